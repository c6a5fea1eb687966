// Decayed linear attention on the tensor cores: 16-bit operands, up to 128 features in a and b, any number in c (in blocks of
// 64 columns).  One CTA walks a segment of one (unit, b, h, column block) in chunks of 128 tokens:
//
//   P   = (a_i . b_j) lambda^(i-j)  for j <= i      S = A B^T in tensor memory; 256 threads weigh, mask and pack it there
//   out = scale * (P C + lambda^(i+1) A X)          X: the state before the chunk, in two 16-bit terms; two accumulators
//   X  <- lambda^128 X + B^T (lambda^(127-j) C)     the weighted C in two 16-bit terms; X itself in fp32 registers
//
// The mirror image in time (n >= t) walks the chunks from the last and mirrors the weights.
//
// Warps: 0-7 weights of P and the outputs, 8-11 weighted C, 12-15 the state, 16 loads and products.  A chunk's product S is
// issued before the chunk before it is finished, and B^T C does not wait for the state: what is serial from chunk to chunk is
// the state's multiply-add, its packing and A X.
//
// Everything that the mask or `lengths` hides is selected away, not multiplied by zero, and rows behind the length are
// cleared in shared memory before a product reads them, so that padding may hold NaN.
#include "decay.h"
#include "launch.h"
#include "tc_common.cuh"
#include "tma_host.h"

namespace flare {

using namespace tc;

namespace {

constexpr int kL = 128;                            // tokens of a chunk
constexpr int kBlk = 128 * 128;                    // bytes of a [128 rows][64] tile

struct DecayMaps {
  CUtensorMap m[4];                                // boxes of [128 tokens][64 features]
  int ia[kDecayUnits], ib[kDecayUnits], ic[kDecayUnits];
};

template <int DK, bool WALK> struct Plan {
  static constexpr int kCB = DK / 64;              // column blocks of a and b
  static constexpr int kStages = WALK && DK == 64 ? 3 : 2;
  static constexpr int kXBuf = DK == 64 ? 2 : 1;   // buffers of the packed state
  static constexpr int kXTile = DK * 128;          // one term of it: [DK][64]
  static constexpr int oA = 0;
  static constexpr int oB = oA + (WALK ? kStages * kCB * kBlk : 0);
  static constexpr int oC = oB + kStages * kCB * kBlk;
  static constexpr int oW = oC + kStages * kBlk;   // weighted C: two terms
  static constexpr int oX = oW + 2 * kBlk;
  static constexpr int oBars = oX + (WALK ? kXBuf * 2 * kXTile : 0);
  static constexpr int kBytes = oBars + 512 + 1024;
  static constexpr int kWarpC = WALK ? 8 : 0, kWarpX = kWarpC + 4, kWarpI = kWarpX + 4;
  static constexpr int kThreads = 32 * (kWarpI + 1);
  static constexpr int kTmem = WALK ? 512 : 64;
  static constexpr int cY = 256, cYx = 320, cKv = WALK ? 384 : 0;      // S of even and odd chunks at 0 and 128
};

__device__ __forceinline__ void arrive_on(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// the hi and lo terms of a pair: lo is what rounding to 16 bits left of each
template <typename T>
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = Op16<T>::pack(x, y);
  const float2 r = Op16<T>::unpack(hi);
  lo = Op16<T>::pack(x - r.x, y - r.y);
}

template <typename T, int DK, bool WALK>
__global__ void __launch_bounds__(Plan<DK, WALK>::kThreads, 1)
k_decay_tc(const __grid_constant__ DecayMaps maps, const __grid_constant__ DecayArgs a, int* status) {
  grid_dep_sync();
  using L = Plan<DK, WALK>;
  constexpr int F = Op16<T>::kFmt, NST = L::kStages, CB = L::kCB;
  constexpr bool kHalfRange = F == 0;              // fp16: the packed state is scaled by a power of two
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::oBars);
  uint64_t *bFullAB = bars, *bFullC = bars + 3, *bS = bars + 6, *bP = bars + 8, *bX = bars + 10, *bYx = bars + 12, *bW = bars + 14,
           *bKv = bars + 15, *bKvFree = bars + 16, *bY = bars + 17, *bYFree = bars + 18;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 20);
  int* abort_flag = reinterpret_cast<int*>(bars + 21);
  float* sExp = reinterpret_cast<float*>(bars + 22);         // 2^e of the packed state, by chunk modulo 4
  uint32_t* sMax = reinterpret_cast<uint32_t*>(bars + 24);   // [2][4]

  const DecayUnit& u = a.u[blockIdx.z];
  const int n_cb = (u.Dc + 63) / 64;
  const int bh = blockIdx.x % (a.B * a.H), cb = blockIdx.x / (a.B * a.H), seg = blockIdx.y;
  if (cb >= n_cb) return;
  const int b = bh / a.H, h = bh % a.H, c0 = 64 * cb;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int live = decay_live(a, b);
  const int n0 = seg * a.seg_len, n1 = min(live, n0 + a.seg_len);
  const int nch = n1 > n0 ? (n1 - n0 + kL - 1) / kL : 0;
  const bool rev = u.rev != 0;
  const float ld = a.log_decay[h], g2 = decay_log2(ld);
  auto first_of = [&](int c) { return n0 + kL * (rev ? nch - 1 - c : c); };      // first token of the c-th chunk in walking order
  auto live_of = [&](int c) { return min(kL, n1 - first_of(c)); };
  const CUtensorMap *mA = &maps.m[maps.ia[blockIdx.z]], *mB = &maps.m[maps.ib[blockIdx.z]], *mC = &maps.m[maps.ic[blockIdx.z]];

  auto load_ab = [&](int c) {
    const int st = c % NST, t0 = first_of(c);
    mbar_expect_tx(bFullAB + st, (WALK ? 2 : 1) * CB * kBlk);
#pragma unroll
    for (int i = 0; i < CB; ++i) {
      if constexpr (WALK) tma_load_4d(smem + L::oA + (st * CB + i) * kBlk, mA, bFullAB + st, 64 * i, t0, h, b);
      tma_load_4d(smem + L::oB + (st * CB + i) * kBlk, mB, bFullAB + st, 64 * i, t0, h, b);
    }
  };
  auto load_c = [&](int c) {
    const int st = c % NST;
    mbar_expect_tx(bFullC + st, kBlk);
    tma_load_4d(smem + L::oC + st * kBlk, mC, bFullC + st, c0, first_of(c), h, b);
  };
  if (tid == 0) {
    for (int i = 0; i < 3; ++i) { mbar_init(bFullAB + i, 1); mbar_init(bFullC + i, 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(bS + i, 1); mbar_init(bP + i, 256); mbar_init(bX + i, 128); mbar_init(bYx + i, 1); }
    mbar_init(bW, 128); mbar_init(bKv, 1); mbar_init(bKvFree, 128); mbar_init(bY, 1); mbar_init(bYFree, 256);
    *abort_flag = 0;
    fence_barrier_init();
    for (int c = 0; c < NST && c < nch; ++c) { load_ab(c); load_c(c); }
  }
  if (warp == 1) tmem_alloc<L::kTmem>(tmem_slot);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // a wait that runs out marks the launch as failed and every later wait returns at once, so that the CTA ends
  auto gave_up = [&] { return *reinterpret_cast<volatile int*>(abort_flag) != 0; };
  auto wait = [&](uint64_t* bar, int parity) { if (!gave_up()) mbar_wait_hot(bar, parity & 1, status, abort_flag); };

  if (warp == L::kWarpI) {
    // ---- loads and products ------------------------------------------------------------------------------------------
    const uint32_t id_s = idesc_f16(128, 128, F, F, 0, 0), id_y = idesc_f16(128, 64, F, F, 0, 1), id_kv = idesc_f16(128, 64, F, F, 1, 1);
    const uint32_t base = smem_u32(smem);
    auto product_s = [&](int c) {
      wait(bFullAB + c % NST, c / NST);
      if (live_of(c) < kL) wait(bW, c);            // rows behind the length are cleared first
      tc_fence_after();
      if (elect_one()) {
        const int st = c % NST;
#pragma unroll
        for (int kk = 0; kk < DK / 16; ++kk) {
          const uint32_t off = (st * CB + kk / 4) * kBlk;
          mma_ss(tmem + 128 * (c & 1), smem_desc<128>(base + L::oA + off) + 2 * (kk & 3), smem_desc<128>(base + L::oB + off) + 2 * (kk & 3), id_s, kk > 0);
        }
        mma_commit(bS + (c & 1));
      }
      __syncwarp();
    };
    if (WALK && nch > 0) product_s(0);
    for (int c = 0; c < nch && !gave_up(); ++c) {
      const int st = c % NST;
      // B^T (weighted C).  For DK = 64 the 128 rows are the 64 features twice (the second block starts where the first does),
      // so that every thread of the state's four warps has half a row to update.
      wait(bFullAB + st, c / NST);
      wait(bW, c);
      if (c > 0) wait(bKvFree, c - 1);
      tc_fence_after();
      if (elect_one()) {
        const uint64_t dB = smem_desc_mn128(base + L::oB + st * CB * kBlk, DK == 128 ? kBlk : 0, 1024);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const uint64_t dW = smem_desc<128>(base + L::oW + t * kBlk);
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) mma_ss(tmem + L::cKv, dB + 128 * kk, dW + 128 * kk, id_kv, t + kk > 0);
        }
        mma_commit(bKv);
      }
      __syncwarp();
      if constexpr (WALK) {
        // c of the chunk before is used up (its product ran ahead of the one just issued).  Before the next S, which may have
        // to wait for that chunk's C.
        if (c > 0 && c - 1 + NST < nch) {
          wait(bY, c - 1);
          if (elect_one()) load_c(c - 1 + NST);
          __syncwarp();
        }
        if (c + 1 < nch) product_s(c + 1);
        wait(bX + (c & 1), c >> 1);
        if (c > 0) wait(bYFree, c - 1);
        tc_fence_after();
        if (elect_one()) {
          const uint32_t x = base + L::oX + (c % L::kXBuf) * 2 * L::kXTile;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const uint64_t dX = smem_desc<128>(x + t * L::kXTile);
#pragma unroll
            for (int kk = 0; kk < DK / 16; ++kk)
              mma_ss(tmem + L::cYx, smem_desc<128>(base + L::oA + (st * CB + kk / 4) * kBlk) + 2 * (kk & 3), dX + 128 * kk, id_y, t + kk > 0);
          }
          mma_commit(bYx + (c & 1));
        }
        __syncwarp();
        if (c + NST < nch) {                       // a and b of this chunk are used up
          wait(bYx + (c & 1), c >> 1);
          if (elect_one()) load_ab(c + NST);
          __syncwarp();
        }
        wait(bP + (c & 1), c >> 1);
        tc_fence_after();
        if (elect_one()) {
          const uint64_t dC = smem_desc<128>(base + L::oC + st * kBlk);
          const uint32_t p = tmem + 128 * (c & 1);
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) mma_ts(tmem + L::cY, p + 8 * (kk & 3) + 64 * (kk >> 2), dC + 128 * kk, id_y, kk > 0);
          mma_commit(bY);
        }
        __syncwarp();
      } else if (c + NST < nch) {
        wait(bKv, c);
        if (elect_one()) { load_ab(c + NST); load_c(c + NST); }
        __syncwarp();
      }
    }
    if (gave_up()) {                               // copies in flight end (within microseconds) before the CTA's memory is given back
      const long long t0 = clock64();
      while (clock64() - t0 < (1LL << 22)) {}
    }
  } else if (warp >= L::kWarpX) {
    // ---- the state -----------------------------------------------------------------------------------------------------
    constexpr int NC = DK == 128 ? 64 : 32;        // columns of a thread
    const int r = tid - 32 * L::kWarpX, d = r & (DK - 1), col = DK == 128 ? 0 : 32 * (r >> 6);
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const long long st_off = (long long)bh * u.Da * u.Dc, seg_off = ((long long)bh * a.n_seg + seg) * u.Da * u.Dc;
    const float* before = nullptr;
    if constexpr (WALK) before = a.n_seg > 1 ? u.seg + seg_off : u.state_in ? u.state_in + st_off : nullptr;
    float X[NC];
#pragma unroll
    for (int j = 0; j < NC; j += 4) {
      float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
      if (before && d < u.Da && c0 + col + j < u.Dc) t = *reinterpret_cast<const float4*>(before + (long long)d * u.Dc + c0 + col + j);
      X[j] = t.x; X[j + 1] = t.y; X[j + 2] = t.z; X[j + 3] = t.w;
    }
    const DecayStep full(ld, kL);
    for (int c = 0; c < nch && !gave_up(); ++c) {
      if constexpr (WALK) {
        float down = 1.f;
        if constexpr (kHalfRange) {
          // the largest magnitude of the tile to 2^13 ... 2^14: X may lie outside fp16's range
          uint32_t top = 0;
#pragma unroll
          for (int j = 0; j < NC; ++j) top = max(top, __float_as_uint(X[j]) & 0x7fffffffu);
          top = __reduce_max_sync(0xffffffffu, top);
          if (lane == 0) sMax[4 * (c & 1) + (warp & 3)] = top;
          asm volatile("bar.sync 1, 128;" ::: "memory");
          const uint4 all = *reinterpret_cast<const uint4*>(sMax + 4 * (c & 1));
          top = max(max(all.x, all.y), max(all.z, all.w));
          const int e = max(-100, min(100, (int)(top >> 23) - 127 - 13));
          down = __uint_as_float((uint32_t)(127 - e) << 23);
          if (r == 0) sExp[c & 3] = __uint_as_float((uint32_t)(127 + e) << 23);
        }
        if (c >= L::kXBuf) wait(bYx + ((c - L::kXBuf) & 1), (c - L::kXBuf) >> 1);
        uint8_t* x = smem + L::oX + (c % L::kXBuf) * 2 * L::kXTile;
#pragma unroll
        for (int j = 0; j < NC; j += 8) {
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) split2<T>(X[j + 2 * i] * down, X[j + 2 * i + 1] * down, hi[i], lo[i]);
          const uint32_t at = swz_off<128>(d, (col + j) / 8);
          *reinterpret_cast<uint4*>(x + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<uint4*>(x + L::kXTile + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        fence_proxy_async();
        arrive_on(bX + (c & 1));
      }
      wait(bKv, c);
      tc_fence_after();
      const int cnt = live_of(c);
      const DecayStep decay = cnt == kL ? full : DecayStep(ld, cnt);
#pragma unroll
      for (int j = 0; j < NC; j += 16) {
        uint32_t v[16];
        tmem_ld16(lane_base + L::cKv + col + j, v);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) X[j + i] = decay(X[j + i]) + __uint_as_float(v[i]);
      }
      tc_fence_before();
      arrive_on(bKvFree);
    }
    float* end = nullptr;
    if constexpr (WALK) end = u.state_out && seg == a.n_seg - 1 ? u.state_out + st_off : nullptr;
    else end = u.seg + seg_off;
    if (end && d < u.Da)
#pragma unroll
      for (int j = 0; j < NC; j += 4)
        if (c0 + col + j < u.Dc) *reinterpret_cast<float4*>(end + (long long)d * u.Dc + c0 + col + j) = make_float4(X[j], X[j + 1], X[j + 2], X[j + 3]);
  } else if (warp >= L::kWarpC) {
    // ---- C weighted by the decay to the chunk's end, in two terms ----------------------------------------------------------
    const int r = tid - 32 * L::kWarpC;
    for (int c = 0; c < nch && !gave_up(); ++c) {
      const int st = c % NST, cnt = live_of(c);
      const float w = exp2f(g2 * (float)(rev ? r : max(0, cnt - 1 - r)));
      wait(bFullC + st, c / NST);
      if (cnt < kL) wait(bFullAB + st, c / NST);
      if (c > 0) wait(bKv, c - 1);                 // the products with the weighted C of the chunk before are done
      uint8_t *src = smem + L::oC + st * kBlk, *hi_t = smem + L::oW, *lo_t = hi_t + kBlk;
      if (r < cnt) {
#pragma unroll
        for (int ch = 0; ch < 8; ++ch) {
          const uint32_t at = swz_off<128>(r, ch);
          const uint4 x = *reinterpret_cast<const uint4*>(src + at);
          uint4 hi, lo;
          const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
          uint32_t hs[4], ls[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = Op16<T>::unpack(xs[i]);
            split2<T>(f.x * w, f.y * w, hs[i], ls[i]);
          }
          hi = make_uint4(hs[0], hs[1], hs[2], hs[3]);
          lo = make_uint4(ls[0], ls[1], ls[2], ls[3]);
          *reinterpret_cast<uint4*>(hi_t + at) = hi;
          *reinterpret_cast<uint4*>(lo_t + at) = lo;
        }
      } else {                                     // behind the length: whatever stands there takes part in no product
        const uint4 z = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int ch = 0; ch < 8; ++ch) {
          const uint32_t at = 128 * r + 16 * ch;
          *reinterpret_cast<uint4*>(src + at) = z;
          *reinterpret_cast<uint4*>(hi_t + at) = z;
          *reinterpret_cast<uint4*>(lo_t + at) = z;
#pragma unroll
          for (int i = 0; i < CB; ++i) *reinterpret_cast<uint4*>(smem + L::oB + (st * CB + i) * kBlk + at) = z;
        }
      }
      fence_proxy_async();
      arrive_on(bW);
    }
  } else if constexpr (WALK) {
    // ---- weights of P, outputs -----------------------------------------------------------------------------------------
    const int r0 = 32 * (warp & 3), r = r0 + lane, hb = warp >> 2;    // token r, half of the columns
    const uint32_t lane_base = tmem + ((uint32_t)r0 << 16);
    // The weights depend on i - j alone, so a thread keeps those of its row for all chunks.
    float w[64];
#pragma unroll
    for (int j = 0; j < 64; ++j) {
      const int dist = rev ? 64 * hb + j - r : r - 64 * hb - j;
      w[j] = dist >= 0 ? exp2f(g2 * (float)dist) : 0.f;
    }
    const float wx = a.scale * exp2f(g2 * (float)(rev ? kL - r : r + 1));
    T* out = static_cast<T*>(u.out) + b * u.os[0] + h * u.os[1] + c0 + 32 * hb;
    const int cols = u.Dc - c0 - 32 * hb;          // of this thread's 32 columns, those that exist

    auto weigh = [&](int c) {
      wait(bS + (c & 1), c >> 1);
      tc_fence_after();
      const int cnt = live_of(c);
      const uint32_t s = lane_base + 128 * (c & 1) + 64 * hb;
      uint32_t v[2][16];
      tmem_ld16(s, v[0]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j0 = 64 * hb + 16 * i;           // the block's first column; the warp's rows are r0 ... r0 + 31
        const bool none = rev ? j0 + 15 < r0 : j0 > r0 + 31, all = (rev ? j0 >= r0 + 31 : j0 + 15 <= r0) && cnt == kL;
        tmem_wait_ld();
        if (i + 1 < 4) tmem_ld16(s + 16 * (i + 1), v[(i + 1) & 1]);
        uint32_t p[8];
        if (none) {
#pragma unroll
          for (int k = 0; k < 8; ++k) p[k] = 0u;
        } else if (all) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            p[k] = Op16<T>::pack(__uint_as_float(v[i & 1][2 * k]) * w[16 * i + 2 * k], __uint_as_float(v[i & 1][2 * k + 1]) * w[16 * i + 2 * k + 1]);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float w0 = w[16 * i + 2 * k], w1 = w[16 * i + 2 * k + 1];
            const float x0 = w0 != 0.f && j0 + 2 * k < cnt ? __uint_as_float(v[i & 1][2 * k]) * w0 : 0.f;
            const float x1 = w1 != 0.f && j0 + 2 * k + 1 < cnt ? __uint_as_float(v[i & 1][2 * k + 1]) * w1 : 0.f;
            p[k] = Op16<T>::pack(x0, x1);
          }
        }
        tmem_st8(s + 8 * i, p);                    // over columns of this thread that are read already
      }
      tmem_wait_st();
      tc_fence_before();
      arrive_on(bP + (c & 1));
    };
    auto store_row = [&](int tok, const uint4 (&o)[4]) {
      T* p = out + (long long)tok * u.os[2];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (8 * i < cols) *reinterpret_cast<uint4*>(p + 8 * i) = o[i];
    };

    if (nch > 0) weigh(0);
    for (int c = 0; c < nch && !gave_up(); ++c) {
      if (c + 1 < nch) weigh(c + 1);
      wait(bY, c);
      tc_fence_after();
      float fx = wx;
      if constexpr (kHalfRange) fx *= sExp[c & 3];
      uint4 o[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t y[16], x[16];
        tmem_ld16(lane_base + L::cY + 32 * hb + 16 * i, y);
        tmem_ld16(lane_base + L::cYx + 32 * hb + 16 * i, x);
        tmem_wait_ld();
        uint32_t q[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
          q[k] = Op16<T>::pack(fmaf(fx, __uint_as_float(x[2 * k]), a.scale * __uint_as_float(y[2 * k])),
                               fmaf(fx, __uint_as_float(x[2 * k + 1]), a.scale * __uint_as_float(y[2 * k + 1])));
        o[2 * i] = make_uint4(q[0], q[1], q[2], q[3]);
        o[2 * i + 1] = make_uint4(q[4], q[5], q[6], q[7]);
      }
      tc_fence_before();
      arrive_on(bYFree);
      const int tok = first_of(c) + r;
      if (tok < n1) store_row(tok, o);
    }
    const uint4 z[4] = {};
    for (int tok = max(n0, live) + (tid & 127); tok < min(a.N, n0 + a.seg_len); tok += 128) {
      T* p = out + (long long)tok * u.os[2];       // rows behind the sequence: zeros
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (8 * i < cols) *reinterpret_cast<uint4*>(p + 8 * i) = z[i];
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc<L::kTmem>(tmem);
}

template <typename T, int DK>
int launch_all(const DecayMaps& maps, const DecayArgs& a, int Dc, cudaStream_t st) {
  using W = Plan<DK, true>;
  using S = Plan<DK, false>;
  int* status = tc_status_ptr();
  if (tc_set_dyn_smem(reinterpret_cast<const void*>(&k_decay_tc<T, DK, true>), W::kBytes) != FLARE_OK ||
      tc_set_dyn_smem(reinterpret_cast<const void*>(&k_decay_tc<T, DK, false>), S::kBytes) != FLARE_OK)
    return FLARE_ECUDA;
  const dim3 grid((unsigned)(a.B * a.H * ((Dc + 63) / 64)), (unsigned)a.n_seg, (unsigned)a.n_units);
  if (a.n_seg > 1) {
    launch_dep(k_decay_tc<T, DK, false>, grid, dim3(S::kThreads), S::kBytes, st, maps, a, status);
    launch_decay_prefix(a, st);
  }
  launch_dep(k_decay_tc<T, DK, true>, grid, dim3(W::kThreads), W::kBytes, st, maps, a, status);
  return FLARE_OK;
}

}  // namespace

bool decay_tc_supported(const DecayArgs& a, int dtype) {
  if (dtype != FLARE_BF16 && dtype != FLARE_F16) return false;
  auto rows = [&](const void* p, const long long (&s)[3], int D) {
    if (D % 8 || reinterpret_cast<uintptr_t>(p) % 16) return false;
    const long long n[3] = {a.B, a.H, a.N};
    for (int i = 0; i < 3; ++i)
      if (n[i] > 1 && (s[i] % 8 || s[i] <= 0 || s[i] >= (1LL << 38))) return false;
    return true;
  };
  for (int i = 0; i < a.n_units; ++i) {
    const DecayUnit& u = a.u[i];
    if (u.Da > 128 || !rows(u.a, u.as, u.Da) || !rows(u.b, u.bs, u.Da) || !rows(u.c, u.cs, u.Dc) || !rows(u.out, u.os, u.Dc)) return false;
    if (reinterpret_cast<uintptr_t>(u.state_in) % 16 || reinterpret_cast<uintptr_t>(u.state_out) % 16) return false;
  }
  return true;
}

// Segments of the token axis: with as many as there are SMs to fill, but a segment of four chunks at least, since every CTA
// has a start-up and the sums of the segments are a pass of their own over b and c.
int decay_tc_segments(int B, int H, int N, int Da, int Dc, int n_units) {
  (void)Da;
  const long long ctas = (long long)B * H * ((Dc + 63) / 64) * n_units;
  long long s = num_sms() / ctas;
  const long long most = ((long long)N + 4 * kL - 1) / (4 * kL);
  if (s > most) s = most;
  if (s > 256) s = 256;
  return s < 1 ? 1 : (int)s;
}

int decay_tc(const DecayArgs& a, int dtype, cudaStream_t st) {
  DecayMaps maps;
  const void* seen[4] = {};
  int n = 0, Da = 0, Dc = 0;
  auto map_of = [&](const void* p, const long long (&s)[3], int D) {
    for (int i = 0; i < n; ++i)
      if (seen[i] == p) return i;
    if (n == 4) return -1;
    // a dimension of one entry has no stride of its own: any valid one
    const uint64_t row = a.N > 1 ? s[2] : D, head = a.H > 1 ? s[1] : row * (uint64_t)a.N, batch = a.B > 1 ? s[0] : head * (uint64_t)a.H;
    if (!make_tile_map_cols(&maps.m[n], p, dtype == FLARE_BF16 ? 1 : 0, D, 64, (uint64_t)a.N, (uint64_t)a.H, (uint64_t)a.B, 2 * row, 2 * head,
                            2 * batch, 128))
      return -1;
    seen[n] = p;
    return n++;
  };
  for (int i = 0; i < a.n_units; ++i) {
    const DecayUnit& u = a.u[i];
    maps.ia[i] = map_of(u.a, u.as, u.Da);
    maps.ib[i] = map_of(u.b, u.bs, u.Da);
    maps.ic[i] = map_of(u.c, u.cs, u.Dc);
    if (maps.ia[i] < 0 || maps.ib[i] < 0 || maps.ic[i] < 0) return FLARE_EUNSUPPORTED;
    Da = u.Da > Da ? u.Da : Da;
    Dc = u.Dc > Dc ? u.Dc : Dc;
  }
  if (dtype == FLARE_BF16) return Da <= 64 ? launch_all<__nv_bfloat16, 64>(maps, a, Dc, st) : launch_all<__nv_bfloat16, 128>(maps, a, Dc, st);
  return Da <= 64 ? launch_all<__half, 64>(maps, a, Dc, st) : launch_all<__half, 128>(maps, a, Dc, st);
}

}  // namespace flare
