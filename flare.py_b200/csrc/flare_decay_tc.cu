// Decayed linear attention on the tensor cores: 16-bit operands, up to 128 features in a and b, any number in c (in blocks of
// 64 columns).  A sequence (one unit, b, h, column block) is taken in chunks of 128 tokens:
//
//   P   = (a_i . b_j) lambda^(i-j)  for j <= i      S = A B^T in tensor memory; 256 threads weigh, mask and pack it there
//   out = scale * (P C + lambda^(i+1) A X)          X: the state before the chunk, in two 16-bit terms; two accumulators
//   X  <- lambda^128 X + B^T (lambda^(127-j) C)     the weighted C in one to three 16-bit terms; X itself in fp32
//
// P and one term of the weighted C are 16-bit numbers, which the products take; the outputs round as much themselves, and are off by
// 1.8 to 2.3e-3 in bf16 where their own rounding alone is 1.7e-3 (fp16 2.5e-4, 2.1e-4).  Where the state is a result, the chunks that
// count in it take two or three terms, or B^T C itself beside two terms of what the weights change (terms_of, near_one).  What is
// rounded to fp16 is first scaled by a power of two: a row of P, the weighted C of a chunk, the packed state.
//
// The mirror image in time (n >= t) walks the chunks from the last and mirrors the weights.
//
// The CTAs of a cluster take the chunks of one sequence in turn.  Everything but X <- ... is theirs alone; X travels from
// CTA to CTA through distributed shared memory (a bulk copy per warp onto the receiver's mbarrier), so what is serial from chunk
// to chunk is one multiply-add of the state and its way to the next SM.  Where even clusters of eight leave SMs idle, the token axis is
// cut into segments as well: k_decay_tc_sums adds up each, k_decay_prefix makes the states before them.
//
// Warps of the walk: 0-7 weights of P, 8-11 weighted C, 12-15 the state, 16-19 outputs, 20 and 21 products, 22 loads.  Everything
// that the mask or `lengths` hides is selected away, not multiplied by zero, and rows behind the length are cleared in shared memory
// before a product reads them, so that padding may hold NaN.
//
// The roles' loops are kept short on purpose: six warps of different roles share a scheduler, and where their loops were unrolled
// they waited for instructions more than for data (152 -> 99 us for 72 sequences of 8192 tokens, D = 128, from that alone).
//
// What bounds it is the way of a chunk through the roles, each a wait: its arrival, the weighted C, B^T C, the state, A X, the
// outputs, and only then its tiles are free.  At B = 4, H = 16, N = 8192, D = 64 bf16 the tensor pipe is busy 30 % of the time,
// the schedulers issue in 47 % of the slots, and HBM moves 3.5 TB/s of the 6.5 that a copy reaches (4.2 with what stays in L2): 64 us
// without a state to return, 82 to 85 with one, 1.8 us a chunk and SM (2.4 with 128 features).
#include <type_traits>
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
  CUtensorMap in[4], out[kDecayUnits];             // boxes of [128 tokens][64 features], of the outputs [32][64]
  int ia[kDecayUnits], ib[kDecayUnits], ic[kDecayUnits];
};

__device__ __forceinline__ void arrive_on(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// A bounded wait, as short in instructions as it can be: the roles of a kernel wait in some thirty places, half of its warps are
// waiting at any time, and what they poll with takes issue slots from those that work.  A try suspends the thread for about a
// hundred clocks; after a second or so of them the wait gives up.
constexpr uint32_t kTries = 1u << 24;
__device__ __forceinline__ bool poll(uint64_t* bar, uint32_t parity) {
  uint32_t tries;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mov.u32 %0, 0;\n"
      "again:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra done;\n\t"
      "add.u32 %0, %0, 1;\n\t"
      "setp.lt.u32 p, %0, %3;\n\t"
      "@p bra again;\n"
      "done:\n\t}"
      : "=&r"(tries) : "r"(smem_u32(bar)), "r"(parity), "n"(kTries) : "memory");
  return tries < kTries;
}
// Whether a phase is over, without waiting for it; the same answer in all lanes of the warp.
__device__ __forceinline__ bool is_over(uint64_t* bar, int parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"(smem_u32(bar)), "r"((uint32_t)parity & 1) : "memory");
  return __all_sync(0xffffffffu, ok != 0);
}
// A thread's waits: once one has run out the others return at once, so that the CTA ends, where the status word gets its bit.
// Warps that meet at a named barrier go through all their chunks all the same.
struct Waits {
  bool dead = false;
  __device__ __forceinline__ void operator()(uint64_t* bar, int parity) {
    if (!dead) dead = !poll(bar, (uint32_t)parity & 1);
  }
  __device__ __forceinline__ void report(int* status) const {
    if (dead && status) atomicOr(status, kErrWaitTimeout);
  }
};
// The wait of a role of several warps: one of them polls, the others sleep at a named barrier.  The polling warps are spread over
// the four schedulers, which the warps' numbers modulo four stand for.
template <int ID, int THREADS>
__device__ __forceinline__ void wait_together(Waits& wait, bool leader, uint64_t* bar, int parity) {
  if (leader) wait(bar, parity);
  asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(THREADS) : "memory");
}
// Position in a ring of N tiles: its index, and the parity of its barrier's phase.
template <int N>
struct Ring {
  int at = 0, phase = 0;
  __device__ __forceinline__ void next() {
    if (++at == N) { at = 0; phase ^= 1; }
  }
};
// A kernel whose waits ran out may have copies in flight: they end (within microseconds) before its memory is given back.
__device__ __forceinline__ void let_copies_end(bool dead) {
  if (!dead) return;
  const long long t0 = clock64();
  while (clock64() - t0 < (1LL << 22)) {}
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t remote(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// bytes of this CTA's shared memory into another's, counted on a barrier over there
__device__ __forceinline__ void copy_to_cta(uint32_t dst, uint32_t src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "r"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, const void* src, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];"
               ::"l"(map), "r"(smem_u32(src)), "r"(c0), "r"(c1), "r"(c2), "r"(c3) : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void tma_prefetch_4d(const CUtensorMap* map, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global [%0, {%1, %2, %3, %4}];" ::"l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3) : "memory");
}
// Two values an instruction.  A pair lives in one 64-bit register from where it is made, so that none is put together twice.
struct F2 {
  uint64_t v;
  __device__ __forceinline__ F2() {}
  __device__ __forceinline__ F2(float x, float y) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y)); }
  __device__ __forceinline__ float2 get() const {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
  }
};
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 floats(uint32_t a, uint32_t b) { return F2(__uint_as_float(a), __uint_as_float(b)); }
// one value twice; volatile, so that it is made where it stands and not again at every use
__device__ __forceinline__ F2 both(float x) {
  F2 r;
  asm volatile("mov.b64 %0, {%1, %1};" : "=l"(r.v) : "f"(x));
  return r;
}
template <typename T> __device__ __forceinline__ F2 unpack2(uint32_t w) {
  const float2 f = Op16<T>::unpack(w);
  return F2(f.x, f.y);
}
template <typename T> __device__ __forceinline__ uint32_t pack2(F2 x) {
  const float2 f = x.get();
  return Op16<T>::pack(f.x, f.y);
}
// the hi and lo terms of a pair: lo is what rounding to 16 bits left of each
template <typename T>
__device__ __forceinline__ void split2(F2 x, F2 minus_one, uint32_t& hi, uint32_t& lo) {
  hi = pack2<T>(x);
  lo = pack2<T>(fma2(unpack2<T>(hi), minus_one, x));
}

// What a chunk is to the CTA that takes it.
struct Span {
  int n0, n1, nch, end;                            // live tokens of the segment, its chunks; live tokens of the sequence
  bool rev;
  __device__ __forceinline__ Span(const DecayArgs& a, int live, int seg, bool reverse) : end(live), rev(reverse) {
    n0 = seg * a.seg_len;
    n1 = min(live, n0 + a.seg_len);
    nch = n1 > n0 ? (n1 - n0 + kL - 1) / kL : 0;
  }
  __device__ __forceinline__ int first(int c) const { return n0 + kL * (rev ? nch - 1 - c : c); }   // of the c-th chunk walked
  __device__ __forceinline__ int live(int c) const { return min(kL, n1 - first(c)); }
  __device__ __forceinline__ int behind(int c) const { return end - first(c) - live(c); }             // live tokens after it
};

// 16-bit terms of a chunk's weighted C.  A chunk counts in the state behind the sequence by the decay over the tokens after it.
// One, two and three bf16 terms leave 2e-3, 3e-6 and 4e-9 of a chunk (fp16: 2e-4, 4e-8): with these borders the state is right
// to 4e-7, as sums in 32 bits are.  Without a state (training) every chunk takes one.
template <typename T>
__device__ __forceinline__ int terms_of(float g2, int behind) {
  const float x = g2 * (float)behind;
  return x > -3.f ? (Op16<T>::kFmt == 1 ? 3 : 2) : x > -13.f ? 2 : 1;
}
// Where the decay over a chunk is small, B^T C itself, which needs no rounding, is taken beside two terms of (weight - 1) C: those
// leave 3e-6 of the 0.24 or less that the weights differ from 1 by.  The third term's second turn at the tiles is spared where
// it would come most often, in heads of long memory.
template <typename T>
__device__ __forceinline__ bool near_one(float g2) { return Op16<T>::kFmt == 1 && fabsf(g2) <= 0.4f / kL; }

// fp16: what is rounded to it is first taken, by a power of two, to where its largest magnitude is 2^13 to 2^14.  The type ends at
// 2^-24 below and at 65504 above: unscaled, values of size 1e-3 would keep 5e-5 of a state and of size 1e-5 3e-3 of a gradient.
// Scaling the weighted C and the rows of P costs fp16 calls 80 -> 94 us for the prompt above, 176 -> 199 for its backward, 135 -> 150
// for that of B = 8, H = 8, N = 2048, 128/32, nothing for one document of 65536 tokens.
__device__ __forceinline__ int exponent_of(uint32_t top) { return max(-100, min(100, (int)(top >> 23) - 127 - 13)); }
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
// The largest magnitude among the pieces of a row, weighted, as its bits.  Values that are not finite have no say in it: they may
// stand in a column of their own.
__device__ __forceinline__ uint32_t top_of_row(int r, int p0, int pieces, float w, const uint8_t* src) {
  const uint32_t row = 128 * r + 16 * (r & 7);
  uint32_t m = 0;
#pragma unroll 4
  for (int ch = p0; ch < p0 + pieces; ++ch) {
    const uint4 x = *reinterpret_cast<const uint4*>(src + (row ^ (16 * ch)));
    m = __vmaxu2(m, __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu), __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu)));
  }
  constexpr uint32_t kInf = 0x7c00u;
  if (max(m & 0xffffu, m >> 16) >= kInf) {
    m = 0;
#pragma unroll 1
    for (int i = 8 * p0; i < 8 * (p0 + pieces); ++i) {
      const uint32_t x = *reinterpret_cast<const uint16_t*>(src + (row ^ (16 * (i >> 3))) + 2 * (i & 7)) & 0x7fffu;
      m = max(m, x < kInf ? x : 0u);
    }
  }
  return __float_as_uint(__half2float(__ushort_as_half((unsigned short)max(m & 0xffffu, m >> 16))) * w);
}

// C weighted by the decay to the chunk's end; a thread takes PIECES of the 16-byte pieces of a row, and of those the first `pieces`
// hold columns.  `which` of its terms are written, bit by bit: 1, 2 and 4 for the first, second and third, to w_t and the tiles
// behind it, but the third alone to w_t.  Rows behind the length are cleared, here and in the tiles of b and c themselves.
template <typename T, int CB, int PIECES = 8>
__device__ __forceinline__ void weigh_c(int r, int p0, int pieces, int cnt, float w, int which, uint8_t* src, uint8_t* w_t, uint8_t* b_t) {
  const uint32_t row = 128 * r + 16 * (r & 7);     // 16-byte piece ch of the swizzled row: row ^ 16 ch
  const F2 w2 = both(w);
  if (r >= cnt) {
    const uint4 z = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 1
    for (int ch = p0; ch < p0 + PIECES; ++ch) {
      const uint32_t at = row ^ (16 * ch);
      *reinterpret_cast<uint4*>(w_t + at) = z;
      if (which & 2) *reinterpret_cast<uint4*>(w_t + kBlk + at) = z;
      if (which == 7) *reinterpret_cast<uint4*>(w_t + 2 * kBlk + at) = z;
      if (which == 4) continue;                    // they are clear, and products may be reading them
      *reinterpret_cast<uint4*>(src + at) = z;
#pragma unroll
      for (int i = 0; i < CB; ++i) *reinterpret_cast<uint4*>(b_t + i * kBlk + at) = z;
    }
  } else if (which == 1) {
    auto weighed = [&](uint32_t x) { return pack2<T>(mul2(unpack2<T>(x), w2)); };
#pragma unroll 4
    for (int ch = p0; ch < p0 + pieces; ++ch) {
      const uint32_t at = row ^ (16 * ch);
      const uint4 x = *reinterpret_cast<const uint4*>(src + at);
      *reinterpret_cast<uint4*>(w_t + at) = make_uint4(weighed(x.x), weighed(x.y), weighed(x.z), weighed(x.w));
    }
  } else {
    const F2 minus_one = both(-1.f);
    uint8_t* third = w_t + (which == 7 ? 2 * kBlk : 0);
#pragma unroll 2
    for (int ch = p0; ch < p0 + pieces; ++ch) {
      const uint32_t at = row ^ (16 * ch);
      const uint4 x = *reinterpret_cast<const uint4*>(src + at);
      uint4 t0, t1;
      F2 rest[4];                                  // what the first term leaves
      auto split = [&](uint32_t v, uint32_t& a0, uint32_t& a1, F2& left) {
        const F2 y = mul2(unpack2<T>(v), w2);
        a0 = pack2<T>(y);
        left = fma2(unpack2<T>(a0), minus_one, y);
        a1 = pack2<T>(left);
      };
      split(x.x, t0.x, t1.x, rest[0]);
      split(x.y, t0.y, t1.y, rest[1]);
      split(x.z, t0.z, t1.z, rest[2]);
      split(x.w, t0.w, t1.w, rest[3]);
      if (which & 1) *reinterpret_cast<uint4*>(w_t + at) = t0;
      if (which & 2) *reinterpret_cast<uint4*>(w_t + kBlk + at) = t1;
      if (which & 4) {
        auto third_of = [&](uint32_t a1, F2 left) { return pack2<T>(fma2(unpack2<T>(a1), minus_one, left)); };
        *reinterpret_cast<uint4*>(third + at) = make_uint4(third_of(t1.x, rest[0]), third_of(t1.y, rest[1]), third_of(t1.z, rest[2]), third_of(t1.w, rest[3]));
      }
    }
  }
  fence_proxy_async();
}

// B^T (first term | second term): 128 x 128, or B^T times one tile: 128 x 64.  For 64 features the 128 rows are the features twice
// (the second block of the operand starts where the first does), so that each of the state's 128 threads has half a row to update.
template <int DK, int F>
__device__ __forceinline__ void product_kv(uint32_t d, uint32_t b_tile, uint32_t w_tile, bool two, bool add) {
  const uint64_t dB = smem_desc_mn128(b_tile, DK == 128 ? kBlk : 0, 1024), dW = smem_desc_mn128(w_tile, kBlk, 1024);
  const uint32_t id = two ? idesc_f16(128, 128, F, F, 1, 1) : idesc_f16(128, 64, F, F, 1, 1);
#pragma unroll 2
  for (int kk = 0; kk < 8; ++kk) mma_ss(d, dB + 128 * kk, dW + 128 * kk, id, add || kk > 0);
}

// ---- the sums of the segments ----------------------------------------------------------------------------------------------
// Warps 0-7 weighted C, 8-11 the sum (in registers), 12 products, 13 loads.
template <int DK> struct SumPlan {
  static constexpr int kCB = DK / 64, kStages = DK == 64 ? 3 : 2;
  static constexpr int oB = 0, oC = kStages * kCB * kBlk, oW = oC + kStages * kBlk, oBars = oW + 6 * kBlk, kBytes = oBars + 256 + 1024;
  static constexpr int kThreads = 448;
};

template <typename T, int DK>
__global__ void __launch_bounds__(SumPlan<DK>::kThreads, 1)
k_decay_tc_sums(const __grid_constant__ DecayMaps maps, const __grid_constant__ DecayArgs a, int* status) {
  grid_dep_sync();
  using L = SumPlan<DK>;
  constexpr int F = Op16<T>::kFmt, NST = L::kStages, CB = L::kCB;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023);   // by an offset: the compiler keeps to shared-memory instructions
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::oBars);
  uint64_t *bFull = bars, *bFree = bars + 3, *bW = bars + 6, *bKv = bars + 8, *bKvFree = bars + 10;      // bW, bKv, bKvFree: two buffers each
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 12);
  uint32_t* sTop = reinterpret_cast<uint32_t*>(bars + 14);   // [8], fp16: the weighing warps' largest magnitudes
  float* sUnit = reinterpret_cast<float*>(bars + 18);        // and what the weighted C of a chunk was divided by, by chunk modulo 4
  constexpr bool kHalfRange = F == 0;
  const DecayUnit& u = a.u[blockIdx.z];
  const int n_cb = (u.Dc + 63) / 64;
  const int bh = blockIdx.x % (a.B * a.H), cb = blockIdx.x / (a.B * a.H), seg = u.rev ? blockIdx.y + 1 : blockIdx.y;
  if (cb >= n_cb) return;
  const int b = bh / a.H, h = bh % a.H, c0 = 64 * cb, tid = threadIdx.x, warp = tid >> 5;
  const float ld = a.log_decay[h], g2 = decay_log2(ld);
  const Span sp(a, decay_live(a, b), seg, u.rev != 0);
  const bool plus = near_one<T>(g2);               // two terms are those beside C itself
  auto terms = [&](int c) {
    const int t = u.state_out ? terms_of<T>(g2, sp.behind(c)) : 1;
    return plus ? min(t, 2) : t;
  };
  auto load = [&](int c, int st) {
    const int t0 = sp.first(c);
    mbar_expect_tx(bFull + st, (CB + 1) * kBlk);
#pragma unroll
    for (int i = 0; i < CB; ++i) tma_load_4d(smem + L::oB + (st * CB + i) * kBlk, &maps.in[maps.ib[blockIdx.z]], bFull + st, 64 * i, t0, h, b);
    tma_load_4d(smem + L::oC + st * kBlk, &maps.in[maps.ic[blockIdx.z]], bFull + st, c0, t0, h, b);
  };
  if (tid == 0) {
    for (int i = 0; i < NST; ++i) { mbar_init(bFull + i, 1); mbar_init(bFree + i, 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(bW + i, 256); mbar_init(bKv + i, 1); mbar_init(bKvFree + i, 128); }
    fence_barrier_init();
    for (int c = 0; c < NST && c < sp.nch; ++c) load(c, c);
  }
  if (warp == 1) tmem_alloc<256>(tmem_slot);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  Waits wait;
  Ring<NST> ring;
  if (warp == 13) {
    const int nch = __reduce_max_sync(0xffffffffu, sp.nch);
    for (int c = 0; c + NST < nch && !wait.dead; ++c) {
      wait(bFree + ring.at, ring.phase);
      if (elect_one()) load(c + NST, ring.at);
      __syncwarp();
      ring.next();
    }
    let_copies_end(wait.dead);
  } else if (warp == 12) {
    const int nch = __reduce_max_sync(0xffffffffu, sp.nch);
    const uint32_t tm = __reduce_max_sync(0xffffffffu, tmem), base = smem_u32(smem);
    for (int c = 0; c < nch && !wait.dead; ++c) {
      wait(bW + (c & 1), c >> 1);
      if (c > 1) wait(bKvFree + (c & 1), (c - 2) >> 1);
      tc_fence_after();
      if (elect_one()) {
        const uint32_t b_at = base + L::oB + ring.at * (CB * kBlk), w_at = base + L::oW + (c & 1) * (3 * kBlk), kv = tm + 128 * (c & 1);
        const int t = terms(c);
        product_kv<DK, F>(kv, b_at, w_at, t > 1, false);
        if (t == 3) product_kv<DK, F>(kv + 64, b_at, w_at + 2 * kBlk, false, true);
        if (t == 2 && plus) product_kv<DK, F>(kv, b_at, base + L::oC + ring.at * kBlk, false, true);
        mma_commit(bKv + (c & 1));
        mma_commit(bFree + ring.at);
      }
      __syncwarp();
      ring.next();
    }
  } else if (warp >= 8) {
    constexpr int NC = DK == 128 ? 64 : 32;        // columns of a thread
    const int r = tid - 256, d = r & (DK - 1), col = DK == 128 ? 0 : 32 * (r >> 6);
    const uint32_t kv = tmem + ((uint32_t)((warp & 3) * 32) << 16) + col;
    float X[NC];
#pragma unroll
    for (int j = 0; j < NC; ++j) X[j] = 0.f;
    const DecayStep full(ld, kL);
    for (int c = 0; c < sp.nch; ++c) {
      const int cnt = sp.live(c);
      const DecayStep decay = cnt == kL ? full : DecayStep(ld, cnt);
      const bool more = terms(c) > 1;
      wait_together<2, 128>(wait, warp == 8, bKv + (c & 1), c >> 1);
      tc_fence_after();
      const float unit = kHalfRange ? sUnit[c & 3] : 1.f;
#pragma unroll
      for (int j = 0; j < NC; j += 16) {
        uint32_t v[16], lo[16];
        tmem_ld16(kv + 128 * (c & 1) + j, v);
        if (more) {
          tmem_ld16(kv + 128 * (c & 1) + 64 + j, lo);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) lo[i] = 0u;
        }
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float x = __uint_as_float(v[i]) + __uint_as_float(lo[i]);
          X[j + i] = decay(X[j + i]) + (kHalfRange ? x * unit : x);
        }
      }
      tc_fence_before();
      arrive_on(bKvFree + (c & 1));
    }
    float* end = u.seg + ((long long)bh * a.n_seg + seg) * u.Da * u.Dc + (long long)d * u.Dc + c0 + col;
    if (d < u.Da)
#pragma unroll
      for (int j = 0; j < NC; j += 4)
        if (c0 + col + j < u.Dc) *reinterpret_cast<float4*>(end + j) = make_float4(X[j], X[j + 1], X[j + 2], X[j + 3]);
  } else {
    const int r = tid & 127, half = tid >> 7;      // row, half of its pieces
    for (int c = 0; c < sp.nch; ++c) {
      const int cnt = sp.live(c);
      float w = exp2f(g2 * (float)(sp.rev ? r : max(0, cnt - 1 - r)));
      if (warp == 1) wait(bFull + ring.at, ring.phase);
      if constexpr (kHalfRange) {
        asm volatile("bar.sync 1, 256;" ::: "memory");
        const uint32_t own = r < cnt ? top_of_row(r, 4 * half, 4, w, smem + L::oC + ring.at * kBlk) : 0u;
        const uint32_t top = __reduce_max_sync(0xffffffffu, own);
        if ((tid & 31) == 0) sTop[warp] = top;
        if (own == 0) w = 0.f;                     // zeros weigh nothing: under growth w times the power of two might overflow
      }
      if (warp == 1 && c > 1) wait(bKv + (c & 1), (c - 2) >> 1);       // the product with what stood here is done
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if constexpr (kHalfRange) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, sTop[i]);
        const int e = exponent_of(top);
        if (tid == 0) sUnit[c & 3] = power_of_two(e);        // the sum of chunk c - 4 has read what stood here: its product is behind
        w *= power_of_two(-e);
      }
      const int t = terms(c);
      weigh_c<T, CB, 4>(r, 4 * half, 4, cnt, t == 2 && plus ? w - 1.f : w, (1 << t) - 1, smem + L::oC + ring.at * kBlk, smem + L::oW + (c & 1) * (3 * kBlk),
                        smem + L::oB + ring.at * (CB * kBlk));
      arrive_on(bW + (c & 1));
      ring.next();
    }
  }
  wait.report(status);
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc<256>(tmem);
}

// ---- the walk --------------------------------------------------------------------------------------------------------------
template <int DK> struct WalkPlan {
  static constexpr int kCB = DK / 64;
  // Tiles in flight: three chunks of 64 features; of 128 features two, and one of b, which is free as soon as S and B^T C have
  // been formed.
  static constexpr int kA = DK == 64 ? 3 : 2, kB = DK == 64 ? 3 : 1, kC = DK == 64 ? 3 : 2;
  static constexpr int kW = 2;                     // tiles for the weighted C: two terms at a time, or two chunks of one
  static constexpr bool kStage = DK == 64;         // outputs leave through shared memory and the TMA
  static constexpr int kXTile = DK * 128;          // one term of the packed state: [DK][64]
  static constexpr int kXPart = 16 + DK * 64;      // a warp's quarter of the state in fp32, as it arrives, behind its largest magnitude
  static constexpr int oA = 0, oB = oA + kA * kCB * kBlk, oC = oB + kB * kCB * kBlk, oW = oC + kC * kBlk, oX = oW + kW * kBlk,
                       oOut = oX + 2 * kXTile, oIn = oOut + (kStage ? kBlk : 0), oBars = oIn + 4 * kXPart, oRows = oBars + 512;
  static constexpr int kBytes = oRows + 6 * 128 + 1024;
  static constexpr int kWarpC = 8, kWarpX = 12, kWarpY = 16, kWarpI = 20, kThreads = 32 * (kWarpI + 3);
  static constexpr int cY = 256, cYx = 320, cKv = 384;       // tensor memory: S of even and odd chunks at 0 and 128
};

template <typename T, int DK, bool STATE>
__global__ void __launch_bounds__(WalkPlan<DK>::kThreads, 1)
k_decay_tc_walk(const __grid_constant__ DecayMaps maps, const __grid_constant__ DecayArgs a, int first, int per_unit, int* status) {
  grid_dep_sync();
  using L = WalkPlan<DK>;
  constexpr int F = Op16<T>::kFmt, CB = L::kCB;
  constexpr bool kHalfRange = F == 0;              // fp16: the packed state is scaled by a power of two, the scale is applied last
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023);   // by an offset: the compiler keeps to shared-memory instructions
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::oBars);
  // bFree: a chunk's outputs are complete, and with them everything that read its tiles.  bFreeB: a single tile of b is free
  // earlier.  bIn: one a warp of the state.
  uint64_t *bFull = bars, *bFullC = bars + 3, *bFree = bars + 6, *bFreeB = bars + 9, *bS = bars + 10, *bP = bars + 12, *bX = bars + 14, *bW = bars + 16,
           *bEv = bars + 18, *bYx = bars + 20, *bKvFree = bars + 21, *bYFree = bars + 22, *bIn = bars + 23;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 27);
  float* sExp = reinterpret_cast<float*>(bars + 28);         // 2^e of the packed state, by chunk modulo 4
  uint32_t* sMax = reinterpret_cast<uint32_t*>(bars + 30);   // [2][4], fp16 of 64 features
  // Rows behind the length are cleared, in the one chunk of a segment that has them.  S waits for that on a barrier of its own: on
  // bW, whose other phases it does not follow, a phase could go by unseen (the wait would then run out) or be taken for the last.
  uint64_t* bClear = bars + 34;
  uint32_t* sTop = reinterpret_cast<uint32_t*>(bars + 36);   // [4], fp16: the weighing warps' largest magnitudes
  float* sUnit = reinterpret_cast<float*>(bars + 38);        // and what the weighted C was divided by, by chunk modulo 4
  uint8_t* sRow = smem + L::oRows;                           // [2][128], fp16: the exponent of the largest P of a row's halves
  int8_t* sPow = reinterpret_cast<int8_t*>(sRow + 256);      // [4][128]: P of a row was divided by 2^this, by chunk modulo 4

  const int size = cluster_size(), rank = cluster_rank(), job = first + blockIdx.x / size;
  const int unit = __reduce_max_sync(0xffffffffu, job / per_unit);       // in a uniform register: it indexes the arguments
  const DecayUnit& u = a.u[unit];
  const int n_cb = (u.Dc + 63) / 64, sequence = job - unit * per_unit, bh = sequence % (a.B * a.H), cb = sequence / (a.B * a.H), seg = blockIdx.y;
  if (cb >= n_cb) return;                          // the whole cluster alike
  const int b = bh / a.H, h = bh % a.H, c0 = 64 * cb;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // Columns that exist: with 128 features the roles leave the others out (half of the state's step where Dv is 32), and what is in
  // them is never stored.  With 64 the state's threads take all theirs at once.
  const int width = DK == 128 ? min(64, u.Dc - c0) : 64;
  const int part = DK == 128 ? 16 + 128 * width : L::kXPart;           // bytes of the state that a warp sends
  const int live = decay_live(a, b);
  const bool rev = u.rev != 0;
  const Span sp(a, live, seg, rev);
  const int mine = (sp.nch - rank + size - 1) / size;        // chunks rank, rank + size, ... are this CTA's: 0, 1, ... below
  const float ld = a.log_decay[h], g2 = decay_log2(ld);
  auto chunk = [&](int i) { return rank + size * i; };
  // The weighted C comes in events e = 0, 1, ...: a chunk of one term is one, in the tiles in turn; two terms are one in both
  // tiles; a third is another, in the first tile.
  const bool plus = STATE && near_one<T>(g2);      // two terms are those beside C itself
  auto terms = [&](int i) {
    const int t = STATE ? terms_of<T>(g2, sp.behind(chunk(i))) : 1;
    return plus ? min(t, 2) : t;
  };

  // a and b of a chunk land on one barrier, c on its own; `at` is the tile in its ring
  auto load = [&](uint8_t* tiles, uint64_t* full, int which, int blocks, int col, int i) {
    for (int k = 0; k < blocks; ++k) tma_load_4d(tiles + k * kBlk, &maps.in[which], full, col + 64 * k, sp.first(chunk(i)), h, b);
  };
  auto load_a = [&](int i, int at) { load(smem + L::oA + at * (CB * kBlk), bFull + at, maps.ia[unit], CB, 0, i); };
  auto load_b = [&](int i, int at, int at_a) {
    mbar_expect_tx(bFull + at_a, 2 * CB * kBlk);
    load(smem + L::oB + at * (CB * kBlk), bFull + at_a, maps.ib[unit], CB, 0, i);
  };
  auto load_c = [&](int i, int at) {
    mbar_expect_tx(bFullC + at, kBlk);
    load(smem + L::oC + at * kBlk, bFullC + at, maps.ic[unit], 1, c0, i);
  };
  if (tid == 0) {
    for (int i = 0; i < 3; ++i) { mbar_init(bFull + i, 1); mbar_init(bFullC + i, 1); mbar_init(bFree + i, 2); }     // bFree: A X and P C
    for (int i = 0; i < 2; ++i) { mbar_init(bS + i, 1); mbar_init(bP + i, 256); mbar_init(bX + i, 128); mbar_init(bW + i, 128); mbar_init(bEv + i, 1); }
    mbar_init(bFreeB, 2); mbar_init(bClear, 128); mbar_init(bYx, 1); mbar_init(bKvFree, 128); mbar_init(bYFree, 128);
    for (int i = 0; i < 4; ++i) mbar_init(bIn + i, 1);
    fence_barrier_init();
    for (int i = 0; i < mine; ++i) {
      if (i < L::kC) load_c(i, i);
      if (i < L::kB) load_b(i, i, i);
      if (i < L::kA) load_a(i, i);
      if (i >= 2) break;
    }
    if (size > 1 && mine > (rank == 0 ? 1 : 0))                           // the first state that comes from another CTA
      for (int i = 0; i < 4; ++i) mbar_expect_tx(bIn + i, part);
  }
  if (warp == 1) tmem_alloc<512>(tmem_slot);
  if (L::kStage && tid == 64) prefetch_tmap(&maps.out[unit]);
  tc_fence_before();
  cluster_sync();                                  // every CTA's barriers stand before a state is sent
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  Waits wait;

  if (warp >= L::kWarpI) {
    // counts and addresses through a warp reduction: the compiler then keeps them, and the descriptors, in uniform registers
    const int n = __reduce_max_sync(0xffffffffu, mine);
    const uint32_t tm = __reduce_max_sync(0xffffffffu, tmem), base = smem_u32(smem);
    constexpr uint32_t id_s = idesc_f16(128, 128, F, F, 0, 0), id_y = idesc_f16(128, 64, F, F, 0, 1);
    auto tile_a = [&](int at) { return smem_desc<128>(base + L::oA + at * (CB * kBlk)); };
    Ring<L::kA> ra;
    Ring<L::kB> rb;
    Ring<L::kC> rc;
    if (warp == L::kWarpI) {
      // ---- S = A B^T and P C -------------------------------------------------------------------------------------------
      auto product_s = [&](int i) {
        wait(bFull + ra.at, ra.phase);
        if (sp.live(chunk(i)) < kL) wait(bClear, 0);
        tc_fence_after();
        if (elect_one()) {
          const uint64_t dA = tile_a(ra.at), dB = smem_desc<128>(base + L::oB + rb.at * (CB * kBlk));
          const uint32_t d = tm + 128 * (i & 1);
#pragma unroll 1
          for (int blk = 0; blk < CB; ++blk)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) mma_ss(d, dA + blk * (kBlk >> 4) + 2 * kk, dB + blk * (kBlk >> 4) + 2 * kk, id_s, blk + kk > 0);
          mma_commit(bS + (i & 1));
          if (L::kB == 1) mma_commit(bFreeB);
        }
        __syncwarp();
        ra.next();
        rb.next();
      };
      constexpr int kAhead = L::kB > 1 ? 1 : 0;    // S comes a chunk ahead of P C where there are tiles for it
      for (int j = 0; j < n + kAhead && !wait.dead; ++j) {
        if (j < n) product_s(j);
        const int i = j - kAhead;
        if (i < 0) continue;
        wait(bFullC + rc.at, rc.phase);            // the weighing warps' wait for c orders only what comes behind their event
        wait(bP + (i & 1), i >> 1);
        if (i > 0) wait(bYFree, i - 1);
        tc_fence_after();
        if (elect_one()) {
          const uint64_t dC = smem_desc<128>(base + L::oC + rc.at * kBlk);
          const uint32_t p = tm + 128 * (i & 1);
#pragma unroll 1
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) mma_ts(tm + L::cY, p + 64 * half + 8 * kk, dC + 512 * half + 128 * kk, id_y, half + kk > 0);
          mma_commit(bFree + rc.at);
        }
        __syncwarp();
        rc.next();
      }
    } else if (warp == L::kWarpI + 1) {
      // ---- B^T C, a chunk ahead where its operands are there, and A X ----------------------------------------------------
      Ring<L::kA> rf;                              // of the operands' barriers, a chunk ahead of ra
      int ev = 0;
      auto product_bc = [&](int i) {
        wait(bFull + rf.at, rf.phase);
        wait(bW + (ev & 1), ev >> 1);
        if (i > 0) wait(bKvFree, i - 1);
        tc_fence_after();
        const int t = terms(i);
        const uint32_t b_at = base + L::oB + rb.at * (CB * kBlk);
        // one product; of two terms and C itself two; of three the first two, and the third by itself when its tile is there
        const int last = t == 3 || (plus && t == 2);
        for (int pass = 0;; ++pass) {
          const uint32_t tile = base + (pass && plus ? L::oC + rf.at * kBlk : L::oW + (t == 1 ? (ev & 1) * kBlk : 0));
          if (elect_one()) {
            product_kv<DK, F>(tm + L::cKv + (pass && !plus ? 64 : 0), b_at, tile, t > 1 && pass == 0, pass > 0);
            if (t == 3 || pass == last) mma_commit(bEv + (ev & 1));
          }
          __syncwarp();
          if (pass == last) break;
          if (t == 3) {
            ++ev;
            wait(bW + (ev & 1), ev >> 1);
            tc_fence_after();
          }
        }
        if (L::kB == 1 && elect_one()) mma_commit(bFreeB);
        __syncwarp();
        ++ev;
        rf.next();
        rb.next();
      };
      for (int i = 0, j = 0; i < n && !wait.dead;) {         // B^T C of chunk j, at most one ahead, or A X of chunk i
        // With two tiles of c the next one's weights may be late: A X does not wait for them then (218 -> 197 us at B = 9,
        // H = 8, N = 8192, D = 128; with three tiles it is better to wait, 126 against 135 us at H = 16, D = 64).
        if (j < n && (j == i || (j == i + 1 && (L::kB > 1 || is_over(bW + (ev & 1), ev >> 1))))) {
          product_bc(j++);
          continue;
        }
        wait(bX + (i & 1), i >> 1);
        if (i > 0) wait(bYFree, i - 1);
        tc_fence_after();
        if (elect_one()) {
          const uint64_t dA = tile_a(ra.at), dX = smem_desc<128>(base + L::oX);
#pragma unroll 1
          for (int blk = 0; blk < 2 * CB; ++blk)   // the blocks of 64 features for the first term, then for the second
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_ss(tm + L::cYx, dA + (blk & (CB - 1)) * (kBlk >> 4) + 2 * kk, dX + 512 * blk + 128 * kk, id_y, blk + kk > 0);
          mma_commit(bYx);
          mma_commit(bFree + ra.at);
        }
        __syncwarp();
        ra.next();
        ++i;
      }
    } else {
      // ---- loads: tiles are refilled when the chunk's products have completed ---------------------------------------------
      static_assert(L::kA == L::kC, "one ring");
      for (int i = 0; i < n && !wait.dead; ++i) {
        if (L::kB == 1 && i + 1 < n) {
          wait(bFreeB, i);
          if (elect_one()) {
            load_b(i + 1, 0, (i + 1) % L::kA);
            if (i + 3 < n) {                       // with so few tiles their way is waited for: it starts in L2
              const int t0 = sp.first(chunk(i + 3));
              for (int k = 0; k < CB; ++k) {
                tma_prefetch_4d(&maps.in[maps.ib[unit]], 64 * k, t0, h, b);
                tma_prefetch_4d(&maps.in[maps.ia[unit]], 64 * k, t0, h, b);
              }
              tma_prefetch_4d(&maps.in[maps.ic[unit]], c0, t0, h, b);
            }
          }
          __syncwarp();
        }
        if (i + L::kA < n) {
          wait(bFree + ra.at, ra.phase);
          if (elect_one()) {
            load_c(i + L::kA, ra.at);              // c first: its weighting starts the chunk's longest chain
            if (L::kB > 1) load_b(i + L::kA, ra.at, ra.at);
            load_a(i + L::kA, ra.at);
          }
          __syncwarp();
          ra.next();
        }
      }
      let_copies_end(wait.dead);
    }
  } else if (warp >= L::kWarpY) {
    // ---- outputs -------------------------------------------------------------------------------------------------------
    const int w = warp & 3, r = 32 * w + lane;     // token
    const uint32_t y_at = tmem + ((uint32_t)(32 * w) << 16) + L::cY, x_at = y_at + (L::cYx - L::cY);
    const float wx_full = a.scale * exp2f(g2 * (float)(rev ? kL - r : r + 1));
    T* out = static_cast<T*>(u.out) + b * u.os[0] + h * u.os[1] + c0;
    const int cols = u.Dc - c0;                    // of the 64 columns, those that exist
    uint8_t* tile = smem + L::oOut + w * 4096;     // the warp's [32 rows][64], swizzled: piece k of a row at row ^ 16 k
    const uint32_t row = 128 * lane + 16 * (lane & 7);
    Ring<L::kA> ra;
    for (int i = 0; i < mine; ++i) {
      const int c = chunk(i), cnt = sp.live(c), tok0 = sp.first(c);
      if constexpr (L::kStage) {                   // the tile of the chunk before has left shared memory
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
      }
      wait_together<5, 128>(wait, w == 0, bFree + ra.at, ra.phase);
      ra.next();
      tc_fence_after();
      // of a mirrored chunk that ends early: by the tokens there are, so that growth (log_decay above 0) stays in range
      const float wx = rev && cnt < kL ? a.scale * exp2f(g2 * (float)max(0, cnt - r)) : wx_full;
      const F2 fx = both(kHalfRange ? wx * sExp[i & 3] : wx), scale2 = both(kHalfRange ? a.scale * power_of_two(sPow[128 * (i & 3) + r]) : 1.f);
      uint32_t y[16], x[16];
      tmem_ld16(y_at, y);
      tmem_ld16(x_at, x);
#pragma unroll 1
      for (int k = 0; 16 * k < width; ++k) {
        uint32_t q[8];
        tmem_wait_ld();
#pragma unroll
        for (int m = 0; m < 8; ++m) {
          F2 in_chunk = floats(y[2 * m], y[2 * m + 1]);
          if constexpr (kHalfRange) in_chunk = mul2(scale2, in_chunk);
          q[m] = pack2<T>(fma2(fx, floats(x[2 * m], x[2 * m + 1]), in_chunk));
        }
        if (16 * (k + 1) < width) {
          tmem_ld16(y_at + 16 * (k + 1), y);
          tmem_ld16(x_at + 16 * (k + 1), x);
        } else {
          tc_fence_before();
          arrive_on(bYFree);
        }
        if (cnt < kL && r >= cnt)                  // rows behind the sequence: zeros
#pragma unroll
          for (int m = 0; m < 8; ++m) q[m] = 0u;
        const uint4 o0 = make_uint4(q[0], q[1], q[2], q[3]), o1 = make_uint4(q[4], q[5], q[6], q[7]);
        if constexpr (L::kStage) {
          *reinterpret_cast<uint4*>(tile + (row ^ (32 * k))) = o0;
          *reinterpret_cast<uint4*>(tile + (row ^ (32 * k + 16))) = o1;
        } else if (tok0 + r < a.N) {
          T* p = out + (long long)(tok0 + r) * u.os[2] + 16 * k;
          if (16 * k < cols) *reinterpret_cast<uint4*>(p) = o0;
          if (16 * k + 8 < cols) *reinterpret_cast<uint4*>(p + 8) = o1;
        }
      }
      if constexpr (L::kStage) {
        fence_proxy_async();
        __syncwarp();
        if (lane == 0 && tok0 + 32 * w < a.N) tma_store_4d(&maps.out[unit], tile, c0, tok0 + 32 * w, h, b);      // clipped at N and the last column
      }
    }
    // chunks of the segment that no live token is in: zeros
    const uint4 z = make_uint4(0u, 0u, 0u, 0u);
    for (int tok = sp.n0 + kL * (sp.nch + rank) + r; tok < min(a.N, sp.n0 + a.seg_len);
         tok = sp.n0 + (tok - sp.n0) / kL * kL + kL * size + r) {
      T* p = out + (long long)tok * u.os[2];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (8 * k < cols) *reinterpret_cast<uint4*>(p + 8 * k) = z;
    }
    if constexpr (L::kStage)
      if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  } else if (warp >= L::kWarpX) {
    // ---- the state -----------------------------------------------------------------------------------------------------
    // It lives in sIn: a thread's quads of columns q = 0, 1, ... stand at 512 q + 16 lane of its warp's quarter.  They are read,
    // packed for this chunk's product, and replaced by the state behind the chunk, which is then copied to the CTA that takes
    // the next one.  That CTA's copy further on cannot arrive here before this one has been read: each waits for the one before.
    constexpr int NC = DK == 128 ? 64 : 32;        // columns of a thread
    const int r = tid - 32 * L::kWarpX, w = warp & 3, d = r & (DK - 1), col = DK == 128 ? 0 : 32 * (r >> 6);
    const uint32_t kv = tmem + ((uint32_t)(w * 32) << 16) + L::cKv + col;
    uint8_t* in = smem + L::oIn + w * L::kXPart + 16 + 16 * lane;
    const long long own = (long long)d * u.Dc + c0 + col;
    const int cols = d < u.Da ? u.Dc - c0 - col : 0;         // of this thread's columns, those that exist
    auto magnitude = [](const float4& x) {
      return max(max(__float_as_uint(x.x) & 0x7fffffffu, __float_as_uint(x.y) & 0x7fffffffu), max(__float_as_uint(x.z) & 0x7fffffffu, __float_as_uint(x.w) & 0x7fffffffu));
    };
    // Values that are not finite have no say in it: one of them, in a column of its own, would scale the others' down to nothing.
    constexpr uint32_t kInf = 0x7f800000u;
    auto finite_magnitude = [](const float4& x) {
      auto of = [](float v) {
        const uint32_t m = __float_as_uint(v) & 0x7fffffffu;
        return m < kInf ? m : 0u;
      };
      return max(max(of(x.x), of(x.y)), max(of(x.z), of(x.w)));
    };
    // fp16: the largest magnitude of the state before chunk c.  Of 128 features it is found as the state is made, and travels
    // with it: a warp's beside its quarter, even and odd chunks apart.  Of 64, whose packing comes last, it is found then.
    constexpr bool kSent = kHalfRange && DK == 128;
    auto note = [&](uint32_t top, int c) {
      top = __reduce_max_sync(0xffffffffu, top);
      if (top >= kInf) {
        top = 0;
#pragma unroll 1
        for (int j = 0; j < width; j += 4) top = max(top, finite_magnitude(*reinterpret_cast<const float4*>(in + 128 * j)));
        top = __reduce_max_sync(0xffffffffu, top);
      }
      if (lane == 0) *reinterpret_cast<uint32_t*>(in - 16 + 4 * (c & 1)) = top;
    };
    auto noted = [&](int c) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) top = max(top, *reinterpret_cast<const uint32_t*>(smem + L::oIn + i * L::kXPart + 4 * (c & 1)));
      return top;
    };
    if (rank == 0) {
      const float* before = a.n_seg > 1 ? u.seg + ((long long)bh * a.n_seg + seg) * u.Da * u.Dc : u.state_in ? u.state_in + (long long)bh * u.Da * u.Dc : nullptr;
      uint32_t top = 0;
#pragma unroll 2
      for (int j = 0; j < NC; j += 4) {
        const float4 x = before && j < cols ? *reinterpret_cast<const float4*>(before + own + j) : make_float4(0.f, 0.f, 0.f, 0.f);
        *reinterpret_cast<float4*>(in + 128 * j) = x;
        if (kSent) top = max(top, magnitude(x));
      }
      if (kSent) note(top, 0);
    }
    const DecayStep full(ld, kL);
    // eight columns of the state before the chunk, packed for the product
    uint8_t* packed = smem + L::oX;
    const F2 minus_one = both(-1.f);
    const uint32_t row = 128 * d + 16 * ((col / 8) ^ (d & 7));         // of the swizzled tile; its piece of columns j: row ^ 2 j
    auto pack = [&](const float4& x0, const float4& x1, float down, int j) {
      uint4 h, l;
      auto term = [&](float a0, float a1, uint32_t& hi, uint32_t& lo) {
        split2<T>(kHalfRange ? F2(a0 * down, a1 * down) : F2(a0, a1), minus_one, hi, lo);
      };
      term(x0.x, x0.y, h.x, l.x);
      term(x0.z, x0.w, h.y, l.y);
      term(x1.x, x1.y, h.z, l.z);
      term(x1.z, x1.w, h.w, l.w);
      const uint32_t at = row ^ (2 * j);
      *reinterpret_cast<uint4*>(packed + at) = h;
      *reinterpret_cast<uint4*>(packed + L::kXTile + at) = l;
    };
    F2 mul, keep;                                  // of the chunk's decay: X <- mul X + keep X
    auto stepped = [&](const float4& x, F2 v0, F2 v1) {
      const F2 a0(x.x, x.y), a1(x.z, x.w);
      const float2 y0 = fma2(mul, a0, fma2(keep, a0, v0)).get(), y1 = fma2(mul, a1, fma2(keep, a1, v1)).get();
      return make_float4(y0.x, y0.y, y1.x, y1.y);
    };
    // the largest magnitude of an fp16 tile to 2^13 ... 2^14: X may lie outside fp16's range
    auto scale_down = [&](uint32_t top, int i) {
      const int e = exponent_of(top);
      if (r == 0) sExp[i & 3] = power_of_two(e);
      return power_of_two(-e);
    };
    auto send = [&](int c) {                       // what this warp has written, to the CTA of the next chunk
      if (size == 1 || c + 1 == sp.nch) return;
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        const uint32_t next = (rank + 1) % size, at = smem_u32(smem + L::oIn + w * L::kXPart);
        copy_to_cta(remote(at, next), at, part, remote(smem_u32(bIn + w), next));
      }
    };
    auto receive = [&](int i, int c) {
      if (size == 1 || c == 0) return;
      for (int k = kSent ? 0 : w; k < (kSent ? 4 : w + 1); ++k) wait(bIn + k, rank == 0 ? i - 1 : i);
      if (lane == 0 && i + 1 < mine) mbar_expect_tx(bIn + w, part);
    };
    int ev = 0;
    for (int i = 0; i < mine; ++i, ++ev) {
      const int c = chunk(i), cnt = sp.live(c);
      const DecayStep decay = cnt == kL ? full : DecayStep(ld, cnt);
      mul = both(decay.mul);
      keep = both(decay.keep);
      const int t = terms(i);
      const bool two = t > 1;
      if (t == 3) ++ev;
      wait_together<4, 128>(wait, w == 2, bEv + (ev & 1), ev >> 1);
      tc_fence_after();
      const float unit = kHalfRange ? sUnit[i & 3] : 1.f;
      if constexpr (DK == 64) {
        // all of a thread's 32 columns in registers: B^T C before the state arrives, then the state behind the chunk, which the
        // next CTA waits for, and last the packing for this chunk's product
        F2 v[16];
#pragma unroll
        for (int j = 0; j < 32; j += 16) {
          uint32_t h[16];
          tmem_ld16(kv + j, h);
          if (two) {
            uint32_t l[16];
            tmem_ld16(kv + 64 + j, l);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 8; ++k) v[j / 2 + k] = add2(floats(h[2 * k], h[2 * k + 1]), floats(l[2 * k], l[2 * k + 1]));
          } else {
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 8; ++k) v[j / 2 + k] = floats(h[2 * k], h[2 * k + 1]);
          }
        }
        tc_fence_before();
        arrive_on(bKvFree);
        if constexpr (kHalfRange) {
          const F2 unit2 = both(unit);
#pragma unroll
          for (int k = 0; k < 16; ++k) v[k] = mul2(v[k], unit2);
        }
        receive(i, c);
        float4 x[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) x[q] = *reinterpret_cast<const float4*>(in + 512 * q);
#pragma unroll
        for (int q = 0; q < 8; ++q) *reinterpret_cast<float4*>(in + 512 * q) = stepped(x[q], v[2 * q], v[2 * q + 1]);
        send(c);
        float down = 1.f;
        if constexpr (kHalfRange) {
          uint32_t top = 0;
#pragma unroll
          for (int q = 0; q < 8; ++q) top = max(top, magnitude(x[q]));
          top = __reduce_max_sync(0xffffffffu, top);
          if (top >= kInf) {
            top = 0;
#pragma unroll
            for (int q = 0; q < 8; ++q) top = max(top, finite_magnitude(x[q]));
            top = __reduce_max_sync(0xffffffffu, top);
          }
          if (lane == 0) sMax[4 * (i & 1) + w] = top;
          asm volatile("bar.sync 1, 128;" ::: "memory");
          const uint4 all = *reinterpret_cast<const uint4*>(sMax + 4 * (i & 1));
          down = scale_down(max(max(all.x, all.y), max(all.z, all.w)), i);
        }
        if (i > 0) wait_together<4, 128>(wait, w == 2, bYx, i - 1);    // the product with the packed state of the chunk before is done
#pragma unroll
        for (int q = 0; q < 8; q += 2) pack(x[q], x[q + 1], down, 4 * q);
      } else {
        if (i > 0) wait_together<4, 128>(wait, w == 2, bYx, i - 1);
        receive(i, c);
        const float down = kSent ? scale_down(noted(c), i) : 1.f;
        uint32_t top = 0;
        auto step = [&](auto more) {               // a loop of its own for each number of terms: it is short, and waited for
#pragma unroll 2
          for (int j = 0; j < width; j += 8) {
            uint32_t h[8], l[8];
            tmem_ld8(kv + j, h);
            if constexpr (more.value) tmem_ld8(kv + 64 + j, l);
            const float4 x0 = *reinterpret_cast<const float4*>(in + 128 * j), x1 = *reinterpret_cast<const float4*>(in + 128 * j + 512);
            pack(x0, x1, down, j);
            tmem_wait_ld();
            auto v = [&](int k) {
              F2 x = floats(h[k], h[k + 1]);
              if constexpr (more.value) x = add2(x, floats(l[k], l[k + 1]));
              if constexpr (kHalfRange) x = mul2(x, both(unit));
              return x;
            };
            const float4 y0 = stepped(x0, v(0), v(2)), y1 = stepped(x1, v(4), v(6));
            *reinterpret_cast<float4*>(in + 128 * j) = y0;
            *reinterpret_cast<float4*>(in + 128 * j + 512) = y1;
            if (kSent) top = max(top, max(magnitude(y0), magnitude(y1)));
          }
        };
        if (two) step(std::true_type{});
        else step(std::false_type{});
        if (kSent) note(top, c + 1);
        send(c);
        tc_fence_before();
        arrive_on(bKvFree);
      }
      fence_proxy_async();
      arrive_on(bX + (i & 1));
    }
    // behind the last chunk (or, without one, behind none: rank 0 then)
    const int last = sp.nch > 0 ? (sp.nch - 1) % size : 0;
    if (u.state_out && seg == a.n_seg - 1 && rank == last)
#pragma unroll 2
      for (int j = 0; j < NC; j += 4)
        if (j < cols) *reinterpret_cast<float4*>(u.state_out + (long long)bh * u.Da * u.Dc + own + j) = *reinterpret_cast<const float4*>(in + 128 * j);
  } else if (warp >= L::kWarpC) {
    // ---- weighted C ----------------------------------------------------------------------------------------------------
    const int r = tid - 32 * L::kWarpC;
    Ring<L::kA> ra;
    Ring<L::kB> rb;
    const float w_full = exp2f(g2 * (float)(rev ? r : kL - 1 - r));
    int ev = 0, before = 1;                        // events so far, terms of the last
    for (int i = 0; i < mine; ++i) {
      const int cnt = sp.live(chunk(i));
      float w = rev || cnt == kL ? w_full : exp2f(g2 * (float)max(0, cnt - 1 - r));
      const int t = terms(i), parts = t == 3 ? 2 : 1;
      const bool leader = warp == L::kWarpC + 2;
      if (leader) {
        wait(bFullC + ra.at, ra.phase);
        if (cnt < kL) wait(bFull + ra.at, ra.phase);
      }
      if constexpr (kHalfRange) {                  // while the product with what stands in w_t may still run
        asm volatile("bar.sync 3, 128;" ::: "memory");
        const uint32_t own = r < cnt ? top_of_row(r, 0, width / 8, w, smem + L::oC + ra.at * kBlk) : 0u;
        const uint32_t top = __reduce_max_sync(0xffffffffu, own);
        if (lane == 0) sTop[warp & 3] = top;
        if (own == 0) w = 0.f;                     // zeros weigh nothing: under growth w times the power of two might overflow
      }
      for (int part = 0; part < parts; ++part, ++ev) {
        // the product with what stood here is done: the event before the last one, or the last where either takes both tiles
        const int back = t > 1 || before > 1 ? 1 : 2;
        if (leader && ev >= back) wait(bEv + ((ev - back) & 1), (ev - back) >> 1);
        asm volatile("bar.sync 3, 128;" ::: "memory");
        if constexpr (kHalfRange) {                // fp16 has one part
          const uint4 tops = *reinterpret_cast<const uint4*>(sTop);
          const int e = exponent_of(max(max(tops.x, tops.y), max(tops.z, tops.w)));
          if (r == 0) sUnit[i & 3] = power_of_two(e);        // chunk i - 4 has been read here: B^T C of i - 2, behind that, is done
          w *= power_of_two(-e);
        }
        weigh_c<T, CB>(r, 0, width / 8, cnt, plus && t == 2 ? w - 1.f : w, part ? 4 : t == 1 ? 1 : 3, smem + L::oC + ra.at * kBlk, smem + L::oW + (t == 1 ? (ev & 1) * kBlk : 0),
                       smem + L::oB + rb.at * (CB * kBlk));
        if (cnt < kL && part == 0) arrive_on(bClear);
        arrive_on(bW + (ev & 1));
        before = t;
      }
      ra.next();
      rb.next();
    }
  } else {
    // ---- weights of P --------------------------------------------------------------------------------------------------
    const int r0 = 32 * (warp & 3), r = r0 + lane, hb = warp >> 2;    // token, half of the columns
    const uint32_t lane_base = tmem + ((uint32_t)r0 << 16);
    // fp16: a row of P is scaled by a power of two of its own before it is rounded, so that products q . k of any size keep their
    // bits, those beyond 65504 too.  The weighted row goes back to tensor memory until its largest is known.
    const float scale_p = kHalfRange ? 1.f : a.scale;
    // The weight lambda^(i-j) of a block of 16 columns is a factor of the column times one of the row and the block.  On the
    // diagonal the latter exceeds 1, up to lambda^-15, and the former makes up for it: products as small as 2^-66 stay normal
    // numbers on the way for every decay above 2^-4 a token; stronger ones take an exponential for each value there.
    // Columns behind the length are zero in S already: its rows of b were cleared.  The mirrored walk, whose weights grow towards
    // them where log_decay is above 0, leaves them out all the same: a weight beyond the range of 32 bits would make them NaN.
    const bool mild = fabsf(g2) <= 4.f;
    F2 wcol[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      wcol[k] = F2(exp2f(g2 * (float)(rev ? 2 * k : 15 - 2 * k)), exp2f(g2 * (float)(rev ? 2 * k + 1 : 14 - 2 * k)));
    for (int i = 0; i < mine; ++i) {
      const uint32_t s = lane_base + 128 * (i & 1) + 64 * hb;
      wait_together<2, 256>(wait, warp == 3, bS + (i & 1), i >> 1);
      tc_fence_after();
      uint32_t top = 0;
      const int cnt = rev ? sp.live(chunk(i)) : kL;
      auto none_of = [&](int j0) { return rev ? j0 + 15 < r0 || j0 >= cnt : j0 > r0 + 31; };
#pragma unroll 1
      for (int k = 0; k < 4; ++k) {
        const int j0 = 64 * hb + 16 * k;           // the block's first column; the warp's rows are r0 ... r0 + 31
        const bool none = none_of(j0), all = rev ? j0 >= r0 + 31 && j0 + 15 < cnt : j0 + 15 <= r0;
        uint32_t p[8];
        if (none) {
          if constexpr (kHalfRange) continue;
#pragma unroll
          for (int m = 0; m < 8; ++m) p[m] = 0u;
        } else {
          uint32_t v[16];
          tmem_ld16(s + 16 * k, v);
          const F2 row = both(scale_p * exp2f(g2 * (float)(rev ? j0 - r : r - j0 - 15)));
          const int d = rev ? j0 - r : r - j0, sign = rev ? 1 : -1;    // i - j of the first column, and its change
          tmem_wait_ld();
          if (all) {
#pragma unroll
            for (int m = 0; m < 8; ++m) {
              const F2 x = mul2(mul2(floats(v[2 * m], v[2 * m + 1]), wcol[m]), row);
              if constexpr (kHalfRange) {
                const float2 f = x.get();
                v[2 * m] = __float_as_uint(f.x);
                v[2 * m + 1] = __float_as_uint(f.y);
              } else {
                p[m] = pack2<T>(x);
              }
            }
          } else if (mild) {
            const int t = r - j0;                  // columns up to t, or from t on
#pragma unroll
            for (int m = 0; m < 8; ++m) {
              const float2 x = mul2(mul2(floats(v[2 * m], v[2 * m + 1]), wcol[m]), row).get();
              v[2 * m] = __float_as_uint(x.x);
              v[2 * m + 1] = __float_as_uint(x.y);
            }
            if (rev) {
#pragma unroll
              for (int m = 0; m < 16; ++m) v[m] = m >= t && m < cnt - j0 ? v[m] : 0u;
            } else {
#pragma unroll
              for (int m = 0; m < 16; ++m) v[m] = m <= t ? v[m] : 0u;
            }
            if constexpr (!kHalfRange)
#pragma unroll
              for (int m = 0; m < 8; ++m) p[m] = Op16<T>::pack(__uint_as_float(v[2 * m]), __uint_as_float(v[2 * m + 1]));
          } else {
#pragma unroll 1
            for (int m = 0; m < 8; ++m) {
              const int d0 = d + sign * (2 * m), d1 = d0 + sign;
              uint32_t s0 = 0, s1 = 0;
#pragma unroll
              for (int q = 0; q < 8; ++q)
                if (q == m) { s0 = v[2 * q]; s1 = v[2 * q + 1]; }
              const float x0 = d0 >= 0 && j0 + 2 * m < cnt ? __uint_as_float(s0) * (scale_p * exp2f(g2 * (float)d0)) : 0.f;
              const float x1 = d1 >= 0 && j0 + 2 * m + 1 < cnt ? __uint_as_float(s1) * (scale_p * exp2f(g2 * (float)d1)) : 0.f;
              const uint32_t t = Op16<T>::pack(x0, x1);
#pragma unroll
              for (int q = 0; q < 8; ++q)
                if (q == m) {
                  if constexpr (kHalfRange) {
                    v[2 * q] = __float_as_uint(x0);
                    v[2 * q + 1] = __float_as_uint(x1);
                  } else {
                    p[q] = t;
                  }
                }
            }
          }
          if constexpr (kHalfRange) {
#pragma unroll
            for (int m = 0; m < 16; ++m) top = max(top, v[m] & 0x7fffffffu);
            tmem_st16(s + 16 * k, v);
          }
        }
        if constexpr (!kHalfRange) tmem_st8(s + 8 * k, p);   // over columns that are read already
      }
      if constexpr (kHalfRange) {
        sRow[128 * hb + r] = (uint8_t)(top >> 23);
        tmem_wait_st();
        asm volatile("bar.sync %0, 64;" ::"r"(6 + (warp & 3)) : "memory");         // the two warps of these rows
        const int e = exponent_of(max(top >> 23, (uint32_t)sRow[128 * (hb ^ 1) + r]) << 23);
        if (hb == 0) sPow[128 * (i & 3) + r] = (int8_t)e;
        const F2 up = both(power_of_two(-e));
#pragma unroll 1
        for (int k = 0; k < 4; ++k) {
          const int j0 = 64 * hb + 16 * k;
          uint32_t p[8];
          if (none_of(j0)) {
#pragma unroll
            for (int m = 0; m < 8; ++m) p[m] = 0u;
          } else {
            uint32_t v[16];
            tmem_ld16(s + 16 * k, v);
            tmem_wait_ld();
#pragma unroll
            for (int m = 0; m < 8; ++m) p[m] = pack2<T>(mul2(floats(v[2 * m], v[2 * m + 1]), up));
          }
          tmem_st8(s + 8 * k, p);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      arrive_on(bP + (i & 1));
    }
  }
  wait.report(status);
  tc_fence_before();
  cluster_sync();                                  // no CTA leaves while another may still write into it
  if (warp == 1) tmem_dealloc<512>(tmem);
}

int launch_walk(const void* kernel, dim3 grid, int threads, int smem, int cluster, cudaStream_t st, const DecayMaps& maps, const DecayArgs& a, int first,
                int per_unit, int* status) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid; cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = cluster > 1 ? 2 : 1;      // a launch of single CTAs that says so takes 1.3 us longer
  void* args[] = {const_cast<DecayMaps*>(&maps), const_cast<DecayArgs*>(&a), &first, &per_unit, &status};
  return cudaLaunchKernelExC(&cfg, kernel, args) == cudaSuccess ? FLARE_OK : FLARE_ECUDA;
}

// How a call is spread: the CTAs of a sequence (a cluster) and the segments of the token axis, whichever the times below say is
// shortest.  Measured (us, 64 / 128 features): a chunk in a CTA 1.9 / 3.0; a chunk's step of the state from CTA to CTA 0.65 /
// 1.2, which bounds what a cluster gains on a long sequence; a chunk's sum 0.7 / 1.1; the ends of a launch 7.  Clusters of
// three, four and eight do not fill every GPC: 45, 33 and 15 of them fit 148 SMs, and one more costs a second wave (97 us in 36
// clusters of four, 72 in 36 of two, at 8192 tokens).  E.g. D = 64, N = 8192: B = 4, H = 8 55 us in clusters of four, 71 of two,
// 73 in four segments; H = 16 79 us in clusters of two, 106 of four, 124 in two segments; B = 1, H = 8, N = 65536 109 us in 18
// segments, 117 in nine of clusters of two.  Over 28 shapes from 200 to 131077 tokens the choice is within 1 % of the best of all
// on average.
// Where the last wave of a launch would leave most SMs idle, the sequences in it are launched by themselves, in clusters that use
// more of them: the backward of B = 4, H = 16, N = 8192, D = 64 takes 148 sequences one to a CTA and 44 in clusters of three:
// 182 us, where 192 clusters of two took 194.  Behind another launch the last of the clusters that fit did not find its place:
// 45 of three took 208 us.
DecaySpread pick_spread(int B, int H, int N, int Da, int Dc, int n_units) {
  const int seqs = B * H * ((Dc + 63) / 64) * n_units;                 // 2^24 * 4 * 3 at most
  const int chunks = (N + kL - 1) / kL, sms = num_sms();
  const bool wide = Da > 64;
  const float chunk = wide ? 3.f : 1.9f, step = wide ? 1.2f : 0.65f, sum = wide ? 1.1f : 0.7f, ends = 7.f;
  constexpr int kSizes[] = {1, 2, 3, 4, 8};
  auto room = [&](int c) { return (c == 8 ? sms * 5 / 6 : c == 4 ? sms * 9 / 10 : c == 3 ? sms * 11 / 12 : sms) / c; };      // clusters that fit
  auto waves = [&](int n, int fit) { return (float)((n + fit - 1) / fit); };
  auto wave = [&](int c, int len) {               // a wave of sequences of so many chunks
    const int own = (len + c - 1) / c;
    return (c > 1 && len * step > own * chunk ? len * step : own * chunk) + ends;
  };
  DecaySpread best = {1, 1, 0, 1};
  float least = 1e30f;
  auto consider = [&](float t, const DecaySpread& s) {
    if (t < least) { least = t; best = s; }
  };
  for (int c : kSizes) {
    const int fit = room(c);
    if (c > chunks || fit < 1) break;
    const int most = chunks / (2 * c), full = seqs <= sms ? sms / (seqs * c) : 0;       // full: segments that fill the GPU once
    consider(waves(seqs, fit) * wave(c, chunks), {c, 1, 0, 1});
    for (int k = 0; k < 3; ++k) {
      int s = k == 0 ? full / 2 : k == 1 ? full : 2 * full;
      s = s < most ? s : most;
      if (s < 2) continue;
      if (s > 256) s = 256;
      const int len = (chunks + s - 1) / s;
      consider(waves(seqs * s, fit) * wave(c, len) + waves(seqs * (s - 1), sms) * (len * sum + ends) + 4.f, {c, s, 0, 1});
    }
    const int whole = seqs / fit, rest = seqs - whole * fit;
    if (whole > 0 && rest > 0)
      for (int r : kSizes) {
        const int places = room(r) - (r > 2);
        if (r <= chunks && places > 0) consider(whole * wave(c, chunks) + waves(rest, places) * wave(r, chunks) + 3.f, {c, 1, rest, r});
      }
  }
  return best;
}

template <typename T, int DK>
int launch_all(const DecayMaps& maps, const DecayArgs& a, int Dc, const DecaySpread& spread, cudaStream_t st) {
  using W = WalkPlan<DK>;
  using S = SumPlan<DK>;
  int* status = tc_status_ptr();
  const void* walk = a.u[0].state_out ? reinterpret_cast<const void*>(&k_decay_tc_walk<T, DK, true>)
                                      : reinterpret_cast<const void*>(&k_decay_tc_walk<T, DK, false>);
  if (tc_set_dyn_smem(walk, W::kBytes) != FLARE_OK) return FLARE_ECUDA;
  const unsigned seqs = (unsigned)(a.B * a.H * ((Dc + 63) / 64));
  if (a.n_seg > 1) {                               // the last segment walked needs no sum
    if (tc_set_dyn_smem(reinterpret_cast<const void*>(&k_decay_tc_sums<T, DK>), S::kBytes) != FLARE_OK) return FLARE_ECUDA;
    launch_dep(k_decay_tc_sums<T, DK>, dim3(seqs, (unsigned)a.n_seg - 1, (unsigned)a.n_units), dim3(S::kThreads), S::kBytes, st, maps, a, status);
    launch_decay_prefix(a, st);
  }
  const unsigned jobs = seqs * (unsigned)a.n_units, rest = (unsigned)spread.rest;
  int rc = launch_walk(walk, dim3((jobs - rest) * spread.cluster, (unsigned)a.n_seg), W::kThreads, W::kBytes, spread.cluster, st, maps, a, 0, (int)seqs, status);
  if (rc == FLARE_OK && rest)
    rc = launch_walk(walk, dim3(rest * spread.rest_cluster, (unsigned)a.n_seg), W::kThreads, W::kBytes, spread.rest_cluster, st, maps, a, (int)(jobs - rest), (int)seqs,
                     status);
  return rc;
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

DecaySpread decay_tc_spread(int B, int H, int N, int Da, int Dc, int n_units) { return pick_spread(B, H, N, Da, Dc, n_units); }

int decay_tc(const DecayArgs& a, int dtype, const DecaySpread& spread, cudaStream_t st) {
  DecayMaps maps;
  const void* seen[4] = {};
  int n = 0, Da = 0, Dc = 0;
  auto make = [&](CUtensorMap* m, const void* p, const long long (&s)[3], int D, int cols, uint32_t rows) {
    // a dimension of one entry has no stride of its own: any valid one
    const uint64_t row = a.N > 1 ? s[2] : D, head = a.H > 1 ? s[1] : row * (uint64_t)a.N, batch = a.B > 1 ? s[0] : head * (uint64_t)a.H;
    return make_tile_map_cols(m, p, dtype == FLARE_BF16 ? 1 : 0, D, cols, (uint64_t)a.N, (uint64_t)a.H, (uint64_t)a.B, 2 * row, 2 * head, 2 * batch, rows);
  };
  auto map_of = [&](const void* p, const long long (&s)[3], int D, int like) {
    // one tensor is an operand of several units; the same address with another shape is another tensor
    for (int i = 0; i < n; ++i)
      if (i == like && seen[i] == p) return i;
    if (n == 4 || !make(&maps.in[n], p, s, D, 64, 128)) return -1;
    seen[n] = p;
    return n++;
  };
  for (int i = 0; i < a.n_units; ++i) {
    const DecayUnit& u = a.u[i];
    Da = u.Da > Da ? u.Da : Da;
    Dc = u.Dc > Dc ? u.Dc : Dc;
    if (!make(&maps.out[i], u.out, u.os, u.Dc, 64, 32)) return FLARE_EUNSUPPORTED;
  }
  // the operands in the order dy v k | (v dy) q | (k q dy): each tensor's map is made once
  const int order[3][3] = {{0, 1, 2}, {1, 0, 3}, {2, 3, 0}};
  for (int i = 0; i < a.n_units; ++i) {
    const DecayUnit& u = a.u[i];
    maps.ia[i] = map_of(u.a, u.as, u.Da, order[i][0]);
    maps.ib[i] = map_of(u.b, u.bs, u.Da, order[i][1]);
    maps.ic[i] = map_of(u.c, u.cs, u.Dc, order[i][2]);
    if (maps.ia[i] < 0 || maps.ib[i] < 0 || maps.ic[i] < 0) return FLARE_EUNSUPPORTED;
  }
  if (dtype == FLARE_BF16) return Da <= 64 ? launch_all<__nv_bfloat16, 64>(maps, a, Dc, spread, st) : launch_all<__nv_bfloat16, 128>(maps, a, Dc, spread, st);
  return Da <= 64 ? launch_all<__half, 64>(maps, a, Dc, spread, st) : launch_all<__half, 128>(maps, a, Dc, spread, st);
}

}  // namespace flare
