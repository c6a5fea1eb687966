// Rotary positions: the pair (x0, x1) of a head's features becomes (x0 cos - x1 sin, x0 sin + x1 cos) * mag with the angle
// position * freqs[i].  Pairs are (i, i + R/2) or (2i, 2i + 1) for the first R features; the rest is copied.
//
// The angle is reduced to a part of a turn in 64 bits (position * freq is off by 0.06 rad at position 10^6 in 32), its sine
// and cosine are taken in 32.  No table is kept: a thread computes the angles of its pairs once and then takes several heads of
// one or two tensors (q and k) one after the other.  Angles made once a block, in shared memory, were slower (81 against 55 us
// for q and k at B = 4, H = 16, N = 8192, D = 64 bf16: two more dependent accesses a head), and so were the loads of four heads
// ahead of their use (82 us: at 111 registers too few threads fit).
// Every element is read and written once, 16 bytes an access; 4.9 TB/s at that size, 74 % of a copy's.  What bounds it is the loads'
// latency: a thread has one head's access in flight, as an output may be its input and loads do not pass stores.
#include <cstdarg>
#include <cstdio>
#include "common.cuh"
#include "launch.h"

namespace flare { void set_last_error(const char* msg); }

namespace flare {
namespace {

constexpr int kThreads = 256;

int refuse(int code, const char* fmt, ...) {
  char msg[400];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg, sizeof(msg), fmt, ap);
  va_end(ap);
  set_last_error(msg);
  return code;
}

struct RotTensor {
  const void* x;
  void* out;
  long long xs[3], os[3];                          // b, h, n
  int H;
};
struct RotArgs {
  RotTensor t[2];
  int B, N, D, half;                               // R = 2 * half features are rotated
  int items, rot_items;                            // pieces of a row: rotated ones first, then copied ones
  int heads, groups;                               // heads of both tensors together; threads that share them
  int heads_inner;                                 // whether heads lie closer together than tokens
  const double* freqs;
  const void* positions;                           // or null: offset + n
  int pos32;
  long long ps[2];                                 // element strides of b, n
  long long offset;
  float mag, sign;
};

template <typename T, int N>
struct alignas(N * sizeof(T)) Pack { T x[N]; };

// VEC elements an access.  Half layout: a rotated item is VEC features at i and VEC at i + half; interleaved: VEC features,
// VEC / 2 pairs (VEC = 1: one pair in two accesses).  A copied item is VEC features.
template <typename T, int VEC, bool INTER>
__global__ void __launch_bounds__(kThreads) k_rotary(const __grid_constant__ RotArgs a) {
  grid_dep_sync();
  using P = Pack<T, VEC>;
  constexpr int PAIRS = INTER && VEC > 1 ? VEC / 2 : VEC;
  constexpr int WIDTH = INTER ? 2 * PAIRS : VEC;   // columns from one rotated item to the next
  // Neighbouring threads go along a row, then along whichever of heads and tokens lies closer in memory.
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x;    // the host keeps items and shares of all tokens below 2^32
  const uint32_t row = i / (uint32_t)a.items, toks = (uint32_t)a.B * (uint32_t)a.N;
  const int item = (int)(i - row * (uint32_t)a.items);
  const uint32_t by = a.heads_inner ? (uint32_t)a.groups : toks, quot = row / by, rest = row - quot * by;
  const uint32_t tok = a.heads_inner ? quot : rest;
  const int share = (int)(a.heads_inner ? rest : quot);
  if (tok >= toks || share >= a.groups) return;
  const int b = (int)(tok / (uint32_t)a.N), n = (int)(tok - (uint32_t)b * (uint32_t)a.N);
  const bool rot = item < a.rot_items;
  const int col = rot ? item * WIDTH : 2 * a.half + (item - a.rot_items) * VEC;
  float cs[PAIRS], sn[PAIRS];
  if (rot) {
    long long pos = n;
    if (a.positions) {
      const long long at = b * a.ps[0] + n * a.ps[1];
      pos = a.pos32 ? (long long)static_cast<const int*>(a.positions)[at] : static_cast<const long long*>(a.positions)[at];
    }
    const double p = (double)(pos + a.offset) * 0.15915494309189533577;      // turns per radian
#pragma unroll
    for (int j = 0; j < PAIRS; ++j) {
      const double turns = p * a.freqs[INTER ? col / 2 + j : col + j];
      sincospif(2.f * (float)(turns - rint(turns)), &sn[j], &cs[j]);
      cs[j] *= a.mag;
      sn[j] *= a.mag * a.sign;
    }
  }
#pragma unroll 8
  for (int hh = share; hh < a.heads; hh += a.groups) {
    const bool second = hh >= a.t[0].H;
    const RotTensor& t = a.t[second ? 1 : 0];
    const int h = second ? hh - a.t[0].H : hh;
    const T* x = static_cast<const T*>(t.x) + b * t.xs[0] + h * t.xs[1] + n * t.xs[2] + col;
    T* o = static_cast<T*>(t.out) + b * t.os[0] + h * t.os[1] + n * t.os[2] + col;
    P u = *reinterpret_cast<const P*>(x);
    if (!rot) {
      *reinterpret_cast<P*>(o) = u;
    } else if constexpr (INTER && VEC == 1) {
      const float x0 = to_f32(u.x[0]), x1 = to_f32(x[1]);
      o[0] = from_f32<T>(x0 * cs[0] - x1 * sn[0]);
      o[1] = from_f32<T>(x0 * sn[0] + x1 * cs[0]);
    } else if constexpr (INTER) {
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) {
        const float x0 = to_f32(u.x[2 * j]), x1 = to_f32(u.x[2 * j + 1]);
        u.x[2 * j] = from_f32<T>(x0 * cs[j] - x1 * sn[j]);
        u.x[2 * j + 1] = from_f32<T>(x0 * sn[j] + x1 * cs[j]);
      }
      *reinterpret_cast<P*>(o) = u;
    } else {
      P w = *reinterpret_cast<const P*>(x + a.half);
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) {
        const float x0 = to_f32(u.x[j]), x1 = to_f32(w.x[j]);
        u.x[j] = from_f32<T>(x0 * cs[j] - x1 * sn[j]);
        w.x[j] = from_f32<T>(x0 * sn[j] + x1 * cs[j]);
      }
      *reinterpret_cast<P*>(o) = u;
      *reinterpret_cast<P*>(o + a.half) = w;
    }
  }
}

template <typename T, int VEC>
int go(RotArgs& a, bool interleaved, cudaStream_t st) {
  a.rot_items = interleaved && VEC > 1 ? 2 * a.half / VEC : a.half / VEC;
  a.items = a.rot_items + (a.D - 2 * a.half) / VEC;
  // Threads that share a token's heads compute its angles each: as many as give the GPU some 4600 threads per SM (55 us where
  // 303,000 threads in all take 61, B = 4, H = 16, N = 8192, D = 64 bf16; beyond that the angles cost more: 62 us at 16 shares).
  const long long threads = (long long)a.B * a.N * a.items;
  constexpr long long kMost = 0xffff0000LL;        // thread numbers are 32-bit
  if (threads > kMost) return refuse(FLARE_EUNSUPPORTED, "rotary: B*N=%lld tokens of %d accesses are too many", (long long)a.B * a.N, a.items);
  long long groups = (4608LL * num_sms() + threads / 2) / threads;
  if (groups > a.heads) groups = a.heads;
  if (groups < 1) groups = 1;
  while (groups > 1 && threads * groups > kMost) --groups;
  a.groups = (int)groups;
  a.heads_inner = a.t[0].xs[1] <= a.t[0].xs[2];
  const dim3 grid((unsigned)((threads * groups + kThreads - 1) / kThreads));
  if (interleaved) launch_dep(k_rotary<T, VEC, true>, grid, dim3(kThreads), 0, st, a);
  else launch_dep(k_rotary<T, VEC, false>, grid, dim3(kThreads), 0, st, a);
  return FLARE_OK;
}

// The widest access (16 bytes, 8 of 16-bit values, one value) that every pointer, stride and column border allows.
template <typename T>
int run(RotArgs& a, bool interleaved, cudaStream_t st) {
  auto fits = [&](int vec) {
    const int bytes = vec * (int)sizeof(T);
    if (a.D % vec || (interleaved ? 2 * a.half : a.half) % vec) return false;
    for (const RotTensor& t : a.t) {
      if (!t.x) continue;
      if (reinterpret_cast<uintptr_t>(t.x) % bytes || reinterpret_cast<uintptr_t>(t.out) % bytes) return false;
      for (int i = 0; i < 3; ++i)
        if (t.xs[i] % vec || t.os[i] % vec) return false;
    }
    return true;
  };
  constexpr int kWide = 16 / sizeof(T);
  if (fits(kWide)) return go<T, kWide>(a, interleaved, st);
  if (sizeof(T) == 2 && fits(4)) return go<T, 4>(a, interleaved, st);
  return go<T, 1>(a, interleaved, st);
}

}  // namespace
}  // namespace flare

using namespace flare;

extern "C" int flare_rotary(int B, int Hq, int Hk, int N, int D, int R, int dtype, const void* q, const int64_t* q_stride, void* q_out,
                            const int64_t* q_out_stride, const void* k, const int64_t* k_stride, void* k_out,
                            const int64_t* k_out_stride, const double* freqs, const void* positions, int positions_are_int32,
                            const int64_t* position_stride, int64_t offset, int interleaved, float mag, int back,
                            flare_stream_t stream) {
  if (B < 1 || Hq < 1 || N < 1 || D < 1 || (k && Hk < 1)) return refuse(FLARE_EINVAL, "rotary: bad sizes B=%d H=%d,%d N=%d D=%d", B, Hq, Hk, N, D);
  if (R < 2 || R % 2 || R > D) return refuse(FLARE_EINVAL, "rotary: R=%d of D=%d features", R, D);
  if (!q || !q_out || !q_stride || !q_out_stride || !freqs || (k && (!k_out || !k_stride || !k_out_stride)) || (positions && !position_stride))
    return refuse(FLARE_EINVAL, "rotary: null pointer");
  if (dtype != FLARE_F32 && dtype != FLARE_F16 && dtype != FLARE_BF16) return refuse(FLARE_EINVAL, "rotary: bad dtype %d", dtype);
  if ((long long)Hq + (k ? Hk : 0) >= 1LL << 30) return refuse(FLARE_EUNSUPPORTED, "rotary: 2^30 heads or more");
  if ((long long)B * N > 0xffff0000LL) return refuse(FLARE_EUNSUPPORTED, "rotary: B*N is too large");
  RotArgs a = {};
  a.t[0].x = q; a.t[0].out = q_out; a.t[0].H = Hq;
  a.t[1].x = k; a.t[1].out = k_out; a.t[1].H = k ? Hk : 0;
  for (int i = 0; i < 3; ++i) {
    a.t[0].xs[i] = q_stride[i]; a.t[0].os[i] = q_out_stride[i];
    if (k) { a.t[1].xs[i] = k_stride[i]; a.t[1].os[i] = k_out_stride[i]; }
  }
  a.B = B; a.N = N; a.D = D; a.half = R / 2;
  a.heads = Hq + a.t[1].H;
  a.freqs = freqs;
  a.positions = positions; a.pos32 = positions_are_int32;
  if (positions) { a.ps[0] = position_stride[0]; a.ps[1] = position_stride[1]; }
  a.offset = offset;
  a.mag = mag;
  a.sign = back ? -1.f : 1.f;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int rc = dtype == FLARE_F32 ? run<float>(a, interleaved != 0, st)
                 : dtype == FLARE_F16 ? run<__half>(a, interleaved != 0, st) : run<__nv_bfloat16>(a, interleaved != 0, st);
  if (rc != FLARE_OK) return rc;
  const cudaError_t e = cudaPeekAtLastError();
  if (e != cudaSuccess) return refuse(FLARE_ECUDA, "rotary: %s", cudaGetErrorString(e));
  return FLARE_OK;
}
