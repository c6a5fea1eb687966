// Linear attention with a decay for each head:  S_t = lambda_h S_{t-1} + k_t v_t^T,  y_t = scale * q_t^T S_t.
//
// This file: the C entries, the fp32-arithmetic kernels (fp32 inputs and every shape and alignment the tensor-core ones of
// flare_decay_tc.cu do not take), the scan over segments, and the single-token form.
//
// The token axis is cut into segments, a CTA each (two CTAs fit an SM).  With one segment a CTA walks its whole sequence; with
// several, pass 1 adds up every segment (sum of lambda^(end-1-n) b_n c_n^T; the last one walked too, which nothing reads),
// k_decay_prefix turns the sums into the states before the segments, and pass 2 walks all segments side by side.  A walk takes 64
// tokens at a time:
//     out = (lambda^(i-j) (a_i . b_j))_{j <= i} C  +  lambda^(i+1) A S,      S <- lambda^64 S + (lambda^(63-j) B)^T C
// The mirror image (n >= t) of the gradients is the same walk over rows taken from the end.
#include <cstdarg>
#include <cstdio>
#include "decay.h"
#include "launch.h"

namespace flare { void set_last_error(const char* msg); }

namespace flare {
namespace {

constexpr int kThreads = 256;
constexpr int kSub = 64;
constexpr int kPitchA = kSub + 4;

int refuse(int code, const char* fmt, ...) {
  char msg[400];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg, sizeof(msg), fmt, ap);
  va_end(ap);
  set_last_error(msg);
  return code;
}

// 16 or 4 bytes into shared memory without waiting for them; zeros where `in` is false
template <int BYTES>
__device__ __forceinline__ void copy_async(float* dst, const void* src, bool in) {
  const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst), n = in ? BYTES : 0;
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(n) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(d), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// rows r < 64 of one operand into shared memory as fp32, zeros behind row cnt and column D.  Row r is token tok0 + r * step.
// fp32 rows are on their way when this returns, 16-bit ones are there.
template <typename T>
__device__ __forceinline__ void load_rows(float* dst, int pitch, const T* src, long long row_stride, int tok0, int step, int cnt,
                                          int col0, int cols, int D, bool vec) {
  const int quads = cols / 4, per_pass = kThreads / quads, r0 = threadIdx.x / quads, c = 4 * (threadIdx.x - r0 * quads), col = col0 + c;
  if (r0 >= per_pass) return;                      // threads beyond whole rows have none
#pragma unroll 4
  for (int r = r0; r < kSub; r += per_pass) {
    const bool in = r < cnt && col < D;
    const T* p = in ? src + (long long)(tok0 + r * step) * row_stride + col : src;
    float* d = dst + r * pitch + c;
    if constexpr (sizeof(T) == 4) {
      if (vec) {                                   // D and every stride a multiple of four elements, bases aligned alike
        copy_async<16>(d, p, in);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) copy_async<4>(d + i, in && col + i < D ? p + i : src, in && col + i < D);
      }
    } else {
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (in && vec) {
        const uint2 t = *reinterpret_cast<const uint2*>(p);
        const T* h = reinterpret_cast<const T*>(&t);
        x = make_float4(to_f32(h[0]), to_f32(h[1]), to_f32(h[2]), to_f32(h[3]));
      } else if (in) {
        x.x = to_f32(p[0]);
        if (col + 1 < D) x.y = to_f32(p[1]);
        if (col + 2 < D) x.z = to_f32(p[2]);
        if (col + 3 < D) x.w = to_f32(p[3]);
      }
      *reinterpret_cast<float4*>(d) = x;
    }
  }
}

template <typename T>
__device__ __forceinline__ bool quads_aligned(const void* p, const long long (&s)[3], int D) {
  return reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T)) == 0 && s[0] % 4 == 0 && s[1] % 4 == 0 && s[2] % 4 == 0 && D % 4 == 0;
}

__device__ __forceinline__ float at4(const float4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// two fp32 values in a register pair, multiplied and added by one instruction
using Pair = unsigned long long;
__device__ __forceinline__ Pair fma_pair(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float2 halves(Pair v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}

// CV columns of a thread: a column block is 16 * CV wide.
template <int CV>
__device__ __forceinline__ void load_cv(const float* p, float (&x)[CV]) {
  if constexpr (CV == 4) {
    const float4 t = *reinterpret_cast<const float4*>(p);
    x[0] = t.x; x[1] = t.y; x[2] = t.z; x[3] = t.w;
  } else {
    const float2 t = *reinterpret_cast<const float2*>(p);
    x[0] = t.x; x[1] = t.y;
  }
}

// WALK: the outputs (and state_out) of a segment from the state before it.  Otherwise its sum alone.
// The next rows of b and c are on their way while these are worked on (bufs = 2), those of a from when the masked products that
// took their place have been read: 303 -> 237 us for the backward of B = 1, H = 8, N = 7000, D = 64 fp32.  c is weighted once, in
// place, not by every thread that reads it.
// What bounds it: the instructions and the shared memory that feed 4 x 4 results a thread.  At B = 4, H = 16, N = 900, D = 64 fp32
// the schedulers issue in 57 % of the slots, the busiest SMs' shared memory moves data 71 % of the time, for 14 TFLOP/s forward
// and 18 backward; blocks of the masked product above the diagonal are left out.  8 x 4 results for each of 128 threads move less
// data and hide less latency: 82 and 235 us instead of 82 and 230 at N = 7000 above, 210 instead of 192 at B = 2, H = 12,
// N = 1300, D = 128.
template <typename T, int CV, bool WALK>
__global__ void __launch_bounds__(kThreads, 2) k_decay_simt(const __grid_constant__ DecayArgs a, int bufs) {
  grid_dep_sync();
  constexpr int DVB = 16 * CV;
  extern __shared__ __align__(16) float sm[];
  const DecayUnit& u = a.u[blockIdx.z];
  const int n_cb = (u.Dc + DVB - 1) / DVB;
  const int bh = blockIdx.x % (a.B * a.H), cb = blockIdx.x / (a.B * a.H), seg = blockIdx.y;
  if (cb >= n_cb) return;
  const int b = bh / a.H, h = bh % a.H;
  const int Da = u.Da, Dap = (Da + 3) & ~3, pitch = Dap + 4, c0 = cb * DVB;
  const int b_size = kSub * pitch, buf_size = b_size + kSub * DVB;
  float* sS = sm;                                  // [Dap][DVB]
  float* sBC = sS + Dap * DVB;                     // bufs times: b [64][pitch], c [64][DVB]
  float* sW = sBC + bufs * buf_size;               // lambda^0 ... lambda^64
  float* sQ = sW + 72;                             // [64][pitch], and the masked products in its place
  float* sA = sQ;                                  // [64][kPitchA]
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const float ld = a.log_decay[h];
  if (tid <= kSub) sW[tid] = exp2f(decay_log2(ld) * (float)tid);
  const int live = decay_live(a, b);
  const int n0 = seg * a.seg_len, n1 = min(live, n0 + a.seg_len), n_end = min(a.N, n0 + a.seg_len);
  const T* pa = static_cast<const T*>(u.a) + b * u.as[0] + h * u.as[1];
  const T* pb = static_cast<const T*>(u.b) + b * u.bs[0] + h * u.bs[1];
  const T* pc = static_cast<const T*>(u.c) + b * u.cs[0] + h * u.cs[1];
  const bool va = WALK && quads_aligned<T>(u.a, u.as, Da), vb = quads_aligned<T>(u.b, u.bs, Da), vc = quads_aligned<T>(u.c, u.cs, u.Dc);
  const long long st_off = (long long)bh * Da * u.Dc;
  const float* before = nullptr;                   // the state before the segment
  if constexpr (WALK) {
    if (a.n_seg > 1) before = u.seg + ((long long)bh * a.n_seg + seg) * Da * u.Dc;
    else if (u.state_in) before = u.state_in + st_off;
  }
  const bool vs = u.Dc % 4 == 0 && reinterpret_cast<uintptr_t>(before) % 16 == 0;
  for (int e = 4 * tid; e < Dap * DVB; e += 4 * kThreads) {
    const int d = e / DVB, c = c0 + e % DVB;
    if (!before || d >= Da || c >= u.Dc) {
      *reinterpret_cast<float4*>(sS + e) = make_float4(0.f, 0.f, 0.f, 0.f);
      continue;
    }
    const float* p = before + (long long)d * u.Dc + c;
    if (vs) {
      copy_async<16>(sS + e, p, true);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) copy_async<4>(sS + e + i, c + i < u.Dc ? p + i : p, c + i < u.Dc);
    }
  }
  T* po = nullptr;
  bool vo = false;
  if constexpr (WALK) {
    po = static_cast<T*>(u.out) + b * u.os[0] + h * u.os[1];
    vo = quads_aligned<T>(u.out, u.os, u.Dc);
  }

  const int subs = n1 > n0 ? (n1 - n0 + kSub - 1) / kSub : 0, step = u.rev ? -1 : 1;
  auto rows_of = [&](int s) { return min(kSub, n1 - n0 - s * kSub); };
  auto first_of = [&](int s) { return u.rev ? n1 - 1 - s * kSub : n0 + s * kSub; };
  auto fetch = [&](int s, int buf) {
    load_rows(sBC + buf * buf_size, pitch, pb, u.bs[2], first_of(s), step, rows_of(s), 0, Dap, Da, vb);
    load_rows(sBC + buf * buf_size + b_size, DVB, pc, u.cs[2], first_of(s), step, rows_of(s), c0, DVB, u.Dc, vc);
  };
  auto fetch_a = [&](int s) { load_rows(sQ, pitch, pa, u.as[2], first_of(s), step, rows_of(s), 0, Dap, Da, va); };
  if (subs > 0) {
    if constexpr (WALK) fetch_a(0);
    fetch(0, 0);
  }
  const DecayStep full(ld, kSub);
  for (int s = 0; s < subs; ++s) {
    const int cnt = rows_of(s), tok0 = first_of(s), buf = bufs == 2 ? s & 1 : 0;
    float *sB = sBC + buf * buf_size, *sC = sB + b_size;
    if (bufs == 1 && s > 0) {
      __syncthreads();
      fetch(s, 0);
    }
    copies_done();
    __syncthreads();
    if (bufs == 2 && s + 1 < subs) fetch(s + 1, buf ^ 1);
    if constexpr (WALK) {
      // (a_i . b_j) for j <= i, thread rows i = ty + 16 p, columns j = tx + 16 r (r > p is above the diagonal), even and odd
      // features apart; and A S
      Pair dot[4][4];
      float out[4][CV] = {};
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int r = 0; r <= p; ++r) dot[p][r] = 0;
      for (int k = 0; k < Dap; k += 4) {
        ulonglong2 x[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) x[p] = *reinterpret_cast<const ulonglong2*>(sQ + (ty + 16 * p) * pitch + k);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const ulonglong2 y = *reinterpret_cast<const ulonglong2*>(sB + (tx + 16 * r) * pitch + k);
#pragma unroll
          for (int p = r; p < 4; ++p) dot[p][r] = fma_pair(x[p].y, y.y, fma_pair(x[p].x, y.x, dot[p][r]));
        }
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          float y[CV];
          load_cv<CV>(sS + (k + kk) * DVB + CV * tx, y);
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            const float2 xx = halves(kk < 2 ? x[p].x : x[p].y);
#pragma unroll
            for (int c = 0; c < CV; ++c) out[p][c] = fmaf(kk % 2 ? xx.y : xx.x, y[c], out[p][c]);
          }
        }
      }
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const float w = sW[ty + 16 * p + 1];
#pragma unroll
        for (int c = 0; c < CV; ++c) out[p][c] *= w;
      }
      __syncthreads();                             // a has been read
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int r = 0; r <= p; ++r) {
          const int i = ty + 16 * p, j = tx + 16 * r;
          const float2 d = halves(dot[p][r]);
          sA[i * kPitchA + j] = j <= i ? (d.x + d.y) * sW[i - j] : 0.f;
        }
      __syncthreads();
#pragma unroll
      for (int jb = 0; jb < 4; ++jb)
        for (int j = 16 * jb; j < 16 * jb + 16; j += 4) {
          float4 x[4];
#pragma unroll
          for (int p = jb; p < 4; ++p) x[p] = *reinterpret_cast<const float4*>(sA + (ty + 16 * p) * kPitchA + j);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            float y[CV];
            load_cv<CV>(sC + (j + kk) * DVB + CV * tx, y);
#pragma unroll
            for (int p = jb; p < 4; ++p)
#pragma unroll
              for (int c = 0; c < CV; ++c) out[p][c] = fmaf(at4(x[p], kk), y[c], out[p][c]);
          }
        }
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const int i = ty + 16 * p, col = c0 + CV * tx;
        if (i >= cnt || col >= u.Dc) continue;
        T* o = po + (long long)(tok0 + i * step) * u.os[2] + col;
        T t[CV];
#pragma unroll
        for (int c = 0; c < CV; ++c) t[c] = from_f32<T>(out[p][c] * a.scale);
        if (vo) {
          struct alignas(CV * sizeof(T)) Pack { T x[CV]; };
          *reinterpret_cast<Pack*>(o) = *reinterpret_cast<const Pack*>(t);
        } else {
#pragma unroll
          for (int c = 0; c < CV; ++c)
            if (col + c < u.Dc) o[c] = t[c];
        }
      }
      __syncthreads();                             // the masked products and c have been read
      if (s + 1 < subs) fetch_a(s + 1);
    }
    for (int e = 4 * tid; e < cnt * DVB; e += 4 * kThreads) {
      const float w = sW[cnt - 1 - e / DVB];
      float4* x = reinterpret_cast<float4*>(sC + e);
      *x = make_float4(x->x * w, x->y * w, x->z * w, x->w * w);
    }
    __syncthreads();
    const DecayStep decay = cnt == kSub ? full : DecayStep(ld, cnt);
    for (int k0 = 4 * ty; k0 < Dap; k0 += 64) {
      float acc[4][CV] = {};
#pragma unroll 4
      for (int i = 0; i < cnt; ++i) {
        const float4 x = *reinterpret_cast<const float4*>(sB + i * pitch + k0);
        float y[CV];
        load_cv<CV>(sC + i * DVB + CV * tx, y);
#pragma unroll
        for (int p = 0; p < 4; ++p)
#pragma unroll
          for (int c = 0; c < CV; ++c) acc[p][c] = fmaf(at4(x, p), y[c], acc[p][c]);
      }
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        float* e = sS + (k0 + p) * DVB + CV * tx;
        float x[CV];
        load_cv<CV>(e, x);
#pragma unroll
        for (int c = 0; c < CV; ++c) x[c] = decay(x[c]) + acc[p][c];
        if constexpr (CV == 4) *reinterpret_cast<float4*>(e) = make_float4(x[0], x[1], x[2], x[3]);
        else *reinterpret_cast<float2*>(e) = make_float2(x[0], x[1]);
      }
    }
  }
  copies_done();                                   // the state, where no token was taken
  __syncthreads();
  float* end = nullptr;
  if constexpr (WALK) {
    if (u.state_out && seg == a.n_seg - 1) end = u.state_out + st_off;
    const int z0 = max(n0, live);                  // rows behind the sequence: zeros
    for (int n = z0 + tid / DVB; n < n_end; n += kThreads / DVB) {
      const int c = c0 + tid % DVB;
      if (c < u.Dc) po[n * u.os[2] + c] = from_f32<T>(0.f);
    }
  } else {
    end = u.seg + ((long long)bh * a.n_seg + seg) * Da * u.Dc;
  }
  if (end)
    for (int e = tid; e < Da * DVB; e += kThreads) {
      const int d = e / DVB, c = c0 + e % DVB;
      if (c < u.Dc) end[(long long)d * u.Dc + c] = sS[e];
    }
}

// sums of the segments -> states before them, in place.  A thread owns one element of one (unit, b, h), and the loads' latency is
// what it waits for: 7 us for 16 heads of 128 x 128 in 8 segments, beside 476 of the kernels around it.
__global__ void __launch_bounds__(256) k_decay_prefix(const __grid_constant__ DecayArgs a) {
  grid_dep_sync();
  const DecayUnit& u = a.u[blockIdx.y];
  const long long per = (long long)u.Da * u.Dc;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long long)a.B * a.H * per) return;
  const int bh = (int)(i / per), b = bh / a.H, h = bh % a.H;
  float* s = u.seg + (long long)bh * a.n_seg * per + i % per;
  float run = u.state_in ? u.state_in[i] : 0.f;
  const float ld = a.log_decay[h];
  const int live = decay_live(a, b);
  const DecayStep full(ld, a.seg_len);
  auto add = [&](int seg, float sum) {
    const int cnt = min(a.seg_len, live - seg * a.seg_len);
    if (cnt == a.seg_len) run = full(run) + sum;
    else if (cnt > 0) run = DecayStep(ld, cnt)(run) + sum;
  };
  constexpr int kAhead = 8;                        // loads in flight: a segment's addition waits for the one before it
  for (int s0 = 0; s0 < a.n_seg; s0 += kAhead) {
    float x[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int seg = u.rev ? a.n_seg - 1 - s0 - j : s0 + j;
      x[j] = s0 + j + 1 < a.n_seg ? s[(long long)seg * per] : 0.f;     // the last one walked has no sum, or one that nobody needs
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (s0 + j >= a.n_seg) break;
      const int seg = u.rev ? a.n_seg - 1 - s0 - j : s0 + j;
      s[(long long)seg * per] = run;
      add(seg, x[j]);
    }
  }
}

// ---- single tokens ---------------------------------------------------------------------------------------------------
// One CTA per (b, h, block of columns); the state stays in registers over the T tokens, so a call reads and writes it once.
// A thread holds ROWS quads of four columns: all its loads are in flight before the first is used.  What bounds it is the state's
// way through HBM, 8 bytes an element: B = 256, H = 16, D = 128 bf16 take 94 us, 5.8 TB/s of the 6.5 that a copy reaches.  A
// small batch is the launch: 5.2 us for B = 4, H = 16, D = 64.
constexpr int kDecThreads = 256;

struct DecodeArgs {
  int B, H, T, Dk, Dv;
  int lanes;                                       // threads beside one another on a row (a power of two): 4 * lanes columns
  float scale;
  const float* log_decay;
  const int* lengths;
  const void *q, *k, *v;
  void* y;
  long long qs[3], ks[3], vs[3], ys[3];
  float* state;
};

template <typename T, int ROWS, bool VEC>
__global__ void __launch_bounds__(kDecThreads) k_decay_decode(const __grid_constant__ DecodeArgs a) {
  grid_dep_sync();
  __shared__ float sQ[256], sK[256];
  __shared__ float4 sY[kDecThreads];
  const int bh = blockIdx.x, b = bh / a.H, h = bh % a.H, tid = threadIdx.x;
  const int lane = tid & (a.lanes - 1), row0 = tid / a.lanes, per_row = kDecThreads / a.lanes;
  const int col = 4 * (blockIdx.y * a.lanes + lane);
  const int live = a.lengths ? max(0, min(a.T, a.lengths[b])) : a.T;
  const T* pq = static_cast<const T*>(a.q) + b * a.qs[0] + h * a.qs[1];
  const T* pk = static_cast<const T*>(a.k) + b * a.ks[0] + h * a.ks[1];
  const T* pv = static_cast<const T*>(a.v) + b * a.vs[0] + h * a.vs[1];
  T* py = static_cast<T*>(a.y) + b * a.ys[0] + h * a.ys[1];
  float* st = a.state + (long long)bh * a.Dk * a.Dv;
  float4 S[ROWS];
  if (live > 0) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int d = row0 + r * per_row;
      S[r] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (d >= a.Dk) continue;
      const float* p = st + (long long)d * a.Dv + col;
      if constexpr (VEC) {
        if (col < a.Dv) S[r] = *reinterpret_cast<const float4*>(p);
      } else {
        if (col < a.Dv) S[r].x = p[0];
        if (col + 1 < a.Dv) S[r].y = p[1];
        if (col + 2 < a.Dv) S[r].z = p[2];
        if (col + 3 < a.Dv) S[r].w = p[3];
      }
    }
  }
  const DecayStep decay(a.log_decay[h], 1);
  for (int t = 0; t < a.T; ++t) {
    T* o = py + (long long)t * a.ys[2];
    if (t >= live) {                               // tokens behind the sequence: zeros, the state as it is
      if (row0 == 0)
        for (int c = 0; c < 4; ++c)
          if (col + c < a.Dv) o[col + c] = from_f32<T>(0.f);
      continue;
    }
    for (int d = tid; d < a.Dk; d += kDecThreads) {
      sQ[d] = to_f32(pq[(long long)t * a.qs[2] + d]);
      sK[d] = to_f32(pk[(long long)t * a.ks[2] + d]);
    }
    float v[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = col + c < a.Dv ? to_f32(pv[(long long)t * a.vs[2] + col + c]) : 0.f;
    __syncthreads();
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int d = row0 + r * per_row;
      if (d >= a.Dk) continue;
      const float k = sK[d], q = sQ[d];
      S[r].x = fmaf(k, v[0], decay(S[r].x)); S[r].y = fmaf(k, v[1], decay(S[r].y));
      S[r].z = fmaf(k, v[2], decay(S[r].z)); S[r].w = fmaf(k, v[3], decay(S[r].w));
      y.x = fmaf(q, S[r].x, y.x); y.y = fmaf(q, S[r].y, y.y); y.z = fmaf(q, S[r].z, y.z); y.w = fmaf(q, S[r].w, y.w);
    }
    sY[tid] = y;
    __syncthreads();
    for (int half = per_row / 2; half > 0; half /= 2) {      // the rows' shares, in a fixed order
      if (row0 < half) {
        const float4 x = sY[tid + half * a.lanes];
        y.x += x.x; y.y += x.y; y.z += x.z; y.w += x.w;
        sY[tid] = y;
      }
      __syncthreads();
    }
    if (row0 == 0) {
      const float r[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (col + c < a.Dv) o[col + c] = from_f32<T>(r[c] * a.scale);
    }
  }
  if (live > 0) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int d = row0 + r * per_row;
      if (d >= a.Dk) continue;
      float* p = st + (long long)d * a.Dv + col;
      if constexpr (VEC) {
        if (col < a.Dv) *reinterpret_cast<float4*>(p) = S[r];
      } else {
        if (col < a.Dv) p[0] = S[r].x;
        if (col + 1 < a.Dv) p[1] = S[r].y;
        if (col + 2 < a.Dv) p[2] = S[r].z;
        if (col + 3 < a.Dv) p[3] = S[r].w;
      }
    }
  }
}

template <typename T>
int run_decode(const DecodeArgs& a0, cudaStream_t st) {
  DecodeArgs a = a0;
  // columns of a CTA: as many as its threads can hold at 16 quads each
  auto rows_of = [&](int lanes) { return (a.Dk + kDecThreads / lanes - 1) / (kDecThreads / lanes); };
  int lanes = 1;
  while (4 * lanes < a.Dv && rows_of(2 * lanes) <= 16) lanes *= 2;
  a.lanes = lanes;
  const int rows = rows_of(lanes);
  const dim3 grid((unsigned)(a.B * a.H), (unsigned)((a.Dv + 4 * lanes - 1) / (4 * lanes)));
  const bool vec = a.Dv % 4 == 0 && reinterpret_cast<uintptr_t>(a.state) % 16 == 0;
  auto go = [&](auto kernel) { launch_dep(kernel, grid, dim3(kDecThreads), 0, st, a); };
  if (rows <= 4) vec ? go(k_decay_decode<T, 4, true>) : go(k_decay_decode<T, 4, false>);
  else vec ? go(k_decay_decode<T, 16, true>) : go(k_decay_decode<T, 16, false>);
  return FLARE_OK;
}

// ---- host side -------------------------------------------------------------------------------------------------------
int pick_segments(int B, int H, int N, int Dc, int n_units) {
  const int cb = (Dc + 63) / 64;
  const long long ctas = (long long)B * H * cb * n_units;
  // Two CTAs an SM and blocks of 64 columns are what up to 124 features have.  Of 125 to 128 one CTA fits (117 kB of shared memory), of
  // more the blocks are 32 columns wide and above 164 one CTA fits again: those grids take two to four waves.
  long long s = 2LL * num_sms() / ctas;
  const long long max_s = ((long long)N + kSub - 1) / kSub;
  if (s > max_s) s = max_s;
  if (s > 256) s = 256;
  return s < 1 ? 1 : (int)s;
}

size_t simt_smem(int Da, int CV, bool walk, int bufs) {
  const int Dap = (Da + 3) & ~3, DVB = 16 * CV, pitch = Dap + 4;
  const size_t f = (size_t)Dap * DVB + bufs * (kSub * pitch + kSub * DVB) + 72 + (walk ? kSub * (pitch > kPitchA ? pitch : kPitchA) : 0);
  return f * sizeof(float);
}

template <typename T, int CV, bool WALK>
void run_simt_pass(const DecayArgs& a, int Da, int Dc, cudaStream_t st) {
  const dim3 grid((unsigned)(a.B * a.H * ((Dc + 16 * CV - 1) / (16 * CV))), (unsigned)a.n_seg, (unsigned)a.n_units);
  // Two tiles of b and c, the next one on its way, unless they would cost the SM its second CTA or do not fit.
  constexpr size_t kOne = 227 * 1024, kTwo = 113 * 1024;
  const size_t one = simt_smem(Da, CV, WALK, 1), two = simt_smem(Da, CV, WALK, 2);
  const int bufs = two <= (one <= kTwo ? kTwo : kOne) ? 2 : 1;
  launch_dep(k_decay_simt<T, CV, WALK>, grid, dim3(kThreads), bufs == 2 ? two : one, st, a, bufs);
}

template <typename T, int CV>
int run_simt_cv(const DecayArgs& a, int Da, int Dc, cudaStream_t st) {
  if (tc_set_dyn_smem(reinterpret_cast<const void*>(&k_decay_simt<T, CV, true>), 227 * 1024) != FLARE_OK ||
      tc_set_dyn_smem(reinterpret_cast<const void*>(&k_decay_simt<T, CV, false>), 227 * 1024) != FLARE_OK)
    return refuse(FLARE_ECUDA, "decay: cudaFuncSetAttribute failed");
  if (a.n_seg > 1) {
    run_simt_pass<T, CV, false>(a, Da, Dc, st);
    launch_decay_prefix(a, st);
  }
  run_simt_pass<T, CV, true>(a, Da, Dc, st);
  return FLARE_OK;
}

// column blocks of 64 where the tiles of Da <= 128 features leave room for two CTAs per SM or one, else of 32
template <typename T>
int run_simt(const DecayArgs& a, int Da, int Dc, cudaStream_t st) {
  return Dc > 32 && Da <= 128 ? run_simt_cv<T, 4>(a, Da, Dc, st) : run_simt_cv<T, 2>(a, Da, Dc, st);
}

int check_problem(const char* what, const FlareDecay* p) {
  if (!p) return refuse(FLARE_EINVAL, "%s: null problem", what);
  if (p->B < 1 || p->H < 1 || p->N < 1) return refuse(FLARE_EINVAL, "%s: bad sizes B=%d H=%d N=%d", what, p->B, p->H, p->N);
  if (p->Dk < 1 || p->Dv < 1 || p->Dk > 256 || p->Dv > 256)
    return refuse(FLARE_EUNSUPPORTED, "%s: Dk=%d Dv=%d, both must be 1 to 256", what, p->Dk, p->Dv);
  if (p->dtype != FLARE_F32 && p->dtype != FLARE_F16 && p->dtype != FLARE_BF16) return refuse(FLARE_EINVAL, "%s: bad dtype %d", what, p->dtype);
  if ((long long)p->B * p->H > (1 << 24)) return refuse(FLARE_EUNSUPPORTED, "%s: B*H > 2^24", what);
  if (p->N > (1 << 30)) return refuse(FLARE_EUNSUPPORTED, "%s: N > 2^30", what);
  return FLARE_OK;
}

DecayArgs base_args(const FlareDecay* p, const float* log_decay, const int* lengths) {
  DecayArgs a = {};
  a.B = p->B; a.H = p->H; a.N = p->N;
  a.scale = p->scale;
  a.log_decay = log_decay;
  a.lengths = lengths;
  return a;
}

void set(long long (&dst)[3], const int64_t* s) { for (int i = 0; i < 3; ++i) dst[i] = s[i]; }

DecayUnit unit(const void* x, const int64_t* xs, const void* y, const int64_t* ys, const void* z, const int64_t* zs, void* out,
               const int64_t* os, int Da, int Dc, int rev) {
  DecayUnit u = {};
  u.a = x; u.b = y; u.c = z; u.out = out;
  set(u.as, xs); set(u.bs, ys); set(u.cs, zs); set(u.os, os);
  u.Da = Da; u.Dc = Dc; u.rev = rev;
  return u;
}

// How a call is cut follows from its sizes alone, for either family, so that the workspace asked for fits both.
struct Plan {
  int simt_segments;
  DecaySpread tc;
  size_t bytes;
};
Plan plan_of(const FlareDecay* p, int units) {
  const int D = p->Dk > p->Dv ? p->Dk : p->Dv, Da = units == 1 ? p->Dk : D, Dc = units == 1 ? p->Dv : D;
  Plan plan = {pick_segments(p->B, p->H, p->N, Dc, units), decay_tc_spread(p->B, p->H, p->N, Da, Dc, units), 0};
  const int s = plan.simt_segments > plan.tc.segments ? plan.simt_segments : plan.tc.segments;
  if (s > 1) plan.bytes = (size_t)units * p->B * p->H * s * p->Dk * p->Dv * sizeof(float);
  return plan;
}

int run(DecayArgs& a, const FlareDecay* p, const Plan& plan, float* ws, cudaStream_t st, const char* what) {
  int Da = 0, Dc = 0;
  for (int i = 0; i < a.n_units; ++i) {
    Da = a.u[i].Da > Da ? a.u[i].Da : Da;
    Dc = a.u[i].Dc > Dc ? a.u[i].Dc : Dc;
  }
  const bool tc = decay_tc_supported(a, p->dtype);
  const int n = tc ? plan.tc.segments : plan.simt_segments;
  const int block = tc ? 128 : kSub;
  a.seg_len = (int)((((long long)p->N + n - 1) / n + block - 1) / block) * block;
  a.n_seg = (p->N + a.seg_len - 1) / a.seg_len;
  for (int i = 0; i < a.n_units; ++i) a.u[i].seg = ws + (size_t)i * p->B * p->H * a.n_seg * p->Dk * p->Dv;
  int rc;
  if (tc) rc = decay_tc(a, p->dtype, plan.tc, st);
  else if (p->dtype == FLARE_F32) rc = run_simt<float>(a, Da, Dc, st);
  else if (p->dtype == FLARE_F16) rc = run_simt<__half>(a, Da, Dc, st);
  else rc = run_simt<__nv_bfloat16>(a, Da, Dc, st);
  if (rc != FLARE_OK) return refuse(rc, "%s: the kernels could not be launched", what);
  const cudaError_t e = cudaPeekAtLastError();
  if (e != cudaSuccess) return refuse(FLARE_ECUDA, "%s: %s", what, cudaGetErrorString(e));
  return FLARE_OK;
}

}  // namespace

void launch_decay_prefix(const DecayArgs& a, cudaStream_t st) {
  const long long n = (long long)a.B * a.H * a.u[0].Da * a.u[0].Dc;        // Da * Dc is Dk * Dv for every unit
  launch_dep(k_decay_prefix, dim3((unsigned)((n + 255) / 256), (unsigned)a.n_units), dim3(256), 0, st, a);
}

}  // namespace flare

using namespace flare;

extern "C" {

size_t flare_decay_workspace_bytes(const FlareDecay* p) { return check_problem("decay", p) == FLARE_OK ? plan_of(p, 1).bytes : 0; }
size_t flare_decay_bwd_workspace_bytes(const FlareDecay* p) { return check_problem("decay_bwd", p) == FLARE_OK ? plan_of(p, 3).bytes : 0; }

int flare_decay_fwd(const FlareDecay* p, const void* q, const void* k, const void* v, const float* log_decay,
                    const int32_t* lengths, void* y, const float* state_in, float* state_out, float* workspace,
                    size_t workspace_bytes, flare_stream_t stream) {
  if (int rc = check_problem("decay", p)) return rc;
  if (!q || !k || !v || !y || !log_decay) return refuse(FLARE_EINVAL, "decay: null pointer");
  const Plan plan = plan_of(p, 1);
  const size_t need = plan.bytes;
  if (need && (!workspace || workspace_bytes < need)) return refuse(FLARE_EWORKSPACE, "decay: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  if (reinterpret_cast<uintptr_t>(workspace) % 16) return refuse(FLARE_EALIGN, "decay: workspace must be 16-byte aligned");
  DecayArgs a = base_args(p, log_decay, lengths);
  a.n_units = 1;
  a.u[0] = unit(q, p->q_stride, k, p->k_stride, v, p->v_stride, y, p->y_stride, p->Dk, p->Dv, 0);
  a.u[0].state_in = state_in;
  a.u[0].state_out = state_out;
  return run(a, p, plan, workspace, static_cast<cudaStream_t>(stream), "decay");
}

int flare_decay_bwd(const FlareDecay* p, const void* q, const void* k, const void* v, const void* dy, const float* log_decay,
                    const int32_t* lengths, void* dq, void* dk, void* dv, float* workspace, size_t workspace_bytes,
                    flare_stream_t stream) {
  if (int rc = check_problem("decay_bwd", p)) return rc;
  if (!q || !k || !v || !dy || !dq || !dk || !dv || !log_decay) return refuse(FLARE_EINVAL, "decay_bwd: null pointer");
  const Plan plan = plan_of(p, 3);
  const size_t need = plan.bytes;
  if (need && (!workspace || workspace_bytes < need)) return refuse(FLARE_EWORKSPACE, "decay_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  if (reinterpret_cast<uintptr_t>(workspace) % 16) return refuse(FLARE_EALIGN, "decay_bwd: workspace must be 16-byte aligned");
  DecayArgs a = base_args(p, log_decay, lengths);
  a.n_units = 3;
  a.u[0] = unit(dy, p->dy_stride, v, p->v_stride, k, p->k_stride, dq, p->dq_stride, p->Dv, p->Dk, 0);
  a.u[1] = unit(v, p->v_stride, dy, p->dy_stride, q, p->q_stride, dk, p->dk_stride, p->Dv, p->Dk, 1);
  a.u[2] = unit(k, p->k_stride, q, p->q_stride, dy, p->dy_stride, dv, p->dv_stride, p->Dk, p->Dv, 1);
  return run(a, p, plan, workspace, static_cast<cudaStream_t>(stream), "decay_bwd");
}

int flare_decay_decode(const FlareDecay* p, const void* q, const void* k, const void* v, const float* log_decay,
                       const int32_t* lengths, void* y, float* state, flare_stream_t stream) {
  if (int rc = check_problem("decay_decode", p)) return rc;
  if (!q || !k || !v || !y || !log_decay || !state) return refuse(FLARE_EINVAL, "decay_decode: null pointer");
  DecodeArgs a = {};
  a.B = p->B; a.H = p->H; a.T = p->N; a.Dk = p->Dk; a.Dv = p->Dv;
  a.scale = p->scale;
  a.log_decay = log_decay; a.lengths = lengths;
  a.q = q; a.k = k; a.v = v; a.y = y;
  set(a.qs, p->q_stride); set(a.ks, p->k_stride); set(a.vs, p->v_stride); set(a.ys, p->y_stride);
  a.state = state;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p->dtype == FLARE_F32) run_decode<float>(a, st);
  else if (p->dtype == FLARE_F16) run_decode<__half>(a, st);
  else run_decode<__nv_bfloat16>(a, st);
  const cudaError_t e = cudaPeekAtLastError();
  if (e != cudaSuccess) return refuse(FLARE_ECUDA, "decay_decode: %s", cudaGetErrorString(e));
  return FLARE_OK;
}

}  // extern "C"
