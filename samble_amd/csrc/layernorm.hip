// Layer normalisation, forward and backward, of (outer, C, inner) tensors over the middle axis:
//     s = x [+ residual],  mean, var over the C values,  xhat = (s - mean) rstd,  y = xhat weight + bias
//     g = dy weight:  ds = rstd (g - mean(g) - xhat mean(g xhat)) [+ gradient that reaches s itself]
//     dweight = sum dy xhat,  dbias = sum dy   over outer and inner
// fp32, fp16 or bf16 in and out; statistics and sums in fp32 from values held in registers: the mean first, then the squares
// of the differences (no sum of squares that cancels).  s is rounded to the tensors' type before it is normalised, so that
// the backward pass, which reads the rounded s, differentiates exactly what the forward computed.
//
// Every byte is touched once (forward: x [residual] in, y [s] out; backward: s, dy in, ds out): the kernels are bound by HBM.
//   inner == 1  rows of C contiguous values.  TPR threads own a row and keep it in registers, in P pieces of 16 bytes each:
//               TPR = 8 .. 64 inside a wave for narrow rows, 256 and 512 above.  Workgroups walk the rows and read the next
//               one ahead.  8192 x 4096 bf16: forward 24 us (5.6 TB/s, part of it from the caches), backward 38 + 4 us.
//   inner > 1   channel-major (B, C, N) tensors: 16 lanes (above 256 channels 8, above 512 4) stand along N (16 bytes each), the
//               other threads along C.
//               32 x 128 x 2048 fp32 with residual: forward 27 us (5.0 TB/s), backward 24.5 + 4 us (4.1 TB/s).
// Pieces are loaded at the alignment of one element, with one short piece at the end of an odd row (4099 x 5001 fp16 with
// residual: forward 36 us, 4.6 TB/s, backward 39 + 5 us; rows of 5000 take 3 % less).  Rows beyond what registers hold (16 384
// 16-bit or 8 192 fp32 values) take the *_loop kernels that read them again from the caches.
// Weight gradients: each workgroup adds its rows in registers and LDS and leaves one line of partial sums; ln_reduce_kernel
// adds the lines in a fixed order (no atomics: run to run identical).
#include "samble_dev.h"

namespace samble {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16;
typedef __bf16 bf16;

template <typename T> struct LnT;
template <> struct LnT<float> { static constexpr int V = 4; typedef u32x4 __attribute__((aligned(4))) piece; };
template <> struct LnT<f16> { static constexpr int V = 8; typedef u32x4 __attribute__((aligned(2))) piece; };
template <> struct LnT<bf16> { static constexpr int V = 8; typedef u32x4 __attribute__((aligned(2))) piece; };

// n of the piece's V values at p (n <= 0: none); the rest are zero
template <typename T>
__device__ __forceinline__ void ln_load(const T* p, long n, float (&v)[LnT<T>::V]) {
  constexpr int V = LnT<T>::V;
  typedef T vec __attribute__((ext_vector_type(V)));
  if (n >= V) {
    const u32x4 raw = *reinterpret_cast<const typename LnT<T>::piece*>(p);
    const vec t = __builtin_bit_cast(vec, raw);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (float)t[e];
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = e < n ? (float)p[e] : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void ln_store(T* p, long n, const float (&v)[LnT<T>::V]) {
  constexpr int V = LnT<T>::V;
  typedef T vec __attribute__((ext_vector_type(V)));
  if (n >= V) {
    vec t;
#pragma unroll
    for (int e = 0; e < V; ++e) t[e] = (T)v[e];
    *reinterpret_cast<typename LnT<T>::piece*>(p) = __builtin_bit_cast(u32x4, t);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < n) p[e] = (T)v[e];
  }
}
// a piece as it stands in memory, and its values: for what is read ahead (4 registers a piece whatever the type)
template <typename T>
__device__ __forceinline__ u32x4 ln_piece(const T* p, long n) {
  constexpr int V = LnT<T>::V;
  typedef T vec __attribute__((ext_vector_type(V)));
  if (n >= V) return *reinterpret_cast<const typename LnT<T>::piece*>(p);
  vec t;
#pragma unroll
  for (int e = 0; e < V; ++e) t[e] = e < n ? p[e] : (T)0.f;
  return __builtin_bit_cast(u32x4, t);
}
template <typename T>
__device__ __forceinline__ void ln_widen(const u32x4& raw, float (&v)[LnT<T>::V]) {
  constexpr int V = LnT<T>::V;
  typedef T vec __attribute__((ext_vector_type(V)));
  const vec t = __builtin_bit_cast(vec, raw);
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = (float)t[e];
}
// weight / bias: fp32 or the tensors' type (one uniform branch); null: `none`
template <typename T>
__device__ __forceinline__ void ln_load_w(const void* w, int w_f32, long c, long n, float none, float (&v)[LnT<T>::V]) {
  constexpr int V = LnT<T>::V;
  if (!w) {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = none;
  } else if (w_f32) {
    const float* p = (const float*)w + c;
    if (n >= V) {
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = p[e];
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = e < n ? p[e] : 0.f;
    }
  } else {
    ln_load<T>((const T*)w + c, n, v);
  }
}
template <typename T>
__device__ __forceinline__ float ln_w1(const void* w, int w_f32, long c, float none) {
  return !w ? none : w_f32 ? ((const float*)w)[c] : (float)((const T*)w)[c];
}

// sums of two values over the TPR threads of a row; every thread of the row gets both.  TPR <= 64: inside the wave
// (`red` unused); above: the waves' sums meet in LDS.  Two barriers: `red` may be reused at once.
template <int TPR>
__device__ __forceinline__ void ln_sum2(float& a, float& b, float* red) {
#pragma unroll
  for (int o = (TPR < 64 ? TPR : 64) / 2; o; o >>= 1) {
    a += __shfl_xor(a, o, 64);
    b += __shfl_xor(b, o, 64);
  }
  if constexpr (TPR > 64) {
    constexpr int NW = TPR / 64;
    const int w = (threadIdx.x % TPR) >> 6;
    if ((threadIdx.x & 63) == 0) {
      red[w] = a;
      red[NW + w] = b;
    }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      a += red[i];
      b += red[NW + i];
    }
    __syncthreads();
  }
}

struct LnArgs {
  const void *x, *res, *w, *b, *dy, *extra;   // extra: gradient that reaches s from elsewhere (backward)
  void *y, *s;                                // forward outputs; backward: y = ds
  float *mean, *rstd, *part;                  // part: (lines, 2, C) partial sums of dweight, dbias
  long outer, inner;                          // rows; columns of a channel-major slice
  long x_os, res_os, dy_os, ex_os;            // strides of the outer axis
  long x_cs, res_cs, dy_cs, ex_cs;            // strides of the channel axis (inner > 1)
  int C, w_f32;
  float eps;
};

// ---- rows (inner == 1) ---------------------------------------------------------------------------------------------------
// A workgroup walks the rows blockIdx.x * RPB + slot, + gridDim.x * RPB, ...  The columns of a thread stay the same, so that
// weight and bias stay in its registers, and the next row is read while the sums of this one are formed.
template <typename T, int TPR, int P>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void ln_rows_fwd_kernel(LnArgs A) {
  constexpr int V = LnT<T>::V, NT = TPR > 256 ? TPR : 256, RPB = NT / TPR;
  __shared__ float red[2 * (TPR > 64 ? TPR / 64 : 1)];
  const int t = threadIdx.x % TPR;
  const long step = (long)gridDim.x * RPB;
  long row = (long)blockIdx.x * RPB + threadIdx.x / TPR;
  u32x4 xr[P], rr[P];
  auto fetch = [&](long row) {
    const long at = row < A.outer ? row : 0;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const long c = (long)(p * TPR + t) * V, n = row < A.outer ? A.C - c : 0;
      xr[p] = ln_piece<T>((const T*)A.x + at * A.x_os + c, n);
      if (A.res) rr[p] = ln_piece<T>((const T*)A.res + at * A.res_os + c, n);
    }
  };
  fetch(row);
  float w[P][V], b[P][V];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const long c = (long)(p * TPR + t) * V;
    ln_load_w<T>(A.w, A.w_f32, c, A.C - c, 1.f, w[p]);
    ln_load_w<T>(A.b, A.w_f32, c, A.C - c, 0.f, b[p]);
  }
  const float cc = (float)A.C;
  for (long r0 = (long)blockIdx.x * RPB; r0 < A.outer; r0 += step, row += step) {
    const bool live = row < A.outer;      // (uniform over the threads of a row; a workgroup per row has no dead rows)
    float v[P][V];
    float sum = 0.f, sq = 0.f;
#pragma unroll
    for (int p = 0; p < P; ++p) ln_widen<T>(xr[p], v[p]);
    if (A.res) {
      T* s = (T*)A.s + (live ? row : 0) * A.C;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const long c = (long)(p * TPR + t) * V;
        float q[V];
        ln_widen<T>(rr[p], q);
#pragma unroll
        for (int e = 0; e < V; ++e) v[p][e] = (float)(T)(v[p][e] + q[e]);
        ln_store<T>(s + c, live ? A.C - c : 0, v[p]);
      }
    }
    if (r0 + step < A.outer) fetch(row + step);
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int e = 0; e < V; ++e) sum += v[p][e];
    ln_sum2<TPR>(sum, sq, red);
    const float mean = sum / cc;   // (a quotient: a constant row has its own value as mean)
    sq = 0.f;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const long c = (long)(p * TPR + t) * V;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        v[p][e] -= mean;
        if (c + e < A.C) sq = fmaf(v[p][e], v[p][e], sq);
      }
    }
    sum = 0.f;
    ln_sum2<TPR>(sq, sum, red);
    const float rstd = 1.f / sqrtf(sq / cc + A.eps);
    if (!live) continue;
    if (t == 0 && A.mean) {
      A.mean[row] = mean;
      A.rstd[row] = rstd;
    }
    T* y = (T*)A.y + row * A.C;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const long c = (long)(p * TPR + t) * V;
      float o[V];
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = fmaf(v[p][e] * rstd, w[p][e], b[p][e]);
      ln_store<T>(y + c, A.C - c, o);
    }
  }
}

// The same walk; the weight gradients add up in a thread's registers, then over the workgroup's rows in LDS, and leave one
// line of partial sums.
constexpr int ln_bwd_threads(int tpr) { return tpr > 512 ? tpr : 512; }

template <typename T, int TPR, int P, bool WG>
__global__ __launch_bounds__(ln_bwd_threads(TPR)) void ln_rows_bwd_kernel(LnArgs A) {
  constexpr int V = LnT<T>::V, NT = ln_bwd_threads(TPR), RPB = NT / TPR;
  constexpr int U = TPR >= 64 ? RPB : NT / 64, W = TPR * P * V;      // sums of the workgroup in LDS: units, columns
  __shared__ float red[RPB][2 * (TPR > 64 ? TPR / 64 : 1)];
  __shared__ float join[WG && U > 1 ? (U - 1) * W : 1];
  constexpr bool kAhead = P * V <= 24;      // (with four 16-bit pieces there are no registers for the next row's)
  const int t = threadIdx.x % TPR, slot = threadIdx.x / TPR;
  const long step = (long)gridDim.x * RPB;
  long row = (long)blockIdx.x * RPB + slot;
  u32x4 xr[P], gr[P];
  float mean, rstd;
  auto fetch = [&](long row) {
    const long at = row < A.outer ? row : 0;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const long c = (long)(p * TPR + t) * V, n = row < A.outer ? A.C - c : 0;
      xr[p] = ln_piece<T>((const T*)A.x + at * A.x_os + c, n);
      gr[p] = ln_piece<T>((const T*)A.dy + at * A.dy_os + c, n);
    }
    mean = A.mean[at];
    rstd = A.rstd[at];
  };
  if (kAhead) fetch(row);
  float w[P][V], dw[P][V], db[P][V];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const long c = (long)(p * TPR + t) * V;
    ln_load_w<T>(A.w, A.w_f32, c, A.C - c, 1.f, w[p]);
#pragma unroll
    for (int e = 0; e < V; ++e) dw[p][e] = db[p][e] = 0.f;
  }
  const float inv = 1.f / (float)A.C;
  for (long r0 = (long)blockIdx.x * RPB; r0 < A.outer; r0 += step, row += step) {
    if (!kAhead) fetch(row);
    float v[P][V], g[P][V];
    float s1 = 0.f, s2 = 0.f;
    const float rs = rstd;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      ln_widen<T>(xr[p], v[p]);
      ln_widen<T>(gr[p], g[p]);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float xh = (v[p][e] - mean) * rs;   // (behind the row's end and in missing rows g = 0: no sum sees it)
        v[p][e] = xh;
        if (WG) {
          dw[p][e] = fmaf(g[p][e], xh, dw[p][e]);
          db[p][e] += g[p][e];
        }
        g[p][e] *= w[p][e];
        s1 += g[p][e];
        s2 = fmaf(g[p][e], xh, s2);
      }
    }
    if (kAhead && r0 + step < A.outer) fetch(row + step);
    ln_sum2<TPR>(s1, s2, red[slot]);
    s1 *= inv;
    s2 *= inv;
    if (row >= A.outer) continue;   // (the barriers of the sums are passed by all threads of the workgroup)
    T* dx = (T*)A.y + row * A.C;
    const T* ex = A.extra ? (const T*)A.extra + row * A.ex_os : nullptr;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const long c = (long)(p * TPR + t) * V, n = A.C - c;
      if (n <= 0) break;
      float o[V];
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = rs * (g[p][e] - s1 - v[p][e] * s2);
      if (ex) {
        float q[V];
        ln_load<T>(ex + c, n, q);
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] += q[e];
      }
      ln_store<T>(dx + c, n, o);
    }
  }
  if constexpr (WG) {
    const int unit = TPR >= 64 ? slot : threadIdx.x >> 6;
    const bool lead = TPR >= 64 || (threadIdx.x & 63) < TPR;
    float* line = A.part + (long)blockIdx.x * 2 * A.C;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int p = 0; p < P; ++p) {
        float a[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          a[e] = k ? db[p][e] : dw[p][e];
#pragma unroll
          for (int o = TPR; o < 64; o <<= 1) a[e] += __shfl_xor(a[e], o, 64);
          if (k) db[p][e] = a[e];
          else dw[p][e] = a[e];
        }
        if (U > 1 && unit && lead) {
#pragma unroll
          for (int e = 0; e < V; ++e) join[(unit - 1) * W + (p * V + e) * TPR + t] = a[e];
        }
      }
      if (U > 1) __syncthreads();
      if (unit == 0 && lead) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
          const long c = (long)(p * TPR + t) * V;
#pragma unroll
          for (int e = 0; e < V; ++e) {
            float a = k ? db[p][e] : dw[p][e];
            for (int u = 1; u < U; ++u) a += join[(u - 1) * W + (p * V + e) * TPR + t];
            if (c + e < A.C) line[k * A.C + c + e] = a;
          }
        }
      }
      if (U > 1) __syncthreads();
    }
  }
}

// any width: one workgroup of 1024 threads per row, the row read once per step (mean, deviations, output)
template <typename T>
__global__ __launch_bounds__(1024) void ln_rows_fwd_loop_kernel(LnArgs A) {
  __shared__ float red[32];
  for (long row = blockIdx.x; row < A.outer; row += gridDim.x) {
  const T* x = (const T*)A.x + row * A.x_os;
  const T* r = A.res ? (const T*)A.res + row * A.res_os : nullptr;
  T* s = A.res ? (T*)A.s + row * A.C : nullptr;
  float sum = 0.f, sq = 0.f;
  for (int c = threadIdx.x; c < A.C; c += 1024) {
    float v = (float)x[c];
    if (r) {
      const T q = (T)(v + (float)r[c]);
      s[c] = q;
      v = (float)q;
    }
    sum += v;
  }
  ln_sum2<1024>(sum, sq, red);
  const T* src = r ? s : x;   // (a thread reads back only what it wrote itself)
  const float mean = sum / (float)A.C;
  sq = 0.f;
  for (int c = threadIdx.x; c < A.C; c += 1024) {
    const float d = (float)src[c] - mean;
    sq = fmaf(d, d, sq);
  }
  sum = 0.f;
  ln_sum2<1024>(sq, sum, red);
  const float rstd = 1.f / sqrtf(sq / (float)A.C + A.eps);
  if (threadIdx.x == 0 && A.mean) {
    A.mean[row] = mean;
    A.rstd[row] = rstd;
  }
  T* y = (T*)A.y + row * A.C;
  for (int c = threadIdx.x; c < A.C; c += 1024) {
    const float w = ln_w1<T>(A.w, A.w_f32, c, 1.f), b = ln_w1<T>(A.b, A.w_f32, c, 0.f);
    y[c] = (T)fmaf(((float)src[c] - mean) * rstd, w, b);
  }
  }
}

template <typename T>
__global__ __launch_bounds__(1024) void ln_rows_bwd_loop_kernel(LnArgs A) {
  __shared__ float red[32];
  for (long row = blockIdx.x; row < A.outer; row += gridDim.x) {
  const T* x = (const T*)A.x + row * A.x_os;
  const T* dy = (const T*)A.dy + row * A.dy_os;
  const float mean = A.mean[row], rstd = A.rstd[row];
  float s1 = 0.f, s2 = 0.f;
  for (int c = threadIdx.x; c < A.C; c += 1024) {
    const float w = ln_w1<T>(A.w, A.w_f32, c, 1.f);
    const float g = (float)dy[c] * w;
    s1 += g;
    s2 = fmaf(g, ((float)x[c] - mean) * rstd, s2);
  }
  ln_sum2<1024>(s1, s2, red);
  s1 /= (float)A.C;
  s2 /= (float)A.C;
  T* dx = (T*)A.y + row * A.C;
  const T* ex = A.extra ? (const T*)A.extra + row * A.ex_os : nullptr;
  for (int c = threadIdx.x; c < A.C; c += 1024) {
    const float w = ln_w1<T>(A.w, A.w_f32, c, 1.f);
    const float o = rstd * ((float)dy[c] * w - s1 - ((float)x[c] - mean) * rstd * s2);
    dx[c] = (T)(ex ? o + (float)ex[c] : o);
  }
  }
}

// dweight / dbias of the same: a thread per column, the rows blockIdx.y, + gridDim.y, ...
template <typename T>
__global__ __launch_bounds__(256) void ln_rows_wgrad_loop_kernel(LnArgs A) {
  const long c = (long)blockIdx.x * 256 + threadIdx.x;
  if (c >= A.C) return;
  float dw = 0.f, db = 0.f;
  for (long row = blockIdx.y; row < A.outer; row += gridDim.y) {
    const float g = (float)((const T*)A.dy)[row * A.dy_os + c];
    dw = fmaf(g, ((float)((const T*)A.x)[row * A.x_os + c] - A.mean[row]) * A.rstd[row], dw);
    db += g;
  }
  float* line = A.part + (long)blockIdx.y * 2 * A.C;
  line[c] = dw;
  line[A.C + c] = db;
}

// ---- channel-major (inner > 1) -------------------------------------------------------------------------------------------
// A workgroup: TN lanes along N (V values each), TC threads along C with channels tc, tc + TC, ...  The pieces stay in
// registers as they were read (4 registers a piece whatever the type); they are widened where they are used.
// sums over the TC threads of every column (K sums of V columns per thread), the same value in every thread
template <int TN, int TC, int KV>
__device__ __forceinline__ void ln_colsum(float (&a)[KV], float* red) {
  constexpr int NW = TN * TC / 64;
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, tn = lane % TN;
#pragma unroll
  for (int o = TN; o < 64; o <<= 1)
#pragma unroll
    for (int e = 0; e < KV; ++e) a[e] += __shfl_xor(a[e], o, 64);
  if (lane < TN) {
#pragma unroll
    for (int e = 0; e < KV; ++e) red[(w * KV + e) * TN + tn] = a[e];
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < KV; ++e) a[e] = 0.f;
  for (int i = 0; i < NW; ++i)
#pragma unroll
    for (int e = 0; e < KV; ++e) a[e] += red[(i * KV + e) * TN + tn];
  __syncthreads();
}

template <typename T, int TN, int TC, int P>
__global__ __launch_bounds__(TN * TC) void ln_chan_fwd_kernel(LnArgs A) {
  constexpr int V = LnT<T>::V;
  __shared__ float red[(TN * TC / 64) * V * TN];
  const int tn = threadIdx.x % TN, tc = threadIdx.x / TN;
  const long per = (A.inner + TN * V - 1) / (TN * V), tiles = per * A.outer;
  for (long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
  const long b = tile / per, n0 = (tile % per) * (TN * V) + tn * V, left = A.inner - n0;
  const T* x = (const T*)A.x + b * A.x_os + n0;
  const long oc = A.inner, ob = b * A.C * A.inner + n0;
  u32x4 raw[P];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int c = p * TC + tc;
    raw[p] = ln_piece<T>(x + (c < A.C ? c : 0) * A.x_cs, c < A.C ? left : 0);
  }
  if (A.res) {
    const T* r = (const T*)A.res + b * A.res_os + n0;
    T* s = (T*)A.s + ob;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int c = p * TC + tc;
      const long n = c < A.C ? left : 0;
      const u32x4 rr = ln_piece<T>(r + (c < A.C ? c : 0) * A.res_cs, n);
      float u[V], q[V];
      ln_widen<T>(raw[p], u);
      ln_widen<T>(rr, q);
      typedef T vec __attribute__((ext_vector_type(V)));
      vec t;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        u[e] += q[e];
        t[e] = (T)u[e];
      }
      raw[p] = __builtin_bit_cast(u32x4, t);
      if (c < A.C) ln_store<T>(s + c * oc, n, u);
    }
  }
  float m[V], q[V];
#pragma unroll
  for (int e = 0; e < V; ++e) m[e] = q[e] = 0.f;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    float u[V];
    ln_widen<T>(raw[p], u);
#pragma unroll
    for (int e = 0; e < V; ++e) m[e] += u[e];
  }
  ln_colsum<TN, TC, V>(m, red);
  const float cc = (float)A.C;
#pragma unroll
  for (int e = 0; e < V; ++e) m[e] /= cc;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    if (p * TC + tc >= A.C) continue;
    float u[V];
    ln_widen<T>(raw[p], u);
#pragma unroll
    for (int e = 0; e < V; ++e) q[e] = fmaf(u[e] - m[e], u[e] - m[e], q[e]);
  }
  ln_colsum<TN, TC, V>(q, red);
#pragma unroll
  for (int e = 0; e < V; ++e) q[e] = 1.f / sqrtf(q[e] / cc + A.eps);
  if (left <= 0) continue;
  if (tc == 0 && A.mean) {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < left) {
        A.mean[b * A.inner + n0 + e] = m[e];
        A.rstd[b * A.inner + n0 + e] = q[e];
      }
  }
  T* y = (T*)A.y + ob;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int c = p * TC + tc;
    if (c >= A.C) continue;
    const float w = ln_w1<T>(A.w, A.w_f32, c, 1.f), bb = ln_w1<T>(A.b, A.w_f32, c, 0.f);
    float u[V];
    ln_widen<T>(raw[p], u);
#pragma unroll
    for (int e = 0; e < V; ++e) u[e] = fmaf((u[e] - m[e]) * q[e], w, bb);
    ln_store<T>(y + c * oc, left, u);
  }
  }
}

template <typename T, int TN, int TC, int P>
__global__ __launch_bounds__(TN * TC) void ln_chan_bwd_kernel(LnArgs A) {
  constexpr int V = LnT<T>::V;
  __shared__ float red[(TN * TC / 64) * 2 * V * TN];
  const int tn = threadIdx.x % TN, tc = threadIdx.x / TN;
  const long per = (A.inner + TN * V - 1) / (TN * V), tiles = per * A.outer;
  const float inv = 1.f / (float)A.C;
  float dw[P], db[P];
#pragma unroll
  for (int p = 0; p < P; ++p) dw[p] = db[p] = 0.f;
  for (long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const long b = tile / per, n0 = (tile % per) * (TN * V) + tn * V, left = A.inner - n0;
    const T* x = (const T*)A.x + b * A.x_os + n0;
    const T* dy = (const T*)A.dy + b * A.dy_os + n0;
    u32x4 xr[P], gr[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int c = p * TC + tc;
      const long n = c < A.C ? left : 0;
      xr[p] = ln_piece<T>(x + (c < A.C ? c : 0) * A.x_cs, n);
      gr[p] = ln_piece<T>(dy + (c < A.C ? c : 0) * A.dy_cs, n);
    }
    float m[V], r[V], s[2 * V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      m[e] = e < left ? A.mean[b * A.inner + n0 + e] : 0.f;
      r[e] = e < left ? A.rstd[b * A.inner + n0 + e] : 0.f;
      s[e] = s[V + e] = 0.f;
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int c = p * TC + tc;
      const float w = c < A.C ? ln_w1<T>(A.w, A.w_f32, c, 1.f) : 0.f;
      float u[V], g[V];
      ln_widen<T>(xr[p], u);
      ln_widen<T>(gr[p], g);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float xh = (u[e] - m[e]) * r[e];
        dw[p] = fmaf(g[e], xh, dw[p]);
        db[p] += g[e];
        s[e] = fmaf(g[e], w, s[e]);
        s[V + e] = fmaf(g[e] * w, xh, s[V + e]);
      }
    }
    ln_colsum<TN, TC, 2 * V>(s, red);
    if (left > 0) {
      const long oc = A.inner;
      T* dx = (T*)A.y + b * A.C * A.inner + n0;
      const T* ex = A.extra ? (const T*)A.extra + b * A.ex_os + n0 : nullptr;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int c = p * TC + tc;
        if (c >= A.C) continue;
        const float w = ln_w1<T>(A.w, A.w_f32, c, 1.f);
        float u[V], g[V];
        ln_widen<T>(xr[p], u);
        ln_widen<T>(gr[p], g);
#pragma unroll
        for (int e = 0; e < V; ++e)
          u[e] = r[e] * (g[e] * w - s[e] * inv - (u[e] - m[e]) * r[e] * (s[V + e] * inv));
        if (ex) {
          ln_widen<T>(ln_piece<T>(ex + c * A.ex_cs, left), g);
#pragma unroll
          for (int e = 0; e < V; ++e) u[e] += g[e];
        }
        ln_store<T>(dx + c * oc, left, u);
      }
    }
  }
  if (!A.part) return;
  float* line = A.part + (long)blockIdx.x * 2 * A.C;
#pragma unroll
  for (int p = 0; p < P; ++p) {
#pragma unroll
    for (int o = 1; o < TN; o <<= 1) {
      dw[p] += __shfl_xor(dw[p], o, 64);
      db[p] += __shfl_xor(db[p], o, 64);
    }
    const int c = p * TC + tc;
    if (tn == 0 && c < A.C) {
      line[c] = dw[p];
      line[A.C + c] = db[p];
    }
  }
}

// any channel count: a thread per column, the channels read once per step
template <typename T>
__global__ __launch_bounds__(256) void ln_chan_fwd_loop_kernel(LnArgs A) {
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < A.outer * A.inner; i += (long)gridDim.x * 256) {
  const long b = i / A.inner, n = i % A.inner;
  const T* x = (const T*)A.x + b * A.x_os + n;
  const T* r = A.res ? (const T*)A.res + b * A.res_os + n : nullptr;
  T* s = A.res ? (T*)A.s + b * A.C * A.inner + n : nullptr;
  float sum = 0.f, sq = 0.f;
  for (int c = 0; c < A.C; ++c) {
    float v = (float)x[c * A.x_cs];
    if (r) {
      const T q = (T)(v + (float)r[c * A.res_cs]);
      s[c * A.inner] = q;
      v = (float)q;
    }
    sum += v;
  }
  const T* src = r ? s : x;
  const long cs = r ? A.inner : A.x_cs;
  const float mean = sum / (float)A.C;
  for (int c = 0; c < A.C; ++c) {
    const float d = (float)src[c * cs] - mean;
    sq = fmaf(d, d, sq);
  }
  const float rstd = 1.f / sqrtf(sq / (float)A.C + A.eps);
  if (A.mean) {
    A.mean[i] = mean;
    A.rstd[i] = rstd;
  }
  T* y = (T*)A.y + b * A.C * A.inner + n;
  for (int c = 0; c < A.C; ++c)
    y[c * A.inner] = (T)fmaf(((float)src[c * cs] - mean) * rstd, ln_w1<T>(A.w, A.w_f32, c, 1.f), ln_w1<T>(A.b, A.w_f32, c, 0.f));
  }
}

template <typename T>
__global__ __launch_bounds__(256) void ln_chan_bwd_loop_kernel(LnArgs A) {
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < A.outer * A.inner; i += (long)gridDim.x * 256) {
  const long b = i / A.inner, n = i % A.inner;
  const T* x = (const T*)A.x + b * A.x_os + n;
  const T* dy = (const T*)A.dy + b * A.dy_os + n;
  const float mean = A.mean[i], rstd = A.rstd[i];
  float s1 = 0.f, s2 = 0.f;
  for (int c = 0; c < A.C; ++c) {
    const float g = (float)dy[c * A.dy_cs] * ln_w1<T>(A.w, A.w_f32, c, 1.f);
    s1 += g;
    s2 = fmaf(g, ((float)x[c * A.x_cs] - mean) * rstd, s2);
  }
  s1 /= (float)A.C;
  s2 /= (float)A.C;
  T* dx = (T*)A.y + b * A.C * A.inner + n;
  const T* ex = A.extra ? (const T*)A.extra + b * A.ex_os + n : nullptr;
  for (int c = 0; c < A.C; ++c) {
    const float g = (float)dy[c * A.dy_cs] * ln_w1<T>(A.w, A.w_f32, c, 1.f);
    const float o = rstd * (g - s1 - ((float)x[c * A.x_cs] - mean) * rstd * s2);
    dx[c * A.inner] = (T)(ex ? o + (float)ex[c * A.ex_cs] : o);
  }
  }
}

// a wave per (channel, slice blockIdx.y of the columns)
template <typename T>
__global__ __launch_bounds__(256) void ln_chan_wgrad_loop_kernel(LnArgs A) {
  const long c = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (c >= A.C) return;
  float dw = 0.f, db = 0.f;
  for (long i = (long)blockIdx.y * 64 + (threadIdx.x & 63); i < A.outer * A.inner; i += (long)gridDim.y * 64) {
    const long b = i / A.inner, n = i % A.inner;
    const float g = (float)((const T*)A.dy)[b * A.dy_os + c * A.dy_cs + n];
    dw = fmaf(g, ((float)((const T*)A.x)[b * A.x_os + c * A.x_cs + n] - A.mean[i]) * A.rstd[i], dw);
    db += g;
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    dw += __shfl_xor(dw, o, 64);
    db += __shfl_xor(db, o, 64);
  }
  if ((threadIdx.x & 63) == 0) {
    float* line = A.part + (long)blockIdx.y * 2 * A.C;
    line[c] = dw;
    line[A.C + c] = db;
  }
}

// dweight, dbias = sums of the lines: 32 columns and 32 slices of the lines per workgroup, added in index order
template <typename T>
__global__ __launch_bounds__(1024) void ln_reduce_kernel(const float* __restrict__ part, long lines, int C, int w_f32, void* dw,
                                                         void* db) {
  __shared__ float red[32][33];
  const int cl = threadIdx.x & 31, sl = threadIdx.x >> 5;
  const long col = (long)blockIdx.x * 32 + cl, cols = 2l * C;
  float a = 0.f;
  if (col < cols) {
    const long step = (lines + 31) / 32, l0 = sl * step, l1 = l0 + step < lines ? l0 + step : lines;
    long l = l0;
    for (; l + 8 <= l1; l += 8) {   // eight loads in flight
      float u[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) u[k] = part[(l + k) * cols + col];
#pragma unroll
      for (int k = 0; k < 8; ++k) a += u[k];
    }
    for (; l < l1; ++l) a += part[l * cols + col];
  }
  red[sl][cl] = a;
  __syncthreads();
  if (sl == 0 && col < cols) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) t += red[k][cl];
    void* out = col < C ? dw : db;
    const long c = col < C ? col : col - C;
    if (!out) return;
    if (w_f32) ((float*)out)[c] = t;
    else ((T*)out)[c] = (T)t;
  }
}

// ---- launches -------------------------------------------------------------------------------------------------------------
// Threads per row and pieces per thread of a width: up to 128 pieces (2 KB rows) stay inside a wave, which needs no barrier;
// wider rows take 256, then 512 threads (the backward's registers: three fp32 arrays beside the two tensors' rows and the next
// ones' end at three pieces of 16-bit values; the widest rows are not read ahead.  4096 x 8192 bf16, backward: 512 threads of
// two pieces 53 us, 256 of four 77 us).
struct LnPlan { int tpr, p; };
static LnPlan ln_plan(int C, int V) {
  const long pieces = ((long)C + V - 1) / V;
  if (pieces <= 8) return {8, 1};
  if (pieces <= 16) return {16, 1};
  if (pieces <= 32) return {32, 1};
  if (pieces <= 64) return {64, 1};
  if (pieces <= 128) return {64, 2};
  if (pieces <= 256) return {256, 1};
  if (pieces <= 512) return {256, 2};
  if (pieces <= 768) return {256, 3};
  if (pieces <= 1024) return {512, 2};
  if (pieces <= 2048) return {512, 4};
  return {0, 0};
}
// Lanes along N: at most 512 threads in a workgroup, whose waves then have 256 registers (8 x 512 x 2048, backward: fp32 29 us, bf16
// 52 us; 1024 threads of 128 registers spill: 160 us, 176 us).  That is room for fp32; the backward of the 16-bit types, eight
// columns a thread, still spills 115 .. 126 registers in all three forms above 128 channels.
constexpr int ln_chan_lanes(int tc) { return tc > 32 ? 512 / tc : 16; }
static LnPlan ln_chan_plan(int C) {   // threads along C, pieces per thread
  if (C <= 16) return {16, 1};
  if (C <= 32) return {16, 2};
  if (C <= 64) return {16, 4};
  if (C <= 128) return {16, 8};
  if (C <= 256) return {32, 8};
  if (C <= 512) return {64, 8};
  if (C <= 1024) return {128, 8};
  return {0, 0};
}
constexpr long kLnGrid = 1 << 20;   // workgroups of a launch at most (a launch holds fewer than 2^32 threads): the kernels walk on
static unsigned ln_grid(long n) { return (unsigned)(n < kLnGrid ? n : kLnGrid); }
constexpr int kLnLoopLines = 128;
// Workgroups of a backward launch at most, each with a line of partial sums: two per CU, and one (of eight waves) for rows of
// two pieces a thread and more, whose next row in flight keeps memory busy and whose lines cost (8192 x 4096 bf16: 256 lines
// 38 + 4 us, 512 lines 45 + 4 us; one piece, 65 536 x 512 bf16: 40 us, 33 us).
constexpr int kLnLines = 512;
// workgroups for n units of work that walk on: at most `most`, each the same number of units
static long ln_even(long n, long most) {
  const long rounds = (n + most - 1) / most;
  return rounds ? (n + rounds - 1) / rounds : 0;
}

template <typename T> static long ln_lines(int C, long outer, long inner) {
  if (inner == 1) {
    const LnPlan pl = ln_plan(C, LnT<T>::V);
    if (!pl.tpr) return outer < kLnLoopLines ? outer : kLnLoopLines;
    const int rpb = ln_bwd_threads(pl.tpr) / pl.tpr;
    return ln_even((outer + rpb - 1) / rpb, pl.p > 1 ? kLnLines / 2 : kLnLines);
  }
  const LnPlan pl = ln_chan_plan(C);
  if (!pl.tpr) {
    const long need = (outer * inner + 63) / 64;
    return need < kLnLoopLines ? need : kLnLoopLines;
  }
  const int tn = ln_chan_lanes(pl.tpr);
  return ln_even(outer * ((inner + tn * LnT<T>::V - 1) / (tn * LnT<T>::V)), kLnLines);
}

template <typename T, int TPR, int P>
static int ln_rows(const LnArgs& A, bool bwd, hipStream_t s) {
  if (!bwd) {
    constexpr int NT = TPR > 256 ? TPR : 256, RPB = NT / TPR;
    // (as many as stand on the card at once: the registers of four pieces halve that)
    const unsigned grid = (unsigned)ln_even((A.outer + RPB - 1) / RPB, 256 * (P < 4 ? 2048 : 1024) / NT);
    hipLaunchKernelGGL((ln_rows_fwd_kernel<T, TPR, P>), dim3(grid), dim3(NT), 0, s, A);
  } else {
    constexpr int NT = ln_bwd_threads(TPR);
    const unsigned grid = (unsigned)ln_lines<T>(A.C, A.outer, 1);
    if (A.part) hipLaunchKernelGGL((ln_rows_bwd_kernel<T, TPR, P, true>), dim3(grid), dim3(NT), 0, s, A);
    else hipLaunchKernelGGL((ln_rows_bwd_kernel<T, TPR, P, false>), dim3(grid), dim3(NT), 0, s, A);
  }
  return (int)hipGetLastError();
}
template <typename T, int TN, int TC, int P>
static int ln_chan(const LnArgs& A, bool bwd, hipStream_t s) {
  constexpr int V = LnT<T>::V;
  const long tiles = A.outer * ((A.inner + TN * V - 1) / (TN * V));
  if (!bwd) hipLaunchKernelGGL((ln_chan_fwd_kernel<T, TN, TC, P>), dim3(ln_grid(tiles)), dim3(TN * TC), 0, s, A);
  else
    hipLaunchKernelGGL((ln_chan_bwd_kernel<T, TN, TC, P>), dim3((unsigned)ln_lines<T>(A.C, A.outer, A.inner)), dim3(TN * TC), 0,
                       s, A);
  return (int)hipGetLastError();
}

template <typename T>
static int ln_launch(const LnArgs& A, bool bwd, hipStream_t s) {
  if (A.inner == 1) {
    const LnPlan pl = ln_plan(A.C, LnT<T>::V);
    switch (pl.tpr * 8 + pl.p) {
      case 8 * 8 + 1: return ln_rows<T, 8, 1>(A, bwd, s);
      case 16 * 8 + 1: return ln_rows<T, 16, 1>(A, bwd, s);
      case 32 * 8 + 1: return ln_rows<T, 32, 1>(A, bwd, s);
      case 64 * 8 + 1: return ln_rows<T, 64, 1>(A, bwd, s);
      case 64 * 8 + 2: return ln_rows<T, 64, 2>(A, bwd, s);
      case 256 * 8 + 1: return ln_rows<T, 256, 1>(A, bwd, s);
      case 256 * 8 + 2: return ln_rows<T, 256, 2>(A, bwd, s);
      case 256 * 8 + 3: return ln_rows<T, 256, 3>(A, bwd, s);
      case 512 * 8 + 2: return ln_rows<T, 512, 2>(A, bwd, s);
      case 512 * 8 + 4: return ln_rows<T, 512, 4>(A, bwd, s);
    }
    if (!bwd) {
      hipLaunchKernelGGL((ln_rows_fwd_loop_kernel<T>), dim3(ln_grid(A.outer)), dim3(1024), 0, s, A);
    } else {
      // (the weight gradients first: the input's gradient may stand in dy's place)
      if (A.part)
        hipLaunchKernelGGL((ln_rows_wgrad_loop_kernel<T>), dim3((A.C + 255) / 256, (unsigned)ln_lines<T>(A.C, A.outer, 1)),
                           dim3(256), 0, s, A);
      hipLaunchKernelGGL((ln_rows_bwd_loop_kernel<T>), dim3(ln_grid(A.outer)), dim3(1024), 0, s, A);
    }
    return (int)hipGetLastError();
  }
  const LnPlan pl = ln_chan_plan(A.C);
  switch (pl.tpr * 8 + pl.p) {
    case 16 * 8 + 1: return ln_chan<T, 16, 16, 1>(A, bwd, s);
    case 16 * 8 + 2: return ln_chan<T, 16, 16, 2>(A, bwd, s);
    case 16 * 8 + 4: return ln_chan<T, 16, 16, 4>(A, bwd, s);
    case 16 * 8 + 8: return ln_chan<T, 16, 16, 8>(A, bwd, s);
    case 32 * 8 + 8: return ln_chan<T, 16, 32, 8>(A, bwd, s);
    case 64 * 8 + 8: return ln_chan<T, ln_chan_lanes(64), 64, 8>(A, bwd, s);
    case 128 * 8 + 8: return ln_chan<T, ln_chan_lanes(128), 128, 8>(A, bwd, s);
  }
  const unsigned grid = ln_grid((A.outer * A.inner + 255) / 256);
  if (!bwd) {
    hipLaunchKernelGGL((ln_chan_fwd_loop_kernel<T>), dim3(grid), dim3(256), 0, s, A);
  } else {
    if (A.part)      // (first, as above)
      hipLaunchKernelGGL((ln_chan_wgrad_loop_kernel<T>), dim3((A.C + 3) / 4, (unsigned)ln_lines<T>(A.C, A.outer, A.inner)),
                         dim3(256), 0, s, A);
    hipLaunchKernelGGL((ln_chan_bwd_loop_kernel<T>), dim3(grid), dim3(256), 0, s, A);
  }
  return (int)hipGetLastError();
}

}  // namespace samble

using namespace samble;

extern "C" size_t samble_ln_ws_bytes(int type, int C, long outer, long inner) {
  const long lines = type == 0 ? ln_lines<float>(C, outer, inner) : ln_lines<f16>(C, outer, inner);
  return (size_t)lines * 2 * C * sizeof(float);
}

extern "C" int samble_launch_ln_fwd(int type, int w_f32, const void* x, long x_os, long x_cs, const void* res, long res_os,
                                    long res_cs, const void* w, const void* b, long outer, int C, long inner, float eps, void* y,
                                    void* sum, float* mean, float* rstd, hipStream_t s) {
  LnArgs A = {};
  A.x = x; A.res = res; A.w = w; A.b = b; A.y = y; A.s = sum; A.mean = mean; A.rstd = rstd;
  A.outer = outer; A.inner = inner; A.x_os = x_os; A.x_cs = x_cs; A.res_os = res_os; A.res_cs = res_cs;
  A.C = C; A.w_f32 = w_f32; A.eps = eps;
  Timed timed(kT_ln_fwd, s);
  return type == 0 ? ln_launch<float>(A, false, s) : type == 1 ? ln_launch<f16>(A, false, s) : ln_launch<bf16>(A, false, s);
}

extern "C" int samble_launch_ln_bwd(int type, int w_f32, const void* x, long x_os, long x_cs, const void* dy, long dy_os,
                                    long dy_cs, const void* extra, long ex_os, long ex_cs, const void* w, const float* mean,
                                    const float* rstd, long outer, int C, long inner, void* dx, void* dw, void* db, float* ws,
                                    hipStream_t s) {
  LnArgs A = {};
  A.x = x; A.dy = dy; A.extra = extra; A.w = w; A.y = dx; A.mean = const_cast<float*>(mean); A.rstd = const_cast<float*>(rstd);
  A.outer = outer; A.inner = inner; A.x_os = x_os; A.x_cs = x_cs; A.dy_os = dy_os; A.dy_cs = dy_cs; A.ex_os = ex_os;
  A.ex_cs = ex_cs; A.C = C; A.w_f32 = w_f32;
  A.part = (dw || db) ? ws : nullptr;
  Timed timed(kT_ln_bwd, s);
  const int rc = type == 0 ? ln_launch<float>(A, true, s) : type == 1 ? ln_launch<f16>(A, true, s) : ln_launch<bf16>(A, true, s);
  if (rc || !A.part) return rc;
  const long lines = type == 0 ? ln_lines<float>(C, outer, inner) : ln_lines<f16>(C, outer, inner);
  const dim3 grid((2l * C + 31) / 32);
  if (type == 1) hipLaunchKernelGGL((ln_reduce_kernel<f16>), grid, dim3(1024), 0, s, A.part, lines, C, w_f32, dw, db);
  else hipLaunchKernelGGL((ln_reduce_kernel<bf16>), grid, dim3(1024), 0, s, A.part, lines, C, w_f32, dw, db);
  return (int)hipGetLastError();
}
