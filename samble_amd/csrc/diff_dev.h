// Shared parts of the differential-attention kernels (diff_attn_fwd.hip, diff_attn_bwd.hip).
//
//     P_m = softmax_j(scale <q_m_i, k_m_j>), m = 1, 2,    out_i = sum_j (P_1 - lam P_2)_ij v_j
//
// Rows.  The G = H / Hkv query heads that share a key head stand together: row r of a (batch item, key head) pair is query
// r / G of head hk G + r % G.  A key head's tiles are then read once for all its query heads, and the sums of shared heads'
// gradients are ordinary sums over rows.
//
// Products.  v_mfma_f32_32x32x16 on fp16 or bf16 operands, fp32 sums.  fp16 / bf16 tensors are operands as they are.  An fp32
// value is three bf16 planes, x = h + m + l, each the rounding of what the ones before it leave: 24 bits, none lost, at fp32's
// own exponents, so that no value depends on the size of its neighbours.  A product takes the six partial products down to
// 2^-16 of the first; the three left out are below 2^-23 of it.  (Two fp16 planes of scaled values take three products: 440
// instead of 600 us for the training step of 32 x 1024 x 4 heads of 16.  But a scale is shared, and what stands 2^20 below
// the largest value that shares it keeps 2^-18 of itself, nothing at 2^40.)  An infinity's or NaN's lower planes are NaN: all sums
// that it enters are NaN.
// Lane l holds
//     A: A[row = l & 31][k = 8 (l >> 5) + e],  B: B[k = 8 (l >> 5) + e][col = l & 31],  e = 0 .. 7
//     D: register r: D[row = crow(r, l >> 5)][col = l & 31]
// The reduced index of a second product stands on the first one's ROW axis: registers 8 t .. 8 t + 7 of a softmax tile are
// then the B operand of step t as they are, with the 16 reduced indices of the step in the order 4 h + {0..3},
// 8 + 4 h + {0..3} for lane half h; ds_read_b64_tr_b16 reads the A operand from row-major tiles in that order.  P and dS
// never leave registers.
//
// Tiles.  A tile is KT rows of two matrices X (two maps of DP elements) and Y (2 DP elements) of 16-bit operands, row-major in
// LDS, 16-byte pieces; NP planes of each.  The pieces of a 256-byte line stand at places turned by a function of the
// line: the four pieces of four rows that half of a transposing read takes fall on sixteen different places, sixteen rows' pieces
// of one column (a quarter of a wave's ds_read_b128) on eight.
#pragma once
#include "diff_args.h"
#include "samble_dev.h"

namespace samble {

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16;
typedef __bf16 bf16;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

template <typename T> struct DaT;      // operand type, planes; kP: the probabilities' scale 2^kP (fp16 operands: off the subnormals)
template <> struct DaT<float> { typedef bf16 E; static constexpr int NP = 3, kP = 0; };
template <> struct DaT<f16> { typedef f16 E; static constexpr int NP = 1, kP = 6; };
template <> struct DaT<bf16> { typedef bf16 E; static constexpr int NP = 1, kP = 0; };

template <typename E> using vec8 = E __attribute__((ext_vector_type(8)));
template <typename E> using vec4 = E __attribute__((ext_vector_type(4)));
template <typename E> using vec2 = E __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// a value that is the same in the whole wave, as one the scalar unit holds
__device__ __forceinline__ int da_uni(int x) { return __builtin_amdgcn_readfirstlane(x); }

__device__ __forceinline__ f32x16 da_mfma(vec8<bf16> a, vec8<bf16> b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 da_mfma(vec8<f16> a, vec8<f16> b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// an operand of eight values: NP planes
template <typename T> struct Frag { vec8<typename DaT<T>::E> p[DaT<T>::NP]; };

template <typename T>
__device__ __forceinline__ f32x16 da_mma(const Frag<T>& a, const Frag<T>& b, f32x16 c) {
  if constexpr (DaT<T>::NP == 1) {
    return da_mfma(a.p[0], b.p[0], c);
  } else {   // the small products first
    c = da_mfma(a.p[2], b.p[0], c);
    c = da_mfma(a.p[0], b.p[2], c);
    c = da_mfma(a.p[1], b.p[1], c);
    c = da_mfma(a.p[1], b.p[0], c);
    c = da_mfma(a.p[0], b.p[1], c);
    return da_mfma(a.p[0], b.p[0], c);
  }
}

// eight fp32 values as an operand.  fp16 / bf16: one rounding to the tensors' own type (half a step of the value; the sums
// that these factors enter stay in fp32); fp32: three planes, no bit lost.
template <typename T>
__device__ __forceinline__ Frag<T> da_pack(const float (&v)[8]) {
  typedef typename DaT<T>::E E;
  constexpr int NP = DaT<T>::NP;
  Frag<T> f;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    f32x2 x = {v[e], v[e + 1]};
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const vec2<E> h = __builtin_convertvector(x, vec2<E>);
      f.p[p][e] = h[0];
      f.p[p][e + 1] = h[1];
      if (p + 1 < NP) {
        x[0] -= (float)h[0];
        x[1] -= (float)h[1];
      }
    }
  }
  return f;
}

// fp16 operands of the backward, P and dS, are held times powers of two (2^11 steps at 2^13, 2^-25 at the low end: half a step is
// 2^-12 of a term as long as that is above 2^-27 of the largest one).
template <typename T> constexpr bool kDaScaled = __is_same(T, f16);
// the power of two that takes a value with these absolute bits to 2^12 .. 2^13 (0: far up)
__device__ __forceinline__ float da_scale(unsigned abs_bits) {
  const unsigned e = max(abs_bits >> 23, 13u);
  return __uint_as_float((266u - e) << 23);
}
// larger of two absolute bits, the second one only if it is finite (an infinity or NaN is one in all its sums, at any scale)
__device__ __forceinline__ unsigned da_max_bits(unsigned a, float x) {
  const unsigned u = __float_as_uint(x) & 0x7fffffffu;
  return u < 0x7f800000u && u > a ? u : a;
}

// eight contiguous values of a tensor, as they are read (held across a tile's computation); ok = false: zeros
template <typename T> struct Raw8;
template <> struct Raw8<float> {
  f32x4 v[2];
  __device__ __forceinline__ void load(const float* p, bool ok) {
    const f32x4 z = {0.f, 0.f, 0.f, 0.f};
    v[0] = ok ? *reinterpret_cast<const f32x4*>(p) : z;
    v[1] = ok ? *reinterpret_cast<const f32x4*>(p + 4) : z;
  }
  __device__ __forceinline__ Frag<float> frag() const {
    float t[8];
    widen(t);
    return da_pack<float>(t);
  }
  __device__ __forceinline__ void widen(float (&t)[8]) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = v[e >> 2][e & 3];
  }
};
template <typename T> struct Raw8 {
  vec8<T> v;
  __device__ __forceinline__ void load(const T* p, bool ok) {
    const u32x4 z = {0, 0, 0, 0};
    v = __builtin_bit_cast(vec8<T>, ok ? *reinterpret_cast<const u32x4*>(p) : z);
  }
  __device__ __forceinline__ Frag<T> frag() const { return Frag<T>{{v}}; }
  __device__ __forceinline__ void widen(float (&t)[8]) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = (float)v[e];
  }
};

// a lane's own row as KS operands (elements 16 s + 8 h .. of a row of n live ones)
template <typename T, int KS>
__device__ __forceinline__ void da_row(const T* p, int n, bool live, int h, Frag<T> (&f)[KS]) {
  Raw8<T> raw[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) raw[s].load(p + 16 * s + 8 * h, live && 16 * s + 8 * h < n);
#pragma unroll
  for (int s = 0; s < KS; ++s) f[s] = raw[s].frag();
}

// byte offset of piece c of a row of 2 DP 16-bit elements, and back from the e-th piece in LDS
template <int DP>
__device__ __forceinline__ int da_turn(int line) {     // what the places of a 256-byte line are turned by (bits 0, 2, 3)
  if constexpr (DP == 16) return line & 1;                                    // four rows a line
  else if constexpr (DP == 32) return ((line & 1) << 2) | ((line >> 1) & 1);  // two rows
  else if constexpr (DP == 64) return ((line & 3) << 2) | ((line >> 2) & 1);  // one row
  else return ((line & 6) << 1) | ((line >> 3) & 1);                          // half a row
}
template <int DP>
__device__ __forceinline__ int da_off(int row, int c) {
  const int e = row * (DP / 4) + c, line = e >> 4;
  return (line << 8) + (((e & 15) ^ da_turn<DP>(line)) << 4);
}
template <int DP>
__device__ __forceinline__ void da_place(int e, int& row, int& c) {
  const int line = e >> 4, q = line * 16 + ((e & 15) ^ da_turn<DP>(line));
  row = q / (DP / 4);
  c = q % (DP / 4);
}

// The LDS addresses a lane reads a tile's operands at: few registers, everything else is an offset of the instruction.
template <int DP>
struct Lane {
  static constexpr int NR = DP >= 64 ? 4 : DP / 16, NC = NR;
  unsigned r[NR], c[NC];
  // row0: the wave's first row of every tile (a multiple of 32)
  __device__ __forceinline__ Lane(int lane, int row0) {
    const int h = lane >> 5, i = lane & 15;
#pragma unroll
    for (int k = 0; k < NR; ++k) r[k] = da_off<DP>(lane & 31, 4 * k + h) + row0 * (4 * DP);
#pragma unroll
    for (int v = 0; v < NC; ++v)
      c[v] = da_off<DP>(4 * h + (i >> 2), 4 * v + 2 * ((lane >> 4) & 1) + ((i >> 1) & 1)) + 8 * (i & 1) + row0 * (4 * DP);
  }
  __device__ __forceinline__ void move(int bytes) {
#pragma unroll
    for (int k = 0; k < NR; ++k) r[k] += bytes;
#pragma unroll
    for (int v = 0; v < NC; ++v) c[v] += bytes;
  }
};

template <typename T, int DP, int KT>
struct Tile {
  static constexpr int NP = DaT<T>::NP;
  static constexpr int kPlane = KT * 4 * DP;          // bytes of one plane of X or Y
  static constexpr int kBytes = 2 * NP * kPlane;      // X planes, then Y planes
  typedef typename DaT<T>::E E;
  typedef __attribute__((address_space(3))) const vec8<E> lds_vec8;

  // A operand, 32 rows row0 .. row0 + 31 of the wave's (a multiple of 32), step ks of the 16-deep steps along the row; X: of
  // map m + (second, the same in the whole wave)
  static __device__ __forceinline__ Frag<T> rows(const Lane<DP>& L, int which, int row0, int ks) {
    return rows_at(L.r[(ks >> 1) & (Lane<DP>::NR - 1)], which * NP, row0, ks);
  }
  static __device__ __forceinline__ Frag<T> map_rows(const Lane<DP>& L, int m, int second, int row0, int ks) {
    constexpr int KS = DP / 16, N = Lane<DP>::NR - 1;
    const int a = m * KS + ks, b = a + KS;
    return rows_at(second ? L.r[(b >> 1) & N] : L.r[(a >> 1) & N], 0, row0, second ? b : a);
  }
  static __device__ __forceinline__ Frag<T> rows_at(unsigned at, int plane, int row0, int ks) {
    Frag<T> f;
    const int o = row0 * (4 * DP) + (ks & 1) * 32 + (ks >> 1) / Lane<DP>::NR * 256;
#pragma unroll
    for (int p = 0; p < NP; ++p) f.p[p] = *(lds_vec8*)(unsigned long)(at + (unsigned)((plane + p) * kPlane + o));
    return f;
  }
  // A operand of the transposed tile: 32 columns col0 .. (a multiple of 32), reduced rows row0 + 16 t + {4 h + 0..3,
  // 8 + 4 h + 0..3}
  static __device__ __forceinline__ Frag<T> cols(const Lane<DP>& L, int which, int row0, int t, int col0) {
    return cols_at(L.c[(col0 >> 5) & (Lane<DP>::NC - 1)], which, row0, t, col0);
  }
  static __device__ __forceinline__ Frag<T> cols_at(unsigned at, int which, int row0, int t, int col0) {
    Frag<T> f;
    const int o = (row0 + 16 * t) * (4 * DP) + col0 / 32 / Lane<DP>::NC * 256;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const unsigned b = at + (unsigned)((which * NP + p) * kPlane + o);
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(unsigned long)b);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(unsigned long)(b + 8 * 4 * DP));
      const vec4<E> x = __builtin_bit_cast(vec4<E>, lo), z = __builtin_bit_cast(vec4<E>, hi);
      f.p[p] = __builtin_shufflevector(x, z, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    return f;
  }
};

// sixteen zero bytes that pieces of rows which do not exist are copied from
__device__ __attribute__((aligned(16))) const unsigned da_zero[4] = {0, 0, 0, 0};

// rows r of the matrices X and Y, r in 0 .. n - 1 where mask (if any) is not 0; other rows are zero
template <typename T>
struct Rows {
  const T *x, *y;
  long x_ms;
  int x_rs, y_rs, n, d;
  const unsigned char* mask;
};

// Tiles on their way from memory to LDS, NT threads together, at LDS address 0.
//   fp16 / bf16: memory to LDS without registers (global_load_lds_dwordx4), two tiles: while one is computed on, the next
//   lands.  The 64 pieces of a wave's copy stand one behind the other in LDS, so the lane picks the piece that belongs there.
//   fp32: through registers, where the values are split into planes; one tile.
// use:  feed.issue(first, row0);  for each tile: { feed.next(L);  [feed.issue(following, row0)];  compute }
// next() is a barrier of the workgroup.
template <typename T, int DP, int KT, int NT>
struct Feed {
  typedef Tile<T, DP, KT> Tl;
  static constexpr bool DMA = Tl::NP == 1;
  static constexpr int kPieces = KT * DP / 4;                    // of X, and of Y
  static constexpr int kPer = (kPieces + NT - 1) / NT;
  static constexpr int kBufs = Tl::kBytes * (DMA ? 2 : 1);
  static constexpr int kLds = kBufs + 32;                        // the tiles, their visible rows (a bit each)
  static_assert(!DMA || kPieces % 64 == 0, "whole waves copy");
  static_assert(!DMA || NT % 256 == 0, "a thread's pieces stand at one place of their rows");
  static_assert(KT <= 128, "room for the visible rows");

  char* lds;
  int tid, wave, cur;       // cur: the buffer that next() left current
  bool bit;
  Raw8<T> x[DMA ? 1 : kPer], y[DMA ? 1 : kPer];

  __device__ __forceinline__ Feed(char* l, int t)
      : lds(l), tid(t), wave(da_uni(t >> 6)), cur(0), bit(false) {}

  __device__ __forceinline__ int after() const { return cur ^ 1; }      // the buffer that issue() fills
  __device__ __forceinline__ unsigned* words(int buf) const { return reinterpret_cast<unsigned*>(lds + kBufs) + 4 * buf; }
  __device__ __forceinline__ void write_words(int buf) {
    if (tid < KT) {
      const unsigned long long w = __ballot(bit);
      if ((tid & 31) == 0) words(buf)[tid >> 5] = (unsigned)(w >> (tid & 32));
    }
  }
  static __device__ __forceinline__ void copy16(const T* g, unsigned off, char* l) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)((const char*)g + off),
                                     (__attribute__((address_space(3))) void*)l, 16, 0, 0);
  }

  __device__ __forceinline__ void issue(const Rows<T>& R, int row0) {
    bit = tid < KT && row0 + tid < R.n && (!R.mask || R.mask[row0 + tid]);
    const T* xt = R.x + (long)row0 * R.x_rs;
    const T* yt = R.y + (long)row0 * R.y_rs;
    if constexpr (DMA) {
      int row, c;
      da_place<DP>(tid, row, c);
      const int map = c / (DP / 8), o = (c % (DP / 8)) * 8;
      // (byte offsets of a tile fit into 32 bits: rows are at most 2^23 elements apart, a map at most 2^28)
      const unsigned xo = (unsigned)(row * R.x_rs + map * (int)R.x_ms + o) * 2u, yo = (unsigned)(row * R.y_rs + c * 8) * 2u;
      constexpr int kRows = NT * 4 / DP;       // rows between a thread's pieces
      char* l = lds + after() * Tl::kBytes + 64 * wave * 16;
      if (R.d == DP && row0 + KT <= R.n && !R.mask) {      // uniform
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          if (kPieces % NT && 64 * wave + NT * i >= kPieces) break;
          copy16(xt + (long)i * kRows * R.x_rs, xo, l + NT * i * 16);
          copy16(yt + (long)i * kRows * R.y_rs, yo, l + NT * i * 16 + Tl::kPlane);
        }
      } else {
#pragma unroll 1
        for (int i = 0; i < kPer; ++i) {
          if (kPieces % NT && 64 * wave + NT * i >= kPieces) break;
          const int r = row0 + row + i * kRows;
          const bool ok = r < R.n && (!R.mask || R.mask[r]);
          const char *px = (const char*)(xt + (long)i * kRows * R.x_rs) + xo, *py = (const char*)(yt + (long)i * kRows * R.y_rs) + yo;
          copy16((const T*)(ok && o < R.d ? px : (const char*)da_zero), 0, l + NT * i * 16);
          copy16((const T*)(ok && c * 8 < 2 * R.d ? py : (const char*)da_zero), 0, l + NT * i * 16 + Tl::kPlane);
        }
      }
      write_words(after());
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int e = tid + NT * i;
        if (kPieces % NT && e >= kPieces) {
          x[i].load(nullptr, false);
          y[i].load(nullptr, false);
          continue;
        }
        const int row = e / (DP / 4), c = e % (DP / 4);
        const int map = c / (DP / 8), o = (c % (DP / 8)) * 8;
        const bool ok = row0 + row < R.n && (!R.mask || R.mask[row0 + row]);
        x[i].load(xt + (unsigned)(row * R.x_rs + map * (int)R.x_ms + o), ok && o < R.d);
        y[i].load(yt + (unsigned)(row * R.y_rs + c * 8), ok && c * 8 < 2 * R.d);
      }
    }
  }
  // the tile issued last, in LDS for every wave; every wave is done with the tile before it.  between(): run by every thread
  // before the last barrier
  template <typename F>
  __device__ __forceinline__ void next(Lane<DP>& L, F between) {
    if constexpr (DMA) {
      between();
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      const int was = cur;
      cur = after();
      L.move((cur - was) * Tl::kBytes);
    } else {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int e = tid + NT * i;
        if (kPieces % NT && e >= kPieces) break;
        const int o = da_off<DP>(e / (DP / 4), e % (DP / 4));
        const Frag<T> fx = x[i].frag(), fy = y[i].frag();
#pragma unroll
        for (int p = 0; p < Tl::NP; ++p) {
          *reinterpret_cast<vec8<typename Tl::E>*>(lds + p * Tl::kPlane + o) = fx.p[p];
          *reinterpret_cast<vec8<typename Tl::E>*>(lds + (Tl::NP + p) * Tl::kPlane + o) = fy.p[p];
        }
      }
      write_words(0);
      between();
      __syncthreads();
    }
  }
  __device__ __forceinline__ void next(Lane<DP>& L) {
    next(L, [] {});
  }
  // visible rows row0 .. row0 + 31 of the current tile, a bit each
  __device__ __forceinline__ unsigned word(int row0) const { return da_uni(words(DMA ? cur : 0)[row0 >> 5]); }
};

// c + the sum of eight operands (of one plane)
template <typename E>
__device__ __forceinline__ float da_sum8(const vec8<E>& v, float c) {
  const vec2<E> one = {(E)1.f, (E)1.f};
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const vec2<E> x = {v[e], v[e + 1]};
    if constexpr (__is_same(E, bf16)) c = __builtin_amdgcn_fdot2_f32_bf16(x, one, c, false);
    else c = __builtin_amdgcn_fdot2(x, one, c, false);
  }
  return c;
}

// whether row j + 4 h of a tile's 32 is visible, h the lane's half: the comparison's result made on the scalar unit
__device__ __forceinline__ bool da_bit(unsigned word, int j) {
  const unsigned lo = (unsigned)((int)(word << (31 - j)) >> 31), hi = (unsigned)((int)(word << (27 - j)) >> 31);
  return __builtin_amdgcn_inverse_ballot_w64(((unsigned long long)hi << 32) | lo);
}

// What rounding x to r leaves, in 2^-7 of half a step of the type: the difference of their fp32 encodings, which counts steps of
// fp32 (x and r have one sign), or where fp16's own steps end, 2^-24 apart, that of their values; an infinity leaves 0.  r and this
// byte give x to 2^-15 (bf16) or 2^-18 of itself, or to 2^-32.
template <typename T> constexpr int kDaRest = __is_same(T, bf16) ? 9 : 6;
template <typename T> __device__ __forceinline__ bool da_fixed(float r) { return __is_same(T, f16) && fabsf(r) < 0x1p-14f; }
template <typename T>
__device__ __forceinline__ int da_rest(float x, T r) {
  const float f = (float)r;
  const int off = (int)(__float_as_uint(x) - __float_as_uint(f)), most = 64 << kDaRest<T>;
  const int steps = off < -most || off > most ? 0 : (off + (1 << (kDaRest<T> - 1))) >> kDaRest<T>;
  return da_fixed<T>(f) ? (int)rintf((x - f) * 0x1p31f) : steps;
}
template <typename T>
__device__ __forceinline__ float da_whole(float r, int rest) {
  const float x = __uint_as_float(__float_as_uint(r) + ((unsigned)rest << kDaRest<T>));
  return da_fixed<T>(r) ? fmaf((float)rest, 0x1p-31f, r) : x;
}
// the pair of them of an element of out and one of out2
template <typename T>
__device__ __forceinline__ unsigned da_rests(float x, T rx, float y, T ry) {
  return (unsigned)((da_rest<T>(x, rx) & 255) | (da_rest<T>(y, ry) & 255) << 8);
}
// words 0, 1 and 2, 3 of the wave's lower half and of its upper half -> words 0, 1 of both in the lower lane, words 2, 3 of both in
// the upper one
__device__ __forceinline__ u32x4 da_halves(u32x4 w) {
  const auto a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false), b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
  const u32x4 r = {a[0], b[0], a[1], b[1]};
  return r;
}

template <typename T>
__device__ __forceinline__ float da_lam(const DaArgs& A, int head) {
  return A.lam_f32 ? ((const float*)A.lam)[head] : (float)((const T*)A.lam)[head];
}
// the position of batch item b's first query (keys <= position are seen), and its keys: under a causal mask those behind the
// last query's position do not exist either.  Both are taken into range here, so that no value of theirs reaches behind the
// tensors (sizes end at 2^30: beyond that, all or none)
__device__ __forceinline__ int da_start(const DaArgs& A, int b) {
  const int s = da_uni(A.q_start ? A.q_start[b] : A.Nk - A.Nq), far = (1 << 30) - 1;
  return s < -far - 2 ? -far - 2 : s > far ? far : s;
}
__device__ __forceinline__ int da_len(const DaArgs& A, int b, int start) {
  const int n = da_uni(A.lengths ? A.lengths[b] : A.Nk), end = A.causal && start + A.Nq < A.Nk ? start + A.Nq : A.Nk;
  return n < 0 || end < 0 ? 0 : n > end ? end : n;
}
// keys that query i sees
__device__ __forceinline__ int da_limit(const DaArgs& A, int len, int start, int i) {
  if (!A.causal) return len;
  const int n = start + i + 1;
  return n < 0 ? 0 : n > len ? len : n;
}

// This workgroup's block and (batch item, key head) pair, of B Hkv x `blocks` (fewer than 2^32); false: none.  Workgroups are
// dealt to the XCDs in turn; the blocks of a pair stand on one XCD, so that its tiles are read once into that XCD's L2.
//   pairs a multiple of 8   every eighth pair on an XCD: items of different lengths are dealt out evenly (32 items of 256 .. 2048
//                           keys, 8 heads of 64, bf16: dk and dv 1100 us, with neighbouring pairs on an XCD 1390 us); under a
//                           causal mask the longest blocks first, over all the XCD's pairs where these are few
//   spread                  the blocks of a pair on all XCDs: where the sweep is as long as the item and an XCD would have
//                           few items (8 items of one head, fp32: 93 us, 99 us)
__device__ __forceinline__ bool da_unit(const DaArgs& A, unsigned grid, unsigned blocks, bool spread, unsigned& blk, unsigned& pair) {
  const unsigned pairs = A.B * A.Hkv, x = blockIdx.x & 7, j = blockIdx.x >> 3;
  if (pairs % 8 == 0 && !spread) {
    const bool order = A.causal && pairs <= 64;
    const unsigned n = order ? pairs / 8 : blocks, q = da_uni(j / n), r = j - q * n;
    blk = order ? q : r;
    pair = 8 * (order ? r : q) + x;
    return blk < blocks && pair < pairs;
  }
  const unsigned unit = spread ? blockIdx.x : x * (grid / 8) + j;
  pair = da_uni(unit / blocks);
  blk = unit - pair * blocks;
  return pair < pairs;
}

__device__ __forceinline__ float da_xor32_sum(float x) {
  const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}

constexpr float kLog2e = 1.4426950408889634f;

}  // namespace samble
