// Shared parts of the differential-attention kernels (diff_attn_fwd.hip, diff_attn_bwd.hip).
//
//     P_m = softmax_j(scale <q_m_i, k_m_j>), m = 1, 2,    out_i = sum_j (P_1 - lam P_2)_ij v_j
//
// Rows.  The G = H / Hkv query heads that share a key head stand together: row r of a (batch item, key head) pair is query
// r / G of head hk G + r % G.  A key head's tiles are then read once for all its query heads, and the sums of shared heads'
// gradients are ordinary sums over rows.
//
// Products.  v_mfma_f32_32x32x16 on fp16 or bf16 operands, fp32 sums.  fp16 / bf16 tensors are operands as they are; an fp32
// tensor is split into three bf16 planes (x = h + m + l, 24 bits; bf16 has fp32's range, so no scale is needed) and a product
// takes the six partial products down to 2^-16 of the first: the error of an fp32 product.  Lane l holds
//     A: A[row = l & 31][k = 8 (l >> 5) + e],  B: B[k = 8 (l >> 5) + e][col = l & 31],  e = 0 .. 7
//     D: register r: D[row = crow(r, l >> 5)][col = l & 31]
// The reduced index of a second product stands on the first one's ROW axis: registers 8 t .. 8 t + 7 of a softmax tile are
// then the B operand of step t as they are, with the 16 reduced indices of the step in the order 4 h + {0..3},
// 8 + 4 h + {0..3} for lane half h; ds_read_b64_tr_b16 reads the A operand from row-major tiles in that order.  P and dS
// never leave registers.
//
// Tiles.  A tile is KT rows of two matrices X (two maps of DP elements) and Y (2 DP elements) of 16-bit operands, row-major in
// LDS, 16-byte pieces; NP planes of each.  Piece c of a row stands at place c ^ f(row): eight rows' pieces of one column (a
// ds_read_b128 of a wave's quarter) and four rows' pairs of pieces (a transposing read) both fall on eight different places
// of a 128-byte line.
#pragma once
#include "diff_args.h"
#include "samble_dev.h"

namespace samble {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16;
typedef __bf16 bf16;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

template <typename T> struct DaT;
template <> struct DaT<float> { typedef bf16 E; static constexpr int NP = 3; };
template <> struct DaT<f16> { typedef f16 E; static constexpr int NP = 1; };
template <> struct DaT<bf16> { typedef bf16 E; static constexpr int NP = 1; };

template <typename E> using vec8 = E __attribute__((ext_vector_type(8)));
template <typename E> using vec4 = E __attribute__((ext_vector_type(4)));

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
  Frag<T> f;
  if constexpr (DaT<T>::NP == 1) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f.p[0][e] = (E)v[e];
  } else {
    float r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      f.p[0][e] = (E)v[e];
      r[e] = v[e] - (float)f.p[0][e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      f.p[1][e] = (E)r[e];
      f.p[2][e] = (E)(r[e] - (float)f.p[1][e]);
    }
  }
  return f;
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
    const float t[8] = {v[0][0], v[0][1], v[0][2], v[0][3], v[1][0], v[1][1], v[1][2], v[1][3]};
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

// byte offset of piece c of a row of 2 DP 16-bit elements
template <int DP>
__device__ __forceinline__ int da_off(int row, int c) {
  if constexpr (DP == 16) {   // two rows of four pieces on a 128-byte line
    const int line = row >> 1;
    return line * 128 + (((((row & 1) << 2) | c) ^ (((line & 1) << 1) | ((line >> 1) & 1))) << 4);
  } else {
    return row * (4 * DP) + ((c ^ (((row & 3) << 1) | ((row >> 2) & 1))) << 4);
  }
}

template <typename T, int DP, int KT>
struct Tile {
  static constexpr int NP = DaT<T>::NP;
  static constexpr int kPlane = KT * 4 * DP;          // bytes of one plane of X or Y
  static constexpr int kBytes = 2 * NP * kPlane;      // X planes, then Y planes
  typedef typename DaT<T>::E E;

  // A operand, 32 rows row0 .. row0 + 31 (a multiple of 32), step ks of the 16-deep steps along the row (X: map m starts at
  // step m DP / 16)
  static __device__ __forceinline__ Frag<T> rows(const char* lds, int which, int row0, int ks, int lane) {
    Frag<T> f;
    const int o = da_off<DP>(row0 + (lane & 31), 2 * ks + (lane >> 5));
#pragma unroll
    for (int p = 0; p < NP; ++p)
      f.p[p] = *reinterpret_cast<const vec8<E>*>(lds + (which * NP + p) * kPlane + o);
    return f;
  }
  // A operand of the transposed tile: 32 columns col0 .. (a multiple of 32), reduced rows row0 + 16 t + {4 h + 0..3,
  // 8 + 4 h + 0..3}
  static __device__ __forceinline__ Frag<T> cols(const char* lds, int which, int row0, int t, int col0, int lane) {
    Frag<T> f;
    const int i = lane & 15, h = lane >> 5;
    const int row = row0 + 16 * t + 4 * h + (i >> 2);
    const int c = col0 / 8 + 2 * ((lane >> 4) & 1) + ((i >> 1) & 1);
    const int o0 = da_off<DP>(row, c) + 8 * (i & 1), o1 = da_off<DP>(row + 8, c) + 8 * (i & 1);
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const char* b = lds + (which * NP + p) * kPlane;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(b + o0));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(b + o1));
      const vec4<E> a = __builtin_bit_cast(vec4<E>, lo), z = __builtin_bit_cast(vec4<E>, hi);
      f.p[p] = __builtin_shufflevector(a, z, 0, 1, 2, 3, 4, 5, 6, 7);
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
  long x_rs, x_ms, y_rs;
  int n, d;
  const unsigned char* mask;
};

// Tiles on their way from memory to LDS, NT threads together.
//   fp16 / bf16: memory to LDS without registers (global_load_lds_dwordx4), two tiles: while one is computed on, the next
//   lands.  The 64 pieces of a wave's copy stand one behind the other in LDS, so the lane picks the piece that belongs there.
//   fp32: through registers, where the values are split into planes; one tile.
// use:  feed.issue(first, row0);  for each tile: { const char* t = feed.next();  [feed.issue(following, row0)];  compute }
// next() is a barrier of the workgroup.
template <typename T, int DP, int KT, int NT>
struct Feed {
  typedef Tile<T, DP, KT> Tl;
  static constexpr bool DMA = Tl::NP == 1;
  static constexpr int kPieces = KT * DP / 4;                    // of X, and of Y
  static constexpr int kPer = (kPieces + NT - 1) / NT;
  static constexpr int kTile = Tl::kBytes + 16 * ((KT / 8 + 15) / 16);   // the tile and its visible rows, a bit each
  static constexpr int kLds = kTile * (DMA ? 2 : 1);
  static_assert(!DMA || kPieces % 64 == 0, "whole waves copy");
  static_assert(NT * 4 / DP % 8 == 0 || kPer == 1, "a thread's pieces stand at one place of their rows");

  char* lds;
  int tid, wave, cur;       // cur: the buffer that next() returns
  bool bit;
  Raw8<T> x[DMA ? 1 : kPer], y[DMA ? 1 : kPer];

  __device__ __forceinline__ Feed(char* l, int t) : lds(l), tid(t), wave(__builtin_amdgcn_readfirstlane(t >> 6)), cur(0), bit(false) {}

  // piece e of a matrix of the tile -> its row and column piece
  static __device__ __forceinline__ void place(int e, int& row, int& c) {
    if constexpr (DP == 16) {
      const int line = e >> 3, q = (e & 7) ^ (((line & 1) << 1) | ((line >> 1) & 1));
      row = line * 2 + (q >> 2);
      c = q & 3;
    } else {
      row = e / (DP / 4);
      c = (e % (DP / 4)) ^ (((row & 3) << 1) | ((row >> 2) & 1));
    }
  }
  static __device__ __forceinline__ void words(char* tile, int tid, bool bit) {
    if (tid < KT) {
      const unsigned long long w = __ballot(bit);
      if ((tid & 31) == 0) reinterpret_cast<unsigned*>(tile + Tl::kBytes)[tid >> 5] = (unsigned)(w >> (tid & 32));
    }
  }
  static __device__ __forceinline__ void copy16(const void* g, char* l) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g,
                                     (__attribute__((address_space(3))) void*)l, 16, 0, 0);
  }

  __device__ __forceinline__ void issue(const Rows<T>& R, int row0) {
    bit = tid < KT && row0 + tid < R.n && (!R.mask || R.mask[row0 + tid]);
    if constexpr (DMA) {
      char* tile = lds + (cur ^ 1) * kTile;
      int row, c;
      place(tid, row, c);
      const int map = c / (DP / 8), o = (c % (DP / 8)) * 8;
      const bool all = R.d == DP && row0 + KT <= R.n && !R.mask;      // uniform
      const long xo = (long)row * R.x_rs + map * R.x_ms + o, yo = (long)row * R.y_rs + c * 8;
      const T* xt = R.x + row0 * R.x_rs;
      const T* yt = R.y + row0 * R.y_rs;
      constexpr int kRows = NT * 4 / DP;       // rows between a thread's pieces
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        if (kPieces % NT && 64 * wave + NT * i >= kPieces) break;
        char* l = tile + (64 * wave + NT * i) * 16;
        const T *px = xt + xo + i * kRows * R.x_rs, *py = yt + yo + i * kRows * R.y_rs;
        if (!all) {
          const int r = row0 + row + i * kRows;
          const bool ok = r < R.n && (!R.mask || R.mask[r]);
          px = ok && o < R.d ? px : (const T*)da_zero;
          py = ok && c * 8 < 2 * R.d ? py : (const T*)da_zero;
        }
        copy16(px, l);
        copy16(py, l + Tl::kPlane);
      }
      words(tile, tid, bit);
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int e = tid + NT * i;
        if (kPieces % NT && e >= kPieces) break;
        const int row = e / (DP / 4), c = e % (DP / 4);
        const int map = c / (DP / 8), o = (c % (DP / 8)) * 8;
        const long r = row0 + row;
        const bool ok = r < R.n && (!R.mask || R.mask[r]);
        x[i].load(R.x + r * R.x_rs + map * R.x_ms + o, ok && o < R.d);
        y[i].load(R.y + r * R.y_rs + c * 8, ok && c * 8 < 2 * R.d);
      }
    }
  }
  // the tile issued last, in LDS for every wave; every wave is done with the tile before it
  __device__ __forceinline__ const char* next() {
    if constexpr (DMA) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      cur ^= 1;
      return lds + cur * kTile;
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
      words(lds, tid, bit);
      __syncthreads();
      return lds;
    }
  }
  static __device__ __forceinline__ unsigned word(const char* tile, int row0) {
    return reinterpret_cast<const unsigned*>(tile + Tl::kBytes)[row0 >> 5];
  }
};

template <typename T>
__device__ __forceinline__ float da_lam(const DaArgs& A, int head) {
  return A.lam_f32 ? ((const float*)A.lam)[head] : (float)((const T*)A.lam)[head];
}
// keys of batch item b, and the position of its first query (keys <= position are seen); both are taken into range here, so
// that no value of theirs reaches behind the tensors
__device__ __forceinline__ int da_len(const DaArgs& A, int b) {
  const int n = A.lengths ? A.lengths[b] : A.Nk;
  return n < 0 ? 0 : n > A.Nk ? A.Nk : n;
}
__device__ __forceinline__ long da_start(const DaArgs& A, int b) { return A.q_start ? (long)A.q_start[b] : (long)A.Nk - A.Nq; }
// keys that query i sees
__device__ __forceinline__ int da_limit(const DaArgs& A, int len, long start, int i) {
  if (!A.causal) return len;
  const long n = start + i + 1;
  return n < 0 ? 0 : n > len ? len : (int)n;
}

// workgroups of one (batch item, key head) on one XCD, so that its keys and values are read once into that XCD's L2:
// workgroups are dealt to the XCDs in turn.  Any bijection is correct.
__device__ __forceinline__ long da_unit(long n) {
  const long per = (n + 7) / 8;
  return (long)(blockIdx.x & 7) * per + (blockIdx.x >> 3);
}

__device__ __forceinline__ float da_xor32_sum(float x) {
  const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}

constexpr float kLog2e = 1.4426950408889634f;

}  // namespace samble
