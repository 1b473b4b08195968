// Differential attention, forward: one pass over the keys with the running maximum and sum of both softmax maps.
// Layout, operands and tiles: diff_dev.h.
//
// A wave owns 32 rows and keeps their Q operands, both maps' statistics and both maps' unnormalised outputs O_1, O_2 in
// registers (the maps' normalisers are known at the end only, so P_1 - lam P_2 cannot be formed before; both maps in one wave
// share every value tile read).  S^T = K Q^T puts a row's logits into one lane column: maxima and sums are lane-local but for
// one exchange of the two halves.
//   RW  waves along the rows, each its own 32
//   KW  waves along the keys of a tile, each its own 32: for few rows (single tokens); their results meet in LDS
//   DW  waves along the value columns
// Few rows against many keys are also split over workgroups (`splits`); diff_join_kernel adds the parts.
#include "diff_dev.h"

namespace samble {

template <typename T, int DP, int RW, int KW, int DW>
struct FwdCfg {
  static constexpr int NW = RW * KW * DW, NT = 64 * NW;
  static constexpr int SUB = KW > 1 ? 1 : (DaT<T>::NP == 1 || DP <= 32) ? 2 : 1;   // 32-key steps of a wave per tile
  static constexpr int KT = 32 * KW * SUB;
  static constexpr int DVT = 2 * DP / 32 / DW;            // 32-column pieces of the outputs per wave
  typedef Tile<T, DP, KT> Tl;
  static constexpr int kMergeFloats = (DVT * 32 + 4) * 64;   // a wave's state
  static constexpr int kMergeBytes = KW > 1 ? kMergeFloats * 4 * (KW / 2) * RW * DW : 0;
  static constexpr int kLds = (Tl::kBytes > kMergeBytes ? Tl::kBytes : kMergeBytes) + KT / 8;
};

// partial results of a split: per row (row order of the pair) m_1, l_1, m_2, l_2, then O_1, O_2 (2 d each)
__device__ __forceinline__ long da_part_floats(int d) { return 4 + 4l * d; }

template <typename T, int DP, int RW, int KW, int DW>
__global__ __launch_bounds__(64 * RW * KW * DW) void diff_fwd_kernel(DaArgs A) {
  typedef FwdCfg<T, DP, RW, KW, DW> Cfg;
  typedef typename Cfg::Tl Tl;
  constexpr int KS = DP / 16, DVT = Cfg::DVT;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  unsigned* words = reinterpret_cast<unsigned*>(smem + Cfg::kLds - Cfg::KT / 8);   // visible keys of the tile, a bit each

  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rw = wave % RW, kw = (wave / RW) % KW, dw = wave / (RW * KW);
  const long rows = (long)A.Nq * A.G;
  const long blocks = (rows + 32 * RW - 1) / (32 * RW);
  const long units = blocks * A.splits * A.B * A.Hkv;
  const long unit = da_unit(units);
  if (unit >= units) return;
  const int split = (int)(unit % A.splits);
  const long rest = unit / A.splits;
  const long blk = blocks - 1 - rest % blocks;      // (under a causal mask the long rows first)
  const int pair = (int)(rest / blocks), b = pair / A.Hkv, hk = pair % A.Hkv;

  const int len = da_len(A, b);
  const long start = da_start(A, b);
  // this lane's row
  const long r = blk * 32 * RW + 32 * rw + (lane & 31);
  const bool live = r < rows;
  const int qi = live ? (int)(r / A.G) : 0, head = hk * A.G + (live ? (int)(r % A.G) : 0);
  const int limit = live ? da_limit(A, len, start, qi) : 0;
  // keys that the last row of the workgroup sees; fewest keys of this wave's rows
  const long last = blk * 32 * RW + 32 * RW - 1;
  const int kmax = da_limit(A, len, start, (int)((last < rows ? last : rows - 1) / A.G));
  const long first = blk * 32 * RW + 32 * rw;
  const int kmin = first + 31 < rows ? da_limit(A, len, start, (int)(first / A.G)) : 0;

  const int tiles = (kmax + Cfg::KT - 1) / Cfg::KT;
  const int t0 = (int)((long)tiles * split / A.splits), t1 = (int)((long)tiles * (split + 1) / A.splits);

  const T* kb = (const T*)A.k + b * A.k_bs + hk * A.k_hs;
  const T* vb = (const T*)A.v + b * A.v_bs + hk * A.v_hs;
  const unsigned char* km = A.key_mask ? A.key_mask + b * A.km_bs : nullptr;

  Frag<T> qf[2][KS];
  {
    const T* qp = (const T*)A.q + b * A.q_bs + qi * A.q_rs + head * A.q_hs;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int o = 16 * s + 8 * h;
        Raw8<T> raw;
        raw.load(qp + m * A.q_ms + o, live && o < A.d);
        qf[m][s] = raw.frag();
      }
  }

  f32x16 o[2][DVT];
  float mx[2] = {kNegInf, kNegInf}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int t = 0; t < DVT; ++t) o[m][t] = zero16();
  const float c = A.scale * kLog2e;

  Stage<T, DP, Cfg::KT, Cfg::NT> st;
  bool bit = false;
  auto load_tile = [&](int t) {
    const int k0 = t * Cfg::KT;
    st.load(tid, A.d, A.k_ms, [&](int row, const T*& px, const T*& py) {
      const long key = k0 + row;
      const bool ok = key < len && (!km || km[key]);
      px = kb + (ok ? key : 0) * A.k_rs;
      py = vb + (ok ? key : 0) * A.v_rs;
      return ok;
    });
    if (tid < Cfg::KT) bit = k0 + tid < len && (!km || km[k0 + tid]);
  };
  if (t0 < t1) load_tile(t0);
  for (int t = t0; t < t1; ++t) {
    __syncthreads();     // the last tile's readers are done
    st.store(smem, tid);
    if (tid < Cfg::KT) {
      const unsigned long long w = __ballot(bit);
      if ((lane & 31) == 0) words[tid >> 5] = (unsigned)(w >> (lane & 32));
    }
    __syncthreads();
    if (t + 1 < t1) load_tile(t + 1);
#pragma unroll
    for (int sub = 0; sub < Cfg::SUB; ++sub) {
      const int row0 = 32 * (kw + sub), k0 = t * Cfg::KT + row0;
      if (k0 >= kmax) continue;   // (uniform; nothing of it is seen)
      f32x16 s[2] = {zero16(), zero16()};
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s[m] = da_mma<T>(Tl::rows(smem, 0, row0, m * KS + ks, lane), qf[m][ks], s[m]);
      const unsigned word = words[row0 >> 5];
      if (word != 0xffffffffu || k0 + 32 > kmin) {
        const unsigned w = word >> (4 * h);
        const int left = limit - k0 - 4 * h;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int j = crow(e, 0);
          const bool see = ((w >> j) & 1) && j < left;
          s[0][e] = see ? s[0][e] : kNegInf;
          s[1][e] = see ? s[1][e] : kNegInf;
        }
      }
      Frag<T> pf[2][2];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        float top = s[m][0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top = fmaxf(top, s[m][e]);
        top = xor32_max(top);
        // the reference of the exponentials follows the maximum only when that has grown by more than 8 (a factor of 256 in
        // the sums): any reference gives the same quotients, and the outputs are rescaled in few of the steps
        if (__any(top * c > mx[m] + 8.f)) {
          const float nm = fmaxf(mx[m], top * c), use = nm == kNegInf ? 0.f : nm;
          const float al = __builtin_amdgcn_exp2f(mx[m] - use);
          l[m] *= al;
#pragma unroll
          for (int dt = 0; dt < DVT; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[m][dt][e] *= al;
          mx[m] = nm;
        }
        const float ref = mx[m] == kNegInf ? 0.f : mx[m];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float p[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            p[e] = __builtin_amdgcn_exp2f(fmaf(s[m][8 * u + e], c, -ref));
            l[m] += p[e];
          }
          pf[m][u] = da_pack<T>(p);
        }
      }
#pragma unroll
      for (int dt = 0; dt < DVT; ++dt)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const Frag<T> vf = Tl::cols(smem, 1, row0, u, 32 * (dw * DVT + dt), lane);
#pragma unroll
          for (int m = 0; m < 2; ++m) o[m][dt] = da_mma<T>(vf, pf[m][u], o[m][dt]);
        }
    }
  }
#pragma unroll
  for (int m = 0; m < 2; ++m) l[m] = da_xor32_sum(l[m]);

  if constexpr (KW > 1) {   // the waves along the keys: pairwise, the upper half hands its state to the lower
    float* f = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int s = KW / 2; s > 0; s >>= 1) {
      __syncthreads();
      if (kw >= s && kw < 2 * s) {
        float* w = f + (long)((kw - s) * RW * DW + rw * DW + dw) * Cfg::kMergeFloats + lane;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          w[(2 * m) * 64] = mx[m];
          w[(2 * m + 1) * 64] = l[m];
#pragma unroll
          for (int dt = 0; dt < DVT; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) w[(4 + (m * DVT + dt) * 16 + e) * 64] = o[m][dt][e];
        }
      }
      __syncthreads();
      if (kw < s) {
        const float* w = f + (long)(kw * RW * DW + rw * DW + dw) * Cfg::kMergeFloats + lane;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const float m2 = w[(2 * m) * 64], l2 = w[(2 * m + 1) * 64];
          const float nm = fmaxf(mx[m], m2), use = nm == kNegInf ? 0.f : nm;
          const float a1 = __builtin_amdgcn_exp2f(mx[m] - use), a2 = __builtin_amdgcn_exp2f(m2 - use);
          mx[m] = nm;
          l[m] = l[m] * a1 + l2 * a2;
#pragma unroll
          for (int dt = 0; dt < DVT; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              o[m][dt][e] = o[m][dt][e] * a1 + w[(4 + (m * DVT + dt) * 16 + e) * 64] * a2;
        }
      }
    }
    if (kw) return;
  }
  if (!live) return;

  if (A.splits > 1) {
    float* w = A.part + (((long)split * A.B * A.Hkv + pair) * rows + r) * da_part_floats(A.d);
    if (dw == 0 && h == 0) {
      const f32x4 head4 = {mx[0], l[0], mx[1], l[1]};
      *reinterpret_cast<f32x4*>(w) = head4;
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int dt = 0; dt < DVT; ++dt)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          const int col = 32 * (dw * DVT + dt) + 8 * q4 + 4 * h;
          if (col < 2 * A.d) {
            const f32x4 v = {o[m][dt][4 * q4], o[m][dt][4 * q4 + 1], o[m][dt][4 * q4 + 2], o[m][dt][4 * q4 + 3]};
            *reinterpret_cast<f32x4*>(w + 4 + 2 * m * A.d + col) = v;
          }
        }
    return;
  }
  const float i1 = l[0] > 0.f ? 1.f / l[0] : l[0] == 0.f ? 0.f : l[0], i2 = l[1] > 0.f ? 1.f / l[1] : l[1] == 0.f ? 0.f : l[1];
  const float lam = da_lam<T>(A, head);
  if (A.lse && dw == 0 && h == 0) {
    float* ls = A.lse + ((long)b * A.H + head) * 2 * A.Nq + qi;
    ls[0] = l[0] == 0.f ? __builtin_huge_valf() : mx[0] + __builtin_amdgcn_logf(l[0]);
    ls[A.Nq] = l[1] == 0.f ? __builtin_huge_valf() : mx[1] + __builtin_amdgcn_logf(l[1]);
  }
  T* out = (T*)A.out + (((long)b * A.Nq + qi) * A.H + head) * 2 * A.d;
  T* out2 = A.out2 ? (T*)A.out2 + (((long)b * A.Nq + qi) * A.H + head) * 2 * A.d : nullptr;
#pragma unroll
  for (int dt = 0; dt < DVT; ++dt)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      const int col = 32 * (dw * DVT + dt) + 8 * q4 + 4 * h;
      if (col >= 2 * A.d) continue;
      typedef T vec __attribute__((ext_vector_type(4)));
      vec a, z;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float o2 = o[1][dt][4 * q4 + e] * i2;
        a[e] = (T)fmaf(-lam, o2, o[0][dt][4 * q4 + e] * i1);
        z[e] = (T)o2;
      }
      *reinterpret_cast<vec*>(out + col) = a;
      if (out2) *reinterpret_cast<vec*>(out2 + col) = z;
    }
}

// adds the splits of a row: 2 d threads' columns, one wave per row
template <typename T>
__global__ __launch_bounds__(256) void diff_join_kernel(DaArgs A) {
  const long rows = (long)A.Nq * A.G, all = rows * A.B * A.Hkv;
  const int lane = threadIdx.x & 63;
  for (long u = (long)blockIdx.x * 4 + (threadIdx.x >> 6); u < all; u += (long)gridDim.x * 4) {
    const long pair = u / rows, r = u % rows;
    const int b = (int)(pair / A.Hkv), hk = (int)(pair % A.Hkv), qi = (int)(r / A.G), head = hk * A.G + (int)(r % A.G);
    const long pf = da_part_floats(A.d), step = all * pf;
    const float* w = A.part + u * pf;
    float m[2] = {kNegInf, kNegInf}, l[2] = {0.f, 0.f};
    for (int s = lane; s < A.splits; s += 64) {
      const f32x4 t = *reinterpret_cast<const f32x4*>(w + s * step);
      m[0] = fmaxf(m[0], t[0]);
      m[1] = fmaxf(m[1], t[2]);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      m[k] = wave_max64(m[k]);
      if (m[k] == kNegInf) m[k] = 0.f;
    }
    const int cols = 2 * A.d;
    float acc[2][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[0][k] = acc[1][k] = 0.f;
    for (int s = 0; s < A.splits; ++s) {
      const float* p = w + s * step;
      const f32x4 t = *reinterpret_cast<const f32x4*>(p);
      const float a0 = __builtin_amdgcn_exp2f(t[0] - m[0]), a1 = __builtin_amdgcn_exp2f(t[2] - m[1]);
      l[0] = fmaf(t[1], a0, l[0]);
      l[1] = fmaf(t[3], a1, l[1]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int c = lane + 64 * k;
        if (c < cols) {
          acc[0][k] = fmaf(p[4 + c], a0, acc[0][k]);
          acc[1][k] = fmaf(p[4 + cols + c], a1, acc[1][k]);
        }
      }
    }
    const float i1 = l[0] > 0.f ? 1.f / l[0] : l[0] == 0.f ? 0.f : l[0], i2 = l[1] > 0.f ? 1.f / l[1] : l[1] == 0.f ? 0.f : l[1];
    const float lam = da_lam<T>(A, head);
    const long o = (((long)b * A.Nq + qi) * A.H + head) * cols;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = lane + 64 * k;
      if (c < cols) {
        const float o2 = acc[1][k] * i2;
        ((T*)A.out)[o + c] = (T)fmaf(-lam, o2, acc[0][k] * i1);
        if (A.out2) ((T*)A.out2)[o + c] = (T)o2;
      }
    }
    if (A.lse && lane == 0) {
      float* ls = A.lse + ((long)b * A.H + head) * 2 * A.Nq + qi;
      ls[0] = l[0] == 0.f ? __builtin_huge_valf() : m[0] + __builtin_amdgcn_logf(l[0]);
      ls[A.Nq] = l[1] == 0.f ? __builtin_huge_valf() : m[1] + __builtin_amdgcn_logf(l[1]);
    }
  }
}

// ---- launches -------------------------------------------------------------------------------------------------------------
struct FwdPlan { bool few; long blocks; int splits; };

// Few rows (at most 32 of a key head) take the kernels whose waves stand along the keys.  Splits: workgroups for two rounds of
// the 256 CUs when rows and heads alone give fewer, each split with at least four tiles of 128 keys (a split costs its
// partial results' way through memory), at most 128.
static FwdPlan fwd_plan(int B, int Nq, int Nk, int H, int Hkv) {
  const long rows = (long)Nq * (H / Hkv), pairs = (long)B * Hkv;
  FwdPlan p;
  p.few = rows <= 32;
  p.blocks = p.few ? 1 : (rows + 127) / 128;
  const long have = p.blocks * pairs;
  long s = 1;
  if (have < 256) {
    s = (512 + have - 1) / have;
    const long most = Nk / 512;
    if (s > most) s = most;
    if (s > 128) s = 128;
    if (s < 1) s = 1;
  }
  p.splits = (int)s;
  return p;
}

template <typename T, int DP, int RW, int KW, int DW>
static int fwd_go(const DaArgs& A, hipStream_t s) {
  typedef FwdCfg<T, DP, RW, KW, DW> Cfg;
  const long rows = (long)A.Nq * A.G, blocks = (rows + 32 * RW - 1) / (32 * RW);
  const long units = blocks * A.splits * A.B * A.Hkv, grid = (units + 7) / 8 * 8;
  if (grid * Cfg::NT >= (1ll << 32)) return -22;
  const void* f = reinterpret_cast<const void*>(diff_fwd_kernel<T, DP, RW, KW, DW>);
  if (Cfg::kLds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, Cfg::kLds);
    if (e != hipSuccess) return (int)e;
  }
  hipLaunchKernelGGL((diff_fwd_kernel<T, DP, RW, KW, DW>), dim3((unsigned)grid), dim3(Cfg::NT), Cfg::kLds, s, A);
  return (int)hipGetLastError();
}

template <typename T>
static int fwd_type(DaArgs& A, hipStream_t s) {
  const FwdPlan p = fwd_plan(A.B, A.Nq, A.Nk, A.H, A.Hkv);
  A.splits = p.splits;
  constexpr bool F = DaT<T>::NP == 3;
  int rc = -22;
  if (A.d <= 16) rc = p.few ? fwd_go<T, 16, 1, 4, 1>(A, s) : fwd_go<T, 16, 4, 1, 1>(A, s);
  else if (A.d <= 32) rc = p.few ? fwd_go<T, 32, 1, 4, 1>(A, s) : fwd_go<T, 32, 4, 1, 1>(A, s);
  else if (A.d <= 64) {
    if constexpr (F) rc = p.few ? fwd_go<T, 64, 1, 2, 2>(A, s) : fwd_go<T, 64, 4, 1, 1>(A, s);
    else rc = p.few ? fwd_go<T, 64, 1, 4, 1>(A, s) : fwd_go<T, 64, 4, 1, 1>(A, s);
  } else if constexpr (!F) {
    if (A.d <= 128) rc = p.few ? fwd_go<T, 128, 1, 2, 2>(A, s) : fwd_go<T, 128, 4, 1, 1>(A, s);
  }
  if (rc || A.splits == 1) return rc;
  const long all = (long)A.Nq * A.H * A.B;
  hipLaunchKernelGGL((diff_join_kernel<T>), dim3((unsigned)((all + 3) / 4 < (1 << 20) ? (all + 3) / 4 : (1 << 20))), dim3(256), 0, s,
                     A);
  return (int)hipGetLastError();
}

}  // namespace samble

using namespace samble;

extern "C" size_t samble_diff_fwd_ws_bytes(int type, int B, int Nq, int Nk, int H, int Hkv, int d) {
  (void)type;
  const FwdPlan p = fwd_plan(B, Nq, Nk, H, Hkv);
  return p.splits == 1 ? 0 : (size_t)p.splits * B * H * Nq * (4 + 4l * d) * sizeof(float);
}

extern "C" int samble_launch_diff_fwd(int type, const DaArgs* args, hipStream_t s) {
  DaArgs A = *args;
  Timed timed(kT_diff_fwd, s);
  return type == 0 ? fwd_type<float>(A, s) : type == 1 ? fwd_type<f16>(A, s) : fwd_type<bf16>(A, s);
}
