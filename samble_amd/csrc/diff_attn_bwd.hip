// Differential attention, backward.  With g = d loss / d out and dA = g v^T:
//     t_m[i] = sum_j P_m dA = g . (P_m v)_i,   dS_1 = P_1 (dA - t_1),   dS_2 = -lam P_2 (dA - t_2)
//     dq_m = scale dS_m k_m,  dk_m = scale dS_m^T q_m,  dv = (P_1 - lam P_2)^T g,  dlam = - sum_i t_2
// The logits are formed again from q and k; P = exp2(logit - lse) with the forward's row statistics.  Two launches, no atomics:
//   diff_dq_kernel   a wave owns 32 rows (layout of the forward): first t_1 = g . out + lam t_2 and t_2 = g . out2 from the
//                    saved outputs, kept for the second launch, then one sweep over the keys
//   diff_dkv_kernel  a wave owns 32 keys and sweeps over the rows of all query heads that share the key head; workgroups
//                    behind the last one sum dlam
// Layout, operands and tiles: diff_dev.h.  The second kernel holds S with the row index on the registers, so that P and dS
// are operands of the sums over rows as they stand.
#include "diff_dev.h"

namespace samble {

template <typename T, int DP>
struct DqCfg {
  static constexpr int SUB = (DaT<T>::NP == 1 || DP <= 32) ? 2 : 1, KT = 32 * SUB;
  typedef Tile<T, DP, KT> Tl;
  static constexpr int DT = DP < 32 ? 1 : DP / 32;     // 32-column pieces of a map's gradient (16 columns: both maps on one)
  static constexpr int kLds = Tl::kBytes + KT / 8;
};

template <typename T, int DP>
__global__ __launch_bounds__(256, 1) void diff_dq_kernel(DaArgs A) {
  typedef DqCfg<T, DP> Cfg;
  typedef typename Cfg::Tl Tl;
  constexpr int KS = DP / 16, DT = Cfg::DT, RW = 4;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  unsigned* words = reinterpret_cast<unsigned*>(smem + Tl::kBytes);

  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
  const int rw = __builtin_amdgcn_readfirstlane(tid >> 6);
  const long rows = (long)A.Nq * A.G, blocks = (rows + 32 * RW - 1) / (32 * RW), units = blocks * A.B * A.Hkv;
  const long unit = da_unit(units);
  if (unit >= units) return;
  const long blk = blocks - 1 - unit % blocks;
  const int pair = (int)(unit / blocks), b = pair / A.Hkv, hk = pair % A.Hkv;
  const int len = da_len(A, b);
  const long start = da_start(A, b);
  const long r = blk * 32 * RW + 32 * rw + (lane & 31);
  const bool live = r < rows;
  const int qi = live ? (int)(r / A.G) : 0, head = hk * A.G + (live ? (int)(r % A.G) : 0);
  const int limit = live ? da_limit(A, len, start, qi) : 0;
  const long last = blk * 32 * RW + 32 * RW - 1;
  const int kmax = da_limit(A, len, start, (int)((last < rows ? last : rows - 1) / A.G));
  const long first = blk * 32 * RW + 32 * rw;
  const int kmin = first + 31 < rows ? da_limit(A, len, start, (int)(first / A.G)) : 0;
  const int tiles = (kmax + Cfg::KT - 1) / Cfg::KT;

  const T* kb = (const T*)A.k + b * A.k_bs + hk * A.k_hs;
  const T* vb = (const T*)A.v + b * A.v_bs + hk * A.v_hs;
  const unsigned char* km = A.key_mask ? A.key_mask + b * A.km_bs : nullptr;

  Frag<T> qf[2][KS], gf[2 * KS];
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
  const float lam = da_lam<T>(A, head);
  float t1 = 0.f, t2 = 0.f;
  {
    const T* gp = (const T*)A.dout + b * A.g_bs + qi * A.g_rs + head * A.g_hs;
    const long at = (((long)b * A.Nq + qi) * A.H + head) * 2 * A.d;
#pragma unroll
    for (int s = 0; s < 2 * KS; ++s) {
      const int o = 16 * s + 8 * h;
      const bool ok = live && o < 2 * A.d;
      Raw8<T> raw, o1, o2;
      raw.load(gp + o, ok);
      o1.load((const T*)A.out + at + o, ok);
      o2.load((const T*)A.out2 + at + o, ok);
      gf[s] = raw.frag();
      float g[8], u[8], w[8];
      raw.widen(g);
      o1.widen(u);
      o2.widen(w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        t1 = fmaf(g[e], u[e], t1);
        t2 = fmaf(g[e], w[e], t2);
      }
    }
    t1 = da_xor32_sum(t1);
    t2 = da_xor32_sum(t2);
    t1 = fmaf(lam, t2, t1);
  }
  const float* ls = A.lse + ((long)b * A.H + head) * 2 * A.Nq + qi;
  const float lse0 = live ? ls[0] : __builtin_huge_valf(), lse1 = live ? ls[A.Nq] : __builtin_huge_valf();
  if (live && h == 0) {
    float* dl = A.delta + ((long)b * A.H + head) * 2 * A.Nq + qi;
    dl[0] = t1;
    dl[A.Nq] = t2;
  }

  f32x16 acc[2][DT];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int t = 0; t < DT; ++t) acc[m][t] = zero16();
  const float c = A.scale * kLog2e;

  Stage<T, DP, Cfg::KT, 256> st;
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
  if (tiles) load_tile(0);
  for (int t = 0; t < tiles; ++t) {
    __syncthreads();
    st.store(smem, tid);
    if (tid < Cfg::KT) {
      const unsigned long long w = __ballot(bit);
      if ((lane & 31) == 0) words[tid >> 5] = (unsigned)(w >> (lane & 32));
    }
    __syncthreads();
    if (t + 1 < tiles) load_tile(t + 1);
#pragma unroll
    for (int sub = 0; sub < Cfg::SUB; ++sub) {
      const int row0 = 32 * sub, k0 = t * Cfg::KT + row0;
      if (k0 >= kmax) continue;
      f32x16 s[2] = {zero16(), zero16()}, da = zero16();
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s[m] = da_mma<T>(Tl::rows(smem, 0, row0, m * KS + ks, lane), qf[m][ks], s[m]);
#pragma unroll
      for (int ks = 0; ks < 2 * KS; ++ks) da = da_mma<T>(Tl::rows(smem, 1, row0, ks, lane), gf[ks], da);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[0][e] = __builtin_amdgcn_exp2f(fmaf(s[0][e], c, -lse0));
        s[1][e] = __builtin_amdgcn_exp2f(fmaf(s[1][e], c, -lse1));
      }
      const unsigned word = words[row0 >> 5];
      if (word != 0xffffffffu || k0 + 32 > kmin) {
        const unsigned w = word >> (4 * h);
        const int left = limit - k0 - 4 * h;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int j = crow(e, 0);
          const bool see = ((w >> j) & 1) && j < left;
          s[0][e] = see ? s[0][e] : 0.f;
          s[1][e] = see ? s[1][e] : 0.f;
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float d1[8], d2[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          d1[e] = s[0][8 * u + e] * (da[8 * u + e] - t1);
          d2[e] = -lam * s[1][8 * u + e] * (da[8 * u + e] - t2);
        }
        const Frag<T> f1 = da_pack<T>(d1), f2 = da_pack<T>(d2);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const Frag<T> k1 = Tl::cols(smem, 0, row0, u, 32 * dt, lane);
          acc[0][dt] = da_mma<T>(k1, f1, acc[0][dt]);
          const Frag<T> k2 = DP < 32 ? k1 : Tl::cols(smem, 0, row0, u, DP + 32 * dt, lane);
          acc[1][dt] = da_mma<T>(k2, f2, acc[1][dt]);
        }
      }
    }
  }
  if (!live) return;
  T* dq = (T*)A.dq + (((long)b * A.Nq + qi) * A.H + head) * 2 * A.d;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int q4 = 0; q4 < (DP < 32 ? 2 : 4); ++q4) {
        const int col = 32 * dt + 8 * q4 + 4 * h, reg = 4 * (q4 + (DP < 32 ? 2 * m : 0));
        if (col >= A.d) continue;
        typedef T vec __attribute__((ext_vector_type(4)));
        vec v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)(A.scale * acc[m][dt][reg + e]);
        *reinterpret_cast<vec*>(dq + m * A.d + col) = v;
      }
}

template <typename T, int DP>
struct DkvCfg {
  static constexpr int NW = DP == 128 ? 2 : 4;
  static constexpr int SUB = (DaT<T>::NP == 1 || DP <= 32) ? (DP == 128 ? 1 : 2) : 1, RT = 32 * SUB;   // rows of a tile
  typedef Tile<T, DP, RT> Tl;
  static constexpr int DT = DP < 32 ? 1 : DP / 32, DVT = 2 * DP / 32;
  static constexpr int kLds = Tl::kBytes + 6 * RT * 4;
};

template <typename T, int DP>
__global__ __launch_bounds__((DkvCfg<T, DP>::NW * 64), 1) void diff_dkv_kernel(DaArgs A, unsigned main_grid) {
  typedef DkvCfg<T, DP> Cfg;
  typedef typename Cfg::Tl Tl;
  constexpr int KS = DP / 16, DT = Cfg::DT, DVT = Cfg::DVT, NW = Cfg::NW, NT = 64 * NW, RT = Cfg::RT;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float* stat = reinterpret_cast<float*>(smem + Tl::kBytes);   // lse_1, lse_2, t_1, t_2, lam [RT], limit (int) [RT]
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;

  if (blockIdx.x >= main_grid) {      // dlam of one head: - sum of t_2 over batch and queries
    const int head = blockIdx.x - main_grid;
    float sum = 0.f;
    const long n = (long)A.B * A.Nq;
    for (long i = tid; i < n; i += NT) sum += A.delta[((i / A.Nq) * A.H + head) * 2 * A.Nq + A.Nq + i % A.Nq];
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (lane == 0) stat[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0) {
      sum = 0.f;
      for (int w = 0; w < NW; ++w) sum += stat[w];
      if (A.lam_f32) ((float*)A.dlam)[head] = -sum;
      else ((T*)A.dlam)[head] = (T)(-sum);
    }
    return;
  }

  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const long rows = (long)A.Nq * A.G;
  const long blocks = ((long)A.Nk + 32 * NW - 1) / (32 * NW), units = blocks * A.B * A.Hkv;
  const long per = main_grid / 8, unit = (long)(blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (unit >= units) return;
  const int blk = (int)(unit % blocks);           // (under a causal mask the keys that most rows see first)
  const int pair = (int)(unit / blocks), b = pair / A.Hkv, hk = pair % A.Hkv;
  const int len = da_len(A, b);
  const long start = da_start(A, b);
  const int key0 = blk * 32 * NW, kw0 = key0 + 32 * wave, key = kw0 + (lane & 31);
  const unsigned char* km = A.key_mask ? A.key_mask + b * A.km_bs : nullptr;
  const bool valid = key < len && (!km || km[key]);
  const bool all_valid = __all(valid);

  Frag<T> kf[2][KS], vf[2 * KS];
  {
    const T* kp = (const T*)A.k + b * A.k_bs + hk * A.k_hs + (long)(valid ? key : 0) * A.k_rs;
    const T* vp = (const T*)A.v + b * A.v_bs + hk * A.v_hs + (long)(valid ? key : 0) * A.v_rs;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int o = 16 * s + 8 * h;
        Raw8<T> raw;
        raw.load(kp + m * A.k_ms + o, valid && o < A.d);
        kf[m][s] = raw.frag();
      }
#pragma unroll
    for (int s = 0; s < 2 * KS; ++s) {
      const int o = 16 * s + 8 * h;
      Raw8<T> raw;
      raw.load(vp + o, valid && o < 2 * A.d);
      vf[s] = raw.frag();
    }
  }
  f32x16 dk[2][DT], dv[DVT];
#pragma unroll
  for (int t = 0; t < DT; ++t) dk[0][t] = dk[1][t] = zero16();
#pragma unroll
  for (int t = 0; t < DVT; ++t) dv[t] = zero16();
  const float c = A.scale * kLog2e;

  // rows that see any key of the workgroup: all behind the first such query
  const long i0 = A.causal ? (key0 - start > 0 ? key0 - start : 0) : 0;
  const long tiles = key0 >= len || i0 >= A.Nq ? 0 : (rows + RT - 1) / RT;
  const long tile0 = tiles ? i0 * A.G / RT : 0;

  Stage<T, DP, RT, NT> st;
  float sv[6] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  auto load_tile = [&](long t) {
    st.load(tid, A.d, A.q_ms, [&](int row, const T*& px, const T*& py) {
      const long r = t * RT + row;
      const bool ok = r < rows;
      const long i = ok ? r / A.G : 0, hd = hk * A.G + (ok ? r % A.G : 0);
      px = (const T*)A.q + b * A.q_bs + i * A.q_rs + hd * A.q_hs;
      py = (const T*)A.dout + b * A.g_bs + i * A.g_rs + hd * A.g_hs;
      return ok;
    });
    if (tid < RT) {
      const long r = t * RT + tid;
      const bool ok = r < rows;
      const int i = ok ? (int)(r / A.G) : 0, hd = hk * A.G + (ok ? (int)(r % A.G) : 0);
      const long at = ((long)b * A.H + hd) * 2 * A.Nq + i;
      sv[0] = ok ? A.lse[at] : __builtin_huge_valf();     // (rows behind the last: P = 0)
      sv[1] = ok ? A.lse[at + A.Nq] : __builtin_huge_valf();
      sv[2] = ok ? A.delta[at] : 0.f;
      sv[3] = ok ? A.delta[at + A.Nq] : 0.f;
      sv[4] = da_lam<T>(A, hd);
      sv[5] = __int_as_float(ok ? da_limit(A, len, start, i) : 0);
    }
  };
  if (tile0 < tiles) load_tile(tile0);
  for (long t = tile0; t < tiles; ++t) {
    __syncthreads();
    st.store(smem, tid);
    if (tid < RT) {
#pragma unroll
      for (int e = 0; e < 6; ++e) stat[e * RT + tid] = sv[e];
    }
    __syncthreads();
    if (t + 1 < tiles) load_tile(t + 1);
#pragma unroll
    for (int sub = 0; sub < Cfg::SUB; ++sub) {
      const int row0 = 32 * sub;
      f32x16 s[2] = {zero16(), zero16()}, da = zero16();
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s[m] = da_mma<T>(Tl::rows(smem, 0, row0, m * KS + ks, lane), kf[m][ks], s[m]);
#pragma unroll
      for (int ks = 0; ks < 2 * KS; ++ks) da = da_mma<T>(Tl::rows(smem, 1, row0, ks, lane), vf[ks], da);
      const int fewest = __builtin_amdgcn_readfirstlane(__float_as_int(stat[5 * RT + row0]));   // (limits rise with the row)
      const bool masked = !all_valid || kw0 + 32 > fewest;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float a[8], d1[8], d2[8];
#pragma unroll
        for (int q4 = 0; q4 < 2; ++q4) {
          const int at = row0 + 16 * u + 8 * q4 + 4 * h;
          const f32x4 l1 = *reinterpret_cast<const f32x4*>(stat + at), l2 = *reinterpret_cast<const f32x4*>(stat + RT + at);
          const f32x4 t1 = *reinterpret_cast<const f32x4*>(stat + 2 * RT + at);
          const f32x4 t2 = *reinterpret_cast<const f32x4*>(stat + 3 * RT + at);
          const f32x4 lm = *reinterpret_cast<const f32x4*>(stat + 4 * RT + at);
          const f32x4 lt = *reinterpret_cast<const f32x4*>(stat + 5 * RT + at);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = 8 * u + 4 * q4 + e;
            float p1 = __builtin_amdgcn_exp2f(fmaf(s[0][i], c, -l1[e])), p2 = __builtin_amdgcn_exp2f(fmaf(s[1][i], c, -l2[e]));
            if (masked) {
              const bool see = valid && key < __float_as_int(lt[e]);
              p1 = see ? p1 : 0.f;
              p2 = see ? p2 : 0.f;
            }
            p2 *= lm[e];
            a[4 * q4 + e] = p1 - p2;
            d1[4 * q4 + e] = p1 * (da[i] - t1[e]);
            d2[4 * q4 + e] = -p2 * (da[i] - t2[e]);
          }
        }
        const Frag<T> af = da_pack<T>(a), f1 = da_pack<T>(d1), f2 = da_pack<T>(d2);
#pragma unroll
        for (int dt = 0; dt < DVT; ++dt) dv[dt] = da_mma<T>(Tl::cols(smem, 1, row0, u, 32 * dt, lane), af, dv[dt]);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const Frag<T> q1 = Tl::cols(smem, 0, row0, u, 32 * dt, lane);
          dk[0][dt] = da_mma<T>(q1, f1, dk[0][dt]);
          const Frag<T> q2 = DP < 32 ? q1 : Tl::cols(smem, 0, row0, u, DP + 32 * dt, lane);
          dk[1][dt] = da_mma<T>(q2, f2, dk[1][dt]);
        }
      }
    }
  }
  if (key >= A.Nk) return;
  typedef T vec __attribute__((ext_vector_type(4)));
  T* dkp = (T*)A.dk + (((long)b * A.Nk + key) * A.Hkv + hk) * 2 * A.d;
  T* dvp = (T*)A.dv + (((long)b * A.Nk + key) * A.Hkv + hk) * 2 * A.d;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int q4 = 0; q4 < (DP < 32 ? 2 : 4); ++q4) {
        const int col = 32 * dt + 8 * q4 + 4 * h, reg = 4 * (q4 + (DP < 32 ? 2 * m : 0));
        if (col >= A.d) continue;
        vec v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)(A.scale * dk[m][dt][reg + e]);
        *reinterpret_cast<vec*>(dkp + m * A.d + col) = v;
      }
#pragma unroll
  for (int dt = 0; dt < DVT; ++dt)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      const int col = 32 * dt + 8 * q4 + 4 * h;
      if (col >= 2 * A.d) continue;
      vec v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (T)dv[dt][4 * q4 + e];
      *reinterpret_cast<vec*>(dvp + col) = v;
    }
}

template <typename T, int DP>
static int bwd_go(const DaArgs& A, hipStream_t s) {
  typedef DqCfg<T, DP> Q;
  typedef DkvCfg<T, DP> K;
  const long rows = (long)A.Nq * A.G, pairs = (long)A.B * A.Hkv;
  const long gq = ((rows + 127) / 128 * pairs + 7) / 8 * 8;
  const long gk = (((long)A.Nk + 32 * K::NW - 1) / (32 * K::NW) * pairs + 7) / 8 * 8;
  if (gq * 256 >= (1ll << 32) || (gk + A.H) * 256 >= (1ll << 32)) return -22;
  if (Q::kLds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(diff_dq_kernel<T, DP>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, Q::kLds);
    if (e != hipSuccess) return (int)e;
  }
  if (K::kLds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(diff_dkv_kernel<T, DP>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, K::kLds);
    if (e != hipSuccess) return (int)e;
  }
  hipLaunchKernelGGL((diff_dq_kernel<T, DP>), dim3((unsigned)gq), dim3(256), Q::kLds, s, A);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  hipLaunchKernelGGL((diff_dkv_kernel<T, DP>), dim3((unsigned)(gk + A.H)), dim3(64 * K::NW), K::kLds, s, A, (unsigned)gk);
  return (int)hipGetLastError();
}

template <typename T>
static int bwd_type(const DaArgs& A, hipStream_t s) {
  if (A.d <= 16) return bwd_go<T, 16>(A, s);
  if (A.d <= 32) return bwd_go<T, 32>(A, s);
  if (A.d <= 64) return bwd_go<T, 64>(A, s);
  if constexpr (DaT<T>::NP == 1) {
    if (A.d <= 128) return bwd_go<T, 128>(A, s);
  }
  return -22;
}

}  // namespace samble

using namespace samble;

extern "C" int samble_launch_diff_bwd(int type, const DaArgs* args, hipStream_t s) {
  Timed timed(kT_diff_bwd, s);
  return type == 0 ? bwd_type<float>(*args, s) : type == 1 ? bwd_type<f16>(*args, s) : bwd_type<bf16>(*args, s);
}
