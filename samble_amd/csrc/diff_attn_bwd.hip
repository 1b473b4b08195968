// Differential attention, backward.  With g = d loss / d out and dA = g v^T:
//     t_m[i] = sum_j P_m dA = g . (P_m v)_i,   dS_1 = P_1 (dA - t_1),   dS_2 = -lam P_2 (dA - t_2)
//     dq_m = scale dS_m k_m,  dk_m = scale dS_m^T q_m,  dv = (P_1 - lam P_2)^T g,  dlam = - sum_i t_2
// The logits are formed again from q and k; P = exp2(logit - lse) with the forward's row statistics.  No atomics:
//   diff_dq_kernel   a wave owns 32 rows (layout of the forward): first t_1 = g . out + lam t_2 and t_2 = g . out2 from the
//                    saved outputs, then one sweep over the keys.  16-bit outputs are rounded, and t of them is off by as much
//                    in all keys of a row: where the row sees one key almost alone, by more than dA - t itself (19 keys, bf16:
//                    dq off by 2.4 times its own rounding; 1.5 times with a whole t).  So the forward leaves a byte beside
//                    each (`rest`), and t has 15 bits at least.  Since sum_j P = 1, sum_j P (dA - t) is what still lacks; t
//                    plus that sum is kept for the second launch, whose dlam adds t over all rows
//                    fp16: dS is held times a power of two of the row, from the largest dA and t so far
//   diff_dkv_kernel  a wave owns 32 keys and sweeps over the rows of all query heads that share the key head, or over a part
//                    of them (`splits`, added by diff_dkv_join_kernel); workgroups behind the last one sum dlam
//                    fp16: P and dS are held times powers of two from the largest |lam| and the largest dA and t of all
//                    rows, which the first launch leaves
// Layout, operands and tiles: diff_dev.h.  The second kernel holds S with the row index on the registers, so that P and dS
// are operands of the sums over rows as they stand.
// P, P_1 - lam P_2 and dS of 16-bit tensors are rounded to the tensors' type, the type of the matrix instructions' operands (two
// planes would double their number): against float64 dq is off by 2.5e-3 and dk by 2.3e-3 of its norm in bf16, where rounding
// the results alone is 1.7e-3 (fp16: 3.2e-4, 2.1e-4); sums are fp32.
//
// Bound: as the forward's, matrix instructions (24 and 32 to a 32 x 32 block of d = 64) and vector ones of a wave in turn.
// 8 x 2048 x 16 heads of 64, bf16, no mask: dq 516 us (800 TFLOP/s), dk and dv 654 us (840); causal on 4 key heads dk and dv
// 418 us; fp32, 32 x 1024 x 4 heads of 16: 198 and 245 us (vector unit 0.6 of the busy cycles, matrix unit 0.5), 8 x 2048 x 8
// heads of 64: 1200 and 1516 us (1030 and 1090 TFLOP/s of the matrix unit's).
#include "diff_dev.h"

namespace samble {

// WPS: waves per SIMD.  Two, but where both maps' operands and gradients need more than 256 registers (8 x 2048 x 8 heads of
// 128, bf16: one wave with 512 registers 639 us, a wave for each map, both forming dA, 1194 us).
template <typename T, int DP>
struct DqCfg {
  static constexpr int RW = 4, NT = 64 * RW, WPS = DP == 128 || (DaT<T>::NP > 1 && DP == 64) ? 1 : 2;
  static constexpr int SUB = 2, KT = 32 * SUB;
  typedef Feed<T, DP, KT, NT> Fd;
  static constexpr int DT = DP < 32 ? 1 : DP / 32;     // 32-column pieces of a map's gradient (16 columns: both maps on one)
  static constexpr int kLds = Fd::kLds;
};

// the waves' largest values (fp16) in the row statistics, behind t_1 and t_2
__host__ __device__ __forceinline__ long da_bound_at(const DaArgs& A) { return 2l * A.B * A.H * A.Nq; }

template <typename T, int DP>
__global__ __launch_bounds__((DqCfg<T, DP>::NT), (DqCfg<T, DP>::WPS)) void diff_dq_kernel(DaArgs A) {
  typedef DqCfg<T, DP> Cfg;
  typedef typename Cfg::Fd Fd;
  typedef typename Fd::Tl Tl;
  constexpr int KS = DP / 16, DT = Cfg::DT, RW = Cfg::RW;
  extern __shared__ __attribute__((aligned(16))) char smem[];

  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
  const int rw = da_uni(tid >> 6);
  const unsigned rows = (unsigned)A.Nq * A.G, blocks = (rows + 32 * RW - 1) / (32 * RW);
  unsigned blk, pr;
  if (!da_unit(A, gridDim.x, blocks, A.lengths && !A.causal && A.Hkv % 8, blk, pr)) return;
  blk = blocks - 1 - blk;      // (under a causal mask the long rows first)
  const int pair = pr, b = da_uni(pair / A.Hkv), hk = pair - b * A.Hkv;
  const int start = da_start(A, b), len = da_len(A, b, start);
  const unsigned first = blk * 32 * RW + 32 * rw, r = first + (lane & 31);
  const bool live = r < rows;
  const int qi = live ? (int)(r / (unsigned)A.G) : 0, head = hk * A.G + (live ? (int)(r % (unsigned)A.G) : 0);
  const int limit = live ? da_limit(A, len, start, qi) : 0;
  const unsigned last = blk * 32 * RW + 32 * RW - 1;
  const int kmax = da_limit(A, len, start, da_uni((last < rows ? last : rows - 1) / (unsigned)A.G));
  const int kmin = first + 31 < rows ? da_limit(A, len, start, da_uni(first / (unsigned)A.G)) : 0;
  const int tiles = (kmax + Cfg::KT - 1) / Cfg::KT;

  const Rows<T> keys = {(const T*)A.k + b * A.k_bs + hk * A.k_hs, (const T*)A.v + b * A.v_bs + hk * A.v_hs, A.k_ms, (int)A.k_rs, (int)A.v_rs,
                        len, A.d, A.key_mask ? A.key_mask + b * A.km_bs : nullptr};
  Fd feed(smem, tid);
  if (tiles) feed.issue(keys, 0);

  Lane<DP> L(lane, 0);
  Frag<T> qf[2][KS], gf[2 * KS];
  const float c = A.scale * kLog2e;
  {
    const T* qp = (const T*)A.q + b * A.q_bs + qi * A.q_rs + head * A.q_hs;
#pragma unroll
    for (int m = 0; m < 2; ++m) da_row<T, KS>(qp + m * A.q_ms, A.d, live, h, qf[m]);
  }
  const float lam = da_lam<T>(A, head);
  float dot[2] = {0.f, 0.f};      // t_1, t_2
  {
    const T* gp = (const T*)A.dout + b * A.g_bs + qi * A.g_rs + head * A.g_hs;
    const long at = (((long)b * A.Nq + qi) * A.H + head) * 2 * A.d;
    da_row<T, 2 * KS>(gp, 2 * A.d, live, h, gf);
    // (four steps' loads in flight, and no branch around them: all of them take registers that the sweep then spills)
#pragma unroll 4
    for (int s = 0; s < 2 * KS; ++s) {
      const int o = 16 * s + 8 * h;
      const bool ok = live && o < 2 * A.d;
      Raw8<T> raw, o1, o2;
      raw.load(gp + o, ok);
      o1.load((const T*)A.out + at + o, ok);
      o2.load((const T*)A.out2 + at + o, ok);
      float g[8], u[8], w[8];
      raw.widen(g);
      o1.widen(u);
      o2.widen(w);
      if constexpr (DaT<T>::NP == 1) {
        const u32x4 none = {0, 0, 0, 0}, pairs = ok && A.rest ? *reinterpret_cast<const u32x4*>(A.rest + 2 * (at + o)) : none;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int pair = (int)(pairs[e >> 1] << (16 * (1 - (e & 1)))) >> 16;
          u[e] = da_whole<T>(u[e], (int)((unsigned)pair << 24) >> 24);
          w[e] = da_whole<T>(w[e], pair >> 8);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        dot[0] = fmaf(g[e], u[e], dot[0]);
        dot[1] = fmaf(g[e], w[e], dot[1]);
      }
    }
    dot[0] = da_xor32_sum(dot[0]);
    dot[1] = da_xor32_sum(dot[1]);
    dot[0] = fmaf(lam, dot[1], dot[0]);
  }
  float lse[2], tm[2], lack[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const long at = (((long)b * A.H + head) * 2 + m) * A.Nq + qi;
    lse[m] = live ? A.lse[at] : __builtin_huge_valf();
    tm[m] = dot[m];
    lack[m] = 0.f;
  }

  f32x16 acc[2][DT];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int t = 0; t < DT; ++t) acc[m][t] = zero16();

  // fp16: dS is held times fscale, a power of two for this lane's row: |dA| and |t| times it are below 2^13
  float fscale = 1.f;
  unsigned fbits = 0;
  if (kDaScaled<T>) {
    fbits = da_max_bits(da_max_bits(0u, tm[0]), tm[1]);
    fscale = da_scale(fbits);
  }

  for (int t = 0; t < tiles; ++t) {
    feed.next(L);
    if (t + 1 < tiles) feed.issue(keys, (t + 1) * Cfg::KT);
#pragma unroll
    for (int sub = 0; sub < Cfg::SUB; ++sub) {
      const int row0 = 32 * sub, k0 = t * Cfg::KT + row0;
      if (k0 >= kmax) continue;
      const unsigned word = keys.mask ? feed.word(row0) : 0xffffffffu;      // (rows end at their limits, at most len)
      f32x16 da = zero16();
#pragma unroll
      for (int ks = 0; ks < 2 * KS; ++ks) da = da_mma<T>(Tl::rows(L, 1, row0, ks), gf[ks], da);
      if (kDaScaled<T>) {
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(da[e]));
        const unsigned now = da_max_bits(0u, xor32_max(top));
        if (__any(now > (fbits | 0x007fffffu))) {     // a larger power of two than so far: few steps
          fbits = max(fbits, now);
          const float to = da_scale(fbits), f = to / fscale;
          fscale = to;
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            lack[m] *= f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
              for (int e = 0; e < 16; ++e) acc[m][dt][e] *= f;
          }
        }
      }
      Frag<T> ds[2][2];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        f32x16 s = zero16();
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s = da_mma<T>(Tl::rows(L, 0, row0, m * KS + ks), qf[m][ks], s);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], c, -lse[m]));
        if (word != 0xffffffffu) {
#pragma unroll
          for (int e = 0; e < 16; ++e) s[e] = da_bit(word, crow(e, 0)) ? s[e] : 0.f;
        }
        if (k0 + 32 > kmin) {
          int left = limit - k0 - 4 * h;
          asm volatile("" : "+v"(left));   // (else the comparisons are made for every tile, in front of the branch)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[e] = crow(e, 0) < left ? s[e] : 0.f;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float p[8];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            p[e] = s[8 * u + e] * (kDaScaled<T> ? fmaf(da[8 * u + e], fscale, -tm[m] * fscale) : da[8 * u + e] - tm[m]);
          if (DaT<T>::NP == 1) lack[m] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
          ds[m][u] = da_pack<T>(p);
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          Frag<T> kf;
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            if (DP >= 32 || m == 0) kf = DP < 32 ? Tl::cols(L, 0, row0, u, 0) : Tl::cols(L, 0, row0, u, m * DP + 32 * dt);
            acc[m][dt] = da_mma<T>(kf, ds[m][u], acc[m][dt]);
          }
        }
    }
  }
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    if (DaT<T>::NP == 1) tm[m] += da_xor32_sum(lack[m]) / fscale;
    if (live && h == 0) A.delta[(((long)b * A.H + head) * 2 + m) * A.Nq + qi] = tm[m];
  }
  if (kDaScaled<T>) {      // the wave's largest, for the second launch
    fbits = max(fbits, da_max_bits(da_max_bits(0u, tm[0]), tm[1]));
#pragma unroll
    for (int o = 32; o; o >>= 1) fbits = max(fbits, (unsigned)__shfl_xor((int)fbits, o, 64));
    if (lane == 0) reinterpret_cast<unsigned*>(A.delta)[da_bound_at(A) + ((long)pair * blocks + blk) * RW + rw] = fbits;
  }
  if (!live) return;
  T* dq = (T*)A.dq + (((long)b * A.Nq + qi) * A.H + head) * 2 * A.d;
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const float f = A.scale * (m ? -lam : 1.f) / fscale;      // dS_2 = -lam P_2 (dA - t_2)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int q4 = 0; q4 < (DP < 32 ? 2 : 4); ++q4) {
        const int col = 32 * dt + 8 * q4 + 4 * h, reg = 4 * (q4 + (DP < 32 ? 2 * m : 0));
        if (col >= A.d) continue;
        typedef T vec __attribute__((ext_vector_type(4)));
        vec v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)(f * acc[m][dt][reg + e]);
        *reinterpret_cast<vec*>(dq + m * A.d + col) = v;
      }
  }
}

// KBW waves along the keys, RWW along the rows of a tile (their sums meet in LDS).  `mirror`: half of a workgroup's keys are
// taken from the front and half from the back, so that under a causal mask, where the first keys are seen by all rows and the
// last ones by few, every workgroup has the same work; the four waves of a key block stand on the four SIMDs.  VL: the values, a
// stationary operand like the keys, stay in LDS instead of registers (64-deep heads and 32-deep ones of fp32: room for a second
// wave on the SIMD; fp32 of 64 and 128-deep heads: room at all).
template <typename T, int DP, int KBW, int RWW>
struct DkvCfg {
  static constexpr int NW = KBW * RWW, NT = 64 * NW, KB = 32 * KBW;
  static constexpr bool VL = DP >= 64 || (DaT<T>::NP > 1 && DP == 32);
  static constexpr int WPS = DP == 128 || (DaT<T>::NP > 1 && DP == 64) ? 1 : 2;      // waves per SIMD the registers allow
  static constexpr int SUB = RWW == 1 && !VL ? 2 : 1, RT = 32 * RWW * SUB;       // rows of a tile
  typedef Feed<T, DP, RT, NT> Fd;
  typedef Tile<T, DP, KB> Vt;
  static constexpr int DT = DP < 32 ? 1 : DP / 32, DVT = 2 * DP / 32;
  static constexpr int kStat = 4 * RT;       // lse_1, lse_2, t_1, t_2 of a tile's rows
  static constexpr int kVal = VL ? DaT<T>::NP * Vt::kPlane : 0;
  static constexpr int kState = (2 * DT + DVT) * 16 * 64;
  static constexpr int kMerge = RWW > 1 ? kState * 4 * KBW : 0;      // one wave's sums per key block at a time
  static constexpr int kBody = Fd::kLds + 2 * kStat * 4;
  static constexpr int kLds = (kBody > kMerge ? kBody : kMerge) + kVal;
};

template <typename T, int DP, int KBW, int RWW>
__global__ __launch_bounds__((DkvCfg<T, DP, KBW, RWW>::NT), (DkvCfg<T, DP, KBW, RWW>::WPS)) void diff_dkv_kernel(DaArgs A,
                                                                                                               unsigned main_grid,
                                                                                                               bool mirror) {
  typedef DkvCfg<T, DP, KBW, RWW> Cfg;
  typedef typename Cfg::Fd Fd;
  typedef typename Fd::Tl Tl;
  constexpr int KS = DP / 16, DT = Cfg::DT, DVT = Cfg::DVT, NT = Cfg::NT, RT = Cfg::RT;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  char* val = smem + Cfg::kLds - Cfg::kVal;
  float* stats = reinterpret_cast<float*>(smem + Fd::kLds);
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;

  if (blockIdx.x >= main_grid) {      // dlam of one head: - sum of t_2 over batch and queries (fewer than 2^31), eight loads in flight
    const int head = blockIdx.x - main_grid;
    const unsigned nq = A.Nq, all = (unsigned)A.B * nq;
    float sum = 0.f;
    for (unsigned first = tid; first < all; first += 8 * NT) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const unsigned e = first + k * NT, bb = e / nq;
        v[k] = e < all ? A.delta[(((long)bb * A.H + head) * 2 + 1) * nq + (e - bb * nq)] : 0.f;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += v[k];
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (lane == 0) stats[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0) {
      sum = 0.f;
      for (int w = 0; w < Cfg::NW; ++w) sum += stats[w];
      if (A.lam_f32) ((float*)A.dlam)[head] = -sum;
      else ((T*)A.dlam)[head] = (T)(-sum);
    }
    return;
  }

  const int wave = da_uni(tid >> 6), kb = wave / RWW, rww = RWW > 1 ? wave % RWW : 0;
  const unsigned blocks = ((unsigned)A.Nk + Cfg::KB - 1) / Cfg::KB;
  unsigned bl, pr;
  if (!da_unit(A, main_grid, blocks * A.splits, false, bl, pr)) return;
  const int split = A.splits > 1 ? bl % A.splits : 0, blk = A.splits > 1 ? bl / A.splits : bl, pair = pr, b = da_uni(pair / A.Hkv), hk = pair - b * A.Hkv;   // (causal: the keys that most rows see first)
  const int start = da_start(A, b), len = da_len(A, b, start);
  // first key of the workgroup's k-th block of 32 (mirrored ones end where the blocks from the front begin: Nk, no key)
  auto block_key = [&](int k) {
    if (!mirror) return blk * Cfg::KB + 32 * k;
    constexpr int HB = KBW / 2;
    if (k < HB) return 32 * (blk * HB + k);
    const int back = (A.Nk + 31) / 32 - 1 - (blk * HB + k - HB);
    return back >= (int)blocks * HB ? 32 * back : A.Nk;
  };
  const int key0 = block_key(0), kw0 = block_key(kb), key = kw0 + (lane & 31);
  const unsigned char* km = A.key_mask ? A.key_mask + b * A.km_bs : nullptr;
  const bool valid = key < len && (!km || km[key]);
  const bool any_valid = __any(valid);

  // rows that see any key of the workgroup: all behind the first such query
  const long i0 = A.causal && key0 > start ? (long)key0 - start : 0;
  const int per_head = (A.Nq + RT - 1) / RT;                            // tiles of a head
  const int tile0 = key0 >= len || i0 >= A.Nq ? per_head : (int)(i0 / RT);
  int g = 0, t = tile0, left = (per_head - tile0) * A.G;      // the tile that comes, tiles to go
  if (A.splits > 1) {      // (sizes end at 2^30 rows: the products fit)
    const int each = left / A.splits, more = left - each * A.splits, first = split * each + (split < more ? split : more);
    left = each + (split < more);
    if (left) {
      g = first / (per_head - tile0);
      t += first - g * (per_head - tile0);
    }
  }
  Rows<T> src = {nullptr, nullptr, A.q_ms, (int)A.q_rs, (int)A.g_rs, A.Nq, A.d, nullptr};
  const T* qb = (const T*)A.q + b * A.q_bs + (long)hk * A.G * A.q_hs;
  const T* gb = (const T*)A.dout + b * A.g_bs + (long)hk * A.G * A.g_hs;
  Fd feed(smem, tid);
  Lane<DP> L(lane, 32 * rww);
  // the rows' statistics go with their tile: copied like it (fp16 / bf16; rows behind the last: zeros), or through registers
  // (fp32; rows behind the last: P = 0)
  float sv[4] = {0.f, 0.f, 0.f, 0.f};
  int buf = 1;               // the statistics that are current; issue() fills the other ones
  auto issue = [&](int g, int t) {
    src.x = qb + g * A.q_hs;
    src.y = gb + g * A.g_hs;
    feed.issue(src, t * RT);
    const long hd = (long)b * A.H + hk * A.G + g;
    const float *ls = A.lse + hd * 2 * A.Nq, *tt = A.delta + hd * 2 * A.Nq;
    if constexpr (Fd::DMA) {
      float* to = stats + (buf ^ 1) * Cfg::kStat;
#pragma unroll
      for (int x = 0; x < 4 * RT / 64; x += Cfg::NW) {
        if (x + wave >= 4 * RT / 64) break;
        const int f = (x + wave) * 64 + lane, row = f % RT, i = t * RT + row;
        const float* from = f < 2 * RT ? ls : tt;
        if ((f / RT) & 1) from += A.Nq;
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void*)(i < A.Nq ? from + i : reinterpret_cast<const float*>(da_zero)),
            (__attribute__((address_space(3))) void*)(to + (x + wave) * 64), 4, 0, 0);
      }
    } else if (tid < RT) {
      const int i = t * RT + tid;
      const bool ok = i < A.Nq;
      sv[0] = ok ? ls[i] : __builtin_huge_valf();
      sv[1] = ok ? (ls + A.Nq)[i] : __builtin_huge_valf();
      sv[2] = ok ? tt[i] : 0.f;
      sv[3] = ok ? (tt + A.Nq)[i] : 0.f;
    }
  };
  if (left) issue(g, t);

  Frag<T> kf[2][KS], vf[Cfg::VL ? 1 : 2 * KS];
  const float c = A.scale * kLog2e;      // logits' base-2 exponents per unit of the products
  {
    const T* kp = (const T*)A.k + b * A.k_bs + hk * A.k_hs + (long)(valid ? key : 0) * A.k_rs;
    const T* vp = (const T*)A.v + b * A.v_bs + hk * A.v_hs;
#pragma unroll
    for (int m = 0; m < 2; ++m) da_row<T, KS>(kp + m * A.k_ms, A.d, valid, h, kf[m]);
    if constexpr (Cfg::VL) {
      for (int e = tid; e < Cfg::KB * DP / 4; e += NT) {
        const int row = e / (DP / 4), pc = e % (DP / 4), kk = block_key(row >> 5) + (row & 31);
        Raw8<T> raw;
        raw.load(vp + (long)kk * A.v_rs + pc * 8, kk < len && (!km || km[kk]) && pc * 8 < 2 * A.d);
        const Frag<T> f = raw.frag();
#pragma unroll
        for (int p = 0; p < Tl::NP; ++p)
          *reinterpret_cast<vec8<typename Tl::E>*>(val + p * Cfg::Vt::kPlane + da_off<DP>(row, pc)) = f.p[p];
      }
    } else {
      da_row<T, 2 * KS>(vp + (long)(valid ? key : 0) * A.v_rs, 2 * A.d, valid, h, vf);
    }
  }
  // fp16: P_1, lam P_2 and their difference are held times 2^kA (below 2^14), dS times 2^kA us (|dA - t| us <= 1)
  float us = 1.f, up = 1.f;      // up = 2^kA
  if constexpr (kDaScaled<T>) {
    const unsigned rows = (unsigned)A.Nq * A.G, waves = (rows + 127) / 128 * 4;
    const unsigned* at = reinterpret_cast<const unsigned*>(A.delta) + da_bound_at(A) + (long)pair * waves;
    unsigned bits = 0;
    for (unsigned e = tid; e < waves; e += NT) bits = max(bits, at[e]);
#pragma unroll
    for (int o = 32; o; o >>= 1) bits = max(bits, (unsigned)__shfl_xor((int)bits, o, 64));
    unsigned* red = reinterpret_cast<unsigned*>(stats + Cfg::kStat);      // (the first tile's statistics land in the other half)
    if (lane == 0) red[wave] = bits;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < Cfg::NW; ++w) bits = max(bits, red[w]);
    float lm = 0.f;
    for (int g = 0; g < A.G; ++g) lm = fmaxf(lm, fabsf(da_lam<T>(A, hk * A.G + g)));
    const int kA = 13 - min(max((int)((__float_as_uint(1.f + lm) >> 23) & 255) - 127, 0), 100);
    us = da_scale(da_uni(bits)) * 0x1p-14f;
    up = __uint_as_float((unsigned)(127 + kA) << 23);
  }
  f32x16 dk[2][DT], dv[DVT];
#pragma unroll
  for (int t = 0; t < DT; ++t) dk[0][t] = dk[1][t] = zero16();
#pragma unroll
  for (int t = 0; t < DVT; ++t) dv[t] = zero16();

  while (left) {
    const float lam = da_lam<T>(A, hk * A.G + g) * (kDaScaled<T> ? up * us : 1.f);
    buf ^= 1;
    float* stat = stats + buf * Cfg::kStat;
    feed.next(L, [&] {
      if (!Fd::DMA && tid < RT) {
#pragma unroll
        for (int e = 0; e < 4; ++e) stat[e * RT + tid] = sv[e];
      }
    });
    const int here = t;
    // the tile behind this one
    if (++t == per_head) {
      t = tile0;
      ++g;
    }
    if (--left) issue(g, t);
#pragma unroll
    for (int sub = 0; sub < Cfg::SUB; ++sub) {
        const int row0 = 32 * (rww + sub);
        const int i0 = here * RT + row0;
        // (uniform in the wave; a workgroup of neighbouring keys has hardly such a step)
        if (RWW > 1 && (!any_valid || i0 >= A.Nq || da_limit(A, len, start, min(i0 + 31, A.Nq - 1)) <= kw0)) continue;
        f32x16 da = zero16();
#pragma unroll
        for (int ks = 0; ks < 2 * KS; ++ks) {
          if constexpr (Cfg::VL) {
            const unsigned at = L.r[(ks >> 1) & (Lane<DP>::NR - 1)] + (unsigned)(Cfg::kLds - Cfg::kVal + (32 * kb - 32 * rww) * 4 * DP - (Fd::DMA ? feed.cur * Tl::kBytes : 0));
            da = da_mma<T>(Tl::rows(L, 1, 32 * sub, ks), Cfg::Vt::rows_at(at, 0, 0, ks), da);
          } else {
            da = da_mma<T>(Tl::rows(L, 1, 32 * sub, ks), vf[ks], da);
          }
        }
        // row i sees the key if i is at least `from`; rows behind the last see nothing.  (A key that does not exist is a column
        // of its own: zeros were read for it, and zeros are written, whatever its sums hold.)
        const int from = key - start;
        const bool masked = (A.causal && kw0 + 31 - start > i0) || i0 + 32 > A.Nq;
        f32x16 s[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          s[m] = zero16();
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) s[m] = da_mma<T>(Tl::rows(L, 0, 32 * sub, m * KS + ks), kf[m][ks], s[m]);
        }
        if (masked) {       // (what a row does not see: exp2 gives 0)
          int low = A.causal ? from - i0 - 4 * h : -32, end = A.Nq - i0 - 4 * h;
          asm volatile("" : "+v"(low), "+v"(end));
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const bool see = crow(e, 0) >= low && crow(e, 0) < end;
#pragma unroll
            for (int m = 0; m < 2; ++m) s[m][e] = see ? s[m][e] : kNegInf;
          }
        }
        // half of the rows at a time: their products run under the other half's exponentials
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float a[8], d1[8], d2[8];
#pragma unroll
          for (int q4 = 0; q4 < 2; ++q4) {
            const float* at = stat + row0 + 16 * u + 8 * q4 + 4 * h;
            const f32x4 l1 = *reinterpret_cast<const f32x4*>(at), l2 = *reinterpret_cast<const f32x4*>(at + RT);
            const f32x4 t1 = *reinterpret_cast<const f32x4*>(at + 2 * RT), t2 = *reinterpret_cast<const f32x4*>(at + 3 * RT);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int i = 8 * u + 4 * q4 + e, j = 4 * q4 + e;
              const float p1 = __builtin_amdgcn_exp2f(fmaf(s[0][i], c, -l1[e])) * (kDaScaled<T> ? up * us : 1.f);
              const float p2 = lam * __builtin_amdgcn_exp2f(fmaf(s[1][i], c, -l2[e]));
              a[j] = (p1 - p2) * (kDaScaled<T> ? 1.f / us : 1.f);
              d1[j] = p1 * (da[i] - t1[e]);
              d2[j] = p2 * (t2[e] - da[i]);
            }
          }
          const Frag<T> af = da_pack<T>(a), f1 = da_pack<T>(d1), f2 = da_pack<T>(d2);
#pragma unroll
          for (int dt = 0; dt < DVT; ++dt) dv[dt] = da_mma<T>(Tl::cols(L, 1, 32 * sub, u, 32 * dt), af, dv[dt]);
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            const Frag<T> q1 = Tl::cols(L, 0, 32 * sub, u, 32 * dt);
            dk[0][dt] = da_mma<T>(q1, f1, dk[0][dt]);
            const Frag<T> q2 = DP < 32 ? q1 : Tl::cols(L, 0, 32 * sub, u, DP + 32 * dt);
            dk[1][dt] = da_mma<T>(q2, f2, dk[1][dt]);
          }
        }
    }
  }
  const float kback = A.scale / (up * us), vback = 1.f / up;
  if constexpr (RWW > 1) {      // the waves along the rows: one after the other onto the first
    float* w = reinterpret_cast<float*>(smem) + kb * Cfg::kState + lane;
    for (int from = 1; from < RWW; ++from) {
      __syncthreads();
      if (rww == from) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            w[(dt * 16 + e) * 64] = dk[0][dt][e];
            w[((DT + dt) * 16 + e) * 64] = dk[1][dt][e];
          }
#pragma unroll
        for (int dt = 0; dt < DVT; ++dt)
#pragma unroll
          for (int e = 0; e < 16; ++e) w[((2 * DT + dt) * 16 + e) * 64] = dv[dt][e];
      }
      __syncthreads();
      if (rww == 0) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            dk[0][dt][e] += w[(dt * 16 + e) * 64];
            dk[1][dt][e] += w[((DT + dt) * 16 + e) * 64];
          }
#pragma unroll
        for (int dt = 0; dt < DVT; ++dt)
#pragma unroll
          for (int e = 0; e < 16; ++e) dv[dt][e] += w[((2 * DT + dt) * 16 + e) * 64];
      }
    }
    if (rww) return;
  }
  if (key >= A.Nk) return;
  const bool part = A.splits > 1;
  float* pp = part ? A.part + ((((long)split * A.B + b) * A.Nk + key) * A.Hkv + hk) * 4 * A.d : nullptr;      // dk, dv of one split
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
        f32x4 x;
        vec v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = valid ? kback * dk[m][dt][reg + e] : 0.f;
          v[e] = (T)x[e];
        }
        if (part) *reinterpret_cast<f32x4*>(pp + m * A.d + col) = x;
        else *reinterpret_cast<vec*>(dkp + m * A.d + col) = v;
      }
#pragma unroll
  for (int dt = 0; dt < DVT; ++dt)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      const int col = 32 * dt + 8 * q4 + 4 * h;
      if (col >= 2 * A.d) continue;
      f32x4 x;
      vec v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = valid ? vback * dv[dt][4 * q4 + e] : 0.f;
        v[e] = (T)x[e];
      }
      if (part) *reinterpret_cast<f32x4*>(pp + 2 * A.d + col) = x;
      else *reinterpret_cast<vec*>(dvp + col) = v;
    }
}

// dk, dv = sums of the splits, in order (a split call has few keys: 32-bit indices)
template <typename T>
__global__ __launch_bounds__(256) void diff_dkv_join_kernel(DaArgs A) {
  const unsigned d = A.d, all = (unsigned)A.B * A.Nk * A.Hkv * d;      // in fours
  for (unsigned i = blockIdx.x * 256 + threadIdx.x; i < all; i += gridDim.x * 256) {
    const float* p = A.part + 4ul * i;
    f32x4 sum = *reinterpret_cast<const f32x4*>(p);
#pragma unroll 4
    for (int s = 1; s < A.splits; ++s) sum += *reinterpret_cast<const f32x4*>(p + 4ul * all * s);
    typedef T vec __attribute__((ext_vector_type(4)));
    vec v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (T)sum[e];
    const unsigned row = i / d, c = 4 * (i - row * d);
    T* to = c < 2 * d ? (T*)A.dk + (unsigned long)row * 2 * d + c : (T*)A.dv + (unsigned long)row * 2 * d + c - 2 * d;
    *reinterpret_cast<vec*>(to) = v;
  }
}

template <typename K>
static int big_lds(K kernel, int bytes) {
  if (bytes <= 64 * 1024) return 0;
  return (int)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

// How dk and dv are divided.
//   half     workgroups of eight waves, 64 keys, four waves along the rows, where blocks of 128 keys are few (64 pairs of 500 rows
//            and 777 keys, fp16, d 32: 448 blocks 34 us, in eight waves 56 us; of 2000 rows and 350 keys, d 64: 192 blocks 114
//            us, in eight waves 106 us).  Under a causal mask more of them, so that the longest blocks, taken first, are not the
//            last to end (32 pairs of 8192 rows and 2048 keys: 512 blocks 581 us, in eight waves 438 us).  Wide heads have one form.
//   splits   of the rows, where even those are fewer than the CUs, under a causal mask fewer than two for each; at least eight
//            tiles of 128 rows to a split (8 pairs of 8192 rows and 2048 keys, causal, bf16, d 64: 157 us, in 2 splits 127 + 8;
//            2 pairs of 32 768 rows and 4096 keys, d 128: 1383 us, in 8 splits 371 + 24)
//   mirror   causal, few and short: keys from both ends in a workgroup
struct DkvPlan { bool half, mirror; int splits; };
static DkvPlan dkv_plan(bool wide, int B, int Nq, int Nk, int H, int Hkv, bool causal) {
  const long rows = (long)Nq * (H / Hkv), blocks = ((long)Nk + 127) / 128 * B * Hkv;
  DkvPlan p;
  p.half = !wide && blocks < (causal ? 1024 : 200);
  const long have = p.half ? 2 * blocks : blocks;
  long s = (causal ? 512 : 256) / have;
  if (s > rows / 1024) s = rows / 1024;
  p.splits = s < 1 ? 1 : s > 16 ? 16 : (int)s;
  p.mirror = p.half && causal && blocks < 256 && p.splits == 1;
  return p;
}
static size_t dkv_part_floats(bool wide, int B, int Nq, int Nk, int H, int Hkv, int d) {      // (causal: at least as many splits)
  const int s = dkv_plan(wide, B, Nq, Nk, H, Hkv, true).splits, t = dkv_plan(wide, B, Nq, Nk, H, Hkv, false).splits;
  return s > 1 || t > 1 ? (size_t)(s > t ? s : t) * B * Nk * Hkv * 4 * d : 0;
}
// t_1, t_2 of the rows, and the largest values of a pair's waves of 32 rows
static size_t bwd_row_floats(int B, int Nq, int H, int Hkv) {
  return ((size_t)B * H * 2 * Nq + ((size_t)Nq * (H / Hkv) + 127) / 128 * 4 * B * Hkv + 3) / 4 * 4;
}

template <typename T, int DP, int KBW, int RWW>
static int dkv_go(const DaArgs& A, bool mirror, hipStream_t s) {
  typedef DkvCfg<T, DP, KBW, RWW> K;
  const long grid = (((long)A.Nk + K::KB - 1) / K::KB * A.splits * A.B * A.Hkv + 7) / 8 * 8;
  if (const int rc = big_lds(diff_dkv_kernel<T, DP, KBW, RWW>, K::kLds)) return rc;
  hipLaunchKernelGGL((diff_dkv_kernel<T, DP, KBW, RWW>), dim3((unsigned)(grid + A.H)), dim3(K::NT), K::kLds, s, A, (unsigned)grid, mirror);
  if (A.splits > 1) {
    const unsigned need = ((unsigned)A.B * A.Nk * A.Hkv * A.d + 255) / 256;
    hipLaunchKernelGGL((diff_dkv_join_kernel<T>), dim3(need < 2048 ? need : 2048), dim3(256), 0, s, A);
  }
  return (int)hipGetLastError();
}

template <typename T, int DP>
static int bwd_go(DaArgs& A, hipStream_t s) {
  typedef DqCfg<T, DP> Q;
  constexpr bool kWide = DP == 128 || (DaT<T>::NP > 1 && DP == 64);
  const long rows = (long)A.Nq * A.G, pairs = (long)A.B * A.Hkv;
  const long grid = ((rows + 127) / 128 * pairs + 7) / 8 * 8, blocks = ((long)A.Nk + 127) / 128 * pairs;
  if (grid * Q::NT >= (1ll << 32) || (blocks + 8 + A.H) * 256 >= (1ll << 32)) return -22;      // (both launches, before the first)
  if (const int rc = big_lds(diff_dq_kernel<T, DP>, Q::kLds)) return rc;
  hipLaunchKernelGGL((diff_dq_kernel<T, DP>), dim3((unsigned)grid), dim3(Q::NT), Q::kLds, s, A);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  const DkvPlan p = dkv_plan(kWide, A.B, A.Nq, A.Nk, A.H, A.Hkv, A.causal);
  A.splits = p.splits;
  A.part = A.delta + bwd_row_floats(A.B, A.Nq, A.H, A.Hkv);
  if constexpr (!kWide) {
    if (p.half) return dkv_go<T, DP, 2, 4>(A, p.mirror, s);
  }
  return dkv_go<T, DP, 4, 1>(A, false, s);
}

template <typename T>
static int bwd_type(DaArgs& A, hipStream_t s) {
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

extern "C" size_t samble_diff_bwd_ws_bytes(int type, int B, int Nq, int Nk, int H, int Hkv, int d) {
  return (bwd_row_floats(B, Nq, H, Hkv) + dkv_part_floats(d > (type == 0 ? 32 : 64), B, Nq, Nk, H, Hkv, d)) * sizeof(float);
}

extern "C" int samble_launch_diff_bwd(int type, const DaArgs* args, hipStream_t s) {
  DaArgs A = *args;
  Timed timed(kT_diff_bwd, s);
  return type == 0 ? bwd_type<float>(A, s) : type == 1 ? bwd_type<f16>(A, s) : bwd_type<bf16>(A, s);
}
