// Differential attention, forward: one pass over the keys with the running maximum and sum of both softmax maps.
// Layout, operands and tiles: diff_dev.h.
//
// A wave owns 32 rows and keeps their Q operands, the softmax statistics and the unnormalised outputs O_1, O_2 in registers
// (the maps' normalisers are known at the end only, so P_1 - lam P_2 cannot be formed before).  S^T = K Q^T puts a row's
// logits into one lane column: maxima and sums are lane-local but for one exchange of the two halves.
//   RW  waves along the rows, each its own 32
//   KW  waves along the keys of a tile, each its own 32: for few rows (single tokens); their results meet in LDS
//   MW  waves along the maps: 1 = both in one wave, which share every value read; 2 where the outputs of two maps would
//       leave no registers (8 x 2048 x 8 heads of 128, bf16: 430 us, with its spills at the ends of the sweep; both maps in
//       one wave of 512 registers 4.5 ms), and for fp32 of 32-deep heads (557 us either way, without spills)
// Few rows against many keys are also split over workgroups (`splits`); diff_join_kernel adds the parts.
//
// Bound.  Many rows: a 32 x 32 block of both maps is 24 matrix instructions (d = 64; 768 cycles) and about 250 vector ones
// (1100 cycles: exponential, sum, maximum, conversion), which two waves of a SIMD can overlap but one wave issues one after
// the other.  8 x 2048 x 16 heads of 64, bf16, no mask: 412 us, 1000 TFLOP/s with both value products counted (a large matrix
// product reaches 1175), 493 us with what the backward needs; causal on 4 key heads 219 us.  fp32, 8 heads: 1000 us, 206
// TFLOP/s of six products each, all that the matrix unit gives.  Single tokens: the cache's bytes.  16 sequences of up to 8192
// keys, 8 key heads of 64, bf16: 80 + 5 us, 4.5 TB/s (fp32, all of 8192: 262 + 5 us, 4.1 TB/s; a tile's planes leave room for one
// workgroup a CU, and none of its loads is in flight while it splits them); one sequence of 128-deep heads: 52 + 9 us, 5.1 TB/s.
// A causal call whose blocks all start at once (2 x 2048, 4 key heads, for training: 95 us) lasts as long as the longest row
// block, alone on its CU at the end.
#include "diff_dev.h"

namespace samble {

template <typename T, int DP, int RW, int KW, int MW>
struct FwdCfg {
  static constexpr int NW = RW * KW * MW, NT = 64 * NW;
  static constexpr bool AHEAD = MW > 1 || DP < 64;            // the next step's logits before this one's exponentials (registers)
  static constexpr int SUB = KW > 1 && RW == 1 ? 1 : 2;                  // 32-key steps of a wave per tile
  static constexpr int KT = 32 * KW * SUB;
  static constexpr int DVT = 2 * DP / 32, MPW = 2 / MW;      // 32-column pieces of an output, maps of a wave
  typedef Feed<T, DP, KT, NT> Fd;
  static constexpr int kState = (DVT * 16 + 3) * MPW * 64;   // floats of a wave's state
  static constexpr int kMergeBytes = KW > 1 ? kState * 4 * (KW / 2) * RW * MW : MW > 1 ? DVT * 16 * 64 * 4 * RW : 0;
  static constexpr int kLds = Fd::kLds > kMergeBytes ? Fd::kLds : kMergeBytes;
};

// partial results of a split: per row (row order of the pair) reference, n, l of each map, two unused, then O_1, O_2 (2 d each)
__host__ __device__ __forceinline__ long da_part_floats(int d) { return 8 + 4l * d; }
__device__ __forceinline__ float da_inv(float l) { return l > 0.f ? 1.f / l : l; }   // (0 for a row without keys, NaN stays)
__device__ __forceinline__ float da_lse(float m, float l, int shift) {      // log2 of the row's sum
  return l == 0.f ? __builtin_huge_valf() : m - (float)shift + __builtin_amdgcn_logf(l);
}

// (Registers are held to two waves per SIMD, so that one wave's matrix instructions run under the other's exponentials; the
// whole file of 512 would put every accumulator into the half that the vector unit cannot read.  128-deep heads spill 22 .. 57
// registers, before and behind the sweep, not in it.)
// (BOTH: the backward comes.)
template <typename T, int DP, int RW, int KW, int MW, bool BOTH>
__global__ __launch_bounds__(64 * RW * KW * MW, 2) void diff_fwd_kernel(DaArgs A) {
  typedef FwdCfg<T, DP, RW, KW, MW> Cfg;
  typedef typename Cfg::Fd Fd;
  typedef typename Fd::Tl Tl;
  constexpr int KS = DP / 16, DVT = Cfg::DVT, MPW = Cfg::MPW;
  extern __shared__ __attribute__((aligned(16))) char smem[];

  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
  const int wave = da_uni(tid >> 6);
  const int rw = wave % RW, kw = KW > 1 ? (wave / RW) % KW : 0, mw = MW > 1 ? wave / (RW * KW) : 0;
  const unsigned rows = (unsigned)A.Nq * A.G;
  const unsigned blocks = (rows + 32 * RW - 1) / (32 * RW);
  unsigned part, pr;
  if (!da_unit(A, gridDim.x, blocks * A.splits, A.lengths && !A.causal && A.Hkv % 8, part, pr)) return;
  const unsigned split = A.splits > 1 ? part % A.splits : 0;
  const int pair = pr, b = da_uni(pair / A.Hkv), hk = pair - b * A.Hkv;
  const unsigned blk = blocks - 1 - (A.splits > 1 ? part / A.splits : part);      // (under a causal mask the long rows first)

  const int start = da_start(A, b), len = da_len(A, b, start);
  // this lane's row
  const unsigned first = blk * 32 * RW + 32 * rw, r = first + (lane & 31);
  const bool live = r < rows;
  const int qi = live ? (int)(r / (unsigned)A.G) : 0, head = hk * A.G + (live ? (int)(r % (unsigned)A.G) : 0);
  const int limit = live ? da_limit(A, len, start, qi) : 0;
  // keys that the last row of the workgroup sees; fewest keys of this wave's rows
  const unsigned last = blk * 32 * RW + 32 * RW - 1;
  const int kmax = da_limit(A, len, start, da_uni((last < rows ? last : rows - 1) / (unsigned)A.G));
  const int kmin = first + 31 < rows ? da_limit(A, len, start, da_uni(first / (unsigned)A.G)) : 0;

  const int tiles = (kmax + Cfg::KT - 1) / Cfg::KT;
  int t0 = 0, t1 = tiles;
  if (A.splits > 1) {
    const int each = da_uni(tiles / A.splits), more = tiles - each * A.splits;
    t0 = split * each + ((int)split < more ? split : more);
    t1 = t0 + each + ((int)split < more);
  }

  const Rows<T> keys = {(const T*)A.k + b * A.k_bs + hk * A.k_hs, (const T*)A.v + b * A.v_bs + hk * A.v_hs, A.k_ms, (int)A.k_rs, (int)A.v_rs,
                        len, A.d, A.key_mask ? A.key_mask + b * A.km_bs : nullptr};
  Fd feed(smem, tid);
  if (t0 < t1) feed.issue(keys, t0 * Cfg::KT);

  Lane<DP> L(lane, 32 * kw * Cfg::SUB);
  Frag<T> qf[MPW][KS];
  const float c = A.scale * kLog2e;      // logits' base-2 exponents per unit of the products
  {
    const T* qp = (const T*)A.q + b * A.q_bs + qi * A.q_rs + head * A.q_hs + mw * A.q_ms;
#pragma unroll
    for (int m = 0; m < MPW; ++m) da_row<T, KS>(qp + m * A.q_ms, A.d, live, h, qf[m]);
  }

  f32x16 o[MPW][DVT];
  // Reference of the exponentials, maximum from which it moves on (minus infinity: no key seen), sums.  The outputs are divided
  // by the sum of the rounded operands (n): a row that sees one key almost alone gives that key's value, whatever its
  // probability was rounded to (100 keys, d 16, bf16: outputs off by 2.1e-3 instead of 2.6e-3 of their norm, their own rounding
  // alone 1.7e-3).  The backward makes its probabilities from the sum before rounding (l, only where it comes; fp32: the same).
  constexpr bool kRounded = DaT<T>::NP == 1;
  float ref[MPW], more_at[MPW], l[MPW], n[MPW];
#pragma unroll
  for (int m = 0; m < MPW; ++m) {
    ref[m] = l[m] = n[m] = 0.f;
    more_at[m] = kNegInf;
#pragma unroll
    for (int t = 0; t < DVT; ++t) o[m][t] = zero16();
  }

  Frag<T> pf[MPW][2];       // the step's probabilities, operands of the value products
  // logits of the 32 keys at L + off
  auto logits = [&](const Lane<DP>& L, int off, f32x16 (&s)[MPW]) {
#pragma unroll
    for (int m = 0; m < MPW; ++m) {
      s[m] = zero16();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s[m] = da_mma<T>(Tl::map_rows(L, m, mw, off, ks), qf[m][ks], s[m]);
    }
  };
  // O += P V of the 32 keys at L + off
  auto values = [&](const Lane<DP>& L, int off) {
#pragma unroll
    for (int dt = 0; dt < DVT; ++dt)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const Frag<T> vf = Tl::cols(L, 1, off, u, 32 * dt);
#pragma unroll
        for (int m = 0; m < MPW; ++m) o[m][dt] = da_mma<T>(vf, pf[m][u], o[m][dt]);
      }
  };
  auto hide = [&](f32x16 (&s)[MPW], int k0, unsigned word) {       // what the rows do not see
    if (word != 0xffffffffu) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const bool see = da_bit(word, crow(e, 0));
#pragma unroll
        for (int m = 0; m < MPW; ++m) s[m][e] = see ? s[m][e] : kNegInf;
      }
    }
    if (k0 + 32 > kmin) {
      int left = limit - k0 - 4 * h;
      asm volatile("" : "+v"(left));   // (else the comparisons are made for every step, in front of the branch)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const bool see = crow(e, 0) < left;
#pragma unroll
        for (int m = 0; m < MPW; ++m) s[m][e] = see ? s[m][e] : kNegInf;
      }
    }
  };
  // The reference of the exponentials follows the maximum only when that has grown by more than 8 (a factor of 256 in the
  // sums): any reference gives the same quotients, and the outputs are rescaled in few of the steps.
  auto refer = [&](const f32x16 (&s)[MPW]) {
    float top[MPW];
    bool more = false;
#pragma unroll
    for (int m = 0; m < MPW; ++m) {
      top[m] = s[m][0];
#pragma unroll
      for (int e = 1; e < 16; ++e) top[m] = fmaxf(top[m], s[m][e]);      // (of this half of the keys: enough for the question)
      more = more || top[m] * c > more_at[m];
    }
    if (__any(more)) {
#pragma unroll
      for (int m = 0; m < MPW; ++m) {
        const float mx = fmaxf(more_at[m] == kNegInf ? kNegInf : ref[m], xor32_max(top[m]) * c);
        const float now = mx == kNegInf ? 0.f : mx;
        const float al = more_at[m] == kNegInf ? 1.f : __builtin_amdgcn_exp2f(ref[m] - now);      // (first: sums of zero)
        l[m] *= al;
        n[m] *= al;
#pragma unroll
        for (int dt = 0; dt < DVT; ++dt)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[m][dt][e] *= al;
        ref[m] = now;
        more_at[m] = mx + 8.f;
      }
    }
  };
  auto weigh = [&](const f32x16 (&s)[MPW], Frag<T> (&f)[MPW][2]) {
#pragma unroll
    for (int m = 0; m < MPW; ++m) {
      const float sub = ref[m] - (float)DaT<T>::kP;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          p[e] = __builtin_amdgcn_exp2f(fmaf(s[m][8 * u + e], c, -sub));
          if (BOTH) l[m] += p[e];
        }
        f[m][u] = da_pack<T>(p);
        if constexpr (kRounded) n[m] = da_sum8(f[m][u].p[0], n[m]);
      }
    }
  };

  for (int t = t0; t < t1; ++t) {
    feed.next(L);
    if (t + 1 < t1) feed.issue(keys, (t + 1) * Cfg::KT);
    f32x16 s[2][MPW];
    logits(L, 0, s[0]);
#pragma unroll
    for (int sub = 0; sub < Cfg::SUB; ++sub) {
      const int row0 = 32 * (kw * Cfg::SUB + sub), k0 = t * Cfg::KT + row0;
      if (sub && k0 >= kmax) break;   // (uniform; nothing of it is seen)
      const unsigned word = keys.mask ? feed.word(row0) : 0xffffffffu;
      hide(s[sub & 1], k0, word);
      refer(s[sub & 1]);
      if (Cfg::AHEAD && sub + 1 < Cfg::SUB) logits(L, 32 * (sub + 1), s[(sub + 1) & 1]);
      weigh(s[sub & 1], pf);
      values(L, 32 * sub);
      if (!Cfg::AHEAD && sub + 1 < Cfg::SUB) logits(L, 32 * (sub + 1), s[(sub + 1) & 1]);
    }
  }
#pragma unroll
  for (int m = 0; m < MPW; ++m) {
    l[m] = da_xor32_sum(l[m]);
    n[m] = kRounded ? da_xor32_sum(n[m]) : l[m];
    if (more_at[m] == kNegInf) ref[m] = kNegInf;
  }

  if constexpr (KW > 1) {   // the waves along the keys: pairwise, the upper half hands its state to the lower
    float* f = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int s = KW / 2; s > 0; s >>= 1) {
      __syncthreads();
      if (kw >= s && kw < 2 * s) {
        float* w = f + ((kw - s) * RW * MW + rw * MW + mw) * Cfg::kState + lane;
#pragma unroll
        for (int m = 0; m < MPW; ++m) {
          w[(3 * m) * 64] = ref[m];
          w[(3 * m + 1) * 64] = n[m];
          w[(3 * m + 2) * 64] = l[m];
#pragma unroll
          for (int dt = 0; dt < DVT; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) w[(3 * MPW + (m * DVT + dt) * 16 + e) * 64] = o[m][dt][e];
        }
      }
      __syncthreads();
      if (kw < s) {
        const float* w = f + (kw * RW * MW + rw * MW + mw) * Cfg::kState + lane;
#pragma unroll
        for (int m = 0; m < MPW; ++m) {
          const float m2 = w[(3 * m) * 64], n2 = w[(3 * m + 1) * 64], l2 = w[(3 * m + 2) * 64];
          const float nm = fmaxf(ref[m], m2), use = nm == kNegInf ? 0.f : nm;
          const float a1 = __builtin_amdgcn_exp2f(ref[m] - use), a2 = __builtin_amdgcn_exp2f(m2 - use);
          ref[m] = nm;
          n[m] = n[m] * a1 + n2 * a2;
          l[m] = l[m] * a1 + l2 * a2;
#pragma unroll
          for (int dt = 0; dt < DVT; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              o[m][dt][e] = o[m][dt][e] * a1 + w[(3 * MPW + (m * DVT + dt) * 16 + e) * 64] * a2;
        }
      }
    }
  }

  if (A.splits > 1) {
    if (kw || !live) return;
    float* w = A.part + (((long)split * A.B * A.Hkv + pair) * rows + r) * da_part_floats(A.d);
#pragma unroll
    for (int m = 0; m < MPW; ++m) {
      if (h == 0) {
        w[3 * (m + mw)] = ref[m];
        w[3 * (m + mw) + 1] = n[m];
        w[3 * (m + mw) + 2] = l[m];
      }
#pragma unroll
      for (int dt = 0; dt < DVT; ++dt)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          const int col = 32 * dt + 8 * q4 + 4 * h;
          if (col < 2 * A.d) {
            const f32x4 v = {o[m][dt][4 * q4], o[m][dt][4 * q4 + 1], o[m][dt][4 * q4 + 2], o[m][dt][4 * q4 + 3]};
            *reinterpret_cast<f32x4*>(w + 8 + 2 * (m + mw) * A.d + col) = v;
          }
        }
    }
    return;
  }
#pragma unroll
  for (int m = 0; m < MPW; ++m) {
    const float inv = da_inv(n[m]);
#pragma unroll
    for (int dt = 0; dt < DVT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[m][dt][e] *= inv;
    if (A.lse && live && kw == 0 && h == 0) A.lse[(((long)b * A.H + head) * 2 + m + mw) * A.Nq + qi] = da_lse(ref[m], l[m], DaT<T>::kP);
  }
  const float* f = reinterpret_cast<const float*>(smem) + rw * DVT * 16 * 64 + lane;   // two waves: the second map's output
  if constexpr (MW > 1) {
    __syncthreads();
    if (mw == 1 && kw == 0) {
#pragma unroll
      for (int dt = 0; dt < DVT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) const_cast<float*>(f)[(dt * 16 + e) * 64] = o[0][dt][e];
    }
    __syncthreads();
    if (mw == 1) return;
  }
  if (kw || !live) return;
  const float lam = da_lam<T>(A, head);
  const long at = (((long)b * A.Nq + qi) * A.H + head) * 2 * A.d;
  auto second = [&](int dt, int i) { return MW > 1 ? f[(dt * 16 + i) * 64] : o[MPW - 1][dt][i]; };
  if constexpr (DaT<T>::NP > 1) {
#pragma unroll
    for (int dt = 0; dt < DVT; ++dt)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const int col = 32 * dt + 8 * q4 + 4 * h;
        if (col >= 2 * A.d) continue;
        f32x4 a, z;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          z[e] = second(dt, 4 * q4 + e);
          a[e] = fmaf(-lam, z[e], o[0][dt][4 * q4 + e]);
        }
        *reinterpret_cast<f32x4*>((float*)A.out + at + col) = a;
        if (A.out2) *reinterpret_cast<f32x4*>((float*)A.out2 + at + col) = z;
      }
  } else {      // two groups of four columns, one of them the other half's: 16 bytes
#pragma unroll
    for (int dt = 0; dt < DVT; ++dt)
#pragma unroll
      for (int q4 = 0; q4 < 4; q4 += 2) {
        const int col = 32 * dt + 8 * (q4 + h);
        if (32 * dt + 8 * q4 >= 2 * A.d) continue;
        u32x4 a, z, r = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          vec4<T> x, y;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = 4 * (q4 + k) + e;
            const float v2 = second(dt, i), v = fmaf(-lam, v2, o[0][dt][i]);
            x[e] = (T)v;
            y[e] = (T)v2;
            if (BOTH) r[2 * k + (e >> 1)] |= da_rests<T>(v, x[e], v2, y[e]) << (16 * (e & 1));
          }
          const u32x2 xw = __builtin_bit_cast(u32x2, x), yw = __builtin_bit_cast(u32x2, y);
          a[2 * k] = xw[0], a[2 * k + 1] = xw[1];
          z[2 * k] = yw[0], z[2 * k + 1] = yw[1];
        }
        *reinterpret_cast<u32x4*>((T*)A.out + at + col) = da_halves(a);
        if (BOTH) {
          if (A.out2) *reinterpret_cast<u32x4*>((T*)A.out2 + at + col) = da_halves(z);
          if (A.rest) *reinterpret_cast<u32x4*>(A.rest + 2 * (at + col)) = da_halves(r);
        }
      }
  }
}

// adds the splits of a row.  NW = 16: a workgroup per row, a wave takes every sixteenth split (many splits, few rows); NW = 1:
// LPR lanes per row.  A lane takes four columns.
template <typename T, int NW, int LPR>
__global__ __launch_bounds__(NW == 1 ? 256 : 64 * NW) void diff_join_kernel(DaArgs A) {
  __shared__ __attribute__((aligned(16))) float red[NW == 1 ? 1 : NW][2][NW == 1 ? 4 : 256 + 4];
  const unsigned rows = (unsigned)A.Nq * A.G;
  const long all = (long)rows * A.B * A.Hkv;
  const int lane = threadIdx.x % LPR, wave = NW == 1 ? 0 : da_uni(threadIdx.x >> 6), cols = 2 * A.d;
  const long pf = da_part_floats(A.d), step = all * pf;
  constexpr int RPB = NW == 1 ? 256 / LPR : 1, kAtOnce = NW == 1 ? 4 : 2;
  for (long u = (long)blockIdx.x * RPB + (NW == 1 ? threadIdx.x / LPR : 0); u < all; u += (long)gridDim.x * RPB) {
    const unsigned pair = (unsigned)(u / rows), r = (unsigned)(u % rows);
    const int b = pair / A.Hkv, hk = pair % A.Hkv, qi = (int)(r / (unsigned)A.G), head = hk * A.G + (int)(r % (unsigned)A.G);
    const float* w = A.part + u * pf;
    float m[2] = {kNegInf, kNegInf};
    for (int s = NW == 1 ? 0 : lane; s < A.splits; s += NW == 1 ? 1 : 64) {
      const f32x4 t = *reinterpret_cast<const f32x4*>(w + s * step);
      m[0] = fmaxf(m[0], t[0]);
      m[1] = fmaxf(m[1], t[3]);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (NW > 1) m[k] = wave_max64(m[k]);
      if (m[k] == kNegInf) m[k] = 0.f;
    }
    const f32x4 none = {0.f, 0.f, 0.f, 0.f};
    f32x4 acc[2] = {none, none};
    float l[2] = {0.f, 0.f}, n[2] = {0.f, 0.f};
    const int c4 = 4 * lane < cols ? 4 * lane : 0;      // (lanes behind the last column: the first ones again, not used)
#pragma unroll kAtOnce
    for (int s = NW == 1 ? 0 : wave; s < A.splits; s += NW) {
      const float* p = w + s * step;
      const f32x4 t = *reinterpret_cast<const f32x4*>(p), t2 = *reinterpret_cast<const f32x4*>(p + 4);
      const f32x4 x = *reinterpret_cast<const f32x4*>(p + 8 + c4), y = *reinterpret_cast<const f32x4*>(p + 8 + cols + c4);
      const float a0 = __builtin_amdgcn_exp2f(t[0] - m[0]), a1 = __builtin_amdgcn_exp2f(t[3] - m[1]);
      n[0] = fmaf(t[1], a0, n[0]);
      l[0] = fmaf(t[2], a0, l[0]);
      n[1] = fmaf(t2[0], a1, n[1]);
      l[1] = fmaf(t2[1], a1, l[1]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        acc[0][e] = fmaf(x[e], a0, acc[0][e]);
        acc[1][e] = fmaf(y[e], a1, acc[1][e]);
      }
    }
    if constexpr (NW > 1) {      // onto the first wave, in order
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        *reinterpret_cast<f32x4*>(&red[wave][k][4 * lane]) = acc[k];
        if (lane == 0) {
          red[wave][k][256] = n[k];
          red[wave][k][257] = l[k];
        }
      }
      __syncthreads();
      if (wave == 0) {
#pragma unroll 1
        for (int i = 1; i < NW; ++i)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            n[k] += red[i][k][256];
            l[k] += red[i][k][257];
            acc[k] += *reinterpret_cast<const f32x4*>(&red[i][k][4 * lane]);
          }
      }
    }
    if (NW == 1 || wave == 0) {
      if (4 * lane < cols) {
        const float i1 = da_inv(n[0]), i2 = da_inv(n[1]), lam = da_lam<T>(A, head);
        const long o = (((long)b * A.Nq + qi) * A.H + head) * cols + 4 * lane;
        typedef T vec __attribute__((ext_vector_type(4)));
        vec a, z;
        u32x2 r = {0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v2 = acc[1][e] * i2, v = fmaf(-lam, v2, acc[0][e] * i1);
          a[e] = (T)v;
          z[e] = (T)v2;
          if constexpr (DaT<T>::NP == 1) r[e >> 1] |= da_rests<T>(v, a[e], v2, z[e]) << (16 * (e & 1));
        }
        *reinterpret_cast<vec*>((T*)A.out + o) = a;
        if (A.out2) *reinterpret_cast<vec*>((T*)A.out2 + o) = z;
        if (DaT<T>::NP == 1 && A.rest) *reinterpret_cast<u32x2*>(A.rest + 2 * o) = r;
      }
      if (A.lse && lane == 0) {
        float* ls = A.lse + ((long)b * A.H + head) * 2 * A.Nq + qi;
        ls[0] = da_lse(m[0], l[0], DaT<T>::kP);
        ls[A.Nq] = da_lse(m[1], l[1], DaT<T>::kP);
      }
    }
    if (NW > 1) __syncthreads();
  }
}

// ---- launches -------------------------------------------------------------------------------------------------------------
struct FwdPlan { bool few; long blocks; int splits; };

// Few rows (at most 32 of a key head) take the kernels whose waves stand along the keys.  Splits: as many as fill the CUs and no
// more, since a part of a second round costs a whole one (8 clouds of 1999 points, one head, fp32, d 64, joins included: 2 splits 155 us, 3
// splits 189 us); each split has at least four tiles of 128 keys, since its partial results go through memory, at most 128.
// Where two workgroups of four waves fit on a CU (not fp32 of 64-deep heads, 98 KB of tiles: 4 x 5 queries, 8 heads of 48, 5000 keys
// 82 us for two places, 54 us for one): as many as fill both places for few rows, and for keys so long that the parts
// are small beside them (4 x 1024 rows, 8 heads of 64, bf16: 2048 keys 85 us, in 2 splits 74 + 18; 4096 keys 163 us, 131 + 18).
static FwdPlan fwd_plan(bool wide, int B, int Nq, int Nk, int H, int Hkv, int d) {
  const long rows = (long)Nq * (H / Hkv), pairs = (long)B * Hkv;
  FwdPlan p;
  p.few = rows <= 32;
  p.blocks = p.few ? 1 : (rows + 127) / 128;
  const long have = p.blocks * pairs, room = (p.few && !(wide && d > 32)) || (d <= (wide ? 16 : 64) && Nk >= 4096) ? 512 : 256;
  long s = room / have;
  const long most = Nk / 512;
  if (s > most) s = most;
  if (s > 128) s = 128;
  p.splits = s < 1 ? 1 : (int)s;
  return p;
}

template <typename T, int DP, int RW, int KW, int DW>
static int fwd_go(const DaArgs& A, hipStream_t s) {
  typedef FwdCfg<T, DP, RW, KW, DW> Cfg;
  const long rows = (long)A.Nq * A.G, blocks = (rows + 32 * RW - 1) / (32 * RW);
  const long units = blocks * A.splits * A.B * A.Hkv, grid = (units + 7) / 8 * 8;
  if (grid * Cfg::NT >= (1ll << 32)) return -22;
  constexpr bool kAlways = DaT<T>::NP > 1;
  const auto f = A.lse ? diff_fwd_kernel<T, DP, RW, KW, DW, true> : diff_fwd_kernel<T, DP, RW, KW, DW, kAlways>;
  if (Cfg::kLds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(f), hipFuncAttributeMaxDynamicSharedMemorySize, Cfg::kLds);
    if (e != hipSuccess) return (int)e;
  }
  hipLaunchKernelGGL(f, dim3((unsigned)grid), dim3(Cfg::NT), Cfg::kLds, s, A);
  return (int)hipGetLastError();
}

template <typename T>
static int fwd_type(DaArgs& A, hipStream_t s) {
  const FwdPlan p = fwd_plan(DaT<T>::NP > 1, A.B, A.Nq, A.Nk, A.H, A.Hkv, A.d);
  A.splits = p.splits;
  constexpr bool F = DaT<T>::NP > 1;
  int rc = -22;
  if (A.d <= 16) rc = p.few ? fwd_go<T, 16, 1, 4, 1>(A, s) : fwd_go<T, 16, 4, 1, 1>(A, s);
  else if (A.d <= 32) rc = p.few ? fwd_go<T, 32, 1, 2, 2>(A, s) : fwd_go<T, 32, 4, 1, F ? 2 : 1>(A, s);
  else if (A.d <= 64) {
    if constexpr (F) rc = p.few ? fwd_go<T, 64, 1, 2, 2>(A, s) : fwd_go<T, 64, 4, 1, 2>(A, s);
    else rc = p.few ? fwd_go<T, 64, 1, 2, 2>(A, s) : fwd_go<T, 64, 4, 1, 1>(A, s);
  } else if constexpr (!F) {
    if (A.d <= 128) rc = p.few ? fwd_go<T, 128, 1, 2, 2>(A, s) : fwd_go<T, 128, 4, 1, 2>(A, s);
  }
  if (rc || A.splits == 1) return rc;
  const long all = (long)A.Nq * A.H * A.B;
  const long most = 1 << 20;      // workgroups of a launch: the kernel walks on
  const int lpr = A.splits >= 16 ? 256 : A.d <= 16 ? 8 : A.d <= 32 ? 16 : A.d <= 64 ? 32 : 64;
  const long need = (all * lpr + 255) / 256;
  const dim3 grid((unsigned)(need < most ? need : most));
  if (lpr == 256) hipLaunchKernelGGL((diff_join_kernel<T, 16, 64>), grid, dim3(1024), 0, s, A);
  else if (lpr == 8) hipLaunchKernelGGL((diff_join_kernel<T, 1, 8>), grid, dim3(256), 0, s, A);
  else if (lpr == 16) hipLaunchKernelGGL((diff_join_kernel<T, 1, 16>), grid, dim3(256), 0, s, A);
  else if (lpr == 32) hipLaunchKernelGGL((diff_join_kernel<T, 1, 32>), grid, dim3(256), 0, s, A);
  else if constexpr (!F) hipLaunchKernelGGL((diff_join_kernel<T, 1, 64>), grid, dim3(256), 0, s, A);
  return (int)hipGetLastError();
}

}  // namespace samble

using namespace samble;

extern "C" size_t samble_diff_fwd_ws_bytes(int type, int B, int Nq, int Nk, int H, int Hkv, int d) {
  const FwdPlan p = fwd_plan(type == 0, B, Nq, Nk, H, Hkv, d);
  return p.splits == 1 ? 0 : (size_t)p.splits * B * H * Nq * da_part_floats(d) * sizeof(float);
}

extern "C" int samble_launch_diff_fwd(int type, const DaArgs* args, hipStream_t s) {
  DaArgs A = *args;
  Timed timed(kT_diff_fwd, s);
  return type == 0 ? fwd_type<float>(A, s) : type == 1 ? fwd_type<f16>(A, s) : fwd_type<bf16>(A, s);
}
