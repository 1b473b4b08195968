// Arguments of the differential-attention launches (abi.hip -> diff_attn_fwd.hip, diff_attn_bwd.hip).
#pragma once

namespace samble {

struct DaArgs {
  const void *q, *k, *v, *lam, *dout;
  long q_bs, q_rs, q_hs, q_ms, k_bs, k_rs, k_hs, k_ms, v_bs, v_rs, v_hs, g_bs, g_rs, g_hs, km_bs;
  const int *lengths, *q_start;
  const unsigned char* key_mask;
  void *out, *out2;          // (B, Nq, H, 2 d); out2 = P_2 v
  signed char* rest;         // (B, Nq, H, 2 d, 2) or null: what the roundings of out and out2 to 16 bits leave (diff_dev.h da_rest)
  float *lse, *delta, *part; // lse: (B, H, 2, Nq); delta: t_1, t_2 alike, then the row blocks' largest values; part: partial results of the splits (forward: of the keys; backward: of the rows)
  void *dq, *dk, *dv, *dlam;
  int B, Nq, Nk, H, Hkv, G, d, causal, lam_f32, splits;
  float scale;
};

}  // namespace samble
