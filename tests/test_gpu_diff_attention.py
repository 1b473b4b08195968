"""Differential attention (samble_amd.attention.differential_attention, csrc/diff_attn_*.hip) against its formulas in float64.

Tolerances are sums of the roundings that the kernels are allowed, per element:
  * U = 2^-24 arithmetic.  A dot product of n terms in fp32 is off by at most (n + 32) U times the sum of magnitudes (fp32
    tensors: the two fp16 planes and three products lose a few U of the same sum, inside the 32).  With L the largest such sum
    over a row's logits, a probability is off by the factor 2 * ((d + 32) U L + 16 U); sums over n keys or rows by n U.
  * h = eps / 2 of the tensors' type: P, P_1 - lam P_2 and dS enter the second products rounded once (fp16 / bf16 only; fp32
    enters whole), saved outputs and results are rounded once.  fp16 adds half a subnormal step, 2^-25, where values are small.
  * fp32 operands are two fp16 planes of scaled values, whose smallest step leaves 2^-25 of the scaled value.  Forward: P
    (sum at least 1) is held times 2^6, 2^-31 of 1.  dv: the maps times 2^12, 2^-37 of 1 and of lam.  dS: times 2^12 and a
    factor that takes |g| |v| to at least 2^-2: 2^-35 |g| |v|.
"""
import math

import pytest
import torch

from samble_amd import _lib

U = 2.0 ** -24
DEV = "cuda"
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _visible(B, Nq, Nk, causal, lengths, q_start, key_mask, device):
    j = torch.arange(Nk, device=device)
    ok = torch.ones((B, Nq, Nk), dtype=torch.bool, device=device)
    if lengths is not None:
        ok &= (j < lengths[:, None])[:, None, :]
    if key_mask is not None:
        ok &= key_mask[:, None, :]
    if causal:
        start = torch.full((B,), Nk - Nq, device=device) if q_start is None else q_start
        ok &= j <= (torch.arange(Nq, device=device)[None, :, None] + start[:, None, None])
    return ok


def _check(q, k, v, lam, g, got, scale, causal, lengths, q_start, key_mask):
    """got = (out[, dq, dk, dv, dlam]) against float64 within the derived bounds; one (batch item, key head) at a time."""
    B, Nq, H, _, d = q.shape
    Nk, Hkv = k.shape[1:3]
    G = H // Hkv
    dt = q.dtype
    half = torch.finfo(dt).eps / 2
    hp = 0.0 if dt == torch.float32 else half       # P and dS as operands
    sub = 2.0 ** -25 if dt == torch.float16 else 0.0
    three = dt == torch.float32
    subp = 2.0 ** -31 if three else sub
    ok_all = _visible(B, Nq, Nk, causal, lengths, q_start, key_mask, q.device)
    lam_err = torch.zeros(H, dtype=torch.float64, device=q.device)
    lam_ref = torch.zeros(H, dtype=torch.float64, device=q.device)

    def held(x, ref, tol, what):
        tol = tol * (1 + 1e-3) + half * ref.abs() + sub + 1e-30
        err = (x.double() - ref).abs()
        bad = (err - tol).max().item() if err.numel() else 0.0
        assert bool(torch.isfinite(x).all()), f"{what}: not finite"
        assert bad <= 0, f"{what}: {bad:.3e} over the bound (worst error {err.max():.3e}, largest value {ref.abs().max():.3e})"

    for b in range(B):
        seen_key = ok_all[b].any(0)
        for hk in range(Hkv):
            # keys that do not exist may hold anything
            kk = torch.where(seen_key[:, None, None], k[b, :, hk].double(), 0.0)       # (Nk, 2, d)
            vv = torch.where(seen_key[:, None], v[b, :, hk].double(), 0.0)             # (Nk, 2d)
            dk_ref, dk_tol = torch.zeros_like(kk), torch.zeros_like(kk)
            dv_ref, dv_tol = torch.zeros_like(vv), torch.zeros_like(vv)
            ok = ok_all[b]
            for hq in range(hk * G, hk * G + G):
                qq, lm = q[b, :, hq].double(), float(lam[hq].double())
                P, dP = [], []
                for m in range(2):
                    s = qq[:, m] @ kk[:, m].T * scale
                    s = torch.where(ok, s, -math.inf)
                    top = s.amax(-1, keepdim=True)
                    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
                    tot = p.sum(-1, keepdim=True)
                    P.append(p / torch.where(tot == 0, 1.0, tot))
                    L = torch.where(ok, qq[:, m].abs() @ kk[:, m].abs().T * scale, 0.0).amax(-1, keepdim=True)
                    dP.append(2 * ((d + 32) * U * L + 16 * U) + Nk * U)                # relative error of the map, per row
                o1, o2 = P[0] @ vv, P[1] @ vv
                av = vv.abs()
                e1 = (P[0] * (dP[0] + hp)) @ av + subp * (ok.double() @ av)            # error of o1, o2 before rounding
                e2 = (P[1] * (dP[1] + hp)) @ av + subp * (ok.double() @ av)
                ref = o1 - lm * o2
                held(got[0][b, :, hq], ref, e1 + abs(lm) * e2 + 4 * U * (o1.abs() + abs(lm) * o2.abs()), f"out b{b} h{hq}")
                if g is None:
                    continue
                gg = g[b, :, hq].double()
                A = P[0] - lm * P[1]
                eA = P[0] * dP[0] + abs(lm) * P[1] * dP[1] + hp * A.abs() + (2.0 ** -37 * (1 + abs(lm)) if three else sub) * ok
                dv_ref += A.T @ gg
                dv_tol += eA.T @ gg.abs() + Nq * G * U * (A.abs().T @ gg.abs())
                dA = gg @ vv.T
                subs = (2.0 ** -35 * (1 + lam.double().abs().max()) * g[b].double().norm(dim=-1).max() * vv.norm(dim=-1).max()
                        if three else sub)
                edA = (2 * d + 32) * U * (gg.abs() @ av.T)
                t2 = (P[1] * dA).sum(-1, keepdim=True)
                t1 = (P[0] * dA).sum(-1, keepdim=True)
                out_err = e1 + abs(lm) * e2 + half * ref.abs() + sub
                out2_err = e2 + half * o2.abs() + sub
                n = (2 * d + 32) * U
                et2 = (gg.abs() * (out2_err + n * o2.abs())).sum(-1, keepdim=True)
                et1 = (gg.abs() * (out_err + n * ref.abs())).sum(-1, keepdim=True) + abs(lm) * et2
                lam_ref[hq] += -t2.sum()
                lam_err[hq] += et2.sum() + Nq * B * U * t2.abs().sum()
                for m, (t, et, sign) in enumerate(((t1, et1, 1.0), (t2, et2, -lm))):
                    dS = sign * P[m] * (dA - t)
                    edS = abs(sign) * P[m] * (edA + et + (dP[m] + 4 * U) * (dA - t).abs()) + hp * dS.abs() + subs * ok
                    dq_ref = scale * dS @ kk[:, m]
                    dq_tol = scale * (edS + Nk * U * dS.abs()) @ kk[:, m].abs()
                    held(got[1][b, :, hq, m], dq_ref, dq_tol, f"dq b{b} h{hq} m{m}")
                    dk_ref[:, m] += scale * dS.T @ qq[:, m]
                    dk_tol[:, m] += scale * (edS + Nq * G * U * dS.abs()).T @ qq[:, m].abs()
            if g is not None:
                held(got[2][b, :, hk], dk_ref, dk_tol, f"dk b{b} hk{hk}")
                held(got[3][b, :, hk], dv_ref, dv_tol, f"dv b{b} hk{hk}")
    if g is not None:
        held(got[4], lam_ref, lam_err + (torch.finfo(got[4].dtype).eps / 2) * lam_ref.abs(), "dlam")


def _inputs(B, Nq, Nk, H, Hkv, d, dtype, seed, packed=False, spread=1.4):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=gen, device=DEV)  # noqa: E731
    if packed:      # rows [Q | K | V] of one projection
        assert Nq == Nk and H == Hkv
        qkv = (spread * rnd(B, Nk, 3 * H * 2 * d)).to(dtype)
        q, k, v = qkv.split(H * 2 * d, 2)
        q, k, v = q.view(B, Nq, H, 2, d), k.view(B, Nk, H, 2, d), v.view(B, Nk, H, 2 * d)
    else:
        q, k = (spread * rnd(B, Nq, H, 2, d)).to(dtype), (spread * rnd(B, Nk, Hkv, 2, d)).to(dtype)
        v = rnd(B, Nk, Hkv, 2 * d).to(dtype)
    lam = (0.2 + 0.6 * torch.rand(H, generator=gen, device=DEV)).to(dtype if seed % 2 else torch.float32)
    g = rnd(B, Nq, H, 2 * d).to(dtype)
    return q, k, v, lam, g, gen


def _masks(kind, B, Nq, Nk, gen):
    lengths = q_start = key_mask = None
    causal = "causal" in kind
    if "lengths" in kind:
        lengths = torch.randint(0, Nk + 1, (B,), generator=gen, device=DEV, dtype=torch.int32)
        lengths[0] = Nk
        if B > 1:
            lengths[1] = 0
        if causal:
            q_start = lengths - Nq
    if "keys" in kind:
        key_mask = torch.rand((B, Nk), generator=gen, device=DEV) > 0.3
        key_mask[-1, : Nk // 2] = False
    return causal, lengths, q_start, key_mask


# B, Nq, Nk, H, Hkv, d, masks
CASES = [
    (1, 1, 1, 1, 1, 8, ""), (2, 1, 33, 4, 4, 16, "lengths"), (3, 5, 7, 2, 1, 24, "keys"), (2, 33, 31, 3, 3, 16, "causal"),
    (2, 31, 65, 4, 2, 32, "causal"), (1, 64, 64, 2, 2, 64, "causal"), (2, 129, 127, 2, 1, 64, "causal lengths"),
    (3, 100, 300, 4, 4, 40, "lengths keys"), (2, 257, 130, 6, 2, 8, "causal keys"), (1, 200, 200, 5, 1, 48, "causal"),
    (2, 96, 515, 2, 2, 56, "lengths"), (1, 1, 700, 8, 1, 64, ""), (4, 3, 2100, 8, 2, 32, "lengths causal"),
    (1, 7, 1500, 40, 8, 16, "keys"), (1, 300, 2600, 2, 2, 16, "causal"), (2, 70, 1, 2, 2, 16, ""),
]
WIDE = [(1, 1, 600, 4, 2, 128, "lengths"), (2, 65, 130, 2, 1, 128, "causal"), (2, 150, 70, 2, 2, 96, "keys"),
        (1, 200, 2100, 1, 1, 72, "causal"), (1, 1, 5000, 4, 1, 128, "")]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES + WIDE, ids=lambda c: "-".join(str(x).replace(" ", "+") or "full" for x in c))
@pytest.mark.parametrize("dtype", list(TYPES))
def test_forward_and_gradients(case, dtype):
    from samble_amd.attention import differential_attention
    B, Nq, Nk, H, Hkv, d, kind = case
    if dtype == "fp32" and d > 64:
        pytest.skip("fp32: d up to 64")
    q, k, v, lam, g, gen = _inputs(B, Nq, Nk, H, Hkv, d, TYPES[dtype], sum(case[:6]))
    causal, lengths, q_start, key_mask = _masks(kind, B, Nq, Nk, gen)
    kw = dict(causal=causal, lengths=lengths, q_start=q_start, key_mask=key_mask)
    leaves = [t.requires_grad_(True) for t in (q, k, v, lam)]
    out = differential_attention(*leaves, **kw)
    grads = torch.autograd.grad(out, leaves, g)
    _check(q.detach(), k.detach(), v.detach(), lam.detach(), g, (out.detach(),) + grads, d ** -0.5, causal, lengths, q_start, key_mask)
    with torch.no_grad():
        assert torch.equal(differential_attention(q, k, v, lam, **kw), out)
    again = torch.autograd.grad(differential_attention(*leaves, **kw), leaves, g)
    assert all(torch.equal(a, b) for a, b in zip(again, grads)), "not the same run to run"


# many pairs of an item and a key head, in the orders that workgroups take them: longest blocks first, keys from both ends, pairs
# dealt to the XCDs one by one or (pairs no multiple of eight; lengths) block by block
MANY = [(32, 130, 520, 8, 8, 16, "causal lengths"), (8, 520, 520, 4, 4, 32, "causal"), (16, 300, 1030, 8, 4, 16, "causal lengths keys"),
        (16, 200, 600, 6, 3, 24, "lengths"), (5, 200, 600, 3, 3, 64, "lengths"), (7, 150, 400, 1, 1, 40, "causal lengths"),
        (8, 1, 700, 8, 1, 64, "lengths"), (4, 3, 2600, 4, 2, 32, "causal lengths")]


@pytest.mark.gpu
@pytest.mark.parametrize("case", MANY, ids=lambda c: "-".join(str(x).replace(" ", "+") or "full" for x in c))
@pytest.mark.parametrize("dtype", list(TYPES))
def test_many_pairs(case, dtype):
    test_forward_and_gradients(case, dtype)


# few keys under many rows: dk and dv as sums of parts of the rows
ROWS = [(1, 2100, 130, 2, 1, 64, ""), (2, 1100, 300, 8, 2, 16, "causal lengths keys"), (1, 3000, 3000, 1, 1, 32, "causal"),
        (1, 1500, 77, 4, 2, 128, "lengths"), (1, 5000, 40, 4, 4, 24, "keys"), (1, 2500, 200, 2, 2, 40, "causal"),
        (1, 1025, 1, 2, 1, 8, "")]


@pytest.mark.gpu
@pytest.mark.parametrize("case", ROWS, ids=lambda c: "-".join(str(x).replace(" ", "+") or "full" for x in c))
@pytest.mark.parametrize("dtype", list(TYPES))
def test_few_keys_under_many_rows(case, dtype):
    test_forward_and_gradients(case, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_long_cache_single_token(dtype):
    from samble_amd.attention import differential_attention
    q, k, v, lam, _, gen = _inputs(2, 1, 20011, 8, 2, 64, TYPES[dtype], 4)
    lengths = torch.tensor([20011, 9001], dtype=torch.int64, device=DEV)
    out = differential_attention(q, k, v, lam, lengths=lengths)
    _check(q, k, v, lam, None, (out,), 0.125, False, lengths, None, None)
    # the cache as a model holds it: heads before positions, longer than what is filled
    cache_k = torch.full((2, 2, 20100, 2, 64), float("nan"), dtype=TYPES[dtype], device=DEV)
    cache_v = torch.full((2, 2, 20100, 128), float("nan"), dtype=TYPES[dtype], device=DEV)
    cache_k[:, :, :20011], cache_v[:, :, :20011] = k.transpose(1, 2), v.transpose(1, 2)
    cache_k[1, :, 9001:], cache_v[1, :, 9001:] = float("nan"), float("inf")
    held = differential_attention(q, cache_k.transpose(1, 2), cache_v.transpose(1, 2), lam, lengths=lengths)
    _check(q, k, v, lam, None, (held,), 0.125, False, lengths, None, None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_strided_operands_scale_and_one_lam(dtype):
    from samble_amd.attention import differential_attention
    q, k, v, lam, g, _ = _inputs(2, 150, 150, 4, 4, 16, TYPES[dtype], 11, packed=True)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    one = torch.tensor(0.35, device=DEV, requires_grad=True)
    out = differential_attention(*leaves, one, scale=0.4)
    grads = torch.autograd.grad(out, leaves + [one], g)
    full = torch.full((4,), 0.35, device=DEV)
    split = torch.autograd.grad(differential_attention(*leaves, full.requires_grad_(True), scale=0.4), leaves + [full], g)
    assert all(torch.equal(a, b) for a, b in zip(grads[:3], split[:3]))
    torch.testing.assert_close(grads[3], split[3].sum(), rtol=1e-5, atol=1e-5)
    _check(q, k, v, full.detach(), g, (out.detach(),) + split, 0.4, False, None, None, None)
    # rows that do not start on 16 bytes, a gradient that is an expanded value, a transposed output gradient
    odd = [torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape).copy_(t.detach()) for t in leaves]
    assert torch.equal(differential_attention(*odd, 0.35, scale=0.4), out)
    ones = torch.autograd.grad(differential_attention(*leaves, 0.35, scale=0.4).sum(), leaves)
    same = torch.autograd.grad(differential_attention(*leaves, 0.35, scale=0.4), leaves, torch.ones_like(out))
    assert all(torch.equal(a, b) for a, b in zip(ones, same))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_axes_of_one_with_any_stride(dtype):
    from samble_amd.attention import differential_attention
    q, k, v, lam, g, _ = _inputs(1, 1, 40, 1, 1, 16, TYPES[dtype], 8)
    odd = lambda t: t.as_strided(t.shape, [s if n > 1 else 2 ** 40 + 3 for s, n in zip(t.stride(), t.shape)])  # noqa: E731
    leaves = [t.requires_grad_(True) for t in (q, k, v, lam)]
    plain = differential_attention(*leaves)
    other = differential_attention(odd(q), odd(k), odd(v), lam)
    assert torch.equal(plain, other)
    for a, b in zip(torch.autograd.grad(plain, leaves, g), torch.autograd.grad(other, leaves, odd(g))):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_nothing_of_missing_keys_is_used(dtype):
    from samble_amd.attention import differential_attention
    q, k, v, lam, g, gen = _inputs(3, 40, 90, 2, 2, 32, TYPES[dtype], 21)
    lengths = torch.tensor([90, 0, 50], dtype=torch.int32, device=DEV)
    mask = torch.rand((3, 90), generator=gen, device=DEV) > 0.4
    gone = ~(mask & (torch.arange(90, device=DEV) < lengths[:, None]))
    res = []
    for filler in (0.0, float("nan"), float("inf"), torch.finfo(TYPES[dtype]).min):
        kk, vv = k.clone(), v.clone()
        kk[gone], vv[gone] = filler, -filler if filler == filler else filler
        leaves = [t.detach().requires_grad_(True) for t in (q, kk, vv, lam)]
        out = differential_attention(*leaves, lengths=lengths, key_mask=mask)
        res.append((out.detach(),) + torch.autograd.grad(out, leaves, g))
    for other in res[1:]:
        assert all(torch.equal(a, b) for a, b in zip(res[0], other))
    out, dq, dk, dv, _ = res[0]
    assert not out[1].any() and not dq[1].any()
    assert not dk[gone].any() and not dv[gone].any()


@pytest.mark.gpu
@pytest.mark.parametrize("Nq,starts", [(1, [40, 5, -3]), (33, [0, 57, -40]), (200, [10, -150, 60])])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_keys_behind_the_last_query_are_not_used(dtype, Nq, starts):
    """A cache with room to grow: what stands behind the positions of the queries has not been written yet."""
    from samble_amd.attention import differential_attention
    q, k, v, lam, g, gen = _inputs(3, Nq, 300, 4, 2, 32, TYPES[dtype], 33)
    start = torch.tensor(starts, dtype=torch.int32, device=DEV)
    gone = torch.arange(300, device=DEV) >= (start + Nq)[:, None]
    res = []
    for filler in (0.0, float("nan"), float("inf")):
        kk, vv = k.clone(), v.clone()
        kk[gone], vv[gone] = filler, filler
        leaves = [t.detach().requires_grad_(True) for t in (q, kk, vv, lam)]
        out = differential_attention(*leaves, causal=True, q_start=start)
        assert torch.equal(differential_attention(q, kk, vv, lam, causal=True, q_start=start), out)
        res.append((out.detach(),) + torch.autograd.grad(out, leaves, g))
    for other in res[1:]:
        assert all(torch.equal(a, b) for a, b in zip(res[0], other))
    assert not res[0][2][gone].any() and not res[0][3][gone].any()
    kk, vv = torch.where(gone[:, :, None, None, None], 0, k), torch.where(gone[:, :, None, None], 0, v)
    _check(q, kk, vv, lam, g, res[0], 32 ** -0.5, True, None, start, None)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [16, 64, 128])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_dlam_is_not_that_of_rounded_outputs(dtype, d):
    """Values 1 and 1 + eps, two in five of them the larger: every output of the second map is 1 + 0.4 eps, which the tensors'
    type rounds to 1 in all rows and columns.  With q = 0 the maps are uniform, and dlam = - Nq 2 d (1 + 0.4 eps) but for fp32
    sums over 2 d columns, Nk keys and Nq rows and a few steps each for the map, its normaliser and t."""
    from samble_amd.attention import differential_attention

    dt = TYPES[dtype]
    Nq, Nk = 40, 320
    eps = torch.finfo(dt).eps
    larger = torch.tensor([0.0, 0.0, 1.0, 0.0, 1.0], device=DEV).repeat(Nk // 5)
    q = torch.zeros(1, Nq, 1, 2, d, dtype=dt, device=DEV)
    k = torch.ones(1, Nk, 1, 2, d, dtype=dt, device=DEV)
    v = (1 + eps * larger).to(dt)[None, :, None, None].expand(1, Nk, 1, 2 * d).contiguous()
    lam = torch.full((1,), 0.5, device=DEV, requires_grad=True)
    out = differential_attention(q, k, v, lam)
    (dlam,) = torch.autograd.grad(out, lam, torch.ones_like(out))
    ref = -Nq * 2 * d * (1 + 0.4 * eps)
    assert abs(dlam.item() - ref) <= (2 * d + Nk + Nq + 96) * U * abs(ref)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["keys", "causal lengths keys"])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_missing_keys_beside_logits_far_below_zero(dtype, kind):
    """Visible logits around -140: a missing key's column, read as zeros, would get probabilities beyond fp32."""
    from samble_amd.attention import differential_attention
    q, k, v, lam, g, gen = _inputs(3, 200, 260, 2, 2, 32, TYPES[dtype], 61, spread=0.3)
    q, k = q + 5, k - 5
    causal, lengths, q_start, key_mask = _masks(kind, 3, 200, 260, gen)
    kw = dict(causal=causal, lengths=lengths, q_start=q_start, key_mask=key_mask)
    leaves = [t.requires_grad_(True) for t in (q, k, v, lam)]
    out = differential_attention(*leaves, **kw)
    grads = torch.autograd.grad(out, leaves, g)
    gone = ~_visible(3, 200, 260, causal, lengths, q_start, key_mask, DEV).any(1)
    assert gone.any() and not grads[1][gone].any() and not grads[2][gone].any()
    _check(*[t.detach() for t in leaves], g, (out.detach(), *grads), 32 ** -0.5, causal, lengths, q_start, key_mask)


@pytest.mark.gpu
def test_lengths_and_starts_out_of_range_are_taken_to_the_nearest():
    from samble_amd.attention import differential_attention
    q, k, v, lam, _, _ = _inputs(4, 6, 20, 2, 2, 16, torch.float32, 3)
    wild = torch.tensor([-5, 1000, 2 ** 40, -(2 ** 40)], device=DEV)
    tame = torch.tensor([0, 20, 20, 0], device=DEV)
    assert torch.equal(differential_attention(q, k, v, lam, lengths=wild), differential_attention(q, k, v, lam, lengths=tame))
    starts = torch.tensor([-100, 2 ** 31 - 1, -2, 3], device=DEV, dtype=torch.int64)
    out = differential_attention(q, k, v, lam, causal=True, q_start=starts)
    assert not out[0].any() and not out[2, :2].any() and out[2, 2].any()
    assert torch.equal(out[1], differential_attention(q, k, v, lam)[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_extreme_logits_and_infinities_stay_in_their_rows(dtype):
    from samble_amd.attention import differential_attention
    q, k, v, lam, g, _ = _inputs(1, 70, 200, 1, 1, 16, TYPES[dtype], 6, spread=12.0)     # logits of several hundred
    leaves = [t.requires_grad_(True) for t in (q, k, v, lam)]
    out = differential_attention(*leaves)
    grads = torch.autograd.grad(out, leaves, g)
    _check(q.detach(), k.detach(), v.detach(), lam.detach(), g, (out.detach(),) + grads, 0.25, False, None, None, None)
    bad = q.detach().clone()
    bad[0, 13] = float("nan")
    bad[0, 44, 0, 0, 3] = float("inf")
    with torch.no_grad():
        res = differential_attention(bad, k, v, lam)
    rows = torch.ones(70, dtype=torch.bool, device=DEV)
    rows[[13, 44]] = False
    assert torch.equal(res[0, rows], out[0, rows]) and torch.isnan(res[0, 13]).all() and not torch.isfinite(res[0, 44]).all()


@pytest.mark.gpu
def test_gradients_against_differences():
    """central differences of a scalar of the output in float64 arithmetic of the formula, at a few coordinates"""
    from samble_amd.attention import differential_attention
    q, k, v, lam, g, _ = _inputs(1, 20, 24, 2, 1, 8, torch.float32, 2)
    leaves = [t.requires_grad_(True) for t in (q, k, v, lam)]
    grads = torch.autograd.grad(differential_attention(*leaves, causal=True), leaves, g)

    def value(q, k, v, lam):
        ok = _visible(1, 20, 24, True, None, None, None, DEV)[0]
        total = 0.0
        for h in range(2):
            p = [torch.softmax((q[0, :, h, m] @ k[0, :, 0, m].T / math.sqrt(8)).masked_fill(~ok, -math.inf), -1) for m in range(2)]
            total += (((p[0] - lam[h] * p[1]) @ v[0, :, 0]) * g[0, :, h].double()).sum()
        return float(total)

    base = [t.detach().double() for t in leaves]
    for n, t in enumerate(base):
        for at in (0, t.numel() // 3, t.numel() - 1):
            for step in (1e-5,):
                lo, hi = t.clone(), t.clone()
                lo.view(-1)[at] -= step
                hi.view(-1)[at] += step
                diff = (value(*base[:n], hi, *base[n + 1:]) - value(*base[:n], lo, *base[n + 1:])) / (2 * step)
                assert abs(diff - grads[n].reshape(-1)[at].item()) <= 1e-5 * (1 + abs(diff)), (n, at)


@pytest.mark.gpu
def test_empty_sizes_and_frozen_inputs():
    from samble_amd.attention import differential_attention
    for B, Nq, Nk in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        q, k, v, lam, _, _ = _inputs(B, Nq, Nk, 2, 1, 16, torch.bfloat16, 1)
        leaves = [t.requires_grad_(True) for t in (q, k, v, lam)]
        out = differential_attention(*leaves)
        assert out.shape == (B, Nq, 2, 32) and not out.any()
        assert all(not t.any() for t in torch.autograd.grad(out.sum(), leaves))
    q, k, v, lam, g, _ = _inputs(1, 9, 9, 2, 2, 16, torch.float32, 1)
    both = torch.autograd.grad(differential_attention(q.requires_grad_(True), k, v.requires_grad_(True), lam), (q, v), g)
    (only,) = torch.autograd.grad(differential_attention(q, k, v.detach(), lam), q, g)
    assert torch.equal(both[0], only)


@pytest.mark.gpu
def test_other_stream_and_graph_replay():
    from samble_amd.attention import differential_attention
    q, k, v, lam, g, gen = _inputs(2, 200, 200, 4, 2, 32, torch.bfloat16, 8)
    tok = q[:, :1]
    leaves = [t.requires_grad_(True) for t in (q, k, v, lam)]

    def step():
        out = differential_attention(*leaves, causal=True)
        return (out.detach(),) + torch.autograd.grad(out, leaves, g)

    def serve():
        with torch.no_grad():
            return differential_attention(tok, long_k, long_v, lam, lengths=lengths)

    long_k, long_v = (torch.randn(s, generator=gen, device=DEV).bfloat16() for s in ((2, 4000, 2, 2, 32), (2, 4000, 2, 64)))
    lengths = torch.tensor([4000, 77], dtype=torch.int32, device=DEV)
    eager, answer = step(), serve()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other, there = step(), serve()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, other)) and torch.equal(answer, there)
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    with torch.cuda.graph(graph2):
        held2 = serve()
    for n in (3999, 1, 0, 2500):
        with torch.no_grad():
            q.copy_(torch.randn(q.shape, generator=gen, device=DEV))
            lengths[0] = n
        graph.replay()
        graph2.replay()
        eager, answer = step(), serve()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, held)) and torch.equal(answer, held2), n


@pytest.mark.gpu
def test_two_threads_on_their_own_streams():
    """Calls of different shapes at the same time, forward and backward, with the layer norm behind them."""
    import threading

    from samble_amd.attention import differential_attention
    from samble_amd.norm import layer_norm

    def work(seed, dims, dtype):
        q, k, v, lam, g, _ = _inputs(*dims, dtype, seed)
        leaves = [t.requires_grad_(True) for t in (q, k, v, lam)]
        y = layer_norm(differential_attention(*leaves, causal=True))
        return (y.detach(), *torch.autograd.grad(y, leaves, g))

    jobs = [(2, (2, 300, 700, 4, 2, 64), torch.bfloat16), (5, (3, 200, 200, 2, 2, 32), torch.float32),
            (8, (1, 2, 9000, 8, 2, 128), torch.float16)]
    alone = [work(*j) for j in jobs]
    torch.cuda.synchronize()
    errors = []

    def run(job, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()) as _:
                for _ in range(10):
                    got = work(*job)
                    torch.cuda.current_stream().synchronize()
                    assert all(torch.equal(a, b) for a, b in zip(got, want))
        except BaseException as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=run, args=(j, w)) for j, w in zip(jobs, alone)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """a cache whose last item starts behind 2^31 elements"""
    from samble_amd.attention import differential_attention
    B, Nk, d = 3, 70000, 64
    k = torch.empty((B, Nk, 64, 2, d), dtype=torch.bfloat16, device=DEV)      # 2^29 elements an item: 1.7e9 in all, with v 3.4e9 bytes each
    v = torch.empty((B, Nk, 64, 2 * d), dtype=torch.bfloat16, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(1)
    for t in (k, v):
        t[2, :, 63] = torch.randn(t[2, :, 63].shape, generator=gen, device=DEV).bfloat16()
        t[0, :, 0] = torch.randn(t[0, :, 0].shape, generator=gen, device=DEV).bfloat16()
    big = torch.as_strided(k, (2, Nk, 2, 2, d), (2 * k.stride(0), k.stride(1), 63 * k.stride(2), d, 1))
    bigv = torch.as_strided(v, (2, Nk, 2, 2 * d), (2 * v.stride(0), v.stride(1), 63 * v.stride(2), 1))
    big[0, :, 1], big[1, :, 0], bigv[0, :, 1], bigv[1, :, 0] = 0.5, 0.25, 1.0, 2.0
    q = torch.randn((2, 1, 2, 2, d), generator=gen, device=DEV).bfloat16()
    lam = torch.tensor([0.3, 0.6], device=DEV)
    out = differential_attention(q, big, bigv, lam)
    copy = differential_attention(q, big.contiguous(), bigv.contiguous(), lam)
    assert torch.equal(out, copy)
    _check(q, big.contiguous(), bigv.contiguous(), lam, None, (out,), d ** -0.5, False, None, None, None)


# ---- the layer ------------------------------------------------------------------------------------------------------------
def _layer_config(C, H, ff):
    from samble_amd.config import to_attr
    one = lambda v: [v]  # noqa: E731
    return to_attr(dict(q_in=one(C), q_out=one(C), k_in=one(C), k_out=one(C), v_in=one(C), v_out=one(C), num_heads=one(H),
                        ff_conv1_channels_in=one(C), ff_conv1_channels_out=one(ff), ff_conv2_channels_in=one(ff),
                        ff_conv2_channels_out=one(C)))


@pytest.mark.gpu
@pytest.mark.parametrize("C,H,ff,N", [(128, 4, 512, 257), (128, 1, 512, 100), (64, 2, 96, 65)])
def test_layer_against_float64(C, H, ff, N):
    """The whole layer, forward and every gradient, with ragged clouds.  Tolerance: the layer chains some ten fp32 stages of
    at most 512-term sums on values of order one; 512 U = 3e-5 per stage, taken against the largest value of each tensor."""
    from samble_amd.attention import DifferentialAttention
    torch.manual_seed(C + H)
    layer = DifferentialAttention(_layer_config(C, H, ff), 0).to(DEV)
    with torch.no_grad():
        for p in (layer.head_norm, layer.norm1, layer.norm2):
            p.weight.add_(0.1 * torch.randn_like(p.weight))
            p.bias.add_(0.1 * torch.randn_like(p.bias))
    B, d = 3, C // (2 * H)
    x = torch.randn(B, C, N, device=DEV, requires_grad=True)
    lengths = torch.tensor([N, N // 2, N - 1], dtype=torch.int32, device=DEV)
    g = torch.randn(B, C, N, device=DEV)
    y = layer(x, lengths=lengths)
    params = dict(layer.named_parameters())
    got = torch.autograd.grad(y, [x, *params.values()], g)

    w = {n: p.detach().double().requires_grad_(True) for n, p in params.items()}
    xd = x.detach().double().requires_grad_(True)

    def norm(t, name, dim):
        r = t.movedim(dim, -1)
        var, mean = torch.var_mean(r, -1, correction=0, keepdim=True)
        return ((r - mean) / torch.sqrt(var + 1e-5) * w[name + ".weight"] + w[name + ".bias"]).movedim(-1, dim)

    def conv(t, name):
        return torch.matmul(w[name + ".weight"][:, :, 0], t)

    q, k, v = (conv(xd, n).transpose(1, 2) for n in ("q_conv", "k_conv", "v_conv"))
    lam = (torch.exp((w["lambda_q1"] * w["lambda_k1"]).sum(-1)) - torch.exp((w["lambda_q2"] * w["lambda_k2"]).sum(-1)) + layer.lambda_init)
    ok = torch.arange(N, device=DEV) < lengths[:, None]
    q, k = (t.reshape(B, N, H, 2, d).permute(0, 2, 3, 1, 4) for t in (q, k))
    v = v.reshape(B, N, H, 2 * d).permute(0, 2, 1, 3)
    p = torch.softmax((torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(d)).masked_fill(~ok[:, None, None, None, :], -math.inf), -1)
    o = torch.matmul(p[:, :, 0] - lam[None, :, None, None] * p[:, :, 1], v).transpose(1, 2)       # (B, N, H, 2d)
    o = norm(o, "head_norm", -1) * (1 - layer.lambda_init)
    z = norm(xd + o.reshape(B, N, C).transpose(1, 2), "norm1", 1)
    ref = norm(z + conv(torch.nn.functional.leaky_relu(conv(z, "ff.0"), 0.2), "ff.2"), "norm2", 1)
    want = torch.autograd.grad(ref, [xd, *w.values()], g.double())
    for name, a, b in zip(["y", "x", *params], (y, *got), (ref, *want)):
        err = ((a.double() - b).abs().max() / b.abs().max()).item()
        assert err <= 10 * 512 * U, f"{name}: {err:.2e}"


def test_layer_refusals():
    from samble_amd.attention import DifferentialAttention
    for C, H in ((128, 3), (128, 16), (256, 1)):
        with pytest.raises(ValueError, match="DifferentialAttention"):
            DifferentialAttention(_layer_config(C, H, 64), 0)
    bad = _layer_config(128, 4, 512)
    bad["v_out"] = [64]
    with pytest.raises(ValueError, match="equal"):
        DifferentialAttention(bad, 0)
    layer = DifferentialAttention(_layer_config(128, 4, 512), 0)
    with pytest.raises(_lib.SambleError, match="GPU"):
        layer(torch.zeros(1, 128, 8))


def test_refusals():
    from samble_amd.attention import differential_attention
    q, k, v, lam = torch.zeros(2, 3, 4, 2, 16), torch.zeros(2, 5, 2, 2, 16), torch.zeros(2, 5, 2, 32), torch.zeros(4)
    good = dict(q=q, k=k, v=v, lam=lam)
    bad = [dict(q=q[0]), dict(k=k.half()), dict(v=v[:, :4]), dict(v=v[..., :16]), dict(k=k[:, :, :, :1]), dict(q=q[:, :, :3]),
           dict(q=q.double(), k=k.double(), v=v.double()), dict(lam=torch.zeros(3)), dict(lam=torch.zeros(4).half()),
           dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
           dict(lengths=torch.zeros(3, dtype=torch.int32)), dict(lengths=torch.zeros(2)), dict(lengths=[5, 5]),
           dict(q_start=torch.zeros(2, dtype=torch.int32)), dict(causal=True, q_start=torch.zeros(1, dtype=torch.int32)),
           dict(key_mask=torch.ones(2, 5)), dict(key_mask=torch.ones(2, 4, dtype=torch.bool)),
           dict(q=q[..., :12], k=k[..., :12], v=v[..., :24]), dict(q=q[..., :0], k=k[..., :0], v=v[..., :0]),
           dict(q=torch.zeros(1, 1, 1, 2, 72), k=torch.zeros(1, 1, 1, 2, 72), v=torch.zeros(1, 1, 1, 144), lam=torch.zeros(1)),
           dict(q=torch.zeros(1, 1, 1, 2, 136).half(), k=torch.zeros(1, 1, 1, 2, 136).half(), v=torch.zeros(1, 1, 1, 272).half(),
                lam=torch.zeros(1))]
    for change in bad:
        with pytest.raises(ValueError, match="differential_attention"):
            differential_attention(**{**good, **change})
    with pytest.raises(_lib.SambleError, match="GPU"):
        differential_attention(**good)


def test_c_entries_refuse_bad_arguments():
    import ctypes
    ok = dict(type=2, lt=2, q=256, k=256, v=256, lam=256, shape=(1, 2, 3, 4, 2, 16),
              st=(256, 128, 32, 16, 192, 64, 32, 16, 192, 64, 32, 0, 256, 128, 32), len=None, qs=None, km=None, causal=0, scale=0.25)

    def call(name, tail, **change):
        a = {**ok, **change}
        args = [(ctypes.c_int64 * len(x))(*x) if isinstance(x, tuple) else x for x in a.values()]
        _lib.call(name, *args, *tail)

    fwd_tail = (256, None, None, None, 0, None)
    bwd_tail = (256, 256, 256, 256, 256, 256, 256, 256, 256, 1 << 20, None)
    bad = [dict(type=4), dict(type=2, lt=1), dict(q=None), dict(k=8), dict(v=257), dict(lam=None), dict(lam=257),
           dict(shape=(0, 2, 3, 4, 2, 16)), dict(shape=(1, 2, 3, 4, 3, 16)), dict(shape=(1, 2, 3, 4, 2, 12)),
           dict(shape=(1, 2, 3, 4, 2, 136)), dict(type=0, lt=0, shape=(1, 2, 3, 4, 2, 72)), dict(shape=(1, 2, 1 << 31, 4, 2, 16)),
           dict(st=(256, 129) + ok["st"][2:]), dict(st=(-256,) + ok["st"][1:]), dict(scale=0.0), dict(scale=float("nan")), dict(qs=256)]
    for change in bad:
        for name, tail in (("samble_diff_attn_fwd", fwd_tail), ("samble_diff_attn_bwd", bwd_tail)):
            with pytest.raises(_lib.SambleError, match=name):
                call(name, tail, **change)
    # more workgroups than a launch holds: refused before anything is launched
    with pytest.raises(_lib.SambleError, match="more rows and heads"):
        call("samble_diff_attn_fwd", fwd_tail, shape=(1 << 24, 1, 1, 4, 4, 16))
    for shape in ((1 << 24, 1, 1, 4, 4, 16), (2, 1, 1 << 30, 1, 1, 8)):
        with pytest.raises(_lib.SambleError, match="more rows and heads"):
            call("samble_diff_attn_bwd", bwd_tail[:-2] + (1 << 40, None), shape=shape)
    with pytest.raises(_lib.SambleError, match="out2 with lse"):
        call("samble_diff_attn_fwd", (256, 256, None, None, 0, None))
    with pytest.raises(_lib.SambleError, match="workspace"):
        call("samble_diff_attn_bwd", bwd_tail[:-2] + (8, None))
    with pytest.raises(_lib.SambleError, match="workspace"):
        call("samble_diff_attn_fwd", fwd_tail, shape=(1, 1, 60000, 4, 2, 16))
    assert _lib.query("samble_diff_attn_fwd_workspace_bytes", 2, (ctypes.c_int64 * 6)(1, 1, 60000, 4, 2, 16)) > 0
    assert _lib.query("samble_diff_attn_fwd_workspace_bytes", 2, None) == 0


@pytest.mark.gpu
def test_forward_mode_is_refused():
    """A tangent is not dropped without a word."""
    from torch.autograd import forward_ad

    from samble_amd.attention import differential_attention
    args = list(_inputs(1, 5, 9, 2, 1, 16, torch.float32, 3)[:4])
    with forward_ad.dual_level():
        plain = differential_attention(*args)
        for n in range(4):
            dual = forward_ad.make_dual(args[n], torch.ones_like(args[n]))
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(RuntimeError):
                    differential_attention(*args[:n], dual, *args[n + 1:])
    assert torch.equal(plain, differential_attention(*args))


def _layer_and_input(C, H, ff, N):
    from samble_amd.attention import DifferentialAttention
    torch.manual_seed(C + H + ff)
    layer = DifferentialAttention(_layer_config(C, H, ff), 0).to(DEV)
    return layer, torch.randn(2, C, N, device=DEV), torch.randn(2, C, N, device=DEV)


def _layer_step(layer, x, g):
    x = x.detach().requires_grad_(True)
    y = layer(x)
    grads = torch.autograd.grad(y.float(), [x, *layer.parameters()], g)
    return [y.detach(), *grads]


LAYERS = [(64, 2, 96, 65), (128, 4, 96, 70), (128, 4, 512, 100), (128, 1, 512, 33)]


def _layer_tolerance(dtype, gradient):
    """Relative to the norm of each tensor.  On the way from the input to the loss and back a value passes at most 16 roundings to
    the 16-bit type (input, weight and result of four products in a row, and the same of their gradients, half of them on either
    way), each of eps / 2, and the result's own; softmax and the three norms pass on up to twice that.  A gradient also jumps where
    a rounding moves a hidden value over the kink of the LeakyReLU (slopes 1 and 0.2).  For normal values with an error of r times
    their norm, r <= 8 eps (the 16 on the way there), signs differ with probability arctan(r) / pi <= r / pi; such an entry is off by 0.8
    beside a slope of sqrt((1 + 0.04) / 2) = 0.72 in the mean square: 1.11 sqrt(r / pi) of the norm."""
    eps = torch.finfo(dtype).eps
    return (2 * 16 + 1) * eps / 2 + (1.11 * math.sqrt(8 * eps / math.pi) if gradient else 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("C,H,ff,N", LAYERS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_layer_under_autocast(C, H, ff, N, dtype):
    """Every width that the constructor takes."""
    layer, x, g = _layer_and_input(C, H, ff, N)
    ref = _layer_step(layer, x, g)
    with torch.autocast("cuda", dtype=dtype):
        got = _layer_step(layer, x, g)
    for name, a, b in zip(["y", "x", *dict(layer.named_parameters())], got, ref):
        assert bool(torch.isfinite(a).all()), name
        err = ((a.double() - b.double()).norm() / b.double().norm()).item()
        assert err <= _layer_tolerance(dtype, name != "y"), f"{name}: {err:.2e}"


@pytest.mark.gpu
@pytest.mark.parametrize("C,H,ff,N", LAYERS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_layer_in_sixteen_bits(C, H, ff, N, dtype):
    """Parameters and tensors of a 16-bit type, against the same values in fp32."""
    layer, x, g = _layer_and_input(C, H, ff, N)
    layer = layer.to(dtype)
    x = x.to(dtype)
    got = _layer_step(layer, x, g)
    assert all(t.dtype == dtype for t in got)
    ref = _layer_step(layer.float(), x.float(), g)
    for name, a, b in zip(["y", "x", *dict(layer.named_parameters())], got, ref):
        assert bool(torch.isfinite(a).all()), name
        err = ((a.double() - b.double()).norm() / b.double().norm()).item()
        assert err <= _layer_tolerance(dtype, name != "y"), f"{name}: {err:.2e}"


# ---- ranges ---------------------------------------------------------------------------------------------------------------
def _exact(q, k, v, lam, g, causal=False):
    """float64 out, dq, dk, dv, dlam of the formulas (no key masks; causal: the queries are the last positions)"""
    leaves = [t.detach().double().requires_grad_(True) for t in (q, k, v, lam)]
    B, Nq, H, _, d = q.shape
    Nk, Hkv = k.shape[1:3]
    qq, kk, vv, lm = leaves
    kk, vv = kk.repeat_interleave(H // Hkv, 2), vv.repeat_interleave(H // Hkv, 2)
    s = torch.matmul(qq.permute(0, 2, 3, 1, 4), kk.permute(0, 2, 3, 4, 1).contiguous()) / math.sqrt(d)
    if causal:
        s = s.masked_fill(~_visible(B, Nq, Nk, True, None, None, None, DEV)[:, None, None], -math.inf)
    p = torch.softmax(s, -1)
    out = torch.matmul(p[:, :, 0] - lm[None, :, None, None] * p[:, :, 1], vv.transpose(1, 2)).transpose(1, 2)
    return (out.detach(), *torch.autograd.grad(out, leaves, g.double()))


def _step(q, k, v, lam, g, **kw):
    from samble_amd.attention import differential_attention
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, lam)]
    out = differential_attention(*leaves, **kw)
    return (out.detach(), *torch.autograd.grad(out, leaves, g))


FP32 = [(2, 70, 130, 4, 2, 16), (1, 150, 333, 2, 2, 32), (1, 65, 200, 2, 1, 64), (2, 1, 1500, 4, 2, 64), (1, 300, 40, 2, 2, 24)]


@pytest.mark.gpu
@pytest.mark.parametrize("case", FP32, ids=lambda c: "-".join(map(str, c)))
def test_fp32_columns_and_keys_of_different_magnitude(case):
    """Columns of v from 2^-40 to 2^40, channels of q and k whose product alone is of order one, keys of v from 2^-20 to 2^20:
    the bound of each element is a few roundings of the magnitudes that the formula itself adds up for it."""
    q, k, v, lam, g, gen = _inputs(*case, torch.float32, 5)
    B, Nq, Nk, H, Hkv, d = case
    power = lambda n, most: torch.exp2(torch.randint(-most, most + 1, (n,), generator=gen, device=DEV).float())  # noqa: E731
    c = power(d, 30)
    q, k = q * c, k / c
    for scaled in (v * power(2 * d, 40), v * power(Nk, 20)[:, None, None]):
        _check(q, k, scaled, lam, g, _step(q, k, scaled, lam, g), d ** -0.5, False, None, None, None)


@pytest.mark.gpu
@pytest.mark.parametrize("case", FP32, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("dtype", list(TYPES))
def test_an_infinity_in_a_visible_value_stays_in_its_column(case, dtype):
    from samble_amd.attention import differential_attention
    q, k, v, lam, _, _ = _inputs(*case, TYPES[dtype], 7)
    plain = differential_attention(q, k, v, lam)
    for bad in (math.inf, -math.inf, math.nan):
        other = v.clone()
        other[0, 3, 0, 5] = bad
        out = differential_attention(q, k, other, lam)
        hit = torch.zeros_like(out, dtype=torch.bool)
        hit[0, :, : case[3] // case[4], 5] = True
        assert torch.equal(out[~hit], plain[~hit]) and not torch.isfinite(out[hit]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("case", FP32, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("exponent", [-100, -80, -60, 60, 80])
def test_fp32_gradients_of_any_size(case, exponent):
    """The gradients are linear in dout, and dq, dk and dlam in v: times a power of two they are the same numbers, as far as
    neither side leaves fp32's range (sums of 2^-24 steps of the largest term, which is far from either end)."""
    q, k, v, lam, g, _ = _inputs(*case, torch.float32, 9)
    one = _step(q, k, v, lam, g)
    for scaled, powers in ((_step(q, k, v, lam, g * 2.0 ** exponent), (0, exponent, exponent, exponent, exponent)),
                           (_step(q, k, v * 2.0 ** exponent, lam, g), (exponent, exponent, exponent, 0, exponent))):
        for name, a, b, e in zip(("out", "dq", "dk", "dv", "dlam"), one, scaled, powers):
            assert bool(torch.isfinite(b).all()), name
            err = (b.double() * 2.0 ** -e - a.double()).norm() / a.double().norm()
            assert err.item() <= 64 * U, f"{name}: {err.item():.2e}"


@pytest.mark.gpu
@pytest.mark.parametrize("small", [2.0 ** -86, 2.0 ** -30])
@pytest.mark.parametrize("causal", [False, True])
def test_fp32_rows_of_small_gradient_before_ordinary_ones(small, causal):
    q, k, v, lam, g, _ = _inputs(1, 400, 400, 2, 2, 32, torch.float32, 13)
    g[:, :128] *= small
    got = _step(q, k, v, lam, g, causal=causal)
    _check(q, k, v, lam, g, got, 32 ** -0.5, causal, None, None, None)
    alone = _step(q, k, v, lam, g[:, :128].repeat(1, 4, 1, 1)[:, :400], causal=causal)
    assert torch.equal(alone[1][:, :128], got[1][:, :128])


@pytest.mark.gpu
@pytest.mark.parametrize("size", [2.0 ** -13, 2.0 ** -10, 1.0, 2.0 ** 10])
@pytest.mark.parametrize("case", [(1, 600, 1000, 8, 1, 16), (2, 500, 700, 4, 2, 32), (1, 257, 900, 8, 2, 64), (1, 200, 2000, 4, 1, 128),
                                  (1, 40, 4000, 2, 2, 64)], ids=lambda c: "-".join(map(str, c)))
def test_fp16_gradients_of_any_size(case, size):
    """dS of a thousand keys is a thousandth of a gradient: as an operand of the type it is held where it has all its bits.
    Bound, against the norm of each gradient in float64: P and dS rounded once each, t from outputs that were rounded once, each
    2^-11 of the terms, whose norm is at most four times the result's (independent signs); the result's own rounding comes on top."""
    q, k, v, lam, g, _ = _inputs(*case, torch.float16, 4)
    g = (g.float() * size).half()
    want = _exact(q, k, v, lam, g)
    for name, a, b in zip(("dq", "dk", "dv", "dlam"), _step(q, k, v, lam, g)[1:], want[1:]):
        assert bool(torch.isfinite(a).all()), name
        own = (b.to(a.dtype).double() - b).norm()
        err = (a.double() - b).norm()
        assert err <= own + 3 * 4 * 2.0 ** -11 * b.norm(), f"{name}: {(err / b.norm()).item():.2e}, rounding alone {(own / b.norm()).item():.2e}"


@pytest.mark.gpu
@pytest.mark.parametrize("lam_value", [0.4, 300.0])
@pytest.mark.parametrize("d", [16, 64, 128])
def test_fp16_terms_beyond_the_type(d, lam_value):
    """Few keys and large gradients: P (dA - t) is beyond 65504, the gradients are not."""
    q, k, v, _, g, _ = _inputs(1, 90, 4, 2, 1, d, torch.float16, 6)
    k, v, g = (0.02 * k.float()).half(), (16 * v.float() / math.sqrt(d / 16)).half(), (4000 * g.float() / max(1.0, lam_value)).half()
    q = (0.02 * q.float()).half()
    lam = torch.full((2,), lam_value, device=DEV)
    want = _exact(q, k, v, lam, g)
    got = _step(q, k, v, lam, g)
    for name, a, b in zip(("out", "dq", "dk"), got, want):
        assert bool(torch.isfinite(a).all()) and float(b.abs().max()) < 60000, name
        err = ((a.double() - b).norm() / b.norm()).item()
        assert err <= 4 * 4 * 2.0 ** -11, f"{name}: {err:.2e}"


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0.0, 64.0])
@pytest.mark.parametrize("case", [(2, 1, 40, 4, 2, 16), (1, 150, 90, 2, 2, 32), (1, 200, 300, 4, 1, 64), (2, 3, 2100, 4, 2, 64),
                                  (1, 70, 130, 2, 1, 128), (1, 2, 3000, 1, 1, 128), (1, 60, 50, 2, 2, 24)],
                         ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_dq_is_not_that_of_rounded_outputs(dtype, case, offset):
    """Keys and values with a large common part: dq is a difference of terms far larger than itself, and a row sum t from outputs
    that were rounded to 16 bits would be off in all of them alike.  Bound of an element, h = eps / 2: half a step of it, dS
    rounded once, P relative (see above), and t off by 2^-7 h of the magnitudes that it sums over (a byte beside each saved value),
    by h of how far the values stand from the output (P is rounded once in the forward's sums and in their divisor alike) and by
    fp32 sums over 2 d columns."""
    B, Nq, Nk, H, Hkv, d = case
    q, k, v, lam, g, _ = _inputs(*case, TYPES[dtype], 4)
    k, v = (1.5 + 0.2 * k.float()).to(k.dtype), (offset + v.float()).to(v.dtype)
    got = _step(q, k, v, lam, g)[1].double()
    h = torch.finfo(TYPES[dtype]).eps / 2
    sub = 2.0 ** -25 if dtype == "fp16" else 0.0
    scale = d ** -0.5
    for b in range(B):
        for hq in range(H):
            kk, vv, gg, lm = k[b, :, hq // (H // Hkv)].double(), v[b, :, hq // (H // Hkv)].double(), g[b, :, hq].double(), float(lam[hq])
            dA, adA = gg @ vv.T, gg.abs() @ vv.abs().T
            P = [torch.softmax(q[b, :, hq, m].double() @ kk[:, m].T * scale, -1) for m in range(2)]
            t2 = (P[1] * dA).sum(-1, keepdim=True)
            t1 = (P[0] * dA).sum(-1, keepdim=True)
            o = [p @ vv for p in P]
            et2 = (gg.abs() * (2.0 ** -7 * h + (2 * d + 32) * U) * o[1].abs()).sum(-1, keepdim=True)
            et1 = (gg.abs() * (2.0 ** -7 * h + (2 * d + 32) * U) * (o[0] - lm * o[1]).abs()).sum(-1, keepdim=True) + lm * et2
            for m, (t, et, sign) in enumerate(((t1, et1, 1.0), (t2, et2, -lm))):
                L = (q[b, :, hq, m].double().abs() @ kk[:, m].abs().T * scale).amax(-1, keepdim=True)
                dP = 2 * ((d + 32) * U * L + 16 * U) + Nk * U
                spread = (P[m] * (gg.abs().T[:, :, None] * (vv.T[:, None] - o[m].T[:, :, None]).abs()).sum(0)).sum(-1, keepdim=True)
                dS = sign * P[m] * (dA - t)
                edS = abs(sign) * P[m] * (et + h * spread + (2 * d + 32) * U * adA + (dP + 4 * U) * (dA - t).abs()) + h * dS.abs()
                ref = scale * dS @ kk[:, m]
                tol = scale * (edS + Nk * U * dS.abs()) @ kk[:, m].abs() * (1 + 1e-3) + h * ref.abs() + sub
                err = (got[b, :, hq, m] - ref).abs()
                assert bool((err <= tol).all()), f"b{b} h{hq} m{m}: {(err - tol).max():.3e} over, error {err.max():.3e}"


@pytest.mark.gpu
@pytest.mark.parametrize("size", [2.0 ** -13, 2.0 ** -18, 2.0 ** -21])
@pytest.mark.parametrize("case", [(2, 150, 90, 2, 2, 32), (1, 200, 300, 4, 1, 64), (2, 3, 2100, 4, 2, 64), (1, 70, 130, 2, 1, 128)],
                         ids=lambda c: "-".join(map(str, c)))
def test_fp16_outputs_below_the_types_normal_numbers(case, size):
    """Values of few steps of 2^-24: the outputs stand among fp16's last steps, but dS, dq and dk do not (gradients of 2^12).  Bound against the norm of each gradient in float64, as above: dS and what t is made of rounded once each."""
    q, k, v, lam, g, _ = _inputs(*case, torch.float16, 8)
    v, g = (v.float() * size).half(), (4096 * g.float()).half()
    want = _exact(q, k, v, lam, g)
    for name, a, b in zip(("dq", "dk", "dv", "dlam"), _step(q, k, v, lam, g)[1:], want[1:]):
        own, err = (b.to(a.dtype).double() - b).norm(), (a.double() - b).norm()
        assert err <= own + 2 * 2.0 ** -11 * b.norm(), f"{name}: {(err / b.norm()).item():.2e}, rounding alone {(own / b.norm()).item():.2e}"


def test_the_rest_of_the_outputs_is_refused_where_there_is_none():
    import ctypes

    from samble_amd import ops
    shape, st = (ctypes.c_int64 * 6)(1, 2, 3, 4, 2, 16), (ctypes.c_int64 * 15)(256, 128, 32, 16, 192, 64, 32, 16, 192, 64, 32, 0, 256, 128, 32)

    def fwd(kind, out2, rest):
        _lib.call("samble_diff_attn_fwd_rest", kind, kind, 256, 256, 256, 256, shape, st, None, None, None, 0, 0.25, 256, out2, out2,
                  rest, None, 0, None)

    def bwd(kind, rest):
        _lib.call("samble_diff_attn_bwd_rest", kind, kind, 256, 256, 256, 256, shape, st, None, None, None, 0, 0.25, 256, 256, 256, rest,
                  256, 256, 256, 256, 256, 256, 1 << 20, None)

    for call in (lambda: fwd(0, 256, 256), lambda: fwd(1, 256, 264), lambda: fwd(2, None, 256), lambda: bwd(0, 256), lambda: bwd(2, 260)):
        with pytest.raises(_lib.SambleError, match="rest"):
            call()
    q = torch.zeros(1, 2, 4, 2, 16, dtype=torch.float16)
    good = torch.zeros(1, 2, 4, 32, 2, dtype=torch.int8)
    ops._rest_shape(q, good)
    ops._rest_shape(q, None)
    for bad in (good.float(), good[..., :1], good.transpose(1, 2), torch.zeros(1, 2, 4, 32, 4, dtype=torch.int8)[..., ::2]):
        with pytest.raises(ValueError, match="rest"):
            ops._rest_shape(q, bad)


@pytest.mark.gpu
@pytest.mark.parametrize("case", [(2, 150, 150, 4, 2, 64), (1, 1500, 130, 2, 1, 32), (2, 2, 2100, 4, 2, 48)], ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("dtype", list(TYPES))
def test_training_step_replayed(case, dtype):
    """Gradients of other sizes at each replay (scales are made anew), the first call of its kind captured where it is the first."""
    q, k, v, lam, g, gen = _inputs(*case, TYPES[dtype], 12)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = _step(q, k, v, lam, g, causal=True)
    for size in (1.0, 2.0 ** -9, 2.0 ** 7, 1.0):
        q.copy_(torch.randn(q.shape, generator=gen, device=DEV))
        g.copy_(size * torch.randn(g.shape, generator=gen, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        eager = _step(q, k, v, lam, g, causal=True)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, held)), size
