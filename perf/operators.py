"""Timed cases of the attention layers' dense operators: differential attention and layer normalisation.

Differential attention (H query heads, Hkv key / value heads, H a multiple of Hkv; per head two maps m = 1, 2 of depth d and
values of depth 2 d, and a learned weight lam per query head):

    P_m = softmax_j(scale <q_m_i, k_m_j>) over the keys that row i may see,   out_i = sum_j (P_1 - lam P_2)_ij v_j

a row that may see no key gives zeros.  Layer normalisation of x (+ residual) over one axis of C channels:

    s = x + residual,  y = (s - mean) / sqrt(var + eps) * weight + bias

`run` computes both either as plain torch expressions in float32 (`own` False) or through this package (`own` True); a
"train" case is the forward pass and the gradients of every input for a given output gradient.
"""
import math

import torch

own = False

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
EPS = 1e-5


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def _attn(name, dtype, mode, batch, heads, kv_heads, depth, queries, keys, mask="none", causal=False):
    return dict(name=name, op="attention", dtype=dtype, mode=mode, batch=batch, heads=heads, kv_heads=kv_heads, depth=depth,
                queries=queries, keys=keys, mask=mask, causal=causal)


def _norm(name, dtype, mode, outer, channels, inner, residual=False, weight_dtype="float32"):
    return dict(name=name, op="norm", dtype=dtype, mode=mode, outer=outer, channels=channels, inner=inner, residual=residual,
                weight_dtype=weight_dtype)


def listed():
    return [
        # one query token against the points of a very small cloud: latency alone
        _attn("attn_one_token_small", "float32", "forward", 1, 4, 4, 16, 1, 33),
        # the attention layer over the 1024 sampled points of 32 clouds, 128 channels in four heads, as it is trained
        _attn("attn_layer_train_fp32", "float32", "train", 32, 4, 4, 16, 1024, 1024),
        # 128 channels in one head, ragged clouds padded to one length, inference
        _attn("attn_padded_clouds_fp32", "float32", "forward", 8, 1, 1, 64, 1999, 1999, mask="lengths"),
        # a long prompt, four query heads on each key head, an odd length
        _attn("attn_prompt_bf16", "bfloat16", "forward", 2, 16, 4, 64, 4001, 4001, causal=True),
        # a training step of the same kind of model
        _attn("attn_causal_train_bf16", "bfloat16", "train", 2, 16, 4, 64, 2048, 2048, causal=True),
        # cross attention of 500 queries to 777 points, holes in the points (a key mask), trained in half precision
        _attn("attn_cross_train_fp16", "float16", "train", 8, 8, 8, 32, 500, 777, mask="keys"),
        # one new token for each of 16 sequences, caches of different lengths
        _attn("attn_one_token_batch_bf16", "bfloat16", "forward", 16, 32, 8, 64, 1, 8192, mask="lengths"),
        # one new token of one sequence with a long cache, wide heads
        _attn("attn_one_token_long_bf16", "bfloat16", "forward", 1, 16, 4, 128, 1, 65536),
        # a handful of rows: latency alone
        _norm("norm_few_rows", "float32", "forward", 7, 128, 1),
        # a prompt's rows in inference
        _norm("norm_rows_bf16", "bfloat16", "forward", 8192, 4096, 1),
        # (B, C, N) as this package's layers hold their tensors, the norm behind a residual add, trained
        _norm("norm_channels_train_fp32", "float32", "train", 32, 128, 2048, residual=True),
        # an odd width and an odd number of rows, weights in the activations' type, trained
        _norm("norm_odd_train_fp16", "float16", "train", 4099, 5001, 1, residual=True, weight_dtype="float16"),
    ]


# bounds of a drawn case, those of the listed ones: (query row, key) pairs over all heads (a plain map is 4 bytes a pair),
# operations and bytes of one pass
MAX_PAIRS, MAX_ATTN_FLOPS, MAX_ATTN_BYTES, MAX_NORM_BYTES = 1 << 28, 1.2e11, 3.5e8, 2.0e8


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    if rng.random() < 0.62:
        while True:
            mode = rng.choice(["token", "forward", "train"])
            dtype = rng.choice(["float32", "float16", "bfloat16"])
            depth = rng.choice([8, 16, 24, 32, 40, 64] + ([] if dtype == "float32" else [96, 128]))
            kv_heads = rng.choice([1, 2, 3, 4, 8])
            heads = kv_heads * rng.choice([1, 1, 2, 4, 5])
            batch = _log_int(rng, 1, 16)
            mask = rng.choice(["none", "lengths", "keys"])
            if mode == "token":
                queries, keys = rng.choice([1, 1, 1, 2, 5]), _log_int(rng, 1, 65536)
                causal = queries > 1
            else:
                keys = _log_int(rng, 16, 4096)
                queries = keys if rng.random() < 0.6 else _log_int(rng, 16, 4096)
                causal = rng.random() < 0.5
            case = _attn("", dtype, "train" if mode == "train" else "forward", batch, heads, kv_heads, depth, queries, keys,
                         mask, causal)
            cost = work(case)
            if (batch * heads * queries * keys <= MAX_PAIRS and cost["flops"] <= MAX_ATTN_FLOPS
                    and cost["bytes"] <= MAX_ATTN_BYTES):
                break
    else:
        while True:
            inner = 1 if rng.random() < 0.6 else _log_int(rng, 2, 4096)
            outer = _log_int(rng, 1, 8192 if inner == 1 else 64)
            channels = _log_int(rng, 8, 8192 if inner == 1 else 1024)
            dtype = rng.choice(["float32", "float16", "bfloat16"])
            case = _norm("", dtype, rng.choice(["forward", "train"]), outer, channels, inner, rng.random() < 0.5,
                         rng.choice(["float32", dtype]))
            if work(case)["bytes"] <= MAX_NORM_BYTES:
                break
    del case["name"]
    return case


def _lengths(case):
    """Key counts of the batch: from all keys down to three tenths of them (their order is the seed's)."""
    B, N = case["batch"], case["keys"]
    if case["mask"] != "lengths":
        return [N] * B
    return [N - int(0.7 * N * b / B) for b in range(B)]


def _starts(case, lengths):
    """Position of a batch item's first query: with lengths, the queries are the last of its keys."""
    return [max(0, n - case["queries"]) for n in lengths] if case["mask"] == "lengths" \
        else [case["keys"] - case["queries"]] * case["batch"]


def _pairs(case):
    """(row, visible key) pairs of one head over the batch."""
    total = 0
    lengths = _lengths(case)
    for n, start in zip(lengths, _starts(case, lengths)):
        if not case["causal"]:
            total += case["queries"] * n
            continue
        first, last = start + 1, start + case["queries"]        # keys seen by the first and the last row, before clipping
        rising = range(max(first, 1), min(last, n) + 1)
        total += (rising[0] + rising[-1]) * len(rising) // 2 if len(rising) else 0
        total += max(0, last - max(n, first - 1)) * n
    return total


def work(case):
    size = torch.empty((), dtype=TYPES[case["dtype"]]).element_size()
    if case["op"] == "norm":
        n = case["outer"] * case["channels"] * case["inner"]
        wsize = torch.empty((), dtype=TYPES[case["weight_dtype"]]).element_size()
        tensors = 2 + (1 if case["residual"] else 0)            # x (residual) y
        flops = 8
        if case["mode"] == "train":
            tensors += 2                                        # dy, dx (the residual's gradient is the same tensor)
            flops += 14
        passes = 4 if case["mode"] == "train" else 2
        return {"bytes": tensors * n * size + passes * case["channels"] * wsize, "flops": flops * n}
    d, H, Hkv, B, Nq = case["depth"], case["heads"], case["kv_heads"], case["batch"], case["queries"]
    q_bytes, kv_rows = B * Nq * H * 2 * d * size, sum(_lengths(case)) * Hkv
    fwd = 2 * q_bytes + kv_rows * 4 * d * size                  # q, k, v in, out
    flops = 8 * d * _pairs(case) * H
    if case["mode"] == "train":
        fwd += 2 * q_bytes + B * case["keys"] * Hkv * 4 * d * size   # d out in, dq, dk, dv out
        flops += 20 * d * _pairs(case) * H
    return {"bytes": fwd, "flops": flops}


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    dt = TYPES[case["dtype"]]
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    host = torch.Generator()
    host.manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=gen, device=dev)  # noqa: E731
    train = case["mode"] == "train"
    state = {"case": case}
    if case["op"] == "norm":
        B, C, N = case["outer"], case["channels"], case["inner"]
        shape = (B, C) if N == 1 else (B, C, N)
        wt = TYPES[case["weight_dtype"]]
        # channels of different offset and spread, as activations have
        spread = (0.5 + torch.rand(C, generator=gen, device=dev)).reshape((1, C) + (1,) * (len(shape) - 2))
        state["x"] = (normal(*shape) * spread + 0.3 * normal(*spread.shape)).to(dt)
        state["weight"] = (1.0 + 0.2 * normal(C)).to(wt)
        state["bias"] = (0.2 * normal(C)).to(wt)
        state["residual"] = normal(*shape).to(dt) if case["residual"] else None
        if train:
            state["grad"] = normal(*shape).to(dt)
            for key in ("x", "weight", "bias", "residual"):
                if state[key] is not None:
                    state[key].requires_grad_(True)
        return state
    B, H, Hkv, d, Nq, Nk = (case[k] for k in ("batch", "heads", "kv_heads", "depth", "queries", "keys"))
    # points and tokens share components: logits with a spread of about two, some rows nearly one-hot
    state["q"] = (1.4 * normal(B, Nq, H, 2, d)).to(dt)
    state["k"] = (1.4 * normal(B, Nk, Hkv, 2, d)).to(dt)
    state["v"] = normal(B, Nk, Hkv, 2 * d).to(dt)
    state["lam"] = (0.2 + 0.6 * torch.rand(H, generator=gen, device=dev)).to(dt)
    lengths = _lengths(case)
    starts = _starts(case, lengths)
    order = torch.randperm(B, generator=host)
    state["lengths"] = state["q_start"] = state["key_mask"] = None
    if case["mask"] == "lengths":
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32)[order].to(dev)
        if case["causal"]:
            state["q_start"] = torch.tensor(starts, dtype=torch.int32)[order].to(dev)
    elif case["mask"] == "keys":
        state["key_mask"] = torch.rand((B, Nk), generator=gen, device=dev) > 0.15
    if train:
        state["grad"] = normal(B, Nq, H, 2 * d).to(dt)
        for key in ("q", "k", "v", "lam"):
            state[key].requires_grad_(True)
    return state


def _visible(state):
    """(B, 1, Nq, 1, Nk) truth values, or None where every row sees every key."""
    case = state["case"]
    B, Nq, Nk = case["batch"], case["queries"], case["keys"]
    dev = state["q"].device
    if case["mask"] == "none" and not case["causal"]:
        return None
    j = torch.arange(Nk, device=dev)
    ok = torch.ones((B, 1, Nk), dtype=torch.bool, device=dev)
    if state["lengths"] is not None:
        ok = ok & (j < state["lengths"][:, None, None])
    if state["key_mask"] is not None:
        ok = ok & state["key_mask"][:, None, :]
    if case["causal"]:
        i = torch.arange(Nq, device=dev)[None, :, None]
        start = Nk - Nq if state["q_start"] is None else state["q_start"][:, None, None]
        ok = ok & (j <= i + start)
    return ok[:, None, :, None, :]


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    if state["case"]["op"] == "norm":
        return _run_norm_own(state) if own else _run_norm_plain(state)
    return _run_attn_own(state) if own else _run_attn_plain(state)


def _run_norm_own(state):
    from samble_amd.norm import layer_norm
    train = state["case"]["mode"] == "train"
    res = state["residual"]
    with torch.set_grad_enabled(train):
        y = layer_norm(state["x"], state["weight"], state["bias"], EPS, dim=1, residual=res)
        if res is not None:
            y, s = y
    if not train:
        return y if res is None else (y, s)
    leaves = [state["x"], state["weight"], state["bias"]]
    dx, dw, db = torch.autograd.grad(y, leaves, state["grad"])
    return (y, dx, dw, db) if res is None else (y, s, dx, dw, db)


def _run_norm_plain(state):
    case = state["case"]
    with torch.no_grad():
        x = state["x"].float()
        dt, wt = state["x"].dtype, state["weight"].dtype
        bc = (1, -1) + (1,) * (x.dim() - 2)
        w, b = state["weight"].float().reshape(bc), state["bias"].float().reshape(bc)
        s = None
        if state["residual"] is not None:
            s = (x + state["residual"].float()).to(dt)
            x = s.float()
        mean = x.mean(1, keepdim=True)
        xc = x - mean
        rstd = 1.0 / torch.sqrt((xc * xc).mean(1, keepdim=True) + EPS)
        xhat = xc * rstd
        y = (xhat * w + b).to(dt)
        if case["mode"] != "train":
            return y if s is None else (y, s)
        dy = state["grad"].float()
        others = [i for i in range(x.dim()) if i != 1]
        db = dy.sum(others).to(wt)
        dw = (dy * xhat).sum(others).to(wt)
        g = dy * w
        dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
        dx = dx.to(dt)
    return (y, dx, dw, db) if s is None else (y, s, dx, dw, db)


def _run_attn_own(state):
    from samble_amd.attention import differential_attention
    train = state["case"]["mode"] == "train"
    with torch.set_grad_enabled(train):
        out = differential_attention(state["q"], state["k"], state["v"], state["lam"], causal=state["case"]["causal"],
                                     lengths=state["lengths"], q_start=state["q_start"], key_mask=state["key_mask"])
    if not train:
        return out
    return (out,) + torch.autograd.grad(out, [state["q"], state["k"], state["v"], state["lam"]], state["grad"])


def _run_attn_plain(state):
    case = state["case"]
    B, H, Hkv, d, Nq, Nk = (case[k] for k in ("batch", "heads", "kv_heads", "depth", "queries", "keys"))
    G = H // Hkv
    dt = state["q"].dtype
    with torch.no_grad():
        # the rows of the heads that share a key head stand together: (2, B Hkv, Nq G, d) against (2, B Hkv, Nk, d)
        q = state["q"].float().reshape(B, Nq, Hkv, G, 2, d).permute(4, 0, 2, 1, 3, 5).reshape(2, B * Hkv, Nq * G, d)
        k = state["k"].float().permute(3, 0, 2, 1, 4).reshape(2, B * Hkv, Nk, d)
        v = state["v"].float().permute(0, 2, 1, 3).reshape(B * Hkv, Nk, 2 * d)
        lam = state["lam"].float().reshape(1, Hkv, 1, G).expand(B, Hkv, Nq, G).reshape(B * Hkv, Nq * G, 1)
        ok = _visible(state)
        if ok is not None:
            ok = ok.expand(B, Hkv, Nq, G, Nk).reshape(B * Hkv, Nq * G, Nk)
        maps = []
        for m in range(2):
            logits = torch.matmul(q[m], k[m].transpose(1, 2).contiguous()) * (1.0 / math.sqrt(d))
            if ok is not None:
                logits = torch.where(ok, logits, -math.inf)
            top = logits.amax(-1, keepdim=True)
            top = torch.where(top == -math.inf, 0.0, top)
            p = torch.exp(logits - top)
            total = p.sum(-1, keepdim=True)
            maps.append(p / torch.where(total == 0, 1.0, total))
        p1, p2 = maps
        a = p1 - lam * p2

        def rows_out(t, width):   # (B Hkv, Nq G, width) -> (B, Nq, H, width)
            return t.reshape(B, Hkv, Nq, G, width).permute(0, 2, 1, 3, 4).reshape(B, Nq, H, width)

        out = rows_out(torch.matmul(a, v), 2 * d).to(dt)
        if case["mode"] != "train":
            return out
        g = state["grad"].float().reshape(B, Nq, Hkv, G, 2 * d).permute(0, 2, 1, 3, 4).reshape(B * Hkv, Nq * G, 2 * d)
        dv = torch.matmul(a.transpose(1, 2).contiguous(), g)
        da = torch.matmul(g, v.transpose(1, 2).contiguous())
        t1, t2 = (p1 * da).sum(-1, keepdim=True), (p2 * da).sum(-1, keepdim=True)
        dlam = -t2.reshape(B, Hkv, Nq, G).sum((0, 2)).reshape(H).to(dt)
        ds = (p1 * (da - t1) * (1.0 / math.sqrt(d)), -lam * p2 * (da - t2) * (1.0 / math.sqrt(d)))
        dq = torch.stack([rows_out(torch.matmul(ds[m], k[m]), d) for m in range(2)], 3).to(dt)
        dk = torch.stack([torch.matmul(ds[m].transpose(1, 2).contiguous(), q[m]).reshape(B, Hkv, Nk, d).permute(0, 2, 1, 3)
                          for m in range(2)], 3).to(dt)
        dv = dv.reshape(B, Hkv, Nk, 2 * d).permute(0, 2, 1, 3).contiguous().to(dt)
    return out, dq, dk, dv, dlam


# ------------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    return _exact_norm(state) if case["op"] == "norm" else _exact_attn(state)


def _exact_norm(state):
    case = state["case"]
    train = case["mode"] == "train"
    x = state["x"].detach()
    s = None
    if state["residual"] is not None:
        s = (x.double() + state["residual"].detach().double()).to(x.dtype)
    z = (x if s is None else s).double().requires_grad_(train)
    w = state["weight"].detach().double().requires_grad_(train)
    b = state["bias"].detach().double().requires_grad_(train)
    rows = z.movedim(1, -1)
    var, mean = torch.var_mean(rows, -1, correction=0, keepdim=True)
    y = ((rows - mean) * (var + EPS).rsqrt() * w + b).movedim(-1, 1)
    first = (y.detach(),) if s is None else (y.detach(), x.double() + state["residual"].detach().double())
    if not train:
        return first[0] if s is None else first
    return first + torch.autograd.grad(y, [z, w, b], state["grad"].double())


def _exact_attn(state):
    case = state["case"]
    train = case["mode"] == "train"
    H, Hkv, d, B = case["heads"], case["kv_heads"], case["depth"], case["batch"]
    leaves = {n: state[n].detach().double().requires_grad_(train) for n in ("q", "k", "v", "lam")}
    grads = {n: torch.zeros_like(t) for n, t in leaves.items()} if train else None
    ok = _visible(state)
    out = torch.zeros(state["q"].shape[:3] + (2 * d,), dtype=torch.float64, device=state["q"].device)
    # one head of one batch item at a time where the maps are large, all rows of a batch item together where they are small
    step = 1 if case["queries"] * case["keys"] > (1 << 18) else Hkv
    for b in range(B):
        for h0 in range(0, Hkv, step):
            kv = range(h0, min(Hkv, h0 + step))
            heads = [h for h in range(H) if h * Hkv // H in kv]
            shared = [h * Hkv // H for h in heads]
            part = [leaves["q"][b][:, heads], leaves["k"][b][:, list(kv)], leaves["v"][b][:, list(kv)], leaves["lam"][heads]]
            part = [t.detach().requires_grad_(train) for t in part]
            q, k, v, lam = part
            local = [s - h0 for s in shared]
            kk, vv = k[:, local], v[:, local]
            energy = torch.einsum("ihmd,jhmd->hmij", q, kk) / d ** 0.5
            if ok is not None:
                seen = ok[b if ok.shape[0] > 1 else 0, 0, :, 0, :]
                energy = energy.masked_fill(~seen, float("-inf"))
                some = seen.any(-1).expand(energy.shape[2])[:, None]
                weights = torch.softmax(energy.masked_fill(~some, 0.0), -1) * some
            else:
                weights = torch.softmax(energy, -1)
            o = torch.einsum("hij,jhe->ihe", weights[:, 0] - lam[:, None, None] * weights[:, 1], vv)
            out[b][:, heads] = o.detach()
            if train:
                gq, gk, gv, gl = torch.autograd.grad(o, part, state["grad"][b][:, heads].double())
                grads["q"][b][:, heads] += gq
                grads["k"][b][:, list(kv)] += gk
                grads["v"][b][:, list(kv)] += gv
                grads["lam"][heads] += gl
    return (out, grads["q"], grads["k"], grads["v"], grads["lam"]) if train else out
