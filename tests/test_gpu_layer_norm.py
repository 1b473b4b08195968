"""Layer normalisation (samble_amd.norm, csrc/layernorm.hip) against its formulas in float64.

Tolerances: one rounding to the output's type (half a step, eps / 2 of the value) plus the fp32 arithmetic.  A sum of n terms
in the kernels' order -- at most 32 values in a thread, ten levels of a tree, up to 64 wave partials -- is off by at most
n_add 2^-24 times the sum of magnitudes, n_add = 32 + 10 + 64; the loop kernels add C / 1024 (rows) or C (columns) values in
a thread instead.  A handful of products and the square root add some 16 roundings more."""
import pytest
import torch

from samble_amd import _lib

U = 2.0 ** -24
DEV = "cuda"


def _ref(x, w, b, eps, dim, dy=None, extra=None):
    """float64: y, magnitude of its terms [, dx, its magnitude, dw, sum |.|, db, sum |.|]"""
    x = x.double().movedim(dim, -1)
    C = x.shape[-1]
    w = torch.ones(C, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(C, dtype=torch.float64, device=x.device) if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    xc = x - mean
    rstd = 1.0 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + eps)
    xh = xc * rstd
    big = (x.abs() + x.abs().mean(-1, keepdim=True)) * rstd       # what xhat is a difference of
    out = [(xh * w + b).movedim(-1, dim), (big * w.abs() + b.abs()).movedim(-1, dim)]
    if dy is not None:
        dy = dy.double().movedim(dim, -1)
        g = dy * w
        m1, m2 = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
        dx = rstd * (g - m1 - xh * m2)
        a1, a2 = g.abs().mean(-1, keepdim=True), (g.abs() * (1 + big)).mean(-1, keepdim=True)
        mag = rstd * (g.abs() + a1 + (1 + big) * a2)
        if extra is not None:
            dx = dx + extra.double().movedim(dim, -1)
            mag = mag + extra.double().movedim(dim, -1).abs()
        rows = tuple(range(x.dim() - 1))
        out += [dx.movedim(-1, dim), mag.movedim(-1, dim), (dy * xh).sum(rows), (dy.abs() * (1 + big)).sum(rows), dy.sum(rows),
                dy.abs().sum(rows)]
    return out


def _close(got, ref, mag, n_add, what):
    tol = torch.finfo(got.dtype).eps / 2 * ref.abs() * (1 + 1e-3) + n_add * U * mag
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25          # half a subnormal step
    err = (got.double() - ref).abs()
    worst = (err - tol).max().item() if err.numel() else 0.0
    assert worst <= 0 and bool(torch.isfinite(got).all()), f"{what}: {worst:.3e} over the bound, worst error {err.max():.3e}"


def _n_add(C, dim_last):
    return 32 + 10 + 64 + 16 + (C // 1024 if dim_last else (C if C > 1024 else 0))


ROWS = [(1, 1), (3, 2), (7, 8), (5, 31), (9, 33), (33, 64), (130, 100), (67, 128), (41, 257), (17, 513), (13, 1000), (11, 1024),
        (9, 1537), (7, 2047), (5, 2049), (6, 3333), (9, 4096), (3, 5001), (4, 6145), (3, 8191), (3, 8200), (2, 16384),
        (2, 16385), (1, 40000), (1037, 24), (2100, 65)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("shape", ROWS, ids=lambda s: f"{s[0]}x{s[1]}")
def test_rows_forward_and_backward(shape, dtype):
    from samble_amd.norm import layer_norm
    R, C = shape
    gen = torch.Generator(device=DEV).manual_seed(R * 7919 + C)
    rnd = lambda *s: torch.randn(s, generator=gen, device=DEV)  # noqa: E731
    wt = torch.float32 if (R + C) % 2 else dtype
    x = (rnd(R, C) * 1.5 + 0.7).to(dtype).requires_grad_(True)
    w, b = (1 + 0.3 * rnd(C)).to(wt).requires_grad_(True), (0.3 * rnd(C)).to(wt).requires_grad_(True)
    dy = rnd(R, C).to(dtype)
    y = layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    ry, my, rdx, mdx, rdw, mdw, rdb, mdb = _ref(x.detach(), w.detach(), b.detach(), 1e-5, 1, dy)
    n = _n_add(C, True)
    _close(y.detach(), ry, my, n, "y")
    _close(dx, rdx, mdx, 2 * n, "dx")
    lines = n + R // 128 + 32 + 32
    _close(dw, rdw, mdw, lines, "dweight")
    _close(db, rdb, mdb, lines, "dbias")
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b), y)
    again = torch.autograd.grad(layer_norm(x, w, b), (x, w, b), dy)
    assert all(torch.equal(p, q) for p, q in zip(again, (dx, dw, db))), "not the same run to run"


LONG = [(70001, 24), (40003, 100), (9001, 300), (5003, 1500), (4099, 5001), (2501, 7777), (2101, 16000)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("shape", LONG, ids=lambda s: f"{s[0]}x{s[1]}")
def test_more_rows_than_the_workgroups_of_a_launch(shape, dtype):
    """Every workgroup walks several rows, the last ones not all of them; residual, and gradients that reach the sum too."""
    from samble_amd.norm import layer_norm
    R, C = shape
    gen = torch.Generator(device=DEV).manual_seed(R + C)
    rnd = lambda *s: torch.randn(s, generator=gen, device=DEV)  # noqa: E731
    x, res = (rnd(R, C) + 0.4).to(dtype).requires_grad_(True), rnd(R, C).to(dtype).requires_grad_(True)
    w, b = (1 + 0.3 * rnd(C)).requires_grad_(True), (0.3 * rnd(C)).requires_grad_(True)
    dy, ds = rnd(R, C).to(dtype), rnd(R, C).to(dtype)
    y, s = layer_norm(x, w, b, residual=res)
    assert torch.equal(s, (x.detach().float() + res.detach().float()).to(dtype))
    dx, dres, dw, db = torch.autograd.grad((y, s), (x, res, w, b), (dy, ds))
    ry, my, rdx, mdx, rdw, mdw, rdb, mdb = _ref(s.detach(), w.detach(), b.detach(), 1e-5, 1, dy, ds)
    n = _n_add(C, True)
    _close(y.detach(), ry, my, n, "y")
    _close(dx, rdx, mdx, 2 * n, "dx")
    assert torch.equal(dx, dres)
    lines = n + R // 128 + 32 + 32
    _close(dw, rdw, mdw, lines, "dweight")
    _close(db, rdb, mdb, lines, "dbias")


CHANNELS = [(1, 1, 2), (2, 8, 5), (3, 16, 64), (2, 17, 65), (2, 33, 127), (3, 64, 200), (2, 128, 2048), (2, 129, 130), (1, 256, 63),
            (2, 257, 66), (2, 512, 40), (1, 513, 33), (2, 1000, 31), (1, 1024, 129), (1, 1025, 50), (700, 20, 3), (3, 128, 1001)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("shape", CHANNELS, ids=lambda s: "x".join(map(str, s)))
def test_channels_with_residual_forward_and_backward(shape, dtype):
    from samble_amd.norm import layer_norm
    B, C, N = shape
    gen = torch.Generator(device=DEV).manual_seed(B * 7919 + C + 31 * N)
    rnd = lambda *s: torch.randn(s, generator=gen, device=DEV)  # noqa: E731
    wt = torch.float32 if (N + C) % 2 else dtype
    x = (rnd(B, C, N) + 0.4).to(dtype).requires_grad_(True)
    res = rnd(B, C, N).to(dtype).requires_grad_(True)
    w, b = (1 + 0.3 * rnd(C)).to(wt).requires_grad_(True), (0.3 * rnd(C)).to(wt).requires_grad_(True)
    dy, ds = rnd(B, C, N).to(dtype), rnd(B, C, N).to(dtype)
    y, s = layer_norm(x, w, b, dim=1, residual=res)
    assert torch.equal(s, (x.detach().float() + res.detach().float()).to(dtype))
    dx, dres, dw, db = torch.autograd.grad((y, s), (x, res, w, b), (dy, ds))
    ry, my, rdx, mdx, rdw, mdw, rdb, mdb = _ref(s.detach(), w.detach(), b.detach(), 1e-5, 1, dy, ds)
    n = _n_add(C, False)
    _close(y.detach(), ry, my, n, "y")
    _close(dx, rdx, mdx, 2 * n, "dx")
    assert torch.equal(dx, dres)
    lines = n + (B * N) // 128 + 8 + 32 + 32
    _close(dw, rdw, mdw, lines, "dweight")
    _close(db, rdb, mdb, lines, "dbias")


@pytest.mark.gpu
def test_strides_axes_and_optional_weights():
    from samble_amd.norm import LayerNorm, layer_norm
    gen = torch.Generator(device=DEV).manual_seed(5)
    base = torch.randn((4, 6, 10, 50), generator=gen, device=DEV)
    w, b = torch.randn(10, generator=gen, device=DEV), torch.randn(10, generator=gen, device=DEV)
    views = [(base[:, :, :, 3:44], 2), (base.permute(0, 2, 1, 3), 1), (base[::2, 1:5], 2), (base.permute(3, 0, 1, 2), -1),
             (base[:, :, :, :10], 3), (base.transpose(2, 3)[:, :, 7:33], 3), (base[:, 0, :, 0], 1), (base[..., ::5], 3)]
    for t, dim in views:
        ry, my = _ref(t, w, b, 1e-3, dim)
        _close(layer_norm(t, w, b, 1e-3, dim), ry, my, 128, f"{tuple(t.shape)} {t.stride()} axis {dim}")
    t = base[0, 0]
    _close(layer_norm(t), *_ref(t, None, None, 1e-5, 1), 128, "no weights")
    v = torch.randn(50, generator=gen, device=DEV)
    _close(layer_norm(t, v), *_ref(t, v, None, 1e-5, 1), 128, "no bias")
    _close(layer_norm(t, None, v), *_ref(t, None, v, 1e-5, 1), 128, "no weight")
    bias = v.clone().requires_grad_(True)
    g = torch.randn_like(t)
    (db,) = torch.autograd.grad(layer_norm(t, None, bias), bias, g)
    torch.testing.assert_close(db, g.sum(0), rtol=1e-5, atol=1e-5)
    mod = LayerNorm(10, dim=1).to(DEV)
    ref = torch.nn.LayerNorm(10).to(DEV)
    ref.load_state_dict(mod.state_dict())
    torch.testing.assert_close(mod(base[0].transpose(0, 1).transpose(0, 1)), ref(base[0].transpose(1, 2)).transpose(1, 2))


@pytest.mark.gpu
def test_gradients_that_come_by_one_output_only():
    from samble_amd.norm import layer_norm
    x, r = (torch.randn(5, 12, device=DEV, requires_grad=True) for _ in range(2))
    w = torch.randn(12, device=DEV, requires_grad=True)
    y, s = layer_norm(x, w, None, residual=r)
    g = torch.randn_like(x)
    dx, dr, dw = torch.autograd.grad(s, (x, r, w), g, retain_graph=True)
    assert torch.equal(dx, g) and torch.equal(dr, g) and not dw.any()
    one = torch.autograd.grad(y, (x, r, w), g)
    ref = _ref((x + r).detach(), w.detach(), None, 1e-5, 1, g)
    _close(one[0], ref[2], ref[3], 256, "dx")
    assert torch.equal(one[0], one[1])
    (only_x,) = torch.autograd.grad(layer_norm(x, w.detach(), None), x, g)
    assert torch.isfinite(only_x).all()


@pytest.mark.gpu
def test_empty_tensors_special_values_and_a_constant_row():
    from samble_amd.norm import layer_norm
    for shape, dim in (((0, 5), 1), ((3, 5, 0), 1), ((0, 4, 7), 1)):
        x = torch.empty(shape, device=DEV, requires_grad=True)
        w = torch.ones(shape[dim], device=DEV, requires_grad=True)
        y = layer_norm(x, w, None, dim=dim)
        dx, dw = torch.autograd.grad(y.sum(), (x, w))
        assert y.shape == x.shape and dx.shape == x.shape and not dw.any()
    x = torch.randn(6, 300, device=DEV)
    x[1, 7], x[3, 0], x[4] = float("nan"), float("inf"), 2.5
    y = layer_norm(x)
    assert torch.isnan(y[1]).all() and torch.isnan(y[3]).any() and not y[4].any()
    keep = [0, 2, 5]
    assert torch.equal(y[keep], layer_norm(x[keep]))
    # a large offset: the deviations are taken from the values, not from a difference of squares
    z = torch.randn(4, 1000, device=DEV) + 4096.0
    _close(layer_norm(z), *_ref(z, None, None, 1e-5, 1), 128, "offset")


@pytest.mark.gpu
def test_more_rows_and_columns_than_workgroups():
    from samble_amd.norm import layer_norm
    x = torch.randn((1 << 20) * 32 + 77, 4, device=DEV)       # 32 rows a workgroup, more than 2^20 workgroups of rows
    y = layer_norm(x)
    tail = slice(-100, None)
    _close(y[tail], *_ref(x[tail], None, None, 1e-5, 1), 128, "last rows")
    _close(y[:100], *_ref(x[:100], None, None, 1e-5, 1), 128, "first rows")


@pytest.mark.gpu
def test_other_stream_and_graph_replay():
    from samble_amd.norm import LayerNorm
    mod = LayerNorm(128, dim=1).to(DEV)
    x = torch.randn(4, 128, 333, device=DEV, requires_grad=True)
    g = torch.randn_like(x)
    eager = torch.autograd.grad(mod(x), [x, *mod.parameters()], g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = torch.autograd.grad(mod(x), [x, *mod.parameters()], g)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = torch.autograd.grad(mod(x), [x, *mod.parameters()], g)
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
        graph.replay()
        eager = torch.autograd.grad(mod(x), [x, *mod.parameters()], g)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, held)), k


def test_refusals():
    from samble_amd.norm import LayerNorm, layer_norm
    x = torch.randn(3, 4)
    for bad in (dict(x=torch.zeros(3, 4, dtype=torch.int32)), dict(x=torch.zeros(3, 4, dtype=torch.float64)),
                dict(x=torch.zeros(())), dict(x=torch.zeros(3, 0)), dict(x=x, weight=torch.ones(3)),
                dict(x=x, weight=torch.ones(4, dtype=torch.float16)), dict(x=x, bias=torch.ones(4, 1)),
                dict(x=x.half(), weight=torch.ones(4), bias=torch.ones(4).half()), dict(x=x, dim=2),
                dict(x=x, residual=torch.zeros(4)), dict(x=x, residual=x.half()), dict(x=x, eps=-1.0), dict(x=x, eps=float("nan"))):
        with pytest.raises(ValueError, match="layer_norm"):
            layer_norm(**bad)
    with pytest.raises(_lib.SambleError, match="GPU"):
        layer_norm(x)
    with pytest.raises(ValueError):
        LayerNorm(0)


def test_c_entries_refuse_bad_arguments():
    fwd = lambda **k: _lib.call("samble_layer_norm_fwd", *({**dict(  # noqa: E731
        t=0, wt=0, x=64, xo=4, xc=1, r=None, ro=0, rc=0, w=None, b=None, outer=2, C=4, inner=1, eps=1e-5, y=64, s=None, m=None,
        rs=None, st=None), **k}).values())
    for bad in (dict(t=3), dict(t=1, wt=2), dict(x=None), dict(outer=0), dict(C=0), dict(inner=-1), dict(y=None), dict(x=66),
                dict(r=64), dict(m=64)):
        with pytest.raises(_lib.SambleError, match="samble_layer_norm_fwd"):
            fwd(**bad)
    assert _lib.query("samble_layer_norm_workspace_bytes", 0, 128, 10, 1) >= 2 * 128 * 4
    assert _lib.query("samble_layer_norm_workspace_bytes", 5, 128, 10, 1) == 0
    with pytest.raises(_lib.SambleError, match="workspace"):
        _lib.call("samble_layer_norm_bwd", 0, 0, 64, 4, 1, 64, 4, 1, None, 0, 0, None, 64, 64, 2, 4, 1, 64, 64, 64, None, 0, None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("shape", [(5, 300, 1), (9, 4099, 1), (3, 8200, 1), (3, 16390, 1), (2, 64, 37), (2, 700, 40), (2, 1030, 50)],
                         ids=lambda s: "x".join(map(str, s)))
def test_input_gradient_in_the_place_of_another_gradient(shape, dtype):
    """The C entry allows dx = dy and dx = extra where those are contiguous: the same bits as into a tensor of its own."""
    outer, C, inner = shape
    gen = torch.Generator(device=DEV).manual_seed(C)
    rnd = lambda *s: torch.randn(s, generator=gen, device=DEV)  # noqa: E731
    x, dy, extra = ((rnd(*shape) + 0.3).to(dtype) for _ in range(3))
    w, mean, rstd = 1 + 0.3 * rnd(C), 0.1 * rnd(outer * inner), 0.5 + rnd(outer * inner).abs()
    kind = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    nbytes = _lib.query("samble_layer_norm_workspace_bytes", kind, C, outer, inner)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=DEV)
    stream = torch.cuda.current_stream().cuda_stream

    def run(dy, extra, dx):
        dw, db = torch.empty((2, C), device=DEV)
        _lib.call("samble_layer_norm_bwd", kind, 0, x.data_ptr(), C * inner, inner, dy.data_ptr(), C * inner, inner,
                  extra.data_ptr(), C * inner, inner, w.data_ptr(), mean.data_ptr(), rstd.data_ptr(), outer, C, inner,
                  dx.data_ptr(), dw.data_ptr(), db.data_ptr(), ws.data_ptr(), nbytes, stream)
        return dx, dw, db

    apart = run(dy, extra, torch.empty_like(x))
    over_dy = dy.clone()
    for a, b in zip(apart, run(over_dy, extra, over_dy)):
        assert torch.equal(a, b), "dx = dy"
    over_extra = extra.clone()
    for a, b in zip(apart, run(dy, over_extra, over_extra)):
        assert torch.equal(a, b), "dx = extra"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_more_channel_slices_than_workgroups_of_a_launch(dtype):
    """A slice of few columns is one workgroup's work, and a launch holds at most 2^20 workgroups: the rest is walked to."""
    from samble_amd.norm import layer_norm
    B, C, N = (1 << 20) + 77, 5, 2
    gen = torch.Generator(device=DEV).manual_seed(9)
    x, r = ((torch.randn((B, C, N), generator=gen, device=DEV) + 0.4).to(dtype) for _ in range(2))
    w, b = (torch.randn(C, generator=gen, device=DEV) for _ in range(2))
    with torch.no_grad():
        y, s = layer_norm(x, w, b, dim=1, residual=r)
    assert torch.equal(s, (x.float() + r.float()).to(dtype))
    for part in (slice(0, 200), slice((1 << 20) - 50, (1 << 20) + 50), slice(B - 200, B)):
        _close(y[part], *_ref(s[part], w, b, 1e-5, 1), 128, str(part))


@pytest.mark.gpu
def test_forward_mode_is_refused():
    """A tangent is not dropped without a word."""
    from torch.autograd import forward_ad

    from samble_amd.norm import layer_norm
    x, t, w = torch.randn(3, 8, device=DEV), torch.randn(3, 8, device=DEV), torch.randn(8, device=DEV)
    with forward_ad.dual_level():
        plain = layer_norm(x, w)
        for kw in (dict(x=forward_ad.make_dual(x, t), weight=w), dict(x=x, weight=forward_ad.make_dual(w, w)),
                   dict(x=x, residual=forward_ad.make_dual(x, t))):
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(RuntimeError):
                    layer_norm(**kw)
    assert torch.equal(plain, layer_norm(x, w))


def test_slices_beyond_the_kernels_indices_are_refused():
    """2^32 + 5 values are not 5, and a 32-bit index does not step past 2^31."""
    from samble_amd.norm import layer_norm
    for n in ((1 << 30) + 1, (1 << 31) - 1, (1 << 32) + 5):
        for shape, dim in (((n,), 0), ((1, n, 2), 1)):
            with pytest.raises(ValueError, match="layer_norm"):
                layer_norm(torch.zeros(()).expand(shape), dim=dim)
    wide = torch.zeros(()).expand(1 << 26)
    with pytest.raises(ValueError, match="2\\^26"):
        layer_norm(wide, wide.clone().requires_grad_(True))
    fwd = [0, 0, 64, 4, 1, None, 0, 0, None, None, 2, 4, 1, 1e-5, 64, None, None, None, None]
    bwd = [0, 0, 64, 4, 1, 64, 4, 1, None, 0, 0, None, 64, 64, 2, 4, 1, 64, 64, 64, 64, 1 << 50, None]
    for n in ((1 << 30) + 1, (1 << 31) - 1):
        for name, args, at in (("samble_layer_norm_fwd", fwd, 11), ("samble_layer_norm_bwd", bwd, 15)):
            with pytest.raises(_lib.SambleError, match=name):
                _lib.call(name, *args[:at], n, *args[at + 1:])
    with pytest.raises(_lib.SambleError, match="2\\^26"):
        _lib.call("samble_layer_norm_bwd", *bwd[:15], 1 << 26, *bwd[16:])
