"""Group norm with an activation (csrc/group_norm.hip) against its formula in 64 bits on the CPU, and its refusals.

Tolerances.  u = eps / 2 of the map's type is the rounding of a result; 32-bit arithmetic in between adds a few 2^-24 of the
terms (x - mean) rstd w and b of z, and of the three terms of dx.  SiLU adds the 32-bit exponential's error (2 ulp + |z| 2^-23).
dw and db are 64-bit sums of products with up to 4 roundings each of 2^-24."""
import contextlib

import pytest
import torch

gpu = pytest.mark.gpu
ACTS = (False, True, 0.01, "silu")
E32 = 2.0 ** -24


def _make(N, C, sp, dtype, layout, seed=0, offset=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, C, *sp, generator=g) * (0.5 + torch.rand(1, C, *[1] * len(sp), generator=g)) + offset * torch.randn(
        1, C, *[1] * len(sp), generator=g)
    dy = torch.randn(N, C, *sp, generator=g)
    w, b = 1 + 0.3 * torch.randn(C, generator=g), 0.3 * torch.randn(C, generator=g)
    x, dy = x.to(dtype), dy.to(dtype)
    return x, dy, w, b


def _place(v, layout):
    v = v.cuda()
    return v.movedim(1, -1).contiguous().movedim(-1, 1) if layout == "last" else v


def _formula(x, dy, G, w, b, eps, relu):
    x, dy = x.double(), dy.double()
    N, C = x.shape[:2]
    one = torch.ones(C, dtype=torch.float64)
    w, b = (one if w is None else w.double()), (0 * one if b is None else b.double())
    w3, b3 = w.reshape(1, C, 1), b.reshape(1, C, 1)
    xs, ds = x.reshape(N, C, -1), dy.reshape(N, C, -1)
    rows = xs.reshape(N, G, -1)
    mean, var = rows.mean(2), rows.var(2, unbiased=False)
    rstd = 1 / (var + eps).sqrt()

    def wide(v):
        return v.repeat_interleave(C // G, 1).unsqueeze(2)
    xhat = (xs - wide(mean)) * wide(rstd)
    z = xhat * w3 + b3
    if relu == "silu":
        s = 1 / (1 + torch.exp(-z))
        y, d = z * s, s * (1 + z * (1 - s))
    else:
        slope = 1.0 if relu is False else 0.0 if relu is True else relu
        d = torch.where(z > 0, 1.0, slope).double()
        y = torch.where(z > 0, z, slope * z if slope else torch.zeros_like(z))
    g = ds * d
    db, dw = g.sum((0, 2)), (g * xhat).sum((0, 2))
    gw = g * w3
    m1 = gw.reshape(N, G, -1).mean(2)
    m2 = (gw * xhat).reshape(N, G, -1).mean(2)
    dx = wide(rstd) * (gw - wide(m1) - xhat * wide(m2))
    mag_y = (xhat * w3).abs() + b3.abs()                                       # terms of z
    mag_dx = wide(rstd) * (gw.abs() + wide(m1).abs() + (xhat * wide(m2)).abs())
    # The group's two means are sums of terms of either sign: their error goes by the terms' magnitudes, not by the sums'.
    # g w is rounded once (slope dy), x - mean three times (x - mh, ml, - ml), the product once, and four products are
    # added in 32 bits (3 more) before 64 bits take over: at most 4 and 8 roundings of a term, so the errors of m1 and m2
    # are at most 4 and 8 x 2^-24 of the means of |g w| and |g w xhat|
    am1 = gw.abs().reshape(N, G, -1).mean(2)
    am2 = (gw * xhat).abs().reshape(N, G, -1).mean(2)
    mag_m = wide(rstd) * (4 * wide(am1) + 8 * xhat.abs() * wide(am2))
    return dict(y=y.reshape(x.shape), dx=dx.reshape(x.shape), dw=dw, db=db, mean=mean, rstd=rstd, mag_y=mag_y.reshape(x.shape),
                mag_dx=mag_dx.reshape(x.shape), mag_dw=(g * xhat).abs().sum((0, 2)), mag_db=g.abs().sum((0, 2)),
                mag_m=mag_m.reshape(x.shape), dgdz=(ds.abs() * w3.abs() * wide(rstd)).reshape(x.shape))


def _close(got, want, tol, what):
    err = (got.double().cpu() - want).abs()
    bad = err > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err - tol).max()):.3e} over its tolerance"


def _check(x, dy, G, w, b, relu, layout, eps=1e-5, dtype=None):
    from boostmvsnerfs_amd import autograd as A
    ref = _formula(x, dy, G, w, b, eps, relu)
    u = torch.finfo(x.dtype).eps / 2
    xg, dyg = _place(x, layout).requires_grad_(), _place(dy, layout)
    wg, bg = (None if v is None else v.cuda().requires_grad_() for v in (w, b))
    y = A.GroupNormAct.apply(xg, G, wg, bg, eps, relu)
    assert y.dtype == x.dtype and y.shape == x.shape and y.stride() == xg.stride()
    y.backward(dyg)
    silu = relu == "silu"
    # y: its rounding + 32-bit rounding of the terms of z (x - mh, - ml, rstd w, *, +; SiLU: exp, +, / on top)
    tol = u * ref["y"].abs() + (6 + (8 + 2 * ref["mag_y"] if silu else 0)) * E32 * ref["mag_y"] + 1e-37
    if x.dtype == torch.float16:
        tol = tol + 2.0 ** -25                                                # (half a step of the subnormal range)
    _close(y.detach(), ref["y"], tol, "y")
    # dx: its rounding + 8 roundings of its terms; SiLU's slope carries z's error (|slope'| <= 0.5 of |dy w rstd|)
    tol = u * ref["dx"].abs() + 8 * E32 * ref["mag_dx"] + E32 * ref["mag_m"] + 1e-37
    if silu:
        tol = tol + ref["dgdz"] * E32 * (16 + 8 * ref["mag_y"])
    if x.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    _close(xg.grad, ref["dx"], tol, "dx")
    for got, key in ((wg, "dw"), (bg, "db")):
        if got is not None:
            uw = torch.finfo(got.dtype).eps / 2
            _close(got.grad, ref[key], uw * ref[key].abs() + (16 if not silu else 64) * E32 * ref["mag_" + key] + 1e-37, key)
            assert got.grad.dtype == got.dtype


# one position / one value a group; odd channel and row counts; slabs of a wide channel axis; groups across slab borders;
# row chunks that end ragged
SHAPES = [(1, 4, (1, 1), 2), (2, 3, (1, 1), 3), (1, 8, (5, 7), 8), (2, 6, (9, 5), 3), (3, 30, (13, 11), 5), (1, 64, (8, 8, 10), 8),
          (2, 320, (9, 9), 32), (1, 1030, (3, 5), 1), (1, 2080, (2, 3), 5), (2, 520, (7,), 4), (1, 7, (129, 131), 1),
          (1, 12, (3, 4099), 4), (5, 24, (1, 17), 24), (1, 1, (33, 3), 1),
          # one launch by 256 and 1024 threads, and just too large for either; groups across the borders of 16-byte accesses
          (2, 8, (32, 32), 2), (2, 8, (32, 33), 2), (2, 8, (64, 64), 2), (2, 8, (64, 65), 2), (2, 60, (21, 20), 6), (1, 24, (90, 31), 8),
          (2, 320, (64, 5), 32), (1, 40, (23, 29), 8), (1, 96, (7, 300), 2)]


@gpu
@pytest.mark.parametrize("layout", ["last", "planar"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, (s[0], s[1], *s[2]))) + f"g{s[3]}")
def test_group_norm_matches_the_formula(shape, dtype, layout):
    N, C, sp, G = shape
    for i, relu in enumerate(ACTS):
        x, dy, w, b = _make(N, C, sp, dtype, layout, seed=i)
        _check(x, dy, G, w, b, relu, layout)


@gpu
@pytest.mark.parametrize("layout", ["last", "planar"])
def test_group_norm_many_chunks_and_the_finishing_launch(layout):
    """Maps whose partial sums come from hundreds of workgroups (with the launch that joins them in front of the second pass)."""
    for N, C, sp, G, dtype in ((1, 8, (640, 517), 1, torch.float32), (2, 64, (131, 128), 64, torch.bfloat16), (1, 256, (96, 97), 1, torch.float32), (1, 19, (200, 150), 19, torch.float16),
                               (3, 30, (131, 97), 30, torch.float32)):
        x, dy, w, b = _make(N, C, sp, dtype, layout, seed=3)
        _check(x, dy, G, w, b, True, layout)


@gpu
def test_group_norm_without_parameters_and_with_16_bit_ones():
    x, dy, w, b = _make(2, 12, (6, 5), torch.bfloat16, "last")
    _check(x, dy, 3, None, None, "silu", "last")
    _check(x, dy, 3, w, None, 0.01, "last")
    _check(x, dy, 3, None, b, True, "planar")
    _check(x, dy, 3, w.bfloat16(), b.bfloat16(), True, "last")


@gpu
def test_group_norm_of_a_large_common_offset():
    """mean / std = 4000: x - mean is exact to x's own rounding (the values are what they are), so nothing else may be lost."""
    x, dy, w, b = _make(2, 8, (31, 33), torch.float32, "last", offset=0.0)
    _check(x + 4000.0, dy, 2, w, b, 0.01, "last")


@gpu
@pytest.mark.parametrize("layout", ["last", "planar"])
def test_group_norm_of_offsets_that_fp32_only_just_holds(layout):
    """mean / std = 5e6: sum x^2 / M - mean^2 in 64 bits would be off by 2^-52 (mean / std)^2 of the variance, half a percent.
    Small maps (one launch), middle and large ones (two launches, with the joining one)."""
    from boostmvsnerfs_amd import ops
    for N, C, sp, G in ((2, 8, (9, 11), 2), (1, 6, (5, 7), 2), (2, 12, (5, 9), 4), (2, 8, (64, 65), 2), (1, 30, (90, 31), 5), (1, 19, (150, 100), 19), (1, 8, (300, 200), 1)):
        x, dy, w, b = _make(N, C, sp, torch.float32, layout, seed=4, offset=0.0)
        x = 3e5 + 0.05 * x
        ref = x.double().reshape(N, G, -1) - 3e5                      # (exact)
        _, mean, rstd = ops.group_norm_fwd(_place(x, layout), G, w.cuda(), b.cuda())
        # 64-bit sums of d = x - pivot over M <= 480000 values lose at most M 2^-52 of the variance, half of that of rstd
        _close(rstd, 1 / (ref.var(2, unbiased=False) + 1e-5).sqrt(), 1e-10 * rstd.double().cpu(), "rstd")
        _close(mean - 3e5, ref.mean(2), 1e-9, "mean")               # (the mean itself is rounded by 2^-53 of 3e5)
        _check(x, dy, G, w, b, 0.01, layout)


@gpu
def test_group_norm_constant_groups_and_zero_eps():
    x = torch.full((2, 4, 6, 5), 3.0)
    _, dy, w, b = _make(2, 4, (6, 5), torch.float32, "last")
    _check(x, dy, 2, w, b, True, "last")           # variance 0: y = act(b)
    x, dy, w, b = _make(1, 4, (6, 5), torch.float32, "last")
    _check(x, dy, 2, w, b, False, "last", eps=0.0)


@gpu
def test_group_norm_other_strides_and_offsets():
    from boostmvsnerfs_amd import autograd as A
    from boostmvsnerfs_amd import ops
    x, dy, w, b = _make(2, 12, (10, 9), torch.float32, "planar")
    ref = _formula(x[:, ::2, 1:, :8], dy[:, ::2, 1:, :8], 3, w[::2], b[::2], 1e-5, True)
    xg, wg, bg = x.cuda()[:, ::2, 1:, :8].requires_grad_(), w.cuda()[::2].requires_grad_(), b.cuda()[::2].requires_grad_()
    y = A.GroupNormAct.apply(xg, 3, wg, bg, 1e-5, True)
    y.sum().backward()                                # (a gradient of stride 0)
    one = _formula(x[:, ::2, 1:, :8], torch.ones(2, 6, 9, 8), 3, w[::2], b[::2], 1e-5, True)
    _close(y.detach(), ref["y"], 8 * E32 * ref["mag_y"] + 1e-37, "y")
    _close(xg.grad, one["dx"], 10 * E32 * one["mag_dx"] + E32 * one["mag_m"], "dx")
    _close(wg.grad, one["dw"], 17 * E32 * one["mag_dw"], "dw")
    # a planar gradient for a channel-last map, and maps that begin at an odd address
    xl, dyp = _place(x, "last").requires_grad_(), dy.cuda()
    ref = _formula(x, dy, 3, w, b, 1e-5, 0.01)
    y = A.GroupNormAct.apply(xl, 3, w.cuda(), b.cuda(), 1e-5, 0.01)
    y.backward(dyp)
    _close(xl.grad, ref["dx"], 9 * E32 * ref["mag_dx"] + E32 * ref["mag_m"], "dx")
    flat = torch.cat([torch.zeros(1), x.flatten()]).cuda()
    y, mean, rstd = ops.group_norm_fwd(flat[1:].view(x.shape), 3, w.cuda(), b.cuda(), 1e-5, 0.01)
    _close(y, ref["y"], 8 * E32 * ref["mag_y"] + 1e-37, "y at an odd address")
    _close(mean, ref["mean"], 1e-14 * (1 + ref["mean"].abs()), "mean")
    _close(rstd, ref["rstd"], 1e-13 * ref["rstd"], "rstd")


@gpu
@pytest.mark.parametrize("layout", ["last", "planar"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_group_norm_gradient_sums_leave_32_bits_after_four_terms(dtype, layout):
    """Large terms among many of 2^-24 of them, which a long sum in 32 bits loses all.  Without an activation g is dy itself, so
    db's error is the sums' alone: three roundings of at most 2^-24 of four terms of one sign, and the result's one (the
    64-bit sums and second-order terms are in the last 2^-4 of a 2^-24)."""
    from boostmvsnerfs_amd import ops
    x = torch.randn(1, 2, 32, 64, generator=torch.Generator().manual_seed(1)).to(dtype)
    i = torch.arange(2048)
    dy = torch.where((i % 8 == 0) & (i < 512), 2.0 ** 10, 2.0 ** -14).to(dtype).view(1, 1, 32, 64).expand(1, 2, 32, 64).contiguous()
    xg, dyg, w, b = _place(x, layout), _place(dy, layout), torch.ones(2).cuda(), torch.zeros(2).cuda()
    _, mean, rstd = ops.group_norm_fwd(xg, 1, w, b)
    db = ops.group_norm_bwd(xg, dyg, 1, w, b, mean, rstd)[2]
    want = dy.double().sum((0, 2, 3))
    _close(db, want, (4 + 2 ** -4) * E32 * want, "db")


@gpu
def test_group_norm_decides_the_sign_at_zero_as_64_bits_do():
    """Values whose exact z is a few 1e-9 off zero, either side: a 32-bit z cannot tell them apart, dx would be off by dy."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(1, 4, 64, 64, generator=g)
    ref = _formula(x, x, 1, None, None, 1e-5, False)
    # b = -xhat of one value per channel, rounded to fp32: |z| there is below 2^-25 |b|
    b = torch.stack([-ref["y"][0, c, 7 + c, 9] for c in range(4)]).float()
    dy = torch.randn(1, 4, 64, 64, generator=g)
    z = ref["y"] + b.double().view(1, 4, 1, 1)
    assert all(0 < abs(float(z[0, c, 7 + c, 9])) < 2 ** -23 for c in range(4))
    for layout in ("last", "planar"):
        _check(x, dy, 1, torch.ones(4), b, True, layout)


@gpu
@pytest.mark.parametrize("layout", ["last", "planar"])
def test_group_norm_nan_and_inf_stay_in_their_group(layout):
    from boostmvsnerfs_amd import ops
    x, dy, w, b = _make(2, 8, (6, 7), torch.float32, layout)
    clean = ops.group_norm_fwd(_place(x, layout), 4, w.cuda(), b.cuda(), 1e-5, True)[0].cpu()
    x[0, 0, 2, 3], x[1, 7, 0, 0] = float("nan"), float("inf")
    y, mean, rstd = ops.group_norm_fwd(_place(x, layout), 4, w.cuda(), b.cuda(), 1e-5, True)
    y = y.cpu()
    assert y[0, :2].isnan().all() and y[1, 6:].isnan().all()
    assert torch.equal(y[0, 2:], clean[0, 2:]) and torch.equal(y[1, :6], clean[1, :6])
    dx, dw, db = ops.group_norm_bwd(_place(x, layout), _place(dy, layout), 4, w.cuda(), b.cuda(), mean, rstd, True)
    dx = dx.cpu()
    assert dx[0, :2].isnan().all() and dx[0, 2:].isfinite().all() and dx[1, :6].isfinite().all()
    assert dw[2:6].isfinite().all() and db[2:6].isfinite().all()


@gpu
def test_group_norm_empty_maps():
    from boostmvsnerfs_amd import autograd as A
    w, b = torch.ones(4, device="cuda", requires_grad=True), torch.ones(4, device="cuda", requires_grad=True)
    for shape in ((0, 4, 3, 3), (2, 4, 0, 3)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        y = A.GroupNormAct.apply(x, 2, w, b, 1e-5, True)
        assert y.shape == x.shape
        w.grad = b.grad = None
        y.sum().backward()
        assert x.grad.shape == x.shape and not w.grad.any() and not b.grad.any()


@gpu
def test_group_norm_is_reproducible_on_another_stream_and_in_a_graph():
    from boostmvsnerfs_amd import ops
    x, dy, w, b = _make(2, 24, (65, 64), torch.float32, "last")
    x, dy, w, b = _place(x, "last"), _place(dy, "last"), w.cuda(), b.cuda()

    def both():
        y, mean, rstd = ops.group_norm_fwd(x, 4, w, b, 1e-5, 0.01)
        return (y, *ops.group_norm_bwd(x, dy, 4, w, b, mean, rstd, 0.01))
    want = [v.clone() for v in both()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    side.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for k in range(3):
        x.add_(0.25 * k)                              # other values: the replay reads the tensors, not what it saw
        want = [v.clone() for v in both()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(out, want)), k


@gpu
def test_group_norm_gradients_against_differences():
    """d(sum y r) / dp against (f(p + h) - f(p - h)) / 2 h of the formula in 64 bits, along random directions."""
    from boostmvsnerfs_amd import autograd as A
    x, r, w, b = _make(2, 6, (5, 7), torch.float32, "last")
    xg, wg, bg = _place(x, "last").requires_grad_(), w.cuda().requires_grad_(), b.cuda().requires_grad_()
    A.GroupNormAct.apply(xg, 3, wg, bg, 1e-5, "silu").backward(_place(r, "last"))
    g = torch.Generator().manual_seed(2)

    def f(x, w, b):
        return float((_formula(x, r, 3, w, b, 1e-5, "silu")["y"] * r.double()).sum())
    x, w, b = x.double(), w.double(), b.double()
    h = 1e-5
    for k, (p, grad) in enumerate(((x, xg.grad), (w, wg.grad), (b, bg.grad))):
        v = torch.randn(p.shape, generator=g).double()
        args = [[x, w, b], [x, w, b]]
        args[0][k], args[1][k] = p + h * v, p - h * v
        want = (f(*args[0]) - f(*args[1])) / (2 * h)
        got = float((grad.double().cpu() * v).sum())
        scale = float((grad.double().cpu() * v).abs().sum())
        # 64-bit differences: h^2 f''' / 6 (h = 1e-5, a smooth function of unit scale) and rounding 1e-16 / h; fp32 gradients 2^-21
        assert abs(got - want) <= scale * (2 ** -20 + 1e-8), (k, got, want)


@gpu
@pytest.mark.parametrize("layout", ["last", "planar"])
def test_group_norm_with_saved_tensors_in_another_layout(layout):
    """Hooks on saved tensors may hand the backward x in other strides (a copy to the host and back does)."""
    from boostmvsnerfs_amd import autograd as A
    x, r, w, b = _make(2, 8, (5, 7), torch.float32, layout)

    def grads(hooks):
        xg, wg, bg = _place(x, layout).requires_grad_(), w.cuda().requires_grad_(), b.cuda().requires_grad_()
        with hooks:
            y = A.GroupNormAct.apply(xg, 4, wg, bg, 1e-5, True)
        return torch.autograd.grad(y, (xg, wg, bg), _place(r, layout))
    want = grads(contextlib.nullcontext())
    other = torch.autograd.graph.saved_tensors_hooks(
        lambda t: t.cpu(), lambda t: t.cuda().transpose(1, -1).contiguous().transpose(1, -1) if t.dim() == 4 and layout == "planar"
        else t.cuda().contiguous())
    for hooks in (torch.autograd.graph.save_on_cpu(), other):
        assert all(torch.equal(u, v) for u, v in zip(grads(hooks), want))


@gpu
def test_group_norm_keeps_no_answer_by_an_arguments_identity():
    from boostmvsnerfs_amd import ops
    x, eps = torch.randn(1, 4, 3, 3, device="cuda"), torch.tensor(1e-5)
    a = ops.group_norm_fwd(x, 2, eps=eps)[0]
    eps.fill_(3.0)
    assert torch.equal(ops.group_norm_fwd(x, 2, eps=eps)[0], ops.group_norm_fwd(x, 2, eps=3.0)[0]) and not torch.equal(a, ops.group_norm_fwd(x, 2, eps=eps)[0])


@gpu
def test_group_norm_refuses_a_second_differentiation():
    from boostmvsnerfs_amd import autograd as A
    x = torch.randn(1, 4, 5, 5, device="cuda", requires_grad=True)
    dx, = torch.autograd.grad(A.GroupNormAct.apply(x, 2, None, None, 1e-5, "silu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="second differentiation"):
        dx.sum().backward()


def test_group_norm_refusals():
    from boostmvsnerfs_amd import ops
    x, w = torch.zeros(1, 4, 2, 2), torch.ones(4)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.group_norm_fwd(x, 2, w, w)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        ops.group_norm_fwd(x.double(), 2)
    with pytest.raises(TypeError, match="expected a tensor"):
        ops.group_norm_fwd([1.0], 2)


def test_group_norm_refuses_maps_whose_launches_would_be_too_large():
    """The host's sizes, in front of any launch: 2^32 threads are one too many."""
    import ctypes as C

    from boostmvsnerfs_amd import _lib
    lib = _lib.load()

    def size(backward=0, **kw):
        return lib.bmv_group_norm_workspace(C.byref(_lib.GroupNormSpec(**{"G": 1, "S": 1, "channels_last": 1, **kw})), backward)
    for backward in (0, 1):
        assert size(backward, N=1 << 23, C=1) > 0 and size(backward, N=1 << 14, C=1 << 10) > 0
        assert size(backward, N=1 << 23, C=1, S=1 << 17, channels_last=0) > 0
        assert size(backward, N=1 << 24, C=1) == -1 and b"too many workgroups" in lib.bmv_last_error()
        assert size(backward, N=(1 << 24) - 1, C=1) == -1             # (with the workgroups of the parameters' gradients)
        assert size(backward, N=1 << 14, C=(1 << 10) + 1) == -1 and b"too large" in lib.bmv_last_error()
        assert size(backward, N=1 << 23, C=1, S=(1 << 17) + 1) == -1 and b"too large" in lib.bmv_last_error()


@gpu
def test_group_norm_of_very_many_groups_that_a_workgroup_would_hold():
    """2^22 groups of 2049 values: held by 1024 threads each they would be 2^32 threads, so they take two launches."""
    from boostmvsnerfs_amd import ops
    x, dy, w, b = _make(512, 1, (2049,), torch.float16, "planar", seed=6)
    ref = _formula(x, dy, 1, w, b, 1e-5, True)
    many = x.cuda().repeat(1 << 13, 1, 1)
    y, mean, rstd = ops.group_norm_fwd(many, 1, w.cuda(), b.cuda(), 1e-5, True)
    _close(y[:512], ref["y"], 2.0 ** -11 * ref["y"].abs() + 6 * E32 * ref["mag_y"] + 2.0 ** -25, "y")
    _close(rstd[:512], ref["rstd"], 1e-12 * ref["rstd"], "rstd")
    for k in range(0, 1 << 22, 512 * 256):
        assert all(torch.equal(v[k:k + 512 * 256].view(256, 512, -1), v[:512].view(1, 512, -1).expand(256, -1, -1)) for v in (y, mean, rstd)), k


@gpu
def test_group_norm_refusals_on_the_gpu():
    from boostmvsnerfs_amd import _lib, ops
    x, w = torch.zeros(1, 4, 2, 2, device="cuda"), torch.ones(4, device="cuda")
    for groups in (0, 3, -2, 8):
        with pytest.raises(ValueError, match="divide"):
            ops.group_norm_fwd(x, groups, w, w)
    with pytest.raises(ValueError, match="weight"):
        ops.group_norm_fwd(x, 2, w[:3], None)
    with pytest.raises(TypeError, match="weight"):
        ops.group_norm_fwd(x, 2, w.half(), w.half())
    with pytest.raises(TypeError, match="one type"):
        ops.group_norm_fwd(x.half(), 2, w.half(), w)
    with pytest.raises(RuntimeError, match="bias: the"):
        ops.group_norm_fwd(x, 2, w, torch.ones(4))
    with pytest.raises(ValueError, match="silu"):
        ops.group_norm_fwd(x, 2, w, w, relu="gelu")
    with pytest.raises(ValueError, match="eps"):
        ops.group_norm_fwd(x, 2, w, w, eps=-1.0)
    with pytest.raises(ValueError, match="N, C"):
        ops.group_norm_fwd(w, 2)
    # what is remembered of a kind of call tells a slope of 1 from a ReLU and of 0 from none
    v = torch.randn(1, 4, 3, 3, device="cuda")
    assert (ops.group_norm_fwd(v, 2, w, w * 0, relu=True)[0] >= 0).all() and (ops.group_norm_fwd(v, 2, w, w * 0, relu=1.0)[0] < 0).any()
    assert (ops.group_norm_fwd(v, 2, w, w * 0, relu=0.0)[0] >= 0).all() and (ops.group_norm_fwd(v, 2, w, w * 0, relu=False)[0] < 0).any()
    y, mean, rstd = ops.group_norm_fwd(x, 2, w, w)
    with pytest.raises(ValueError, match="dy"):
        ops.group_norm_bwd(x, y.half(), 2, w, w, mean, rstd)
    with pytest.raises(ValueError, match="mean"):
        ops.group_norm_bwd(x, y, 2, w, w, mean.float(), rstd)
    lib = _lib.load()
    import ctypes as C
    assert lib.bmv_group_norm_workspace(C.byref(_lib.GroupNormSpec(N=1, C=4, G=3, S=4, channels_last=1)), 0) == -1
    assert b"multiple" in lib.bmv_last_error()
