"""Newton-Schulz orthogonalisation and the optimiser step around it (csrc/newton_schulz.hip) against the formula in 64 bits on
the CPU, and their refusals.

Tolerance of an iterate, in the Frobenius norm: a product L R^T over k terms in fp32 (three-piece operands: dropped products
below 3 x 2^-24 of a term, then fp32 sums) is off by at most eps_k |L|_F |R|_F with eps_k = 2^-24 (4 + 2 sqrt(k)) -- one
rounding of each operand, of the result, and k roundings of partial sums of random sign.  A step turns errors of its three products
into at most (|b| + 2 |c| |A|) dA |X| + |c| d(AA) |X| + d(QX) of X, and an error of X into at most L of it, L = max |p'| of the
polynomial p = a s + b s^3 + c s^5 over the iterate's singular values (of the divided differences as well, which p' bounds).
That sum is computed along the 64-bit iteration; bf16 and fp16 results add half a step of their rounding.

For bf16 matrices the operands have two pieces: each is off by at most 2^-18 of itself, and mid mid (2^-18) is dropped, so a term
l r is off by at most 3 x 2^-18 of itself, of random sign: a product by 3 x 2^-18 sqrt(sum_k |l_k|^2 |r_k|^2) over the columns
l_k, r_k (twice that is allowed: in X X^T the same rounding stands on both sides)."""
import math

import pytest
import torch

gpu = pytest.mark.gpu
COEFFS = (3.4445, -4.7750, 2.0315)


def _iterate(u, steps=5, coeffs=COEFFS, eps=1e-7, two=False):
    """(the iterate, its tolerance in the Frobenius norm) of u, in 64 bits; `two`: with operands of two pieces."""
    a, b, c = coeffs
    two = two or u.dtype == torch.bfloat16
    u = u.double()
    x = u / max(float(u.norm()), eps)
    tall = x.shape[0] > x.shape[1]
    x = x.mT if tall else x
    m, n = x.shape
    unit = 2.0 ** -24

    def off(l, r):                                     # of l r, the columns of l against the rows of r
        k = l.shape[1]
        d = unit * (4 + 2 * math.sqrt(k)) * float(l.norm()) * float(r.norm())
        return d + (6 * 2.0 ** -18 * float((l.norm(dim=0) * r.norm(dim=1)).norm()) if two else 0.0)
    tol = 2 * unit * float(x.norm())
    for _ in range(steps):
        A = x @ x.mT
        Q = a * torch.eye(m, dtype=torch.float64) + b * A + c * (A @ A)
        s = max(float(torch.linalg.matrix_norm(x, 2)), 1e-300)
        grid = torch.linspace(0, s, 200, dtype=torch.float64)
        lip = float((a + 3 * b * grid ** 2 + 5 * c * grid ** 4).abs().max())
        dA, dAA = off(x, x.mT), off(A, A)
        local = ((abs(b) + 2 * abs(c) * s * s) * dA + abs(c) * dAA) * s + off(Q, x)
        tol = lip * tol + local
        x = Q @ x
    return (x.mT if tall else x), tol


def _grad(m, n, seed=0, rank=3, noise=0.1):
    g = torch.Generator().manual_seed(seed)
    return 1e-2 * (noise * torch.randn(m, n, generator=g) + torch.randn(m, rank, generator=g) @ torch.randn(rank, n, generator=g))


def _check(got, u, steps=5, coeffs=COEFFS, eps=1e-7):
    want, tol = _iterate(u, steps, coeffs, eps)
    u_out = torch.finfo(got.dtype).eps / 2
    err = float((got.double().cpu() - want).norm())
    small = 2.0 ** -25 * math.sqrt(want.numel()) if got.dtype == torch.float16 else 0.0      # half a step of fp16's subnormals
    assert err <= tol + u_out * float(want.norm()) + small, (tuple(u.shape), err, tol)
    return err, tol


SHAPES = [(1, 1), (1, 7), (9, 1), (2, 2), (3, 64), (8, 27), (16, 200), (35, 4), (64, 24), (33, 32), (63, 65), (64, 64), (64, 1728),
          (65, 40), (80, 100), (127, 129), (128, 63), (8, 4000), (128, 1024), (1025, 100), (128, 2048), (97, 2049), (128, 4097), (33, 1000), (5, 16384), (17, 16385), (60, 1153), (112, 288), (112, 289), (96, 1200), (128, 128), (128, 515), (129, 129), (130, 1000), (333, 257), (256, 384), (700, 90)]


@pytest.fixture(params=["short", "blocks", "tiles"])
def way(request):
    """Short sides of up to 128 one launch a step (default), all through 64 x 64 blocks where those are taken (default above 128),
    all through the tiles of the large ones."""
    from boostmvsnerfs_amd import _lib
    _lib.set_tuning("BMV_NS_SHORT", None if request.param == "short" else 0)
    _lib.set_tuning("BMV_NS_BLOCK_K", {"short": None, "blocks": 1 << 20, "tiles": 0}[request.param])
    yield request.param
    _lib.set_tuning("BMV_NS_SHORT", None)
    _lib.set_tuning("BMV_NS_BLOCK_K", None)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_newton_schulz_matches_the_formula(dtype, way):
    from boostmvsnerfs_amd import ops
    mats = [_grad(m, n, seed=i).to(dtype) for i, (m, n) in enumerate(SHAPES)]
    on_gpu = [v.cuda() for v in mats]
    before = [v.clone() for v in on_gpu]
    out = ops.newton_schulz(on_gpu)
    for got, u, src, keep in zip(out, mats, on_gpu, before):
        assert got.shape == u.shape and got.dtype == dtype and torch.equal(src, keep)
        _check(got, u)
    # the same call again is the same bit for bit; a matrix alone is cut along k in other places (sums of fp32 in another order),
    # so it agrees within the tolerance
    for got, again in zip(out, ops.newton_schulz(on_gpu)):
        assert torch.equal(got, again), got.shape
    for src, u in zip(on_gpu, mats):
        _check(ops.newton_schulz(src), u)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_sixteen_bit_matrices_are_computed_as_fp32_ones(dtype, way):
    """A 16-bit matrix' result is the fp32 result of the same values rounded once, a 16-bit weight's step the fp32 step rounded
    once: bit for bit, because the way, the operands and the order of the sums go by the sizes alone."""
    from boostmvsnerfs_amd import ops
    mats = [_grad(m, n, seed=i).to(dtype).cuda() for i, (m, n) in enumerate(SHAPES)]
    for steps in (5, 8):
        for got, want in zip(ops.newton_schulz(mats, steps=steps), ops.newton_schulz([v.float() for v in mats], steps=steps)):
            assert torch.equal(got, want.to(dtype)), (steps, got.shape)
    for m, n in ((700, 90), (333, 1000), (1024, 1100)):                     # ... alone as well
        u = _grad(m, n, 7).to(dtype).cuda()
        assert torch.equal(ops.newton_schulz(u), ops.newton_schulz(u.float()).to(dtype)), (m, n)
    g = torch.Generator().manual_seed(3)
    params = [torch.randn(v.shape, generator=g).to(dtype).cuda() for v in mats]
    momenta = [1e-2 * torch.randn(v.shape, generator=g).cuda() for v in mats]
    p32, m32 = [p.float() for p in params], [m.clone() for m in momenta]
    ops.muon_step(params, mats, momenta, 0.02, weight_decay=0.01)
    ops.muon_step(p32, [v.float() for v in mats], m32, 0.02, weight_decay=0.01)
    for p, m, q, k in zip(params, momenta, p32, m32):
        assert torch.equal(m, k) and torch.equal(p, q.to(dtype)), p.shape


@gpu
def test_newton_schulz_is_as_exact_as_the_iteration_in_fp32(way):
    """Within four times the error of the same iteration in fp32 products (four: two roundings for its one at the operands'
    pieces, and the spread of one random error against another), on flat and on decaying spectra."""
    from boostmvsnerfs_amd import ops

    def fp32(u):
        a, b, c = COEFFS
        x = u / u.norm()
        for _ in range(5):
            A = x @ x.mT
            x = a * x + (b * A + c * (A @ A)) @ x
        return x
    for k, (m, n, rank, noise) in enumerate([(64, 200, 3, 0.1), (128, 128, 3, 0.1), (128, 1000, 128, 1.0), (256, 300, 5, 0.01), (200, 200, 200, 1.0)]):
        u = _grad(m, n, k, rank, noise)
        want, _ = _iterate(u)
        base = float((fp32(u).double() - want).norm() / want.norm())
        err = float((ops.newton_schulz(u.cuda()).double().cpu() - want).norm() / want.norm())
        assert err <= 4 * base + 2.0 ** -24, (m, n, err, base)


@gpu
def test_newton_schulz_large_matrices():
    from boostmvsnerfs_amd import ops
    for m, n in ((1024, 1100), (1500, 520)):
        u = _grad(m, n, 7)
        _check(ops.newton_schulz(u.cuda()), u)


def _through_tiles(mats, **kw):
    from boostmvsnerfs_amd import _lib, ops
    _lib.set_tuning("BMV_NS_SHORT", 0)
    _lib.set_tuning("BMV_NS_BLOCK_K", 0)
    try:
        return ops.newton_schulz(mats, **kw)
    finally:
        _lib.set_tuning("BMV_NS_SHORT", None)
        _lib.set_tuning("BMV_NS_BLOCK_K", None)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_newton_schulz_whole_tiles_and_cut_ones_in_one_launch(dtype):
    """Lists of more than 512 tiles: 512 are a workgroup each, the rest is cut along k.  40 matrices of 15 symmetric tiles and 25
    others (600 and 1000 a launch), tall and wide, on and off the tiles' borders; the matrices repeat, so that each is in whole
    tiles and in cut ones."""
    kinds = [_grad(m, n, seed).to(dtype) for seed, (m, n) in enumerate([(520, 600), (600, 520), (513, 640), (640, 577), (640, 640)])]
    on_gpu = [v.cuda() for v in kinds]
    refs = [_iterate(u) for u in kinds]
    out = _through_tiles(on_gpu * 8)
    again = _through_tiles(on_gpu * 8)
    u_out = torch.finfo(dtype).eps / 2
    for k, (got, twice) in enumerate(zip(out, again)):
        want, tol = refs[k % 5]
        small = 2.0 ** -25 * math.sqrt(want.numel()) if dtype == torch.float16 else 0.0
        assert torch.equal(got, twice), k
        assert float((got.double().cpu() - want).norm()) <= tol + u_out * float(want.norm()) + small, (k, tuple(want.shape))


@gpu
def test_newton_schulz_tiles_of_more_than_one_super_row():
    """A short side of nine tiles: the second super-row of both enumerations, alone (all cut) and twelve times (540 symmetric
    tiles and 972 others: whole and cut)."""
    u = _grad(1100, 1030, 5)
    want, tol = _iterate(u)
    for got in _through_tiles([u.cuda()]) + _through_tiles([u.cuda()] * 12):
        assert float((got.double().cpu() - want).norm()) <= tol + 2.0 ** -24 * float(want.norm())


@gpu
def test_newton_schulz_lists_that_fill_the_card():
    """bf16 symmetric products in blocks of 128 x 64, which are taken where the list keeps the compute units busy: panels of one
    to four, sides on and off their borders, tall and wide, two lengths of k.  And a large matrix alone."""
    from boostmvsnerfs_amd import _lib, ops
    sizes = [(129, 140), (256, 256), (257, 400), (300, 150), (384, 129), (130, 131), (400, 512), (511, 385)]
    mats = [_grad(*sizes[i % len(sizes)], seed=i).bfloat16() for i in range(64)]
    on_gpu = [v.cuda() for v in mats]
    _lib.set_tuning("BMV_NS_BLOCK_K", 1)
    try:
        out, again = ops.newton_schulz(on_gpu), ops.newton_schulz(on_gpu)
    finally:
        _lib.set_tuning("BMV_NS_BLOCK_K", None)
    for got, twice, u in zip(out, again, mats):
        assert torch.equal(got, twice)
        _check(got, u)
    u = _grad(1500, 1450, 9).bfloat16()
    _check(ops.newton_schulz(u.cuda()), u)


@gpu
def test_newton_schulz_orthogonalises():
    """After enough steps of the classical cubic (1.5, -0.5, 0) the result is the orthogonal factor itself."""
    from boostmvsnerfs_amd import ops
    for m, n in ((24, 40), (40, 24), (140, 150)):
        u = _grad(m, n, 3, rank=min(m, n), noise=1.0)
        got = ops.newton_schulz(u.cuda(), steps=30, coeffs=(1.5, -0.5, 0.0)).double().cpu()
        U, _, V = torch.linalg.svd(u.double(), full_matrices=False)
        # the fixed point is stable (p'(1) = 0): what stays is one step's own error
        eps = 2.0 ** -24 * (4 + 2 * math.sqrt(max(m, n)))
        assert float((got - U @ V).norm()) <= 8 * eps * min(m, n), (m, n)


@gpu
def test_newton_schulz_steps_coefficients_and_lists():
    from boostmvsnerfs_amd import ops
    u = _grad(20, 30, 1)
    for steps in (1, 2, 3, 8):
        _check(ops.newton_schulz(u.cuda(), steps=steps), u, steps)
    _check(ops.newton_schulz(u.cuda(), coeffs=(2.0, -1.5, 0.5)), u, coeffs=(2.0, -1.5, 0.5))
    # a large eps damps: the norm does not count below it
    _check(ops.newton_schulz(u.cuda(), eps=10.0), u, eps=10.0)
    # more matrices than a launch's table holds, of mixed types, one of them a convolution kernel of other strides, one empty
    g = torch.Generator().manual_seed(4)
    mats = [torch.randn(1 + i % 9, 3 + 5 * (i % 7), generator=g).to((torch.float32, torch.bfloat16)[i % 2]) for i in range(90)]
    conv = torch.randn(16, 8, 3, 3, generator=g)
    on_gpu = [v.cuda() for v in mats] + [conv.cuda().to(memory_format=torch.channels_last), torch.empty(3, 0, device="cuda"),
                                         torch.randn(40, 50, generator=g).cuda().t()]
    out = ops.newton_schulz(on_gpu)
    for got, v in zip(out, mats):
        _check(got, v)
    _check(out[90].flatten(1), conv.flatten(1))
    assert out[91].shape == (3, 0)
    _check(out[92], on_gpu[92].cpu())
    assert ops.newton_schulz([]) == []


@gpu
def test_newton_schulz_zero_tiny_and_non_finite(way):
    from boostmvsnerfs_amd import ops
    u = _grad(24, 40, 2)
    mats = [u * 0, u * 1e-12, u * 1e-30, u * 1e12, u.clone(), u.clone(), u]
    mats[4][3, 5] = float("nan")
    mats[5][0, 0] = float("inf")
    out = ops.newton_schulz([v.cuda() for v in mats])
    assert not out[0].any()
    for k in (1, 2, 3, 6):
        _check(out[k], mats[k])
    assert out[4].isnan().all() and out[5].isnan().any()
    # (what is below eps is divided by eps: 1e-30 stays tiny, and finite)
    assert float(out[2].abs().max()) < 1e-18


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nesterov,scale,decay", [(True, "shape", 0.0), (False, "rms", 0.1), (True, "none", 0.01)])
def test_muon_step_matches_the_formula(dtype, nesterov, scale, decay, way):
    from boostmvsnerfs_amd import ops
    shapes = [(8, 27), (64, 24), (1, 12), (128, 63), (130, 140), (16, 8, 3, 3), (200, 40)]
    g = torch.Generator().manual_seed(11)
    lr, mu = 0.02, 0.9
    params = [torch.randn(s, generator=g).to(dtype) for s in shapes]
    momenta = [torch.zeros(s) for s in shapes]
    pg, mg = [p.cuda() for p in params], [m.cuda() for m in momenta]
    for it in range(3):
        grads = [torch.randn(s, generator=g).mul(0.1).to(dtype) for s in shapes]
        params, momenta = [p.cpu() for p in pg], [m.cpu() for m in mg]        # (every step from the state that is there)
        ops.muon_step(pg, [v.cuda() for v in grads], mg, lr, mu, nesterov, decay, scale)
        for p, gr, m, pn, mn in zip(params, grads, momenta, pg, mg):
            gd, md = gr.double(), m.double()
            moved = mu * md + (1 - mu) * gd
            # two products and a sum, with mu and 1 - mu rounded to fp32
            off = (mn.double().cpu() - moved).abs() - 4 * 2.0 ** -24 * ((mu * md).abs() + ((1 - mu) * gd).abs()) - 1e-40
            assert float(off.max()) <= 0, (tuple(p.shape), float(off.max()))
            u = ((1 - mu) * gd + mu * moved if nesterov else moved).flatten(1)
            o, tol = _iterate(u, two=dtype == torch.bfloat16)
            rows, cols = u.shape
            s = {"shape": math.sqrt(max(1, rows / cols)), "rms": 0.2 * math.sqrt(max(rows, cols)), "none": 1.0}[scale]
            want = p.double().flatten(1) * (1 - lr * decay) - lr * s * o
            # the iterate's tolerance, its input's (U is off by a few 2^-24 of |U|, which the steps can amplify as they do X's own
            # error: the tolerance begins with 2 x 2^-24 |X|, so four times as much again), and the roundings of the update
            u_out = torch.finfo(dtype).eps / 2
            lim = lr * s * 5 * tol + (u_out + 4 * 2.0 ** -24) * float(want.norm()) + 4 * 2.0 ** -24 * float(p.double().norm())
            if dtype == torch.float16:
                lim += 2.0 ** -25 * math.sqrt(want.numel())
            err = float((pn.double().cpu().flatten(1) - want).norm())
            assert err <= lim, (tuple(p.shape), err, lim)


@gpu
def test_muon_step_bumps_versions_and_takes_other_strides():
    from boostmvsnerfs_amd import ops
    g = torch.Generator().manual_seed(1)
    p0, gr = torch.randn(16, 8, 3, 3, generator=g).cuda(), torch.randn(16, 8, 3, 3, generator=g).cuda()
    pa, ma = p0.clone(), torch.zeros_like(p0)
    pb = p0.to(memory_format=torch.channels_last)
    mb = torch.zeros_like(pb)
    va, vb = pa._version, pb._version
    ops.muon_step([pa], [gr], [ma], 0.1)
    ops.muon_step([pb], [gr.to(memory_format=torch.channels_last)], [mb], 0.1)
    assert torch.equal(pa, pb) and torch.equal(ma, mb) and pa._version > va and pb._version > vb
    assert pb.is_contiguous(memory_format=torch.channels_last)
    # a saved weight that a step changed is noticed
    w = torch.nn.Parameter(p0[:, :, 0, 0].clone())
    y = (torch.randn(3, 8, device="cuda", requires_grad=True) @ w.t())
    ops.muon_step([w], [gr[:, :, 0, 0]], [torch.zeros_like(w)], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@gpu
def test_iterates_on_another_stream_and_in_a_graph():
    from boostmvsnerfs_amd import ops
    mats = [_grad(m, n, i).cuda() for i, (m, n) in enumerate([(8, 27), (128, 128), (140, 300)])]
    params, momenta = [torch.randn_like(v) for v in mats], [torch.zeros_like(v) for v in mats]
    want = [v.clone() for v in ops.newton_schulz(mats)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.newton_schulz(mats)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        out = ops.newton_schulz(mats)
    with torch.cuda.graph(g2):
        ops.muon_step(params, mats, momenta, 0.1, weight_decay=0.01)
    for k in range(3):
        for v in mats:
            v.mul_(1 + k).add_(1e-3)
        pe, me = [p.clone() for p in params], [m.clone() for m in momenta]
        want = [v.clone() for v in ops.newton_schulz(mats)]
        ops.muon_step(pe, mats, me, 0.1, weight_decay=0.01)
        torch.cuda.synchronize()
        g1.replay(), g2.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k
        assert all(torch.equal(a, b) for a, b in zip(params + momenta, pe + me)), k


def test_refusals():
    from boostmvsnerfs_amd import ops
    m = torch.zeros(4, 4)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.newton_schulz(m)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.muon_step([m], [m], [m], 0.1)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        ops.newton_schulz([m.double()])
    with pytest.raises(TypeError, match="expected a tensor"):
        ops.newton_schulz([3.0])
    with pytest.raises(ValueError, match="steps"):
        ops.newton_schulz(m, steps=0)
    with pytest.raises(ValueError, match="eps"):
        ops.newton_schulz(m, eps=0.0)
    with pytest.raises(ValueError, match="1 params, 2 grads"):
        ops.muon_step([m], [m, m], [m], 0.1)
    with pytest.raises(ValueError, match="scale"):
        ops.muon_step([m], [m], [m], 0.1, scale="other")
    with pytest.raises(ValueError, match="momentum"):
        ops.muon_step([m], [m], [m], 0.1, momentum=1.0)


def test_overlaps_are_refused_by_the_entry_points():
    """Checked on the host, in front of any launch: addresses that are never read."""
    import ctypes as C

    from boostmvsnerfs_amd import _lib
    lib = _lib.load()

    def ptrs(*v):
        return (C.c_void_p * len(v))(*v)
    rows, cols, one = (C.c_int * 2)(4, 4), (C.c_int * 2)(8, 8), (C.c_float * 2)(1, 1)
    A, B, G, M, N, W = 0x1000000, 0x2000000, 0x3000000, 0x4000000, 0x5000000, 0x6000000

    def step(p, g, m):
        return lib.bmv_muon_step(2, ptrs(*p), ptrs(*g), ptrs(*m), rows, cols, one, 0, 0.9, 1, 1.0, 5, *COEFFS, 1e-7, C.c_void_p(W), 1 << 40, None)
    for p, g, m in (((A, A), (G, G), (M, N)), ((A, A + 64), (G, G), (M, N)), ((A, B), (A, G), (M, N)), ((A, B), (G, G), (M, M)),
                    ((A, B), (G, G), (M, B)), ((A, B), (G, M + 4), (M, N))):
        assert step(p, g, m) == -1 and b"overlaps" in lib.bmv_last_error()
    assert lib.bmv_newton_schulz(2, ptrs(A, B), ptrs(G, A), rows, cols, 0, 5, *COEFFS, 1e-7, C.c_void_p(W), 1 << 40, None) == -1
    assert b"overlaps" in lib.bmv_last_error()
    assert lib.bmv_newton_schulz_workspace(1, (C.c_int * 1)(0), (C.c_int * 1)(4), 0) == -1
    need = lib.bmv_newton_schulz_workspace(2, rows, cols, 0)
    assert lib.bmv_newton_schulz(2, ptrs(A, B), ptrs(G, M), rows, cols, 0, 5, *COEFFS, 1e-7, C.c_void_p(W), need - 1, None) == -1
    assert b"too small" in lib.bmv_last_error()
    assert lib.bmv_newton_schulz(1, ptrs(A), ptrs(G), rows, cols, 7, 5, *COEFFS, 1e-7, C.c_void_p(W), 1 << 40, None) == -1


def test_strided_tensors_that_share_elements_are_found():
    """The host's check against marking every byte, for slices, permutations and windows of one storage."""
    from boostmvsnerfs_amd.ops import _written_twice

    def marked(tensors, size):
        seen = torch.zeros(size, dtype=torch.int32)
        base = tensors[0].untyped_storage().data_ptr()
        for t in tensors:
            at = torch.zeros(t.shape, dtype=torch.long) + (t.data_ptr() - base)
            for d, (s, n) in enumerate(zip(t.stride(), t.shape)):
                at = at + (torch.arange(n) * s * t.element_size()).view([-1 if k == d else 1 for k in range(t.dim())])
            for b in range(t.element_size()):
                seen.index_add_(0, at.flatten() + b, torch.ones(at.numel(), dtype=torch.int32))
        return bool((seen > 1).any())
    flat = torch.zeros(4096)
    wide = flat[:960].view(8, 120)
    half = flat.view(torch.bfloat16)
    cube = flat[:1920].view(4, 8, 6, 10)
    cases = [[wide[:, :40], wide[:, 40:]], [wide[:, :41], wide[:, 40:]], [wide[:, ::2], wide[:, 1::2]], [wide[:, ::2], wide[:, 1::3]],
             [wide[::2], wide[1::2]], [wide[:4].t(), wide[4:].t()], [wide[:5].t(), wide[4:].t()], [wide.t(), wide[3:4, 7:9]],
             [wide, flat[960:968].view(2, 4)], [wide, flat[959:967].view(2, 4)], [cube[:, :4], cube[:, 4:]],
             [cube.permute(0, 2, 3, 1)[:2], cube.permute(3, 2, 1, 0)[..., 2:]], [cube.permute(0, 2, 3, 1)[:3], cube.permute(3, 2, 1, 0)[..., 2:]],
             [cube[..., 0], cube[..., 9], cube[..., 4:6]], [cube[..., 0], cube[..., 5], cube[..., 4:6]],
             [wide[:, :40], half[80:160].view(8, 10)], [wide[:, 40:80], half[:80].view(8, 10)], [wide[:, :40], half[81:160]],
             [flat[:64].view(8, 8), flat[:64].view(8, 8).t()], [wide[:, 0:1], wide[:, 1:2]], [flat[:1].expand(4), wide[1:]], [flat[5:6].expand(2, 3)],
             [flat.as_strided((4, 4), (2, 1))], [flat.as_strided((4, 4), (4, 1)), flat.as_strided((4, 4), (4, 1), 16)]]
    found = [marked(c, 4 * 4096) for c in cases]
    assert [_written_twice(c) for c in cases] == found and 8 < sum(found) < 20
    g = torch.Generator().manual_seed(0)
    hits = 0
    for _ in range(300):                                     # two windows of one grid, at random
        pair = []
        for _ in range(2):
            (a, b), (c, d) = (sorted(torch.randint(0, 13, (2,), generator=g).tolist()) for _ in range(2))
            s, k = (int(torch.randint(1, 4, (1,), generator=g)) for _ in range(2))
            v = flat[:156].view(12, 13)[a:b + 1:s, c:d + 1:k]
            pair.append(v.t() if torch.randint(0, 2, (1,), generator=g) else v)
        want = marked(pair, 4 * 4096)
        hits += want
        assert _written_twice(pair) == want, [(v.shape, v.stride(), v.storage_offset()) for v in pair]
    assert 50 < hits < 250


@gpu
def test_muon_step_of_slices_of_one_tensor():
    """Column slices of one weight step as weights of their own where they are disjoint, and are refused where they are not."""
    from boostmvsnerfs_amd import ops
    g = torch.Generator().manual_seed(5)
    w, gr = torch.randn(12, 40, generator=g).cuda(), torch.randn(12, 40, generator=g).cuda()
    cut = [(0, 15), (15, 40)]
    want = [w[:, a:b].contiguous() for a, b in cut]
    kept, m0 = w.clone(), [torch.zeros_like(v) for v in want]
    ops.muon_step(want, [gr[:, a:b].contiguous() for a, b in cut], m0, 0.1)
    for cols, bad in ((cut, False), ([(0, 16), (15, 40)], True), ([(0, 40), (15, 20)], True)):
        w.copy_(kept)
        parts, grads = [w[:, a:b] for a, b in cols], [gr[:, a:b] for a, b in cols]
        momenta = [torch.zeros(v.shape, device="cuda") for v in parts]
        if bad:
            with pytest.raises(RuntimeError, match="overlaps"):
                ops.muon_step(parts, grads, momenta, 0.1)
            assert torch.equal(w, kept) and not any(m.any() for m in momenta)
        else:
            ops.muon_step(parts, grads, momenta, 0.1)
            assert all(torch.equal(a, b) for a, b in zip(parts + momenta, want + m0))
    # a weight that is one element many times, and a strided momentum over a dense weight
    one = torch.zeros(1, 4, device="cuda").expand(3, 4)
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.muon_step([one], [torch.ones(3, 4, device="cuda")], [torch.zeros(3, 4, device="cuda")], 0.1)
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.muon_step([w[:4]], [gr[:4]], [w.as_strided((4, 40), (80, 1))], 0.1)


@gpu
def test_refusals_on_the_gpu():
    from boostmvsnerfs_amd import ops
    m = torch.zeros(4, 4, device="cuda")
    with pytest.raises(ValueError, match="matrix"):
        ops.newton_schulz(m[0])
    with pytest.raises(ValueError, match=r"grads\[0\]"):
        ops.muon_step([m], [m.half()], [m], 0.1)
    with pytest.raises(ValueError, match=r"momenta\[0\]"):
        ops.muon_step([m], [m], [m.half()], 0.1)
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.muon_step([m, m], [m.clone(), m.clone()], [m.clone(), m.clone()], 0.1)
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.muon_step([m], [m], [m.clone()], 0.1)
    wide = torch.zeros(8, 4, device="cuda").t()                # (goes through a copy)
    for other in (wide, wide.t()):
        with pytest.raises(RuntimeError, match="overlaps"):
            ops.muon_step([wide, other], [wide.clone(), other.clone()], [torch.zeros_like(wide), torch.zeros_like(other)], 0.1)
