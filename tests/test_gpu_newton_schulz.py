"""GPU: orthogonalised updates (ops.orthogonalize) and the Muon step (optim.muon_step, optim.Muon) against the
same chain in 64 bits.

Tolerance, norm-wise (Frobenius), with e = 2^-22, what a pair of halves and a product of pairs without lo lo
keep, and s the largest singular value of a step's X.  A step p(X) = a X + b A X + c A A X rounds:
  A once in the product and once when it is split, relative to |X| |X|': taken as independent roundings that is
  2 e s |X| in norm, times |b| s after the product with X; c A A X takes A's two roundings twice and its own two;
  Q is split once, |Q| s <= (|a| + |b| s^2 + |c| s^4), the product Q X rounds once and X once more when it is split:
      delta = e |X| (3 |a| + (2 + 3) |b| s^2 + (6 + 3) |c| s^4)
An error passes through the following steps by at most L = max |p'| on [0, s] each (the divided differences of the
odd polynomial p).  tolerance = sum over the steps of delta times the later L, plus e for the first split of X; a
result of a 16-bit type adds half a step of it.  The sum is loose for small errors of early steps, so a test of
its own compares with the error of the fp32 chain."""
import copy
import math

import pytest
import torch

from dance_amd import config, modules, ops, optim, synthetic

pytestmark = pytest.mark.gpu

COEFF = (3.4445, -4.7750, 2.0315)


def _chain(m, steps=5, eps=1e-7, coeff=COEFF):
    """in m's type, on the CPU"""
    a, b, c = coeff
    x = m.t() if m.size(0) > m.size(1) else m
    x = x / max(float(x.double().norm()), eps)
    for _ in range(steps):
        g = x @ x.t()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.t() if m.size(0) > m.size(1) else x


def _norm_tolerance(m, want, dtype, steps=5, eps=1e-7, coeff=COEFF):
    a, b, c = coeff
    e = 2.0 ** -22
    x = m.t() if m.size(0) > m.size(1) else m
    x = x / max(float(x.norm()), eps)
    total = e * float(x.norm())
    for _ in range(steps):
        top = float(torch.linalg.matrix_norm(x, 2))
        grid = torch.linspace(0, top, 1001, dtype=torch.float64)
        slope = float((a + 3 * b * grid ** 2 + 5 * c * grid ** 4).abs().max())
        delta = e * float(x.norm()) * (3 * abs(a) + 5 * abs(b) * top ** 2 + 9 * abs(c) * top ** 4)
        total = slope * total + delta
        g = x @ x.t()
        x = a * x + (b * g + c * (g @ g)) @ x
    half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    return total + half * (float(want.norm()) + total) + 1e-30


def _check(got, m, dtype, what, **kw):
    """got (rows, columns) of the chain over m (fp64, CPU)"""
    want = _chain(m, **kw)
    off = float((got.detach().double().cpu() - want).norm())
    tol = _norm_tolerance(m, want, dtype, **kw)
    assert off <= tol, "%s: off by %.3g, tolerance %.3g" % (what, off, tol)


def _matrix(m, n, seed, kind="noise"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((m, n), generator=g)
    if kind == "gradient":                       # a few strong directions and noise, small in value
        k = min(4, m, n)
        x = (torch.randn((m, k), generator=g) @ torch.randn((k, n), generator=g) + 0.3 * x) * 1e-3
    return x


SHAPES = [(1, 1), (1, 288), (2, 64), (32, 9), (32, 288), (64, 256), (63, 65), (65, 63), (128, 1152), (127, 130),
          (256, 1024), (200, 333), (333, 200), (5, 700), (700, 5), (320, 2304), (64, 64), (129, 129)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize(device, shape, dtype):
    for seed, kind in ((1, "noise"), (2, "gradient")):
        x = _matrix(*shape, seed, kind).to(dtype)
        got = ops.orthogonalize(x.to(device))
        assert got.dtype == dtype and got.shape == x.shape and got.is_contiguous()
        _check(got, x.double(), dtype, "%s %s %s" % (shape, dtype, kind))


def test_as_accurate_as_the_fp32_chain(device):
    """pairs of halves carry 22 bits where fp32 carries 24: at most four times the fp32 chain's error, over matrices
    large enough that neither error is an accident"""
    for m, n in ((128, 1152), (256, 1024), (320, 320)):
        for seed, kind in ((21, "noise"), (22, "gradient")):
            x = _matrix(m, n, seed, kind)
            want = _chain(x.double())
            off32 = float((_chain(x).double() - want).norm())
            off = float((ops.orthogonalize(x.to(device)).double().cpu() - want).norm())
            assert off <= 4 * off32, (m, n, kind, off, off32)


def test_orthogonal_it_is(device):
    """singular values of a well conditioned matrix end where the coefficients put them"""
    for m, n in ((64, 256), (256, 64), (128, 1152)):
        s = torch.linalg.svdvals(ops.orthogonalize(_matrix(m, n, 3).to(device)).double().cpu())
        assert 0.65 < float(s.min()) and float(s.max()) < 1.25
    # the cubic chain of classical coefficients converges to the orthogonal factor itself
    x = _matrix(48, 80, 4)
    got = ops.orthogonalize(x.to(device), steps=30, coefficients=(1.5, -0.5, 0.0)).double().cpu()
    u, s, v = torch.linalg.svd(x.double(), full_matrices=False)
    # every singular value has converged; what is left is the last step's rounding, r products of 2^-22
    assert float((got - u @ v).abs().max()) < 48 * 2.0 ** -22 * 4


@pytest.mark.parametrize("shape", [(96, 150), (90, 100), (32, 500), (33, 34), (1, 3000), (16, 1500), (17, 17)])
def test_around_one_workgroup(device, shape):
    """sizes on both sides of what one workgroup keeps in its LDS, and of its 16 and 32 wide tiles"""
    for dtype in (torch.float32, torch.bfloat16):
        for x in (_matrix(*shape, 31).to(dtype), _matrix(*shape, 32, "gradient").to(dtype).t()):
            _check(ops.orthogonalize(x.to(device)), x.double(), dtype, "%s %s" % (tuple(x.shape), dtype))


@pytest.mark.parametrize("shape", [(100, 9000), (128, 20011), (20000, 65)])
def test_long_narrow(device, shape):
    """up to 128 rows and so many columns that a workgroup has several tiles of them; the Muon step too"""
    x = _matrix(*shape, 33)
    _check(ops.orthogonalize(x.to(device), steps=2), x.double(), torch.float32, str(shape), steps=2)
    p, g, m = (_matrix(*shape, 34 + i).to(device) for i in range(3))
    before = [(p.clone(), m.clone())]
    optim.muon_step([p], [g], [m], lr=0.1)
    _muon_check([p], [g], [m], before, torch.float32, 0.1, 0.95, True, 0.0, "long")


@pytest.mark.parametrize("batch,shape", [(2, (600, 5000)), (18, (600, 640)), (3, (1100, 1100))])
def test_enough_for_large_tiles(device, batch, shape):
    """batches whose products have tiles enough of 128 x 128 for the whole chip: the bits of single calls, whose tiles
    are of 64 x 64"""
    x = torch.stack([_matrix(*shape, 40 + i, "gradient" if i % 2 else "noise") for i in range(batch)])
    got = ops.orthogonalize(x.to(device), steps=2)
    for i in (0, batch - 1):
        assert torch.equal(ops.orthogonalize(x[i].to(device), steps=2), got[i]), i
    _check(got[batch - 1], x[batch - 1].double(), torch.float32, "%d of %s" % (batch, shape), steps=2)


def test_identities_to_the_bit(device):
    """a transposed matrix, a power of two, one of a batch, any strides: the same bits"""
    x = _matrix(96, 200, 5).to(device)
    got = ops.orthogonalize(x)
    assert torch.equal(ops.orthogonalize(x.t()), got.t())
    assert torch.equal(ops.orthogonalize(x * 2.0 ** 20), got) and torch.equal(ops.orthogonalize(x * 2.0 ** -10), got)
    others = torch.stack([_matrix(96, 200, 6 + i).to(device) for i in range(3)] + [x])
    assert torch.equal(ops.orthogonalize(others)[3], got)
    assert torch.equal(ops.orthogonalize(others.reshape(2, 2, 96, 200))[1, 1], got)
    many = x.expand(101, -1, -1)                 # more than one launch's items, a batch stride of zero
    out = ops.orthogonalize(many)
    assert torch.equal(out[0], got) and torch.equal(out[100], got) and torch.equal(out[57], got)
    wide = torch.zeros((96, 450), device=device)
    wide[:, 1:401:2] = x
    assert torch.equal(ops.orthogonalize(wide[:, 1:401:2]), got)
    for _ in range(3):
        assert torch.equal(ops.orthogonalize(x), got)


def test_scales_zero_and_not_finite(device):
    x = _matrix(40, 70, 7)
    for k in (1e-6, 1e12, 1e18, 1e30):           # squares that over- and underflow fp32
        _check(ops.orthogonalize((x * k).to(device)), (x * k).double(), torch.float32, "times %g" % k)
    # a norm below eps is not normalised away
    tiny = x * 1e-12
    _check(ops.orthogonalize(tiny.to(device)), tiny.double(), torch.float32, "below eps")
    assert not bool(ops.orthogonalize(torch.zeros((40, 70), device=device)).any())
    row = x.clone()
    row[3] = 0                                   # a row without an entry stays one
    assert not bool(ops.orthogonalize(row.to(device))[3].any())
    for bad in (float("nan"), float("inf")):
        batch = torch.stack([x, x])
        batch[1, 2, 3] = bad
        got = ops.orthogonalize(batch.to(device))
        assert bool(got[1].isnan().all()) and torch.equal(got[0], ops.orthogonalize(x.to(device)))


def test_steps_and_coefficients(device):
    x = _matrix(50, 90, 8)
    for kw in (dict(steps=1), dict(steps=2), dict(steps=8), dict(coeff=(2.0, -1.5, 0.5)), dict(steps=3, eps=50.0)):
        call = {("coefficients" if k == "coeff" else k): v for k, v in kw.items()}
        _check(ops.orthogonalize(x.to(device), **call), x.double(), torch.float32, str(kw), **kw)


def test_refusals(device):
    x = _matrix(8, 16, 9).to(device)
    for match, call in (("GPU tensors", lambda: ops.orthogonalize(x.cpu())),
                        (r"\(\.\.\., m, n\)", lambda: ops.orthogonalize(x[0])),
                        (r"\(\.\.\., m, n\)", lambda: ops.orthogonalize(x.double())),
                        ("steps", lambda: ops.orthogonalize(x, steps=0)),
                        ("steps", lambda: ops.orthogonalize(x, steps=2.5)),
                        ("steps", lambda: ops.orthogonalize(x, steps=101)),
                        ("eps", lambda: ops.orthogonalize(x, eps=0.0)),
                        ("eps", lambda: ops.orthogonalize(x, eps=float("nan"))),
                        ("coefficients", lambda: ops.orthogonalize(x, coefficients=(1.0, 2.0))),
                        ("coefficients", lambda: ops.orthogonalize(x, coefficients=(1.0, float("inf"), 0.0))),
                        ("not differentiable", lambda: ops.orthogonalize(x.clone().requires_grad_(True)))):
        with pytest.raises(RuntimeError, match=match):
            call()
    for shape in ((0, 8, 16), (3, 0, 16), (2, 8, 0), (0, 5)):
        assert ops.orthogonalize(torch.empty(shape, device=device)).shape == shape
    with torch.no_grad():
        assert not ops.orthogonalize(x.clone().requires_grad_(True)).requires_grad


def test_sizes_past_the_library_s_integers(device):
    """refused before anything is allocated or launched"""
    one = torch.zeros((1, 1), device=device)
    for big in (one.expand(2 ** 32, 1), one.expand(2 ** 16, 2 ** 15), one[None].expand(2 ** 31, 1, 1)):
        with pytest.raises(RuntimeError, match="2\\^31"):
            ops.orthogonalize(big)
    p, m = (torch.empty((2 ** 31, 1), device=device, dtype=torch.float16) for _ in range(2))
    with pytest.raises(RuntimeError, match="2\\^31"):
        optim.muon_step([p], [p], [m], lr=0.1)


# ------------------------------------------------------------------------------------------- Muon
def _muon_check(params, grads, buffers, before, dtype, lr, momentum, nesterov, weight_decay, what):
    """params, buffers after a step that started from `before`"""
    for p, g, m, (p0, m0) in zip(params, grads, buffers, before):
        rows = p.size(0)
        p64, g64, m64 = (t.detach().double().cpu().reshape(rows, -1) for t in (p0, g, m0))
        half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
        want_m = momentum * m64 + (1 - momentum) * g64
        tol = 4 * 2.0 ** -24 * (momentum * m64.abs() + (1 - momentum) * g64.abs()) + half * want_m.abs() + 2.0 ** -133
        if dtype == torch.float16:
            tol = tol + 2.0 ** -25
        assert bool(((m.detach().double().cpu().reshape(rows, -1) - want_m).abs() <= tol).all()), what + ": momentum"
        u = momentum * want_m + (1 - momentum) * g64 if nesterov else want_m
        o = _chain(u)
        step = lr * math.sqrt(max(1.0, rows / u.size(1)))
        want_p = p64 * (1 - lr * weight_decay) - step * o
        # the chain's error; three roundings of fp32; the momentum's rounding turned by the chain like its own first one
        tol = step * 2 * _norm_tolerance(u, o, torch.float32) + (3 * 2.0 ** -24 + half) * float(want_p.norm()) + 1e-12
        off = float((p.detach().double().cpu().reshape(rows, -1) - want_p).norm())
        assert off <= tol, "%s: parameter off by %.3g, tolerance %.3g" % (what, off, tol)


MIX = [(128, 258, 9), (128, 128, 9), (64, 256, 1), (2, 64, 1), (256, 256, 3, 3), (1, 32, 3, 3), (32, 1, 3, 3), (7, 3), (3, 7)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_muon_step(device, dtype):
    for nesterov, weight_decay in ((True, 0.0), (False, 0.1)):
        params = [_matrix(s[0], math.prod(s[1:]), i).reshape(s).mul(0.05).to(dtype).to(device) for i, s in enumerate(MIX)]
        grads = [_matrix(s[0], math.prod(s[1:]), 50 + i, "gradient").reshape(s).mul(30.0).to(dtype).to(device) for i, s in enumerate(MIX)]
        buffers = [_matrix(s[0], math.prod(s[1:]), 90 + i, "gradient").reshape(s).mul(30.0).to(dtype).to(device) for i, s in enumerate(MIX)]
        before = [(p.clone(), m.clone()) for p, m in zip(params, buffers)]
        kept = [g.clone() for g in grads]
        optim.muon_step(params, grads, buffers, lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=weight_decay)
        _muon_check(params, grads, buffers, before, dtype, 0.02, 0.9, nesterov, weight_decay, str((dtype, nesterov)))
        assert all(torch.equal(a, b) for a, b in zip(kept, grads))


def test_muon_more_matrices_than_a_launch_takes(device):
    params = [_matrix(16 + i % 3, 40, i).to(device) for i in range(100)]
    grads = [_matrix(16 + i % 3, 40, 200 + i).to(device) for i in range(100)]
    buffers = [torch.zeros_like(p) for p in params]
    before = [(p.clone(), m.clone()) for p, m in zip(params, buffers)]
    optim.muon_step(params, grads, buffers, lr=0.1)
    _muon_check(params, grads, buffers, before, torch.float32, 0.1, 0.95, True, 0.0, "100 matrices")


def test_muon_memory_layouts(device):
    """channels_last weights stay as they are laid out; a gradient of other strides is copied; views of one flat
    storage at any element alignment; what lies around them is left alone"""
    w = _matrix(24, 45, 1).reshape(24, 5, 3, 3).to(device)
    g = _matrix(24, 45, 2).reshape(24, 5, 3, 3).to(device)
    one, grad_cl = w.clone(), g.to(memory_format=torch.channels_last)
    two = w.to(memory_format=torch.channels_last).clone(memory_format=torch.preserve_format)
    m1, m2 = torch.zeros_like(one), torch.zeros_like(two, memory_format=torch.preserve_format)
    before = [(one.clone(), m1.clone())]
    optim.muon_step([one], [grad_cl], [m1], lr=0.1)
    optim.muon_step([two], [g], [m2], lr=0.1)
    assert not two.is_contiguous() and m2.stride() == two.stride()
    for p, m in ((one, m1), (two, m2)):
        _muon_check([p], [g], [m], before, torch.float32, 0.1, 0.95, True, 0.0, "layout")
    for dtype in (torch.float32, torch.bfloat16):
        flat = torch.full((3, 1000), 7.0, device=device, dtype=dtype)
        sizes = [(3, 7), (5, 11), (9, 4)]
        views, at = [[], [], []], 1
        for i, s in enumerate(sizes):
            for k in range(3):
                v = flat[k, at:at + s[0] * s[1]].view(s)
                v.copy_(_matrix(*s, 10 * i + k))
                views[k].append(v)
            at += s[0] * s[1] + 1
        before = [(p.clone(), m.clone()) for p, m in zip(views[0], views[2])]
        optim.muon_step(views[0], views[1], views[2], lr=0.1)
        _muon_check(views[0], views[1], views[2], before, dtype, 0.1, 0.95, True, 0.0, "views")
        at = 0
        for s in sizes:
            assert bool((flat[:, at] == 7.0).all())
            at += s[0] * s[1] + 1
        assert bool((flat[:, at:] == 7.0).all())


def test_muon_refusals(device):
    p = torch.zeros((4, 6), device=device)
    z = torch.zeros_like
    for match, call in (
            ("GPU tensors", lambda: optim.muon_step([p.cpu()], [z(p).cpu()], [z(p).cpu()], lr=0.1)),
            ("1 params, 0 grads", lambda: optim.muon_step([p], [], [z(p)], lr=0.1)),
            ("matrices", lambda: optim.muon_step([p[0]], [z(p[0])], [z(p[0])], lr=0.1)),
            ("matrices", lambda: optim.muon_step([p.double()], [z(p)], [z(p)], lr=0.1)),
            ("a gradient", lambda: optim.muon_step([p], [z(p).half()], [z(p)], lr=0.1)),
            ("a gradient", lambda: optim.muon_step([p], [z(p)[:2]], [z(p)], lr=0.1)),
            ("a momentum buffer", lambda: optim.muon_step([p], [z(p)], [torch.zeros((6, 4), device=device)], lr=0.1)),
            ("equal strides", lambda: optim.muon_step([p], [z(p)], [torch.zeros((6, 4), device=device).t()], lr=0.1)),
            ("rows outermost", lambda: optim.muon_step([p.t()], [z(p).t()], [z(p).t()], lr=0.1)),
            ("rows outermost", lambda: optim.muon_step([p[:, ::2]], [z(p)[:, ::2]], [z(p)[:, ::2]], lr=0.1)),
            ("appears twice", lambda: optim.muon_step([p, p], [z(p), z(p)], [z(p), z(p)], lr=0.1)),
            ("steps", lambda: optim.muon_step([p], [z(p)], [z(p)], lr=0.1, steps=0)),
            ("requirement failed", lambda: optim.muon_step([p], [z(p)], [z(p)], lr=float("nan")))):
        with pytest.raises(RuntimeError, match=match):
            call()
    assert not bool(p.any())
    optim.muon_step([], [], [], lr=0.1)
    optim.muon_step([torch.zeros((0, 4), device=device)], [torch.zeros((0, 4), device=device)], [torch.zeros((0, 4), device=device)], lr=0.1)
    for bad in (lambda: optim.Muon([torch.zeros(3, requires_grad=True)]), lambda: optim.Muon([p], lr=-1.0),
                lambda: optim.Muon([p], momentum=1.0), lambda: optim.Muon([p], weight_decay=-0.1)):
        with pytest.raises(ValueError):
            bad()


def test_muon_optimizer(device):
    """torch.optim's manners: groups, parameters without a gradient, state_dict, closures, versions"""
    a, b, c = (torch.nn.Parameter(_matrix(*s, i).to(device)) for i, s in enumerate(((12, 30), (40, 8), (6, 6))))
    opt = optim.Muon([dict(params=[a], lr=0.5), dict(params=[b, c], weight_decay=0.2)], lr=0.1, momentum=0.8)
    a.grad, b.grad = _matrix(12, 30, 5).to(device), _matrix(40, 8, 6).to(device)
    was = [t.detach().clone() for t in (a, b, c)]
    version = a._version
    assert opt.step(lambda: 3.0) == 3.0
    assert a._version > version and torch.equal(c, was[2]) and c not in opt.state
    zeros = [torch.zeros_like(t) for t in (a, b)]
    for t, w, z, lr, wd in ((a, was[0], zeros[0], 0.5, 0.0), (b, was[1], zeros[1], 0.1, 0.2)):
        _muon_check([t], [t.grad], [opt.state[t]["momentum_buffer"]], [(w, z)], torch.float32, lr, 0.8, True, wd, "optimizer")
    # a saved and loaded optimizer goes on the same way
    a2, b2, c2 = (torch.nn.Parameter(t.detach().clone()) for t in (a, b, c))
    other = optim.Muon([dict(params=[a2]), dict(params=[b2, c2])])
    other.load_state_dict(copy.deepcopy(opt.state_dict()))     # (a shallow one shares its tensors with opt)
    a2.grad, b2.grad = a.grad.clone(), b.grad.clone()
    opt.step()
    other.step()
    assert torch.equal(a, a2) and torch.equal(b, b2)
    # a tensor saved for a backward pass and changed by the step is noticed
    y = (a * a).sum()
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_optimizer_step_captured(device):
    """refused before the momentum buffers exist (a replay would clear them); afterwards replays are eager steps"""
    weights = [[torch.nn.Parameter(_matrix(*s, i).to(device)) for i, s in enumerate(((40, 70), (150, 160)))] for _ in range(2)]
    opts = [optim.Muon(w, lr=0.1, weight_decay=0.1) for w in weights]
    for w in weights:
        for i, p in enumerate(w):
            p.grad = _matrix(*p.shape, 10 + i).to(device)
    fresh = optim.Muon([torch.nn.Parameter(weights[0][0].detach().clone())])
    fresh.param_groups[0]["params"][0].grad = weights[0][0].grad.clone()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before the one that is captured"):
        with torch.cuda.graph(graph):
            fresh.step()
    for opt in opts:
        opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opts[0].step()
    for turn in range(4):
        for w in weights:
            for i, p in enumerate(w):
                p.grad.copy_(_matrix(*p.shape, 20 + 2 * turn + i).to(device))
        graph.replay()
        opts[1].step()
        torch.cuda.synchronize()
        for a, b in zip(*weights):
            assert torch.equal(a, b) and torch.equal(opts[0].state[a]["momentum_buffer"], opts[1].state[b]["momentum_buffer"]), turn


def test_inference_tensors(device):
    """made under inference_mode, they carry no version"""
    with torch.inference_mode():
        p, g, m = (_matrix(30, 50, i).to(device) for i in range(3))
        before = [(p.clone(), m.clone())]
        optim.muon_step([p], [g], [m], lr=0.1)
        _muon_check([p], [g], [m], before, torch.float32, 0.1, 0.95, True, 0.0, "inference")
        assert ops.orthogonalize(g).is_inference() and ops.group_norm_act(g, 5).is_inference()


def test_modules_repack_after_a_step(device):
    """the heads cache weights packed for their kernels; a step on them must be seen"""
    cfg = config.dance_r50(num_sampling=128, num_convs=2)
    net = modules.RefineNet(cfg)
    synthetic.fill_state_dict_(net.state_dict(), 3)
    net = net.to(device).eval()
    feats = synthetic.make_smooth_features(1, 256, 24, 32, 5).to(device)
    with torch.no_grad():
        first = net._features(feats)[1].clone()
        packed = net._packed
        weights = [p for p in net.parameters() if p.dim() >= 2]
        for i, p in enumerate(weights):
            p.grad = torch.randn(p.shape, generator=torch.Generator().manual_seed(i)).to(device)
        optim.Muon(weights, lr=0.01).step()
        second = net._features(feats)[1]
    assert net._packed is not packed and not torch.equal(first, second)


def test_streams_and_captured_graphs(device):
    """on a stream of its own beside another call, and captured: replayed steps on changing gradients equal eager ones"""
    x = _matrix(128, 300, 11).to(device)
    want = ops.orthogonalize(x)
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        first = ops.orthogonalize(x)
    second = ops.orthogonalize(x)
    torch.cuda.current_stream(device).wait_stream(side)
    assert torch.equal(first, want) and torch.equal(second, want)
    params = [_matrix(*s, i).to(device) for i, s in enumerate(((64, 200), (20, 30), (150, 40)))]
    grads, buffers = [torch.zeros_like(p) for p in params], [torch.zeros_like(p) for p in params]
    eager = [[t.clone() for t in ts] for ts in (params, grads, buffers)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        optim.muon_step(params, grads, buffers, lr=0.1)
    for seed in (1, 2, 3, 4):
        for i, (g, e) in enumerate(zip(grads, eager[1])):
            new = _matrix(*g.shape, 100 * seed + i).to(device)
            g.copy_(new)
            e.copy_(new)
        graph.replay()
        optim.muon_step(*eager, lr=0.1)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(params + buffers, eager[0] + eager[2])), seed


BOTH = [(64, 200), (150, 140), (20, 30), (200, 9, 3, 3), (128, 700), (300, 301), (257, 129)]


@pytest.mark.parametrize("repeat", [1, 9])
def test_narrow_and_wide_matrices_beside_each_other(device, repeat):
    """both sides of 128 rows in one step, which then runs on two streams; also more of each than one launch takes.  Each
    matrix gets the bits it has alone, but for the two that alone fit one workgroup's LDS, where the order of the sums
    is another (_muon_check holds for all)"""
    shapes = BOTH * repeat + [(140, 150)] * (repeat * repeat // 2)
    def lists():
        return [[_matrix(s[0], math.prod(s[1:]), 1000 * k + i).reshape(s).to(device) for i, s in enumerate(shapes)] for k in range(3)]
    params, grads, buffers = lists()
    optim.muon_step(params, grads, buffers, lr=0.1)
    alone = lists()
    before = [(p.clone(), m.clone()) for p, m in zip(alone[0], alone[2])]
    for i in range(len(shapes)):
        optim.muon_step(*[[t[i]] for t in alone], lr=0.1)
    for i, s in enumerate(shapes):
        assert s in ((20, 30), (64, 200)) or torch.equal(params[i], alone[0][i]), (i, s)
        assert torch.equal(buffers[i], alone[2][i]), (i, s)
    _muon_check(params[:7], grads, buffers, before, torch.float32, 0.1, 0.95, True, 0.0, "both")


@pytest.mark.parametrize("narrow,wide", [(60, 3), (3, 60), (100, 50)])
def test_many_of_one_kind_beside_few_of_the_other(device, narrow, wide):
    """the launches of one kind reuse their part of the workspace while the other kind's may still run"""
    shapes = [(100, 300 + i % 3) for i in range(narrow)] + [(400, 500 + i % 2) for i in range(wide)]
    def lists():
        return [[_matrix(*s, 1000 * k + i).to(device) for i, s in enumerate(shapes)] for k in range(3)]
    params, grads, buffers = lists()
    alone = lists()
    for _ in range(3):
        optim.muon_step(params, grads, buffers, lr=0.1)
    for _ in range(3):
        optim.muon_step(*[t[:narrow] for t in alone], lr=0.1)
        optim.muon_step(*[t[narrow:] for t in alone], lr=0.1)
    assert all(torch.equal(a, b) for a, b in zip(params + buffers, alone[0] + alone[2]))


def test_captured_on_two_streams(device):
    """the fork into the step's own stream and the join are part of a captured graph; two graphs and eager steps in turn,
    captured and replayed on a stream of the caller's"""
    def state():
        return [[_matrix(s[0], math.prod(s[1:]), 100 * k + i).reshape(s).to(device) for i, s in enumerate(BOTH)] for k in range(3)]
    captured, eager = [state(), state()], [state(), state()]
    stream = torch.cuda.Stream(device)
    graphs = [torch.cuda.CUDAGraph() for _ in captured]
    for graph, s in zip(graphs, captured):
        stream.wait_stream(torch.cuda.current_stream(device))
        with torch.cuda.graph(graph, stream=stream):
            optim.muon_step(*s, lr=0.1)
    for turn in range(4):
        for k in (0, 1):
            for a, b in zip(captured[k][1], eager[k][1]):
                new = _matrix(a.size(0), a.numel() // a.size(0), 10000 * turn + a.numel() + k).reshape(a.shape).to(device)
                a.copy_(new)
                b.copy_(new)
            stream.wait_stream(torch.cuda.current_stream(device))
            with torch.cuda.stream(stream):
                graphs[k].replay()
            optim.muon_step(*eager[k], lr=0.1)
            torch.cuda.synchronize()
        for k in (0, 1):
            assert all(torch.equal(a, b) for a, b in zip(captured[k][0] + captured[k][2], eager[k][0] + eager[k][2])), (turn, k)


def test_a_failing_step_is_joined(device):
    """an error from the library is raised with the step's own stream joined, and the next step is right"""
    params, grads, buffers = ([_matrix(s[0], math.prod(s[1:]), 100 * k + i).reshape(s).to(device) for i, s in enumerate(BOTH[:2])]
                              for k in range(3))
    kept = [p.clone() for p in params]
    with pytest.raises(RuntimeError, match="requirement failed"):
        optim.muon_step(params, grads, buffers, lr=float("nan"))
    assert all(torch.equal(a, b) for a, b in zip(params, kept))
    before = [(p.clone(), m.clone()) for p, m in zip(params, buffers)]
    optim.muon_step(params, grads, buffers, lr=0.1)
    _muon_check(params, grads, buffers, before, torch.float32, 0.1, 0.95, True, 0.0, "after an error")


def test_training_a_norm_layer_stack(device):
    """the operators as they are used together: conv -> group norm + activation layers, backward, Muon on the
    convolutions; parameters after the step against the formulas in 64 bits"""
    g = torch.Generator().manual_seed(7)
    convs = [torch.nn.Conv2d(ci, co, 3, padding=1, bias=False).to(device).to(memory_format=torch.channels_last)
             for ci, co in ((16, 32), (32, 32))]
    for conv in convs:
        with torch.no_grad():
            conv.weight.copy_(torch.randn(conv.weight.shape, generator=g) * 0.1)
    affine = [(torch.ones(32, device=device, requires_grad=True), torch.zeros(32, device=device, requires_grad=True)) for _ in convs]
    x = torch.randn((2, 16, 20, 24), generator=g).to(device).to(memory_format=torch.channels_last)

    def forward(norm):
        y = x
        for conv, (w, b) in zip(convs, affine):
            y = norm(conv(y), w, b)
        return (y * y).mean()

    leaves = [c.weight for c in convs] + [t for pair in affine for t in pair]
    got = torch.autograd.grad(forward(lambda y, w, b: ops.group_norm_act(y.contiguous(memory_format=torch.channels_last), 8, w, b)), leaves)
    want = torch.autograd.grad(forward(lambda y, w, b: torch.relu(torch.nn.functional.group_norm(y, 8, w, b))), leaves)
    for a, b in zip(got, want):
        # both are fp32 passes over the same sums of 2 * 480 pixels: each within (960 u + a few) of the magnitudes
        assert float((a - b).norm()) <= 1e-4 * float(b.norm())
    opt = optim.Muon([c.weight for c in convs], lr=0.05)
    before = [(c.weight.detach().clone(memory_format=torch.preserve_format), torch.zeros_like(c.weight)) for c in convs]
    for c, d in zip(convs, got):
        c.weight.grad = d
    opt.step()
    # (columns in logical order on both sides)
    _muon_check([c.weight.contiguous() for c in convs], [c.weight.grad.contiguous() for c in convs],
                [opt.state[c.weight]["momentum_buffer"].contiguous() for c in convs],
                [(p.contiguous(), m.contiguous()) for p, m in before], torch.float32, 0.05, 0.95, True, 0.0, "stack")


def test_optimizer_state_of_another_memory_format(device):
    """a state saved from contiguous weights carries on with channels_last ones"""
    g = torch.Generator().manual_seed(77)
    shape = (48, 20, 3, 3)
    start, grads = torch.randn(shape, generator=g), [torch.randn(shape, generator=g).to(device) for _ in range(3)]
    p = torch.nn.Parameter(start.to(device))
    opt = optim.Muon([p], lr=0.05)
    p.grad = grads[0]
    opt.step()
    q = torch.nn.Parameter(p.detach().to(memory_format=torch.channels_last))
    other = optim.Muon([q], lr=0.05)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    for grad in grads[1:]:
        before = [(q.detach().clone(), other.state[q]["momentum_buffer"].clone())]
        p.grad = q.grad = grad
        opt.step()
        other.step()
        _muon_check([q], [grad], [other.state[q]["momentum_buffer"]], before, torch.float32, 0.05, 0.95, True, 0.0, "loaded")
    m, n = opt.state[p]["momentum_buffer"], other.state[q]["momentum_buffer"]
    assert n.stride() == q.stride() != p.stride() and torch.equal(m, n)
