"""GPU: group norm with an activation on channels-last maps (ops.group_norm_act) and its gradients, against
the same formulas in 64 bits and, for the gradients, against differences of them.

Tolerances (u = 2^-24, half a step of fp32).  The statistics are fp64, so xh = ((x - mhi) - mlo) rstd carries
two subtractions, the rounding of rstd and a product: 4u.  z = fma(xh, w, beta) adds u |z|:
    |dz| <= 5u (|xh w| + |beta|), taken as 6u.
SiLU: its slope is at most 1.1; the exponential's argument and its own error give (|z| + 4) u on the sigmoid,
two more operations u each.  Gradients: sums in fp32 of at most N_T terms a thread (chunks of 8 pixels a
thread at these sizes) and a tree above them, so a sum is off by at most (N_T + 10) u of the sum of
magnitudes.  On top comes half a step of the output's type."""
import pytest
import torch
import torch.utils.checkpoint

from dance_amd import modules, ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
N_T = 32
SMALLEST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def _oracle(x, groups, weight, bias, act, dy=None, eps=1e-5):
    """{name: (value, tolerance)} in fp64; x (B, C, *spatial)"""
    b, c = x.shape[:2]
    shape = x.shape
    x = x.detach().double().reshape(b, c, -1)
    one = lambda t, v: (torch.full((c,), v, dtype=torch.float64, device=x.device) if t is None else t.detach().double())[None, :, None]
    w, be = one(weight, 1.0), one(bias, 0.0)
    gx = x.reshape(b, groups, -1)
    mean = gx.mean(2, keepdim=True)
    var = ((gx - mean) ** 2).mean(2, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xh = ((gx - mean) * rstd).reshape(x.shape)
    z = xh * w + be
    tz = 6 * U * ((xh * w).abs() + be.abs())
    s = torch.sigmoid(z)
    if act == "relu":
        y, ty = torch.where(z > 0, z, torch.where(z.isnan(), z, torch.zeros_like(z))), tz
    elif act == "silu":
        y, ty = z * s, 1.1 * tz + (z * s).abs() * (z.abs() + 6) * U
    else:
        y, ty = z, tz
    out = {"y": (y.reshape(shape), ty.reshape(shape))}
    if dy is None:
        return out
    dy = dy.detach().double().reshape(x.shape)
    if act == "relu":
        dz, tdz = dy * (z > 0), torch.zeros_like(z)
    elif act == "silu":
        dz = dy * (s + z * s * (1 - s))
        tdz = dy.abs() * (0.5 * tz + 1.2 * (z.abs() + 8) * U)
    else:
        dz, tdz = dy, torch.zeros_like(z)

    def per_group(t):
        return t.reshape(b, groups, -1).mean(2, keepdim=True).expand(b, groups, gx.size(2)).reshape(x.shape)

    r = rstd.expand_as(gx).reshape(x.shape)
    wdz = dz * w
    m1, m2 = per_group(wdz), per_group(wdz * xh)
    dx = r * (wdz - m1 - xh * m2)
    sums = (N_T + 10) * U
    twdz = tdz * w.abs()
    tdx = r * (twdz + per_group(twdz) + xh.abs() * per_group(twdz * xh.abs()) + 4 * U * (wdz.abs() + m1.abs())
               + 9 * U * (xh * m2).abs() + sums * per_group(wdz.abs())
               + xh.abs() * (sums + 5 * U) * per_group((wdz * xh).abs())) + 2 * U * dx.abs()
    out["dx"] = (dx.reshape(shape), tdx.reshape(shape))
    out["dweight"] = ((dz * xh).sum((0, 2)), ((sums + 5 * U) * (dz * xh).abs() + tdz * xh.abs()).sum((0, 2)))
    out["dbias"] = (dz.sum((0, 2)), (sums * dz.abs() + tdz).sum((0, 2)))
    return out


def _check(got, want, what):
    value, tol = want
    assert got.shape == value.shape, what
    tol = tol + torch.finfo(got.dtype).eps / 2 * (value.abs() + tol) + SMALLEST[got.dtype]
    off = (got.detach().double() - value).abs()
    assert torch.equal(got.isnan(), value.isnan()), what + ": NaNs elsewhere"
    bad = (off > tol) & ~value.isnan()
    assert not bool(bad.any()), "%s: %d values off, worst %.3g of the tolerance" % (
        what, int(bad.sum()), float((off / tol.clamp_min(1e-300)).nan_to_num().max()))


def _map(shape, dtype, device, seed, mean=0.5):
    """a channels-last map, every channel with a mean and a spread of its own"""
    g = torch.Generator().manual_seed(seed)
    b, c = shape[:2]
    t = torch.randn((b,) + tuple(shape[2:]) + (c,), generator=g) * (0.5 + torch.rand((c,), generator=g))
    return (t + mean * torch.randn((c,), generator=g)).to(dtype).to(device).movedim(-1, 1)


def _affine(c, dtype, device, seed):
    g = torch.Generator().manual_seed(1000 + seed)
    return ((1 + 0.2 * torch.randn((c,), generator=g)).to(dtype).to(device),
            (0.2 * torch.randn((c,), generator=g)).to(dtype).to(device))


SHAPES = [((1, 256, 25, 38), 32), ((2, 256, 7, 9), 32), ((1, 1, 1, 2), 1), ((3, 96, 13, 17), 32), ((2, 5, 3, 41), 1),
          ((2, 7, 8, 8), 7), ((1, 64, 1, 1), 4), ((4, 24, 2, 3), 8), ((2, 260, 5, 5), 5), ((1, 1024, 3, 3), 32),
          ((1, 2046, 2, 2), 2), ((2, 33, 61), 3), ((6, 48), 4), ((1, 16, 5, 4, 3), 4), ((1, 8, 90, 91), 8)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_forward_and_gradients(device, shape, groups, dtype):
    for i, act in enumerate(("relu", "silu", None)):
        x = _map(shape, dtype, device, 7 + i).requires_grad_(True)
        w, be = _affine(shape[1], (torch.float32, dtype)[i % 2], device, i)
        w.requires_grad_(True)
        be.requires_grad_(True)
        dy = _map(shape, dtype, device, 70 + i)
        with torch.no_grad():
            alone = ops.group_norm_act(x, groups, w, be, act=act)
        y = ops.group_norm_act(x, groups, w, be, act=act)
        assert torch.equal(y, alone) and y.dtype == dtype and ops._channels_last_strides(y) is not None
        dx, dw, db = torch.autograd.grad(y, (x, w, be), dy)
        assert dx.dtype == dtype and dw.dtype == w.dtype and db.dtype == be.dtype
        want = _oracle(x, groups, w, be, act, dy)
        for name, got in (("y", y), ("dx", dx), ("dweight", dw), ("dbias", db)):
            _check(got, want[name], "%s %s %s %s" % (shape, dtype, act, name))


def test_memory_layouts(device):
    """what is read in place (channel and batch slices, an expanded batch), what is copied (a crop), the
    values the same in every case"""
    base = _map((4, 40, 12, 10), torch.float32, device, 3)
    w, be = _affine(24, torch.float32, device, 3)
    for what, x in (("channel slice", base[:, 9:33]), ("batch slice", base[1::2, :24]), ("crop", base[:, :24, 2:9, 1:8]),
                    ("expanded batch", base[:1, 3:27].expand(3, -1, -1, -1)), ("rows", base[:, :24, 4:7])):
        y = ops.group_norm_act(x, 6, w, be)
        _check(y, _oracle(x, 6, w, be, "relu")["y"], what)
        dense = x.permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2)
        assert torch.equal(ops.group_norm_act(dense, 6, w, be), y), what
        # the gradient's memory in any layout as well: dense NCHW, an expanded scalar
        xr = x.detach().requires_grad_(True)
        dy = torch.randn(x.shape, device=device)
        for d in (dy, dy[:1, :1, :1, :1].expand(x.shape), dy.permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2)):
            dx, = torch.autograd.grad(ops.group_norm_act(xr, 6, w, be), xr, d)
            _check(dx, _oracle(x, 6, w, be, "relu", d)["dx"], what + " dx")
    one = torch.zeros(1, device=device)                   # weights that are strided views
    y = ops.group_norm_act(base[:, :24], 6, torch.stack([w, w], 1)[:, 0], one.expand(24))
    assert torch.equal(y, ops.group_norm_act(base[:, :24], 6, w, torch.zeros(24, device=device)))


def test_unaligned_maps(device):
    """pixels and bases that are not 16-byte aligned, every type, and odd channel counts behind them"""
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        buf = torch.randn((2, 9, 11, 65), device=device).to(dtype)
        for lo, c, groups in ((1, 64, 8), (3, 40, 5), (1, 63, 7), (2, 9, 3)):
            x = buf.permute(0, 3, 1, 2)[:, lo:lo + c]
            w, be = _affine(c, torch.float32, device, c)
            xr = x.detach().requires_grad_(True)
            y = ops.group_norm_act(xr, groups, w, be, act="silu")
            dy = torch.randn((2, 9, 11, c + 1), device=device).to(dtype)[..., 1:].permute(0, 3, 1, 2)
            dx, = torch.autograd.grad(y, xr, dy)
            want = _oracle(x, groups, w, be, "silu", dy)
            _check(y, want["y"], "y")
            _check(dx, want["dx"], "dx")


def test_means_far_from_the_spread(device):
    """a mean ten thousand times the spread: the variance must not cancel, x - mean must keep its bits"""
    g = torch.Generator().manual_seed(1)
    x = (1.0e4 + torch.randn((2, 16, 16, 32), generator=g)).to(device).permute(0, 3, 1, 2)
    w, be = _affine(32, torch.float32, device, 1)
    xr = x.detach().requires_grad_(True)
    y = ops.group_norm_act(xr, 4, w, be)
    dy = torch.randn(x.shape, device=device)
    dx, = torch.autograd.grad(y, xr, dy)
    want = _oracle(x, 4, w, be, "relu", dy)
    _check(y, want["y"], "y")
    _check(dx, want["dx"], "dx")
    # groups without any spread: xh = 0, y = act(beta)
    flat = torch.full((1, 4, 4, 8), 3.25, device=device).permute(0, 3, 1, 2)
    y = ops.group_norm_act(flat, 2, *_affine(8, torch.float32, device, 2), act=None)
    assert torch.equal(y, _affine(8, torch.float32, device, 2)[1][None, :, None, None].expand_as(y))


def test_relu_gradient_at_the_border(device):
    """z exactly zero (beta = 0 at the group's mean) has no gradient; z next to zero goes by its fp64 sign"""
    x = torch.tensor([-2.0, -1.0, 0.0, 1.0, 2.0], device=device).reshape(1, 1, 5).requires_grad_(True)
    y = ops.group_norm_act(x, 1)
    dy = torch.ones_like(y)
    want = _oracle(x, 1, None, None, "relu", dy)
    dx, = torch.autograd.grad(y, x, dy)
    _check(dx, want["dx"], "dx")
    # beta cancels the second-largest value's term to fp32 rounding: both signs of z there
    g = torch.Generator().manual_seed(5)
    for k in range(16):
        xk = torch.randn((1, 64, 1), generator=g).to(device)
        x64 = xk.double().flatten()
        xh = (x64 - x64.mean()) / torch.sqrt(((x64 - x64.mean()) ** 2).mean() + 1e-5)
        be = (-xh).float()                                 # z = xh + rn(-xh): a rounding error, either sign
        xk.requires_grad_(True)
        dx, = torch.autograd.grad(ops.group_norm_act(xk, 1, None, be), xk, torch.ones_like(xk))
        _check(dx, _oracle(xk, 1, None, be, "relu", torch.ones_like(xk))["dx"], "border %d" % k)


def test_nan_and_infinities_stay_in_their_group(device):
    for bad in (float("nan"), float("inf"), -float("inf")):
        x = _map((2, 16, 6, 6), torch.float32, device, 5)
        x[1, 5, 3, 3] = bad
        for act in ("relu", "silu", None):
            y = ops.group_norm_act(x, 4, act=act)
            assert bool(y[1, 4:8].isnan().all())
            y[1, 4:8] = 0
            assert bool(y.isfinite().all())


def test_parts_that_are_not_wanted(device):
    x = _map((2, 12, 5, 5), torch.float32, device, 6)
    w, be = _affine(12, torch.float32, device, 6)
    dy = _map((2, 12, 5, 5), torch.float32, device, 8)
    for mask in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 1, 0)):
        leaves = [t.detach().clone(memory_format=torch.preserve_format).requires_grad_(bool(m)) for t, m in zip((x, w, be), mask)]
        y = ops.group_norm_act(leaves[0], 3, leaves[1], leaves[2], act="silu")
        y.backward(dy)
        want = _oracle(x, 3, w, be, "silu", dy)
        for t, m, name in zip(leaves, mask, ("dx", "dweight", "dbias")):
            assert (t.grad is not None) == bool(m)
            if m:
                _check(t.grad, want[name], name)
    # no affine parameters, one of them, and an eps of its own
    for ww, bb in ((None, None), (w, None), (None, be)):
        xr = x.detach().requires_grad_(True)
        y = ops.group_norm_act(xr, 3, ww, bb, eps=0.25)
        dx, = torch.autograd.grad(y, xr, dy)
        want = _oracle(x, 3, ww, bb, "relu", dy, eps=0.25)
        _check(y, want["y"], "y")
        _check(dx, want["dx"], "dx")


def test_gradients_against_differences(device):
    """the directional derivative of the fp64 forward by central differences (error h^2 / 6 of the third
    derivative, far below 1e-6 at h = 1e-4) against the kernels' gradients"""
    x = _map((2, 8, 5, 7), torch.float32, device, 9).requires_grad_(True)
    w, be = _affine(8, torch.float32, device, 9)
    w.requires_grad_(True)
    be.requires_grad_(True)
    dy = _map((2, 8, 5, 7), torch.float32, device, 10)
    for act in ("silu", None):
        grads = torch.autograd.grad(ops.group_norm_act(x, 2, w, be, act=act), (x, w, be), dy)
        g = torch.Generator().manual_seed(2)
        for k in range(3):
            leaves = [t.detach().double() for t in (x, w, be)]
            d = torch.randn(leaves[k].shape, generator=g, dtype=torch.float64).to(device)
            ends = []
            for h in (1e-4, -1e-4):
                moved = [t + h * d if i == k else t for i, t in enumerate(leaves)]
                ends.append((_oracle(moved[0], 2, moved[1], moved[2], act)["y"][0] * dy.double()).sum())
            slope = float((ends[0] - ends[1]) / 2e-4)
            got = float((grads[k].double() * d).sum())
            scale = float((grads[k].double() * d).abs().sum())
            # differences: cancellation 1e-16 |f| / h; the kernel: (N_T + 20) u of the magnitudes
            assert abs(got - slope) <= 1e-6 * scale + (N_T + 20) * U * scale, (act, k)


def test_empty_and_refusals(device):
    w = torch.ones(8, device=device, requires_grad=True)
    for shape in ((0, 8, 4, 4), (2, 8, 0, 4), (0, 8)):
        x = torch.empty(shape, device=device).to(memory_format=torch.channels_last if len(shape) == 4 else torch.contiguous_format)
        x.requires_grad_(True)
        y = ops.group_norm_act(x, 2, w)
        assert y.shape == shape
        dx, dw = torch.autograd.grad(y.sum(), (x, w))
        assert dx.shape == shape and torch.equal(dw, torch.zeros_like(w))
    x = _map((2, 8, 4, 4), torch.float32, device, 1)
    w, be = _affine(8, torch.float32, device, 1)
    for match, call in (
            ("channels-last", lambda: ops.group_norm_act(x.contiguous(), 2, w, be)),
            ("GPU tensors", lambda: ops.group_norm_act(x.cpu(), 2)),
            ("GPU tensors", lambda: ops.group_norm_act(x, 2, w.cpu())),
            ("do not divide", lambda: ops.group_norm_act(x, 3)),
            ("do not divide", lambda: ops.group_norm_act(x, 0)),
            ("fp32, fp16 or bf16", lambda: ops.group_norm_act(x.double(), 2)),
            ("weight must be", lambda: ops.group_norm_act(x, 2, w[:4])),
            ("bias must be", lambda: ops.group_norm_act(x, 2, w, be.double())),
            ("differ in type", lambda: ops.group_norm_act(x, 2, w, be.half())),
            ("act is", lambda: ops.group_norm_act(x, 2, act="gelu")),
            ("eps", lambda: ops.group_norm_act(x, 2, eps=-1.0)),
            ("eps", lambda: ops.group_norm_act(x, 2, eps=float("nan"))),
            ("dimension", lambda: ops.group_norm_act(x.flatten(), 2)),
            ("requirement failed", lambda: ops.group_norm_act(torch.zeros((1, 2052), device=device), 1))):
        with pytest.raises(RuntimeError, match=match):
            call()
    # a second derivative is refused, not wrong
    xr = x.detach().requires_grad_(True)
    dx, = torch.autograd.grad(ops.group_norm_act(xr, 2, act="silu").sum(), xr, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def test_two_runs_give_the_same_bits(device):
    x = _map((2, 256, 50, 76), torch.float32, device, 12).requires_grad_(True)
    w, be = _affine(256, torch.float32, device, 12)
    w.requires_grad_(True)
    be.requires_grad_(True)
    dy = _map((2, 256, 50, 76), torch.float32, device, 13)
    first = None
    for _ in range(4):
        y = ops.group_norm_act(x, 32, w, be)
        out = (y,) + torch.autograd.grad(y, (x, w, be), dy)
        first = first or out
        assert all(torch.equal(a, b) for a, b in zip(out, first))


def test_streams_and_captured_graphs(device):
    """on a stream of its own; captured with its backward pass and replayed on new inputs, eager calls between"""
    shape = (2, 64, 20, 30)
    w, be = _affine(64, torch.float32, device, 14)
    w.requires_grad_(True)
    be.requires_grad_(True)
    x = _map(shape, torch.float32, device, 15).requires_grad_(True)
    dy = _map(shape, torch.float32, device, 16)

    def step():
        y = ops.group_norm_act(x, 8, w, be, act="silu")
        return (y.detach(),) + torch.autograd.grad(y, (x, w, be), dy)

    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    eager = step()
    with torch.cuda.stream(side):
        other = step()
        step()
    torch.cuda.current_stream(device).wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    del eager, other
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (20, 21, 22):
        with torch.no_grad():
            x.copy_(_map(shape, torch.float32, device, seed))
            dy.copy_(_map(shape, torch.float32, device, seed + 50))
        graph.replay()
        got = [t.clone() for t in held]
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), seed


def test_offsets_past_32_bits(device):
    """a slice of a buffer of more than 2^32 elements: the last pixels lie behind 32-bit offsets"""
    pixels, width, c = 1_050_000, 4100, 8
    buf = torch.zeros((pixels, width), dtype=torch.float16, device=device)
    assert buf.numel() > 2 ** 32
    x = buf[:, :c]
    x.copy_(torch.randn((pixels, c), device=device))
    m = buf.as_strided((1, c, 1, pixels), (0, 1, 0, width))
    w, be = _affine(c, torch.float32, device, 4)
    y = ops.group_norm_act(m, 2, w, be)
    dense = x.contiguous().reshape(1, 1, pixels, c).permute(0, 3, 1, 2)
    assert torch.equal(y, ops.group_norm_act(dense, 2, w, be))
    assert float(y[..., -4096:].float().abs().max()) > 0.5


def test_conv_layers_use_it_when_asked(device, monkeypatch):
    """modules._ConvNormAct under autograd with DANCE_GROUPNORM=hip against the stock path; a channels-first map stays on
    the stock path.  The sums of both are of at most 960 fp32 terms (576 * 2^-24 = 3.4e-5 of their absolute sum for the
    convolution alone, forward and backward), and where |z| is below 1e-3, which the two may see on either side of the
    ReLU's border, the gradient is zero: 1e-4 of the norms, 1e-3 of the weight's (sums of cancelling terms)."""
    g = torch.Generator().manual_seed(3)
    layer = modules._ConvNormAct(64, 96, 1, "GN").to(device).to(memory_format=torch.channels_last)
    with torch.no_grad():
        for p in layer.parameters():
            p.copy_(torch.randn(p.shape, generator=g) * (0.05 if p.dim() == 4 else 0.3) + (p.dim() == 1))
    x = torch.randn((2, 64, 20, 24), generator=g).to(device)
    dy = torch.randn((2, 96, 20, 24), generator=g).to(device)
    with torch.no_grad():
        z = layer.norm.to(device)(torch.nn.functional.conv2d(x, layer.weight, layer.bias, padding=1))
    dy = dy * (z.abs() > 1e-3)
    calls = []
    real = ops.group_norm_act
    monkeypatch.setattr(ops, "group_norm_act", lambda *a, **k: calls.append(1) or real(*a, **k))
    results = {}
    for knob in ("torch", "hip"):
        monkeypatch.setenv("DANCE_GROUPNORM", knob)
        xr = x.to(memory_format=torch.channels_last).requires_grad_(True)
        y = layer(xr)
        results[knob] = (y,) + torch.autograd.grad(y, [xr] + list(layer.parameters()), dy)
        assert len(calls) == (knob == "hip")
    for i, (a, b) in enumerate((a.detach(), b.detach()) for a, b in zip(results["hip"], results["torch"])):
        assert a.shape == b.shape and float((a - b).norm()) <= (1e-4 if i < 2 else 1e-3) * float(b.norm())
    monkeypatch.setattr(ops, "is_channels_last", lambda t: False)
    assert layer(x).shape == dy.shape
    assert len(calls) == 1


@pytest.mark.parametrize("dtype,c,lo,hi", [(torch.float32, 72, 0, 72), (torch.float32, 75, 1, 73), (torch.bfloat16, 143, 3, 139)])
def test_maps_larger_than_the_cache(device, dtype, c, lo, hi):
    """maps of more than 64 MB are read and written past the cache: aligned, and at odd elements with channels around
    them, which get a gradient of zero.  (A thread sums 16 pixels at these sizes, half of N_T.)"""
    full = _map((2, c, 257, 463), dtype, device, c).permute(0, 2, 3, 1).contiguous().requires_grad_(True)
    x = full.permute(0, 3, 1, 2)[:, lo:hi]
    assert x.numel() * x.element_size() >= 64e6
    w, be = (t.requires_grad_(True) for t in _affine(hi - lo, torch.float32, device, c))
    y = ops.group_norm_act(x, 8, w, be)
    dy = _map(tuple(x.shape), dtype, device, c + 1)
    dfull, dw, db = torch.autograd.grad(y, (full, w, be), dy)
    want = _oracle(x, 8, w, be, "relu", dy)
    for name, got in (("y", y), ("dx", dfull.permute(0, 3, 1, 2)[:, lo:hi]), ("dweight", dw), ("dbias", db)):
        _check(got, want[name], name)
    assert not bool(dfull[..., :lo].any()) and not bool(dfull[..., hi:].any())


def test_more_images_or_channels_than_a_call_takes(device):
    one = torch.zeros((1, 8), device=device)
    for big in (one.expand(65536, 8), one.expand(2 ** 32 + 1, 8), torch.zeros((1, 8192), device=device)):
        with pytest.raises(RuntimeError, match="at most 65535 images and 4096 channels"):
            ops.group_norm_act(big, 1)
    assert ops.group_norm_act(one.expand(65535, 8), 1).shape == (65535, 8)


@pytest.mark.parametrize("shape,groups", [((65535, 4), 2), ((300, 40, 9, 9), 8), ((600, 256, 3, 3), 32), ((40, 64, 70, 71), 8),
                                          ((17, 96, 50, 50), 4), ((129, 75, 2, 3), 5)])
def test_many_images(device, shape, groups):
    """whole maps a workgroup, and the parameters' gradients over many images"""
    for dtype in (torch.float32, torch.bfloat16):
        x = _map(shape, dtype, device, 3).requires_grad_(True)
        w, be = (t.requires_grad_(True) for t in _affine(shape[1], torch.float32, device, 3))
        dy = _map(shape, dtype, device, 4)
        y = ops.group_norm_act(x, groups, w, be, act="silu")
        got = torch.autograd.grad(y, (x, w, be), dy)
        want = _oracle(x, groups, w, be, "silu", dy)
        for name, t in zip(("y", "dx", "dweight", "dbias"), (y,) + got):
            _check(t, want[name], "%s %s %s" % (shape, dtype, name))
        only, = torch.autograd.grad(ops.group_norm_act(x.detach(), groups, w, be, act="silu"), (w,), dy)
        assert torch.equal(only, got[1])


@pytest.mark.parametrize("pin", [False, True])
@pytest.mark.parametrize("dtype,lo", [(torch.float32, 0), (torch.float32, 1), (torch.bfloat16, 0), (torch.float16, 3)])
@pytest.mark.parametrize("hw", [(9, 11), (70, 71)])
def test_saved_tensors_in_host_memory(device, hw, dtype, lo, pin):
    """save_on_cpu gives the map back in other strides, pinned also channels first: the same bits as without it"""
    x = _map((2, 40 + lo, *hw), dtype, device, 30)[:, lo:].requires_grad_(True)
    w, be = _affine(40, dtype, device, 30)
    w.requires_grad_(True)
    be.requires_grad_(True)
    dy = _map((2, 40, *hw), dtype, device, 31)
    y = ops.group_norm_act(x, 8, w, be, act="silu")
    want = (y.detach(),) + torch.autograd.grad(y, (x, w, be), dy)
    with torch.autograd.graph.save_on_cpu(pin_memory=pin):
        y = ops.group_norm_act(x, 8, w, be, act="silu")
    got = (y.detach(),) + torch.autograd.grad(y, (x, w, be), dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("mean,spread,first", [(1e6, 0.1, 0.0), (1e5, 1e-2, 0.0), (1e4, 1e-3, 0.0), (-1e4, 1e-2, 0.0),
                                               (1e4, 1e-2, -1e6), (3.0, 1.0, 1e5)])
@pytest.mark.parametrize("shape,groups", [((1, 32, 200, 304), 4), ((2, 30, 150, 130), 5), ((2, 16, 16, 32), 4), ((3, 10, 5, 7), 2)])
def test_any_mean_and_any_first_value(device, shape, groups, mean, spread, first):
    """the statistics keep their bits at any ratio of mean and spread that fp32 values can have, also where a group's
    first value (`first` away from the others) is not like them.  To the tolerances above comes what a mean far from the
    values' spread adds: its low float is rounded, U |mlo| <= U^2 |mean|, and the oracle's own mean; 2 U^2 |mean| of x
    are e = 2 U^2 |mean| rstd of xh, in every place that xh has."""
    g = torch.Generator().manual_seed(11)
    b, c = shape[:2]
    x = mean + spread * torch.randn((b, *shape[2:], c), generator=g)
    x[:, 0, 0, ::c // groups] += first
    x = x.to(device).permute(0, 3, 1, 2).requires_grad_(True)
    w, be = _affine(c, torch.float32, device, 11)
    w.requires_grad_(True)
    be.requires_grad_(True)
    dy = torch.randn((b, *shape[2:], c), generator=g).to(device).permute(0, 3, 1, 2)
    y = ops.group_norm_act(x, groups, w, be, act=None)
    dx, dw, db = torch.autograd.grad(y, (x, w, be), dy)
    want = _oracle(x, groups, w, be, None, dy)
    gx = x.detach().double().reshape(b, groups, -1)
    far = gx.mean(2, keepdim=True)
    rstd = 1 / torch.sqrt(((gx - far) ** 2).mean(2, keepdim=True) + 1e-5)
    e = 2 * U * U * far.abs() * rstd
    wdz = (dy.double() * w.detach().double()[None, :, None, None]).reshape(gx.shape)
    xh = (gx - far) * rstd
    of_dx = rstd * e * ((wdz * xh).mean(2, keepdim=True).abs() + xh.abs() * wdz.abs().mean(2, keepdim=True))
    each = e.expand(gx.shape).reshape(shape)
    more = {"y": each * w.detach().double().abs()[None, :, None, None], "dx": of_dx.reshape(shape),
            "dweight": (dy.double().abs() * each).sum((0, 2, 3)), "dbias": 0.0}
    for name, got in (("y", y), ("dx", dx), ("dweight", dw), ("dbias", db)):
        _check(got, (want[name][0], want[name][1] + more[name]), name)


@pytest.mark.parametrize("shape,groups", [((1, 4093, 2, 2), 4093), ((300, 4072, 1), 4072), ((1, 4078, 2, 2), 2039),
                                          ((2, 4096, 3, 1), 4096), ((2, 4095, 2), 9)])
def test_thousands_of_groups(device, shape, groups):
    """groups of a channel or two, as many as there can be"""
    x = _map(shape, torch.bfloat16, device, 40).requires_grad_(True)
    w, be = _affine(shape[1], torch.float32, device, 40)
    w.requires_grad_(True)
    be.requires_grad_(True)
    dy = _map(shape, torch.bfloat16, device, 41)
    y = ops.group_norm_act(x, groups, w, be, act="silu")
    got = (y,) + torch.autograd.grad(y, (x, w, be), dy)
    want = _oracle(x, groups, w, be, "silu", dy)
    for name, value in zip(("y", "dx", "dweight", "dbias"), got):
        _check(value, want[name], name)


def test_conv_layers_under_autocast(device, monkeypatch):
    """DANCE_GROUPNORM=hip returns the stock path's type: fp32, from the 16-bit output of the convolution"""
    layer = modules._ConvNormAct(32, 64, 1, "GN").to(device).to(memory_format=torch.channels_last)
    layer.use_hip = False
    x = _map((2, 32, 9, 10), torch.float32, device, 50)
    results = {}
    for knob in ("torch", "hip"):
        monkeypatch.setenv("DANCE_GROUPNORM", knob)
        for dtype in (torch.float16, torch.bfloat16):
            with torch.autocast("cuda", dtype=dtype):
                results[knob, dtype] = layer(x)
    with torch.no_grad():
        for dtype in (torch.float16, torch.bfloat16):
            want, got = results["torch", dtype], results["hip", dtype]
            assert got.dtype == want.dtype == torch.float32
            conv = torch.nn.functional.conv2d(x.to(dtype), layer.weight.to(dtype), padding=1)
            _check(got, _oracle(conv, 32, layer.norm.weight, layer.norm.bias, "relu")["y"], str(dtype))


def test_conv_layers_of_more_channels_than_a_call_takes(device, monkeypatch):
    """stay on the stock path"""
    monkeypatch.setenv("DANCE_GROUPNORM", "hip")
    layer = modules._ConvNormAct(4, 2080, 1, "GN").to(device).to(memory_format=torch.channels_last)
    layer.use_hip = False
    x = _map((1, 4, 5, 6), torch.float32, device, 51)
    assert ops.is_channels_last(_map((1, 2048, 2, 2), torch.float32, device, 52))
    assert ops.is_channels_last(_map((1, 4096, 2, 2), torch.bfloat16, device, 52))
    assert not ops.is_channels_last(_map((1, 2052, 2, 2), torch.float32, device, 52))
    assert not ops.is_channels_last(_map((70000, 4), torch.float32, device, 52))
    assert layer(x).shape == (1, 2080, 5, 6)


def test_checkpointed(device):
    """torch.utils.checkpoint gives back tensors of a second forward call: the same bits as without it"""
    x = _map((2, 40, 21, 23), torch.float32, device, 60)[:, 4:36].requires_grad_(True)
    w, be = _affine(32, torch.float32, device, 60)
    w.requires_grad_(True)
    be.requires_grad_(True)
    dy = _map((2, 32, 21, 23), torch.float32, device, 61)

    def layer(t):
        return ops.group_norm_act(ops.group_norm_act(t, 8, w, be), 4, w, be, act="silu")

    y = layer(x)
    want = (y.detach(),) + torch.autograd.grad(y, (x, w, be), dy)
    y = torch.utils.checkpoint.checkpoint(layer, x, use_reentrant=False)
    got = (y.detach(),) + torch.autograd.grad(y, (x, w, be), dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
