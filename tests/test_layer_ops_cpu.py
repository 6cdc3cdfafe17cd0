"""CPU: the group-norm entry points report bad arguments before anything is enqueued."""
import contextlib
import ctypes

import pytest
import torch

from dance_amd import _lib, ops, optim

BAD = 1                                                    # hipErrorInvalidValue


def _norm(**over):
    a = dict(x=None, image=0, pixel=8, dtype=0, w=None, b=None, affine=0, eps=1e-5, act=1, groups=2, y=None, saved=None,
             ws=None, ws_bytes=0, n=1, c=8, hw=4, stream=None)
    a.update(over)
    return _lib.lib().dance_group_norm_act(*a.values())


def _norm_backward(**over):
    a = dict(dy=None, dy_image=0, dy_pixel=8, x=None, image=0, pixel=8, dtype=0, affine=0, act=1, groups=2,
             saved=None, dx=None, dw=None, db=None, ws=None, ws_bytes=0, n=1, c=8, hw=4, stream=None)
    a.update(over)
    return _lib.lib().dance_group_norm_act_backward(*a.values())


@pytest.mark.parametrize("over", [dict(dtype=3), dict(affine=-1), dict(act=9), dict(groups=3), dict(groups=0), dict(c=0),
                                  dict(c=2052, groups=1), dict(c=4104, groups=1, dtype=2), dict(eps=-1.0), dict(eps=float("nan")),
                                  dict(image=-1), dict(pixel=-8), dict(n=-1), dict(hw=-1), dict(), dict(n=70000)])
def test_group_norm_refuses(over):
    assert _norm(**over) == BAD and b"requirement failed" in _lib.lib().dance_last_error()
    if "eps" not in over:
        assert _norm_backward(**over) == BAD


def test_group_norm_empty_calls_do_nothing():
    assert _norm(n=0) == 0 and _norm(hw=0) == 0


def test_group_norm_workspace():
    """none for maps of one launch; otherwise large enough for every group's sums, and refused one byte short"""
    size = _lib.lib().dance_group_norm_workspace_bytes
    assert size(1, 2052, 4, 1, 0, 0) == 0 and size(1, 8, 4, 3, 0, 0) == 0 and size(0, 8, 4, 2, 0, 0) == 0
    fake = ctypes.c_void_p(64)                             # never reached: the size is looked at first
    for dtype in (0, 1, 2):
        assert size(1, 8, 1, 2, dtype, 0) == 0 and size(1, 8, 1, 2, dtype, 1) == 0
        assert size(3, 8, 1, 2, dtype, 1) == 3 * 8 * 16     # a channel's two sums of every image
        need = size(2, 256, 60800, 32, dtype, 0)
        assert need >= 2 * 32 * 16 and size(2, 256, 60800, 32, dtype, 1) >= 2 * 256 * 16
        big = dict(x=fake, y=fake, saved=fake, n=2, c=256, hw=60800, groups=32, dtype=dtype)
        assert _norm(ws=fake, ws_bytes=need - 1, **big) == BAD and _norm(ws=None, ws_bytes=need, **big) == BAD


@pytest.mark.parametrize("b,c,hw,groups", [(1, 4093, 4, 4093), (300, 4072, 1, 4072), (1, 4078, 4, 2039)])
def test_group_norm_of_thousands_of_groups(b, c, hw, groups):
    """no slab of them fits a compute unit's LDS with its groups' statistics and channels' constants: the form of three
    launches, which has a workspace"""
    assert _lib.lib().dance_group_norm_workspace_bytes(b, c, hw, groups, 2, 0) >= b * groups * 16


def test_group_norm_needs_a_gpu_tensor():
    with pytest.raises(RuntimeError, match="GPU tensors"):
        ops.group_norm_act(torch.zeros((1, 8, 2, 2)), 2)


def test_channels_last_strides():
    s = ops._channels_last_strides
    t = torch.zeros((2, 5, 7, 12))                         # (B, H, W, C)
    nchw = t.permute(0, 3, 1, 2)
    assert s(nchw) == (5 * 7 * 12, 12) and s(nchw[:, 3:9]) == (5 * 7 * 12, 12)
    assert s(nchw[:, :, 1:3]) == (5 * 7 * 12, 12)          # whole rows
    assert s(nchw[:, :, :, 1:3]) is None                   # a crop inside the rows
    assert s(nchw.contiguous()) is None
    assert s(nchw[:1].expand(4, -1, -1, -1))[0] == 0
    assert s(torch.zeros((3, 6))) == (6, 6)
    assert s(torch.zeros((3, 1, 4, 4))) == (16, 1)         # one channel: any layout
    assert s(torch.zeros((3, 6, 1, 1))) == (6, 6)


def _orth(**over):
    a = dict(x=None, bs=0, rs=8, cs=1, dtype=0, out=None, batch=1, m=4, n=8, steps=5, a=3.4445, b=-4.775, c=2.0315, eps=1e-7,
             ws=None, ws_bytes=0, stream=None)
    a.update(over)
    return _lib.lib().dance_orthogonalize(*a.values())


@pytest.mark.parametrize("over", [dict(dtype=7), dict(steps=0), dict(steps=101), dict(a=float("nan")), dict(c=float("inf")),
                                  dict(eps=0.0), dict(eps=float("nan")), dict(rs=-1), dict(bs=-1), dict(cs=-1), dict(m=-1),
                                  dict(batch=-1), dict(m=1 << 16, n=1 << 15), dict()])
def test_orthogonalize_refuses(over):
    assert _orth(**over) == BAD and b"requirement failed" in _lib.lib().dance_last_error()


def test_orthogonalize_empty_and_workspace():
    assert _orth(batch=0) == 0 and _orth(m=0) == 0 and _orth(n=0) == 0
    size = _lib.lib().dance_orthogonalize_workspace_bytes
    assert size(0, 4, 8) == 0 and size(1, 0, 8) == 0 and size(1, 1 << 16, 1 << 15) == 0
    assert size(1, 1, 2 ** 31 - 1) == 0 and _orth(m=1, n=2 ** 31 - 1) == BAD          # the padded side would not fit an int
    assert size(1, 64, 200) == 0 and size(48, 32, 9) == 0   # a compute unit's LDS holds the whole chain
    need = size(3, 100, 500)
    assert need >= 3 * 4 * 100 * 500                        # up to 128 rows: X in place, 4 bytes each
    assert size(3, 200, 500) >= 3 * 16 * 200 * 500          # more: two layouts, two steps
    fake = ctypes.c_void_p(64)
    good = dict(x=fake, out=fake, batch=3, m=100, n=500)
    assert _orth(ws=fake, ws_bytes=need - 1, **good) == BAD and _orth(ws=None, ws_bytes=need, **good) == BAD
    assert _orth(ws=ctypes.c_void_p(72), ws_bytes=need, **good) == BAD
    assert size(1000, 100, 500) < 1000 * need / 3           # of the matrices of one launch


def _muon(items, **over):
    a = dict(items=items, count=1, dtype=0, lr=0.1, momentum=0.9, nesterov=1, wd=0.0, steps=5, a=3.4445, b=-4.775, c=2.0315,
             eps=1e-7, ws=None, ws_bytes=0, stream=None, side=None)
    a.update(over)
    return _lib.lib().dance_muon_step(*a.values())


def test_muon_refuses():
    items = (_lib.MuonItemStruct * 2)()
    for it in items:
        it.param, it.grad, it.momentum, it.rows, it.cols = 64, 64, 64, 200, 300
    size = _lib.lib().dance_muon_workspace_bytes
    need = size(items, 2)
    assert need > size(items, 1) > 0 and size(items, 0) == 0
    fake = ctypes.c_void_p(64)
    assert _muon(items, count=0) == 0 and _muon(None, count=0) == 0
    good = dict(count=2, ws=fake, ws_bytes=need)
    for over in (dict(count=-1), dict(dtype=5), dict(lr=float("nan")), dict(momentum=float("inf")), dict(wd=float("nan")),
                 dict(steps=0), dict(eps=-1.0), dict(b=float("nan")), dict(ws_bytes=need - 1), dict(ws=None)):
        assert _muon(items, **{**good, **over}) == BAD, over
    for field, bad in (("param", 0), ("grad", 0), ("momentum", 0), ("rows", 0), ("cols", -1), ("rows", 1 << 30)):
        keep = getattr(items[1], field)
        setattr(items[1], field, bad)
        assert _muon(items, **good) == BAD, field
        setattr(items[1], field, keep)


def test_muon_workspace_keeps_the_kinds_apart():
    """matrices of up to 128 rows and the others run beside each other on two streams, and more of a kind than one launch
    takes follow each other: what one kind uses must not depend on how many launches the other one takes"""
    def size(*shapes):
        items = (_lib.MuonItemStruct * len(shapes))()
        for it, s in zip(items, shapes):
            it.param, it.grad, it.momentum, it.rows, it.cols = 64, 64, 64, s[0], s[1]
        return _lib.lib().dance_muon_workspace_bytes(items, len(shapes))
    narrow, wide = [(100, 900)], [(200, 300)]
    for n, w in ((1, 1), (48, 5), (60, 5), (5, 60), (100, 100)):
        assert size(*narrow * n, *wide * w) == size(*narrow * n) + size(*wide * w)
        assert size(*narrow * n) == size(*narrow * min(n, 48)) and size(*wide * w) == size(*wide * min(w, 48))


def test_muon_item_layout_matches_header():
    assert ctypes.sizeof(_lib.MuonItemStruct) == 3 * 8 + 2 * 4


def test_newton_schulz_needs_gpu_tensors_and_matrices():
    from dance_amd import optim

    with pytest.raises(RuntimeError, match="GPU tensors"):
        ops.orthogonalize(torch.zeros((4, 4)))
    with pytest.raises(RuntimeError, match="GPU tensors"):
        optim.muon_step([torch.zeros((4, 4))], [torch.zeros((4, 4))], [torch.zeros((4, 4))], lr=0.1)
    with pytest.raises(ValueError, match="not a matrix"):
        optim.Muon([torch.zeros(4, requires_grad=True)])
    with pytest.raises(RuntimeError, match="steps"):
        optim.Muon([torch.zeros((4, 4), requires_grad=True)], steps=0)


def test_rows_outermost():
    from dance_amd.optim import _rows_outermost as f

    t = torch.zeros((6, 4, 3, 3))
    assert f(t) and f(t.to(memory_format=torch.channels_last)) and f(t[2:4]) and f(t[:1, 1:2])
    assert not f(t.transpose(0, 1)) and not f(t[:, ::2]) and not f(t[::2]) and not f(t[:, :, :2])
    assert f(torch.zeros((1, 9)).t()) and not f(torch.zeros((3, 9)).t())


class _Kernels:
    """In the library's place: the backward call reads x where and as it is told to (and nowhere outside the tensors of
    `held`), so that a CPU tensor can stand for the GPU's."""

    def __init__(self, held):
        self.held, self.called, self.read = held, False, None

    def dance_group_norm_saved_bytes(self, b, c, groups):
        return 64

    def dance_group_norm_workspace_bytes(self, *sizes):
        return 0

    def dance_group_norm_act(self, *args):
        return 0

    def dance_group_norm_act_backward(self, dy, dy_image, dy_pixel, x, image, pixel, *rest):
        self.called = True
        if not self.held:
            return 0
        b, c, hw = rest[-4:-1]
        if x in self.held:
            t = self.held[x]
            left = t.untyped_storage().nbytes() // 4 - t.storage_offset()
            assert (b - 1) * image + (hw - 1) * pixel + c <= left, "reads past the end of x"
        values = (ctypes.c_float * ((b - 1) * image + (hw - 1) * pixel + c)).from_address(x)
        self.read = [[[values[i * image + p * pixel + ch] for p in range(hw)] for ch in range(c)] for i in range(b)]
        return 0


@pytest.fixture
def on_cpu(monkeypatch):
    """ops' group norm on CPU tensors, up to the library's calls"""
    kernels = _Kernels({})
    monkeypatch.setattr(ops, "_need_gpu", lambda *tensors: None)
    monkeypatch.setattr(ops, "lib", lambda: kernels)
    monkeypatch.setattr(ops, "on_device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(ops, "stream_of", lambda device: 0)
    return kernels


def _slice(shape, channels):
    """a channels-last map, the first channel of a wider one left out"""
    b, c, h, w = shape
    wide = torch.arange(b * h * w * (c + channels), dtype=torch.float32).reshape(b, h, w, c + channels)
    return wide.permute(0, 3, 1, 2)[:, channels:]


@pytest.mark.parametrize("channels", [0, 1])
@pytest.mark.parametrize("unpack", [lambda t: t, torch.clone, lambda t: torch.empty(t.shape, dtype=t.dtype).copy_(t),
                                    lambda t: t[..., None].expand(*t.shape, 2).contiguous()[..., 0]],
                         ids=["same", "dense", "channels_first", "spread"])
def test_group_norm_backward_reads_what_a_hook_gives_back(on_cpu, unpack, channels):
    """saved-tensor hooks (torch's save_on_cpu among them) give x back in other strides"""
    x = _slice((2, 8, 4, 5), channels).requires_grad_(True)

    def back(t):
        t = unpack(t)
        on_cpu.held[t.data_ptr()] = t
        return t

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), back):
        y = ops.group_norm_act(x, 4)
        y.backward(torch.ones_like(y))
    assert on_cpu.read == x.detach().flatten(2).tolist()


@pytest.mark.parametrize("unpack", [lambda t: t.double(), lambda t: t[:1], lambda t: t.half(), lambda t: t.to("meta")])
def test_group_norm_backward_refuses_other_saved_tensors(on_cpu, unpack):
    x = _slice((2, 8, 4, 5), 0).requires_grad_(True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), unpack):
        y = ops.group_norm_act(x, 4, torch.ones(8, requires_grad=True))
        with pytest.raises(RuntimeError, match="saved-tensor hook"):
            y.backward(torch.ones_like(y))
    assert not on_cpu.called


def test_tangents_are_refused(on_cpu, monkeypatch):
    """forward-mode derivatives: dual tensors, and those that torch.func.jvp makes"""
    x, t = _slice((2, 8, 4, 5), 0), torch.ones((2, 8, 4, 5))
    w, tw = torch.ones(8), torch.ones(8)
    monkeypatch.setattr(optim, "_need_gpu", lambda *tensors: None)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual
        with torch.no_grad():
            for args in ((dual(x, t), 4), (x, 4, dual(w, tw)), (x, 4, w, dual(w, tw))):
                with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    ops.group_norm_act(*args)
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            ops.orthogonalize(dual(x, t))
        for k in range(3):
            lists = [[torch.ones((4, 6))] for _ in range(3)]
            lists[k] = [dual(torch.ones((4, 6)), torch.ones((4, 6)))]
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                optim.muon_step(*lists, lr=0.1)
        assert ops.group_norm_act(x, 4, w).shape == x.shape         # a level alone is no reason
    for f in (lambda v: ops.group_norm_act(v, 4), ops.orthogonalize):
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            torch.func.jvp(f, (x,), (t,))
    assert not on_cpu.called


def test_muon_lays_out_buffers_of_another_memory_format(monkeypatch):
    """a state loaded from contiguous weights into channels_last ones, a module converted after its first step"""
    taken = []
    monkeypatch.setattr(optim, "muon_step", lambda params, grads, buffers, **settings: taken.extend(buffers))
    shapes = [(8, 4, 3, 3), (8, 4, 1, 1), (6, 5)]

    def optimizer(memory_format):
        params = [torch.nn.Parameter(torch.zeros(s)) for s in shapes]
        for p in params:
            p.data = p.data.to(memory_format=memory_format) if p.dim() == 4 else p.data
            p.grad = torch.zeros_like(p)
        return optim.Muon(params), params

    opt, params = optimizer(torch.contiguous_format)
    opt.step()
    with torch.no_grad():
        for m in taken:
            m.copy_(torch.arange(m.numel()).reshape(m.shape))
    want = [m.clone() for m in taken]
    other, others = optimizer(torch.channels_last)
    other.load_state_dict(opt.state_dict())
    for p in params[:2]:
        p.data = p.data.to(memory_format=torch.channels_last)
        p.grad = torch.zeros_like(p)
    for o, ps in ((other, others), (opt, params)):
        taken.clear()
        o.step()
        assert [m.stride() for m in taken] == [p.stride() for p in ps]
        assert all(torch.equal(m, v) for m, v in zip(taken, want))
        held = list(taken)
        taken.clear()
        o.step()
        assert all(m is h for m, h in zip(taken, held))


@pytest.mark.parametrize("m,n", [(1, 10 ** 7), (8, 10 ** 6), (128, 1152), (100, 500), (65, 40000), (128, 128), (129, 129), (144, 1296),
                                 (1024, 4096), (200, 500), (46000, 46000), (130, 16 * 10 ** 6), (4000, 300), (300, 10 ** 5)])
def test_orthogonalize_workspace_as_documented(m, n):
    size = _lib.lib().dance_orthogonalize_workspace_bytes
    r, k = sorted((s + 127) // 128 * 128 for s in (m, n))
    each = 1024 * k + 2 ** 17 if r == 128 else 16 * r * k + 10 * r * r + 2 ** 24 + 2 ** 17
    for batch in (1, 3, 48, 1000):
        assert size(batch, m, n) <= min(batch, 48) * each
    assert size(1, m, n) >= (512 if r == 128 else 16 * r) * k
