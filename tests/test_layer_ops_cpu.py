"""CPU: the group-norm entry points report bad arguments before anything is enqueued."""
import ctypes

import pytest
import torch

from dance_amd import _lib, ops

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
