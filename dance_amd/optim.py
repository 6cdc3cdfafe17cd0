"""Muon: momentum SGD whose update is orthogonalised (ops.orthogonalize), for the weight matrices of heads that are trained
as torch modules (this package's own only infer).

A parameter of more than two dimensions is its (first dimension, the rest) matrix: a convolution's weight is
(out channels, in channels * taps).  Vectors (biases, norm weights) are not Muon's: give them to another
optimizer.  The whole step -- momentum, Nesterov's look-ahead, the chain of products, the parameter update --
shares its launches among all matrices of one type and device, whatever their shapes: one launch where each fits a
compute unit, else one chain of them for up to 128 rows and one for the others.

The reference trains with Detectron2's SGD (train_net.py:22-70) and has no counterpart.
"""
import struct
import threading

import torch

from ._lib import MuonItemStruct, check, lib, on_device, ptr, stream_of
from .ops import DTYPE_CODES, MOST_ELEMENTS, NS_COEFFICIENTS, _need_gpu, _no_tangents, _scratch, check_newton_schulz


NARROW_ROWS = 128           # up to so many rows (of the smaller side) a step of the chain is a launch of its own

_SIDE = threading.local()    # a thread may be capturing its stream into a graph while another one steps


def _side_stream(dev):
    """-> a stream of this thread's and two events to fork into it and join it with"""
    kept = _SIDE.__dict__
    if dev not in kept:
        kept[dev] = torch.cuda.Stream(dev), torch.cuda.Event(), torch.cuda.Event()
    return kept[dev]


def _rows_outermost(t):
    """Is t's memory dense with its first dimension outermost?  (contiguous or channels_last weights; the order
    of the columns does not matter, orthogonalisation commutes with permuting them)"""
    if t.is_contiguous():
        return True
    dense = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride()[1:], t.shape[1:]) if sz > 1):
        if stride != dense:
            return False
        dense *= size
    return t.size(0) == 1 or t.stride(0) == dense


def _refuse(what, p, g, m):
    _need_gpu(p, g, m)
    if p.dim() < 2 or p.dtype not in DTYPE_CODES:
        raise RuntimeError("%s: matrices of fp32, fp16 or bf16 expected, got a %s parameter of shape %s"
                           % (what, p.dtype, tuple(p.shape)))
    for name, t in (("gradient", g), ("momentum buffer", m)):
        if t.shape != p.shape or t.dtype != p.dtype or t.device != p.device:
            raise RuntimeError("%s: a %s %s %s on %s for a parameter %s %s on %s"
                               % (what, name, tuple(t.shape), t.dtype, t.device, tuple(p.shape), p.dtype, p.device))


@torch.no_grad()
def muon_step(params, grads, momentum_buffers, *, lr, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, eps=1e-7,
              coefficients=NS_COEFFICIENTS):
    """One Muon step, in place on params and momentum_buffers (equally long lists of tensors):

        m <- momentum m + (1 - momentum) g,   u = momentum m + (1 - momentum) g (nesterov) or m
        p <- p (1 - lr weight_decay) - lr sqrt(max(1, rows / columns)) orthogonalize(u)

    A parameter, its gradient and its buffer are of one type (fp32, fp16, bf16), device and shape; the parameter
    and its buffer dense with equal strides, rows outermost.  No tensor may appear twice among params and
    buffers."""
    what = "muon_step"
    steps, eps, (a, b, c) = check_newton_schulz(what, steps, eps, coefficients)
    if not len(params) == len(grads) == len(momentum_buffers):
        raise RuntimeError("%s: %d params, %d grads, %d momentum buffers"
                           % (what, len(params), len(grads), len(momentum_buffers)))
    _no_tangents(what, *params, *grads, *momentum_buffers)
    # checked a property at a time over the lists, which takes Python a third of the time of a matrix at a time
    shapes, dtypes, places = ([t.shape for t in params], [t.dtype for t in params], [t.get_device() for t in params])
    for other in (grads, momentum_buffers):
        if [t.shape for t in other] != shapes or [t.dtype for t in other] != dtypes or [t.get_device() for t in other] != places:
            break
    else:
        other = None
    if other is not None or min(places, default=0) < 0 or min(map(len, shapes), default=2) < 2 or \
            not DTYPE_CODES.keys() >= set(dtypes):
        for p, g, m in zip(params, grads, momentum_buffers):
            _refuse(what, p, g, m)
    strides = [t.stride() for t in params]
    for p, m, stride in zip(params, momentum_buffers, strides):
        if (m.stride() != stride or not (p.is_contiguous() or _rows_outermost(p))) and p.numel():
            raise RuntimeError("%s: parameter and momentum buffer must be dense, rows outermost, with equal strides, got %s "
                               "and %s of shape %s" % (what, stride, m.stride(), tuple(p.shape)))
    grads = [g if g.stride() == stride else torch.empty_strided(g.shape, stride, dtype=g.dtype, device=g.device).copy_(g)
             for g, stride in zip(grads, strides)]
    # {(device, type): [device, dance_muon_item's fields one after the other, a narrow matrix among them?, a wide one?]}
    chains, written = {}, []
    for p, g, m, shape, dtype, index in zip(params, grads, momentum_buffers, shapes, dtypes, places):
        size = shape.numel()
        if size == 0:
            continue
        if size > MOST_ELEMENTS:
            raise RuntimeError("%s: a matrix of more than 2^31 - 129 elements: %s" % (what, tuple(shape)))
        rows = shape[0]
        cols = size // rows
        chain = chains.get((index, dtype))
        if chain is None:
            chain = chains[index, dtype] = [p.device, [], False, False]
        chain[1] += (p.data_ptr(), g.data_ptr(), m.data_ptr(), rows, cols)
        chain[3 if rows > NARROW_ROWS and cols > NARROW_ROWS else 2] = True
        written += (p, m)
    places = [at for chain in chains.values() for k in (0, 2) for at in chain[1][k::5]]
    if len(set(places)) != len(places):
        raise RuntimeError("%s: a parameter or momentum buffer appears twice" % what)
    h = lib()
    for (_, dtype), (dev, fields, narrow, wide) in chains.items():
        count = len(fields) // 5
        items = (MuonItemStruct * count).from_buffer_copy(struct.pack("@" + "PPPii" * count, *fields))
        nbytes = h.dance_muon_workspace_bytes(items, count)
        with on_device(dev):
            ws, cur, side = _scratch(nbytes, dev), None, None
            if narrow and wide:                  # beside each other on two streams (the refinement net's weights: 276 against
                                                 # 322 us), since each leaves compute units idle between its launches
                cur, (side, fork, join) = torch.cuda.current_stream(dev), _side_stream(dev)
                fork.record(cur)
                side.wait_event(fork)
            code = h.dance_muon_step(items, count, DTYPE_CODES[dtype], lr, momentum, int(bool(nesterov)), weight_decay, steps, a,
                                     b, c, eps, ptr(ws), nbytes, stream_of(dev), None if side is None else side.cuda_stream)
            if side is not None:
                join.record(side)                # also where the call failed half way: the workspace is freed next
                cur.wait_event(join)
            check(code, what)
    # written behind autograd's back: what caches by version (saved tensors, the modules' packed weights) must see it
    # (inference tensors have no version)
    if any(map(torch.is_inference, written)):
        written = [t for t in written if not t.is_inference()]
    if written:
        torch.autograd.graph.increment_version(written)


class Muon(torch.optim.Optimizer):
    """torch.optim optimizer over muon_step.  Every parameter a matrix (two dimensions or more, the first one the
    rows); parameters without a gradient are left as they are.  A momentum buffer in another memory format than its
    parameter's (a loaded state, a module converted after its first step) is laid out again.  A step can be captured into a graph once every
    momentum buffer exists; its replays keep the settings, lr among them, that it was captured with."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, eps=1e-7,
                 coefficients=NS_COEFFICIENTS):
        steps, eps, coefficients = check_newton_schulz("Muon", steps, eps, coefficients)
        if not (lr >= 0 and 0 <= momentum < 1 and weight_decay >= 0):
            raise ValueError("Muon: lr and weight_decay must not be negative, momentum in [0, 1), got %r, %r, %r"
                             % (lr, weight_decay, momentum))
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      eps=eps, coefficients=coefficients))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() < 2:
                shape = tuple(p.shape)
                self.param_groups.pop()
                raise ValueError("Muon: a parameter of shape %s is not a matrix; give it to another optimizer" % (shape,))

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            for p in params:
                held = self.state[p].get("momentum_buffer")
                if held is not None and (held.stride() == p.stride() or held.shape != p.shape):
                    continue
                if p.is_cuda and torch.cuda.is_current_stream_capturing():
                    # (a replay would make the buffer again)
                    raise RuntimeError("Muon: take a step before the one that is captured into a graph")
                if held is None:
                    self.state[p]["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                else:                            # of a loaded state, or from before the module took another memory format
                    self.state[p]["momentum_buffer"] = torch.empty_like(p, dtype=held.dtype, device=held.device,
                                                                        memory_format=torch.preserve_format).copy_(held)
            muon_step(params, [p.grad for p in params], [self.state[p]["momentum_buffer"] for p in params],
                      **{k: v for k, v in group.items() if k in ("lr", "momentum", "nesterov", "weight_decay", "steps", "eps",
                                                                 "coefficients")})
        return loss
