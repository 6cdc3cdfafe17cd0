"""Muon: momentum SGD whose update is orthogonalised (ops.orthogonalize), for the weight matrices of the heads.

A parameter of more than two dimensions is its (first dimension, the rest) matrix: a convolution's weight is
(out channels, in channels * taps).  Vectors (biases, norm weights) are not Muon's: give them to another
optimizer.  The whole step -- momentum, Nesterov's look-ahead, the chain of products, the parameter update --
is one chain of launches for all matrices of one type and device, whatever their shapes.

The reference trains with Detectron2's SGD (train_net.py:22-70) and has no counterpart.
"""
import torch

from ._lib import MuonItemStruct, check, lib, on_device, stream_of
from .ops import DTYPE_CODES, NS_COEFFICIENTS, _need_gpu, _scratch, check_newton_schulz


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
    chains, seen = {}, set()
    for p, g, m in zip(params, grads, momentum_buffers):
        _need_gpu(p, g, m)
        if p.dim() < 2 or p.dtype not in DTYPE_CODES:
            raise RuntimeError("%s: matrices of fp32, fp16 or bf16 expected, got a %s parameter of shape %s"
                               % (what, p.dtype, tuple(p.shape)))
        for name, t in (("gradient", g), ("momentum buffer", m)):
            if t.shape != p.shape or t.dtype != p.dtype or t.device != p.device:
                raise RuntimeError("%s: a %s %s %s on %s for a parameter %s %s on %s"
                                   % (what, name, tuple(t.shape), t.dtype, t.device, tuple(p.shape), p.dtype, p.device))
        if p.numel() == 0:
            continue
        if m.stride() != p.stride() or not _rows_outermost(p):
            raise RuntimeError("%s: parameter and momentum buffer must be dense, rows outermost, with equal strides, got %s "
                               "and %s of shape %s" % (what, p.stride(), m.stride(), tuple(p.shape)))
        for t in (p, m):
            if t.data_ptr() in seen:
                raise RuntimeError("%s: a parameter or momentum buffer appears twice" % what)
            seen.add(t.data_ptr())
        if g.stride() != p.stride():
            g = torch.empty_strided(p.shape, p.stride(), dtype=p.dtype, device=p.device).copy_(g)
        chains.setdefault((p.device, p.dtype), []).append((p, g, m))
    h = lib()
    for (dev, dtype), chain in chains.items():
        items = (MuonItemStruct * len(chain))()
        for it, (p, g, m) in zip(items, chain):
            it.param, it.grad, it.momentum = p.data_ptr(), g.data_ptr(), m.data_ptr()
            it.rows, it.cols = p.size(0), p.numel() // p.size(0)
        nbytes = h.dance_muon_workspace_bytes(items, len(chain))
        ws = _scratch(nbytes, dev)
        with on_device(dev):
            check(h.dance_muon_step(items, len(chain), DTYPE_CODES[dtype], lr, momentum, int(bool(nesterov)), weight_decay,
                                    steps, a, b, c, eps, ws.data_ptr() if nbytes else None, nbytes, stream_of(dev)), what)
        # written behind autograd's back: what caches by version (saved tensors, the modules' packed weights) must see it
        torch.autograd.graph.increment_version([t for p, _, m in chain for t in (p, m)])


class Muon(torch.optim.Optimizer):
    """torch.optim optimizer over muon_step.  Every parameter a matrix (two dimensions or more, the first one the
    rows); parameters without a gradient are left as they are."""

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
                if "momentum_buffer" not in self.state[p]:
                    self.state[p]["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.preserve_format)
            muon_step(params, [p.grad for p in params], [self.state[p]["momentum_buffer"] for p in params],
                      **{k: v for k, v in group.items() if k in ("lr", "momentum", "nesterov", "weight_decay", "steps", "eps",
                                                                 "coefficients")})
        return loss
