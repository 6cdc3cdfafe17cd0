"""What the training-side layer operators of dance_amd are measured on: group norm with an activation on
channels_last maps (alone and with its backward pass), the orthogonalised update and the optimizer step
built on it.

A case is a dict of plain values.  `run` is one pass over what `prepare` made: in the plain form
(`own` false) elementary torch operations in 32 bits, with `own` true the calls a user of dance_amd makes.
`exact` evaluates the same definitions in 64 bits.

    group norm    x (B, C, H, W), groups of C/G channels;  mu, var over a group's channels and pixels
                  xh = (x - mu) / sqrt(var + eps),  z = xh * weight + bias,  y = act(z)
                  backward, dz = dy * act'(z):  dbias = sum dz,  dweight = sum dz xh  (over B, H, W)
                  dx = (w dz - mean_group(w dz) - xh mean_group(w dz xh)) / sqrt(var + eps)
    orthogonalize X = M / max(|M|_F, eps), then `steps` times  A = X X',  X <- a X + (b A + c A A) X
    Muon step     m <- mu m + (1 - mu) g,  u = mu m + (1 - mu) g  (Nesterov),  O = orthogonalize(u)
                  p <- p (1 - lr wd) - lr sqrt(max(1, rows / columns)) O
"""
import math

import torch

own = False

EPS = 1e-5                                   # nn.GroupNorm's
NS_STEPS, NS_EPS = 5, 1e-7
NS_A, NS_B, NS_C = 3.4445, -4.7750, 2.0315
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}

# matrices of one snake net of the shipped DANCE configuration, Conv1d weights as (out, in * taps): the head
# block, the residual blocks, the fusion layer and the three prediction layers
SNAKE_NET = [(128, 258, 9)] + [(128, 128, 9)] * 7 + [(256, 1024, 1), (256, 1280, 1), (64, 256, 1), (2, 64, 1)]
MODELS = {
    # RefineNet: three deformers and the two 3x3 layers of bottom_out
    "refine": SNAKE_NET * 3 + [(256, 256, 3, 3)] * 2,
    # one deformer alone
    "snake": SNAKE_NET,
    # the two 3x3 layers of bottom_out
    "bottom": [(256, 256, 3, 3)] * 2,
    # the attention map's producer: small and narrow matrices, one of a single row
    "attender": [(32, 1, 3, 3), (32, 32, 3, 3), (1, 32, 3, 3)],
}


# ------------------------------------------------------------------------------------------ cases
def _gn(name, b, c, h, w, groups, dtype, act, train, affine="fp32", skip=0):
    return {"name": name, "kind": "group_norm", "b": b, "c": c, "h": h, "w": w, "groups": groups, "dtype": dtype,
            "affine": affine, "act": act, "train": train, "skip": skip}


def _ns(name, batch, m, n, dtype):
    return {"name": name, "kind": "orthogonalize", "batch": batch, "m": m, "n": n, "dtype": dtype}


def listed():
    return [
        # the coarsest pyramid level of one 800 x 1216 image: a call whose latency is what counts
        _gn("gn_p5_one_image", 1, 256, 25, 38, 32, "fp32", "relu", False),
        # the stride-4 map of one image under half precision
        _gn("gn_p2_bf16", 1, 256, 200, 304, 32, "bf16", "relu", False),
        # a 257-channel map whose first channel, the attention plane, is skipped: no aligned pixel
        _gn("gn_p3_skip_plane", 2, 256, 100, 152, 32, "fp32", "silu", False, skip=1),
        # eight images' stride-4 maps: the largest call of batched inference
        _gn("gn_p2_eight_images", 8, 256, 200, 304, 32, "fp32", "relu", False),
        # a training step's layer on the coarsest level, mixed precision
        _gn("gn_train_p5_bf16", 2, 256, 25, 38, 32, "bf16", "relu", True),
        # the same on the stride-4 maps of two images a GPU, fp32
        _gn("gn_train_p2", 2, 256, 200, 304, 32, "fp32", "relu", True),
        # odd map, groups of three channels, half-precision affine parameters
        _gn("gn_train_odd_fp16", 3, 96, 67, 101, 32, "fp16", "silu", True, affine="fp16"),
        # one prediction layer's gradient: the smallest matrix product chain
        _ns("ns_prediction", 1, 64, 256, "fp32"),
        # the residual blocks of three deformers in one batch
        _ns("ns_residual_blocks", 21, 128, 1152, "fp32"),
        # a wide backbone-sized pair, half precision
        _ns("ns_wide_bf16", 2, 1024, 4096, "bf16"),
        # an optimizer step over the whole refinement head
        {"name": "muon_refine_net", "kind": "muon", "model": "refine", "dtype": "fp32"},
        # an optimizer step over the attention map's producer: launches and little else
        {"name": "muon_attender", "kind": "muon", "model": "attender", "dtype": "fp32"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["group_norm", "group_norm", "group_norm", "orthogonalize", "orthogonalize", "muon"])
    if kind == "group_norm":
        train = rng.random() < 0.5
        groups = rng.choice([1, 2, 4, 8, 16, 32])
        c = groups * _log_int(rng, 1, max(1, 512 // groups))
        limit = (2 if train else 8) * 256 * 200 * 304
        b = rng.randint(1, 8)
        # at least two values a group: of one there is no variance
        pixels = _log_int(rng, max(2, 16 // c + 1), max(2, min(limit // (b * c), 200 * 304)))
        h = max(1, _log_int(rng, 1, max(1, math.isqrt(pixels))))
        w = max(2, pixels // h)
        dtype = rng.choice(["fp32", "bf16", "fp16"])
        return {"kind": kind, "b": b, "c": c, "h": h, "w": w, "groups": groups, "dtype": dtype,
                "affine": rng.choice(["fp32", dtype]), "act": rng.choice(["relu", "silu", "none"]), "train": train,
                "skip": rng.choice([0, 0, 0, 1])}
    if kind == "orthogonalize":
        small = _log_int(rng, 2, 1024)
        wide = _log_int(rng, small, min(4096, 64 * small))
        batch = rng.choice([1, 1, 2, 3, 8, 21])
        while batch > 2 and batch * small * small * wide > 2 * 1024 * 1024 * 4096:
            batch //= 2
        m, n = (small, wide) if rng.random() < 0.7 else (wide, small)
        return {"kind": kind, "batch": batch, "m": m, "n": n, "dtype": rng.choice(["fp32", "fp32", "bf16", "fp16"])}
    # a stack of convolutions of one width, one input layer and one output layer: a head of another size
    return {"kind": kind, "model": "stack", "width": _log_int(rng, 8, 256), "inputs": rng.randint(1, 64),
            "outputs": rng.randint(1, 81), "layers": rng.randint(1, 6), "dtype": rng.choice(["fp32", "bf16"])}


def _shapes(case):
    if case["model"] != "stack":
        return MODELS[case["model"]]
    w = case["width"]
    return [(w, case["inputs"], 3, 3)] + [(w, w, 3, 3)] * case["layers"] + [(case["outputs"], w, 1, 1)]


# ----------------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, g):
    return torch.randn(shape, generator=g, device="cuda")


def _gradient(shape, g):
    """A weight's gradient: a few strong directions (the batch's common ones) and noise, small in value."""
    m, n = shape[0], math.prod(shape[1:])
    k = min(4, m, n)
    return ((_randn((m, k), g) @ _randn((k, n), g) / math.sqrt(k) + 0.3 * _randn((m, n), g)) * 1e-3).reshape(shape)


def prepare(case, seed):
    g = _generator(seed)
    dt = DTYPES[case["dtype"]]
    if case["kind"] == "group_norm":
        b, c, h, w, skip = case["b"], case["c"], case["h"], case["w"], case["skip"]
        # a convolution's output: every channel has a mean and a spread of its own
        nhwc = _randn((b, h, w, c + skip), g) * (0.5 + torch.rand((c + skip,), generator=g, device="cuda"))
        nhwc = (nhwc + 0.5 * _randn((c + skip,), g)).to(dt)
        at = DTYPES[case["affine"]]
        state = {"x": nhwc.permute(0, 3, 1, 2)[:, skip:], "weight": (1 + 0.2 * _randn((c,), g)).to(at),
                 "bias": (0.2 * _randn((c,), g)).to(at)}
        if case["train"]:
            state["dy"] = _randn((b, h, w, c), g).to(dt).permute(0, 3, 1, 2)
            for k in ("x", "weight", "bias"):
                state[k].requires_grad_(True)
        return {"case": case, **state}
    if case["kind"] == "orthogonalize":
        return {"case": case, "m": torch.stack([_gradient((case["m"], case["n"]), g) for _ in range(case["batch"])]).to(dt)}
    shapes = _shapes(case)
    # parameters, gradients and momentum as views of one flat storage each, as data-parallel buckets hold them
    state = {"case": case}
    for key in ("params", "grads", "buffers"):
        parts = [_randn(s, g) / math.sqrt(math.prod(s[1:])) if key == "params" else _gradient(s, g) for s in shapes]
        state["flat_" + key] = flat = torch.cat([t.flatten() for t in parts]).to(dt)
        state[key] = [t.view(s) for t, s in zip(flat.split([t.numel() for t in parts]), shapes)]
    return state


# ------------------------------------------------------------------------------------ plain forms
def _plain_group_norm(x, weight, bias, groups, act, dy):
    b, c, h, w = x.shape
    x32 = x.detach().permute(0, 2, 3, 1).float().reshape(b, h * w, groups, c // groups)
    g32, b32 = (t.detach().float().reshape(groups, c // groups) for t in (weight, bias))
    mean = x32.mean(dim=(1, 3), keepdim=True)
    d = x32 - mean
    rstd = 1.0 / torch.sqrt((d * d).mean(dim=(1, 3), keepdim=True) + EPS)
    xh = d * rstd
    z = xh * g32 + b32
    s = 1.0 / (1.0 + torch.exp(-z)) if act == "silu" else None
    y = torch.where(z <= 0, torch.zeros_like(z), z) if act == "relu" else z * s if act == "silu" else z

    def nchw(t):
        return t.reshape(b, h, w, c).permute(0, 3, 1, 2)

    y = nchw(y).to(x.dtype)
    if dy is None:
        return y
    dy32 = dy.permute(0, 2, 3, 1).float().reshape(b, h * w, groups, c // groups)
    if act == "relu":
        # which side of zero z lies on is decided in 64 bits
        x64 = x32.double()
        m64 = x64.mean(dim=(1, 3), keepdim=True)
        x64 = x64 - m64
        z64 = x64 / torch.sqrt((x64 * x64).mean(dim=(1, 3), keepdim=True) + EPS) * g32.double() + b32.double()
        dz = torch.where(z64 > 0, dy32, torch.zeros_like(dy32))
    elif act == "silu":
        dz = dy32 * (s * (1.0 + z * (1.0 - s)))
    else:
        dz = dy32
    dbias = dz.sum(dim=(0, 1)).reshape(c)
    dweight = (dz * xh).sum(dim=(0, 1)).reshape(c)
    wdz = dz * g32
    dx = (wdz - wdz.mean(dim=(1, 3), keepdim=True) - xh * (wdz * xh).mean(dim=(1, 3), keepdim=True)) * rstd
    return y, nchw(dx).to(x.dtype), dweight.to(weight.dtype), dbias.to(bias.dtype)


def _plain_orthogonalize(m):
    """(batch, rows, columns) -> the same, fp32"""
    x = m.float()
    tall = x.size(1) > x.size(2)
    if tall:
        x = x.transpose(1, 2).contiguous()
    x = x / torch.sqrt((x * x).sum(dim=(1, 2), keepdim=True)).clamp_min(NS_EPS)
    for _ in range(NS_STEPS):
        a = torch.bmm(x, x.transpose(1, 2).contiguous())
        x = NS_A * x + torch.bmm(NS_B * a + NS_C * torch.bmm(a, a), x)
    return x.transpose(1, 2) if tall else x


def _by_shape(shapes):
    groups = {}
    for i, s in enumerate(shapes):
        groups.setdefault(tuple(s), []).append(i)
    return groups.values()


def _plain_muon(params, grads, buffers):
    for ids in _by_shape([p.shape for p in params]):         # matrices of one shape go together
        dt, shape = params[ids[0]].dtype, params[ids[0]].shape
        rows = shape[0]
        g = torch.stack([grads[i].reshape(rows, -1) for i in ids]).float()
        m = torch.stack([buffers[i].reshape(rows, -1) for i in ids]).float() * MOMENTUM + g * (1 - MOMENTUM)
        o = _plain_orthogonalize(m * MOMENTUM + g * (1 - MOMENTUM))
        p = torch.stack([params[i].reshape(rows, -1) for i in ids]).float() * (1 - LR * DECAY)
        p = (p - LR * math.sqrt(max(1.0, rows / o.size(2))) * o).to(dt)
        m = m.to(dt)
        for k, i in enumerate(ids):
            params[i].copy_(p[k].reshape(shape))
            buffers[i].copy_(m[k].reshape(shape))


def run(state):
    case = state["case"]
    if case["kind"] == "group_norm":
        act = None if case["act"] == "none" else case["act"]
        x, weight, bias, dy = state["x"], state["weight"], state["bias"], state.get("dy")
        if not own:
            return _plain_group_norm(x, weight, bias, case["groups"], act, dy)
        from dance_amd import ops
        y = ops.group_norm_act(x, case["groups"], weight, bias, eps=EPS, act=act)
        if dy is None:
            return y
        return (y.detach(),) + torch.autograd.grad(y, (x, weight, bias), dy)
    if case["kind"] == "orthogonalize":
        if not own:
            return _plain_orthogonalize(state["m"]).to(state["m"].dtype)
        from dance_amd import ops
        return ops.orthogonalize(state["m"], steps=NS_STEPS, eps=NS_EPS, coefficients=(NS_A, NS_B, NS_C))
    if not own:
        _plain_muon(state["params"], state["grads"], state["buffers"])
    else:
        from dance_amd import optim
        optim.muon_step(state["params"], state["grads"], state["buffers"], lr=LR, momentum=MOMENTUM, nesterov=True,
                        weight_decay=DECAY, steps=NS_STEPS, eps=NS_EPS, coefficients=(NS_A, NS_B, NS_C))
    return {"params": state["flat_params"], "buffers": state["flat_buffers"]}


# ------------------------------------------------------------------------------------------- work
def _chain_flops(m, n):
    """The Newton-Schulz chain on the smaller Gram matrix: its two symmetric products by half."""
    r, k = min(m, n), max(m, n)
    return NS_STEPS * (r * (r + 1) * k + r * r * (r + 1) + 2 * r * r * k)


def work(case):
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if case["kind"] == "group_norm":
        items = case["b"] * case["c"] * case["h"] * case["w"]
        # forward: x in, y out; with the backward pass dy in and dx out as well
        return {"bytes": items * size * (4 if case["train"] else 2), "flops": items * (24 if case["train"] else 8)}
    if case["kind"] == "orthogonalize":
        return {"bytes": 2 * case["batch"] * case["m"] * case["n"] * size,
                "flops": case["batch"] * _chain_flops(case["m"], case["n"])}
    mats = [(s[0], math.prod(s[1:])) for s in _shapes(case)]
    # parameter and momentum read and written, the gradient read
    return {"bytes": sum(5 * m * n * size for m, n in mats), "flops": sum(_chain_flops(m, n) for m, n in mats)}


# ------------------------------------------------------------------------------------------ exact
def _exact_group_norm(x, weight, bias, groups, act, dy):
    x = x.detach().double()
    gx = x.reshape(x.size(0), groups, -1)
    var, mean = torch.var_mean(gx, dim=2, correction=0, keepdim=True)
    inv = torch.rsqrt(var + EPS)
    xh = ((gx - mean) * inv).reshape(x.shape)
    wt, bs = (t.detach().double()[None, :, None, None] for t in (weight, bias))
    z = xh * wt + bs
    y = torch.where(z > 0, z, torch.zeros_like(z)) if act == "relu" else z * torch.sigmoid(z) if act == "silu" else z
    if dy is None:
        return y
    dz = dy.double()
    if act == "relu":
        dz = dz * (z > 0)
    elif act == "silu":
        s = torch.sigmoid(z)
        dz = dz * (s + z * s * (1 - s))
    wdz = (dz * wt).reshape(gx.shape)
    gxh = xh.reshape(gx.shape)
    dx = inv * (wdz - wdz.mean(2, keepdim=True) - gxh * (wdz * gxh).mean(2, keepdim=True))
    return y, dx.reshape(x.shape), (dz * xh).sum(dim=(0, 2, 3)), dz.sum(dim=(0, 2, 3))


def _exact_orthogonalize(m):
    """The chain with its products taken from the right: X (a + b X'X + c (X'X)^2), by products with X alone."""
    x = m.double()
    x = x / max(float(torch.linalg.norm(x)), NS_EPS)
    for _ in range(NS_STEPS):
        gx = (x @ x.t()) @ x if x.size(0) <= x.size(1) else x @ (x.t() @ x)
        ggx = (x @ x.t()) @ gx if x.size(0) <= x.size(1) else gx @ (x.t() @ x)
        x = NS_A * x + NS_B * gx + NS_C * ggx
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "group_norm":
        act = None if case["act"] == "none" else case["act"]
        return _exact_group_norm(s["x"], s["weight"], s["bias"], case["groups"], act, s.get("dy"))
    if case["kind"] == "orthogonalize":
        return torch.stack([_exact_orthogonalize(m) for m in s["m"]])
    params, buffers = [], []
    for p, g, b in zip(s["params"], s["grads"], s["buffers"]):
        g64, p64 = g.double().flatten(1), p.double().flatten(1)
        m64 = torch.lerp(b.double().flatten(1), g64, 1 - MOMENTUM)
        o = _exact_orthogonalize(torch.lerp(g64, m64, MOMENTUM))
        p64 = p64 - LR * (DECAY * p64 + math.sqrt(max(1.0, p64.size(0) / p64.size(1))) * o)
        params.append(p64.flatten())
        buffers.append(m64.flatten())
    return {"params": torch.cat(params), "buffers": torch.cat(buffers)}
