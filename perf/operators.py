"""What the framework's Muon and group-norm operators cost: cases, inputs, plain forms and 64-bit values.

Four kinds of case:
  ns       Newton-Schulz orthogonalisation of one matrix or a stack of them (``ops.kernels.newton_schulz``)
  muon     one Muon step over a list of weight matrices (``ops.kernels.muon_step``, what ``ops.optim.FusedMuon`` runs)
  gn_fwd   group norm + activation over channels-last activations (``ops.kernels.gn_fwd``)
  gn_bwd   its backward pass (``ops.kernels.gn_bwd``)

``own`` selects what ``run`` calls: the framework's kernels, or the same mathematics in elementary torch operations.
"""
import math

import torch

own = False

COEFFS = (3.4445, -4.7750, 2.0315)
STEPS = 5
NS_EPS = 1e-7
GN_EPS = 1e-5
LR, MOMENTUM, WEIGHT_DECAY = 1e-3, 0.95, 0.1
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# [rows, cols] of VGG16's thirteen convolution weights as matrices: output channels x (9 * input channels)
VGG16_CONVS = ((64, 27), (64, 576), (128, 576), (128, 1152), (256, 1152), (256, 2304), (256, 2304), (512, 2304),
               (512, 4608), (512, 4608), (512, 4608), (512, 4608), (512, 4608))


def listed():
    return [
        # the update of one 64-channel convolution: every product is tiny, the number of launches counts
        dict(name="ns_64x576", kind="ns", batch=1, rows=64, cols=576, dtype="f32", rank=16),
        # one of the 512-channel convolutions
        dict(name="ns_512x4608", kind="ns", batch=1, rows=512, cols=4608, dtype="bf16", rank=64),
        # a stack of tall matrices of odd sizes: neither side a multiple of anything
        dict(name="ns_3x1001x333", kind="ns", batch=3, rows=1001, cols=333, dtype="f32", rank=40),
        # the second classifier layer, square
        dict(name="ns_4096x4096", kind="ns", batch=1, rows=4096, cols=4096, dtype="bf16", rank=256),
        # optimizer step over VGG16's convolution weights
        dict(name="muon_vgg16_convs", kind="muon", shapes="vgg16", rows=0, cols=0, dtype="f32", rank=32),
        # optimizer step over VGG16's first classifier layer: the largest matrix of the model, bf16 gradients
        dict(name="muon_4096x25088", kind="muon", shapes="one", rows=4096, cols=25088, dtype="bf16", rank=64),
        # four images per GPU, last block: latency
        dict(name="gn_fwd_4x14x14x512", kind="gn_fwd", n=4, h=14, w=14, c=512, groups=32, act="relu", dtype="bf16"),
        # first block at 64 images per GPU: the largest activation
        dict(name="gn_fwd_64x224x224x64", kind="gn_fwd", n=64, h=224, w=224, c=64, groups=32, act="relu", dtype="bf16"),
        # odd spatial size and a channel count that is no multiple of 8
        dict(name="gn_fwd_5x27x19x60_silu", kind="gn_fwd", n=5, h=27, w=19, c=60, groups=12, act="silu", dtype="f32"),
        # four images per GPU, fourth block
        dict(name="gn_bwd_4x28x28x512", kind="gn_bwd", n=4, h=28, w=28, c=512, groups=32, act="relu", dtype="bf16"),
        # third block at 64 images per GPU
        dict(name="gn_bwd_64x56x56x256", kind="gn_bwd", n=64, h=56, w=56, c=256, groups=32, act="relu", dtype="bf16"),
        # odd sizes in half precision
        dict(name="gn_bwd_7x33x45x72_silu", kind="gn_bwd", n=7, h=33, w=45, c=72, groups=9, act="silu", dtype="f16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("ns", "muon", "gn_fwd", "gn_bwd"))
    if kind in ("ns", "muon"):
        rows, cols = _log_int(rng, 16, 2500), _log_int(rng, 16, 2500)
        if rng.random() < 0.3:
            cols = min(4 * cols, 8000)
        rank = _log_int(rng, 1, min(rows, cols))
        if kind == "muon":
            return dict(kind=kind, shapes="one", rows=rows, cols=cols, dtype=rng.choice(("f32", "bf16")), rank=rank)
        return dict(kind=kind, batch=rng.randint(1, 4), rows=rows, cols=cols, dtype=rng.choice(("f32", "bf16")), rank=rank)
    dtype = rng.choice(("bf16", "f16", "f32"))
    groups = rng.choice((1, 3, 4, 8, 16, 32))
    c = groups * _log_int(rng, 1, max(2, 768 // groups))
    n, h, w = _log_int(rng, 1, 96), _log_int(rng, 1, 160), _log_int(rng, 1, 160)
    while n * h * w * c > 60_000_000:
        n, h, w = (n + 1) // 2, (3 * h + 3) // 4, (3 * w + 3) // 4
    # a sign that f32 cannot decide is one whole gradient: the ReLU goes with the types whose values are coarse
    act = rng.choice(("none", "silu")) if dtype == "f32" else rng.choice(("none", "relu", "silu"))
    return dict(kind=kind, n=n, h=h, w=w, c=c, groups=groups, act=act, dtype=dtype)


def _shapes(case):
    return list(VGG16_CONVS) if case["shapes"] == "vgg16" else [(case["rows"], case["cols"])]


def _gradient(g, rows, cols, rank, dtype, scale=1e-3):
    """What a backward pass leaves: a product of activations and output gradients (few strong directions, as many
    as there are samples) over a floor of noise, at the magnitude of a mean over a batch."""
    rank = min(rank, rows, cols)
    x = torch.randn(rows, rank, generator=g, device="cuda") @ torch.randn(rank, cols, generator=g, device="cuda")
    x = x / math.sqrt(rank) + 0.1 * torch.randn(rows, cols, generator=g, device="cuda")
    return (x * scale).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    kind = case["kind"]
    if kind == "ns":
        xs = [_gradient(g, case["rows"], case["cols"], case["rank"], dt) for _ in range(case["batch"])]
        return dict(kind=kind, x=torch.stack(xs) if case["batch"] > 1 else xs[0])
    if kind == "muon":
        params, grads, bufs, lps = [], [], [], []
        for rows, cols in _shapes(case):
            params.append(torch.randn(rows, cols, generator=g, device="cuda") * math.sqrt(2.0 / max(rows, cols)))
            grads.append(_gradient(g, rows, cols, case["rank"], dt))
            bufs.append(_gradient(g, rows, cols, case["rank"], torch.float32))
            lps.append(params[-1].to(torch.bfloat16))
        return dict(kind=kind, params=params, grads=grads, bufs=bufs, lps=lps)
    shape = (case["n"], case["h"], case["w"], case["c"])
    c, groups = case["c"], case["groups"]
    # pre-activations: a mean and a spread of their own for every channel
    mean = 0.5 * torch.randn(c, generator=g, device="cuda")
    std = 0.5 + torch.rand(c, generator=g, device="cuda")
    x = (torch.randn(shape, generator=g, device="cuda") * std + mean).to(dt)
    st = dict(kind=kind, x=x, groups=groups, act=case["act"],
              gamma=1.0 + 0.2 * torch.randn(c, generator=g, device="cuda"),
              beta=0.2 * torch.randn(c, generator=g, device="cuda"))
    if kind == "gn_bwd":
        st["dy"] = torch.randn(shape, generator=g, device="cuda").to(dt)
        st["stats"] = _gn_stats(x, groups)          # what the forward pass left
        st["dgamma"] = torch.empty(c, device="cuda")
        st["dbeta"] = torch.empty(c, device="cuda")
    return st


# ------------------------------------------------------------------ plain forms
def _newton_schulz(x):
    a, b, c = COEFFS
    tall = x.shape[-2] > x.shape[-1]
    x = x.float()
    if tall:
        x = x.transpose(-2, -1)
    # (a sum of up to 10^8 squares: in 64 bits)
    norm = x.double().square().sum((-2, -1), keepdim=True).sqrt()
    x = (x / (norm + NS_EPS)).float()
    for _ in range(STEPS):
        s = x @ x.transpose(-2, -1)
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.transpose(-2, -1) if tall else x


def _muon_step(st):
    for p, g, m, lp in zip(st["params"], st["grads"], st["bufs"], st["lps"]):
        d = g.float()
        m.mul_(MOMENTUM).add_(d, alpha=1 - MOMENTUM)
        o = _newton_schulz((1 - MOMENTUM) * d + MOMENTUM * m)
        p.mul_(1 - LR * WEIGHT_DECAY).add_(o, alpha=-LR * 0.2 * math.sqrt(max(p.shape)))
        lp.copy_(p)
    return dict(params=st["params"], bufs=st["bufs"], lps=st["lps"])


def _gn_stats(x, groups):
    n, c = x.shape[0], x.shape[-1]
    v = x.reshape(n, -1, groups, c // groups).double()
    mean = v.mean((1, 3), keepdim=True)
    var = (v - mean).square().mean((1, 3))
    return torch.stack((mean.view(n, groups), (var + GN_EPS).rsqrt()), -1).float()


def _gn_plain_stats(x, groups):
    n, c = x.shape[0], x.shape[-1]
    v = x.reshape(n, -1, groups, c // groups).float()
    mean = v.mean((1, 3), keepdim=True)
    var = (v - mean).square().mean((1, 3))
    return torch.stack((mean.view(n, groups), (var + GN_EPS).rsqrt()), -1)


def _gn_xhat(x, stats, groups):
    n, c = x.shape[0], x.shape[-1]
    v = x.reshape(n, -1, groups, c // groups).to(stats.dtype)
    return (v - stats[:, None, :, None, 0]) * stats[:, None, :, None, 1]


def _gn_fwd(st):
    x, groups = st["x"], st["groups"]
    stats = _gn_plain_stats(x, groups)
    z = _gn_xhat(x, stats, groups).reshape(x.shape) * st["gamma"] + st["beta"]
    if st["act"] == "relu":
        z = z.clamp_min(0)
    elif st["act"] == "silu":
        z = z / (1 + torch.exp(-z))
    return z.to(x.dtype), stats


def _gn_act_grad(z, dy, act):
    if act == "relu":
        return torch.where(z > 0, dy, torch.zeros_like(dy))
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return dy * s * (1 + z * (1 - s))
    return dy


def _gn_bwd(st):
    x, groups, gamma = st["x"], st["groups"], st["gamma"]
    n, c = x.shape[0], x.shape[-1]
    xhat = _gn_xhat(x, st["stats"], groups)                                          # [n, hw, g, c/g]
    dz = _gn_act_grad(xhat.reshape(n, -1, c) * gamma + st["beta"], st["dy"].float().reshape(n, -1, c), st["act"])
    dbeta = dz.sum((0, 1))
    dgamma = (dz * xhat.reshape(n, -1, c)).sum((0, 1))
    dxhat = (dz * gamma).view_as(xhat)
    m1 = dxhat.mean((1, 3), keepdim=True)
    m2 = (dxhat * xhat).mean((1, 3), keepdim=True)
    dx = (dxhat - m1 - xhat * m2) * st["stats"][:, None, :, None, 1]
    return dx.reshape(x.shape).to(x.dtype), dgamma, dbeta


def run(state):
    kind = state["kind"]
    if own:
        from distributed_training_pytorch_amd.ops import kernels as K
        if kind == "ns":
            return K.newton_schulz(state["x"], steps=STEPS, coeffs=COEFFS, eps=NS_EPS, out_dtype=torch.bfloat16)
        if kind == "muon":
            K.muon_step(state["params"], state["grads"], state["bufs"], state["lps"], lr=LR, momentum=MOMENTUM,
                        nesterov=True, weight_decay=WEIGHT_DECAY, steps=STEPS, coeffs=COEFFS, eps=NS_EPS,
                        adjust_lr="match_rms_adamw")
            return dict(params=state["params"], bufs=state["bufs"], lps=state["lps"])
        if kind == "gn_fwd":
            return K.gn_fwd(state["x"], state["gamma"], state["beta"], state["groups"], eps=GN_EPS, act=state["act"])
        dx = K.gn_bwd(state["x"], state["dy"], state["gamma"], state["beta"], state["stats"], state["groups"],
                      state["dgamma"], state["dbeta"], act=state["act"])
        return dx, state["dgamma"], state["dbeta"]
    if kind == "ns":
        return _newton_schulz(state["x"]).to(torch.bfloat16)
    if kind == "muon":
        return _muon_step(state)
    return _gn_fwd(state) if kind == "gn_fwd" else _gn_bwd(state)


# ------------------------------------------------------------------ what a pass cannot do without
def _ns_flops(rows, cols):
    # one Gram matrix and one product with the input (the first symmetric: half of it), and between them the
    # products of symmetric m x m matrices (half of each) that the polynomials of STEPS steps need:
    # A*A, P*A, P*(P*A), P*Q a step; the first has no Q yet, the last needs no next A
    m, n = min(rows, cols), max(rows, cols)
    return 3.0 * m * m * n + (4 * STEPS - 3) * float(m) ** 3


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
    kind = case["kind"]
    if kind == "ns":
        n = case["batch"] * case["rows"] * case["cols"]
        return dict(bytes=n * (size + 2), flops=case["batch"] * _ns_flops(case["rows"], case["cols"]))
    if kind == "muon":
        n = sum(r * c for r, c in _shapes(case))
        # gradient and momentum read, momentum written, weights read and written, bf16 copy written
        return dict(bytes=n * (size + 4 + 4 + 4 + 4 + 2), flops=sum(_ns_flops(r, c) for r, c in _shapes(case)))
    n = case["n"] * case["h"] * case["w"] * case["c"]
    if kind == "gn_fwd":
        return dict(bytes=2 * n * size, flops=10.0 * n)
    return dict(bytes=3 * n * size, flops=20.0 * n)


# ------------------------------------------------------------------ the definitions in 64 bits
def _orthogonalised(u):
    a, b, c = COEFFS
    y = u.double()
    y = y / (torch.linalg.vector_norm(y) + NS_EPS)
    for _ in range(STEPS):
        if y.shape[0] <= y.shape[1]:
            s = torch.mm(y, y.t())
            y = a * y + b * torch.mm(s, y) + c * torch.mm(s, torch.mm(s, y))
        else:
            s = torch.mm(y.t(), y)
            y = a * y + b * torch.mm(y, s) + c * torch.mm(torch.mm(y, s), s)
    return y


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "ns":
        x = st["x"]
        return torch.stack([_orthogonalised(v) for v in x]) if x.dim() == 3 else _orthogonalised(x)
    if kind == "muon":
        params, bufs = [], []
        for p, g, m in zip(st["params"], st["grads"], st["bufs"]):
            m64 = MOMENTUM * m.double() + (1 - MOMENTUM) * g.double()
            o = _orthogonalised(MOMENTUM * m64 + (1 - MOMENTUM) * g.double())
            params.append(p.double() * (1 - LR * WEIGHT_DECAY) - LR * 0.2 * math.sqrt(max(p.shape)) * o)
            bufs.append(m64)
        return dict(params=params, bufs=bufs, lps=params)
    # one image at a time
    groups, act = case["groups"], case["act"]
    n, c = case["n"], case["c"]
    gamma, beta = st["gamma"].double().view(groups, -1, 1), st["beta"].double().view(groups, -1, 1)
    ys, stats = [], []
    dgamma, dbeta = torch.zeros_like(gamma), torch.zeros_like(beta)
    for i in range(n):
        v = st["x"][i].double().reshape(-1, c).t().reshape(groups, c // groups, -1)      # [g, c/g, hw]
        mu = v.mean((1, 2), keepdim=True)
        sd = torch.sqrt(((v - mu) ** 2).mean((1, 2), keepdim=True) + GN_EPS)
        xh = (v - mu) / sd
        z = gamma * xh + beta
        if kind == "gn_fwd":
            out = torch.relu(z) if act == "relu" else z * torch.sigmoid(z) if act == "silu" else z
            stats.append(torch.stack((mu.flatten(), 1 / sd.flatten()), -1))
        else:
            dy = st["dy"][i].double().reshape(-1, c).t().reshape(groups, c // groups, -1)
            if act == "relu":
                dz = dy * (z > 0)
            elif act == "silu":
                s = torch.sigmoid(z)
                dz = dy * (s + z * s * (1 - s))
            else:
                dz = dy
            dgamma += (dz * xh).sum(2, keepdim=True)
            dbeta += dz.sum(2, keepdim=True)
            e = dz * gamma
            out = (e - e.mean((1, 2), keepdim=True) - xh * (e * xh).mean((1, 2), keepdim=True)) / sd
        ys.append(out.reshape(c, -1).t().reshape(st["x"][i].shape))
    if kind == "gn_fwd":
        return torch.stack(ys), torch.stack(stats)
    return torch.stack(ys), dgamma.flatten(), dbeta.flatten()
