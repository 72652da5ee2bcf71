"""The operators of ``dd3d_amd.ops`` for ragged channels-last rows -- group norm with an activation, its first and second gradient, dropout
from a counter-based generator, and the two in one pass -- as cases that can be timed, beside their plain form in elementary torch.

A batch of clouds is a matrix of rows ``x[M, C]``; cloud ``b`` owns the rows ``seg_off[b] : seg_off[b + 1]``.  Group norm takes its
statistics over the rows of one cloud and the ``C / G`` channels of one group.  Dropout keeps element (row, channel) by word ``channel % 4``
of Philox4x32-10 at counter ``(row * ceil(C / 4) + channel // 4, call)`` under key ``seed``.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_EPS = 1e-5


# ------------------------------------------------------------------------------------------------------------------------- cases
def _case(name, op, rows, clouds, channels, groups, dtype, act="none", p=0.0, spread=0.3):
    return {"name": name, "op": op, "rows": rows, "clouds": clouds, "channels": channels, "groups": groups, "dtype": dtype, "act": act, "p": p,
            "spread": spread}


def listed():
    return [
        # one class's synthetic clouds (10 clouds of 250 points) through a frozen network: a call where latency counts
        _case("norm_syn_class", "norm", 2157, 10, 128, 8, "f32", "relu"),
        # the real digits of all ten classes in evaluation, half precision
        _case("norm_digits_bf16", "norm", 209920, 2560, 128, 32, "bf16", "gelu"),
        # a training step's norm over one class of real digits
        _case("train_class", "train", 21000, 256, 128, 8, "f32", "silu"),
        # ... and over all ten classes at once (the class-batched step)
        _case("train_digits", "train", 209920, 2560, 128, 8, "f32", "silu"),
        # few clouds of very different sizes (scenes): the long ones do not fit one compute unit
        _case("train_scenes_bf16", "train", 400003, 7, 96, 6, "bf16", "gelu", spread=1.5),
        # gradient matching: the synthetic clouds of ten classes, differentiated twice
        _case("second_syn", "second", 21570, 100, 128, 8, "f32", "silu"),
        # ... and of the forty classes with 1024 points a cloud
        _case("second_shells", "second", 300000, 400, 128, 16, "f32", "gelu", spread=0.1),
        # dropout in front of a classifier: one feature row a cloud
        _case("dropout_head", "dropout", 256, 256, 1024, 1, "f32", p=0.5),
        # dropout on the voxel rows of a large batch, half precision
        _case("dropout_rows_bf16", "dropout", 800001, 1, 128, 1, "bf16", p=0.1),
        # the level of a network in one pass, at widths that fill no vector, with clouds from nothing to a few thousand rows
        _case("block_odd_f16", "block", 30011, 97, 100, 5, "f16", "silu", p=0.3, spread=1.2),
        # ... over the real clouds of a large configuration
        _case("block_shells", "block", 400000, 512, 128, 8, "f32", "gelu", p=0.2, spread=0.15),
    ]


def draw(rng):
    op = rng.choice(["norm", "train", "second", "dropout", "block"])
    channels = rng.choice([rng.randint(8, 64), 4 * rng.randint(4, 48), 8 * rng.randint(4, 40), 64, 128, 256])
    most = min(400000, 38000000 // channels)   # elements of the largest listed case that is differentiated twice
    rows = int(round(math.exp(rng.uniform(math.log(64), math.log(most)))))
    clouds = max(1, min(3000, int(rows / math.exp(rng.uniform(math.log(16), math.log(4 * rows))))))
    groups = rng.choice([d for d in range(1, channels + 1) if channels % d == 0 and (d <= 32 or d == channels)])
    return {"op": op, "rows": rows, "clouds": clouds, "channels": channels, "groups": groups, "dtype": rng.choice(["f32", "bf16", "f16"]),
            # a derivative that jumps has no value next to its border, so those activations are drawn for the forward pass only
            "act": "none" if op == "dropout" else rng.choice(["relu", "silu", "gelu", "leaky_relu", "none"] if op == "norm" else ["silu", "gelu", "none"]),
            "p": rng.choice([0.1, 0.25, 0.5, 0.7]) if op in ("dropout", "block") else 0.0, "spread": rng.choice([0.1, 0.4, 1.0, 1.5])}


def prepare(case, seed):
    dev = torch.device("cuda")
    host, gen = torch.Generator().manual_seed(seed), torch.Generator(device=dev).manual_seed(seed)
    M, B, C, t = case["rows"], case["clouds"], case["channels"], _TYPES[case["dtype"]]
    share = torch.exp(case["spread"] * torch.randn(B, generator=host, dtype=torch.float64))
    ends = torch.round(torch.cumsum(share, 0) / share.sum() * M).to(torch.int32)
    ends[-1] = M
    seg_off = torch.cat([torch.zeros(1, dtype=torch.int32), ends])
    randn = lambda *shape: torch.randn(shape, generator=gen, device=dev)  # noqa: E731
    state = dict(case, seg_off=seg_off.to(dev), x=(randn(M, C) * torch.exp(0.3 * randn(C)) + 0.5 * randn(C)).to(t).requires_grad_(),
                 key=torch.tensor([0x1234567890ABCDEF ^ seed, seed], dtype=torch.int64, device=dev))
    if case["op"] != "norm":
        state["dy"] = randn(M, C).to(t)
    if case["op"] != "dropout":
        state["w"], state["b"] = (1 + 0.2 * randn(C)).requires_grad_(), (0.2 * randn(C)).requires_grad_()
    if case["op"] == "second":
        state["dy"].requires_grad_()
        state["ggx"], state["ggw"], state["ggb"] = randn(M, C).to(t), randn(C), randn(C)
    return state


def work(case):
    M, C, op = case["rows"], case["channels"], case["op"]
    size = 4 if case["dtype"] == "f32" else 2
    # matrices [M, C] that go in and out: x -> y;  x, dy -> y, dx;  x, dy, ggx -> y, dx, d(dy), d(x);  x, dy -> y, dx
    mats = {"norm": 2, "train": 4, "second": 7, "dropout": 4, "block": 4}[op]
    flops = {"norm": 20, "train": 50, "second": 110, "dropout": 50, "block": 100}[op]
    vecs = {"norm": 2, "train": 4, "second": 8, "dropout": 0, "block": 4}[op]
    return {"bytes": mats * M * C * size + vecs * C * 4 + (case["clouds"] + 1) * 4, "flops": flops * M * C}


# ------------------------------------------------------------------------------------------------------------------- the plain form
def _cut(v):
    return v & 0xFFFFFFFF


def _wide_product(a, m):
    """High and low 32 bits of a * m (a: int64 tensor of 32-bit words, m: 32-bit constant) without leaving 63 bits."""
    low, high = a * (m & 0xFFFF), a * (m >> 16)
    mid = (low >> 16) + high
    return mid >> 16, _cut((_cut(mid) << 16) | (low & 0xFFFF))


def _keep(case, key):
    """Truth values [M, C]: the elements that dropout keeps."""
    M, C = case["rows"], case["channels"]
    quads = (C + 3) // 4
    block = torch.arange(M * quads, dtype=torch.int64, device=key.device)
    k0, k1 = _cut(key[0]), _cut(key[0] >> 32)
    c0, c1, c2, c3 = _cut(block), block >> 32, _cut(key[1]).expand_as(block), _cut(key[1] >> 32).expand_as(block)
    for _ in range(10):
        h0, l0 = _wide_product(c0, 0xD2511F53)
        h1, l1 = _wide_product(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = _cut(k0 + 0x9E3779B9), _cut(k1 + 0xBB67AE85)
    words = torch.stack([c0, c1, c2, c3], 1).view(M, 4 * quads)[:, :C]
    return words >= round(case["p"] * 2.0 ** 32)


def _act(name, u, order):
    """phi(u), phi'(u), phi''(u) up to ``order``, elementwise."""
    if name in ("none", "relu", "leaky_relu"):
        slope = {"none": 1.0, "relu": 0.0, "leaky_relu": 0.01}[name]
        up = u > 0
        d = torch.where(up, 1.0, slope)
        return [torch.where(up, u, u * slope), d, torch.zeros_like(u)][: order + 1]
    if name == "silu":
        s = 1 / (1 + torch.exp(-u))
        t = s * (1 - s)
        return [u * s, s + u * t, t * (2 + u * (1 - 2 * s))][: order + 1]
    cdf, pdf = 0.5 * (1 + torch.erf(u * math.sqrt(0.5))), torch.exp(-0.5 * u * u) / math.sqrt(2 * math.pi)
    return [u * cdf, cdf + u * pdf, pdf * (2 - u * u)][: order + 1]


class _Clouds:
    """Sums over (cloud, group), taken in 64 bits."""

    def __init__(self, case, seg_off):
        self.G, self.Cg = case["groups"], case["channels"] // case["groups"]
        ends = seg_off[1:].long()
        row = torch.arange(case["rows"], device=ends.device)
        self.ids = torch.searchsorted(ends, row, right=True)
        self.many = max(1, 65536 // case["clouds"])   # partial sums a cloud: additions to one place wait for each other
        self.part = self.ids * self.many + row % self.many
        self.n = ((ends - seg_off[:-1]) * self.Cg).clamp(min=1).double()[:, None]

    def mean(self, t):
        rows = t.double().view(t.shape[0], self.G, self.Cg).sum(2)
        parts = torch.zeros(self.many * len(self.n), self.G, dtype=rows.dtype, device=rows.device).index_add(0, self.part, rows)
        return parts.view(-1, self.many, self.G).sum(1) / self.n

    def spread(self, s):
        """[B, G] -> [M, C], 32 bits"""
        return s.float()[self.ids].repeat_interleave(self.Cg, 1)


def _plain(state):
    op, x = state["op"], state["x"].detach()
    t, x = x.dtype, x.float()
    keep, scale = (_keep(state, state["key"]), 1 / (1 - state["p"])) if state["p"] > 0 else (None, 1.0)
    drop = (lambda v: torch.where(keep, v * scale, 0.0)) if keep is not None else (lambda v: v)  # noqa: E731
    if op == "dropout":
        return drop(x).to(t), drop(state["dy"].float()).to(t)
    w, b, name = state["w"].detach(), state["b"].detach(), state["act"]
    cl = _Clouds(state, state["seg_off"])
    cen = x - cl.spread(cl.mean(x))
    cen = cen - cl.spread(cl.mean(cen))
    r = cl.spread(1 / torch.sqrt(cl.mean(cen * cen) + _EPS))
    xh = cen * r
    f = _act(name, w * xh + b, 2 if op == "second" else 0 if op == "norm" else 1)
    y = drop(f[0]).to(t)
    if op == "norm":
        return y
    dy = state["dy"].detach().float()
    total = lambda v: v.double().sum(0).float()  # noqa: E731
    g = drop(dy) * f[1]
    h = g * w
    m1, m2 = cl.spread(cl.mean(h)), cl.spread(cl.mean(h * xh))
    first = (y, (r * (h - m1 - xh * m2)).to(t), total(g * xh), total(g))
    if op != "second":
        return first
    P, q, s = state["ggx"].float(), state["ggw"], state["ggb"]
    mp, mp2, mph = (cl.spread(cl.mean(v)) for v in (P, P * xh, P * h))
    v = r * (P - mp - xh * mp2)
    gb = w * v + q * xh + s
    ub = gb * dy * f[2]
    X = -r * (h * mp2 + P * m2) + q * g + w * ub
    ddx = r * (X - cl.spread(cl.mean(X)) - xh * (cl.spread(cl.mean(X * xh)) + r * (mph - mp * m1 - mp2 * m2)))
    return first + ((gb * f[1]).to(t), ddx.to(t), total(g * v + ub * xh), total(ub))


# ------------------------------------------------------------------------------------------------------------- the framework's calls
def run(state):
    if not own:
        with torch.no_grad():
            return _plain(state)
    from dd3d_amd import ops
    op, x = state["op"], state["x"]
    if op == "dropout":
        y = ops.dropout(x, state["p"], state["key"])
        return (y.detach(),) + torch.autograd.grad(y, x, state["dy"])
    w, b = state["w"], state["b"]
    norm = lambda: ops.group_norm(x, state["seg_off"], state["groups"], w, b, eps=_EPS, activation=state["act"],  # noqa: E731
                                  dropout=state["p"], key=state["key"] if state["p"] > 0 else None)
    if op == "norm":
        with torch.no_grad():
            return norm()
    y = norm()
    if op != "second":
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b), state["dy"])
    first = torch.autograd.grad(y, (x, w, b), state["dy"], create_graph=True)
    second = torch.autograd.grad(first, (state["dy"], x, w, b), (state["ggx"], state["ggw"], state["ggb"]))
    return (y.detach(),) + tuple(v.detach() for v in first) + second


# --------------------------------------------------------------------------------------------------- the definition, in 64 bits
def _philox_words(seed, call, blocks, dev):
    """The four words of Philox4x32-10 at counters (block, call), each [blocks] int64."""
    ctr = [torch.arange(blocks, device=dev) % (1 << 32), torch.arange(blocks, device=dev) // (1 << 32)]
    ctr += [torch.full((blocks,), (call >> s) % (1 << 32), device=dev) for s in (0, 32)]
    for r in range(10):
        ka, kb = (seed % (1 << 32) + r * 0x9E3779B9) % (1 << 32), ((seed >> 32) % (1 << 32) + r * 0xBB67AE85) % (1 << 32)
        out = []
        for word, mul in ((ctr[0], 0xD2511F53), (ctr[2], 0xCD9E8D57)):
            lo, hi = word % 65536, word // 65536
            low = lo * mul                                   # < 2^48
            high = hi * mul + low // 65536                   # < 2^49: the product shifted down by 16 bits
            out.append((high // 65536, high % 65536 * 65536 + low % 65536))
        (h0, l0), (h1, l1) = out
        ctr = [h1 ^ ctr[1] ^ ka, l1, h0 ^ ctr[3] ^ kb, l0]
    return ctr


def exact(case, seed):
    state = prepare(case, seed)
    M, C, G, op = case["rows"], case["channels"], case["groups"], case["op"]
    dev = state["x"].device
    D = None
    if case["p"] > 0:
        quads = -(-C // 4)
        words = torch.stack(_philox_words(0x1234567890ABCDEF ^ seed, seed, M * quads, dev), -1).reshape(M, 4 * quads)[:, :C]
        D = (words.double() / 2.0 ** 32 >= round(case["p"] * 2.0 ** 32) / 2.0 ** 32).double() / (1.0 - case["p"])
        del words
    x = state["x"].detach().double().requires_grad_()
    if op == "dropout":
        return (x * D).detach(), state["dy"].double() * D
    w, b = (state[k].detach().double().requires_grad_() for k in ("w", "b"))
    lens = (state["seg_off"][1:] - state["seg_off"][:-1]).long()
    ids = torch.repeat_interleave(torch.arange(case["clouds"], device=dev), lens)
    n = (lens.clamp(min=1).double() * (C // G))[:, None]

    class Sum(torch.autograd.Function):
        """Sums over clouds [M, G] -> [B, G]; its gradient is the gather, and the gather's gradient the sum."""

        @staticmethod
        def forward(ctx, t):
            return torch.segment_reduce(t, "sum", lengths=lens, axis=0, unsafe=True)

        @staticmethod
        def backward(ctx, g):
            return Gather.apply(g)

    class Gather(torch.autograd.Function):
        @staticmethod
        def forward(ctx, t):
            return t.index_select(0, ids)

        @staticmethod
        def backward(ctx, g):
            return Sum.apply(g.contiguous())

    rows = x.view(M, G, C // G)
    cen = rows - Gather.apply(Sum.apply(rows.sum(2)) / n)[:, :, None]
    var = Sum.apply((cen * cen).sum(2)) / n
    u = (cen / Gather.apply(torch.sqrt(var + _EPS))[:, :, None]).reshape(M, C) * w + b
    act = {"none": lambda v: v, "relu": lambda v: v.clamp(min=0), "leaky_relu": lambda v: torch.maximum(v, 0.01 * v),
           "silu": lambda v: v * torch.sigmoid(v), "gelu": lambda v: v * torch.erfc(-v / math.sqrt(2.0)) / 2}[case["act"]]
    y = act(u) if D is None else act(u) * D
    if op == "norm":
        return y.detach()
    dy = state["dy"].detach().double().requires_grad_()
    first = torch.autograd.grad(y, (x, w, b), dy, create_graph=op == "second")
    out = (y.detach(),) + tuple(v.detach() for v in first)
    if op == "second":
        second = torch.autograd.grad(first, (dy, x, w, b), tuple(state[k].double() for k in ("ggx", "ggw", "ggb")), allow_unused=True)
        # with the identity for an activation the bias meets no second derivative
        out += tuple(torch.zeros_like(v) if g is None else g for v, g in zip((dy, x, w, b), second))
    return out
