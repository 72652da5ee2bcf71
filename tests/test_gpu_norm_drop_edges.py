"""Group norm and dropout at the edges of their range, on the GPU.  Reference and counts of roundings: oracle/norm_drop_ref.py."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import norm_drop_ref as R
from tests.test_gpu_norm_drop import BF16, F16, F32, MIXED, SEED, batch, check, dev, key, through_autograd


def seg_on_device(seg):
    return torch.tensor(seg, dtype=torch.int32, device=dev())


# ---------------------------------------------------------------------------------------------------------- huge pre-activations
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("act", ["none", "relu", "leaky_relu", "silu", "gelu"])
def test_an_infinite_bias_gives_an_infinite_activation(act, dtype):
    from dd3d_amd import ops
    seg, t = batch(MIXED, 16, dtype, seed=31)
    d = {k: v.to(dev()) for k, v in t.items()}
    call = lambda b: ops.group_norm(d["x"], seg_on_device(seg), 4, d["w"], b, activation=act)  # noqa: E731
    b = d["b"].clone()
    b[5] = math.inf
    y, plain = call(b), call(d["b"])
    others = [c for c in range(16) if c != 5]
    assert bool((y[:, 5] == math.inf).all()) and torch.equal(y[:, others], plain[:, others])


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_huge_finite_preactivations_twice_differentiated(act, dtype):
    """u^2 leaves fp32 from 1.8e19 on, where the density that multiplies it is zero; every channel is a group of its own, so that no tolerance
    grows with the neighbour's bias."""
    seg, t = batch(MIXED, 8, dtype, seed=32)
    t["b"] = torch.tensor([1e20, -1e20, 3e38, -3e38, 2e19, -2e19, 0.5, -0.5])
    check(through_autograd(t, seg_on_device(seg), 8, 2, activation=act, eps=1e-2), seg, t, 8, act, eps=1e-2)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_the_activations_element_by_element(act, dtype):
    """weight = 0 makes the bias the pre-activation, and each result is held against its own size, not its cloud's.  GELU's tail Q = e t P(t): the
    exponent a^2 / 2 is off by 5 half steps of itself (two roundings of the factor, squared, and one of the square); the hardware's exponential and
    reciprocal, nine steps of the polynomial and two products come to less than 24 half steps; the short polynomial for half-width values is off by
    8.3e-6.  SiLU's exponent u is off by 2 half steps, its exponential, sum, reciprocal and product by less than 12."""
    from dd3d_amd import ops
    C = 4096
    u = torch.linspace(-12, 12, C)
    b = u.to(dev()).requires_grad_()
    x = torch.randn(3, C, generator=torch.Generator().manual_seed(38)).to(dtype).to(dev())
    dy = torch.zeros_like(x)
    dy[1] = 1.0                                    # the bias' gradient is one row's derivative
    y = ops.group_norm(x, seg_on_device([0, 3]), 64, torch.zeros(C, device=dev()), b, activation=act)
    db, = torch.autograd.grad(y, b, dy)
    u = u.double()
    a, half = u.abs(), 2.0 ** -24
    if act == "gelu":
        tail = lambda v: torch.special.erfc(v / math.sqrt(2)) / 2  # noqa: E731  (1 + erf, and so torch's ndtr, has no digit of it left below -8)
        Q, n = tail(a), torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)
        f, d = u * tail(-u), tail(-u) + u * n
        steps = (2.5 * a * a + 24) * half
        value, slope = a * Q * (steps + (8.3e-6 if dtype != F32 else 0.0)) + half * u.clamp(min=0), (Q + a * n) * steps + half * (u > 0)
    else:
        s = torch.sigmoid(u)
        f, d = u * s, s * (1 + u * (1 - s))
        steps = (2 * a + 12) * half
        value, slope = f.abs() * steps, s * (1 + a) * steps
    if dtype != F32:                               # the rounding to the rows' type, of fp16's subnormal numbers at least 2^-25
        value = value + f.abs() * torch.finfo(dtype).eps / 2 * 1.001 + (2.0 ** -25 if dtype == F16 else 0.0)
    assert bool(((y.detach().cpu().double() - f).abs() <= value).all())
    assert bool(((db.cpu().double() - d).abs() <= slope).all())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_gelu_at_minus_infinity_is_its_limit(dtype):
    from dd3d_amd import ops
    seg, t = batch(MIXED, 8, dtype, seed=36)
    y = ops.group_norm(t["x"].to(dev()), seg_on_device(seg), 2, None, torch.full((8,), -math.inf, device=dev()), activation="gelu")
    assert not y.any()


# ------------------------------------------------------------------------------------------------------------ clouds without spread
LENGTHS = [32, 5, 1, 82, 700, 3001, 9000, 20011]


@pytest.mark.parametrize("C,G", [(16, 4), (16, 1), (7, 7), (24, 2), (12, 3), (128, 8), (128, 32), (2048, 1)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("value", [100.3, 3.1, -1e17])
def test_a_constant_cloud_is_a_cloud_of_zeros(C, G, dtype, value):
    """x - mean is zero whatever the constant, also where neither it nor 1 / count is a sum of few powers of two: value and gradients
    are those of a cloud of zeros, bit for bit."""
    lens = LENGTHS if C <= 128 else [82, 5, 1500]
    seg, t = batch(lens, C, dtype, seed=33)
    so = seg_on_device(seg)
    t["x"] = torch.zeros_like(t["x"])
    want = through_autograd(t, so, G, 2, activation="silu")
    t["x"] = torch.full_like(t["x"], value)
    got = through_autograd(t, so, G, 2, activation="silu")
    for k in want:
        assert torch.equal(got[k], want[k]), k


@pytest.mark.parametrize("lens,C,G", [([32, 45, 7, 1, 60], 16, 4), ([82] * 50, 128, 8), ([30, 9], 10, 5)])
@pytest.mark.parametrize("shift", [3000.0, 1e6])
def test_the_mean_is_off_by_its_own_rounding(lens, C, G, shift):
    """A thread's mean is corrected by the mean of its differences and rounded once, and so is the cloud's: two half steps, and the
    differences' own roundings (at most 2^10 additions of numbers below 2^4: less than an eighth of the half step at 3000)."""
    from dd3d_amd import _lib as L
    seg, t = batch(lens, C, F32, seed=34)
    x, so, B, M = (t["x"].clamp(-7, 7) + shift).to(dev()), seg_on_device(seg), len(lens), seg[-1]
    y, mean, rstd = torch.empty_like(x), torch.empty(B, G, device=dev()), torch.empty(B, G, device=dev())
    n = L.lib.dd3d_group_norm_ws_bytes(M, C, B, G, 0)
    ws = torch.empty(max(1, n), dtype=torch.uint8, device=dev())
    L.call("dd3d_group_norm_fwd", L.ptr(x), 0, M, C, L.ptr(so), B, G, None, None, 0, 1e-5, 0, 0.0, 0.0, None, L.ptr(y), L.ptr(mean), L.ptr(rstd), L.ptr(ws),
           ws.numel(), L.stream())
    half = 2.0 ** (math.floor(math.log2(shift)) - 24)
    for b, (r0, r1) in enumerate(zip(seg[:-1], seg[1:])):
        want = x[r0:r1].double().reshape(r1 - r0, G, -1).mean((0, 2))
        assert float((mean[b].double() - want).abs().max()) <= 2.125 * half


def test_a_spike_in_a_clouds_first_element_costs_no_accuracy():
    """The first element serves as a reference for the sums; every element but that one lies next to the mean in units of the spread, and its
    value comes out to the roundings of the mean (two half steps of |mean|) and of its own three operations."""
    from dd3d_amd import ops
    seg, t = batch([82, 700, 9000], 16, F32, seed=37)
    for r in seg[:-1]:
        t["x"][r, ::4] = 1e6
    y = ops.group_norm(t["x"].to(dev()), seg_on_device(seg), 4).cpu().double()
    for r0, r1 in zip(seg[:-1], seg[1:]):
        x = t["x"][r0:r1].double().reshape(r1 - r0, 4, 4)
        mean = x.mean((0, 2), keepdim=True)
        sd = torch.sqrt(((x - mean) ** 2).mean((0, 2), keepdim=True) + 1e-5)
        want = (x - mean) / sd
        # (the spread is a sum of squares of at most 2^18 elements, some 30 half steps in partial sums)
        allow = (4 * mean.abs() / sd + 40 * want.abs()) * 2.0 ** -24
        assert bool(((y[r0:r1].reshape(r1 - r0, 4, 4) - want).abs() <= allow).all())


@pytest.mark.parametrize("C,G", [(43, 43), (16, 16), (8, 2), (64, 64), (16, 4)])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_values_that_lie_close_together(C, G, act):
    """Clouds of a few rows a thousandth apart: half a step of the mean is a visible part of their spread, and is not in the results.  Held against
    the count of roundings without the conditioning (largest value over spread) that the other tests grant."""
    lens = [2, 3, 2, 1, 4, 2, 40, 2, 700] * 6
    seg, t = batch(lens, C, F32, seed=41)
    base = t["x"][torch.tensor(seg[:-1])].repeat_interleave(torch.tensor(lens), 0)
    t["x"] = base + 1e-3 * torch.randn(base.shape, generator=torch.Generator().manual_seed(42))
    got = through_autograd(t, seg_on_device(seg), G, 2, activation=act)
    ref = R.group_norm(t["x"], seg, G, t["w"], t["b"], 1e-5, act, dy=t["dy"], ggx=t["ggx"], ggw=t["ggw"], ggb=t["ggb"], order=2)
    for n, v in got.items():
        far = R.off(n, v, ref, F32, torch.ones(()))
        assert far <= 1, f"{n}: {far:.3g} times what its roundings allow"


@pytest.mark.parametrize("C,G", [(16, 4), (7, 7), (24, 2), (128, 8)])
def test_the_mean_in_two_floats(C, G):
    """Sums of differences below 2^4: at most 64 in a thread, 128 over threads and 64 for chunks, windows and reciprocals, a half step each."""
    from dd3d_amd import _lib as L
    for dtype in (F32, BF16):
        lens = [32, 45, 0, 1, 700, 9000, 20011]
        seg, t = batch(lens, C, dtype, seed=43)
        x, so, B, M = (t["x"].float().clamp(-7, 7) + 1e6).to(dtype).to(dev()), seg_on_device(seg), len(lens), seg[-1]
        y, mean, rstd = torch.empty_like(x), torch.full((2, B, G), 7.0, device=dev()), torch.empty(B, G, device=dev())
        ws = torch.empty(max(1, L.lib.dd3d_group_norm_ws_bytes(M, C, B, G, 0)), dtype=torch.uint8, device=dev())
        L.call("dd3d_group_norm_fwd", L.ptr(x), 0 if dtype == F32 else 2, M, C, L.ptr(so), B, G, None, None, 0, 1e-5, 16, 0.0, 0.0, None, L.ptr(y), L.ptr(mean),
               L.ptr(rstd), L.ptr(ws), ws.numel(), L.stream())
        if dtype != F32:
            assert bool((mean[1] == 7.0).all())      # half-width rows leave the second floats alone
            continue
        assert float(mean[1].abs().max()) <= 2.0 ** -5      # half a step at 2^19
        for b, (r0, r1) in enumerate(zip(seg[:-1], seg[1:])):
            want = x[r0:r1].double().reshape(r1 - r0, G, -1).mean((0, 2)) if r1 > r0 else torch.zeros(G, dtype=torch.float64, device=dev())
            assert float((mean[:, b].double().sum(0) - want).abs().max()) <= 256 * 2.0 ** -24 * 2.0 ** 4


@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
@pytest.mark.parametrize("value,eps", [(2.0 ** 57, 1e-5), (2.0 ** 20, 1e-30), (2.0 ** 70, 1e-36)])
@pytest.mark.parametrize("C,G,dtype", [(16, 4, F32), (9, 3, F32), (32, 2, BF16)])
def test_rows_that_are_not_there_add_nothing_to_a_constant_cloud(act, value, eps, C, G, dtype):
    """Zeros stand in for rows behind a chunk's last one.  They lie far from a constant cloud's mean in units of its spread, and what is
    computed from them may leave fp32; the gradients stay those of a cloud of zeros."""
    seg, t = batch([32, 5, 700, 9000], C, dtype, seed=35)
    so = seg_on_device(seg)
    t["x"] = torch.zeros_like(t["x"])
    want = through_autograd(t, so, G, 2, 0.2, activation=act, eps=eps)
    assert all(bool(torch.isfinite(v).all()) for v in want.values())
    t["x"] = torch.full_like(t["x"], value)
    got = through_autograd(t, so, G, 2, 0.2, activation=act, eps=eps)
    for k in want:
        assert torch.equal(got[k], want[k]), k


# ------------------------------------------------------------------------------------------------------- forward-mode derivatives
def test_forward_mode_derivatives_are_refused_not_lost():
    from torch.autograd import forward_ad
    from dd3d_amd import ops
    x, so = torch.randn(40, 8, device=dev()), torch.tensor([0, 40], dtype=torch.int32, device=dev())
    w, v = torch.ones(8, device=dev()), torch.randn(40, 8, device=dev())
    k = key()
    want = ops.group_norm(x, so, 2, w), ops.dropout(x, 0.3, k)
    with forward_ad.dual_level():
        xd, wd = forward_ad.make_dual(x, v), forward_ad.make_dual(w, torch.ones_like(w))
        calls = [lambda: ops.dropout(xd, 0.3, k), lambda: ops.group_norm(xd, so, 2, w), lambda: ops.group_norm(x, so, 2, wd),
                 lambda: ops.group_norm(x, so, 2, None, wd)]
        for call in calls:
            with pytest.raises(NotImplementedError):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError):
                call()
        # a tangent on the incoming gradient, in the first and in the second backward pass
        xr, gd = x.clone().requires_grad_(), forward_ad.make_dual(torch.ones_like(x), v)
        for y in (ops.dropout(xr, 0.3, k), ops.group_norm(xr, so, 2, w)):
            for again in (False, True):
                with pytest.raises(NotImplementedError):
                    torch.autograd.grad(y, xr, gd, retain_graph=True, create_graph=again)
        dx, = torch.autograd.grad(ops.group_norm(xr, so, 2, w), xr, v, create_graph=True)
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(dx, xr, gd)
        # without a tangent the calls are the ordinary ones
        assert torch.equal(ops.group_norm(x, so, 2, w), want[0]) and torch.equal(ops.dropout(x, 0.3, k), want[1])


# ------------------------------------------------------------------------------------------------- wide slabs, and beyond 32 bits
@pytest.mark.parametrize("C,G", [(4096, 1), (4096, 2), (2047, 1), (2052, 1)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_slabs_of_more_than_256_vectors_cut_by_windows(C, G, dtype):
    seg, t = batch([1500, 3, 700], C, dtype, seed=39)
    check(through_autograd(t, seg_on_device(seg), G, 2, 0.2, activation="silu"), seg, t, G, "silu", 0.2)


def test_gradients_of_elements_beyond_32_bits():
    """2^31 + elements: the last rows' gradients, first and second, and the mask drawn again for them.  The first cloud is all zeros with zero
    gradients, so the parameters' are sums over the last two."""
    from dd3d_amd import ops
    M, C, G, p = 16_800_000, 128, 8, 0.5
    seg, t = batch([200, 300], C, BF16, seed=40)
    wide = lambda v: torch.cat([torch.zeros(M - 500, C, dtype=BF16, device=dev()), v.to(dev())])  # noqa: E731
    x, dy = wide(t["x"]).requires_grad_(), wide(t["dy"]).requires_grad_()
    w, b = t["w"].to(dev()).requires_grad_(), t["b"].to(dev()).requires_grad_()
    y = ops.group_norm(x, seg_on_device([0, M - 500, M - 300, M]), G, w, b, activation="silu", dropout=p, key=key())
    first = torch.autograd.grad(y, (x, w, b), dy, create_graph=True)
    second = torch.autograd.grad(first, (dy, x, w, b), (wide(t["ggx"]), t["ggw"].to(dev()), t["ggb"].to(dev())))
    D = R.keep_mask(500, C, p, SEED, 5, first_row=M - 500).double() / (1 - p)
    ref = R.group_norm(t["x"], seg, G, t["w"], t["b"], name="silu", D=D, dy=t["dy"], ggx=t["ggx"], ggw=t["ggw"], ggb=t["ggb"], order=2)
    for n, v in zip(("dx", "dw", "db", "ddy", "ddx", "ddw", "ddb"), (*first, *second)):
        far = R.off(n, v[-500:] if v.dim() == 2 else v, ref, v.dtype, ref["cond"][0])
        assert far <= 1, f"{n}: {far:.3g} times what its roundings allow"
    assert not first[0][:-500].any() and not second[1][:-500].any()
