"""Group norm with an activation (value, first and second gradient), counter-based dropout, and the two in one pass, on the GPU against the
float64 restatement (oracle/norm_drop_ref.py): every type, ragged and empty clouds, odd widths, unaligned and strided rows, rows in no
cloud, values that are not finite, other streams, captured graphs.  The tolerances are the oracle's count of fp32 half steps plus one
rounding to the rows' type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import norm_drop_ref as R

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
SEED = 0x0123456789ABCDEF


def dev():
    return torch.device("cuda:0")


def key(call=5, seed=SEED):
    return torch.tensor([seed, call], dtype=torch.int64, device=dev())


def offsets(lens, start=0):
    return [start + int(v) for v in torch.cat([torch.zeros(1, dtype=torch.long), torch.cumsum(torch.tensor(lens), 0)])]


def batch(lens, C, dtype, seed=0, start=0, behind=0, shift=0.4, pdtype=F32):
    g = torch.Generator().manual_seed(seed)
    seg = offsets(lens, start)
    M = seg[-1] + behind
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    t = dict(x=(rn(M, C) * torch.exp(0.3 * rn(C)) + shift * rn(C)).to(dtype), dy=rn(M, C).to(dtype), w=(1 + 0.3 * rn(C)).to(pdtype), b=(0.3 * rn(C)).to(pdtype),
             ggx=rn(M, C).to(dtype), ggw=rn(C).to(pdtype), ggb=rn(C).to(pdtype))
    return seg, t


def factors(M, C, p, call=5):
    return None if p == 0 else R.keep_mask(M, C, p, SEED, call).double() / (1 - p) if p < 1 else torch.zeros(M, C, dtype=torch.float64)


def keep_off_the_border(seg, t, G, act, eps):
    """No gradient flows into an element whose pre-activation lies next to a jump of the derivative: it may fall on either side."""
    if act in ("relu", "leaky_relu"):
        u = R.group_norm(t["x"], seg, G, t["w"], t["b"], eps, "none")["y"][0]
        t["dy"] = torch.where(u.abs() < 1e-3, torch.zeros(()), t["dy"].float()).to(t["dy"].dtype)


def through_autograd(t, seg_off, G, order, p=0.0, affine=(True, True), **kw):
    from dd3d_amd import ops
    d = {k: v.to(dev()) for k, v in t.items()}
    x, dy = d["x"].requires_grad_(), d["dy"].requires_grad_()
    w, b = (d[n].requires_grad_() if on else None for n, on in zip("wb", affine))
    y = ops.group_norm(x, seg_off, G, w, b, dropout=p, key=key() if p else None, **kw)
    out = {"y": y}
    if order >= 1:
        ins = [(n, v) for n, v in (("x", x), ("w", w), ("b", b)) if v is not None]
        first = torch.autograd.grad(y, [v for _, v in ins], dy, create_graph=order == 2)
        out |= {"d" + n: v for (n, _), v in zip(ins, first)}
    if order == 2:
        cot = [d["gg" + n] for n, _ in ins]
        second = torch.autograd.grad(first, [dy] + [v for _, v in ins], cot)
        out |= {"ddy": second[0]} | {"dd" + n: v for (n, _), v in zip(ins, second[1:])}
    return out


def check(got, seg, t, G, act, p=0.0, eps=1e-5, slope=0.01, order=2, affine=(True, True)):
    M, C = t["x"].shape
    w, b, ggw, ggb = (t[n] if on else None for n, on in (("w", affine[0]), ("b", affine[1]), ("ggw", affine[0]), ("ggb", affine[1])))
    ref = R.group_norm(t["x"], seg, G, w, b, eps, act, slope, factors(M, C, p), t["dy"], t["ggx"], ggw, ggb, order=order)
    for n, v in got.items():
        dt = t["w"].dtype if n in ("dw", "db", "ddw", "ddb") else t["x"].dtype
        assert v.dtype == dt
        far = R.off(n, v, ref, dt, ref["cond"][0])
        assert far <= 1, f"{n}: {far:.3g} times what its roundings allow"


def check_some(got, lens, every, seg, t, G, act, order):
    """The matrices' rows of the last four clouds and of one cloud in ``every``."""
    some = [i + i // every % 4 for i in range(0, len(lens) - 4, every)] + list(range(len(lens) - 4, len(lens)))
    rows = torch.tensor([r for i in some for r in range(seg[i], seg[i + 1])])
    part = {k: v[rows] if v.shape[0] == seg[-1] else v for k, v in t.items()}
    check({n: got[n].cpu()[rows] for n in ("y", "dx", "ddy", "ddx")[:2 * order]}, offsets([lens[i] for i in some]), part, G, act, order=order)


MIXED = [5, 0, 1, 37, 2, 0, 82, 250, 3]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("act", ["none", "relu", "leaky_relu", "silu", "gelu"])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_every_type_and_activation_twice_differentiated(dtype, act, p):
    seg, t = batch(MIXED, 32, dtype, seed=1)
    keep_off_the_border(seg, t, 4, act, 1e-5)
    so = torch.tensor(seg, dtype=torch.int32, device=dev())
    check(through_autograd(t, so, 4, 2, p, activation=act, negative_slope=0.2), seg, t, 4, act, p, slope=0.2)


@pytest.mark.parametrize("lens,C,G", [([1], 1, 1), ([2, 1], 3, 3), (MIXED, 3, 1), (MIXED, 5, 5), (MIXED, 7, 1), (MIXED, 10, 2), (MIXED, 12, 4), (MIXED, 24, 3),
                                      (MIXED, 36, 6), (MIXED, 100, 5), (MIXED, 128, 128), (MIXED, 128, 32), (MIXED, 128, 1), (MIXED, 130, 10),
                                      ([40, 9], 1030, 5), ([17], 4096, 2), ([300], 1000, 1), ([2100, 3, 900], 48, 6), ([5000], 16, 2), ([1] * 50, 64, 4),
                                      ([12] * 70, 40, 10)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_shapes(lens, C, G, dtype):
    seg, t = batch(lens, C, dtype, seed=C + G)
    so = torch.tensor(seg, dtype=torch.int32, device=dev())
    eps = 1e-2    # groups of one or two elements: their variance may be anything, the conditioning counted is 1 / sqrt(eps) at most
    check(through_autograd(t, so, G, 2, 0.25, activation="silu", eps=eps), seg, t, G, "silu", 0.25, eps=eps)


@pytest.mark.parametrize("lens", [[70001, 3, 0, 20011], [1, 40000, 1], [3000, 3000, 3001, 2999, 100], [260] * 40 + [9000]])
@pytest.mark.parametrize("C,G,dtype", [(16, 4, F32), (24, 1, F16), (9, 3, F32)])
def test_long_clouds(lens, C, G, dtype):
    seg, t = batch(lens, C, dtype, seed=7)
    so = torch.tensor(seg, dtype=torch.int32, device=dev())
    check(through_autograd(t, so, G, 2, 0.1, activation="gelu"), seg, t, G, "gelu", 0.1)
    keep_off_the_border(seg, t, G, "relu", 1e-5)
    check(through_autograd(t, so, G, 2, 0.0, activation="relu"), seg, t, G, "relu", 0.0)


@pytest.mark.parametrize("lens,C,G,dtype", [([2] * 2500, 8, 1, F32), ([1, 4, 2] * 900, 12, 3, BF16), ([90] * 40, 128, 8, F16), ([82] * 300, 64, 4, F32)])
def test_many_short_clouds(lens, C, G, dtype):
    """More clouds than workgroups leave parts of the parameter gradients for: one workgroup takes several."""
    seg, t = batch(lens, C, dtype, seed=21)
    so = torch.tensor(seg, dtype=torch.int32, device=dev())
    check(through_autograd(t, so, G, 2, 0.2, activation="silu", eps=1e-2), seg, t, G, "silu", 0.2, eps=1e-2)


@pytest.mark.parametrize("rows", [1, 31, 32, 33, 63, 64, 65, 255, 256, 257, 511, 512, 513, 1023, 1024, 1025, 2047, 2049, 4097])
def test_lengths_about_the_chunk_and_window_sizes(rows):
    lens = [rows, 2, rows + 1]
    for C, G, dtype in ((16, 2, F32), (32, 1, BF16), (128, 32, F16)):
        seg, t = batch(lens, C, dtype, seed=rows)
        so = torch.tensor(seg, dtype=torch.int32, device=dev())
        check(through_autograd(t, so, G, 2, 0.1, activation="silu", eps=1e-2), seg, t, G, "silu", 0.1, eps=1e-2)


def test_everything_dropped_and_next_to_it():
    seg, t = batch(MIXED, 16, F32, seed=22)
    so = torch.tensor(seg, dtype=torch.int32, device=dev())
    got = through_autograd(t, so, 4, 2, 1.0, activation="silu")
    assert not any(bool(v.any()) for k, v in got.items()), "p = 1 leaves nothing"
    check(through_autograd(t, so, 4, 2, 0.999, activation="silu"), seg, t, 4, "silu", 0.999)


def test_two_calls_at_once():
    """Two streams, one pair of parameters: neither call sees the other's workspace."""
    from dd3d_amd import ops
    so = torch.tensor(offsets([6000, 40, 9000] + [70] * 50), dtype=torch.int32, device=dev())
    xs = [torch.randn(18540, 64, device=dev(), generator=torch.Generator(dev()).manual_seed(i)).requires_grad_() for i in range(2)]
    w, b = torch.rand(64, device=dev()).requires_grad_(), torch.rand(64, device=dev()).requires_grad_()
    run = lambda x: torch.autograd.grad(ops.group_norm(x, so, 8, w, b, activation="gelu", dropout=0.1, key=key()).square().sum(), (x, w, b))  # noqa: E731
    want = [[g.clone() for g in run(x)] for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(3):
        got = []
        for x, s in zip(xs, streams):
            with torch.cuda.stream(s):
                got.append(run(x))
        torch.cuda.synchronize()
        for o, r in zip(got, want):
            assert all(torch.equal(a, c) for a, c in zip(o[1:], r[1:])) and torch.equal(o[0], r[0])


@pytest.mark.parametrize("affine", [(False, False), (True, False), (False, True)])
def test_without_weight_or_bias(affine):
    seg, t = batch(MIXED, 16, F32, seed=3)
    so = torch.tensor(seg, dtype=torch.int32, device=dev())
    check(through_autograd(t, so, 2, 2, affine=affine, activation="silu"), seg, t, 2, "silu", affine=affine)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_parameters_of_the_rows_type(dtype):
    seg, t = batch(MIXED, 16, dtype, seed=4, pdtype=dtype)
    so = torch.tensor(seg, dtype=torch.int32, device=dev())
    check(through_autograd(t, so, 2, 2, activation="gelu"), seg, t, 2, "gelu")


@pytest.mark.parametrize("lens,start,behind", [(MIXED, 3, 41), ([0, 0], 2, 5), ([6000, 2], 700, 5000)])
def test_rows_in_no_cloud_are_zero_and_leave_the_others_alone(lens, start, behind):
    seg, t = batch(lens, 20, F32, seed=5, start=start, behind=behind)
    for k in ("x", "dy", "ggx"):     # what they hold does not matter, not even to the sums
        t[k][:start] = float("nan")
        t[k][seg[-1]:] = float("inf")
    so = torch.tensor(seg, dtype=torch.int32, device=dev())
    got = through_autograd(t, so, 4, 2, activation="silu")
    for k in ("y", "dx", "ddy", "ddx"):
        assert not got[k][:start].any() and not got[k][seg[-1]:].any(), k
    check(got, seg, t, 4, "silu")


def test_no_rows_and_no_clouds():
    from dd3d_amd import ops
    for M, seg in ((0, [0]), (0, [0, 0, 0]), (7, [0])):
        x = torch.full((M, 8), 3.0, device=dev(), requires_grad=True)
        w = torch.ones(8, device=dev(), requires_grad=True)
        y = ops.group_norm(x, torch.tensor(seg, dtype=torch.int32, device=dev()), 2, w, activation="relu")
        assert y.shape == (M, 8) and not y.any()
        dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y), create_graph=True)
        assert not dx.any() and not dw.any()
        assert not torch.autograd.grad(dw.sum(), x)[0].any()


def test_rows_behind_the_last_one_are_not_touched():
    from dd3d_amd import _lib as L
    x, seg = torch.randn(50, 12, device=dev()), torch.tensor([0, 20, 40], dtype=torch.int32, device=dev())
    y = torch.full((50, 12), 7.0, device=dev())
    ws = torch.empty(max(1, L.lib.dd3d_group_norm_ws_bytes(40, 12, 2, 3, 0)), dtype=torch.uint8, device=dev())
    L.call("dd3d_group_norm_fwd", L.ptr(x), 0, 40, 12, L.ptr(seg), 2, 3, None, None, 0, 1e-5, 0, 0.0, 0.0, None, L.ptr(y), None, None, L.ptr(ws), ws.numel(), L.stream())
    assert bool((y[40:] == 7.0).all()) and bool((y[:40] != 7.0).all())
    # offsets beyond the rows (a bound that is too small) are cut, not followed
    far = torch.tensor([0, 20, 400], dtype=torch.int32, device=dev())
    L.call("dd3d_group_norm_fwd", L.ptr(x), 0, 40, 12, L.ptr(far), 2, 3, None, None, 0, 1e-5, 0, 0.0, 0.0, None, L.ptr(y), None, None, L.ptr(ws), ws.numel(), L.stream())
    assert bool((y[40:] == 7.0).all())


def test_values_that_are_not_finite_stay_in_their_cloud_and_group():
    seg, t = batch([30, 40, 6000, 5], 16, F32, seed=6)
    so = torch.tensor(seg, dtype=torch.int32, device=dev())
    bad = {k: v.clone() for k, v in t.items()}
    bad["x"][35, 5] = float("nan")        # cloud 1, group 1
    bad["x"][100, 14] = float("inf")      # cloud 2, group 3
    a, z = through_autograd(t, so, 4, 2, activation="silu"), through_autograd(bad, so, 4, 2, activation="silu")
    hit = torch.zeros(seg[-1], 16, dtype=torch.bool, device=dev())
    hit[30:70, 4:8] = hit[70:6070, 12:16] = True
    for k in ("y", "dx", "ddy", "ddx"):
        assert torch.equal(a[k][~hit], z[k][~hit]), k
    assert bool(z["y"][30:70, 4:8].isnan().all()) and bool(z["y"][70:6070, 12:16].isnan().all())
    assert bool(torch.isfinite(z["dw"][[0, 1, 2, 3, 8, 9, 10, 11]]).all()) and bool(z["dw"][4:8].isnan().all())


def test_equal_rows_have_no_variance():
    from dd3d_amd import ops
    x = torch.tensor([3.25, -1.5]).repeat_interleave(8).repeat(50, 1).to(dev())
    y = ops.group_norm(x, torch.tensor([0, 50], dtype=torch.int32, device=dev()), 2, activation="none")
    assert not y.any()


@pytest.mark.parametrize("shift", [100.0, 3000.0])
def test_a_mean_far_above_the_spread(shift):
    """The conditioning (largest value over spread) is counted: a variance as mean of squares minus squared mean would miss it by far."""
    seg, t = batch([40, 700, 5000], 8, F32, seed=8)
    t["x"] = t["x"] + shift
    so = torch.tensor(seg, dtype=torch.int32, device=dev())
    check(through_autograd(t, so, 2, 2, activation="silu"), seg, t, 2, "silu")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("C", [8, 32])
def test_unaligned_and_strided_rows(dtype, C):
    from dd3d_amd import ops
    seg, t = batch(MIXED, C, dtype, seed=9)
    M = seg[-1]
    so = torch.tensor(seg, dtype=torch.int32, device=dev())
    wide = torch.zeros(M, 2 * C + 1, dtype=dtype, device=dev())
    wide[:, 1:C + 1] = t["x"].to(dev())
    flat = torch.zeros(M * C + 1, dtype=dtype, device=dev())
    flat[1:] = t["x"].reshape(-1).to(dev())
    dy = t["dy"].to(dev()).t().contiguous().t()          # columns first
    w, b = t["w"].to(dev()), t["b"].to(dev())
    for x in (wide[:, 1:C + 1], flat[1:].view(M, C), t["x"].to(dev()).t().contiguous().t()):
        x = x.detach().requires_grad_()
        y = ops.group_norm(x, so, 4, w, b, activation="gelu", dropout=0.2, key=key())
        dx, = torch.autograd.grad(y, x, dy)
        check({"y": y, "dx": dx}, seg, t, 4, "gelu", 0.2, order=1)
    wflat = torch.zeros(C + 1, device=dev())
    wflat[1:] = w
    y = ops.group_norm(t["x"].to(dev()), so, 4, wflat[1:], b, activation="gelu")
    check({"y": y}, seg, t, 4, "gelu", 0.0, order=0)


def test_an_expanded_gradient():
    from dd3d_amd import ops
    seg, t = batch(MIXED, 16, F32, seed=10)
    t["dy"] = torch.ones_like(t["dy"])
    x = t["x"].to(dev()).requires_grad_()
    ops.group_norm(x, torch.tensor(seg, dtype=torch.int32, device=dev()), 4, t["w"].to(dev()), t["b"].to(dev()), activation="silu").sum().backward()
    check({"dx": x.grad}, seg, t, 4, "silu", order=1)


def test_only_what_is_asked_for_is_computed_and_it_is_the_same():
    from dd3d_amd import ops
    seg, t = batch(MIXED, 16, F32, seed=11)
    so = torch.tensor(seg, dtype=torch.int32, device=dev())
    full = through_autograd(t, so, 4, 2, activation="silu")
    d = {k: v.to(dev()) for k, v in t.items()}
    for n in ("x", "w", "b"):
        v = {k: d[k].detach().clone().requires_grad_(k == n) for k in ("x", "w", "b")}
        y = ops.group_norm(v["x"], so, 4, v["w"], v["b"], activation="silu")
        assert torch.equal(y, full["y"]) and torch.equal(torch.autograd.grad(y, v[n], d["dy"])[0], full["d" + n])
    with torch.no_grad():
        assert torch.equal(ops.group_norm(d["x"], so, 4, d["w"], d["b"], activation="silu"), full["y"])
    # one cotangent at a time: the second gradient is linear in the three
    v = {k: d[k].detach().clone().requires_grad_() for k in ("x", "w", "b", "dy")}
    first = torch.autograd.grad(ops.group_norm(v["x"], so, 4, v["w"], v["b"], activation="silu"), (v["x"], v["w"], v["b"]), v["dy"], create_graph=True)
    parts = [torch.autograd.grad(f, v["x"], d["gg" + n], retain_graph=True)[0].double() for f, n in zip(first, "xwb")]
    assert float((sum(parts) - full["ddx"].double()).abs().max() / full["ddx"].abs().max()) < 1e-5
    with pytest.raises(RuntimeError):
        ddx, = torch.autograd.grad(first[0], v["x"], d["ggx"], create_graph=True)
        torch.autograd.grad(ddx.sum(), v["x"])      # a third differentiation is refused


def test_gradient_equals_differences_of_the_value():
    """Directional derivative of the fp32 kernel by central differences.  h = 2^-6: the difference misses the derivative by h^2/6 of a third
    derivative of order one (4e-5) and by the roundings of the two values over 2h (about sqrt(N) 2^-24 2^6 / 2 of |dy|: 2e-6 per element)."""
    from dd3d_amd import ops
    seg, t = batch([40, 90, 5000], 16, F32, seed=12)
    so = torch.tensor(seg, dtype=torch.int32, device=dev())
    d = {k: v.to(dev()) for k, v in t.items()}
    f = lambda **o: (ops.group_norm(*(o.get(k, d[k]) for k in ("x",)), so, 4, o.get("w", d["w"]), o.get("b", d["b"]), activation="gelu").double() * d["dy"].double()).sum()  # noqa: E731
    got = through_autograd(t, so, 4, 1, activation="gelu")
    h = 2.0 ** -6
    for n in ("x", "w", "b"):
        u = d["gg" + n]
        num = (f(**{n: d[n] + h * u}) - f(**{n: d[n] - h * u})) / (2 * h)
        want = (got["d" + n].double() * u.double()).sum()
        size = (got["d" + n].double() * u.double()).abs().sum()
        assert abs(float(num - want)) <= 1e-3 * float(size)


# ------------------------------------------------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(1, 1), (7, 3), (33, 4), (5, 1024), (250, 128), (3, 5, 9), (4099,), (64, 7), (1000, 36), ()])
@pytest.mark.parametrize("p", [0.1, 0.5, 1.0])
def test_dropout_equals_the_generator_word_by_word(dtype, shape, p):
    from dd3d_amd import ops
    g = torch.Generator().manual_seed(1)
    x, dy = (3 * torch.randn(shape, generator=g)).to(dtype), torch.randn(shape, generator=g).to(dtype)
    xd = x.to(dev()).requires_grad_()
    y = ops.dropout(xd, p, key(call=-3))
    dx, = torch.autograd.grad(y, xd, dy.to(dev()))
    assert y.dtype == dtype and y.shape == x.shape
    for got, src in ((y, x), (dx, dy)):
        want, keep = R.dropout(src.reshape(shape or (1, 1)), p, SEED, -3)
        got = got.detach().cpu().double().reshape(want.shape)
        assert torch.equal(got != 0, keep & (src.reshape(want.shape) != 0) if p < 1 else torch.zeros_like(keep))
        # the factor is rounded to fp32, then the product, then to the type: two half steps of fp32 and one of the type
        assert bool(((got - want).abs() <= want.abs() * (2 * 2.0 ** -24 + torch.finfo(dtype).eps / 2) + 2.0 ** -25 * (dtype == F16)).all())


def test_dropout_unaligned_strided_and_special():
    from dd3d_amd import ops
    x = torch.randn(40, 32, device=dev())
    k = key()
    want = ops.dropout(x, 0.4, k)
    flat = torch.zeros(40 * 32 + 1, device=dev())
    flat[1:] = x.reshape(-1)
    assert torch.equal(ops.dropout(flat[1:].view(40, 32), 0.4, k), want)
    assert torch.equal(ops.dropout(x.t().contiguous().t(), 0.4, k), want)
    assert ops.dropout(x, 0.0, k) is x and ops.dropout(x[:0], 0.5, k).shape == (0, 32)
    bad = x.clone()
    bad[want == 0] = float("nan")
    assert torch.equal(ops.dropout(bad, 0.4, k), want)      # a dropped element is zero whatever it held
    assert not torch.equal(ops.dropout(x, 0.4, key(call=6)), want) and not torch.equal(ops.dropout(x, 0.4, key(seed=SEED + 1)), want)
    # twice differentiable: the gradient of <dropout(x), v>^2 / 2 twice
    xr = x.clone().requires_grad_()
    v = torch.randn_like(x)
    s, = torch.autograd.grad((ops.dropout(xr, 0.4, k) * v).sum().square() / 2, xr, create_graph=True)
    vd = ops.dropout(v, 0.4, k)
    assert torch.allclose(torch.autograd.grad((s * v).sum(), xr)[0], (vd * v).sum() * vd, rtol=1e-4, atol=1e-4)


def test_the_fused_mask_is_the_separate_one():
    from dd3d_amd import ops
    for C, G, dtype in ((128, 8, F32), (100, 5, F16), (9, 3, F32), (64, 64, BF16)):
        seg, t = batch(MIXED, C, dtype, seed=13)
        so = torch.tensor(seg, dtype=torch.int32, device=dev())
        x = t["x"].to(dev())
        plain = ops.group_norm(x, so, G, activation="gelu")
        fused = ops.group_norm(x, so, G, activation="gelu", dropout=0.5, key=key())
        both = ops.dropout(plain, 0.5, key())
        # the factor 2 rounds nothing among normal numbers.  An fp16 value below 2^-14 (GELU's tail) was rounded to a multiple of 2^-24
        # before it was doubled, off by 2^-25 at most and by 2^-24 doubled; the fused one is rounded once, off by 2^-25
        normal = plain.abs().float() >= torch.finfo(dtype).tiny
        assert torch.equal(fused[normal], both[normal])
        assert float((fused.float() - both.float()).abs().max()) <= (2.0 ** -24 + 2.0 ** -25 if dtype == F16 else torch.finfo(dtype).tiny)


def test_equal_inputs_give_equal_bits():
    for lens, C in ((MIXED, 64), ([20000, 5, 300], 16)):
        seg, t = batch(lens, C, F32, seed=14)
        so = torch.tensor(seg, dtype=torch.int32, device=dev())
        a, b = (through_autograd(t, so, 4, 2, 0.2, activation="silu") for _ in range(2))
        for k in a:
            assert torch.equal(a[k], b[k]), k


def test_another_stream_than_the_default_one():
    seg, t = batch([300, 4000, 7], 32, F32, seed=15)
    so = torch.tensor(seg, dtype=torch.int32, device=dev())
    want = through_autograd(t, so, 4, 2, 0.2, activation="silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = through_autograd(t, so, 4, 2, 0.2, activation="silu")
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for k in want:
        assert torch.equal(want[k], got[k]), k


def test_key_stream():
    from dd3d_amd import ops
    state = ops.random_state(42, dev())
    keys = [ops.random_key(state).tolist() for _ in range(3)]
    assert keys == [[42, 0], [42, 1], [42, 2]] and state.tolist() == [42, 3]


def test_a_state_used_as_a_key_is_not_read_after_it_changed():
    from dd3d_amd import ops
    state = ops.random_state(42, dev())
    x = torch.randn(40, 32, device=dev(), requires_grad=True)
    so = torch.tensor([0, 40], dtype=torch.int32, device=dev())
    for call in (lambda: ops.dropout(x, 0.4, state), lambda: ops.group_norm(x, so, 4, dropout=0.4, key=state)):
        y = call()
        torch.autograd.grad(y.sum(), x, retain_graph=True)
        ops.random_key(state)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y.sum(), x)


def test_more_clouds_than_workgroups():
    """70 000 clouds of a row or two, on at most 32 768 forward and 2048 backward workgroups; every 500th cloud is compared."""
    lens = [1, 2, 0, 2] * 17500
    seg, t = batch(lens, 16, F32, seed=17)
    got = through_autograd(t, torch.tensor(seg, dtype=torch.int32, device=dev()), 4, 1, activation="silu")
    check_some(got, lens, 500, seg, t, 4, "silu", 1)


@pytest.mark.parametrize("C,G,dtype", [(256, 256, F32), (256, 256, BF16), (256, 64, F16)])
def test_as_many_groups_as_channels_and_many_clouds(C, G, dtype):
    lens = [30, 45, 0, 1] * 300
    seg, t = batch(lens, C, dtype, seed=18)
    got = through_autograd(t, torch.tensor(seg, dtype=torch.int32, device=dev()), G, 2, activation="silu")
    check_some(got, lens, 100, seg, t, G, "silu", 2)


def test_a_captured_step_draws_a_new_mask_at_every_replay():
    from dd3d_amd import ops
    seg, t = batch([300, 4000, 7], 32, F32, seed=16)
    so = torch.tensor(seg, dtype=torch.int32, device=dev())
    d = {k: v.to(dev()) for k, v in t.items()}
    state, cell = ops.random_state(9, dev()), {}

    def step(k, x, w, b):
        y = ops.group_norm(x, so, 4, w, b, activation="silu", dropout=0.3, key=k)
        first = torch.autograd.grad(y, (x, w, b), d["dy"], create_graph=True)
        return [y.detach(), *(f.detach() for f in first), *torch.autograd.grad(first, (x, w), (d["ggx"], d["ggw"], d["ggb"]))]

    leaves = lambda: [d[n].clone().requires_grad_() for n in "xwb"]  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(ops.random_key(state), *leaves())
    torch.cuda.current_stream().wait_stream(side)
    mine = leaves()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cell["key"] = ops.random_key(state)
        cell["out"] = step(cell["key"], *mine)
    seen = []
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        k = cell["key"].clone()
        assert k.tolist() == [9, 1 + i]      # the call drawn before capture was number 0
        for a, b in zip(cell["out"], step(k, *leaves())):
            assert torch.equal(a, b)
        seen.append(cell["out"][0].clone())
    assert not any(torch.equal(seen[0], s) for s in seen[1:])


def test_two_captured_graphs_replayed_side_by_side():
    from dd3d_amd import ops
    so = torch.tensor(offsets([3000, 9000, 40]), dtype=torch.int32, device=dev())
    xs = [torch.randn(12040, 32, device=dev(), generator=torch.Generator(dev()).manual_seed(i)).requires_grad_() for i in range(2)]
    w = torch.ones(32, device=dev(), requires_grad=True)
    run = lambda x: torch.autograd.grad(ops.group_norm(x, so, 4, w, activation="gelu").square().sum(), (x, w))  # noqa: E731
    want = [[g.clone() for g in run(x)] for x in xs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(x))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, r in zip(outs, want):
            for a, b in zip(o, r):
                assert torch.allclose(a, b, rtol=1e-5, atol=1e-5)


def test_elements_beyond_32_bits():
    """2^31 + elements: the last rows' addresses and the generator's counter pass 32 bits."""
    from dd3d_amd import ops
    M, C = 16_800_000, 128                              # 2.15e9 bf16 elements
    x = torch.zeros(M, C, dtype=BF16, device=dev())
    tail = torch.randn(500, C, generator=torch.Generator().manual_seed(1)).to(BF16)
    x[-500:] = tail.to(dev())
    so = torch.tensor([0, M - 500, M - 300, M], dtype=torch.int32, device=dev())
    y = ops.group_norm(x, so, 8, activation="silu", dropout=0.5, key=key())
    D = R.keep_mask(500, C, 0.5, SEED, 5, first_row=M - 500).double() * 2
    ref = R.group_norm(tail, [0, 200, 500], 8, name="silu", D=D)
    assert R.off("y", y[-500:], ref, BF16, ref["cond"][0]) <= 1
    assert not y[:-500].any()
    z = ops.dropout(x, 0.5, key())
    assert torch.equal(z[-500:].cpu().double(), tail.double() * D)


# ---------------------------------------------------------------------------------------------------- a run of them together
def test_modules_on_a_sparse_tensor_and_the_matching_gradient():
    """conv -> group norm + SiLU + dropout -> average pooling -> group norm + GELU -> global pooling -> dropout -> linear, the parameters'
    gradients matched against constants with the squared distance, and the result differentiated into the features: the whole in
    float64 on the CPU, with the kernels' own masks."""
    from dd3d_amd import nn as ME, ops
    from dd3d_amd.sparse import TensorField
    torch.manual_seed(0)
    B, n = 6, 60
    coords = torch.cat([torch.cat([torch.full((n, 1), float(i)), torch.zeros(n, 1), torch.randint(0, 14, (n, 2)).float()], 1) for i in range(B)])
    feats = torch.randn(B * n, 4)
    conv = ME.MinkowskiConvolution(4, 24, kernel_size=3, dimension=3).to(dev())
    gn1 = ME.MinkowskiGroupNorm(4, 24, activation="silu", dropout=0.2, seed=5).to(dev())
    pool = ME.MinkowskiAvgPooling(2, 2, dimension=3)
    gn2 = ME.MinkowskiGroupNorm(3, 24, activation="gelu").to(dev())
    gap, drop, lin = ME.MinkowskiGlobalAvgPooling(), ME.MinkowskiDropout(0.3, seed=6).to(dev()), ME.MinkowskiLinear(24, 5).to(dev())
    with torch.no_grad():
        for m in (gn1, gn2):
            m.weight.add_(0.2 * torch.randn(1, 24, device=dev()))
            m.bias.add_(0.2 * torch.randn(1, 24, device=dev()))
    labels = torch.arange(B) % 5
    params = [gn1.weight, gn1.bias, gn2.weight, gn2.bias, lin.linear.weight, lin.linear.bias]
    f = feats.to(dev()).requires_grad_()
    with ops.true_second_order():
        s0 = TensorField(features=f, coordinates=coords.to(dev()), device=dev(), num_clouds=B).sparse()
        s1 = gn1(conv(s0))
        s2 = gn2(pool(s1))
        logits = lin(drop(gap(s2))).F
    ce = torch.nn.functional.cross_entropy(logits, labels.to(dev()))
    gw = torch.autograd.grad(ce, params, create_graph=True)
    target = [0.1 * torch.randn(p.shape, generator=torch.Generator().manual_seed(i)) for i, p in enumerate(params)]
    loss = sum((a - t.to(dev())).square().sum() for a, t in zip(gw, target))
    grad, = torch.autograd.grad(loss, f)

    cm = s0.coordinate_manager
    M1, M2 = cm.num_rows(1), cm.num_rows(2)
    inv = cm.levels[1].inv[:B * n].long().cpu()
    nbr, kids = cm.kernel_map(1, 1, 3)[0][:, :M1].long().cpu(), cm.kernel_map(1, 2, 2)[0][:, :M2].long().cpu()
    segs = [[int(v) for v in cm.seg_off(ts)] for ts in (1, 2)]
    F = feats.double().requires_grad_()
    P = [p.detach().double().cpu().requires_grad_() for p in params]
    W = conv.kernel.detach().double().cpu()
    take = lambda X, at: torch.cat([X, X.new_zeros(1, X.shape[1])])[at]  # noqa: E731  (-1: the row of zeros)
    x0 = torch.zeros(M1, 4, dtype=torch.float64).index_add(0, inv, F) / torch.bincount(inv, minlength=M1)[:, None]
    y = sum(take(x0, nbr[k]) @ W[k] for k in range(27))

    def norm(X, seg, G, w, b):
        parts = []
        for r0, r1 in zip(seg[:-1], seg[1:]):
            Z = X[r0:r1].reshape(r1 - r0, G, -1)
            Z = Z - Z.mean((0, 2), keepdim=True)
            parts.append((Z / torch.sqrt((Z * Z).mean((0, 2), keepdim=True) + 1e-5)).reshape(r1 - r0, -1))
        return torch.cat(parts) * w + b

    a1 = torch.nn.functional.silu(norm(y, segs[0], 4, P[0], P[1])) * R.keep_mask(M1, 24, 0.2, 5, 0).double() / 0.8
    have = (kids >= 0).double().sum(0)[:, None]
    a2 = torch.nn.functional.gelu(norm(sum(take(a1, kids[k]) for k in range(8)) / have, segs[1], 3, P[2], P[3]))
    pooled = torch.stack([a2[r0:r1].mean(0) for r0, r1 in zip(segs[1][:-1], segs[1][1:])]) * R.keep_mask(B, 24, 0.3, 6, 0).double() / 0.7
    out = pooled @ P[4].t() + P[5]
    rgw = torch.autograd.grad(torch.nn.functional.cross_entropy(out, labels), P, create_graph=True)
    rloss = sum((a - t.double()).square().sum() for a, t in zip(rgw, target))
    rgrad, = torch.autograd.grad(rloss, F)
    assert float((logits.detach().cpu().double() - out).abs().max()) < 1e-4 * float(out.abs().max())
    for a, r in zip(gw, rgw):
        assert float((a.detach().cpu().double() - r).abs().max()) < 1e-4 * float(r.abs().max())
    assert float(loss) == pytest.approx(float(rloss), rel=1e-4)
    assert float((grad.cpu().double() - rgrad).abs().max()) < 1e-4 * float(rgrad.abs().max())
    # evaluation: no mask, and the generator stands still
    gn1.eval()
    drop.eval()
    with torch.no_grad():
        assert drop(s2) is s2 and torch.equal(gn1(conv(s0)).F, gn1(conv(s0)).F)
    assert gn1.rng_state.tolist() == [5, 1] and drop.rng_state.tolist() == [6, 1]
