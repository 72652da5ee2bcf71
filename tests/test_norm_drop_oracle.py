"""CPU checks of the float64 restatement of group norm + activation and counter-based dropout (oracle/norm_drop_ref.py): against torch's
autograd on the definition (first and second gradient), finite differences and the generator's published vectors; and of everything the
package refuses without a GPU."""
import numpy as np
import pytest
import torch

from oracle import norm_drop_ref as R

SEG = [0, 5, 5, 6, 17]


def definition(x, seg, G, w, b, eps, name, slope, D):
    Cg, parts = x.shape[1] // G, []
    for r0, r1 in zip(seg[:-1], seg[1:]):
        X = x[r0:r1].reshape(r1 - r0, G, Cg)
        if r1 > r0:
            cen = X - X.mean((0, 2), keepdim=True)
            X = cen / torch.sqrt((cen * cen).mean((0, 2), keepdim=True) + eps)
        parts.append(X.reshape(r1 - r0, G * Cg))
    u = torch.cat(parts) * w + b
    f = {"none": lambda t: t, "relu": torch.relu, "leaky_relu": lambda t: torch.nn.functional.leaky_relu(t, slope),
         "silu": lambda t: t * torch.sigmoid(t), "gelu": lambda t: t * 0.5 * (1 + torch.erf(t / 2 ** 0.5))}[name](u)
    return f * D


@pytest.mark.parametrize("name", ["none", "relu", "leaky_relu", "silu", "gelu"])
@pytest.mark.parametrize("C,G", [(6, 2), (5, 5), (4, 1)])
def test_formulas_equal_autograd_of_the_definition(name, C, G):
    g = torch.Generator().manual_seed(C * 10 + G)
    rn = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    M = SEG[-1]
    x, w, b, dy = (t.requires_grad_() for t in (1.5 * rn(M, C) + 0.3, 1 + 0.3 * rn(C), 0.3 * rn(C), rn(M, C)))
    D = (torch.rand(M, C, generator=g) > 0.3).double() / 0.7
    P, q, s = rn(M, C), rn(C), rn(C)
    y = definition(x, SEG, G, w, b, 1e-3, name, 0.2, D)
    first = torch.autograd.grad(y, (x, w, b), dy, create_graph=True)
    second = torch.autograd.grad(first, (dy, x, w, b), (P, q, s), allow_unused=True)
    ref = R.group_norm(x, SEG, G, w, b, 1e-3, name, 0.2, D, dy, P, q, s, order=2)
    for k, t in zip(("y", "dx", "dw", "db", "ddy", "ddx", "ddw", "ddb"), (y, *first, *second)):
        t = torch.zeros(C, dtype=torch.float64) if t is None else t.detach()
        assert (ref[k][0] - t).abs().max() <= 1e-9 * (1 + t.abs().max()), k
        assert (ref[k][0].abs() <= ref[k][1] * (1 + 1e-9)).all(), k + ": a result beyond the size of its terms"


def test_gradients_equal_finite_differences():
    g = torch.Generator().manual_seed(3)
    rn = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x, w, b, dy, P, q, s = rn(17, 6), 1 + 0.2 * rn(6), 0.2 * rn(6), rn(17, 6), rn(17, 6), rn(6), rn(6)
    one = lambda k, x, w, b, dy: R.group_norm(x, SEG, 3, w, b, 1e-2, "gelu", dy=dy, ggx=P, ggw=q, ggb=s, order=2)[k][0]  # noqa: E731
    h, dirs = 1e-6, {"x": rn(17, 6), "w": rn(6), "b": rn(6), "dy": rn(17, 6)}
    for k, d in dirs.items():
        at = dict(x=x, w=w, b=b, dy=dy)
        up, down = dict(at, **{k: at[k] + h * d}), dict(at, **{k: at[k] - h * d})
        if k != "dy":
            num = ((one("y", **up) - one("y", **down)) * dy).sum() / (2 * h)
            assert num == pytest.approx(float((one("d" + k, **at) * d).sum()), rel=1e-6)
        num = sum(((one(n, **up) - one(n, **down)) * c).sum() for n, c in (("dx", P), ("dw", q), ("db", s))) / (2 * h)
        assert num == pytest.approx(float((one("d" + ("dy" if k == "dy" else "d" + k), **at) * d).sum()), rel=1e-6)


def test_random_words_are_the_published_ones():
    w = lambda *v: np.array(v, dtype=np.uint32)  # noqa: E731
    assert R.philox4x32(w(0, 0, 0, 0), w(0, 0)).tolist() == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    f = 0xffffffff
    assert R.philox4x32(w(f, f, f, f), w(f, f)).tolist() == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    assert R.philox4x32(w(0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), w(0xa4093822, 0x299f31d0)).tolist() == [
        0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]


def test_kept_share_and_independence_of_calls():
    a, b = R.keep_mask(500, 128, 0.3, 7, 0), R.keep_mask(500, 128, 0.3, 7, 1)
    n = a.numel()
    for m in (a, b):      # a binomial share: five standard deviations
        assert abs(float(m.double().mean()) - 0.7) < 5 * (0.21 / n) ** 0.5
    assert abs(float((a & b).double().mean()) - 0.49) < 5 * (0.25 / n) ** 0.5
    assert torch.equal(R.keep_mask(100, 9, 0.5, 1, 2, first_row=37), R.keep_mask(137, 9, 0.5, 1, 2)[37:])


# ------------------------------------------------------------------------------------------------------------------- refusals
def test_c_entry_points_refuse_bad_arguments_before_any_launch():
    from dd3d_amd import _lib as L
    lib, one = L.lib, 256      # a non-null address: nothing is launched, so nothing reads it
    ws = lib.dd3d_group_norm_ws_bytes
    assert ws(1000, 128, 10, 8, 0) >= 0 and ws(1000, 128, 10, 8, 2) > 0
    assert ws(-1, 128, 10, 8, 0) == -1 and ws(10, 10, 1, 3, 0) == -1 and ws(10, 8, 1, 2, 3) == -1
    assert ws(2 ** 31, 8, 1, 2, 0) == -2 and ws(10, 4098, 1, 2, 0) == -2

    def fwd(dtype=0, M=10, C=8, seg=one, B=1, G=2, w=one, b=one, pdt=0, eps=1e-5, act=0, slope=0.1, p=0.0, key=None, x=one, y=one, mean=None, rstd=None):
        return lib.dd3d_group_norm_fwd(x, dtype, M, C, seg, B, G, w, b, pdt, eps, act, slope, p, key, y, mean, rstd, None, 0, None)
    for bad in (dict(dtype=3), dict(dtype=-1), dict(M=-1), dict(C=0), dict(C=9), dict(G=0), dict(B=-1), dict(seg=None), dict(pdt=1), dict(eps=0.0),
                dict(eps=float("nan")), dict(eps=1e-40), dict(eps=float("inf")), dict(act=5), dict(act=-1), dict(slope=float("nan")), dict(p=-0.1), dict(p=1.5), dict(p=float("nan")), dict(p=0.5),
                dict(x=None), dict(y=None), dict(mean=one), dict(rstd=one)):
        assert fwd(**bad) == -1, bad
    for bad in (dict(M=2 ** 31), dict(C=4098, G=2), dict(B=2 ** 30, G=8)):
        assert fwd(**bad) == -2, bad

    def bwd(second=False, dy=one, x=one, mean=one, rstd=one, C=8):
        head = (0, 10, C, one, 1, 2, one, one, 0, 0, 0.1, 0.0, None, mean, rstd)
        if second:
            return lib.dd3d_group_norm_bwd2(None, None, None, dy, x, *head, one, one, one, one, None, 0, None)
        return lib.dd3d_group_norm_bwd(dy, x, *head, one, one, one, None, 0, None)
    for second in (False, True):
        for bad in (dict(dy=None), dict(x=None), dict(mean=None), dict(rstd=None), dict(C=7)):
            assert bwd(second, **bad) == -1, (second, bad)
    assert bwd(True) == -3
    drop = lambda p=0.5, key=one, rows=4, C=4, dt=0, x=one: lib.dd3d_dropout(x, dt, rows, C, p, key, one, None)  # noqa: E731
    for bad in (dict(p=-1.0), dict(p=2.0), dict(key=None), dict(rows=-1), dict(C=-1), dict(dt=7), dict(x=None)):
        assert drop(**bad) == -1, bad
    assert drop(rows=2 ** 50, C=2 ** 20) == -2 and drop(rows=0, x=None) == 0
    assert lib.dd3d_random_key(None, one, None) == -1


def test_rows_and_clouds_whose_counters_would_leave_32_bits_are_refused():
    """A walk over rows steps by up to 4096 (a chunk), one over clouds by up to 32 768 (a launch's workgroups), and tests for the end after the step."""
    from dd3d_amd import _lib as L, ops
    lib, one, most = L.lib, 256, 2 ** 31 - 65536
    assert most - 1 + 32768 < 2 ** 31
    ws = lib.dd3d_group_norm_ws_bytes
    for order in (0, 1, 2):
        assert ws(most, 1, 1, 1, order) >= 0 and ws(1000, 1, most, 1, order) >= 0 and ws(1000, 8, most // 8, 8, order) >= 0
        for bad in ((most + 1, 1, 1, 1), (2 ** 31 - 1, 1, 1, 1), (1000, 1, most + 1, 1), (1000, 1, 2 ** 31 - 1, 1), (1000, 8, most // 8 + 1, 8)):
            assert ws(*bad, order) == -2, bad
    for M, B in ((most + 1, 1), (2 ** 31 - 1, 1), (10, most + 1), (10, 2 ** 31 - 1)):
        head = (0, M, 1, one, B, 1, one, one, 0)
        assert lib.dd3d_group_norm_fwd(one, *head, 1e-5, 0, 0.0, 0.0, None, one, None, None, None, 0, None) == -2
        assert lib.dd3d_group_norm_bwd(one, one, *head, 0, 0.0, 0.0, None, one, one, one, one, one, None, 0, None) == -2
        assert lib.dd3d_group_norm_bwd2(None, None, None, one, one, *head, 0, 0.0, 0.0, None, one, one, one, one, one, one, None, 0, None) == -2
    rows, seg = torch.empty(most + 1, 1, device="meta"), torch.empty(2, dtype=torch.int32, device="meta")
    with pytest.raises(ValueError, match="rows"):
        ops.group_norm(rows, seg, 1)
    with pytest.raises(ValueError, match="clouds times groups"):
        ops.group_norm(rows[:10], torch.empty(most + 2, dtype=torch.int32, device="meta"), 1)
    with pytest.raises(ValueError, match="clouds times groups"):
        ops.group_norm(torch.empty(10, 8, device="meta"), torch.empty(most // 8 + 2, dtype=torch.int32, device="meta"), 8)


def test_python_entry_points_refuse_bad_arguments():
    from dd3d_amd import nn as ME, ops
    x, seg, key = torch.zeros(6, 8), torch.tensor([0, 6], dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    gn = lambda x=x, seg=seg, G=2, w=None, b=None, **k: ops.group_norm(x, seg, G, w, b, **k)  # noqa: E731
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        gn()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.dropout(x, 0.5, key)
    with pytest.raises(RuntimeError):
        gn(x=x.double())
    with pytest.raises(RuntimeError):
        ops.dropout(x.long(), 0.5, key)
    for bad in (dict(x=x[0]), dict(G=3), dict(G=0), dict(G=16), dict(seg=seg.long()), dict(seg=seg[None]), dict(seg=seg[:0]), dict(w=torch.ones(7)),
                dict(w=torch.ones(8, dtype=torch.float64)), dict(w=torch.ones(8, dtype=torch.bfloat16)), dict(activation="tanh"), dict(eps=0.0),
                dict(eps=float("nan")), dict(eps=1e-40), dict(eps=float("inf")), dict(negative_slope=float("nan")), dict(dropout=1.2, key=key), dict(dropout=-0.1, key=key), dict(dropout=0.3),
                dict(dropout=0.3, key=key.int()), dict(dropout=0.3, key=key[:1]), dict(x=torch.zeros(2, 4100), G=1)):
        with pytest.raises(ValueError):
            gn(**bad)
    with pytest.raises(ValueError):
        gn(x=x.half(), w=torch.ones(8).half(), b=torch.ones(8))
    for bad in (dict(p=2.0, key=key), dict(p=float("nan"), key=key), dict(p=0.5, key=None), dict(p=0.5, key=key.float())):
        with pytest.raises(ValueError):
            ops.dropout(x, **bad)
    with pytest.raises(ValueError):
        ops.random_key(torch.zeros(3, dtype=torch.int64))
    for bad in (lambda: ME.MinkowskiDropout(1.5), lambda: ME.MinkowskiGroupNorm(3, 8), lambda: ME.MinkowskiGroupNorm(2, 8, activation="tanh"),
                lambda: ME.MinkowskiGroupNorm(2, 8, dropout=-1)):
        with pytest.raises(ValueError):
            bad()


def test_modules_keep_the_norms_parameters_and_no_generator_state():
    from dd3d_amd import nn as ME, ops
    m = ME.MinkowskiGroupNorm(4, 16, activation="silu", dropout=0.1, seed=3)
    assert {k: tuple(v.shape) for k, v in m.state_dict().items()} == {"weight": (1, 16), "bias": (1, 16)}
    assert m.rng_state.tolist() == [3, 0] and not list(ME.MinkowskiGroupNorm(4, 16, affine=False).parameters())
    assert ops.random_state(2 ** 64 - 1).tolist() == [-1, 0] and ops.random_state(-5).tolist() == [-5, 0]
    torch.manual_seed(11)
    a = ME.MinkowskiDropout().rng_state
    torch.manual_seed(11)
    assert torch.equal(a, ME.MinkowskiDropout().rng_state)
    assert ME.MinkowskiDropout(0.5).eval()(x := object()) is x and ME.MinkowskiDropout(0.0)(x) is x
    assert "activation=silu" in repr(m) and "p=0.5" in repr(ME.MinkowskiDropout())


def test_the_module_takes_its_own_number_of_channels_only():
    """Without weight and bias a tensor of another width would be normalised in groups that nobody asked for."""
    from types import SimpleNamespace
    from dd3d_amd import nn as ME
    x = SimpleNamespace(F=torch.zeros(6, 16), coordinate_manager=SimpleNamespace(seg_off=lambda ts: torch.tensor([0, 6], dtype=torch.int32)), tensor_stride=1)
    for affine in (False, True):
        with pytest.raises(ValueError, match="8 channels got 16"):
            ME.MinkowskiGroupNorm(2, 8, affine=affine)(x)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ME.MinkowskiGroupNorm(2, 16, affine=False)(x)


def test_a_fraction_of_groups_is_refused_by_name():
    from dd3d_amd import ops
    with pytest.raises(ValueError, match="do not divide into 2.5 groups"):
        ops.group_norm(torch.zeros(6, 5), torch.tensor([0, 6], dtype=torch.int32), 2.5)


def test_the_flag_of_the_two_float_means_takes_no_other_number():
    from dd3d_amd import _lib as L
    def fwd(act):
        return L.lib.dd3d_group_norm_fwd(256, 0, 1000, 8, 256, 1, 2, None, None, 0, 1e-5, act, 0.0, 0.0, None, 256, None, None, None, 0, None)
    for act in (5, 16 + 5, 15, 32, 48, -1, -16, -12):
        assert fwd(act) == -1, act
    for act in (0, 4, 16, 16 + 4):
        assert fwd(act) == -3, act      # as far as the workspace, which is missing
