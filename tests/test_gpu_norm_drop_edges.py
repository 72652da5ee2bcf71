"""Group norm and dropout at the edges of their range, on the GPU.  Reference and counts of roundings: oracle/norm_drop_ref.py."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import norm_drop_ref as R
from tests.test_gpu_norm_drop import BF16, F16, F32, MIXED, batch, check, dev, through_autograd


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
def test_gelu_at_minus_infinity_is_its_limit(dtype):
    from dd3d_amd import ops
    seg, t = batch(MIXED, 8, dtype, seed=36)
    y = ops.group_norm(t["x"].to(dev()), seg_on_device(seg), 2, None, torch.full((8,), -math.inf, device=dev()), activation="gelu")
    assert not y.any()
