"""Decoupled weight decay of ops.adam_step_tensors, p (1 - lr wd), at the values where p - lr wd p is something else: infinite parameters and
zeros; and groups without decay beside groups that decay, which keep the bits of ops.adam_step_multi.  Needs a GPU."""
import math

import pytest
import torch

from neural_invertible_warp_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
ODD = [math.inf, -math.inf, math.nan, 0.0, -0.0, 3.4028234663852886e38, 1e-45, -1e-45]


def state(n, seed, still, dtype=F32):
    """one tensor of n parameters, every 16th of them one of ODD (those of `still` have no gradient and no moments: their update is 0)"""
    r = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda: torch.randn(n, device=DEV, generator=r)
    p, g, m, v = rand(), rand(), rand() * 0.3, rand().square() * 0.2 + 1e-12
    for k, x in enumerate(ODD):
        p[16 + 2 * k::16 * len(ODD)] = x
        if still:
            for t in (g, m, v):
                t[16 + 2 * k::16 * len(ODD)] = 0.0
    s = dict(params=[p.to(dtype)], grads=[g], exp_avg=[m], exp_avg_sq=[v])
    if dtype != F32:
        s["master"] = [p]
    return s


def copy(s):
    return {k: [x.clone() for x in v] for k, v in s.items()}


def same_bits(a, b):
    return torch.equal(a.view(torch.int32), b.view(torch.int32))


@pytest.mark.parametrize("n", [5, 1000, 70001])
@pytest.mark.parametrize("still", [False, True])
@pytest.mark.parametrize("max_norm", [None, math.inf])
@pytest.mark.parametrize("where", ["host", "device"])
def test_a_group_without_decay_keeps_its_bits_beside_one_that_decays(n, still, max_norm, where):
    a, b = state(n, 1, still), state(n, 2, still)
    want, other = copy(b), copy(a)
    lr, step = [1e-2, 1e-3], [4, 9]
    decay = dict(weight_decay=[0.1, 0.0]) if where == "host" else dict(decay_dev=torch.tensor([1e-3, 0.0], device=DEV))
    for _ in range(3):
        ops.adam_step_tensors([a, b], lr=lr, step=step, max_norm=max_norm, **decay)
        ops.adam_step_multi([(*[want[k][0] for k in ("params", "grads", "exp_avg", "exp_avg_sq")], lr[1], step[1])])
        ops.adam_step_tensors([other], lr=lr[0], step=step[0], weight_decay=0.1, max_norm=max_norm)
    for k in ("params", "exp_avg", "exp_avg_sq"):
        assert same_bits(b[k][0], want[k][0]), k
        assert same_bits(a[k][0], other[k][0]), k                            # and the decaying group is what it is alone


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("n", [5, 70001])
@pytest.mark.parametrize("rate", [1e-9, 1e-3, 0.5, 1.0, 3.0])
@pytest.mark.parametrize("where", ["host", "device"])
def test_decay_of_infinities_and_zeros_is_the_product(dtype, n, rate, where):
    """elements whose update is 0 become p (1 - rate), in 64 bits and rounded once (the rate itself is rounded to fp32: half a step of
    rate p more)"""
    s = state(n, 3, True, dtype)
    rate = float(torch.tensor(rate, dtype=F32))
    w = s["params" if dtype == F32 else "master"][0]
    still = (s["grads"][0] == 0) & (s["exp_avg"][0] == 0)
    before = w.double()
    decay = dict(lr=1.0, step=1, weight_decay=rate) if where == "host" else \
        dict(lr=0.0, step=0, hyper_dev=torch.tensor([ops.adam_hyper(1.0, 1)], device=DEV, dtype=F32), decay_dev=torch.tensor([rate], device=DEV))
    ops.adam_step_tensors([s], **decay)
    want, got = (before * (1.0 - rate))[still], w[still].double()
    rounded = want.to(F32).double()                                          # (twice the largest fp32 value rounds to infinity)
    assert torch.equal(rounded.isnan(), got.isnan()) and torch.equal(rounded.isinf(), got.isinf())
    inf, finite = rounded.isinf(), rounded.isfinite()
    assert torch.equal(rounded[inf], got[inf])
    assert bool(((got - want).abs()[finite] <= 2.0 ** -24 * (1 + 1e-6) * (want.abs() + rate * before[still].abs())[finite] + 2.0 ** -150).all())
    zero = before[still] == 0
    assert torch.equal(want[zero].signbit(), got[zero].signbit())
    if dtype != F32:
        assert torch.equal(s["params"][0].view(torch.int16), w.to(dtype).view(torch.int16)) or bool((s["params"][0].isnan() == w.isnan()).all())
