"""clip_grads and adam_step_tensors write tensors by their addresses: autograd's version counters have to count it, so that a backward through a
saved tensor that they overwrote is an error and no wrong gradient.  Needs a GPU."""
import math

import pytest
import torch

from neural_invertible_warp_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def state(n=300, dtype=torch.float32):
    s = dict(params=[torch.randn(n, device=DEV).to(dtype).requires_grad_(), torch.randn(7, device=DEV).to(dtype).requires_grad_()])
    s["grads"] = [torch.randn_like(p).detach() for p in s["params"]]
    s["exp_avg"] = [torch.zeros(p.shape, device=DEV) for p in s["params"]]
    s["exp_avg_sq"] = [torch.zeros(p.shape, device=DEV) for p in s["params"]]
    if dtype != torch.float32:
        s["master"] = [p.detach().float() for p in s["params"]]
    return s


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("max_norm", [None, 1.0])
def test_a_backward_through_an_updated_parameter_is_an_error(dtype, kept, max_norm):
    s = state(dtype=dtype)
    table = ops.AdamTable([s]) if kept else [s]
    for _ in range(2):                                                       # (a kept table at every call, not at its first alone)
        y = sum((p * p).sum() for p in s["params"])
        before = {k: [t._version for t in v] for k, v in s.items()}
        ops.adam_step_tensors(table, lr=1e-2, step=1, max_norm=max_norm)
        for k, v in s.items():
            assert all((t._version > b) == (k != "grads") for t, b in zip(v, before[k])), k
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()


@pytest.mark.parametrize("kept", [False, True])
def test_a_backward_through_a_clipped_gradient_is_an_error(kept):
    p = torch.randn(50, device=DEV, requires_grad=True)
    g, = torch.autograd.grad((p ** 3).sum(), p, create_graph=True)
    y = (g * g).sum()
    given = ops.TensorTable([g.detach()]) if kept else [g.detach()]          # (a detached tensor shares its version counter)
    assert math.isfinite(float(ops.grad_norm(given)))
    torch.autograd.grad(y, p, retain_graph=True)                             # a norm writes nothing
    ops.clip_grads(given, 1e-3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, p)


def test_outputs_are_counted_and_their_sources_are_not():
    g, out = torch.randn(90, device=DEV), torch.zeros(90, device=DEV)
    a, b = g._version, out._version
    ops.clip_grads([g], 1e-3, out=[out])
    assert g._version == a and out._version > b


def test_views_count_in_what_they_are_views_of():
    bucket = torch.randn(1000, device=DEV)
    views, other = list(bucket.split([10, 490, 500])), bucket.view(10, 100)
    before = bucket._version
    ops.clip_grads(ops.TensorTable(views), 1e-3)
    assert bucket._version > before and other._version == bucket._version == views[1]._version


def test_tensors_made_in_inference_mode_have_no_counter():
    with torch.inference_mode():
        g = torch.randn(90, device=DEV)
        ops.clip_grads([g], 1e-3)
    norm = ops.clip_grads([g, torch.randn(5, device=DEV)], 1e-3)
    assert math.isfinite(float(norm))
