"""The operators over lists of many tensors (ops.grad_norm, ops.clip_grads, ops.adam_step_tensors; csrc/niw_optim.hip) against their
formulas in 64 bits.

Tolerances are counted roundings: fp32 half a step is H = 2^-24 of the value, bf16 2^-8, fp16 2^-11 (and half of the smallest fp16 step,
2^-25, below its normal range)."""
import math
import random
import threading

import pytest
import torch

from neural_invertible_warp_amd import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
H = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


def rand(n, dtype=F32, scale=1.0, seed=0, offset=0):
    """n values in a tensor that begins `offset` elements behind an allocation's start"""
    g = torch.Generator(device=DEV).manual_seed(seed * 7919 + n)
    return (torch.randn(n + offset, device=DEV, generator=g) * scale).to(dtype)[offset:]


def exact_norm(tensors, kind=2.0):
    if not any(t.numel() for t in tensors):
        return 0.0
    if kind == 2.0:
        return math.sqrt(sum(float(t.double().square().sum()) for t in tensors))
    return max(float(t.double().abs().max()) for t in tensors if t.numel())


def check_norm(norm, tensors, kind=2.0):
    """sum in 64 bits (its own rounding is below 1e-12), then the root rounded to fp32 once"""
    want = exact_norm(tensors, kind)
    assert norm.dtype == F32 and norm.shape == () and norm.device == torch.device(DEV)
    assert abs(float(norm) - want) <= H * want * (1 + 1e-6), (float(norm), want)


def coefficient(norm, max_norm):
    return min(1.0, max_norm / (norm + 1e-6))


def check_clipped(out, before, c):
    """c rounded to fp32, the product rounded to fp32, the result rounded to its type; c = 1 is exact"""
    want = before.double() * c
    tol = want.abs() * ((HALF[out.dtype] if out.dtype != F32 else 0.0) + 2 * H) * (1 + 1e-3) + TINY[out.dtype]
    assert bool(((out.double() - want).abs() <= tol).all()), float((out.double() - want).abs().max())


LENGTHS = [[1], [2, 1], [255], [256], [257], [1023, 1025], [16383], [16384], [16385], [65537], [0, 5, 0, 16384 * 3 + 1], [1000003], [7] * 250, [3, 70001] * 61,
           [0], [17_000_003], [9_000_001, 1, 8_388_608]]


@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda v: f"{len(v)}x{max(v)}")
@pytest.mark.parametrize("kept", [False, True])
def test_norm(lengths, dtype, kind, kept):
    tensors = [rand(n, dtype, seed=i, offset=i % 3) for i, n in enumerate(lengths)]
    given = ops.TensorTable(tensors) if kept else tensors
    check_norm(ops.grad_norm(given, norm_type=kind), tensors, kind)
    total = ops.grad_total(given, norm_type=kind)
    assert total.dtype == torch.float64 and total.shape == (1,)
    want = exact_norm(tensors, kind) ** (2 if kind == 2.0 else 1)
    assert abs(float(total) - want) <= 1e-12 * want


def test_norm_of_nothing():
    for nothing in ([], [None], [torch.empty(0, device=DEV)]):
        assert float(ops.grad_norm(nothing)) == 0.0 and float(ops.grad_norm(nothing, norm_type=math.inf)) == 0.0
        assert float(ops.grad_total(nothing)) == 0.0
        assert float(ops.clip_grads(nothing, 1.0)) == 0.0


@pytest.mark.parametrize("kind", [2.0, math.inf])
def test_norm_of_mixed_types_orders_and_shapes(kind):
    t = [rand(600, BF16).view(20, 30).t(), rand(1, F32).view(()), rand(24, F16).view(2, 3, 4).permute(2, 0, 1), rand(5000, F32), None, rand(64, BF16).view(1, 64, 1)]
    check_norm(ops.grad_norm(t, norm_type=kind), [x for x in t if x is not None], kind)
    same = rand(1000)
    check_norm(ops.grad_norm([same, same]), [same, same])                    # the same tensor twice counts twice
    check_norm(ops.grad_norm(same), [same])                                  # one tensor, no list


@pytest.mark.parametrize("scale", [1e-30, 3e-39, 1e25, 1e38])
def test_norm_neither_overflows_nor_underflows(scale):
    t = [rand(3000, F32).clamp(-3, 3) * scale, rand(50, F32).clamp(-3, 3) * scale]
    check_norm(ops.grad_norm(t), t) if scale < 1e38 else None
    want = sum(float(x.double().square().sum()) for x in t)
    assert math.isfinite(want) and abs(float(ops.grad_total(t)) - want) <= 1e-12 * want


@pytest.mark.parametrize("where", [0, 4097, 69999])
@pytest.mark.parametrize("dtype", TYPES)
def test_norm_of_what_is_not_finite(dtype, where):
    for value, want in ((math.inf, math.inf), (-math.inf, math.inf), (math.nan, math.nan)):
        t = [rand(333, dtype), rand(70000, dtype, seed=1)]
        t[1][where] = value
        for kind in (2.0, math.inf):
            got = float(ops.grad_norm(t, norm_type=kind))
            assert got == want or (math.isnan(got) and math.isnan(want))
        t[0][7] = math.inf                                                   # an infinity beside it: a NaN stays a NaN
        got = float(ops.grad_norm(t, norm_type=math.inf))
        assert got == want or (math.isnan(got) and math.isnan(want))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_offsets_that_pass_32_bits(dtype):
    n = (1 << 31) + 77 if dtype == BF16 else (1 << 30) + 77                  # more than 2^32 bytes
    x = torch.zeros(n, device=DEV, dtype=dtype)
    places = [0, 1, n // 2, (1 << 31) // (2 if dtype == F32 else 1) - 1, n - 2, n - 1]
    for i, p in enumerate(places):
        x[p] = float(i + 1)
    want = math.sqrt(sum((i + 1) ** 2 for i in range(len(places))))
    assert abs(float(ops.grad_norm([x])) - want) <= H * want
    norm = ops.clip_grads([x], want / 4)
    assert abs(float(norm) - want) <= H * want
    c = coefficient(want, want / 4)
    got = torch.stack([x[p] for p in places])
    check_clipped(got, torch.arange(1, len(places) + 1, device=DEV, dtype=dtype), c)
    assert int((x != 0).sum()) == len(places)


# ------------------------------------------------------------------------------------------ clipping
OUTS = [(F32, None), (BF16, None), (F16, None), (F32, F32), (BF16, F32), (F16, F32), (BF16, BF16), (F32, BF16), (F16, F16), (BF16, F16)]


@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("dtype,out_dtype", OUTS, ids=str)
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda v: f"{len(v)}x{max(v)}")
@pytest.mark.parametrize("kept", [False, True])
def test_clip(lengths, dtype, out_dtype, kind, kept):
    before = [rand(n, dtype, seed=i, offset=i % 3) for i, n in enumerate(lengths)]
    g = [x.clone() for x in before]
    out = None if out_dtype is None else [torch.empty(n, device=DEV, dtype=out_dtype) for n in lengths]
    want = exact_norm(before, kind)
    max_norm = 0.37 * want + 1e-3 * (want == 0)
    norm = ops.clip_grads(ops.TensorTable(g, out=out), max_norm, norm_type=kind) if kept else ops.clip_grads(g, max_norm, norm_type=kind, out=out)
    check_norm(norm, before, kind)
    for x, b, o in zip(g, before, g if out is None else out):
        check_clipped(o, b, coefficient(want, max_norm))
        assert out is None or torch.equal(x, b)


@pytest.mark.parametrize("dtype", TYPES)
def test_clip_leaves_what_lies_between_and_behind_the_tensors(dtype):
    flat = rand(300000, dtype, seed=5)
    before = flat.clone()
    cuts = [(1, 5), (5, 8), (11, 20011), (20012, 20013), (20480, 20480), (30003, 299990)]
    views = [flat[a:b] for a, b in cuts]
    norm = ops.clip_grads(views, 0.5)
    inside = torch.zeros(300000, dtype=torch.bool, device=DEV)
    for a, b in cuts:
        inside[a:b] = True
    assert torch.equal(flat[~inside], before[~inside])
    check_norm(norm, [before[inside]])
    check_clipped(flat[inside], before[inside], coefficient(exact_norm([before[inside]]), 0.5))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("max_norm", [1e9, math.inf])
def test_clip_under_the_limit_changes_nothing(dtype, max_norm):
    g = [rand(n, dtype, seed=n) for n in (1, 300, 70001)]
    before = [x.clone() for x in g]
    out = [torch.full_like(x, 7.0) for x in g]
    ops.clip_grads(g, max_norm)
    ops.clip_grads(g, max_norm, out=out)
    assert all(torch.equal(a, b) and torch.equal(a, o) for a, b, o in zip(g, before, out))


def test_clip_follows_its_formula_where_the_norm_is_not_finite():
    for value in (math.inf, math.nan):
        g = [rand(5000), rand(77, BF16)]
        g[0][11] = value
        norm = float(ops.clip_grads(g, 1.0))
        if math.isnan(value):
            assert math.isnan(norm) and all(bool(x.isnan().all()) for x in g)
        else:
            assert norm == math.inf and bool(g[0][11].isnan()) and int(g[0].isnan().sum()) == 1 and float(g[0].nan_to_num().abs().max()) == 0.0 and bool((g[1] == 0).all())
        g = [rand(5000), rand(77, BF16)]
        before = [x.clone() for x in g]
        g[0][11] = before[0][11] = value
        ops.clip_grads(g, math.inf)
        assert all(torch.equal(a.nan_to_num(nan=5.0), b.nan_to_num(nan=5.0)) for a, b in zip(g, before))
    zeros = [torch.zeros(300, device=DEV)]
    assert float(ops.clip_grads(zeros, 0.0)) == 0.0 and not bool(zeros[0].any())
    g = [rand(300)]
    ops.clip_grads(g, 0.0)
    assert not bool(g[0].any())


def test_clip_of_permuted_tensors_pairs_elements_by_their_place():
    g = rand(60).view(3, 4, 5).permute(2, 0, 1)
    out = torch.empty(3, 4, 5, device=DEV).permute(2, 0, 1)
    ops.clip_grads([g], 0.1, out=[out])
    check_clipped(out, g, coefficient(exact_norm([g]), 0.1))


def test_clip_refuses_tensors_that_share_memory():
    x = rand(100)
    for lists in ([x, x], [x, x[50:]], [x[:60], x[59:]]):
        with pytest.raises(_lib.NiwError, match="overlap"):
            ops.clip_grads(lists, 1.0)
        ops.grad_norm(lists)
    with pytest.raises(_lib.NiwError, match="overlap"):
        ops.clip_grads([x[:50]], 1.0, out=[x[10:60]])
    ops.clip_grads([x[:50], x[50:]], 1.0)


def test_total_of_several_shares():
    """two ranks' shares: their totals, summed, clip each share by the global norm"""
    a, b = [rand(5000), rand(7, BF16)], [rand(3000, F16)]
    want = exact_norm(a + b)
    total = ops.grad_total(a) + ops.grad_total(b)
    before = [x.clone() for x in a + b]
    for share in (a, b):
        norm = ops.clip_grads(share, 3.0, total=total)
        assert abs(float(norm) - want) <= H * want * (1 + 1e-6)
    for x, y in zip(a + b, before):
        check_clipped(x, y, coefficient(want, 3.0))
    assert abs(float(ops.clip_grads([], 3.0, total=total)) - want) <= H * want * (1 + 1e-6)          # a rank whose share is empty
    with pytest.raises(_lib.NiwError, match="grad_total"):
        ops.clip_grads(a, 1.0, total=torch.zeros(1, device=DEV))


# ------------------------------------------------------------------------------------------ Adam
def adam_state(lengths, pt, gt, seed=0, offset=0, scale=1.0):
    params = [rand(n, F32, seed=4 * i + seed, offset=offset) for i, n in enumerate(lengths)]
    master = None if pt == F32 else [p.clone() for p in params]
    mk = lambda j, f: [f(rand(n, F32, seed=4 * i + j + seed, offset=(i * j) % 3 if offset else 0)) for i, n in enumerate(lengths)]
    return dict(params=[p.to(pt) for p in params] if pt != F32 else params, grads=[rand(n, gt, scale=scale, seed=4 * i + 1 + seed, offset=offset) for i, n in enumerate(lengths)],
                exp_avg=mk(2, lambda x: x * 0.3 * scale), exp_avg_sq=mk(3, lambda x: x * x * 0.2 * scale ** 2 + 1e-12 * scale ** 2), master=master)


def copy_state(s):
    return {k: None if v is None else [x.clone() for x in v] for k, v in s.items()}


def check_adam(after, before, c, lr, step, decay, b1=0.9, b2=0.999, eps=1e-8):
    """Each quantity against the formula in 64 bits, with its roundings counted in H (|x|(1+H) slack aside):
    g: the product c g and c itself (2);  m: w1 (1), g - m (1) and g's own, the fma (1);  v: w2 and w2 g and g twice (6) of its new part, b2 and the
    product (2) of its old, the fma (1);  the update: m's and v's errors, then sqrt, bias correction and its division, eps, the sum, the division,
    the step size (7);  p: the decay's coefficient, its fma (1 of p), the last fma (1)."""
    for i in range(len(before["params"])):
        g, m0, v0 = (before[k][i].double() for k in ("grads", "exp_avg", "exp_avg_sq"))
        w0 = (before["params"] if before["master"] is None else before["master"])[i].double()
        g = g * c
        m = m0 + (1 - b1) * (g - m0)
        v = b2 * v0 + (1 - b2) * g * g
        bc1, bc2 = 1 - b1 ** step, math.sqrt(1 - b2 ** step)
        denom = v.sqrt() / bc2 + eps
        p1 = w0 - lr * decay * w0
        u = lr / bc1 * m / denom
        em = H * (m.abs() + (1 - b1) * (2 * (g - m0).abs() + 2 * g.abs()))
        ev = H * (v + 2 * b2 * v0 + 6 * (1 - b2) * g * g)
        rel_denom = ev / (2 * v).clamp_min(1e-300) + 5 * H
        eu = lr / bc1 * (em / denom + m.abs() / denom * (rel_denom + 2 * H))
        ep = H * (p1.abs() + lr * decay * w0.abs()) + eu + H * (p1 - u).abs()
        slack, least = 1 + 1e-3, 1e-37
        assert bool(((after["exp_avg"][i].double() - m).abs() <= em * slack + least).all())
        assert bool(((after["exp_avg_sq"][i].double() - v).abs() <= ev * slack + least).all())
        w = (after["params"] if after["master"] is None else after["master"])[i]
        assert bool(((w.double() - (p1 - u)).abs() <= ep * slack + least).all())
        if after["master"] is not None:
            assert torch.equal(after["params"][i], w.to(after["params"][i].dtype))          # the rounded master copy
        assert torch.equal(after["grads"][i], before["grads"][i])


COMBOS = [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)]


@pytest.mark.parametrize("pt,gt", COMBOS, ids=str)
@pytest.mark.parametrize("lengths", [[1], [255, 0, 257], [16385], [5] * 150, [1023, 70001, 2], [4_500_001], [17_000_003, 5]], ids=lambda v: f"{len(v)}x{max(v)}")
@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("clip,decay,offset", [(None, 0.0, 0), (0.5, 0.1, 0), (1e9, 0.01, 1), (0.3, 0.0, 3)])
def test_adam(lengths, pt, gt, clip, decay, offset, kept):
    s = adam_state(lengths, pt, gt, offset=offset)
    before = copy_state(s)
    lr, step = 1e-2, 7
    norm = ops.adam_step_tensors(ops.AdamTable([s]) if kept else [s], lr=lr, step=step, weight_decay=decay, max_norm=clip)
    if clip is None:
        assert norm is None
    else:
        check_norm(norm, before["grads"])
    check_adam(s, before, 1.0 if clip is None else coefficient(exact_norm(before["grads"]), clip), lr, step, decay)


def test_adam_groups_have_their_own_values():
    a, b, e = adam_state([300, 5000], F32, F32), adam_state([77], BF16, BF16, seed=50), dict(params=[], grads=[], exp_avg=[], exp_avg_sq=[])
    before = [copy_state(a), copy_state(b)]
    want = exact_norm(a["grads"] + b["grads"])
    norm = ops.adam_step_tensors([a, e, b], lr=[1e-3, 1.0, 2e-2], step=[3, 1, 900], weight_decay=[0.0, 0.0, 0.2], max_norm=want / 2, norm_type=2)
    check_norm(norm, before[0]["grads"] + before[1]["grads"])
    check_adam(a, before[0], coefficient(want, want / 2), 1e-3, 3, 0.0)
    check_adam(b, before[1], coefficient(want, want / 2), 2e-2, 900, 0.2)


def test_adam_without_a_clip_that_bites_has_the_bits_of_adam_step_multi():
    lengths = [530052, 165900, 2304, 1]
    a = adam_state(lengths, F32, F32)
    for x, value in ((a["params"][0], math.inf), (a["params"][1], -math.inf), (a["exp_avg"][0], 0.0), (a["exp_avg_sq"][0], 0.0)):
        x[5::1000] = value
    b, c = copy_state(a), copy_state(a)
    rows = lambda s: [(s["params"][i], s["grads"][i], s["exp_avg"][i], s["exp_avg_sq"][i], 1e-3, 5) for i in range(len(lengths))]
    for _ in range(3):
        ops.adam_step_multi(rows(a))
        ops.adam_step_tensors([b], lr=1e-3, step=5)
        ops.adam_step_tensors([c], lr=1e-3, step=5, max_norm=math.inf)
    for k in ("params", "exp_avg", "exp_avg_sq"):
        bits = lambda s: [x.view(torch.int32) for x in s[k]]
        assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(bits(a), bits(b), bits(c)))
    assert math.isinf(float(a["params"][0][5])) and math.isinf(float(c["params"][1][5]))


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_adam_skips_a_norm_that_is_not_finite(value):
    s = adam_state([5000, 33], BF16, F32)
    s["grads"][1][5] = value
    before = copy_state(s)
    norm = float(ops.adam_step_tensors([s], lr=1e-2, step=2, weight_decay=0.1, max_norm=1.0, skip_nonfinite=True))
    assert math.isnan(norm) if math.isnan(value) else norm == math.inf
    for k in ("params", "master", "exp_avg", "exp_avg_sq"):
        assert all(torch.equal(x, y) for x, y in zip(s[k], before[k]))
    s["grads"][1][5] = before["grads"][1][5] = 0.5
    ops.adam_step_tensors([s], lr=1e-2, step=2, weight_decay=0.1, max_norm=1.0, skip_nonfinite=True)
    check_adam(s, before, coefficient(exact_norm(before["grads"]), 1.0), 1e-2, 2, 0.1)


def test_adam_reads_its_scalars_from_the_device():
    s = adam_state([3000, 7], F32, F32)
    t = copy_state(s)
    hyper = torch.tensor([ops.adam_hyper(1e-2, 4)], device=DEV, dtype=F32)
    decay = torch.tensor([1e-2 * 0.1], device=DEV, dtype=F32)
    ops.adam_step_tensors([s], lr=1e-2, step=4, weight_decay=0.1, max_norm=0.2)
    ops.adam_step_tensors([t], lr=0.0, step=0, max_norm=0.2, hyper_dev=hyper, decay_dev=decay)
    for k in ("params", "exp_avg", "exp_avg_sq"):
        assert all(torch.equal(x, y) for x, y in zip(s[k], t[k]))
    with pytest.raises(_lib.NiwError, match="decay_dev"):
        ops.adam_step_tensors([t], lr=0.0, step=0, weight_decay=0.1, hyper_dev=hyper)
    with pytest.raises(_lib.NiwError, match="hyper_dev"):
        ops.adam_step_tensors([t], lr=0.0, step=0, hyper_dev=hyper[:, :1])


def test_adam_of_permuted_tensors_and_none_gradients():
    mk = lambda seed: rand(60, seed=seed).view(3, 4, 5).permute(2, 0, 1)
    s = dict(params=[mk(1), rand(4)], grads=[mk(2), None], exp_avg=[mk(3), rand(4)], exp_avg_sq=[mk(4) ** 2, rand(4)], master=None)
    s["exp_avg_sq"][0] = torch.empty(3, 4, 5, device=DEV).permute(2, 0, 1).copy_(s["exp_avg_sq"][0])
    before = {k: None if v is None else [None if x is None else x.clone() for x in v] for k, v in s.items()}
    ops.adam_step_tensors([s], lr=1e-2, step=1, max_norm=0.5)
    first = lambda d: {k: None if v is None else v[:1] for k, v in d.items()}
    check_adam(first(s), first(before), coefficient(exact_norm([before["grads"][0]]), 0.5), 1e-2, 1, 0.0)
    assert torch.equal(s["params"][1], before["params"][1]) and torch.equal(s["exp_avg"][1], before["exp_avg"][1])


def test_adam_offsets_that_pass_32_bits():
    n = (1 << 30) + 77                                                       # more than 2^32 bytes in every tensor
    z = lambda: torch.zeros(n, device=DEV)
    s = dict(params=[z()], grads=[z()], exp_avg=[z()], exp_avg_sq=[z()])
    places = [0, n // 2, (1 << 30) - 1, 1 << 30, n - 1]
    for i, p in enumerate(places):
        s["grads"][0][p] = float(i + 1)
    norm = ops.adam_step_tensors([s], lr=1e-2, step=1, max_norm=math.inf)
    want = math.sqrt(55.0)
    assert abs(float(norm) - want) <= H * want
    got = torch.stack([s["params"][0][p] for p in places]).double()
    assert bool(((got + 1e-2).abs() < 1e-6).all())                           # Adam's first step: lr against the gradient's sign
    assert int((s["params"][0] != 0).sum()) == len(places) == int((s["exp_avg"][0] != 0).sum())


# ------------------------------------------------------------------------------------------ how they are used together
def test_a_run_of_steps_against_64_bits():
    """norm for the log, clip into fp32 buckets, Adam under the clip: eight steps of bf16 parameters with master copies, gradients that change"""
    lengths = [1000, 33, 70001, 1]
    s = adam_state(lengths, BF16, BF16)
    table = ops.AdamTable([s])
    grads = ops.TensorTable(s["grads"])
    bucket = torch.zeros(sum(lengths), device=DEV)
    views = list(bucket.split(lengths))
    into = ops.TensorTable(s["grads"], out=views)
    for step in range(1, 9):
        for i, g in enumerate(s["grads"]):
            g.copy_(rand(lengths[i], BF16, scale=10.0 ** (step % 3 - 1), seed=100 * step + i))
        before = copy_state(s)
        want = exact_norm(s["grads"])
        logged = ops.grad_norm(grads)
        clipped = ops.clip_grads(into, 2.0)
        used = ops.adam_step_tensors(table, lr=1e-3, step=step, weight_decay=0.01, max_norm=2.0)
        check_norm(logged, s["grads"])
        assert float(logged) == float(clipped) == float(used)
        for v, g in zip(views, before["grads"]):
            check_clipped(v, g, coefficient(want, 2.0))
        check_adam(s, before, coefficient(want, 2.0), 1e-3, step, 0.01)


def test_the_same_call_gives_the_same_bits():
    g = [rand(n, BF16, seed=i) for i, n in enumerate([70001, 5, 300000] * 60)]
    first = ops.grad_total(g)
    for _ in range(5):
        assert torch.equal(ops.grad_total(g), first)


def test_on_a_stream_of_its_own_beside_a_busy_one():
    side = torch.cuda.Stream()
    g = [rand(300000, BF16), rand(77)]
    want = exact_norm(g)
    before = [x.clone() for x in g]
    side.wait_stream(torch.cuda.current_stream())
    a = rand(2048 * 2048).view(2048, 2048)
    for _ in range(20):
        a = a @ a * 1e-3
    with torch.cuda.stream(side):
        norm = ops.clip_grads(g, 1.0)
        again = ops.grad_norm(g)
    torch.cuda.current_stream().wait_stream(side)
    check_norm(norm, before)
    for x, b in zip(g, before):
        check_clipped(x, b, coefficient(want, 1.0))
    check_norm(again, g)


def test_two_threads_at_once():
    lists = [[rand(50000, BF16, seed=k), rand(3, seed=k)] for k in range(2)]
    want = [exact_norm(l) for l in lists]
    wrong = []

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            torch.cuda.current_stream().wait_event(ready)
            for _ in range(50):
                if abs(float(ops.grad_norm(lists[k])) - want[k]) > H * want[k] * 1.001:
                    wrong.append(k)

    ready = torch.cuda.Event()
    ready.record()
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


def test_captured_and_replayed():
    """two graphs of the same tables, replayed in turn with eager calls between: every replay against the eager result"""
    lengths = [70001, 5, 1000] * 50
    s = adam_state(lengths, BF16, BF16)
    e = copy_state(s)
    table, eager = ops.AdamTable([s]), ops.AdamTable([e])
    grads, egrads = ops.TensorTable(s["grads"]), ops.TensorTable(e["grads"])
    hyper, decay = torch.zeros(1, 2, device=DEV), torch.zeros(1, device=DEV)
    kw = dict(lr=0.0, step=0, hyper_dev=hyper, decay_dev=decay)
    hyper.copy_(torch.tensor([ops.adam_hyper(1e-3, 1)]))
    scratch = copy_state(s)
    ops.adam_step_tensors([scratch], max_norm=1.0, **kw)                     # warm-up outside the capture
    torch.cuda.synchronize()
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(one):
        norm1 = ops.grad_norm(grads)
        clipped1 = ops.clip_grads(grads, 40.0)
    with torch.cuda.graph(two):
        norm2 = ops.adam_step_tensors(table, max_norm=30.0, **kw)
    for step in range(1, 6):
        for i, n in enumerate(lengths):
            new = rand(n, BF16, seed=1000 * step + i)
            s["grads"][i].copy_(new)
            e["grads"][i].copy_(new)
        hyper.copy_(torch.tensor([ops.adam_hyper(1e-3 / step, step)]))
        decay.fill_(1e-5 * step)
        one.replay()
        want = ops.clip_grads(egrads, 40.0)
        two.replay()
        used = ops.adam_step_tensors(eager, max_norm=30.0, **kw)
        torch.cuda.synchronize()
        assert float(norm1) == float(clipped1) == float(want) and float(norm2) == float(used)
        for k in ("params", "master", "grads", "exp_avg", "exp_avg_sq"):
            assert all(torch.equal(x, y) for x, y in zip(s[k], e[k])), (step, k)


def test_two_graphs_of_one_table_at_the_same_time():
    """each graph has a workspace of its own: replayed on two streams at once, against lists that change in between"""
    g = [rand(n, BF16, seed=n) for n in (3_000_001, 5, 70001)]
    table = ops.TensorTable(g)
    ops.grad_norm(table)
    torch.cuda.synchronize()
    graphs, results, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for kind in (2.0, math.inf):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            results.append([ops.grad_norm(table, norm_type=kind) for _ in range(8)])
    for trial in range(5):
        for i, x in enumerate(g):
            x.copy_(rand(x.numel(), BF16, seed=trial * 10 + i))
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for norms, kind in zip(results, (2.0, math.inf)):
            for n in norms:
                check_norm(n, g, kind)


def test_a_table_is_built_in_front_of_a_capture_a_list_may_be_gathered_inside():
    g = [rand(n, BF16, seed=n) for n in (70001, 3, 500)]
    want = exact_norm(g)
    ops.grad_norm(g)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(_lib.NiwError, match="before the capture"):
            ops.TensorTable(g)
        norm = ops.grad_norm(g)                                              # its image is stored by the graph itself
    for scale in (1.0, 2.0, 1.0):
        for x, y in zip(g, [rand(n, BF16, seed=n) for n in (70001, 3, 500)]):
            x.copy_(y * scale)
        graph.replay()
        junk = torch.full((1 << 20,), float("nan"), device=DEV)
        torch.cuda.synchronize()
        assert abs(float(norm) - scale * want) <= H * scale * want * 1.001
        del junk


def test_a_table_serves_streams_other_than_the_one_it_was_built_on():
    g = [rand(n, F32, seed=n) for n in (300001, 5)]
    want = exact_norm(g)
    torch.cuda.synchronize()
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        table = ops.TensorTable(g)
    with torch.cuda.stream(other):
        norm = ops.grad_norm(table)
        del table                                                            # its memory is not handed out again before `other` has read it
    with torch.cuda.stream(side):
        junk = [torch.zeros(64, device=DEV, dtype=torch.uint8) for _ in range(8)]
    torch.cuda.synchronize()
    assert abs(float(norm) - want) <= H * want * 1.001 and len(junk) == 8


@pytest.mark.parametrize("count", [1, 2, 63, 64, 65, 127, 128, 129, 4095, 4096, 4097, 9000])
def test_lists_of_many_tensors(count):
    """every tensor of the list is found: each has a value of its own"""
    flat = torch.arange(1, count + 1, device=DEV, dtype=F32)
    g = [flat[i:i + 1] for i in range(count)]
    want = math.sqrt(sum((i + 1) ** 2 for i in range(count)))
    norm = ops.clip_grads(g, want / 2)
    assert abs(float(norm) - want) <= H * want * 1.001
    check_clipped(flat, torch.arange(1, count + 1, device=DEV, dtype=F32), coefficient(want, want / 2))


def test_random_lists():
    """lists of random lengths, types and places in one buffer, against 64 bits"""
    r = random.Random(3)
    for trial in range(12):
        flat = {t: rand(400000, t, seed=trial) for t in TYPES}
        at, views = {t: 0 for t in TYPES}, []
        for _ in range(r.randint(1, 300)):
            t = r.choice(TYPES)
            n = min(int(10 ** r.uniform(0, 5)), 400000 - at[t])
            views.append(flat[t][at[t]:at[t] + n])
            at[t] += n + r.choice([0, 0, 1, 3])
            at[t] = min(at[t], 400000)
        before = [v.clone() for v in views]
        norm = ops.clip_grads(views, 1.0)
        check_norm(norm, before)
        c = coefficient(exact_norm(before), 1.0)
        for v, b in zip(views, before):
            check_clipped(v, b, c)


# ------------------------------------------------------------------------------------------ tensors that are not dense
def strided(shape, form, dtype=F32, seed=0):
    """(tensor of random values, the memory it lies in): laid out otherwise than in order"""
    turned, n = tuple(reversed(shape)), math.prod(shape)
    if form == "dense":
        whole = rand(n, dtype, seed=seed).view(shape)
        return whole, whole
    if form == "reversed":                                                                       # the first dimension innermost
        whole = rand(n, dtype, seed=seed).view(turned)
        return whole.permute(*range(len(shape) - 1, -1, -1)), whole
    if form == "columns":
        whole = rand(math.prod(shape[:-1]) * (2 * shape[-1] + 3), dtype, seed=seed).view(*shape[:-1], -1)
        return whole[..., 2:2 + shape[-1]], whole
    assert form == "rows"
    whole = rand(2 * n, dtype, seed=seed).view(2 * shape[0], *shape[1:])
    return whole[::2], whole


FORMS = ["dense", "reversed", "columns", "rows"]
SHAPES = [(7,), (129, 65), (1, 300), (300, 1), (3, 5, 130), (2, 40000)]


@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("dtype", TYPES)
def test_norm_of_strided_and_expanded_tensors(dtype, kind):
    t = [strided(s, f, dtype, seed=i)[0] for i, (s, f) in enumerate((s, f) for s in SHAPES for f in FORMS)]
    t += [rand(65, dtype, seed=99).expand(40, 65), rand(1, dtype, seed=98).view(1, 1).expand(90, 70), rand(33, dtype).view(33, 1).expand(33, 5)]
    check_norm(ops.grad_norm(t, norm_type=kind), t, kind)
    check_norm(ops.grad_norm(ops.TensorTable(t), norm_type=kind), t, kind)


@pytest.mark.parametrize("out_form", [None] + FORMS)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype,out_dtype", [(F32, F32), (BF16, F32), (F16, F16)], ids=str)
def test_clip_of_strided_tensors(form, out_form, dtype, out_dtype):
    pairs = [strided(s, form, dtype, seed=i) for i, s in enumerate(SHAPES)]
    g, before, whole = [p[0] for p in pairs], [p[0].clone() for p in pairs], [p[1].clone() for p in pairs]
    outs = None if out_form is None else [strided(s, out_form, out_dtype, seed=50 + i) for i, s in enumerate(SHAPES)]
    around = pairs if outs is None else outs
    kept = [p[1].clone() for p in around]
    want = exact_norm(before)
    norm = ops.clip_grads(g, want / 3, out=None if outs is None else [o[0] for o in outs])
    check_norm(norm, before)
    for i, (o, memory) in enumerate(around):
        check_clipped(o, before[i], coefficient(want, want / 3))
        o.zero_()                                                            # what lies between the elements is as it was
        view = kept[i].as_strided(o.shape, o.stride(), o.storage_offset() - memory.storage_offset())
        view.zero_()
        assert torch.equal(memory, kept[i])
    assert outs is None or all(torch.equal(p[1], w) for p, w in zip(pairs, whole))


def test_clip_of_shared_elements_is_refused_their_norm_is_not():
    for g in (rand(6).expand(4, 6), rand(40).as_strided((5, 4), (3, 1))):
        check_norm(ops.grad_norm([g]), [g])
        with pytest.raises(_lib.NiwError, match="overlap.*stretches of a list of 1"):
            ops.clip_grads([g], 1.0)
        out = torch.empty(g.shape, device=DEV)
        before = g.clone()
        ops.clip_grads([g], 0.5, out=[out])
        check_clipped(out, before, coefficient(exact_norm([before]), 0.5))
        with pytest.raises(_lib.NiwError, match="overlap"):
            ops.clip_grads([out], 0.5, out=[g])


@pytest.mark.parametrize("pt,gt", [(F32, F32), (BF16, BF16), (F16, F32)], ids=str)
@pytest.mark.parametrize("forms", [("columns", "dense", "dense", "dense", "dense"), ("dense", "reversed", "dense", "dense", "dense"), ("reversed",) * 5,
                                   ("rows", "columns", "reversed", "dense", "columns"), ("dense", "expanded", "dense", "rows", "dense")], ids="-".join)
def test_adam_of_strided_tensors(pt, gt, forms):
    shapes, s = [(129, 65), (3, 5, 70), (2, 20000)], dict(params=[], grads=[], exp_avg=[], exp_avg_sq=[], master=None if pt == F32 else [])
    for i, shape in enumerate(shapes):
        p = strided(shape, forms[0], pt, seed=10 * i)[0]
        s["params"].append(p)
        s["grads"].append(rand(shape[-1], gt, seed=10 * i + 1).expand(shape) if forms[1] == "expanded" else strided(shape, forms[1], gt, seed=10 * i + 1)[0])
        s["exp_avg"].append(strided(shape, forms[2], F32, seed=10 * i + 2)[0])
        s["exp_avg_sq"].append(strided(shape, forms[3], F32, seed=10 * i + 3)[0].square_())
        if pt != F32:
            s["master"].append(strided(shape, forms[4], F32, seed=10 * i + 4)[0].copy_(p))
    before = copy_state(s)
    want = exact_norm(before["grads"])
    norm = ops.adam_step_tensors([s], lr=1e-2, step=4, weight_decay=0.1, max_norm=want / 2)
    check_norm(norm, before["grads"])
    check_adam(s, before, coefficient(want, want / 2), 1e-2, 4, 0.1)


def test_adam_refuses_shared_elements_that_it_writes():
    for key in ("params", "exp_avg", "exp_avg_sq"):
        s = {k: [rand(24, seed=i).view(4, 6).square_()] for i, k in enumerate(("params", "grads", "exp_avg", "exp_avg_sq"))}
        s[key] = [rand(6).expand(4, 6)]
        with pytest.raises(_lib.NiwError, match="overlap"):
            ops.AdamTable([s])
