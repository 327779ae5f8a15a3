"""CPU: what the operators over lists of many tensors (gradient norm, clipping, Adam under the clip) refuse, at the C boundary and in the
Python wrappers.  Nothing is launched: every check runs on the host, in front of the first launch."""
import ctypes
import math

import numpy as np
import pytest
import torch

from neural_invertible_warp_amd import _lib, ops


def err():
    return _lib.load().niw_last_error_string().decode()


def grads(*rows):
    a = (_lib.GradTensor * max(len(rows), 1))()
    for c, (g, o, n, d, od) in zip(a, rows):
        c.grad, c.out, c.n, c.dtype, c.out_dtype = g, o, n, d, od
    return a


def grad_table(rows, for_clip):
    """-> (return code, table); the image goes nowhere near a GPU"""
    lib = _lib.load()
    image, t = ctypes.create_string_buffer(max(lib.niw_table_bytes(len(rows)), 16)), _lib.Table()
    return lib.niw_grad_table(grads(*rows), len(rows), for_clip, image, ctypes.byref(t)), t


@pytest.mark.parametrize("row,what", [
    ((None, None, 4, 0, 0), "null pointer"),
    ((1024, 1024, -1, 0, 0), "n=-1"),
    ((1024, 1024, 1 << 60, 0, 0), "n="),
    ((1024, 1024, 4, 3, 0), "dtype 3"),
    ((1026, 1026, 4, 0, 0), "aligned"),
    ((1025, 1025, 4, 1, 1), "aligned"),
])
def test_c_grad_table_refuses_a_bad_descriptor(row, what):
    for for_clip in (0, 1):
        assert grad_table([row], for_clip)[0] == -1 and what in err()


@pytest.mark.parametrize("rows,what", [
    ([(1024, None, 4, 0, 0)], "null pointer in output"),
    ([(1024, 2048, 4, 0, 7)], "dtype 7"),
    ([(1024, 2050, 4, 0, 0)], "aligned"),
    ([(1024, 1024, 4, 1, 0)], "changes its type"),
])
def test_c_grad_table_for_clipping_refuses_a_bad_output(rows, what):
    assert grad_table(rows, 1)[0] == -1 and what in err()
    assert grad_table(rows, 0)[0] == 0                                        # (the norm does not look at outputs)


@pytest.mark.parametrize("rows,ok", [
    ([(1024, 1024, 4, 0, 0), (1040, 1040, 4, 0, 0)], True),                  # neighbours that touch
    ([(1024, 1024, 4, 0, 0), (1024, 1024, 4, 0, 0)], False),                 # the same tensor twice
    ([(1024, 1024, 4, 0, 0), (1036, 1036, 4, 0, 0)], False),                 # one element shared
    ([(1024, 2048, 4, 0, 0), (1024, 4096, 4, 0, 0)], True),                  # one gradient into two outputs
    ([(1024, 2048, 4, 0, 0), (4096, 2060, 4, 0, 0)], False),                 # outputs that overlap
    ([(1024, 1028, 4, 0, 0)], False),                                        # an output that runs over its own gradient
    ([(1024, 2048, 4, 1, 0), (2056, 8192, 4, 1, 0)], False),                 # an output over another gradient
    ([(1024, 1024, 400, 0, 0), (1100, 4096, 1, 0, 0)], False),               # a gradient inside another that is written
    ([(1024, 1024, 0, 0, 0), (1024, 1024, 0, 0, 0)], True),                  # nothing at the same place
    ([(8192, 8192, 4, 0, 0), (1024, 1024, 4000, 0, 0)], False),              # a long one from before
])
def test_c_overlap_check(rows, ok):
    rc, t = grad_table(rows, 1)
    assert (rc == 0) == ok and (ok or "overlap" in err())
    assert grad_table(rows, 0)[0] == 0                                        # the norm may read whatever it likes


def test_c_table_counts_what_it_holds():
    rc, t = grad_table([(1024, 1024, 4, 0, 0), (None, None, 0, 0, 0), (1 << 20, 1 << 20, 100000, 1, 1)], 1)
    assert rc == 0 and t.slots == 2 and t.image is None and t.bytes % 16 == 0 and t.chunks == 1 + -(-100000 // t.chunk)
    assert t.bytes <= _lib.load().niw_table_bytes(3)
    rc, t = grad_table([(1 << 40, 1 << 40, 1 << 33, 0, 0)], 1)
    assert rc == 0 and t.chunks == (1 << 33) // t.chunk
    assert grad_table([], 1)[1].slots == 0


def test_c_lists_whose_launch_could_not_be_counted_are_refused():
    """a launch has less than 2^32 threads: 2^24 workgroups of 256, one per 1024 elements of an update and per 2048 (or 4096) of a clip"""
    far = 1 << 60
    assert grad_table([(1024, 2048, 1 << 44, 0, 0)] * 3, 0)[0] == -1 and "chunks" in err()
    assert grad_table([(1024, 1024, (1 << 35) - (1 << 15), 0, 0)], 1)[0] == 0
    assert grad_table([(1024, 1024, 1 << 35, 0, 0)], 1)[0] == -1 and "chunks" in err()
    assert grad_table([(1024, 1024, 1 << 35, 0, 0)], 0)[0] == 0
    big = dict(param=far, grad=2 * far, exp_avg=3 * far, exp_avg_sq=4 * far)
    assert adam_table(n=(1 << 34) - (1 << 14), **big)[0] == 0
    assert adam_table(n=1 << 34, **big)[0] == -1 and "chunks" in err()


@pytest.mark.parametrize("lengths", [[1], [4096], [4097], [530052, 530052, 165900, 2304], [5] * 3000, [100000] * 100, [1 << 20] * 5, [1 << 20] * 16, [3, 7]])
@pytest.mark.parametrize("offset", [0, 2, 126])
def test_c_kept_tables_cut_small_lists_into_pieces(lengths, offset):
    """the image of a kept table holds every element of every tensor once, in order, and fits the size that was asked for"""
    lib = _lib.load()
    rows, at = [], (1 << 30) + offset
    for n in lengths:
        rows.append((at, at, n, 1, 1))
        at += 2 * n + 64
    image, t = ctypes.create_string_buffer(lib.niw_table_bytes(len(rows))), _lib.Table()
    assert lib.niw_grad_table(grads(*rows), len(rows), 3, image, ctypes.byref(t)) == 0
    assert t.bytes <= len(image) and t.slots >= len(rows)
    slots = [(int.from_bytes(image.raw[32 * i:32 * i + 8], "little"), int.from_bytes(image.raw[32 * i + 16:32 * i + 24], "little"),
              int.from_bytes(image.raw[32 * i + 24:32 * i + 28], "little")) for i in range(t.slots)]
    k, chunks = 0, 0
    for begin, _, n, _, _ in rows:
        here = begin
        while here < begin + 2 * n:
            assert slots[k][0] == here and slots[k][2] == chunks
            here += 2 * slots[k][1]
            chunks += -(-slots[k][1] // t.chunk)
            k += 1
        assert here == begin + 2 * n
    assert k == t.slots and chunks == t.chunks
    first = [int.from_bytes(image.raw[32 * t.slots + 4 * i:32 * t.slots + 4 * i + 4], "little") for i in range(t.slots)]
    assert first == [s[2] for s in slots]


def test_c_calls_refuse_bad_arguments():
    lib = _lib.load()
    t = grad_table([(1024, 1024, 4, 0, 0)], 1)[1]
    t.image = 4096
    norm_only = grad_table([(1024, 1024, 4, 0, 0)], 0)[1]
    norm_only.image = 4096
    R = ctypes.byref
    assert lib.niw_grad_table(None, 1, 0, 4096, R(_lib.Table())) == -1 and "1 tensors" in err()
    assert lib.niw_grad_table(None, -1, 0, 4096, R(_lib.Table())) == -1 and "-1 tensors" in err()
    assert lib.niw_grad_table(grads((1024, 1024, 4, 0, 0)), 1, 0, None, R(_lib.Table())) == -1 and "null pointer" in err()
    assert lib.niw_grad_table(grads((1024, 1024, 4, 0, 0)), 1, 4, 4096, R(_lib.Table())) == -1 and "flags 4" in err()
    assert lib.niw_adam_table(adam_row(), 1, 1, 1, 4096, R(_lib.Table())) == -1 and "flags 1" in err()
    assert lib.niw_table_bytes(-1) == 0
    assert lib.niw_table_store(None, 16, 4096, None) == -1 and "null" in err()
    assert lib.niw_table_store(4096, 16, 4097, None) == -1 and "misaligned" in err()
    assert lib.niw_table_store(4096, 15, 4096, None) == -1 and "15 bytes" in err()
    assert lib.niw_grad_norm(None, 0, 4096, 4096, None, None) == -1 and "null pointer" in err()
    assert lib.niw_grad_norm(R(t), 2, 4096, 4096, None, None) == -1 and "kind 2" in err()
    assert lib.niw_grad_norm(R(t), 0, None, 4096, None, None) == -1 and "null pointer" in err()
    assert lib.niw_grad_norm(R(t), 0, 4096, None, None, None) == -1 and "null pointer" in err()
    for bad in (-1.0, math.nan, -math.inf):
        assert lib.niw_grad_clip(R(t), 0, bad, None, 4096, None, None) == -1 and "max_norm" in err()
    assert lib.niw_grad_clip(R(t), 5, 1.0, None, 4096, None, None) == -1 and "kind 5" in err()
    assert lib.niw_grad_clip(R(t), 0, 1.0, None, None, None, None) == -1 and "null pointer" in err()
    assert lib.niw_grad_clip(R(norm_only), 0, 1.0, None, 4096, None, None) == -1 and "form 1" in err()
    t.image = None
    assert lib.niw_grad_norm(R(t), 0, 4096, 4096, None, None) == -1 and "not stored" in err()
    t.image = 4100
    assert lib.niw_grad_norm(R(t), 0, 4096, 4096, None, None) == -1 and "not stored" in err()
    h = (_lib.AdamHyper * 1)(_lib.AdamHyper(lr=1e-3, step=1))
    assert lib.niw_adam_step_tensors(R(norm_only), h, 0.9, 0.999, 1e-8, None, None, None, None) == -1 and "form 1" in err()


def adam_row(**kw):
    r = _lib.AdamTensor(param=1024, grad=2048, exp_avg=4096, exp_avg_sq=8192, master=None, n=4, param_dtype=0, grad_dtype=0, group=0)
    for k, v in kw.items():
        setattr(r, k, v)
    return (_lib.AdamTensor * 1)(r)


def adam_table(n_groups=1, **kw):
    lib = _lib.load()
    image, t = ctypes.create_string_buffer(lib.niw_table_bytes(1)), _lib.Table()
    return lib.niw_adam_table(adam_row(**kw), 1, n_groups, 0, image, ctypes.byref(t)), t


@pytest.mark.parametrize("change,what", [
    (dict(param=None), "null pointer"), (dict(grad=None), "null pointer"), (dict(exp_avg=None), "null pointer"), (dict(exp_avg_sq=None), "null pointer"),
    (dict(n=-4), "n=-4"), (dict(param_dtype=5, master=16384), "dtype 5"), (dict(grad_dtype=-1), "dtype 0 / -1"), (dict(group=1), "group 1 of 1"),
    (dict(group=-1), "group -1"), (dict(master=16384), "master copy"), (dict(param_dtype=1), "master copy"), (dict(exp_avg=4098), "aligned"),
    (dict(param_dtype=1, master=16385), "aligned"), (dict(n_groups=0), "1..8 groups"), (dict(n_groups=9), "1..8 groups"),
    (dict(exp_avg=1024), "overlap"), (dict(exp_avg_sq=4100), "overlap"), (dict(grad=1024), "overlap"), (dict(param_dtype=1, master=1028), "overlap"),
])
def test_c_adam_table_refuses(change, what):
    assert adam_table(**change)[0] == -1 and what in err()


def test_c_adam_refuses_bad_arguments():
    lib = _lib.load()
    rc, t = adam_table()
    t.image = 4096
    assert rc == 0
    step = lambda h, b1=0.9, b2=0.999, eps=1e-8, hd=None, dd=None, clip=None: lib.niw_adam_step_tensors(ctypes.byref(t), h, b1, b2, eps, hd, dd, clip, None)
    H = lambda **kw: (_lib.AdamHyper * 1)(_lib.AdamHyper(**{**dict(lr=1e-3, weight_decay=0.0, step=1), **kw}))
    assert step(None) == -1 and "null pointer" in err()
    assert step(H(step=0)) == -1 and "step=0" in err()
    assert step(H(lr=math.nan)) == -1 and "lr=" in err()
    assert step(H(weight_decay=-0.1)) == -1 and "weight_decay" in err()
    assert step(H(weight_decay=0.1), hd=64) == -1 and "decay_dev" in err()
    for kw in (dict(b1=1.0), dict(b2=1.0), dict(b1=-0.1), dict(eps=-1e-8), dict(b2=math.nan)):
        assert step(H(), **kw) == -1 and "beta1" in err()
    clip = lambda **kw: ctypes.byref(_lib.AdamClip(**{**dict(max_norm=1.0, kind=0, workspace=4096), **kw}))
    assert step(H(), clip=clip(max_norm=-1.0)) == -1 and "max_norm" in err()
    assert step(H(), clip=clip(kind=9)) == -1 and "kind 9" in err()
    assert step(H(), clip=clip(workspace=None)) == -1 and "null pointer" in err()


# ------------------------------------------------------------------------------------------ Python wrappers (CPU tensors: refused last)
def z(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("tensors,out,what", [
    ([z(4, dtype=torch.float64)], None, "float64"),
    ([z(4, dtype=torch.int32)], None, "int32"),
    ([3.0], None, "float"),
    ([z(600000)[::2]], None, "300000 stretches of 1 elements"),
    ([z(600, 500).t()], [z(500, 600)], "300000 stretches of 1 elements"),
    ([z(4).to_sparse()], None, "sparse"),
    ([z(4)], [], "1 tensors and 0 outputs"),
    ([z(4), z(4)], [z(4), None], "some tensors only"),
    ([z(4)], [z(5)], "agree in shape"),
    ([z(4, 6)], [z(4, 6).t()], "agree in shape"),
    ([z(8)[::2]], [z(2, 2)], "agree in shape"),
    ([z(4)], [z(4, dtype=torch.int64)], "int64"),
    ([torch._neg_view(z(4))], None, "negated"),
    ([z(4)], None, "expected CUDA/HIP"),
    ([z(0)], None, "expected CUDA/HIP"),
])
def test_tensor_table_refuses(tensors, out, what):
    with pytest.raises(_lib.NiwError, match=what):
        ops.TensorTable(tensors, out=out)


def test_rows_of_a_list_have_the_layout_of_the_descriptors():
    """the columns the wrappers fill are the fields of include/niw.h"""
    for row, struct in ((ops._GRAD_ROW, _lib.GradTensor), (ops._ADAM_ROW, _lib.AdamTensor)):
        assert row.itemsize == ctypes.sizeof(struct)
        assert [(n, row.fields[n][1]) for n in row.names] == [(n, getattr(struct, n).offset) for n, _ in struct._fields_]


def strided(shape, form, dtype=torch.float32):
    """a tensor of that shape, laid out otherwise than in order"""
    n = len(shape)
    if form == "dense":
        return torch.empty(shape, dtype=dtype)
    if form == "reversed":                                                                       # the first dimension innermost
        return torch.empty(shape[::-1], dtype=dtype).permute(*range(n - 1, -1, -1))
    if form == "columns":
        return torch.empty((*shape[:-1], 2 * shape[-1] + 3), dtype=dtype)[..., 2:2 + shape[-1]]
    if form == "rows":
        return torch.empty((2 * shape[0], *shape[1:]), dtype=dtype)[::2]
    assert form == "expanded"
    return torch.empty((1, *shape[1:]), dtype=dtype).expand(shape)


FORMS = ["dense", "reversed", "columns", "rows", "expanded"]


def addresses(t):
    """of every element, in the order of its index"""
    at = np.zeros(t.shape, np.int64)
    for d, n in enumerate(t.shape):
        at += (np.arange(n) * t.stride(d)).reshape([-1 if k == d else 1 for k in range(t.dim())])
    return (t.data_ptr() + at * t.element_size()).reshape(-1)


@pytest.mark.parametrize("second", FORMS)
@pytest.mark.parametrize("first", FORMS)
@pytest.mark.parametrize("shape", [(1,), (7,), (5, 6), (1, 6), (5, 1), (3, 4, 5), (2, 1, 3, 4), (0, 4), (4, 0)])
def test_stretches_pair_the_elements_that_belong_together(shape, first, second):
    """over all stretches, the pairs of addresses walked are those of the elements of equal index, each once"""
    a, b = strided(shape, first), strided(shape, second, torch.bfloat16)
    length, (at, to) = ops._runs([a, b], "pair")
    walked = [(int(x) + 4 * j, int(y) + 2 * j) for x, y in zip(at, to) for j in range(length)]
    assert sorted(walked) == sorted(zip(addresses(a).tolist(), addresses(b).tolist()))


@pytest.mark.parametrize("form,length,count", [("dense", 120, 1), ("reversed", 120, 1), ("columns", 6, 20), ("rows", 30, 4), ("expanded", 30, 4)])
def test_stretches_are_as_long_as_the_layout_allows(form, length, count):
    got, (at,) = ops._runs([strided((4, 5, 6), form)], "tensor")
    assert (got, len(at)) == (length, count)


def test_rows_of_a_mixed_list():
    """entries in step keep one row, the others have one per stretch, in the entries' order"""
    t = [z(5), z(3, 8)[:, 2:6], z(0), z(4, 6).t(), z(0, 4)[:, 1:3], z(6)]
    out = [z(5), z(3, 4), z(0), z(4, 6).t(), z(0, 2), z(2, 3)]
    cols = dict(grad=[x.data_ptr() for x in t], out=[x.data_ptr() for x in out], n=[x.numel() for x in t], dtype=0, out_dtype=0)
    rows = ops._rows(ops._GRAD_ROW, cols, ("grad", "out"), False, (t, out), "tensor")
    assert [int(n) for n in rows["n"] if n] == [5, 4, 4, 4, 24, 6]
    full = rows[rows["n"] > 0]
    assert full["grad"].tolist() == [t[0].data_ptr()] + [t[1].data_ptr() + 32 * k for k in range(3)] + [t[3].data_ptr(), t[5].data_ptr()]
    assert full["out"].tolist() == [out[0].data_ptr()] + [out[1].data_ptr() + 16 * k for k in range(3)] + [out[3].data_ptr(), out[5].data_ptr()]


@pytest.mark.parametrize("tensors,overlap", [
    (lambda: [z(1, 4).expand(3, 4)], True), (lambda: [z(12).as_strided((3, 4), (2, 1))], True), (lambda: [z(4, 6)[:, :3]], False),
    (lambda: (lambda x: [x[:, :3], x[:, 3:]])(z(4, 6)), False), (lambda: (lambda x: [x[:, :4], x[:, 3:]])(z(4, 6)), True),
    (lambda: (lambda x: [x[::2], x[1::2]])(z(9)), False), (lambda: [z(6, 4).t()], False),
])
def test_written_stretches_that_overlap_are_refused(tensors, overlap):
    """what has a norm need not be clippable in place: elements that several indices share would be scaled several times"""
    t = tensors()
    cols = dict(grad=[x.data_ptr() for x in t], out=[x.data_ptr() for x in t], n=[x.numel() for x in t], dtype=0, out_dtype=0)
    rows = ops._rows(ops._GRAD_ROW, cols, ("grad", "out"), False, (t, t), "tensor")
    lib, table = _lib.load(), _lib.Table()
    image = np.zeros(lib.niw_table_bytes(len(rows)), np.uint8)
    for flags, refused in ((0, False), (ops.TABLE_CLIP, overlap)):
        code = lib.niw_grad_table(rows.ctypes.data, len(rows), flags, image.ctypes.data, ctypes.byref(table))
        assert code == (-1 if refused else 0)
        assert not refused or "overlap" in err()


def test_none_entries_are_left_out_before_any_check():
    with pytest.raises(_lib.NiwError, match="expected CUDA/HIP"):
        ops.TensorTable([None, z(4)], out=[None, z(4)])


@pytest.mark.parametrize("call,what", [
    (lambda t: ops.grad_norm(t, norm_type=1), "norm_type"),
    (lambda t: ops.grad_norm(t, norm_type=-math.inf), "norm_type"),
    (lambda t: ops.clip_grads(t, -1.0), "max_norm"),
    (lambda t: ops.clip_grads(t, math.nan), "max_norm"),
    (lambda t: ops.clip_grads(t, 1.0, total=z(1)), "grad_total"),
    (lambda t: ops.clip_grads(t, 1.0, out=[]), "when it is built"),
])
def test_wrappers_refuse(call, what):
    with pytest.raises(_lib.NiwError, match=what):
        call(ops.TensorTable([]))


def group(**kw):
    g = dict(params=[z(4)], grads=[z(4)], exp_avg=[z(4)], exp_avg_sq=[z(4)])
    g.update(kw)
    return g


@pytest.mark.parametrize("groups,what", [
    ([], "1..8 groups"), ([group()] * 9, "1..8 groups"),
    ([group(lr=[1.0])], "unknown keys"), ([group(grads=None)], "needs params"), ([group(grads=[])], "differ in length"),
    ([group(exp_avg=[z(4, dtype=torch.bfloat16)])], "expected float32"), ([group(params=[z(4, dtype=torch.bfloat16)])], "master copy"),
    ([group(master=[z(4)])], "has none"), ([group(grads=[z(5)])], "agree in shape"),
    ([group(params=[z(2, 3)], grads=[z(3, 2)], exp_avg=[z(2, 3)], exp_avg_sq=[z(2, 3).t()])], "agree in shape"),
    ([group(params=[z(4, dtype=torch.bfloat16)], master=[z(5)])], "agree in shape"),
    ([group(grads=[z(8)[::2]], exp_avg=[z(5)])], "agree in shape"), ([group()], "expected CUDA/HIP"), ([group(grads=[z(4, dtype=torch.float64)])], "float64"),
])
def test_adam_table_refuses(groups, what):
    with pytest.raises(_lib.NiwError, match=what):
        ops.AdamTable(groups)


@pytest.mark.parametrize("kw,what", [
    (dict(lr=[1e-3, 1e-3]), "lr: 2 values for 1 groups"), (dict(step=[]), "step: 0 values"), (dict(weight_decay=[0.1] * 3), "weight_decay: 3"),
    (dict(skip_nonfinite=True), "go with max_norm"), (dict(total=z(1, dtype=torch.float64)), "go with max_norm"), (dict(max_norm=-2.0), "max_norm"),
    (dict(max_norm=1.0, norm_type=3), "norm_type"), (dict(hyper_dev=z(2)), "float32 CUDA"), (dict(max_norm=1.0, total=z(1)), "grad_total"),
])
def test_adam_step_tensors_refuses(kw, what):
    empty = ops.AdamTable([dict(params=[], grads=[], exp_avg=[], exp_avg_sq=[])])
    with pytest.raises(_lib.NiwError, match=what):
        ops.adam_step_tensors(empty, **{**dict(lr=1e-3, step=1), **kw})


@pytest.mark.parametrize("optim,what", [
    (dict(clip_norm=-1.0), "from 0 on"), (dict(clip_norm=float("nan")), "from 0 on"), (dict(clip_norm=True), "from 0 on"), (dict(clip_norm="much"), "from 0 on"), (dict(clip_norm=[1]), "from 0 on"),
    (dict(skip_nonfinite=True), "goes with optim.clip_norm"),
])
def test_trainer_options_are_checked(optim, what):
    from neural_invertible_warp_amd import engine
    with pytest.raises(_lib.NiwError, match=what):
        engine.ClippedAdam(optim)


def test_trainer_without_the_option_has_no_clip():
    from neural_invertible_warp_amd import engine
    assert engine.ClippedAdam({}).max_norm is None and engine.ClippedAdam(dict(clip_norm=0)).max_norm == 0.0
    assert engine.clip_options(dict(clip_norm="1e-3", skip_nonfinite=True)) == (1e-3, True)      # as the command line's yaml reads it


def test_torch_optimizers_refuse_to_leave_a_step_out():
    from neural_invertible_warp_amd.model import nerf
    from neural_invertible_warp_amd.util import edict
    m = nerf.Model.__new__(nerf.Model)
    with pytest.raises(_lib.NiwError, match="does not"):
        m.setup_optimizer(edict(optim=edict(algo="AdamW", lr=1e-3, clip_norm=1.0, skip_nonfinite=True)))
