"""optim.clip_norm through the trainers, the models and the command line: the global gradient norm over all trained groups, clipping by it
inside the Adam launch (engine.ClippedAdam over ops.adam_step_tensors), in place on the torch.optim path (ops.clip_grads)."""
import math

import pytest
import torch

from tests.test_gpu_fused_step import _trainer
from tests.test_gpu_optim import H, check_adam, check_norm, coefficient

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def clipped(cfg, clip_norm, fused=True, **kw):
    """the fused-step tests' trainer with a clip: the option is read when the trainer is built"""
    from neural_invertible_warp_amd import engine
    tr, var = _trainer(cfg, fused, **kw)
    tr.opt.optim.clip_norm = clip_norm
    tr.clip = engine.ClippedAdam(tr.opt.optim)
    return tr, var


def iterations(tr, var, steps):
    return [{k: float(v.detach()) for k, v in tr.train_iteration(type(var)(var)).items()} for _ in range(steps)]


@pytest.mark.parametrize("cfg", ["cfg3_barf_inn_llff", "cfg2_nerf_inn_llff_hier", "dtu"])
def test_a_clip_that_never_bites_changes_no_bit(cfg):
    a, va = _trainer(cfg, True)
    b, vb = clipped(cfg, math.inf)
    c, vc = clipped(cfg, 1e9)
    la, lb, lc = (iterations(t, v, 5) for t, v in ((a, va), (b, vb), (c, vc)))
    assert la == lb == lc
    assert a.grad_norm is None
    for other in (b, c):
        assert all(torch.equal(x, y) for x, y in zip(a._flats() + a.m + a.v, other._flats() + other.m + other.v))
        check_norm(other.grad_norm, [other.bucket.flat])


@pytest.mark.parametrize("cfg", ["cfg2_nerf_inn_llff_hier", "dtu"])
def test_a_clip_that_bites_against_64_bits(cfg):
    tr, var = clipped(cfg, 1e-3)
    for it in range(3):
        before = [f.clone() for f in tr._flats()], [x.clone() for x in tr.m], [x.clone() for x in tr.v]
        tr.train_iteration(type(var)(var))
        check_norm(tr.grad_norm, [tr.bucket.flat])
        c = coefficient(float(tr.bucket.flat.double().norm()), 1e-3)
        assert c < 0.5
        for i, flat in enumerate(tr._flats()):
            g = [tr.bucket.segment(i)]
            check_adam(dict(params=[flat], grads=g, exp_avg=[tr.m[i]], exp_avg_sq=[tr.v[i]], master=None),
                       dict(params=[before[0][i]], grads=g, exp_avg=[before[1][i]], exp_avg_sq=[before[2][i]], master=None), c, tr.learning_rate(i, it), it + 1, 0.0)


def test_the_mirror_and_the_one_call_iteration_clip_alike():
    a, va = clipped("cfg2_nerf_inn_llff_hier", 1e-3, fused=False)
    b, vb = clipped("cfg2_nerf_inn_llff_hier", 1e-3)
    for _ in range(4):
        a.train_iteration(type(va)(va))
        b.train_iteration(type(vb)(vb))
        assert float(a.grad_norm) == float(b.grad_norm)
    assert all(torch.equal(x, y) for x, y in zip(a._flats(), b._flats()))


@pytest.mark.parametrize("cfg", ["cfg3_barf_inn_llff", "dtu"])
def test_captured_iterations_clip_like_launched_ones(cfg):
    a, va = clipped(cfg, 1e-3)
    b, vb = clipped(cfg, 1e-3, hip_graph=True)
    for it in range(8):
        la, lb = a.train_iteration(type(va)(va)), b.train_iteration(type(vb)(vb), replay=it != 5)
        torch.cuda.synchronize()
        assert {k: float(v.detach()) for k, v in la.items()} == {k: float(v.detach()) for k, v in lb.items()}
        assert float(a.grad_norm) == float(b.grad_norm), it
        junk = torch.full((1 << 18,), float("nan"), device=DEV)              # the program's own work between two replays
        del junk
    assert b._captured is not None
    assert all(torch.equal(x, y) for x, y in zip(a._flats() + a.m + a.v, b._flats() + b.m + b.v))


def test_a_group_that_is_not_trained_is_neither_counted_nor_moved():
    tr, var = clipped("cfg3_barf_inn_llff", 1e-3)
    tr.trainable[-1] = False
    latent = tr._flats()[-1].clone()
    tr.train_iteration(type(var)(var))
    check_norm(tr.grad_norm, [tr.bucket.segment(i) for i in range(len(tr.bucket.groups) - 1)])
    assert torch.equal(tr._flats()[-1], latent)


def test_skip_nonfinite_leaves_a_step_out():
    from neural_invertible_warp_amd import engine
    tr, var = clipped("cfg3_barf_inn_llff", 1.0)
    tr.opt.optim.skip_nonfinite = True
    tr.clip = engine.ClippedAdam(tr.opt.optim)
    tr.train_iteration(type(var)(var))
    before = [f.clone() for f in tr._flats() + tr.m + tr.v]
    tr._forward_backward(type(var)(var), tr.it)
    tr.bucket.flat[12345] = math.inf
    tr._optimizer_step(tr.it)
    assert float(tr.grad_norm) == math.inf
    assert all(torch.equal(x, y) for x, y in zip(tr._flats() + tr.m + tr.v, before))
    tr.train_iteration(type(var)(var))
    assert math.isfinite(float(tr.grad_norm)) and not torch.equal(tr._flats()[0], before[0])


def test_the_table_follows_buffers_that_move():
    tr, var = clipped("cfg3_barf_inn_llff", 1e-3)
    ref, vr = clipped("cfg3_barf_inn_llff", 1e-3)
    for it in range(4):
        if it == 2:
            tr.m = [x.clone() for x in tr.m]
        tr.train_iteration(type(var)(var))
        ref.train_iteration(type(vr)(vr))
    assert all(torch.equal(x, y) for x, y in zip(tr._flats() + tr.m + tr.v, ref._flats() + ref.m + ref.v))


def test_vanilla_trainer_clips():
    from neural_invertible_warp_amd import configs, engine

    def make(clip_norm):
        opt = configs.cfg1_nerf_llff_repr(device=DEV)
        opt.nerf.rand_rays, opt.nerf.sample_intvs, opt.nerf.sample_intvs_fine, opt.max_iter = 4 * 40, 16, 16, 40
        opt.optim.clip_norm = clip_norm
        return engine.NeRFTrainer(opt, 4, seed=2), engine.synthetic_scene(opt, 4)
    (a, va), (b, vb), (c, vc) = make(None), make(1e6), make(1e-3)
    la, lb = iterations(a, va, 4), iterations(b, vb, 4)
    assert la == lb and all(torch.equal(x, y) for x, y in zip(a._flats(), b._flats())) and a.grad_norm is None
    check_norm(b.grad_norm, [b.bucket.flat])
    before = [f.clone() for f in c._flats()], [x.clone() for x in c.m], [x.clone() for x in c.v]
    c.train_iteration(type(vc)(vc))
    factor = coefficient(float(c.bucket.flat.double().norm()), 1e-3)
    assert factor < 1
    for i, flat in enumerate(c._flats()):
        g = [c.bucket.segment(i)]
        check_adam(dict(params=[flat], grads=g, exp_avg=[c.m[i]], exp_avg_sq=[c.v[i]], master=None),
                   dict(params=[before[0][i]], grads=g, exp_avg=[before[1][i]], exp_avg_sq=[before[2][i]], master=None), factor, c.lr0, 1, 0.0)


COMMON = ["--data.image_size=[24,32]", "--freq.val=100", "--freq.ckpt=100", "--freq.scalar=1", "--max_iter=3"]


def norms_of(text):
    return [float(w.split("=")[1]) for w in text.split() if w.startswith("grad_norm=")]


def test_command_line_trains_under_a_clip(tmp_path, capsys):
    from neural_invertible_warp_amd import train
    args = ["--model=barf_inn_llff", "--yaml=barf_inn_llff", "--barf_c2f=[0.1,0.5]", "--loss_weight.global_alignment=2", "--data.dataset=synthetic",
            "--nerf.rand_rays=288", "--nerf.sample_intvs=32", f"--output_root={tmp_path}"] + COMMON
    plain = train.main(args + ["--name=a"])
    assert not norms_of(capsys.readouterr().out)
    free = train.main(args + ["--name=b", "--optim.clip_norm=.inf"])
    assert len(norms_of(capsys.readouterr().out)) == 3
    assert all(torch.equal(x, y) for x, y in zip(plain.trainer._flats(), free.trainer._flats()))
    tight = train.main(args + ["--name=c", "--optim.clip_norm=1e-3", "--optim.skip_nonfinite"])
    assert len(norms_of(capsys.readouterr().out)) == 3 and tight.trainer.clip.max_norm == 1e-3 and tight.trainer.clip.skip_nonfinite


@pytest.mark.parametrize("args", [
    ["--model=nerf", "--yaml=nerf_llff_repr", "--data.dataset=synthetic", "--nerf.rand_rays=288", "--nerf.sample_intvs=16", "--nerf.sample_intvs_fine=16"],
    ["--model=barf_inn_dtu", "--yaml=barf_inn_dtu", "--barf_c2f=[0.1,0.5]", "--loss_weight.global_alignment=3", "--data.dataset=dtu", "--data.synthetic_fallback",
     "--nerf.rand_rays=192", "--nerf.sample_intvs=32", "--data.train_sub=3", "--optim.test_iter=3"],
], ids=["nerf", "dtu"])
def test_torch_optimizers_see_clipped_gradients(args, tmp_path, capsys):
    """another optim.algo than Adam: torch.optim steps by .grad, which the clip has scaled in place"""
    from neural_invertible_warp_amd import train
    m = train.main(args + COMMON + ["--optim.algo=AdamW", "--optim.clip_norm=1e-3", f"--output_root={tmp_path}", "--name=t"])
    assert m.trainer is None
    norms = norms_of(capsys.readouterr().out)
    assert len(norms) == 3 and all(n > 1e-3 for n in norms)
    optimizers = [m.optim] + ([m.optim_pose] if hasattr(m, "optim_pose") else [])
    left = math.sqrt(sum(float(p.grad.double().square().sum()) for o in optimizers for g in o.param_groups for p in g["params"] if p.grad is not None))
    # every gradient is off by half a step of the factor, of the product and of its own rounding at most: so is their norm
    want = 1e-3 * float(m.grad_norm) / (float(m.grad_norm) + 1e-6)
    assert abs(left - want) <= 4 * H * want


def test_two_ranks_clip_by_the_norm_of_the_exchanged_gradients(tmp_path):
    """two gloo ranks on this GPU, each with its share of the rays: both log the same norms -- that of the summed gradients -- and stay equal"""
    import os
    import re
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    args = ["--model=barf_inn_llff", "--yaml=barf_inn_llff", "--barf_c2f=[0.1,0.5]", "--loss_weight.global_alignment=2", "--data.dataset=synthetic",
            "--data.image_size=[24,32]", "--nerf.rand_rays=288", "--nerf.sample_intvs=32", "--freq.val=2", "--freq.ckpt=100", "--freq.scalar=1",
            "--optim.clip_norm=1e-3", "--optim.skip_nonfinite", f"--output_root={tmp_path}", "--name=clip", "--max_iter=4"]
    procs = []
    for rank in range(2):
        env = dict(os.environ, MASTER_ADDR="127.0.0.1", MASTER_PORT="29677", RANK=str(rank), WORLD_SIZE="2", LOCAL_RANK="0", NIW_DIST_BACKEND="gloo")
        procs.append(subprocess.Popen([sys.executable, "-m", "neural_invertible_warp_amd.train"] + args, cwd=root, env=env, stdout=subprocess.PIPE,
                                      stderr=subprocess.PIPE, text=True))
    try:
        outs = [p.communicate(timeout=100) for p in procs]
    finally:
        for p in procs:
            if p.poll() is None:
                p.kill()
    for p, (out, err) in zip(procs, outs):
        assert p.returncode == 0, err[-2000:]
    val = [[l for l in out.splitlines() if l.startswith("[val it 4]")] for out, _ in outs]
    assert val[0] and val[0] == val[1], val
    norms = [re.findall(r"grad_norm=(\S+)", out) for out, _ in outs]
    assert len(norms[0]) >= 3 and norms[0] == norms[1]
    assert all(math.isfinite(float(n)) and float(n) > 1e-3 for n in norms[0])
