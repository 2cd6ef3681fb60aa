"""the mapper with mapping.optimizer adamw / adamw8bit and mapping.grad_clip: the optimizers that SLAM builds, what they hold, and one map
iteration's step against torch.optim.AdamW and the clipping formula in 64 bits."""
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


def _pipeline(**mapping):
    from remixfusion_amd.config import synthetic_config
    from remixfusion_amd.pipeline import MappingPipeline
    cfg = synthetic_config("office0")
    cfg["cam"].update({"H": 120, "W": 160, "fx": 144.0, "fy": 144.0, "cx": 79.5, "cy": 59.5})
    cfg["volume"].update({"voxel_size": 0.04, "trunc": 0.15})
    cfg["mapping"].update({"first_iters": 5, "sample": 512, **mapping})
    return MappingPipeline(cfg, n_frames=20)


def _run(pipe, n=12):               # the mapper fires at frames 6 and 11
    frames = pipe.prefetch(list(range(n)))
    pipe.start(frames[0])
    for i in range(1, n):
        pipe.step(i, frames[i])
    torch.cuda.synchronize()
    return frames


@pytest.mark.parametrize("kind", ["adamw", "adamw8bit"])
@pytest.mark.parametrize("clip", [None, 0.5])
def test_the_mapper_runs_with_it(kind, clip):
    from remixfusion_amd.optim import AdamW
    pipe = _pipeline(optimizer=kind, grad_clip=clip)
    before = [p.detach().clone() for p in pipe.model.parameters() if p.requires_grad and p.numel()]
    _run(pipe)
    assert int(pipe.slam.mapping_idx[0]) == 10
    for opt in (pipe.slam.map_optimizer, pipe.slam.rba_optimizer):
        assert type(opt) is AdamW and opt.max_grad_norm == clip
        assert (opt.grad_norm is None) == (clip is None)
        if clip is not None:
            assert bool(torch.isfinite(opt.grad_norm)) and float(opt.grad_norm) > 0
    table = pipe.model.embed_res_fn.params
    st = pipe.slam.map_optimizer.state[table]
    assert st["exp_avg"].dtype == (torch.uint8 if kind == "adamw8bit" else torch.float32) and float(st["step"]) == 5 + 2 * 5
    for w in pipe.model.decoder_res.parameters():
        assert pipe.slam.map_optimizer.state[w]["exp_avg"].dtype == torch.float32
    assert all(g["weight_decay"] in (0.0, 1e-6) for g in pipe.slam.map_optimizer.param_groups)
    after = [p.detach() for p in pipe.model.parameters() if p.requires_grad and p.numel()]
    assert all(bool(torch.isfinite(a).all()) and not torch.equal(a, b) for a, b in zip(after, before))


@pytest.mark.parametrize("kind", ["adamw", "adamw8bit"])
def test_one_map_iteration_is_the_formula(kind):
    """gradients of one iteration, then the step: parameters against AdamW in fp64 from the same moments"""
    pipe = _pipeline(optimizer=kind, grad_clip=0.5)
    _run(pipe, 7)
    opt, d = pipe.slam.map_optimizer, pipe.mapper._direct_iterations()
    batch = pipe.dataset[6]
    rays = torch.cat([batch["direction"], batch["rgb"], batch["depth"][..., None]], -1).reshape(-1, 7).to(pipe.device)
    poses = pipe.slam.est_c2w_data[0:7:pipe.config["mapping"]["keyframe_every"]].clone()
    d.map_gradients(rays, poses)
    params = [p for g in opt.param_groups for p in g["params"]]
    grads = [p.grad.double() for p in params]
    avg, avg_sq = opt.moments()
    old = [(p.detach().double(), m.double(), v.double()) for p, m, v in zip(params, avg, avg_sq)]
    norm = torch.sqrt(sum((g * g).sum() for g in grads))
    opt.step()
    c = min(1.0, 0.5 / (float(norm) + 1e-6))
    assert abs(float(opt.grad_norm) - float(norm)) <= 1e-6 * float(norm)
    i = 0
    for g in opt.param_groups:
        for p in g["params"]:
            k = float(opt.state[p]["step"])
            x, m, v = old[i]
            m, v = 0.9 * m + 0.1 * grads[i] * c, 0.99 * v + 0.01 * (grads[i] * c) ** 2
            up = g["lr"] / (1 - 0.9 ** k) * m / ((v / (1 - 0.99 ** k)).sqrt() + g["eps"])
            want = x - g["lr"] * g["weight_decay"] * x - up
            # u = 2^-24: the parameter's own rounding, 16 u of the update, and m's terms of opposite sign (4 u of each) over the root of v
            spread = g["lr"] / (1 - 0.9 ** k) * (0.9 * old[i][1].abs() + 0.1 * grads[i].abs() * c) / ((v / (1 - 0.99 ** k)).sqrt() + g["eps"])
            tol = 2.0 ** -24 * (2 * x.abs() + want.abs() + 16 * up.abs() + 4 * spread) + 2.0 ** -126
            # (roots of second moments under 2^-126, gradients under 1e-19, are not resolved: they count as 2^-126)
            tiny = v < 2.0 ** -120
            assert bool(((p.detach().double() - want).abs() <= tol)[~tiny].all()), (kind, tuple(p.shape))
            assert bool(((p.detach().double() - x).abs()[tiny] <= 2 * g["lr"] + tol[tiny]).all())
            i += 1


def test_the_autograd_formulation_runs_with_it():
    pipe = _pipeline(optimizer="adamw8bit", grad_clip=0.5, direct_iterations=False)
    _run(pipe)
    assert int(pipe.slam.mapping_idx[0]) == 10 and pipe.mapper._direct_iterations() is None
    assert float(pipe.slam.map_optimizer.state[pipe.model.embed_res_fn.params]["step"]) == 5 + 2 * 5
    assert all(bool(torch.isfinite(p).all()) for p in pipe.model.parameters() if p.requires_grad)


def test_what_the_configuration_refuses():
    with pytest.raises(ValueError):
        _pipeline(optimizer="sgd")
    with pytest.raises(ValueError):
        _pipeline(grad_clip=1.0)


def _rank(rank, world, port, out_dir):
    import torch.distributed as dist
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    torch.cuda.set_device(0)
    from remixfusion_amd import _lib as L
    from remixfusion_amd.dist import ShardedPipeline
    from test_dist_gpu import _small_cfg
    cfg = _small_cfg("center", "auto")
    cfg["mapping"].update(optimizer="adamw8bit", grad_clip=0.5)
    pipe = ShardedPipeline(cfg, dist, rank, world, n_frames=20, seed=5)
    frames = pipe.prefetch(list(range(8)))
    pipe.start(frames[0])
    for i in range(1, 8):
        pipe.step(i, frames[i])
    out = {"mode": type(pipe.mapper._direct).__name__, "table": pipe.model.embed_res_fn.params.detach().cpu()}
    st = pipe.slam.map_optimizer.state[pipe.model.embed_res_fn.params]
    out.update({k: v.cpu() for k, v in st.items()})
    # a rank whose state went astray gets rank 0's back: codes and the exponents that belong to them
    if rank == 1:
        st["exponents"].fill_(3)
        st["exp_avg"].fill_(9)
    pipe.sync_replicas()
    out.update({"again_" + k: v.cpu() for k, v in st.items()})
    pipe.mapper._direct, pipe.mapper.config["mapping"]["shard_field"] = None, "levels"
    try:
        pipe.mapper._direct_iterations()
        out["levels"] = "taken"
    except L.RfxError as e:
        out["levels"] = str(e)
    torch.save(out, os.path.join(out_dir, f"r{rank}.pt"))
    dist.barrier()
    dist.destroy_process_group()


def test_two_ranks_keep_identical_states(tmp_path):
    """one scene on two ranks (gloo, both on this GPU): replicated table, all-reduced gradients, the same 8-bit step on every rank"""
    import torch.multiprocessing as mp
    from test_dist_gpu import _free_port
    mp.spawn(_rank, args=(2, _free_port(), str(tmp_path)), nprocs=2, join=True)
    a, b = (torch.load(tmp_path / f"r{r}.pt") for r in range(2))
    assert a["mode"] == b["mode"] == "ShardedIterations" and a["levels"] == b["levels"] != "taken"
    assert a["exp_avg"].dtype == torch.uint8 and float(a["step"]) == 6 + 5
    for k in ("table", "exp_avg", "exp_avg_sq", "exponents", "step"):
        assert torch.equal(a[k], b[k]), k
    for k in ("exp_avg", "exp_avg_sq", "exponents"):
        assert torch.equal(a["again_" + k], a[k]) and torch.equal(b["again_" + k], a[k]), k
