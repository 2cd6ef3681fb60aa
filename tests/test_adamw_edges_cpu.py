"""remixfusion_amd.optim.AdamW and clip_grad_norm_ without a GPU: groups and states that come from outside, what a plan holds on to."""
import copy
import gc
import weakref

import pytest
import torch

from remixfusion_amd import _lib as L


@pytest.fixture(scope="module", autouse=True)
def built():
    from remixfusion_amd.build import build_host, build_library
    build_library()
    build_host()


def _param():
    p = torch.nn.Parameter(torch.linspace(-1, 1, 12))
    p.grad = torch.ones(12)
    return p


@pytest.mark.parametrize("group", [{"amsgrad": True}, {"differentiable": True}, {"state_bits": 16}, {"seed": -1}, {"seed": 1 << 32}, {"seed": 0.5}])
def test_groups_that_are_refused_however_they_come(group):
    """as a group that joins, as a loaded one, as one that was changed in place: nothing of the optimizer moves"""
    from remixfusion_amd.optim import AdamW
    p = _param()
    opt = AdamW([p], lr=0.05)
    opt.step()
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [_param()], **group})
    assert len(opt.param_groups) == 1
    saved = copy.deepcopy(opt.state_dict())
    saved["param_groups"][0].update(group, lr=7.0)
    moments = opt.state[p]["exp_avg"]
    with pytest.raises(ValueError):
        opt.load_state_dict(saved)
    assert opt.param_groups[0]["lr"] == 0.05 and opt.state[p]["exp_avg"] is moments
    assert all(opt.param_groups[0].get(k) != v for k, v in group.items())
    opt.param_groups[0].update(group)
    before = p.detach().clone()
    with pytest.raises((ValueError, L.RfxError)):
        opt.step()
    assert torch.equal(p.detach(), before) and float(opt.state[p]["step"]) == 1.0


def test_a_run_with_amsgrad_is_not_resumed_without_it():
    from remixfusion_amd.optim import AdamW
    p, q = _param(), _param()
    theirs = torch.optim.AdamW([q], amsgrad=True)
    theirs.step()
    opt = AdamW([p])
    with pytest.raises(ValueError):
        opt.load_state_dict(theirs.state_dict())
    assert not opt.state and opt.param_groups[0]["amsgrad"] is False
    for kind in (torch.optim.AdamW, torch.optim.Adam):          # as torch's AdamW takes them: the decay stays apart from the gradient
        opt.load_state_dict(kind([_param()]).state_dict())
        assert opt.param_groups[0]["decoupled_weight_decay"] is True
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [_param()], "decoupled_weight_decay": False})
    opt.param_groups[0]["decoupled_weight_decay"] = False
    with pytest.raises(ValueError):
        opt.step()


def test_clip_takes_torchs_arguments():
    from remixfusion_amd.optim import clip_grad_norm_
    for kw in ({"foreach": None}, {"foreach": False}, {"foreach": True}, {"error_if_nonfinite": True, "foreach": False, "norm_type": 3.0}):
        p, q = _param(), _param()
        assert torch.equal(clip_grad_norm_([p], 0.5, **kw), torch.nn.utils.clip_grad_norm_([q], 0.5, **kw)) and torch.equal(p.grad, q.grad)


def test_a_plan_keeps_no_state_alive():
    """an optimizer's state that is cleared is freed, and no other tensor at its address is taken for it"""
    p = _param()
    state = {p: {"step": torch.zeros(()), "exp_avg": torch.zeros(12), "exp_avg_sq": torch.zeros(12), "name": "p"}}
    groups = [dict(params=[p], state_bits=32, master_weights=False, capturable=False, seed=0)]
    plan = L.host().Plan([(p, 0, 0)], groups, state)
    seen = [weakref.ref(state[p][k]) for k in ("step", "exp_avg", "exp_avg_sq")]
    state.clear()
    gc.collect()
    assert all(r() is None for r in seen)
    state[p] = {"step": torch.zeros(()), "exp_avg": torch.zeros(12), "exp_avg_sq": torch.zeros(12), "name": "p"}
    assert plan.step(groups, state, -1.0, 0) == L.host().STALE
    state.clear()
    assert plan.step(groups, state, -1.0, 0) == L.host().STALE
    state[p] = None
    assert plan.step(groups, state, -1.0, 0) == L.host().STALE


def test_eight_bit_moments_on_the_cpu_say_what_they_need():
    """a device run's state loaded without one: it can be kept and saved, its values are read on a device"""
    from remixfusion_amd.optim import AdamW
    p = _param()
    opt = AdamW([p], state_bits=8)
    codes = torch.arange(12, dtype=torch.uint8)
    opt.load_state_dict({"state": {0: {"step": torch.tensor(3.0), "exp_avg": codes, "exp_avg_sq": codes.clone(),
                                       "exponents": torch.zeros(2, 1, dtype=torch.int8)}}, "param_groups": opt.state_dict()["param_groups"]})
    assert torch.equal(opt.state_dict()["state"][0]["exp_avg"], codes)
    with pytest.raises(L.RfxError, match="device"):
        opt.moments()
