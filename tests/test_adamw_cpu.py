"""remixfusion_amd.optim.AdamW and clip_grad_norm_ without a GPU: CPU parameters take torch's own step, what has no CPU path is
refused, and the C entry points check their arguments before anything is launched."""
import copy
import ctypes as C
import math

import pytest
import torch

from remixfusion_amd import _lib as L


@pytest.fixture(scope="module", autouse=True)
def built():
    from remixfusion_amd.build import build_host, build_library
    build_library()
    build_host()


def _pair(**kw):
    from remixfusion_amd.optim import AdamW
    p = torch.nn.Parameter(torch.linspace(-1, 1, 12).reshape(3, 4).clone())
    q = torch.nn.Parameter(p.detach().clone())
    return p, q, AdamW([p], lr=0.05, betas=(0.9, 0.99), weight_decay=0.1, **kw), torch.optim.AdamW([q], lr=0.05, betas=(0.9, 0.99), weight_decay=0.1)


def test_cpu_parameters_take_torchs_step_and_hooks_fire_once():
    p, q, ours, ref = _pair()
    pre, post = [], []
    g = torch.Generator().manual_seed(3)
    for it in range(4):
        grad = torch.randn(p.shape, generator=g)
        p.grad, q.grad = grad.clone(), grad.clone()
        if it == 1:
            h0 = ours.register_step_pre_hook(lambda *a: pre.append(it))
            h1 = ours.register_step_post_hook(lambda *a: post.append(it))
        if it == 3:
            h0.remove(); h1.remove()
        ours.step(); ref.step()
        assert torch.equal(p.detach(), q.detach())
    assert pre == [1, 2] and post == [1, 2]
    third = torch.optim.AdamW([torch.nn.Parameter(torch.zeros(3, 4))])
    third.load_state_dict(ours.state_dict())
    assert float(third.state[third.param_groups[0]["params"][0]]["step"]) == 4.0


def test_copies_and_state_dicts_keep_what_is_ours():
    p, q, ours, ref = _pair(state_bits=8, master_weights=True, seed=7, max_grad_norm=0.5)
    twin = copy.deepcopy(ours)
    assert twin.max_grad_norm == 0.5 and twin.param_groups[0]["state_bits"] == 8 and twin.param_groups[0]["seed"] == 7
    ours.add_param_group({"params": [torch.nn.Parameter(torch.zeros(2))], "state_bits": 32})
    assert [g["state_bits"] for g in ours.param_groups] == [8, 32]
    assert ours.state_dict()["param_groups"][1]["master_weights"] is True
    ours.load_state_dict({"state": {}, "param_groups": [{"params": [0], "lr": 0.5, "betas": (0.8, 0.9), "eps": 1e-8, "weight_decay": 0.0},
                                                        {"params": [1], "lr": 0.5, "betas": (0.8, 0.9), "eps": 1e-8, "weight_decay": 0.0}]})
    assert [g["state_bits"] for g in ours.param_groups] == [8, 32] and ours.param_groups[0]["lr"] == 0.5     # what a foreign dict lacks stays
    avg, avg_sq = ours.moments()
    assert len(avg) == 2 and avg[0].shape == (3, 4) and float(avg_sq[1].abs().sum()) == 0.0                  # no state yet: zeros


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_a_device_runs_state_steps_on_the_cpu(dtype):
    """moments in fp32, as a device holds them whatever the parameter's type"""
    from remixfusion_amd.optim import AdamW
    p, q = (torch.nn.Parameter(torch.linspace(-1, 1, 12).to(dtype)) for _ in range(2))
    ours, ref = AdamW([p], lr=0.05), torch.optim.AdamW([q], lr=0.05)
    state = {"step": torch.tensor(3.0), "exp_avg": torch.full((12,), 0.3), "exp_avg_sq": torch.full((12,), 0.7)}
    for o in (ours, ref):
        o.load_state_dict({"state": {0: copy.deepcopy(state)}, "param_groups": ref.state_dict()["param_groups"]})
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    ours.step(); ref.step()
    assert torch.equal(p.detach(), q.detach()) and float(ours.state[p]["step"]) == 4.0


def test_what_has_no_cpu_path_is_refused():
    for kw in ({"state_bits": 8}, {"master_weights": True}, {"max_grad_norm": 1.0}):
        p, q, ours, ref = _pair(**kw)
        p.grad = torch.ones_like(p)
        before = p.detach().clone()
        with pytest.raises(L.RfxError):
            ours.step()
        assert torch.equal(p.detach(), before)


def test_constructor_refusals():
    from remixfusion_amd.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(3))
    for kw in ({"amsgrad": True}, {"differentiable": True}, {"state_bits": 16}, {"max_grad_norm": -1.0}, {"max_grad_norm": math.nan},
               {"seed": -1}, {"seed": 1 << 32}, {"lr": torch.tensor(0.1)}, {"lr": -1.0}, {"betas": (1.0, 0.9)}):
        with pytest.raises(ValueError):
            AdamW([p], **kw)
    with pytest.raises(ValueError), pytest.warns(UserWarning):                          # the same parameter twice in a group
        AdamW([p, p])
    opt = AdamW([p])
    with pytest.raises(ValueError):
        opt.max_grad_norm = -0.5
    opt.max_grad_norm = 2
    assert opt.max_grad_norm == 2.0


def test_clip_on_the_cpu_is_torchs():
    from remixfusion_amd.optim import clip_grad_norm_
    p, q = torch.nn.Parameter(torch.zeros(5)), torch.nn.Parameter(torch.zeros(5))
    p.grad, q.grad = torch.arange(5.0), torch.arange(5.0)
    assert torch.equal(clip_grad_norm_([p], 1.0), torch.nn.utils.clip_grad_norm_([q], 1.0)) and torch.equal(p.grad, q.grad)
    assert float(clip_grad_norm_([torch.nn.Parameter(torch.zeros(2))], 1.0)) == 0.0     # no gradient at all
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError):
            clip_grad_norm_([p], bad)


# ---- the C boundary: every refusal comes before a launch, so none of this needs a device -------------------------------------
A = 1 << 20                                                                             # stands for device memory: never read


def _tensor(**kw):
    t = L.AdamwTensor(A, A + 4096, A + 8192, A + 12288, A + 16384, None, None, 8, 0, 0, 0, 0)
    for k, v in kw.items():
        setattr(t, k, v)
    return t


def _group(**kw):
    g = L.AdamwGroup(0.1, 0.9, 0.99, 1e-8, 0.0, None, 1, 0, 32, 0, 0)
    for k, v in kw.items():
        setattr(g, k, v)
    return g


def _call(t, g, count=1, groups=1, ws=None, ws_bytes=0, clip=None, limit=0.0):
    arr = (L.AdamwTensor * 1)(t) if t is not None else None
    garr = (L.AdamwGroup * 1)(g) if g is not None else None
    return L.load().rfx_adamw_step(C.addressof(arr) if arr else None, count, C.addressof(garr) if garr else None, groups,
                                 C.addressof(clip) if clip else None, limit, None, ws, ws_bytes, None)


def test_struct_layouts_match_the_library():
    lib = L.load()
    assert lib.rfx_adamw_tensor_bytes() == C.sizeof(L.AdamwTensor) == 80
    assert lib.rfx_adamw_group_bytes() == C.sizeof(L.AdamwGroup) == 72
    assert C.sizeof(L.MomentTensor) == 48 and C.sizeof(L.GradTensor) == 24


@pytest.mark.parametrize("t", [dict(param=None), dict(grad=None), dict(exp_avg=None), dict(exp_avg_sq=None), dict(n=-1), dict(group=1),
                               dict(group=-1), dict(dtype=3), dict(dtype=-1), dict(master=A), dict(param=A + 2), dict(grad=A + 1),
                               dict(exp_avg=A + 2), dict(dtype=1, param=A + 1), dict(dtype=1, master=A + 2)])
def test_adamw_step_refuses_bad_tensors(t):
    assert _call(_tensor(**t), _group()) == -1


@pytest.mark.parametrize("g", [dict(state_bits=16), dict(beta1=1.0), dict(beta2=-0.1), dict(beta1=math.nan), dict(eps=-1.0), dict(step=0),
                               dict(lr_dev=A)])
def test_adamw_step_refuses_bad_groups(g):
    assert _call(_tensor(), _group(**g)) == -1


def test_adamw_step_refusals_and_empty_calls():
    assert _call(_tensor(exponents=None), _group(state_bits=8)) == -1
    assert _call(_tensor(exp_avg=A + 1), _group(state_bits=8)) == -1
    assert _call(None, None, 0, 0) == 0 and _call(None, _group()) == -1 and _call(_tensor(), None) == -1
    assert _call(_tensor(), _group(), -1) == -1 and _call(_tensor(), _group(), 1, 0) == -1
    assert _call(_tensor(n=0, param=None), _group()) == 0                               # no elements: nothing to launch
    assert _call(_tensor(n=1 << 52), _group()) == -3 and _call(_tensor(n=(1 << 63) - 1), _group()) == -1
    assert _call(_tensor(n=(1 << 34) + (1 << 20)), _group()) == -3                     # more blocks than a launch counts threads for
    lib = L.load()
    assert lib.rfx_adamw_workspace_bytes(0) == 0 and lib.rfx_adamw_workspace_bytes(-3) == 0 and lib.rfx_adamw_workspace_bytes(3) >= 48
    grads = (L.GradTensor * 1)(L.GradTensor(A + 4096, 8, 0, 0))
    for ws, n in ((None, 0), (A, 15), (A + 8, 1 << 16)):                                # a count on the device, or a norm, needs the workspace
        assert _call(_tensor(step_dev=A), _group(), ws=ws, ws_bytes=n) == -4
        assert _call(_tensor(), _group(), ws=ws, ws_bytes=n, clip=grads, limit=1.0) == -4
    for limit in (-1.0, math.nan):
        assert _call(_tensor(), _group(), ws=A, ws_bytes=1 << 16, clip=grads, limit=limit) == -1
    grads[0].dtype = 7
    assert _call(_tensor(), _group(), ws=A, ws_bytes=1 << 16, clip=grads, limit=1.0) == -1


def test_norm_scale_and_moments_refusals():
    lib = L.load()

    def grads(**kw):
        t = L.GradTensor(A, 8, 0, 0)
        for k, v in kw.items():
            setattr(t, k, v)
        return (L.GradTensor * 1)(t)

    def norm(t, count=1, kind=2, limit=1.0, clip=A, ws=A, ws_bytes=1 << 16):
        return lib.rfx_grad_norm(C.addressof(t) if t else None, count, kind, limit, clip, None, ws, ws_bytes, None)

    for kw in (dict(grad=None), dict(n=-1), dict(dtype=3), dict(grad=A + 2), dict(dtype=2, grad=A + 1)):
        assert norm(grads(**kw)) == -1 and lib.rfx_grad_scale(C.addressof(grads(**kw)), 1, A, None) == -1
        assert lib.rfx_grad_clip(C.addressof(grads(**kw)), 1, 2, 1.0, None, A, 1 << 16, None) == -1
    ok = grads()
    assert norm(None) == -1 and norm(ok, -1) == -1 and norm(ok, clip=None) == -1 and norm(ok, clip=A + 4) == -1
    assert norm(ok, limit=-1.0) == -1 and norm(ok, limit=math.nan) == -1 and norm(ok, kind=1) == -3
    assert norm(ok, ws=None) == -4 and norm(ok, ws_bytes=7) == -4 and norm(ok, ws=A + 4) == -4
    assert lib.rfx_grad_clip(C.addressof(ok), 1, 2, 1.0, None, A, 7, None) == -4 and lib.rfx_grad_clip(C.addressof(ok), 1, 3, 1.0, None, A, 1 << 16, None) == -3
    assert lib.rfx_grad_norm_workspace_bytes(-1) == 0 and lib.rfx_grad_norm_workspace_bytes(1) >= 2048
    assert lib.rfx_grad_scale(C.addressof(ok), 1, None, None) == -1 and lib.rfx_grad_scale(C.addressof(ok), 1, A + 4, None) == -1 and lib.rfx_grad_scale(None, 0, A, None) == 0
    m = L.MomentTensor(A, A, A, A, A, 8)
    for k in ("exp_avg", "exp_avg_sq", "exponents", "out_avg", "out_avg_sq"):
        bad = (L.MomentTensor * 1)(m)
        setattr(bad[0], k, None)
        assert lib.rfx_adamw_moments(C.addressof(bad), 1, None) == -1
    bad = (L.MomentTensor * 1)(m)
    bad[0].exp_avg = A + 1
    assert lib.rfx_adamw_moments(C.addressof(bad), 1, None) == -1
    assert lib.rfx_adamw_moments(None, 0, None) == 0 and lib.rfx_adamw_moments(None, 1, None) == -1
