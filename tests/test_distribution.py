"""Distributions over classes without a GPU: the float64 oracle against autograd, differences and closed
forms; refusals of the Python entry points and of the C ABI (nothing is launched)."""
import math

import pytest
import torch
import torch.nn.functional as F

from depth_estimation_amd import _lib
from oracle import distribution as ref

INF = float("inf")


def _rows(n, V, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(n, V, generator=g, dtype=torch.float64) * spread, g


# --------------------------------------------------------------------------- the oracle itself

@pytest.mark.parametrize("scale", [1.0, -1.0, 0.5])
def test_oracle_log_probs_is_log_softmax_and_its_gradient_is_autograds(scale):
    x, g = _rows(7, 19)
    idx = torch.tensor([0, 18, 5, -1, 19, 3, 3])
    gl, gh = torch.randn(7, generator=g, dtype=torch.float64), torch.randn(7, generator=g, dtype=torch.float64)
    out = ref.log_probs(x, idx, scale, top=4)
    xr = x.clone().requires_grad_(True)
    logp = F.log_softmax(xr * scale, -1)
    lp = torch.where((idx >= 0) & (idx < 19), logp.gather(-1, idx.clamp(0, 18)[:, None])[:, 0], 0.0)
    ent = torch.distributions.Categorical(logits=xr * scale).entropy()
    assert torch.allclose(out["log_prob"], lp) and torch.allclose(out["entropy"], ent)
    top = logp.detach().topk(4, -1)
    assert torch.equal(out["top_index"].long(), top.indices) and torch.allclose(out["top_log_prob"], top.values)
    want, = torch.autograd.grad([lp, ent], [xr], [gl, gh])
    assert torch.allclose(ref.log_probs_grad(x, idx, scale, gl, gh), want, atol=1e-12)


@pytest.mark.parametrize("renormalise", [False, True])
@pytest.mark.parametrize("scale", [1.0, -0.7])
def test_oracle_distill_gradient_against_differences(scale, renormalise):
    x, g = _rows(5, 11, seed=3)
    idx = torch.tensor([[0, 4, 7], [10, 10, 2], [3, -1, 5], [-1, -1, 11], [6, 1, 0]])   # twice, padding, none
    val = F.log_softmax(torch.randn(5, 4, generator=g, dtype=torch.float64), -1)[:, :3]
    out = ref.distill(x, val, idx, scale, renormalise)
    eps = 1e-5
    for j in range(11):
        d = torch.zeros(5, 11, dtype=torch.float64)
        d[:, j] = eps
        num = (ref.distill(x + d, val, idx, scale, renormalise)["loss"]
               - ref.distill(x - d, val, idx, scale, renormalise)["loss"]) / (2 * eps)
        assert torch.allclose(out["grad"][:, j], num, atol=1e-8), j
    assert out["loss"][3] == 0 and (out["grad"][3] == 0).all()


def test_oracle_distill_of_a_full_list_is_the_divergence_and_vanishes_for_equal_distributions():
    x, g = _rows(4, 6, seed=5)
    t = torch.randn(4, 6, generator=g, dtype=torch.float64)
    idx = torch.arange(6).expand(4, 6)
    out = ref.distill(x, F.log_softmax(t, -1), idx)
    want = F.kl_div(F.log_softmax(x, -1), F.log_softmax(t, -1), log_target=True, reduction="none").sum(-1)
    assert torch.allclose(out["loss"], want)
    same = ref.distill(x, F.log_softmax(x, -1)[:, :3], idx[:, :3])
    assert same["loss"].abs().max() < 1e-12 and same["grad"].abs().max() < 1e-12


def test_oracle_masked_and_empty_rows():
    x, _ = _rows(3, 5, seed=1)
    x[0] = -INF
    x[1, 1:] = -INF
    idx = torch.tensor([2, 0, 4])
    out = ref.log_probs(x, idx, 1.0, top=5)
    assert out["log_prob"][0] == -INF and out["entropy"][0] == 0 and out["top_index"][0].tolist() == [0, 1, 2, 3, 4]
    assert out["log_prob"][1] == 0 and out["entropy"][1] == 0
    one = torch.ones(3, dtype=torch.float64)
    g = ref.log_probs_grad(x, idx, 1.0, one, one)
    assert g.isfinite().all() and (g[0] == 0).all()
    lowest = torch.full((1, 8), torch.finfo(torch.float32).min)
    assert abs(float(ref.log_probs(lowest, torch.tensor([3]))["entropy"]) - math.log(8)) < 1e-12


# ----------------------------------------------------------------------------------- refusals

def _desc(outer=2, classes=8, inner=1, scale=1.0, dtype=0, entries=2, flags=0):
    import ctypes
    return ctypes.byref(_lib.DwDistDesc(outer, classes, inner, (2, 1, 1), scale, dtype, entries, flags))


BAD = [(dict(classes=0), -2), (dict(classes=(1 << 28) + 1), -2), (dict(outer=-1), -2), (dict(inner=-1), -2),
       (dict(entries=-1), -2), (dict(entries=65), -2), (dict(dtype=3), -5), (dict(dtype=-1), -5), (dict(flags=64), -5),
       (dict(scale=0.0), -5), (dict(scale=INF), -5), (dict(scale=float("nan")), -5),
       (dict(outer=1 << 41), -2), (dict(outer=1 << 39, inner=1 << 39), -2), (dict(outer=1 << 30, classes=1 << 27), -2),
       # more threads than a launch can have
       (dict(outer=1 << 24, classes=5000), -2), (dict(outer=1 << 26, classes=2100), -2), (dict(outer=1 << 38, classes=8), -2),
       (dict(outer=1 << 26, inner=64, classes=1), -2)]


@pytest.mark.parametrize("kw,code", BAD)
def test_abi_refuses_bad_problems_before_touching_a_pointer(kw, code):
    lib = _lib.lib()
    d = _desc(**kw)
    assert lib.dw_log_probs_workspace_bytes(d) == code
    assert lib.dw_log_probs_fwd(d, None, None, None, None, None, None, None, None, 0, None) == code
    assert lib.dw_log_probs_bwd(d, None, None, None, None, None, None, None) == code
    assert lib.dw_distill_workspace_bytes(d) == code
    assert lib.dw_distill_fwd(d, None, None, None, None, None, None, 0, None) == code
    assert lib.dw_distill_bwd(d, None, None, None, None, None, None, None) == code


@pytest.mark.parametrize("scale", [3e38, -3e38, 2.0 ** 121, 2.0 ** -121, -1e-37, 1e-45])
def test_abi_refuses_scales_whose_exponents_leave_float32(scale):
    # (3e38 log2 e is infinite: every row's maximum would give 0 * inf)
    test_abi_refuses_bad_problems_before_touching_a_pointer(dict(scale=scale), -5)
    lib = _lib.lib()
    for ok in (2.0 ** 120, -(2.0 ** -120)):
        assert lib.dw_log_probs_workspace_bytes(_desc(scale=ok)) == 0 == lib.dw_distill_workspace_bytes(_desc(scale=ok))


def test_abi_refuses_null_pointers_small_workspaces_and_misfit_lists():
    lib = _lib.lib()
    x = 256   # stands for a device pointer: nothing is launched
    assert lib.dw_log_probs_workspace_bytes(None) == -1 and lib.dw_distill_workspace_bytes(None) == -1
    d = _desc()
    assert lib.dw_log_probs_fwd(d, None, x, x, x, x, x, x, None, 0, None) == -1
    assert lib.dw_log_probs_fwd(d, x, None, x, x, x, x, x, None, 0, None) == -1      # log_prob without an index
    assert lib.dw_log_probs_fwd(d, x, x, x, x, None, x, x, None, 0, None) == -1      # entries without their outputs
    assert lib.dw_log_probs_bwd(d, x, x, None, x, x, x, None) == -1
    assert lib.dw_log_probs_bwd(d, x, None, x, x, None, x, None) == -1               # its gradient without an index
    assert lib.dw_log_probs_bwd(d, x, x, x, x, x, None, None) == -1
    assert lib.dw_distill_fwd(d, x, x, None, x, x, None, 0, None) == -1
    assert lib.dw_distill_bwd(d, x, x, x, None, x, x, None) == -1
    assert lib.dw_log_probs_workspace_bytes(_desc(classes=1, entries=2)) == -2       # more top classes than classes
    assert lib.dw_log_probs_workspace_bytes(_desc(flags=4)) == -5                    # a flag of the other operator
    assert lib.dw_distill_workspace_bytes(_desc(entries=0)) == -2
    assert lib.dw_distill_workspace_bytes(_desc(flags=8 | 16)) == -5
    one_long_row = _desc(outer=1, classes=1 << 20, entries=4)
    n = lib.dw_log_probs_workspace_bytes(one_long_row)
    assert n > 0 and n % 256 == 0
    assert lib.dw_log_probs_fwd(one_long_row, x, x, x, x, x, x, x, None, n, None) == -1
    assert lib.dw_log_probs_fwd(one_long_row, x, x, x, x, x, x, x, x, n - 1, None) == -3
    assert lib.dw_log_probs_fwd(one_long_row, x, x, x, x, x, x, x, x + 8, n, None) == -3
    assert lib.dw_distill_workspace_bytes(one_long_row) > 0
    assert lib.dw_distill_fwd(one_long_row, x, x, x, x, x, x, 0, None) == -3
    # nothing to do: no pointer is needed
    assert lib.dw_log_probs_fwd(_desc(outer=0), None, None, None, None, None, None, None, None, 0, None) == 0
    assert lib.dw_distill_bwd(_desc(inner=0), None, None, None, None, None, None, None) == 0


def test_header_and_binding_agree():
    import os
    import re
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = open(os.path.join(root, "include", "depthwarp.h")).read()
    for name, value in re.findall(r"#define\s+(DW_(?:DIST|DTYPE)_\w+)\s+(\d+)", text):
        assert getattr(_lib, name) == int(value)
    import ctypes
    assert ctypes.sizeof(_lib.DwDistDesc) == 64


def test_python_refuses_cpu_tensors():
    from depth_estimation_amd.distribution import distill_loss, log_probs
    with pytest.raises(_lib.DepthwarpError):
        log_probs(torch.zeros(2, 4), torch.zeros(2, dtype=torch.long))
    with pytest.raises(_lib.DepthwarpError):
        distill_loss(torch.zeros(2, 4), torch.zeros(2, 2), torch.zeros(2, 2, dtype=torch.long))


# ------------------------------------------------------------- the documented use, as it is written

def documented_loss():
    """`distribution_loss` of the integration guide's example, over whatever `depth_estimation_amd.distribution` offers now."""
    import os
    import re
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = open(os.path.join(root, "INTEGRATION.md")).read()
    block, = [b for b in re.findall(r"```python\n(.*?)```", text, re.S) if "distill_loss" in b]
    names = {"torch": torch}
    exec(block, names)
    return names["distribution_loss"]


def check_documented_loss(device):
    loss_of = documented_loss()
    g = torch.Generator().manual_seed(0)
    cost = torch.randn(1, 16, 4, 5, generator=g) * 2
    gt = torch.randint(1, 16, (1, 4, 5), generator=g).float()
    gt[0, 1] = 0.0          # no ground truth
    gt[0, 2] = 40.0         # beyond the range
    nothing = torch.full((1, 3, 4, 5), -1)
    t = torch.full((1, 3, 4, 5), -2.0)

    def run(cost, gt, t=t, ti=nothing):
        c = cost.to(device).requires_grad_(True)
        loss = loss_of(c, gt.to(device), t.to(device), ti.to(device))
        grad, = torch.autograd.grad(loss, c)
        return float(loss.detach()), grad.cpu()

    loss, grad = run(cost, gt)
    logp = F.log_softmax(-cost.double(), 1)
    at = gt.long().clamp(0, 15)[:, None]
    want = -logp.gather(1, at)[:, 0][:, [0, 3]].mean()
    assert abs(loss - float(want)) < 1e-5
    # to lower the loss, the true bin's cost falls and the others' rise; where nothing is known, nothing changes
    hit = torch.zeros_like(cost).scatter_(1, at, 1.0).bool()
    known = torch.tensor([True, False, False, True])[None, None, :, None].expand_as(cost)
    assert (grad[hit & known] > 0).all() and (grad[~hit & known] < 0).all() and (grad[~known] == 0).all()
    # a pixel whose log-probability is 0 counts in the mean
    sure = cost.clone()
    sure[0, :, 0] = torch.where(hit[0, :, 0], -200.0, 200.0)
    want = -F.log_softmax(-sure.double(), 1).gather(1, at)[:, 0][:, [0, 3]].mean()
    assert abs(run(sure, gt)[0] - float(want)) < 1e-5
    # a crop without ground truth
    loss, grad = run(cost, torch.zeros_like(gt))
    assert loss == 0 and (grad == 0).all()
    # the teacher's bins become likelier
    ti = nothing.clone()
    ti[0, 0] = 7
    loss, grad = run(cost, torch.zeros_like(gt), torch.full_like(t, -0.01), ti)
    assert loss > 0 and (grad[0, 7] > 0).all()


def test_the_documented_loss_makes_the_true_bin_cheaper(monkeypatch):
    from depth_estimation_amd import distribution

    def log_probs(x, index, scale=1.0):
        logp = F.log_softmax(x * scale, 1)
        given = (index >= 0) & (index < x.shape[1])
        at = logp.gather(1, index.clamp(0, x.shape[1] - 1)[:, None])[:, 0]
        return distribution.LogProbs(torch.where(given, at, 0.0), -(logp.exp() * logp).sum(1), None, None)

    def distill_loss(x, t, ti, scale=1.0):
        last = [v.movedim(1, -1) for v in (x, t, ti)]
        return ref.distill(*last, scale)["loss"].float()

    monkeypatch.setattr(distribution, "log_probs", log_probs)
    monkeypatch.setattr(distribution, "distill_loss", distill_loss)
    check_documented_loss("cpu")


# ------------------------------------------------------------------------------------ tracing

def _fake_problem(mode, dtype=torch.float32):
    with mode:
        x = torch.empty(2, 20, 4, 6, device="cuda:0", dtype=dtype)
        idx = torch.empty(2, 4, 6, device="cuda:0", dtype=torch.long)
        t = torch.empty(2, 5, 4, 6, device="cuda:0")
        ti = torch.empty(2, 5, 4, 6, device="cuda:0", dtype=torch.int32)
    return x, idx, t, ti


def test_calls_on_tensors_without_data_give_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from depth_estimation_amd.distribution import distill_loss, log_probs
    mode = FakeTensorMode()
    x, idx, t, ti = _fake_problem(mode, torch.bfloat16)

    def check():
        out = log_probs(x, idx, top=3)
        loss = distill_loss(x, t, ti)
        assert out.log_prob.shape == out.entropy.shape == loss.shape == (2, 4, 6)
        assert out.top_log_prob.shape == out.top_index.shape == (2, 3, 4, 6) and out.top_index.dtype == torch.int32
        assert out.log_prob.dtype == loss.dtype == torch.float32 and out.entropy.device == x.device
        bare = log_probs(x)
        assert bare.log_prob is None and bare.top_index is None and bare.entropy.shape == (2, 4, 6)
        with pytest.raises(TypeError):
            log_probs(x, idx.float())
        with pytest.raises(ValueError):
            distill_loss(x, t, ti[:, :4])

    with mode:
        check()
    check()   # the tensors' own class is enough


def test_traced_graphs_hold_the_operators_and_what_decides_them():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    from depth_estimation_amd.distribution import distill_loss, log_probs

    def f(x, idx, t, ti):
        o = log_probs(x, idx, scale=-2.0, top=3)
        loss = distill_loss(x, t, ti, renormalise=True)
        return o.log_prob, o.top_index, loss

    mode = FakeTensorMode()
    args = _fake_problem(mode)
    with mode:
        graph = make_fx(f)(*args)
    calls = {n.target: n for n in graph.graph.nodes if n.op == "call_function"}
    lp, ds = calls[torch.ops.depthwarp.log_probs.default], calls[torch.ops.depthwarp.distill_loss.default]
    assert lp.args[2:] == (1, -2.0, 3) and ds.args[3:] == (1, 1.0, True)
    assert not any("eager" in str(t) or "empty" in str(t) for t in calls)
