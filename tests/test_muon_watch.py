"""FusedMuon (hidden matrices by orthogonalised momentum, the rest by AdamW), DINOLoss.watch / prototype_log_probs, and
the two together in training steps."""
import math

import numpy as np
import pytest
import torch

from tests.test_ortho import recurrence

gpu = pytest.mark.gpu
DEV = "cuda"


def _setup(dtype, nsteps=4, **kw):
    from dino_amd.components.loss import DINOLoss
    from dino_amd.optim import FusedMuon
    from dino_amd.utils import get_params_groups
    from tests.golden_spec import TINY, tiny_crops
    from tests.helpers_model import build_pair
    student, teacher = build_pair(TINY, dtype)
    crops = [c.to(DEV) for c in tiny_crops()]
    loss_fn = DINOLoss(TINY["head"]["out_dim"], len(crops), 0.04, 0.04, 0, nsteps).to(DEV)
    return student, teacher, loss_fn, FusedMuon(get_params_groups(student), student, teacher, **kw), crops


def _backward(student, teacher, loss_fn, opt, crops, it):
    with torch.no_grad():
        t = teacher(crops[:2])
    s = student(crops)
    loss = loss_fn(s, t, it)
    opt.zero_grad()
    loss.backward()
    return loss


@gpu
@pytest.mark.parametrize("nesterov,scale", [(True, "rms"), (False, "spectral")])
def test_step_matches_the_formula(nesterov, scale):
    """Two steps: matrices against the recurrence in 64 bits (tolerance: lr * scale times that of the orthogonalised update,
    plus fp32 roundings of the weight), the others against torch.optim.AdamW, the teacher against the EMA of the result."""
    from dino_amd.optim import is_hidden_matrix
    student, teacher, loss_fn, opt, crops = _setup(torch.float32, nesterov=nesterov, scale=scale, momentum=0.9)
    for g in opt.param_groups:
        g["lr"] = 1e-3
    opt.param_groups[0]["weight_decay"] = 0.05
    names = dict(student.named_parameters())
    hidden = {k for k, p in names.items() if is_hidden_matrix(k, p)}
    assert any("qkv" in k for k in hidden) and any("head.mlp" in k for k in hidden)
    assert not any("last_layer" in k or "pos_embed" in k or "patch" in k or k.endswith("bias") for k in hidden)
    buf = {k: torch.zeros(names[k].shape, dtype=torch.float64) for k in hidden}
    rest = {k: p.detach().clone().requires_grad_(True) for k, p in names.items() if k not in hidden and p.requires_grad}
    wd = {id(p): g["weight_decay"] for g in opt.param_groups for p in g["params"]}
    ref = torch.optim.AdamW([{"params": [rest[k]], "weight_decay": wd[id(names[k])]} for k in rest], lr=1e-3)
    for it in range(2):
        _backward(student, teacher, loss_fn, opt, crops, it)
        before = {k: p.detach().double().cpu() for k, p in names.items()}
        tb = {k: p.detach().double().cpu() for k, p in teacher.named_parameters()}
        grads = {k: p.grad.detach().double().cpu() for k, p in names.items() if p.grad is not None}
        for k, p in rest.items():
            p.grad = names[k].grad.detach().clone()
        ref.step()
        opt.step(ema_momentum=0.75)
        for k in hidden:
            buf[k] = 0.9 * buf[k] + grads[k]
            u = grads[k] + 0.9 * buf[k] if nesterov else buf[k]
            r, c = u.shape
            parts = 3 if "qkv" in k else 1
            sc = 0.2 * max(r // parts, c) ** 0.5 if scale == "rms" else max(1.0, r / parts / c) ** 0.5
            got = names[k].detach().double().cpu()
            for a in range(parts):
                sl = slice(a * (r // parts), (a + 1) * (r // parts))
                o, tol = recurrence(u[sl])
                want = before[k][sl] * (1 - 1e-3 * 0.05) - 1e-3 * sc * o
                d = torch.linalg.vector_norm(got[sl] - want).item()
                assert d <= 1e-3 * sc * tol + 4 * 2.0 ** -24 * torch.linalg.vector_norm(want).item(), (k, a, d)
        for k, p in rest.items():
            # fp32 AdamW twice: a few roundings of the weight and of a step of at most lr
            tol = 8 * 2.0 ** -24 * (names[k].detach().abs().max().item() + 1e-3) + 1e-3 * 2e-5
            assert (names[k].detach() - p.detach()).abs().max().item() <= tol, k
        for k, p in teacher.named_parameters():
            want = 0.75 * tb[k] + 0.25 * names[k].detach().double().cpu()
            assert (p.detach().double().cpu() - want).abs().max().item() <= 4 * 2.0 ** -24 * (want.abs().max().item() + 1e-30), k


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_checkpoint_goes_on_where_it_stopped(dtype, tmp_path):
    from dino_amd.utils.train_utils import train_step
    lr, wd, mom = np.full(4, 1e-3), np.full(4, 0.04), np.full(4, 0.99)
    runs = []
    for stop in (False, True):
        student, teacher, loss_fn, opt, crops = _setup(dtype)
        for it in range(3):
            if stop and it == 2:
                path = tmp_path / "c.pt"
                torch.save({"s": student.state_dict(), "t": teacher.state_dict(), "o": opt.state_dict(),
                            "l": loss_fn.state_dict()}, path)
                ck = torch.load(path, weights_only=True)
                student, teacher, loss_fn, opt, crops = _setup(dtype)
                student.load_state_dict(ck["s"])
                teacher.load_state_dict(ck["t"])
                loss_fn.load_state_dict(ck["l"])
                opt.load_state_dict(ck["o"])
            train_step(student, teacher, loss_fn, opt, crops, it, lr, wd, mom, 3.0, 0)
        runs.append({k: p.detach().clone() for k, p in student.named_parameters()})
    for k in runs[0]:
        # the backward pass adds some gradients with float atomics: the last bits of AdamW's side may differ
        d = (runs[0][k].float() - runs[1][k].float()).abs().max().item()
        assert d <= 2e-4, (k, d)


@gpu
def test_matrices_without_a_gradient_stay_and_follow_the_teacher():
    student, teacher, loss_fn, opt, crops = _setup(torch.float32)
    _backward(student, teacher, loss_fn, opt, crops, 0)
    name = "backbone.blocks.0.mlp.fc1.weight"
    p = dict(student.named_parameters())[name]
    p.grad = None
    w = p.detach().clone()
    t0 = dict(teacher.named_parameters())[name].detach().clone()
    opt.step(ema_momentum=0.5)
    assert torch.equal(p.detach(), w) and (opt.state[p]["exp_avg"] == 0).all()
    assert torch.allclose(dict(teacher.named_parameters())[name], 0.5 * t0 + 0.5 * w, atol=1e-7)


def _plain_watch(s, t, center, ncrops, temp, stemp):
    s, t = s.double().cpu(), t.double().cpu()
    B = t.shape[0] // 2
    lt = torch.log_softmax((t - center.double().cpu()) / temp, 1)
    ls = torch.log_softmax(s / stemp, 1)
    best = (t.float() - center.cpu()).argmax(1)
    agree, assigned = [], []
    for c in range(ncrops):
        for b in range(B):
            mine = [best[v * B + b].item() for v in range(2) if v != c]
            row = c * B + b
            agree.append(float(s[row].argmax().item() in mine))
            assigned += [ls[row, m].item() for m in mine]
    return {"teacher_entropy": -(lt.exp() * lt).sum(1).mean().item(), "student_entropy": -(ls.exp() * ls).sum(1).mean().item(),
            "agreement": sum(agree) / len(agree), "assigned_log_prob": sum(assigned) / len(assigned),
            "prototypes_used": float(len(set(best.tolist())))}


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_watch_matches_plain_code(dtype):
    from dino_amd.components.loss import DINOLoss
    B, ncrops, K = 5, 6, 700
    g = torch.Generator().manual_seed(1)
    s = (torch.randn(ncrops * B, K, generator=g) * 0.3).to(dtype)
    t = (torch.randn(2 * B, K, generator=g) * 0.3).to(dtype)
    s[:B] += t[B:] * 2                                   # some agreement
    loss_fn = DINOLoss(K, ncrops, 0.04, 0.04, 0, 3).to(DEV)
    loss_fn.center.copy_(torch.randn(1, K, generator=g) * 0.1)
    c = loss_fn.center.clone()
    got = loss_fn.watch(s.to(DEV), t.to(DEV), 1)
    want = _plain_watch(s, t, c, ncrops, 0.04, 0.1)
    assert set(got) == set(want) and torch.equal(loss_fn.center, c)
    for k in want:
        assert got[k].dim() == 0 and abs(got[k].item() - want[k]) <= 2e-5 * (1 + abs(want[k])), (k, got[k].item(), want[k])


@gpu
def test_no_hidden_matrix_is_adamw():
    """select can take none: then every parameter is AdamW's."""
    from dino_amd.optim import FusedAdamW
    from dino_amd.utils import get_params_groups
    runs = []
    for muon in (True, False):
        student, teacher, loss_fn, opt, crops = _setup(torch.float32, select=lambda k, p: False)
        if not muon:
            opt = FusedAdamW(get_params_groups(student), student, teacher)
        _backward(student, teacher, loss_fn, opt, crops, 0)
        g = {k: p.grad.clone() for k, p in student.named_parameters() if p.grad is not None}
        runs.append((g, {k: p.detach().clone() for k, p in student.named_parameters()}, opt, student))
    for g, _, opt, student in runs:                       # the same gradients for both (they are added with float atomics)
        for k, p in student.named_parameters():
            if p.grad is not None:
                p.grad.copy_(runs[0][0][k])
        opt.step(ema_momentum=0.9)
    a, b = (dict(r[3].named_parameters()) for r in runs)
    for k in a:
        assert torch.equal(a[k], b[k]), k


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prototype_log_probs_and_its_gradient(dtype):
    from dino_amd.components import prototype_log_probs
    g = torch.Generator().manual_seed(2)
    x = (torch.randn(7, 513, generator=g) * 0.3).to(dtype)
    c = torch.randn(1, 513, generator=g) * 0.1
    tgt = torch.randint(0, 513, (7,), generator=g)
    tgt[3] = -1
    w = torch.randn(7, generator=g)
    xd = x.to(DEV).requires_grad_(True)
    r = prototype_log_probs(xd, tgt.to(DEV), center=c.to(DEV), temperature=0.1, topk=3)
    assert r.log_prob.shape == (7,) and r.top_index.shape == (7, 3) and not r.top_index.requires_grad
    (r.log_prob * w.to(DEV)).sum().add(r.entropy.sum() * 0.5).add(r.top_log_prob[:, 1].sum()).backward()
    x64 = x.double().requires_grad_(True)
    lp = torch.log_softmax((x64 - c.double()) / 0.1, 1)
    top = (x.float() - c).topk(3, 1).indices
    ref = (torch.where(tgt >= 0, lp.gather(1, tgt.clamp(min=0)[:, None])[:, 0], 0.0) * w).sum() \
        - 0.5 * (lp.exp() * lp).sum() + lp.gather(1, top)[:, 1].sum()
    ref.backward()
    half = torch.finfo(dtype).eps / 2
    tol = half * x64.grad.abs() + 1e-4 * 10 * lp.exp().detach() + 1e-5      # 1e-4: fp32 of z up to 30, times p / temperature
    assert ((xd.grad.double().cpu() - x64.grad).abs() <= tol).all()
    assert torch.equal(r.top_index.cpu(), top)
    with torch.no_grad():
        only = prototype_log_probs(xd, topk=0, temperature=0.1)
    assert only.log_prob is None and only.top_index is None
    e = prototype_log_probs(xd, None, temperature=0.1).entropy            # entropy alone has a gradient too
    (gx,) = torch.autograd.grad(e.sum(), xd)
    assert gx.abs().sum() > 0


@gpu
def test_differentiable_form_refuses_capture():
    from dino_amd import ops
    from dino_amd.components import prototype_log_probs
    x = torch.randn(3, 40, device=DEV, requires_grad=True)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    refused = False
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        try:
            prototype_log_probs(x, None)
        except RuntimeError:
            refused = True
        r = ops.logprob_fwd(x.detach(), None, topk=1)                     # the captured form
    graph.replay()
    torch.cuda.synchronize()
    assert refused and torch.equal(r.top_index[:, 0], x.argmax(1))


@gpu
def test_training_with_both_together():
    """Steps as train_one_epoch runs them: FusedMuon with the watch beside the loss; taking the watch changes no weight."""
    from dino_amd.utils.train_utils import train_one_epoch
    nsteps = 3
    finals, stats = [], []
    for every in (0, 2):
        student, teacher, loss_fn, opt, crops = _setup(torch.float32, nsteps=nsteps)
        loader = [([c.clone() for c in crops], None) for _ in range(nsteps)]
        st = train_one_epoch(student, teacher, teacher, loss_fn, loader, opt, np.full(nsteps, 5e-4),
                             np.full(nsteps, 0.04), np.full(nsteps, 0.99), 0, 1, None, 3.0, 1, 0, None, -1, watch_every=every)
        finals.append({k: p.detach().clone() for k, p in student.named_parameters()})
        stats.append(st)
    assert "teacher_entropy" not in stats[0] and set(stats[0]) <= set(stats[1])
    K = loss_fn.center.numel()
    assert 0 <= stats[1]["teacher_entropy"] <= math.log(K) + 1e-4 and 1 <= stats[1]["prototypes_used"] <= K
    assert math.isfinite(stats[1]["assigned_log_prob"]) and 0 <= stats[1]["agreement"] <= 1
    assert math.isfinite(stats[1]["loss"]) and abs(stats[0]["loss"] - stats[1]["loss"]) <= 1e-5 * abs(stats[0]["loss"])
    for k in finals[0]:
        assert (finals[0][k] - finals[1][k]).abs().max().item() <= 1e-4, k      # float atomics in the backward pass


def test_refusals_on_the_cpu():
    from dino_amd._lib import DinoHipError
    from dino_amd.components import prototype_log_probs
    from dino_amd.components.loss import DINOLoss
    from dino_amd.optim import FusedMuon, is_hidden_matrix
    p = torch.nn.Parameter(torch.zeros(4, 4))
    for kw in (dict(momentum=1.0), dict(momentum=-0.1), dict(scale="other")):
        with pytest.raises(ValueError):
            FusedMuon([p], torch.nn.Linear(2, 2), **kw)
    for kw in (dict(ns_steps=0), dict(ns_coeffs=(1.0, 2.0)), dict(ns_coeffs=(20.0, 0.0, 0.0)), dict(ns_eps=-1.0)):
        with pytest.raises(DinoHipError):
            FusedMuon([p], torch.nn.Linear(2, 2), **kw)
    loss_fn = DINOLoss(10, 4, 0.04, 0.04, 0, 3)
    with pytest.raises(ValueError):
        loss_fn.watch(torch.zeros(7, 10), torch.zeros(4, 10), 0)            # 4 crops of 2 images are 8 rows
    lazy = torch.zeros(8, 10)
    lazy._dino_lazy = object()
    with pytest.raises(ValueError):
        loss_fn.watch(lazy, torch.zeros(4, 10), 0)
    with pytest.raises(ValueError):
        prototype_log_probs(torch.zeros(2, 5), center=torch.zeros(5, requires_grad=True))
    assert is_hidden_matrix("backbone.blocks.3.attn.qkv.weight", p) and is_hidden_matrix("head.mlp.2.weight", p)
    assert not is_hidden_matrix("head.last_layer.weight_v", p) and not is_hidden_matrix("backbone.norm.weight", p[0])
    assert not is_hidden_matrix("backbone.patch_embed.proj.weight", torch.zeros(4, 3, 2, 2))
