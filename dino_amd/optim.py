"""FusedAdamW and FusedMuon over the student's flat parameter buffer.

FusedAdamW: torch.optim.AdamW semantics (reference dino.py:251, train_utils.py:56-59,131)
as ONE streaming kernel over the student's flat parameter buffer, fused with the per-tensor
gradient clip factor, the momentum-teacher EMA (train_utils.py:152-162) and the refresh of
the bf16 weight shadows of student and teacher.

FusedMuon: the hidden matrices by orthogonalised momentum (all of them in one sequence of launches), everything else by
the same AdamW pass, which also does the EMA and the shadows of both.

They subclass torch.optim.Optimizer so param_groups / state_dict keep the reference's shape
(the step loop rewrites param_groups[i]["lr"/"weight_decay"] every iteration).
"""
import time

import numpy as np
import torch

from . import ops
from .utils.utils import _unwrap


class FusedAdamW(torch.optim.Optimizer):
    def __init__(self, params, student, teacher=None, lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
                 weight_decay=1e-2, amsgrad=False, maximize=False):
        if amsgrad or maximize:
            raise NotImplementedError("FusedAdamW: amsgrad / maximize are off in the reference (dino.py:251)")
        # the remaining keys are what torch.optim.AdamW keeps in every param_group: a checkpoint written
        # here has the reference's optimizer layout key for key (tests/golden/ops.npz ckpt/manifest_json)
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, amsgrad=False,
                        maximize=False, foreach=None, capturable=False, differentiable=False, fused=None,
                        decoupled_weight_decay=True)
        super().__init__(params, defaults)
        self._student = _unwrap(student)
        self._teacher = None if teacher is None else _unwrap(teacher)
        self._st = None
        self._hp_host = None

    _NBUF = 3   # pinned hyper-parameter tables in rotation (see step())

    def _bind(self):
        st = self._student.store()
        if st is self._st:
            return st
        # the store was re-materialised (student.to(), DataParallel's re-bind): the row counters are the live
        # step counts -- write them back before state[p]["step"] is re-read below, or AdamW's bias corrections
        # would restart at t = 1 on carried-over moments (no-op after load_state_dict, which clears _st)
        self._sync_step_state()
        self._st = st
        n, dev = st.layout.total, st.device
        self.exp_avg = torch.zeros(n, dtype=torch.float32, device=dev)
        self.exp_avg_sq = torch.zeros(n, dtype=torch.float32, device=dev)
        self._name_of = {id(p): k for k, p in st.params.items()}
        row_of = {k: i for i, k in enumerate(st.layout.names)}
        nt = len(st.layout.names)
        # a table the GPU may still be reading is never rewritten: _NBUF pinned tables in rotation, each
        # guarded by an event recorded behind its host -> device copy
        self._hp_host = [torch.zeros((nt, 8), dtype=torch.float32).pin_memory() for _ in range(self._NBUF)]
        self._hp_np = [h.numpy() for h in self._hp_host]
        self._hp_event = [None] * self._NBUF
        self.host_wait_s = 0.0
        self._hp_turn = 0
        self._hp_dev = torch.zeros((nt, 8), dtype=torch.float32, device=dev)
        # per group: the parameters in table-row order, for one vectorised fill per group
        self._rows, self._params = [], []
        self._steps = np.zeros(nt, dtype=np.float64)   # torch.optim.AdamW's state[p]["step"], by row
        for group in self.param_groups:
            rows = []
            for p in group["params"]:
                k = self._name_of.get(id(p))
                if k is None:
                    raise ValueError("FusedAdamW: parameter does not belong to the student store")
                rows.append(row_of[k])
                s = self.state[p]
                prev_m, prev_v = s.get("exp_avg"), s.get("exp_avg_sq")
                s.setdefault("step", torch.tensor(0.0))
                self._steps[row_of[k]] = float(s["step"])
                s["exp_avg"] = st.layout.view(self.exp_avg, k)
                s["exp_avg_sq"] = st.layout.view(self.exp_avg_sq, k)
                if prev_m is not None:
                    s["exp_avg"].copy_(prev_m)
                    s["exp_avg_sq"].copy_(prev_v)
            self._rows.append(np.asarray(rows, dtype=np.int64))
            self._params.append(list(group["params"]))
        return st

    def _sync_step_state(self):
        """state[p]["step"] (what torch.optim.AdamW keeps, and what a checkpoint stores) from the row
        counters the step loop maintains."""
        if self._st is None:
            return
        for rows, params in zip(self._rows, self._params):
            for r, p in zip(rows, params):
                self.state[p]["step"] = torch.tensor(float(self._steps[r]))

    def state_dict(self):
        self._sync_step_state()
        return super().state_dict()

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        self._st = None  # re-bind: copies the loaded moments and step counts into the flat buffers
        self._bind()

    @torch.no_grad()
    def step(self, closure=None, ema_momentum=None, clip_coef=None):
        """One AdamW update.  ema_momentum: if given (and a teacher was passed) the teacher EMA
        k <- m k + (1-m) q runs in the same pass.  clip_coef: optional device fp32 [ntensors]
        per-tensor gradient scale from utils.grad_stats_async(materialize=False)."""
        st = self._bind()
        if st.pending_bwd:
            raise RuntimeError(
                f"FusedAdamW.step(): {st.pending_bwd} recorded backbone pass(es) of the student were never "
                "back-propagated, so this step's gradients are incomplete.  Run inference under "
                "torch.no_grad() or drop the outputs of forward passes you do not back-propagate.")
        turn = self._hp_turn
        self._hp_turn = (turn + 1) % self._NBUF
        if self._hp_event[turn] is not None:
            t0 = time.perf_counter()
            self._hp_event[turn].synchronize()   # its last copy (NBUF steps ago) has been consumed
            self.host_wait_s += time.perf_counter() - t0   # host time spent throttled, not issuing
        hp = self._hp_np[turn]
        hp[:] = 0.0
        for group, rows, params in zip(self.param_groups, self._rows, self._params):
            if not len(rows):
                continue
            b1, b2 = group["betas"]
            # torch skips a parameter without a gradient: no moment update, no decay, no step count
            active = np.fromiter((p.grad is not None for p in params), dtype=bool, count=len(params))
            active = self._split_off(group, rows, active, hp)
            r = rows[active]
            self._steps[r] += 1
            t = self._steps[r]
            hp[r, 0], hp[r, 1] = group["lr"], group["weight_decay"]
            hp[r, 2], hp[r, 3], hp[r, 4] = 1 - b1 ** t, 1 - b2 ** t, 1.0
        # inactive rows keep lr = 0; give them benign bias corrections (never read when inactive)
        np.maximum(hp[:, 2:4], 1e-30, out=hp[:, 2:4])
        self._hp_dev.copy_(self._hp_host[turn], non_blocking=True)
        ev = self._hp_event[turn] or torch.cuda.Event()
        ev.record()
        self._hp_event[turn] = ev
        g0 = self.param_groups[0]
        tst = None
        m = 1.0
        if ema_momentum is not None and self._teacher is not None:
            tst = self._teacher.store()
            tst.managed = True
            if tst.layout.total != st.layout.total:
                raise ValueError("teacher and student layouts differ")
            m = float(ema_momentum)
        self._before_adamw(st, clip_coef)
        ops.adamw_ema(st.flat, st.grad_flat, self.exp_avg, self.exp_avg_sq,
                      None if tst is None else tst.flat,
                      st.shadow if st.bf16 else None,
                      None if tst is None else (tst.shadow if tst.bf16 else None),
                      st.chunks, self._hp_dev, clip_coef, g0["betas"][0], g0["betas"][1], g0["eps"],
                      m, 1.0 - m)
        st.refresh_derived()
        if tst is not None:
            tst.refresh_derived()
        return None

    def _split_off(self, group, rows, active, hp):
        """Which of a group's rows AdamW updates (a subclass takes some for itself and fills their hp rows)."""
        return active

    def _before_adamw(self, st, clip_coef):
        """Updates of the rows that _split_off took; AdamW's pass then does their EMA and shadows."""

    def zero_grad(self, set_to_none: bool = True):
        st = self._bind()
        if set_to_none:
            for p in st.params.values():
                p.grad = None
        st.grad_flat.zero_()
        st._need_zero = False


class FusedMuon(FusedAdamW):
    """Muon for the hidden matrices of the backbone's blocks and the head's MLP (2-D weights; qkv as three matrices),
    AdamW for everything else -- embeddings, norms, biases, the prototypes -- in one step() with FusedAdamW's contract.

        buf = momentum * buf + grad;  u = grad + momentum * buf  (nesterov) or buf
        weight = weight * (1 - lr * weight_decay) - lr * scale * orthogonalize(u)

    scale: "rms" = 0.2 * sqrt(max(rows, cols)), which gives the update the size of AdamW's, so one learning-rate schedule
    serves both; "spectral" = sqrt(max(1, rows / cols)).  select(name, parameter) -> bool chooses the matrices.
    state[p]["exp_avg"] of a matrix is its momentum buffer (and its "exp_avg_sq" stays zero): checkpoints keep AdamW's
    layout."""

    def __init__(self, params, student, teacher=None, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
                 momentum=0.95, nesterov=True, ns_steps=5, ns_coeffs=ops.NS_COEFFS, ns_eps=1e-7, scale="rms", select=None):
        if not 0.0 <= momentum < 1.0:
            raise ValueError(f"FusedMuon: momentum {momentum} is not in [0, 1)")
        if scale not in ("rms", "spectral"):
            raise ValueError(f"FusedMuon: scale is \"rms\" or \"spectral\", got {scale!r}")
        ops.OrthoPlan([], steps=ns_steps, coeffs=ns_coeffs, eps=ns_eps)          # refuses what no step could use
        super().__init__(params, student, teacher, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay)
        self.momentum, self.nesterov = float(momentum), bool(nesterov)
        self.ns_steps, self.ns_coeffs, self.ns_eps = ns_steps, ns_coeffs, float(ns_eps)
        self.scale, self._select = scale, select if select is not None else is_hidden_matrix

    def _bind(self):
        old = self._st
        st = super()._bind()
        if st is not old:
            names = [k for k in st.layout.names if st.params[k].requires_grad and self._select(k, st.params[k])]
            for k in names:
                if st.params[k].dim() != 2:
                    raise ValueError(f"FusedMuon: {k} is not a matrix")
            index = {k: i for i, k in enumerate(st.layout.names)}
            mine = set(index[k] for k in names)
            keep = torch.tensor([int(t) in mine for t in st.layout.chunks[:, 0]], dtype=torch.bool)
            self._mchunks = st.layout.chunks[keep].contiguous().to(st.device)
            self._update = torch.zeros(st.layout.total, dtype=torch.float32, device=st.device)
            self._ortho = torch.zeros(st.layout.total, dtype=torch.bfloat16, device=st.device)
            self._mscale = np.zeros(len(st.layout.names))
            mats = []                                 # (update, ortho) views
            for k in names:
                r, c = st.params[k].shape
                parts = 3 if k.endswith("attn.qkv.weight") and r == 3 * c else 1
                rr = r // parts
                self._mscale[index[k]] = 0.2 * max(rr, c) ** 0.5 if self.scale == "rms" else max(1.0, rr / c) ** 0.5
                shape = (parts, rr, c)
                mats.append((st.layout.view(self._update, k).view(shape), st.layout.view(self._ortho, k).view(shape)))
            self._plan = ops.OrthoPlan([u for u, _ in mats], [o for _, o in mats], steps=self.ns_steps,
                                       coeffs=self.ns_coeffs, eps=self.ns_eps)
        return st

    def _split_off(self, group, rows, active, hp):
        mine = self._mscale[rows] != 0
        take = rows[mine & active]
        hp[take, 0], hp[take, 1] = group["lr"], group["weight_decay"]
        hp[take, 5], hp[take, 6] = 1.0, self._mscale[take]
        self._steps[take] += 1
        return active & ~mine

    def _before_adamw(self, st, clip_coef):
        if not self._plan.out:
            return
        ops.muon_momentum(st.grad_flat, self.exp_avg, self._update, self._mchunks, self._hp_dev, clip_coef,
                          self.momentum, self.nesterov)
        self._plan.run()
        ops.muon_apply(st.flat, self._ortho, self._mchunks, self._hp_dev)


def is_hidden_matrix(name, param):
    """The weights that act on hidden features: linear layers of the blocks and of the head's MLP (not the patch or
    position embeddings, norms, biases, or the prototypes)."""
    return (param.dim() == 2 and name.endswith(".weight")
            and ("blocks." in name or ".mlp" in "." + name) and "last_layer" not in name)


@torch.no_grad()
def update_teacher(student, teacher, m):
    """Stand-alone momentum-teacher update (the inline loop of train_utils.py:152-162) for
    callers that step a stock optimizer: one launch over the flat buffers."""
    s, t = _unwrap(student).store(), _unwrap(teacher).store()
    m = float(m)
    ops.ema(t.flat, s.flat, t.shadow if t.bf16 else None, m, 1.0 - m)
    t.refresh_derived()
