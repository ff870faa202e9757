"""Cases over which the prototype log probabilities and the orthogonalised updates are measured.

`own` false computes each operator from elementary torch operations in 32 bits; `own` true makes the calls of
dino_amd.  exact() is the definition in 64 bits."""
import math

import torch

own = False

DEV = "cuda"
COEFFS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7
_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _lp(name, rows, protos, dtype, targets, topk, temp, centred, masked, grad):
    return {"name": name, "kind": "logprob", "rows": rows, "protos": protos, "dtype": dtype, "targets": targets,
            "topk": topk, "temp": temp, "centred": centred, "masked": masked, "grad": grad}


def _ns(name, shapes, dtype, strided=False):
    return {"name": name, "kind": "ortho", "shapes": shapes, "dtype": dtype, "strided": strided}


def listed():
    return [
        # one crop's teacher output against the 65 536 prototypes: looking at a single image, latency counts
        _lp("logprob one crop", 1, 65536, "bf16", 1, 5, 0.04, True, False, False),
        # the teacher's two global crops of a batch of 256: entropy, assigned prototypes and the best eight, centred
        _lp("logprob teacher batch", 512, 65536, "bf16", 1, 8, 0.04, True, False, False),
        # the student's ten local crops of that batch, with the gradient: distillation onto given prototypes
        _lp("logprob student grad", 2560, 65536, "bf16", 1, 0, 0.1, False, False, True),
        # a small head of odd width in fp32, several assigned prototypes a row, some masked, some rows with none left
        _lp("logprob odd fp32 grad", 333, 8191, "fp32", 4, 3, 0.1, True, True, True),
        # every patch token of 64 global crops (197 tokens) against a small head, with the gradient
        _lp("logprob patch tokens grad", 12608, 4096, "bf16", 1, 2, 0.1, False, False, True),
        # one projection of ViT-Ti: the smallest update
        _ns("ortho one 192", "1x192x192", "fp32"),
        # every hidden matrix of ViT-S/16's twelve blocks: q, k, v and proj apart, fc1, fc2
        _ns("ortho ViT-S", "48x384x384,12x1536x384,12x384x1536", "fp32"),
        # the same of ViT-L/14's twenty-four blocks: the largest
        _ns("ortho ViT-L", "96x1024x1024,24x4096x1024,24x1024x4096", "fp32"),
        # the DINO head's MLP for ViT-S (384 -> 2048 -> 2048 -> 256), bf16 momentum
        _ns("ortho head", "1x2048x384,1x2048x2048,1x256x2048", "bf16"),
        # odd sizes: ViT-L/14's patch projection (3 * 14 * 14 = 588 columns) and ragged matrices, rows of a wider buffer
        _ns("ortho odd strided", "1x1024x588,3x251x1000,2x77x65,1x1x300", "fp32", True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        protos = _log_int(rng, 64, 100000)
        rows = _log_int(rng, 1, max(1, min(16384, 160_000_000 // protos)))
        return {"kind": "logprob", "rows": rows, "protos": protos, "dtype": rng.choice(["bf16", "fp32"]),
                "targets": rng.choice([1, 1, 2, 5]), "topk": rng.choice([0, 1, 4, 10, 20]),
                "temp": rng.choice([0.04, 0.07, 0.1, 1.0]), "centred": rng.random() < 0.5,
                "masked": rng.random() < 0.3, "grad": rng.random() < 0.5}
    parts, left = [], 40e9
    for _ in range(rng.randint(1, 4)):
        r, c = _log_int(rng, 16, 2200), _log_int(rng, 16, 2200)
        m, n = min(r, c), max(r, c)
        cost = 4.0 * m * m * n + 2.0 * m ** 3
        batch = max(1, min(_log_int(rng, 1, 24), int(left / cost)))
        parts.append("%dx%dx%d" % (batch, r, c))
        left = max(0.0, left - batch * cost)
    return {"kind": "ortho", "shapes": ",".join(parts), "dtype": rng.choice(["fp32", "bf16"]),
            "strided": rng.random() < 0.3}


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = _DT[case["dtype"]]
    if case["kind"] == "ortho":
        # a momentum: a few strong directions whose weights fall off, over noise of every direction; small numbers
        ups = []
        for b, r, c in _shapes(case):
            k = max(1, min(r, c, 16))
            w = torch.arange(1, k + 1, device=DEV, dtype=torch.float32).rsqrt()
            u = (torch.randn(b, r, k, generator=g, device=DEV) * w) @ torch.randn(b, k, c, generator=g, device=DEV)
            u = (u + torch.randn(b, r, c, generator=g, device=DEV)) * 1e-3
            if case["strided"]:
                wide = torch.zeros((b, r, c + 24), dtype=dt, device=DEV)
                wide[:, :, 8:8 + c] = u.to(dt)
                ups.append(wide[:, :, 8:8 + c])
            else:
                ups.append(u.to(dt))
        return {"case": case, "updates": ups}
    R, K, T = case["rows"], case["protos"], case["targets"]
    # similarities of a normalised bottleneck with the prototypes: a narrow bulk, a few near ones
    x = torch.randn(R, K, generator=g, device=DEV).mul_(0.12)
    near = torch.randint(0, K, (R, 4), generator=g, device=DEV)
    x.scatter_add_(1, near, torch.rand(R, 4, generator=g, device=DEV) * 0.6)
    tgt = torch.randint(0, K, (R, T), generator=g, device=DEV)
    tgt[:, 0] = near[:, 0]
    if case["masked"]:
        x.masked_fill_(torch.rand(R, K, generator=g, device=DEV) < 0.1, -math.inf)
        x[::7] = -math.inf                    # rows whose mask leaves nothing
        tgt[1::5, -1] = -1                    # an absent target
    center = torch.randn(K, generator=g, device=DEV) * 0.05 if case["centred"] else None
    s = {"case": case, "logits": x.to(dt), "targets": tgt, "center": center}
    if case["grad"]:
        s["g_logp"] = torch.randn(R, T, generator=g, device=DEV) / R
        s["g_ent"] = torch.randn(R, generator=g, device=DEV) / R
    return s


def _plain_logprob(s):
    case, tgt = s["case"], s["targets"]
    x = s["logits"].to(torch.float32)
    d = x - s["center"] if s["center"] is not None else x
    md = d.max(1, keepdim=True).values
    empty = md == -math.inf
    zs = (d - torch.where(empty, torch.zeros_like(md), md)) / case["temp"]
    e = torch.exp(zs)
    tot = e.sum(1, keepdim=True)
    lp = zs - torch.log(tot)                                   # -inf - -inf in an empty row
    lp = torch.where(empty, torch.full_like(lp, -math.inf), lp)
    p = torch.where(empty, torch.zeros_like(e), e / tot)
    plp = torch.where(p > 0, p * torch.where(p > 0, lp, torch.zeros_like(lp)), torch.zeros_like(p))
    ent = -plp.sum(1)
    have = tgt >= 0
    at = tgt.clamp(min=0)
    logp = torch.where(have, lp.gather(1, at), torch.zeros((), device=DEV))
    out = {"log_prob": logp, "entropy": ent}
    if case["topk"]:
        idx = torch.sort(d, dim=1, descending=True, stable=True).indices[:, :case["topk"]]
        out["top_index"] = idx
        out["top_log_prob"] = lp.gather(1, idx)
    if case["grad"]:
        gl = torch.where(have & ~empty, s["g_logp"], torch.zeros((), device=DEV))
        dz = -p * gl.sum(1, keepdim=True) - s["g_ent"][:, None] * (plp + p * ent[:, None])
        dz.scatter_add_(1, at, gl)
        out["dlogits"] = (dz / case["temp"]).to(s["logits"].dtype)
    return out


def _plain_ortho(s):
    a, b, c = COEFFS
    outs = []
    for u in s["updates"]:
        x = u.to(torch.float32)
        flip = x.shape[1] > x.shape[2]
        x = x.transpose(1, 2).contiguous() if flip else x.contiguous()
        x = x / (torch.sqrt((x * x).sum((1, 2), keepdim=True)) + EPS)
        for _ in range(5):
            g = torch.matmul(x, x.transpose(1, 2))
            x = a * x + torch.matmul(b * g + c * torch.matmul(g, g), x)
        outs.append((x.transpose(1, 2) if flip else x).contiguous().to(torch.bfloat16))
    return outs


def run(state):
    case = state["case"]
    if not own:
        return _plain_ortho(state) if case["kind"] == "ortho" else _plain_logprob(state)
    from dino_amd import ops
    if case["kind"] == "ortho":
        return ops.orthogonalize(state["updates"], steps=5, coeffs=COEFFS, eps=EPS)
    r = ops.logprob_fwd(state["logits"], state["targets"], center=state["center"], temp=case["temp"], topk=case["topk"])
    out = {"log_prob": r.log_prob, "entropy": r.entropy}
    if case["topk"]:
        out["top_index"], out["top_log_prob"] = r.top_index, r.top_log_prob
    if case["grad"]:
        out["dlogits"] = ops.logprob_bwd(state["logits"], r, targets=state["targets"], center=state["center"],
                                         temp=case["temp"], dlog_prob=state["g_logp"], dentropy=state["g_ent"])
    return out


def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "ortho":
        nbytes = flops = 0.0
        for b, r, c in _shapes(case):
            m, n = min(r, c), max(r, c)
            nbytes += b * r * c * (es + 2.0)
            # the two symmetric products need half of their entries
            flops += 5.0 * b * (m * (m + 1.0) * n + m * (m + 1.0) * m + 2.0 * m * m * n)
        return {"bytes": nbytes, "flops": flops}
    R, K, T = case["rows"], case["protos"], case["targets"]
    n = float(R) * K
    nbytes = n * es * (2 if case["grad"] else 1) + (4.0 * K if case["centred"] else 0.0)
    nbytes += R * (T * 12.0 + 4.0 + case["topk"] * 12.0) + (R * (T + 1) * 4.0 if case["grad"] else 0.0)
    return {"bytes": nbytes, "flops": n * (12.0 if case["grad"] else 6.0)}


def exact(case, seed):
    s = prepare(case, seed)
    f8 = torch.float64
    if case["kind"] == "ortho":
        a, b, c = COEFFS
        outs = []
        for u in s["updates"]:
            y = torch.empty(u.shape, dtype=f8, device=DEV)
            for i in range(u.shape[0]):
                v = u[i].to(f8)
                v = v / (torch.linalg.vector_norm(v) + EPS)
                tall = v.shape[0] > v.shape[1]
                for _ in range(5):          # the Gram matrix of the shorter side, on that side
                    q = v.T @ v if tall else v @ v.T
                    q = b * q + c * (q @ q)
                    v = a * v + (v @ q if tall else q @ v)
                y[i] = v
            outs.append(y)
        return outs
    tau = float(case["temp"])
    x = s["logits"].to(f8)
    if s["center"] is not None:
        x = x - s["center"].to(f8)
    x = x / tau
    lse = torch.logsumexp(x, 1, keepdim=True)
    none = torch.isneginf(lse)
    lp = torch.where(none, torch.full_like(x, -math.inf), x - lse)
    pr = torch.exp(lp)
    h = -torch.xlogy(pr, pr).sum(1)
    tgt = s["targets"]
    given = tgt >= 0
    safe = tgt.clamp(min=0)
    logp = torch.where(given, torch.take_along_dim(lp, safe, 1), torch.zeros((), dtype=f8, device=DEV))
    out = {"log_prob": logp, "entropy": h}
    if case["topk"]:
        out["top_index"] = None
        out["top_log_prob"] = torch.topk(lp, case["topk"], dim=1).values
    if case["grad"]:
        gl = s["g_logp"].to(f8) * (given & ~none)
        dz = torch.zeros_like(x).scatter_add_(1, safe, gl) - pr * gl.sum(1, keepdim=True)
        dz -= s["g_ent"].to(f8)[:, None] * (torch.xlogy(pr, pr) + pr * h[:, None])
        out["dlogits"] = dz / tau
    return out
