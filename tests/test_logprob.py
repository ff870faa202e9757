"""Log probabilities of given prototypes, entropy and best prototypes (ops.logprob_fwd / logprob_bwd) against the
definition in 64 bits, and their refusals."""
import math

import pytest
import torch

from dino_amd import ops
from dino_amd._lib import DinoHipError

gpu = pytest.mark.gpu
NEG = -math.inf
U32 = 2.0 ** -24                                    # half a step of fp32, relative


def reference(x, targets, center, temp, topk, dlp=None, dent=None, dtop=None):
    """Everything in 64 bits on the CPU; the order of the best by the fp32 difference (ties: lowest index)."""
    d32 = x.float() - center if center is not None else x.float()
    d = d32.double()
    md = d.max(1, keepdim=True).values
    none = md == NEG
    zs = (d - md.masked_fill(none, 0.0)) / temp
    lp = zs - torch.logsumexp(zs, 1, keepdim=True)
    lp = lp.masked_fill(none, NEG)
    p = lp.exp()
    plp = torch.where(p > 0, p * lp, torch.where(p == 0, 0.0, math.nan))
    ent = -plp.sum(1)
    given = targets >= 0
    at = targets.clamp(min=0)
    out = {"lp": torch.where(given, lp.gather(1, at), 0.0), "ent": ent, "zs": zs}
    if topk:
        out["idx"] = torch.sort(d32, dim=1, descending=True, stable=True).indices[:, :topk]
        out["top"] = lp.gather(1, out["idx"])
    dz = torch.zeros_like(d)
    mag = torch.zeros_like(d)                       # sum of the magnitudes that make up dz
    if dlp is not None:
        g = dlp.double() * (given & ~none)
        dz += torch.zeros_like(d).scatter_add_(1, at, g) - p * g.sum(1, keepdim=True)
        mag += torch.zeros_like(d).scatter_add_(1, at, g.abs()) + p * g.abs().sum(1, keepdim=True)
    if dtop is not None:
        g = dtop.double() * ~none
        dz += torch.zeros_like(d).scatter_add_(1, out["idx"], g) - p * g.sum(1, keepdim=True)
        mag += torch.zeros_like(d).scatter_add_(1, out["idx"], g.abs()) + p * g.abs().sum(1, keepdim=True)
    if dent is not None:
        g = dent.double()[:, None]
        dz -= g * (plp + p * ent[:, None])
        mag += g.abs() * (plp.abs() + p * ent[:, None].abs())
    out["dx"], out["mag"] = dz / temp, mag / temp
    return out


def delta(x, center, temp, zs):
    """Relative error of one e^zs and of the sums over them, from the kernel's roundings: zs = (d - md) * (1 / temp) has
    three of them and passes through log2(e) (two more) and exp2 (2 ulp), all but the last times |zs| <= 110 (beyond it
    e is 0); d itself is rounded at |d|; 64 values are added in sequence, then ten levels of a tree; log and the final
    subtraction add a few.  8 |zs| + 160 covers these, 2 |d| / temp the rounding of d."""
    d = (x.float() - center if center is not None else x.float()).double()
    fin = torch.where(torch.isfinite(d) & (d.abs() < 1e30), d.abs(), 0.0)
    z = torch.where(torch.isfinite(zs), zs.abs(), 0.0).clamp(max=110.0).max(1).values
    near = torch.where(zs > -110, fin, torch.zeros_like(fin)).max(1).values
    return U32 * (8 * z + 160 + (2 * near / temp if center is not None else 0.0))


def make(R, K, dtype, T, seed, masked=False, scale=0.12):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, K, generator=g) * scale
    tgt = torch.randint(0, K, (R, T), generator=g)
    if masked:
        x[torch.rand(R, K, generator=g) < 0.3] = NEG
        x[::3] = NEG
        tgt[1::2, -1] = -1
    x = x.to(dtype)
    c = torch.randn(K, generator=g) * 0.05
    return x, tgt, c, g


def near(got, want, tol):
    got = got.detach().cpu().double()
    # what fp32 cannot hold rounds to infinity: (-3.4e38 - 3) / 0.04 = -8.5e39, and the largest fp32 is 3.4e38
    want = torch.where(want.abs() > torch.finfo(torch.float32).max, want.sign() * math.inf, want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    both = got == want                               # infinities and exact ones
    off = torch.where(both | torch.isnan(want), torch.zeros_like(got), (got - want).abs() - tol)
    assert (off <= 0).all(), (off.max().item(), off.argmax().item())


def check(x, tgt, c, temp, topk, g, grads=True):
    R, K = x.shape
    T = tgt.shape[1]
    dlp = torch.randn(R, T, generator=g) if grads else None
    dent = torch.randn(R, generator=g) if grads else None
    dtop = torch.randn(R, topk, generator=g) if grads and topk else None
    ref = reference(x.cpu(), tgt, c, temp, topk, dlp, dent, dtop)
    cu = lambda t: None if t is None else t.cuda()   # noqa: E731
    xd = x if x.is_cuda else x.cuda()
    got = ops.logprob_fwd(xd, cu(tgt), center=cu(c), temp=temp, topk=topk)
    dl = delta(x.cpu(), c, temp, ref["zs"])
    near(got.log_prob, ref["lp"], dl[:, None] + U32 * ref["lp"].abs().nan_to_num(0, 0, 0))
    near(got.entropy, ref["ent"], dl * (1 + math.log(K)))
    if topk:
        assert torch.equal(got.top_index.cpu(), ref["idx"])
        near(got.top_log_prob, ref["top"], dl[:, None] + U32 * ref["top"].abs().nan_to_num(0, 0, 0))
    if grads:
        dx = ops.logprob_bwd(xd, got, targets=cu(tgt), center=cu(c), temp=temp, dlog_prob=cu(dlp), dentropy=cu(dent),
                             dtop_log_prob=cu(dtop))
        assert dx.dtype == x.dtype and dx.shape == x.shape
        half = torch.finfo(x.dtype).eps / 2
        # p is off by dl relative, log p and H inside by dl absolute; fp32 sums of the T + topk gradients
        tol = ref["mag"] * (dl[:, None] + (T + topk + 4) * U32) + 2 * dl[:, None] * (1 + math.log(K)) * (
            dent.abs().double()[:, None] * ref["zs"].exp() / temp).nan_to_num(0) + half * ref["dx"].abs() + 1e-37
        near(dx, ref["dx"], tol.nan_to_num(0))
    return got


# every variant of the kernel (one wave, 1 to 8 vectors; one chunk; many chunks), ends inside a vector
SIZES = [(1, 1), (3, 2), (5, 9), (4, 65), (7, 512), (2, 777), (3, 1025), (2, 2047), (3, 4096), (2, 4097), (5, 8191),
         (1, 16385), (2, 65536), (9, 65537), (1, 100003), (3, 9000), (2, 16384),
         (2, 524289), (1, 1048576), (70001, 33)]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R,K", SIZES)
def test_matches_the_definition(R, K, dtype):
    x, tgt, c, g = make(R, K, dtype, 2, R * 7 + K)
    check(x, tgt, c, 0.04, min(K, 5), g)
    check(x, tgt, None, 1.0, min(K, 64), g)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R,K", [(6, 9), (7, 700), (6, 4097), (6, 70001)])
def test_masked_and_empty_rows(R, K, dtype):
    x, tgt, c, g = make(R, K, dtype, 3, K, masked=True)
    for topk in (1, min(K, 9)):
        check(x, tgt, c, 0.1, topk, g)


@gpu
@pytest.mark.parametrize("K", [300, 20000])
def test_rows_masked_by_the_lowest_value(K):
    x, tgt, _, g = make(4, K, torch.float32, 1, 5)
    low = torch.finfo(torch.float32).min
    x[0, : K // 2] = low
    x[1] = low                                       # all equal: a uniform row, not an empty one
    x[2, 1:] = low
    got = check(x, tgt, None, 0.04, 4, g)
    assert abs(got.entropy[1].item() - math.log(K)) < 1e-5 and got.entropy[2].item() == 0.0


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K", [300, 20000])
@pytest.mark.parametrize("base", [-1e9, 3e7, 1e20, -1e33])
def test_rows_far_from_zero(base, K, dtype):
    """A finite mask value in every column, or in all but one, and values that differ in their last bit only: what counts
    is the distance to the row's largest.  The temperature is a power of two, so z of the definition is exact."""
    low = torch.tensor(base, dtype=dtype)
    high = torch.nextafter(low, torch.tensor(math.inf, dtype=dtype))
    x = low.repeat(4, K)
    x[1, K // 2:] = high
    x[2, K // 3] = high
    x[3, 5] = 0.25
    tgt = torch.tensor([[0], [K - 1], [K // 3], [5]])
    g = torch.Generator().manual_seed(K)
    got = check(x, tgt, None, 2.0 ** -5, 3, g)
    assert abs(got.entropy[0].item() - math.log(K)) < 1e-5


@gpu
@pytest.mark.parametrize("K", [200, 5000, 70000])
def test_nan_and_infinity_stay_in_their_row(K):
    x, tgt, c, g = make(6, K, torch.float32, 1, 6)
    x[1, K // 3] = math.nan
    x[3, K - 1] = math.inf
    x[4] = NEG
    x[4, 0] = math.nan
    got = ops.logprob_fwd(x.cuda(), tgt.cuda(), center=c.cuda(), temp=0.1, topk=3)
    dx = ops.logprob_bwd(x.cuda(), got, targets=tgt.cuda(), center=c.cuda(), temp=0.1,
                         dlog_prob=torch.ones(6, 1, device="cuda"))
    bad = torch.tensor([False, True, False, True, True, False])
    for t in (got.log_prob[:, 0], got.entropy, got.top_log_prob[:, 0], dx[:, 1]):
        assert torch.equal(torch.isnan(t).cpu(), bad)
    assert got.top_index[1, 0] == K // 3 and got.top_index[3, 0] == K - 1 and got.top_index[4, 0] == 0
    fine = [0, 2, 5]
    ref = reference(x[fine], tgt[fine], c, 0.1, 3)
    assert torch.equal(got.top_index[fine].cpu(), ref["idx"])


@gpu
@pytest.mark.parametrize("K", [100, 4096, 40000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ties_go_to_the_lowest_index(K, dtype):
    x = torch.zeros(5, K, dtype=dtype)
    x[1, K // 2:] = 1.0
    x[2, ::3] = -0.0                                 # equal to +0
    x[3] = torch.arange(K).remainder(3).to(dtype)
    x[4] = NEG
    x[4, K - 3:] = 2.0
    got = ops.logprob_fwd(x.cuda(), None, topk=min(K, 64))
    want = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, : min(K, 64)]
    assert torch.equal(got.top_index.cpu(), want)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("order", [1, -1])
def test_sorted_rows(dtype, order):
    x = (torch.arange(30000) * (order * 1e-4)).repeat(2, 1).to(dtype)
    got = ops.logprob_fwd(x.cuda(), None, topk=20)
    want = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :20]
    assert torch.equal(got.top_index.cpu(), want)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("off,pad", [(0, 8), (1, 3), (7, 13)])
def test_strided_rows_of_any_alignment(dtype, off, pad):
    R, K = 5, 5003
    x, tgt, c, g = make(R, K, dtype, 2, 11)
    wide = torch.full((R, K + off + pad), 77.0, dtype=dtype, device="cuda")
    wide[:, off:off + K] = x.cuda()
    view = wide[:, off:off + K]
    check(view, tgt, c, 0.1, 4, g)
    out = torch.full_like(wide, 55.0)
    got = ops.logprob_fwd(view, tgt.cuda(), temp=0.1)
    ops.logprob_bwd(view, got, targets=tgt.cuda(), temp=0.1, dentropy=torch.ones(R, device="cuda"),
                    dlogits=out[:, off:off + K])
    assert (out[:, :off] == 55).all() and (out[:, off + K:] == 55).all()      # nothing beside the rows is written


@gpu
def test_repeated_targets_add_up_and_absent_ones_count_nothing():
    x, _, c, g = make(3, 1000, torch.float32, 1, 3)
    tgt = torch.tensor([[5, 5, 5, -1], [7, 999, 7, 0], [-1, -1, -1, -1]])
    check(x, tgt, c, 0.1, 3, g)
    got = ops.logprob_fwd(x.cuda(), tgt.cuda(), temp=0.1)
    dx = ops.logprob_bwd(x.cuda(), got, targets=tgt.cuda(), temp=0.1, dlog_prob=torch.ones(3, 4, device="cuda"))
    assert (dx[2] == 0).all() and (got.log_prob[2] == 0).all()


@gpu
def test_targets_outside_the_columns_give_nan_and_no_gradient():
    x, _, _, _ = make(2, 300, torch.float32, 1, 3)
    tgt = torch.tensor([[300, 1], [-2, 2 ** 40]])
    got = ops.logprob_fwd(x.cuda(), tgt.cuda())
    assert torch.isnan(got.log_prob).cpu().tolist() == [[True, False], [True, True]]
    dx = ops.logprob_bwd(x.cuda(), got, targets=tgt.cuda(), dlog_prob=torch.ones(2, 2, device="cuda"))
    assert torch.isfinite(dx).all() and (dx[1] == 0).all()


@gpu
def test_many_targets_no_targets_no_rows():
    x, _, c, g = make(2, 9000, torch.bfloat16, 1, 4)
    tgt = torch.randint(0, 9000, (2, 1000), generator=g)
    check(x, tgt, c, 0.1, 0, g)
    got = ops.logprob_fwd(x.cuda(), None, topk=2)
    assert got.log_prob.shape == (2, 0)
    got = ops.logprob_fwd(torch.empty(0, 9000, device="cuda"), torch.empty(0, 1, dtype=torch.int64, device="cuda"), topk=2)
    assert got.entropy.shape == (0,) and got.top_index.shape == (0, 2)
    dx = ops.logprob_bwd(torch.empty(0, 9000, device="cuda"), got, dentropy=torch.empty(0, device="cuda"))
    assert dx.shape == (0, 9000)


@gpu
def test_offsets_past_32_bits():
    """bf16 rows whose elements lie beyond 2^32 bytes and 2^31 elements."""
    R, K = 34000, 65536
    x = torch.zeros((R, K), dtype=torch.bfloat16, device="cuda")
    x[-1, 12345] = 3.0
    tgt = torch.full((R, 1), 12345, dtype=torch.int64, device="cuda")
    got = ops.logprob_fwd(x, tgt, topk=1)
    want = 3.0 - math.log(K - 1 + math.exp(3.0))
    assert abs(got.log_prob[-1, 0].item() - want) < 1e-5 and got.top_index[-1, 0] == 12345
    assert abs(got.log_prob[0, 0].item() + math.log(K)) < 1e-5
    ops.logprob_bwd(x, got, targets=tgt, dlog_prob=torch.ones(R, 1, device="cuda"), dlogits=x)     # in place
    assert abs(x[-1, 12345].item() - (1 - math.exp(want))) < 4e-3 and x[-1, 0].item() < 0


@gpu
def test_gradient_against_differences():
    g = torch.Generator().manual_seed(9)
    x = torch.randn(2, 37, generator=g)
    c = torch.randn(37, generator=g) * 0.1
    tgt = torch.tensor([[3, 36], [0, 3]])
    w = torch.randn(2, 2, generator=g)
    v = torch.randn(2, generator=g)
    got = ops.logprob_fwd(x.cuda(), tgt.cuda(), center=c.cuda(), temp=0.5)
    dx = ops.logprob_bwd(x.cuda(), got, targets=tgt.cuda(), center=c.cuda(), temp=0.5, dlog_prob=w.cuda(),
                         dentropy=v.cuda()).cpu().double()

    def f(x64):
        lp = torch.log_softmax((x64 - c.double()) / 0.5, 1)
        return (lp.gather(1, tgt) * w).sum() - ((lp.exp() * lp).sum(1) * v).sum()
    h = 1e-5
    for r in range(2):
        for k in range(37):
            e = torch.zeros(2, 37, dtype=torch.float64)
            e[r, k] = h
            num = (f(x.double() + e) - f(x.double() - e)) / (2 * h)
            assert abs(num.item() - dx[r, k].item()) < 2e-5        # h^2 f''' and the kernel's fp32, both below 1e-5


@gpu
def test_side_stream_and_two_graphs():
    """Two captured graphs (each with its own workspace) and eager calls between their replays."""
    xs = [make(3, 20000, torch.bfloat16, 1, s)[0].cuda() for s in (1, 2)]
    tgt = torch.tensor([[5], [6], [7]], device="cuda")
    ones = torch.ones(3, 1, device="cuda")
    want = [ops.logprob_fwd(x, tgt, temp=0.1, topk=4) for x in xs]
    wdx = [ops.logprob_bwd(x, w, targets=tgt, temp=0.1, dlog_prob=ones) for x, w in zip(xs, want)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.logprob_fwd(xs[0], tgt, temp=0.1, topk=4)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got.entropy, want[0].entropy)
    graphs, outs = [], []
    for x in xs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            r = ops.logprob_fwd(x, tgt, temp=0.1, topk=4)
            dx = ops.logprob_bwd(x, r, targets=tgt, temp=0.1, dlog_prob=ones)
        graphs.append(gr)
        outs.append((r, dx))
    for _ in range(3):
        for gr in graphs:
            gr.replay()
        ops.logprob_fwd(xs[0], tgt, temp=0.1, topk=4)
        torch.cuda.synchronize()
        for (r, dx), w, v in zip(outs, want, wdx):
            assert torch.equal(r.log_prob, w.log_prob) and torch.equal(r.top_index, w.top_index)
            assert torch.equal(r.entropy, w.entropy) and torch.equal(dx, v)


def test_refusals_on_the_cpu(monkeypatch):
    x = torch.zeros(2, 9)
    with pytest.raises(DinoHipError):
        ops.logprob_fwd(x)                                          # no CPU path
    monkeypatch.setattr(ops, "_dev", lambda *a: None)               # the checks behind it, without a GPU
    i64 = torch.int64
    bad = [
        dict(targets=torch.zeros(2, dtype=i64)), dict(targets=torch.zeros(3, 1, dtype=i64)),
        dict(targets=torch.zeros(2, 1, dtype=torch.int32)), dict(targets=torch.zeros(2, 5000, dtype=i64)),
        dict(center=torch.zeros(8)), dict(center=torch.zeros(9, dtype=torch.bfloat16)),
        dict(temp=0.0), dict(temp=-1.0), dict(temp=math.nan), dict(temp=math.inf), dict(temp=1e-39),
        dict(topk=10), dict(topk=-1), dict(topk=1.5),
    ]
    for kw in bad:
        with pytest.raises(DinoHipError):
            ops.logprob_fwd(x, **kw)
    with pytest.raises(DinoHipError):
        ops.logprob_fwd(torch.zeros(2, 200), topk=65)
    for odd in (torch.zeros(9), torch.zeros(2, 9, 1), torch.zeros(9, 2).t(), torch.zeros(2, 0), torch.zeros(1, 9).expand(2, 9)):
        with pytest.raises(DinoHipError):
            ops.logprob_fwd(odd)


def test_backward_refusals_on_the_cpu(monkeypatch):
    monkeypatch.setattr(ops, "_dev", lambda *a: None)
    i64, bf = torch.int64, torch.bfloat16
    x, tgt = torch.zeros(2, 9), torch.zeros(2, 1, dtype=i64)
    r = ops.LogProbs(torch.zeros(2, 1), torch.zeros(2), torch.zeros(2, 2), torch.zeros(2, 3), torch.zeros(2, 3, dtype=i64))
    bad = [
        dict(dlog_prob=torch.zeros(2, 1)), dict(targets=tgt, dlog_prob=torch.zeros(2, 2)),
        dict(targets=tgt, dlog_prob=torch.zeros(2, 1, dtype=bf)), dict(dentropy=torch.zeros(3)),
        dict(dentropy=torch.zeros(2, dtype=torch.float64)), dict(dtop_log_prob=torch.zeros(2, 2)),
        dict(dtop_log_prob=torch.zeros(3, 2).t()), dict(dlogits=torch.zeros(2, 9, dtype=bf)), dict(dlogits=torch.zeros(2, 8)),
        dict(dlogits=torch.zeros(9, 2).t()), dict(dlogits=torch.zeros(1, 9).expand(2, 9)), dict(temp=0.0),
        dict(fwd=r._replace(stats=torch.zeros(3, 2))), dict(fwd=r._replace(entropy=torch.zeros(2, 1))),
        dict(fwd=r._replace(top_index=torch.zeros(2, 3, dtype=torch.int32))),
        dict(fwd=r._replace(top_index=None, top_log_prob=None), dtop_log_prob=torch.zeros(2, 3)),
    ]
    for kw in bad:
        with pytest.raises(DinoHipError):
            ops.logprob_bwd(x, kw.pop("fwd", r), **kw)


def test_entry_points_refuse_bad_arguments():
    import ctypes

    from dino_amd import _lib
    lib = _lib.load()
    n = ctypes.c_int64(0)
    assert lib.dino_logprob_workspace(4, 1 << 21, 0, ctypes.byref(n)) == -3
    assert lib.dino_logprob_workspace(4, 10, 11, ctypes.byref(n)) == -1
    assert lib.dino_logprob_workspace(4, 100, 65, ctypes.byref(n)) == -1
    assert lib.dino_logprob_workspace(4, 65536, 8, ctypes.byref(n)) == 0 and n.value > 0
    # a missing pointer, an unknown type, a short stride, a short workspace: refused before any launch
    one = ctypes.c_void_p(16)
    def fwd(dtype=0, x=one, ld=65536, K=65536, inv=1.0, T=1, tg=one, ws=None, wsb=0):
        return lib.dino_logprob_fwd(dtype, x, ld, 4, K, None, inv, tg, T, 0, one, one, one, None, None, ws, wsb, None)
    assert fwd() == -1 and fwd(dtype=2) == -1 and fwd(x=None) == -1 and fwd(ld=5) == -1 and fwd(tg=None) == -1
    assert fwd(inv=0.0) == -1 and fwd(inv=float("nan")) == -1 and fwd(K=1 << 21, ld=1 << 21) == -3 and fwd(ws=one, wsb=8) == -1
