"""Orthogonalised updates (ops.orthogonalize) against the Newton-Schulz recurrence in 64 bits, and their refusals."""
import ctypes
import math

import pytest
import torch

from dino_amd import _lib, ops
from dino_amd._lib import DinoHipError

gpu = pytest.mark.gpu
NS = ops.NS_COEFFS
SPLIT_ABOVE = 16.0


def recurrence(u, steps=5, coeffs=NS, eps=1e-7):
    """(result, tolerance) in 64 bits on the CPU.  The tolerance is on the Frobenius norm of the difference.

    A step rounds X, A and B to fp16 (half a step: 2^-11 of an element).  X's rounding is multiplied by the later steps, by
    at most the product of their a (derivative at 0, the largest); while that is above 8 X is a pair of fp16 (2^-22), so the
    limit of 16 below allows more than is used.  A's and B's multiply X from the left and stay relative to it.  Counted here:
    three roundings of rms half / sqrt(3) a step, all growing, of a whole fp16 from a growth of 16 down, of 2^-20 before.
    Independent roundings add in squares; three times that is allowed.  The bf16 result adds half a step, 2^-8, of itself.
    fp32 sums of K terms stay below 2^-24 sqrt(K), less than 2^-20 for the sizes here."""
    x = u.double()
    x = x / (torch.linalg.vector_norm(x) + eps)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    cs = [coeffs] * steps if not isinstance(coeffs[0], (tuple, list)) else list(coeffs)
    grow = [math.prod(max(1.0, abs(c[0])) for c in cs[s + 1:]) for s in range(steps)]
    var = 0.0
    for (a, b, c), g in zip(cs, grow):
        half = 2.0 ** -20 if g > SPLIT_ABOVE else 2.0 ** -11
        mag = max(1.0, abs(a), abs(b) / 2, abs(c))
        var += 3 * (half / math.sqrt(3) * g * mag * torch.linalg.vector_norm(x).item()) ** 2
        q = x @ x.T
        x = a * x + (b * q + c * (q @ q)) @ x
    x = x.T if tall else x
    return x, 3 * math.sqrt(var) + 2.0 ** -8 * torch.linalg.vector_norm(x).item()


def momentum(shape, seed, kind="momentum"):
    g = torch.Generator().manual_seed(seed)
    r, c = shape[-2:]
    if kind == "noise":
        return torch.randn(*shape, generator=g)
    k = max(1, min(r, c, 4))
    lead = shape[:-2]
    u = torch.randn(*lead, r, k, generator=g) @ torch.randn(*lead, k, c, generator=g)
    return (u + 0.1 * torch.randn(*shape, generator=g)) * 1e-3


def off(got, u, **kw):
    want, tol = recurrence(u.cpu(), **kw)
    d = torch.linalg.vector_norm(got.detach().cpu().double() - want).item()
    assert d <= tol, (d, tol, d / max(torch.linalg.vector_norm(want).item(), 1e-30))
    return d / max(torch.linalg.vector_norm(want).item(), 1e-30)


SHAPES = [(1, 1), (1, 300), (300, 1), (2, 3), (31, 33), (32, 32), (64, 65), (77, 65), (128, 128), (129, 127), (192, 192),
          (251, 1000), (1000, 251), (384, 384), (384, 1536), (1536, 384), (588, 300)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind", ["momentum", "noise"])
def test_matches_the_recurrence(shape, dtype, kind):
    u = momentum(shape, shape[0] * 3 + shape[1], kind).to(dtype)
    got = ops.orthogonalize(u.cuda())
    assert got.dtype == torch.bfloat16 and got.shape == u.shape
    off(got, u)


@gpu
def test_many_items_in_one_call():
    shapes = [(3, 96, 200), (40, 70), (1, 130, 33), (2, 256, 256), (0, 50, 60)] + [(17 + i, 40) for i in range(40)]
    ups = [momentum(s, i).to(torch.float32 if i % 3 else torch.bfloat16) for i, s in enumerate(shapes)]
    got = ops.orthogonalize([u.cuda() for u in ups])
    assert isinstance(got, list) and len(got) == len(ups)
    for u, o in zip(ups, got):
        assert o.shape == u.shape
        for a, b in zip(u.reshape(-1, *u.shape[-2:]), o.reshape(-1, *o.shape[-2:])):
            off(b, a)
    again = ops.orthogonalize([u.cuda() for u in ups])
    assert all(torch.equal(a, b) for a, b in zip(got, again))            # no schedule in the result


@gpu
@pytest.mark.parametrize("shape", [(25, 1000, 1030), (25, 1030, 1000)])
def test_large_tiles_with_tiny_matrices_beside_them(shape):
    """Enough work for the 256 x 256 tiles, which then also take matrices that fill a corner of one."""
    big = momentum(shape, 11)
    small = [momentum((3, 5, 7), 1), momentum((2, 64, 300), 2), momentum((65, 1), 3)]
    got = ops.orthogonalize([big.cuda()] + [u.cuda() for u in small])
    for i in (0, 24):
        off(got[0][i], big[i])
    for u, o in zip(small, got[1:]):
        for a, b in zip(u.reshape(-1, *u.shape[-2:]), o.reshape(-1, *o.shape[-2:])):
            off(b, a)
    again = ops.orthogonalize(big.cuda())
    assert torch.equal(again, got[0])


@gpu
@pytest.mark.parametrize("steps", [1, 2, 3, 5, 7])
def test_steps_and_coefficients(steps):
    u = momentum((100, 180), 5)
    off(ops.orthogonalize(u.cuda(), steps=steps), u, steps=steps)
    off(ops.orthogonalize(u.cuda(), steps=steps, coeffs=(1.5, -0.5, 0.0)), u, steps=steps, coeffs=(1.5, -0.5, 0.0))
    cs = [(4.0, -6.0, 2.7)] * (steps - 1) + [(1.875, -1.25, 0.375)]
    if steps < 3:
        off(ops.orthogonalize(u.cuda(), steps=steps, coeffs=cs), u, steps=steps, coeffs=cs)
    else:   # 0.55 -> 1.34 -> 2.66 -> 33 (steps = 3) and on from there: past the 12 that fp16 has room for, refused
        with pytest.raises(DinoHipError):
            ops.orthogonalize(u.cuda(), steps=steps, coeffs=cs)
    cs = [NS] * (steps - 1) + [(1.875, -1.25, 0.375)]
    off(ops.orthogonalize(u.cuda(), steps=steps, coeffs=cs), u, steps=steps, coeffs=cs)


@gpu
@pytest.mark.parametrize("scale", [1e-30, 1e-9, 1e25])
def test_scale_of_the_update(scale):
    """The squares of 1e-30 and 1e25 do not fit fp32: the norm is summed in 64 bits.  eps is part of the formula."""
    u = momentum((60, 90), 2, "noise") * scale
    off(ops.orthogonalize(u.cuda(), eps=0.0), u, eps=0.0)
    off(ops.orthogonalize(u.cuda()), u)


@gpu
@pytest.mark.parametrize("shape", [(4, 1000, 1030), (4, 1030, 1000), (2, 1000, 1030), (10, 450, 1500)])
def test_middle_tiles_with_tiny_matrices_beside_them(shape):
    """Enough work for the 128 x 128 tiles (and, for the last, 64 x 64 ones beside them)."""
    big = momentum(shape, 12)
    small = [momentum((3, 5, 7), 1), momentum((65, 129), 3)]
    got = ops.orthogonalize([big.cuda()] + [u.cuda() for u in small])
    for i in (0, shape[0] - 1):
        off(got[0][i], big[i])
    for u, o in zip(small, got[1:]):
        for a, b in zip(u.reshape(-1, *u.shape[-2:]), o.reshape(-1, *o.shape[-2:])):
            off(b, a)
    assert torch.equal(ops.orthogonalize(big.cuda()), got[0])


@gpu
@pytest.mark.parametrize("shape", [(32704, 32768), (32768, 16400)])
def test_largest_matrices(shape):
    """Offsets up to the last byte that a matrix may have (2^31).  Zeros but for blocks in the corners and between: rows and
    columns of zeros stay zeros, and every block takes the recurrence from its part of the whole norm."""
    r, c = shape
    at = [(0, 0), (r // 2 + 3, c // 3 + 1), (r - 90, c - 120)]
    u = torch.zeros(shape, device="cuda")
    blocks = [momentum((90, 120), 60 + i, "noise") for i in range(3)]
    for (y, x), b in zip(at, blocks):
        u[y:y + 90, x:x + 120] = b.cuda()
    got = ops.orthogonalize(u)
    whole = math.sqrt(sum(b.double().square().sum().item() for b in blocks))
    inside = 0
    for (y, x), b in zip(at, blocks):
        o = got[y:y + 90, x:x + 120]
        inside += torch.count_nonzero(o).item()
        off(o, b, eps=whole - torch.linalg.vector_norm(b.double()).item() + 1e-7)
    assert torch.count_nonzero(got).item() == inside > 0


@gpu
@pytest.mark.parametrize("scale,eps", [(1e-38, 0.0), (1e-41, 0.0), (1e-41, 1e-40), (1e-10, 1e20), (1e-3, 1e29)])
def test_norms_at_the_end_of_the_range(scale, eps):
    """1 / |U| is past fp32's range, or |U| / eps far below fp16's."""
    u = momentum((60, 90), 4, "noise") * scale
    off(ops.orthogonalize(u.cuda(), eps=eps), u, eps=eps)
    off(ops.orthogonalize(u.t().contiguous().cuda(), eps=eps), u.t().contiguous(), eps=eps)


@gpu
def test_zeros_and_bad_numbers_stay_in_their_matrix():
    u = momentum((5, 70, 90), 3).cuda()
    clean = ops.orthogonalize(u)
    v = u.clone()
    v[1] = 0
    v[2, 3, 4] = math.nan
    v[3, 69, 89] = math.inf
    got = ops.orthogonalize(v)
    assert torch.equal(got[0], clean[0]) and torch.equal(got[4], clean[4])
    assert (got[1] == 0).all() and torch.isnan(got[2]).any() and torch.isnan(got[3]).any()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_inputs_and_outputs(dtype):
    u = momentum((3, 50, 77), 4).to(dtype)
    wide = torch.full((3, 53, 91), 7.0, dtype=dtype, device="cuda")
    wide[:, 1:51, 5:82] = u.cuda()
    out = torch.full((4, 60, 83), 9.0, dtype=torch.bfloat16, device="cuda")
    view = out[1:, 2:52, 3:80]
    got = ops.orthogonalize(wide[:, 1:51, 5:82], out=view)
    assert got.data_ptr() == view.data_ptr()
    for a, b in zip(u, got):
        off(b, a)
    out[1:, 2:52, 3:80] = 9.0
    assert (out == 9.0).all()                               # nothing beside the matrices was written
    t = momentum((77, 50), 6).to(dtype)
    b = torch.empty((77, 64), dtype=dtype, device="cuda")
    b[:, :50] = t.cuda()
    off(ops.orthogonalize(b[:, :50]), t)


@gpu
def test_in_place_over_a_bf16_update():
    u = momentum((96, 160), 7).to(torch.bfloat16)
    d = u.cuda()
    ops.orthogonalize(d, out=d)
    off(d, u)


@gpu
def test_singular_values_end_near_one():
    u = torch.randn(200, 320, generator=torch.Generator().manual_seed(1)) @ torch.diag(torch.logspace(0, -1, 320))
    s = torch.linalg.svdvals(ops.orthogonalize(u.cuda()).float().cpu())
    assert 0.6 < s.min() and s.max() < 1.25


@gpu
def test_side_stream_and_two_graphs():
    us = [momentum((2, 130, 200), s).cuda() for s in (1, 2)]
    want = [ops.orthogonalize(u) for u in us]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.orthogonalize(us[0])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want[0])
    graphs, outs = [], []
    for u in us:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.orthogonalize(u))
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
        ops.orthogonalize(us[1])
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)


def test_refusals_on_the_cpu(monkeypatch):
    with pytest.raises(DinoHipError):
        ops.orthogonalize(torch.zeros(4, 4))                # no CPU path
    monkeypatch.setattr(ops, "_dev", lambda *a: None)
    monkeypatch.setattr(ops, "_on", lambda d: ops._NO_GUARD)
    u = torch.zeros(4, 6)
    for kw in (dict(steps=0), dict(steps=17), dict(steps=2.0), dict(coeffs=(1.0, 2.0)), dict(coeffs=[(1, 2, 3)] * 4),
               dict(eps=-1.0), dict(eps=math.nan), dict(out=torch.zeros(4, 6)), dict(out=torch.zeros(6, 4, dtype=torch.bfloat16))):
        with pytest.raises(DinoHipError):
            ops.orthogonalize(u, **kw)
    for bad in (torch.zeros(4), torch.zeros(2, 2, 2, 2), torch.zeros(6, 4).t(), torch.zeros(1, 6).expand(4, 6),
                torch.zeros(1, 4, 6).expand(3, 4, 6), torch.zeros(0, 6)):
        with pytest.raises(DinoHipError):
            ops.orthogonalize(bad)
    with pytest.raises(TypeError):
        ops.orthogonalize(torch.zeros(4, 6, dtype=torch.float16))
    with pytest.raises(DinoHipError):
        ops.orthogonalize([u, u], out=[torch.zeros(4, 6, dtype=torch.bfloat16)])
    twice = torch.zeros(4, 6, dtype=torch.bfloat16)
    with pytest.raises(DinoHipError):
        ops.orthogonalize([u, u], out=[twice, twice])
    assert ops.orthogonalize([]) == []


def test_entry_point_refuses_bad_arguments():
    lib = _lib.load()
    n = ctypes.c_int64(0)

    def item(rows=4, cols=6, batch=1, dtype=0, ld=6):
        it = (_lib.OrthoItem * 1)()
        it[0].inp = it[0].out = 4096
        it[0].rows, it[0].cols, it[0].batch, it[0].dtype, it[0].in_ld, it[0].out_ld = rows, cols, batch, dtype, ld, ld
        return it
    assert lib.dino_ortho_workspace(item(), 1, ctypes.byref(n)) == 0 and n.value > 0
    assert lib.dino_ortho_workspace(item(rows=0), 1, ctypes.byref(n)) == -1
    assert lib.dino_ortho_workspace(item(dtype=3), 1, ctypes.byref(n)) == -1
    assert lib.dino_ortho_workspace(item(rows=40000, cols=4), 1, ctypes.byref(n)) == -3
    assert lib.dino_ortho_workspace(item(rows=32768, cols=32768), 1, ctypes.byref(n)) == -3
    assert lib.dino_ortho_workspace(item(batch=1 << 25), 1, ctypes.byref(n)) == -3
    c = (ctypes.c_float * 48)(*([3.4445, -4.7750, 2.0315] * 16))
    ws = ctypes.c_void_p(1 << 20)
    big = 1 << 40

    def run(it, steps=5, coeffs=c, eps=1e-7, w=ws, nb=big):
        return lib.dino_ortho(it, 1, steps, coeffs, eps, w, nb, None)
    assert run(item(), steps=0) == -1 and run(item(), steps=17) == -1 and run(item(), eps=-1.0) == -1
    assert run(item(), w=None) == -1 and run(item(), nb=16) == -1 and run(item(), w=ctypes.c_void_p(8)) == -1
    assert run(item(ld=5)) == -1
    wild = (ctypes.c_float * 15)(*([20.0, 0.0, 0.0] * 5))
    assert run(item(), coeffs=wild) == -1                    # singular values past what fp16 holds
    nan = (ctypes.c_float * 15)(*([math.nan, 0.0, 0.0] * 5))
    assert run(item(), coeffs=nan) == -1
    assert lib.dino_ortho(None, 0, 5, c, 1e-7, None, 0, None) == 0
