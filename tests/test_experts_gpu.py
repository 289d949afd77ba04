"""Routed experts on the GPU against plain forms in 64 bits.

Tolerances: an output of 16 bits is rounded once (half a step, ``eps / 2`` of the value); a sum of n products held
in fp32 is off by at most n steps of 2^-23 of the sum of their magnitudes (the tensor cores may truncate, so a whole
step for each addition).  Both are computed per element."""
import math

import pytest
import torch

from flare_b200._native import default_status
from flare_b200.models.layers import BatchedExpertMoE, TokenMixLargeMoe
from flare_b200.ops.experts import (MAX_EXPERTS, MAX_GROUPS, ExpertRoute, combine_rows, combine_rows_reference,
                                    e4m3_checkpoint_reference, expert_mlp, grouped_linear, route_topk, route_topk_reference, swiglu)
from test_experts import check_route, hard_logits

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def within(got, want, slack, note=""):
    """|got - want| <= half a step of got's type + slack, elementwise (``want`` in 64 bits)."""
    fi = torch.finfo(got.dtype)
    off = (got.double() - want).abs() - (fi.eps / 2 * want.abs() + fi.smallest_normal * fi.eps + slack)
    assert not got.isnan().any(), note
    assert bool((off <= 0).all()), f"{note}: {off.max().item():.3g} over at {(off > 0).double().mean().item():.3g} of the values"


# -------------------------------------------------------------------- routing
@pytest.mark.parametrize("S,B,E,k,dtype", [
    (1, 1, 1, 1, FP32), (1, 3, 8, 8, BF16), (1, 255, 9, 2, FP16), (1, 512, 16, 3, FP32), (1, 513, 17, 3, BF16),
    (2, 1, 5, 2, FP32), (3, 300, 33, 4, FP32), (1, 700, 65, 2, BF16), (1, 600, 129, 2, FP32), (2, 40, 257, 32, BF16),
    (1, 20, MAX_EXPERTS, 32, FP32), (300, 3, 4, 1, FP32)])
def test_route(cuda, S, B, E, k, dtype):
    lg = hard_logits(S, B, E, S + B + E, dtype)
    leaf = lg.to(cuda).requires_grad_(True)
    route = route_topk(leaf, k)
    check_route(ExpertRoute(*(t.detach().cpu() for t in route)), lg, k)
    ref = lg.double().requires_grad_(True)
    want = route_topk_reference(ref, k)
    # exponentials within 2 steps, k additions and one division
    within(route.weights.cpu(), want.weights, (k + 6) * 2 ** -23 * want.weights.detach())
    g = torch.randn(want.weights.shape, dtype=torch.float64, generator=torch.Generator().manual_seed(1)).float()
    route.weights.backward(g.to(cuda))
    want.weights.backward(g.double())
    slack = 4 * (k + 6) * 2 ** -23 * g.abs().max().item()
    within(leaf.grad.cpu(), ref.grad, slack)


def test_route_large_matches_plain(cuda):
    lg = torch.randn(2, 40000, 60, device=cuda).to(BF16)
    lg[:, 30000:] = -math.inf
    a, b = route_topk(lg, 3), route_topk_reference(lg, 3)
    for n in ("experts", "offsets", "rows", "row_of"):
        assert torch.equal(getattr(a, n), getattr(b, n)), n


def test_route_views_and_repeats(cuda):
    big = torch.randn(50, 3, 40, device=cuda)
    view = big.transpose(0, 1)[:, ::2, 3:20]  # slots of other strides, unit inner stride
    assert view.stride(2) == 1 and not view.is_contiguous()
    a, b = route_topk(view, 2), route_topk(view.contiguous(), 2)
    c = route_topk(big.permute(1, 2, 0)[:, :, :17], 2)  # inner stride not 1: copied
    for u, v in zip(a, b):
        assert torch.equal(u, v)
    check_route(ExpertRoute(*(t.cpu() for t in c)), big.permute(1, 2, 0)[:, :, :17].cpu(), 2)


def test_route_nan_and_infinity(cuda):
    lg = torch.tensor([[0.0, math.nan, 3.0, math.inf], [math.inf, 1.0, -math.inf, math.inf], [-math.nan, 0.0, 0.0, 9.0]], device=cuda)
    r = route_topk(lg, 2)
    assert r.experts.tolist() == [[1, 3], [0, 3], [0, 3]] and r.weights.isnan().all()


# ------------------------------------------------------------ grouped products
def offsets_of(sizes, before, cuda):
    return torch.tensor([before] + [before + sum(sizes[:i + 1]) for i in range(len(sizes))], dtype=torch.int32, device=cuda)


def exact_linear(x, w, b, off, dy, rows=None):
    """Values and the sums of magnitudes that bound them: y, dx (of the rows), dw, db."""
    off = off.tolist()
    R = dy.shape[0]
    xd, wd, dyd = x.double(), w.double(), dy.double()
    xr = xd if rows is None else xd[rows.long().clamp(min=0)]
    y, ay = torch.zeros(R, w.shape[2], dtype=torch.float64, device=x.device), torch.zeros(R, w.shape[2], dtype=torch.float64, device=x.device)
    dx, ax = torch.zeros_like(xr), torch.zeros_like(xr)
    dw, aw = torch.zeros_like(wd), torch.zeros_like(wd)
    db, ab = (torch.zeros(w.shape[0], w.shape[2], dtype=torch.float64, device=x.device) for _ in range(2))
    for g in range(w.shape[0]):
        lo, hi = off[g], off[g + 1]
        if hi > lo:
            a, d = xr[lo:hi], dyd[lo:hi]
            bias = b[g].double() if b is not None else torch.zeros(w.shape[2], dtype=torch.float64, device=x.device)
            y[lo:hi], ay[lo:hi] = a @ wd[g] + bias, a.abs() @ wd[g].abs() + bias.abs()
            dx[lo:hi], ax[lo:hi] = d @ wd[g].t(), d.abs() @ wd[g].abs().t()
            dw[g], aw[g] = a.t() @ d, a.abs().t() @ d.abs()
            db[g], ab[g] = d.sum(0), d.abs().sum(0)
    return (y, ay), (dx, ax), (dw, aw), (db, ab)


SIZES = {
    "one row": [1],
    "one each": [1] * 9,
    "empty ends": [0, 5, 0, 0, 130, 1, 0],
    "one tile": [128, 128],
    "past a tile": [129, 127, 257],
    "large": [700, 1, 900, 0, 333],
    "many small": [(i * 7) % 5 for i in range(300)],
    "more than are sorted": [(i * 5) % 4 for i in range(600)],
    "long, sums in chunks": [1, 4095, 0, 5000, 32, 100, 0],
}


@pytest.mark.parametrize("K,N,dtype", [(8, 8, BF16), (64, 64, FP16), (72, 136, BF16), (200, 328, FP16), (520, 264, BF16), (136, 1032, BF16)])
@pytest.mark.parametrize("sizes", list(SIZES))
def test_grouped_linear(cuda, sizes, K, N, dtype):
    gen = torch.Generator(device="cuda").manual_seed(K + N)
    sz = SIZES[sizes]
    before, after = (3, 70) if len(sz) > 2 else (0, 0)
    off = offsets_of(sz, before, cuda)
    R, G = before + sum(sz) + after, len(sz)
    x = torch.randn(R, K, device=cuda, generator=gen).to(dtype).requires_grad_(True)
    w = (torch.randn(G, K, N, device=cuda, generator=gen) / K ** 0.5).to(dtype).requires_grad_(True)
    b = torch.randn(G, N, device=cuda, generator=gen).to(dtype).requires_grad_(True)
    dy = torch.randn(R, N, device=cuda, generator=gen).to(dtype)
    y = grouped_linear(x, w, b, offsets=off)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    want = exact_linear(x.detach(), w.detach(), b.detach(), off, dy)
    for name, got, (v, mag), n in zip(("y", "dx", "dw", "db"), (y.detach(), dx, dw, db), want, (K + 1, N, max(sz), max(sz))):
        within(got, v, (n + 2) * 2 ** -23 * mag, name)
    out = torch.ones(R, dtype=torch.bool, device=cuda)
    out[before:before + sum(sz)] = False
    assert not y[out].any() and not dx[out].any()  # rows of no group
    default_status(cuda).check()


@pytest.mark.parametrize("T,S,E,k,K,N,dtype", [
    (1, 1, 4, 2, 64, 128, BF16), (3, 2, 5, 1, 40, 24, FP16), (130, 1, 3, 3, 136, 264, BF16), (1500, 1, 2, 2, 512, 320, BF16),
    (700, 3, 7, 2, 200, 96, FP16)])
def test_grouped_linear_gathered(cuda, T, S, E, k, K, N, dtype):
    gen = torch.Generator(device="cuda").manual_seed(T + K)
    lg = torch.randn(S, T, E, device=cuda, generator=gen)
    lg[torch.rand(S, T, E, device=cuda, generator=gen) < 0.2] = -math.inf
    route = route_topk(lg, k)
    x = torch.randn(S * T, K, device=cuda, generator=gen).to(dtype).requires_grad_(True)
    w = (torch.randn(S, E, K, N, device=cuda, generator=gen) / K ** 0.5).requires_grad_(True)  # float32 parameters
    b = torch.randn(S, E, N, device=cuda, generator=gen).requires_grad_(True)
    dy = torch.randn(S * T * k, N, device=cuda, generator=gen).to(dtype)
    y = grouped_linear(x, w, b, route=route)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert dw.dtype == FP32 and dw.shape == w.shape and db.shape == b.shape
    wq = w.detach().to(dtype).view(S * E, K, N)
    (y0, ay), (dr, ar), (dw0, aw), (db0, ab) = exact_linear(x.detach(), wq, b.detach().view(S * E, N), route.offsets, dy, route.rows)
    within(y.detach(), y0, (K + 3) * 2 ** -23 * ay, "y")
    flat = ExpertRoute(*route)
    dx0, ax = combine_rows_reference(dr, flat), combine_rows_reference(ar, flat)
    within(dx, dx0, (N + k + 2) * 2 ** -23 * ax, "dx")
    n = int((route.offsets[1:] - route.offsets[:-1]).max()) + 2
    within(dw, dw0.view_as(w), n * 2 ** -23 * aw.view_as(w), "dw")
    within(db, db0.view_as(b), n * 2 ** -23 * ab.view_as(b), "db")
    # with the same rows laid out by hand: the same bits
    laid = x.detach()[route.rows.long().clamp(min=0)]
    assert torch.equal(grouped_linear(laid, w, b, offsets=route.offsets).detach(), y.detach())


def test_grouped_linear_other_rows_stay_out(cuda):
    """Infinities and NaN of one group, of rows of no group, and of another group's weights reach nothing else."""
    sizes, K, N = [70, 3, 90, 40], 72, 40
    off = offsets_of(sizes, 5, cuda)
    R = 5 + sum(sizes) + 30
    x, dy = torch.randn(R, K, device=cuda).to(BF16), torch.randn(R, N, device=cuda).to(BF16)
    w = torch.randn(4, K, N, device=cuda).to(BF16)
    for clean in (0, 2):
        xs, ws, ds = x.clone(), w.clone(), dy.clone()
        lo, hi = off[clean].item(), off[clean + 1].item()
        keep = torch.zeros(R, dtype=torch.bool, device=cuda)
        keep[lo:hi] = True
        for t, bad in ((xs, math.nan), (ds, math.inf)):
            t[~keep] = bad
        for g in range(4):
            if g != clean:
                ws[g] = math.nan
        outs = []
        for a, b, d in ((x, w, dy), (xs, ws, ds)):
            a, b = a.clone().requires_grad_(True), b.clone().requires_grad_(True)
            y = grouped_linear(a, b, offsets=off)
            da, db = torch.autograd.grad(y, (a, b), d)
            outs.append((y[lo:hi].detach(), da[lo:hi], db[clean]))
        for u, v in zip(*outs):
            assert torch.equal(u, v)


def test_grouped_linear_views(cuda):
    """Strided, offset and misaligned operands give what their copies give."""
    off = offsets_of([40, 0, 55], 0, cuda)
    base = torch.randn(96, 200, device=cuda).to(BF16)
    w0 = torch.randn(3, 48, 64, device=cuda).to(BF16)
    big = torch.randn(3 * 64 * 48 + 1, device=cuda).to(BF16)
    for x in (base[:95, 8:56], base[:95, 3:51], base.t()[:48, :95].t(), base[1:, 100:148], base[:1, 8:56].expand(95, 48)):
        for w in (w0, w0.transpose(1, 2).contiguous().transpose(1, 2), big[1:].view(3, 48, 64)):
            a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
            c, d = x.contiguous().clone().requires_grad_(True), w.contiguous().clone().requires_grad_(True)
            y, z = grouped_linear(a, b, offsets=off), grouped_linear(c, d, offsets=off)
            assert torch.equal(y, z)
            g = torch.randn(64, 95, device=cuda).to(BF16).t()  # a gradient of other strides
            for u, v in zip(torch.autograd.grad(y, (a, b), g), torch.autograd.grad(z, (c, d), g.contiguous())):
                assert torch.equal(u, v)


def test_grouped_linear_gradients_by_differences(cuda):
    """The derivative along random directions against central differences of the 64-bit sum."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    route = route_topk(torch.randn(90, 5, device=cuda, generator=gen), 2)
    x, w = torch.randn(90, 64, device=cuda, generator=gen).to(BF16), torch.randn(5, 64, 32, device=cuda, generator=gen).to(BF16)
    b, dy = torch.randn(5, 32, device=cuda, generator=gen), torch.randn(180, 32, device=cuda, generator=gen).to(BF16)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(grouped_linear(*leaves, route=route), leaves, dy)

    def f(x, w, b):
        return (exact_linear(x, w, b, route.offsets, dy, route.rows)[0][0] * dy.double()).sum().item()

    base = [x.double(), w.double(), b.double()]
    for i, grad in enumerate(grads):
        d = torch.randn(grad.shape, device=cuda, dtype=torch.float64, generator=gen)
        h = 1e-4
        up, dn = [t.clone() for t in base], [t.clone() for t in base]
        up[i] += h * d
        dn[i] -= h * d
        diff = (f(*up) - f(*dn)) / (2 * h)
        mine = (grad.double() * d).sum().item()
        # f is linear in each operand; grad's rounding is at most half a step of each value
        assert abs(diff - mine) <= (torch.finfo(grad.dtype).eps / 2 + 1e-5) * (grad.double() * d).abs().sum().item() + 1e-5


def test_grouped_linear_repeats_bit_for_bit(cuda):
    route = route_topk(torch.randn(3000, 6, device=cuda), 2)
    x = torch.randn(3000, 264, device=cuda).to(BF16).requires_grad_(True)
    w = torch.randn(6, 264, 520, device=cuda).to(BF16).requires_grad_(True)
    b = torch.randn(6, 520, device=cuda).to(BF16).requires_grad_(True)
    dy = torch.randn(6000, 520, device=cuda).to(BF16)
    runs = []
    for _ in range(3):
        y = grouped_linear(x, w, b, route=route)
        runs.append((y.detach(), *torch.autograd.grad(y, (x, w, b), dy)))
    for r in runs[1:]:
        for u, v in zip(r, runs[0]):
            assert torch.equal(u, v)


def test_grouped_linear_bad_offsets_are_reported(cuda):
    """Offsets that fall or leave the rows: clamped, reported, nothing outside the output is touched."""
    x, w = torch.randn(20, 16, device=cuda).to(BF16), torch.randn(3, 16, 8, device=cuda).to(BF16)
    st = default_status(cuda)
    st.check()
    for off in ([0, 5, 9, 400], [0, 12, 7, 20], [-4, 5, 9, 20]):
        grouped_linear(x, w, offsets=torch.tensor(off, dtype=torch.int32, device=cuda))
        with pytest.raises(RuntimeError, match="out of range"):
            st.check("offsets")


@pytest.mark.parametrize("R,off", [
    (12, [0, 7, 2, 12]), (16, [9, 3, 12, 14, -5, 11]), (14, [3] + [(i * 37) % 14 for i in range(80)]), (700, [0, 400, 130, 650, 10, 700]),
    (700, [650, 20, 300, 900, 100]), (5000, [(i * 977) % 5000 for i in range(601)]), (9000, [0, 8000, 4000, 8500, 100, 9000]),
    (9000, [(i * 1117) % 9000 for i in range(41)])])
def test_grouped_linear_falling_offsets_share_no_row(cuda, R, off):
    """A group starts at the largest offset up to its own, as on the CPU: no row is computed twice, and each call gives the
    bits that the rising offsets give."""
    gen = torch.Generator(device="cuda").manual_seed(R)
    G, top, rising = len(off) - 1, 0, []
    for o in off:
        top = max(top, min(max(o, 0), R))
        rising.append(top)
    x, dy = torch.randn(R, 40, device=cuda, generator=gen).to(BF16), torch.randn(R, 72, device=cuda, generator=gen).to(BF16)
    w, b = torch.randn(G, 40, 72, device=cuda, generator=gen).to(BF16), torch.randn(G, 72, device=cuda, generator=gen)
    st = default_status(cuda)
    st.check()
    outs = []
    for o in (off, rising):
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        y = grouped_linear(*leaves, offsets=torch.tensor(o, dtype=torch.int32, device=cuda))
        outs.append((y.detach(), *torch.autograd.grad(y, leaves, dy)))
        if o is off:
            with pytest.raises(RuntimeError, match="out of range"):
                st.check("offsets")
    st.check()
    for name, u, v in zip(("y", "dx", "dw", "db"), *outs):
        assert torch.equal(u, v), name
    on_cpu = grouped_linear(x.cpu().double(), w.cpu().double(), b.cpu().double(), offsets=torch.tensor(off, dtype=torch.int32))
    assert torch.equal(on_cpu, grouped_linear(x.cpu().double(), w.cpu().double(), b.cpu().double(), offsets=torch.tensor(rising, dtype=torch.int32)))
    mag = grouped_linear(x.cpu().double().abs(), w.cpu().double().abs(), b.cpu().double().abs(), offsets=torch.tensor(rising, dtype=torch.int32))
    within(outs[0][0].cpu(), on_cpu, 43 * 2 ** -23 * mag)


@pytest.mark.parametrize("R,G", [(9000, 1), (5000, 3)])
def test_grouped_linear_in_slices(cuda, R, G):
    """Few groups of a small weight: the weight gradient's rows are cut into slices, written and accumulated."""
    gen = torch.Generator(device="cuda").manual_seed(R)
    sizes = [R] if G == 1 else [R - 70, 0, 70]
    off = offsets_of(sizes, 0, cuda)
    x, dy = torch.randn(R, 40, device=cuda, generator=gen).to(BF16), torch.randn(R, 72, device=cuda, generator=gen).to(BF16)
    w = torch.randn(G, 40, 72, device=cuda, generator=gen).to(BF16).requires_grad_(True)
    b = torch.randn(G, 72, device=cuda, generator=gen).requires_grad_(True)
    y = grouped_linear(x, w, b, offsets=off)
    dw, db = torch.autograd.grad(y, (w, b), dy)
    _, _, (dw0, aw), (db0, ab) = exact_linear(x, w.detach(), b.detach(), off, dy)
    within(dw, dw0, (R + 2) * 2 ** -23 * aw, "dw")
    within(db, db0, (R + 2) * 2 ** -23 * ab, "db")
    p = torch.nn.Parameter(w.detach())
    p._flare_grad = torch.ones_like(p, dtype=FP32)
    grouped_linear(x, p, offsets=off).backward(dy)
    within(p._flare_grad, 1 + dw0, (R + 3) * 2 ** -23 * (1 + aw), "accumulated")


@pytest.mark.parametrize("N", [8, 72, 520])
@pytest.mark.parametrize("sizes", [
    [9000], [8193], [31, 1, 32, 33, 63, 64, 65, 0, 127, 129, 95, 10000], [8191, 1, 0, 8192, 64, 1, 63], [5000, 5000],
    [160 * 7 + 1, 160 * 9 - 1, 160, 20000, 159, 161, 0], [(i * 13) % 67 for i in range(520)], [1] * 17 + [4095, 4097, 513, 511]])
def test_grouped_linear_sums_lose_no_row(cuda, sizes, N):
    """Weight and bias gradients of small whole numbers are exact in float32 whatever the order: groups that end just before,
    on and after the borders of steps, chunks and slices, written in float32 and added to a flat buffer."""
    gen = torch.Generator(device="cuda").manual_seed(N + len(sizes))
    off = offsets_of(sizes, 2, cuda)
    R, G, K = 2 + sum(sizes) + 3, len(sizes), 40
    x, dy = (torch.randint(-3, 4, (R, n), device=cuda, generator=gen).to(BF16) for n in (K, N))
    w, b = (torch.randn(G, *n, device=cuda, generator=gen).requires_grad_(True) for n in ((K, N), (N,)))
    dw, db = torch.autograd.grad(grouped_linear(x, w, b, offsets=off), (w, b), dy)
    assert dw.dtype == db.dtype == FP32
    _, _, (dw0, _), (db0, _) = exact_linear(x, w.detach(), b.detach(), off, dy)  # sums below 2^18
    assert torch.equal(dw.double(), dw0) and torch.equal(db.double(), db0)
    p, q = torch.nn.Parameter(w.detach()), torch.nn.Parameter(b.detach())
    p._flare_grad, q._flare_grad = torch.full_like(p, 5.0), torch.full_like(q, -7.0)
    grouped_linear(x, p, q, offsets=off).backward(dy)
    assert torch.equal(p._flare_grad.double(), dw0 + 5) and torch.equal(q._flare_grad.double(), db0 - 7)


def test_grouped_linear_very_long_group(cuda):
    """One of 300 groups has nearly all of 70 million rows: cut into slices (its sums of small whole numbers are exact)."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    sizes = [i % 3 for i in range(150)] + [70_000_000] + [i % 5 for i in range(149)]
    off = offsets_of(sizes, 0, cuda)
    R = sum(sizes)
    x, dy = (torch.randint(-3, 4, (R, 8), device=cuda, generator=gen, dtype=torch.int8).to(BF16) for _ in range(2))
    w, b = torch.zeros(300, 8, 8, device=cuda, requires_grad=True), torch.zeros(300, 8, device=cuda, requires_grad=True)
    dw, db = torch.autograd.grad(grouped_linear(x, w, b, offsets=off), (w, b), dy)
    default_status(cuda).check()
    at = off.tolist()
    for g in (149, 150, 151, 299):
        want, sums = torch.zeros(8, 8, dtype=torch.float64, device=cuda), torch.zeros(8, dtype=torch.float64, device=cuda)
        for lo in range(at[g], at[g + 1], 1 << 22):
            hi = min(lo + (1 << 22), at[g + 1])
            want += x[lo:hi].double().t() @ dy[lo:hi].double()
            sums += dy[lo:hi].double().sum(0)
        assert torch.equal(dw[g].double(), want) and torch.equal(db[g].double(), sums)


def test_grouped_linear_frozen_operands(cuda):
    """Only what requires a gradient gets one: the bias alone, the input alone, the weight alone."""
    route = route_topk(torch.randn(300, 4, device=cuda), 2)
    x, dy = torch.randn(300, 32, device=cuda).to(BF16), torch.randn(600, 48, device=cuda).to(BF16)
    w, b = torch.randn(4, 32, 48, device=cuda).to(BF16), torch.randn(4, 48, device=cuda).to(BF16)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(grouped_linear(*leaves, route=route), leaves, dy)
    for i in range(3):
        args = [x, w, b]
        args[i] = args[i].clone().requires_grad_(True)
        got, = torch.autograd.grad(grouped_linear(*args, route=route), args[i], dy)
        assert torch.equal(got, want[i])


def test_grouped_linear_flat_gradients(cuda):
    """A parameter bound to a flat fused optimizer gets its gradient added there in fp32, micro-step by micro-step."""
    route = route_topk(torch.randn(100, 4, device=cuda), 2)
    x, dy = torch.randn(100, 32, device=cuda).to(BF16), torch.randn(200, 48, device=cuda).to(BF16)
    w = torch.nn.Parameter(torch.randn(2, 2, 32, 48, device=cuda).to(BF16))
    b = torch.nn.Parameter(torch.randn(2, 2, 48, device=cuda).to(BF16))
    free = [t.detach().float().requires_grad_(True) for t in (w, b)]
    want = torch.autograd.grad(grouped_linear(x, *free, route=route), free, dy)
    w._flare_grad, b._flare_grad = torch.ones_like(w, dtype=FP32), torch.ones_like(b, dtype=FP32)
    for _ in range(2):
        grouped_linear(x, w, b, route=route).backward(dy)
    assert w.grad is None and b.grad is None
    for p, g in ((w, want[0]), (b, want[1])):
        torch.testing.assert_close(p._flare_grad, 1 + 2 * g, rtol=2 ** -22, atol=2 ** -21)  # two fp32 additions


# -------------------------------------------------------------------- SwiGLU
def exact_swiglu(x, dy):
    h = x.shape[1] // 2
    up, gate, d = x[:, :h].double(), x[:, h:].double(), dy.double()
    s = torch.sigmoid(gate)
    return up * gate * s, torch.cat([d * gate * s, d * up * s * (1 + gate * (1 - s))], 1)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("R,h", [(1, 1), (3, 7), (5, 8), (2, 31), (300, 33), (17, 64), (1000, 200), (9, 1000), (4, 2056), (2, 2500)])
@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_swiglu(cuda, R, h, dtype, checkpoint):
    gen = torch.Generator(device="cuda").manual_seed(R + h)
    x = (torch.randn(R, 2 * h, device=cuda, generator=gen) * torch.exp(torch.randn(R, 1, device=cuda, generator=gen))).to(dtype)
    dy = torch.randn(R, h, device=cuda, generator=gen).to(dtype)
    leaf = x.clone().requires_grad_(True)
    y = swiglu(leaf, checkpoint=checkpoint)
    dx, = torch.autograd.grad(y, leaf, dy)
    at = e4m3_checkpoint_reference(x.cpu()).to(cuda) if checkpoint else x
    want, _ = exact_swiglu(x, dy)
    _, dwant = exact_swiglu(at, dy)
    # the exponential is off by 2 + 1.2 |gate| steps at most, the division and three products by 6 more
    def slack(v):
        gate = v[:, h:].double().abs()
        return (8 + 2 * gate) * 2 ** -23
    within(y.detach(), want, slack(x) * want.abs(), "y")
    up, gate, d = at[:, :h].double().abs(), at[:, h:].double().abs(), dy.double().abs()
    s = torch.sigmoid(at[:, h:].double())
    within(dx, dwant, torch.cat([slack(at) * d * gate * s, 2 * slack(at) * d * up * s * (1 + gate)], 1), "dx")
    assert torch.equal(swiglu(x, checkpoint=checkpoint), y.detach())  # without a gradient: the same values


def test_swiglu_extremes(cuda):
    """Large and small magnitudes, infinities and NaN: others of the group keep their checkpoint; nothing overflows that the
    result does not."""
    x = torch.zeros(4, 128, device=cuda)
    x[0] = torch.logspace(-40, 38, 128)
    x[1, 64:] = -torch.logspace(-3, 30, 64)
    x[1, :64] = 1e30
    x[2, 5], x[2, 69], x[2, 70] = math.inf, math.nan, 2.0
    x[2, :5] = 1.0
    x[3] = 2.0 ** -140
    leaf = x.clone().requires_grad_(True)
    y = swiglu(leaf, checkpoint="e4m3")
    dx, = torch.autograd.grad(y, leaf, torch.ones_like(y))
    want, _ = exact_swiglu(x, torch.ones_like(y))
    ok = torch.isfinite(want) & (want.abs() < 3e38)
    assert torch.isfinite(y[ok]).all()
    big = want.abs() > 1e-30
    assert ((y.double() - want).abs()[ok & big] <= (8 + 2 * x[:, 64:].double().abs())[ok & big] * 2 ** -23 * want.abs()[ok & big]).all()
    at = e4m3_checkpoint_reference(x.cpu()).to(cuda)
    _, dwant = exact_swiglu(at, torch.ones_like(y))
    assert torch.equal(dx.isnan(), dwant.isnan())


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
@pytest.mark.parametrize("h", [64, 37])
def test_swiglu_gates_whose_sigmoid_leaves_float32(cuda, h, checkpoint, dtype):
    """Gates from -78 down, where the sigmoid is below float32's normal range but its product with up or dy is not."""
    big = 3e4 if dtype == FP16 else 1e36
    gen = torch.Generator(device="cuda").manual_seed(h)
    gate = -torch.linspace(78, 110, 40 * h, device=cuda).view(40, h)
    gate[-1] = -torch.linspace(110, 700, h, device=cuda)
    gate[::3, ::2] = torch.randn(14, (h + 1) // 2, device=cuda, generator=gen)  # ordinary ones beside them
    up = big * torch.randn(40, h, device=cuda, generator=gen)
    x, dy = torch.cat([up, gate], 1).to(dtype), (big * torch.randn(40, h, device=cuda, generator=gen)).to(dtype)
    if dtype != FP16:
        dy[:, 1::2] = torch.randn(40, h // 2, device=cuda, generator=gen).to(dtype)
        dy[::3, ::2] = 1.0  # ordinary gates: results within the type's range
    leaf = x.clone().requires_grad_(True)
    y = swiglu(leaf, checkpoint=checkpoint)
    dx, = torch.autograd.grad(y, leaf, dy)
    at = e4m3_checkpoint_reference(x.cpu()).to(cuda) if checkpoint else x
    want, dwant = exact_swiglu(x, dy)[0], exact_swiglu(at, dy)[1]
    most = torch.finfo(dtype).max
    def slack(v):  # as in test_swiglu; 8 steps for the eighth power and five roundings where the 64-bit form is taken
        return (13 + 2 * v[:, h:].double().abs().clamp(max=100)) * 2 ** -23
    ok = want.abs() < most
    within(y.detach()[ok], want[ok], (slack(x) * want.abs())[ok], "y")
    g, d, u = at[:, h:].double(), dy.double(), at[:, :h].double()
    s = torch.sigmoid(g)
    mag = torch.cat([(d * g * s).abs(), (d * u * s).abs() * (1 + g.abs())], 1)
    ok = dwant.abs() < most * 0.99
    within(dx[ok], dwant[ok], (2 * slack(at).repeat(1, 2) * mag)[ok], "dx")
    if dtype != FP16 and checkpoint is None:  # what is tested here: results that are not small
        assert int(((want.abs() > 1e-3) & (x[:, h:] < -88)).sum()) > h


def test_swiglu_views(cuda):
    base = torch.randn(50, 300, device=cuda).to(BF16)
    for x in (base[:, 4:132], base[:, 3:131], base[::2, 8:72], base.t()[:128].t(), base[:1, :64].expand(9, 64)):
        a, b = x.detach().requires_grad_(True), x.contiguous().clone().requires_grad_(True)
        for checkpoint in (None, "e4m3"):
            y, z = swiglu(a, checkpoint=checkpoint), swiglu(b, checkpoint=checkpoint)
            assert torch.equal(y, z)
            g = torch.randn(y.shape[1], y.shape[0], device=cuda).to(BF16).t()
            assert torch.equal(torch.autograd.grad(y, a, g)[0], torch.autograd.grad(z, b, g.contiguous())[0])


def test_swiglu_checkpoint_memory(cuda):
    """The input can go after the call: what is kept is a byte a value and a byte for each 32."""
    x = torch.randn(4096, 2048, device=cuda).to(BF16).requires_grad_(True)
    held = []
    for checkpoint in (None, "e4m3"):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        h = x * 1  # an intermediate that nothing else holds
        y = swiglu(h, checkpoint=checkpoint)
        del h
        held.append(torch.cuda.memory_allocated() - before - y.numel() * 2)
        del y
    assert held[0] >= x.numel() * 2 and held[1] <= x.numel() * (1 + 1 / 32) + 4096


# --------------------------------------------------------------- combination
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("S,T,E,k,N", [(1, 1, 1, 1, 1), (1, 5, 4, 4, 8), (2, 70, 7, 3, 33), (1, 300, 9, 9, 264), (1, 900, 5, 2, 1500), (1, 40, 40, 32, 24)])
def test_combine(cuda, S, T, E, k, N, dtype):
    gen = torch.Generator(device="cuda").manual_seed(T + N)
    lg = torch.randn(S, T, E, device=cuda, generator=gen)
    if E > 1:
        lg[torch.rand(S, T, E, device=cuda, generator=gen) < 0.2] = -math.inf
        lg[:, T // 2] = -math.inf
    route = route_topk(lg, k)
    z = torch.randn(S * T * k, N, device=cuda, generator=gen).to(dtype)
    dy = torch.randn(S * T, N, device=cuda, generator=gen).to(dtype)
    total = int(route.offsets[-1])
    z[total:] = math.nan  # rows behind the last group are not read
    for weighted in (True, False):
        a, w = z.clone().requires_grad_(True), route.weights.clone().requires_grad_(True)
        y = combine_rows(a, route, w if weighted else None)
        grads = torch.autograd.grad(y, (a, w) if weighted else (a,), dy)
        b, v = z.double().requires_grad_(True), route.weights.double().requires_grad_(True)
        want = combine_rows_reference(b, route, v if weighted else None)
        mag = combine_rows_reference(z.double().abs(), route, route.weights.double() if weighted else None)
        ref = torch.autograd.grad(want, (b, v) if weighted else (b,), dy.double())
        within(y.detach(), want.detach(), (k + 1) * 2 ** -23 * mag)
        within(grads[0][:total], ref[0][:total], 2 ** -23 * ref[0][:total].abs())
        assert not grads[0][total:].any()
        if weighted:
            zz, at = torch.cat([z[:total].double().abs(), z.new_zeros(1, N).double()]), route.row_of.view(S * T, k).long()
            m = (zz[torch.where(at < 0, total, at)] * dy.double().abs().unsqueeze(1)).sum(-1).view(w.shape)
            within(grads[1], ref[1], (N + 2) * 2 ** -23 * m)
            assert not grads[1][route.experts < 0].any()


def test_combine_views(cuda):
    route = route_topk(torch.randn(60, 4, device=cuda), 2)
    base = torch.randn(120, 100, device=cuda).to(BF16)
    for z in (base[:, 8:72], base[:, 1:65], base.t()[:64].t().contiguous().t().contiguous().t(), base[:1, :64].expand(120, 64)):
        w = route.weights.to(BF16)  # weights of another type are used in float32
        assert torch.equal(combine_rows(z, route, w), combine_rows(z.contiguous(), route, w.float()))


def test_combination_ignores_weights_where_there_is_no_choice(cuda):
    route = route_topk(torch.tensor([[0.0, 1.0, -math.inf], [-math.inf] * 3, [-math.inf, 2.0, -math.inf]], device=cuda), 2)
    z = torch.ones(6, 4, device=cuda, requires_grad=True)
    for bad in (math.nan, math.inf):
        w = torch.where(route.experts < 0, bad, route.weights).requires_grad_(True)
        y = combine_rows(z, route, w)
        assert torch.equal(y, combine_rows(z, route, route.weights))
        dz, dw = torch.autograd.grad(y, (z, w), torch.ones_like(y))
        assert torch.isfinite(dz).all() and torch.isfinite(dw).all() and not dw[route.experts < 0].any()


# ------------------------------------------------------------ used together
def plain_mlp(x, lg, wu, bu, wd, bd, k, checkpoint):
    """The block in 64 bits from the definition, its activations rounded where the kernels store them (rounding passes
    gradients on).  With a checkpoint the activation's gradient is taken at the checkpoint's values."""
    S, T, E = lg.shape
    h = wd.shape[-2]

    class Round(torch.autograd.Function):
        @staticmethod
        def forward(ctx, v):
            return v.to(BF16).double()

        @staticmethod
        def backward(ctx, g):
            return g.to(BF16).double()

    class At(torch.autograd.Function):  # the value of v, the derivative at the checkpoint
        @staticmethod
        def forward(ctx, v):
            ctx.save_for_backward(e4m3_checkpoint_reference(v.to(BF16)).double() if checkpoint else v)
            return v[:, :h] * torch.nn.functional.silu(v[:, h:])

        @staticmethod
        def backward(ctx, g):
            v, = ctx.saved_tensors
            s = torch.sigmoid(v[:, h:])
            return torch.cat([g * v[:, h:] * s, g * v[:, :h] * s * (1 + v[:, h:] * (1 - s))], 1)

    route = route_topk_reference(lg, k)
    flat = x.reshape(S * T, -1)
    y = torch.zeros(S * T, wd.shape[-1], dtype=torch.float64, device=x.device)
    experts, weights = route.experts.view(S * T, k), route.weights.view(S * T, k)
    for s in range(S):
        for e in range(E):
            for j in range(k):
                t = (experts[s * T:(s + 1) * T, j] == e).nonzero().squeeze(1) + s * T
                if t.numel():
                    u = Round.apply(flat[t] @ wu[s, e] + bu[s, e])
                    z = Round.apply(Round.apply(At.apply(u)) @ wd[s, e] + bd[s, e])
                    y = y.index_add(0, t, weights[t, j:j + 1] * z)
    return y.view(S, T, -1)


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
@pytest.mark.parametrize("S,T,E,k,d,h", [(1, 1, 4, 2, 64, 128), (2, 90, 5, 2, 64, 96), (1, 700, 3, 1, 136, 264)])
def test_expert_mlp(cuda, S, T, E, k, d, h, checkpoint):
    gen = torch.Generator(device="cuda").manual_seed(T)
    def rnd(*shape, scale=1.0):
        return (torch.randn(*shape, device=cuda, generator=gen) * scale).to(BF16)
    x, lg = rnd(S, T, d), rnd(S, T, E)
    params = [rnd(S, E, d, 2 * h, scale=d ** -0.5), rnd(S, E, 2 * h, scale=0.1), rnd(S, E, h, d, scale=h ** -0.5), rnd(S, E, d, scale=0.1)]
    dy = rnd(S, T, d)
    mine = [t.clone().requires_grad_(True) for t in (x, lg, *params)]
    ref = [t.double().requires_grad_(True) for t in (x, lg, *params)]
    y, want = expert_mlp(*mine, top_k=k, checkpoint=checkpoint), plain_mlp(*ref, k, checkpoint)
    grads, wants = torch.autograd.grad(y, mine, dy), torch.autograd.grad(want, ref, dy.double())
    # Every stored value is off by at most half a step (2^-8 in bf16).  A value that lies within fp32 error of a
    # rounding border may fall on its other side (one step, 2^-7, in a few places): at most six stored values lie
    # between an input and an output, so in the norm nothing is further off than 6 * 2^-8.
    for name, a, b in zip(("y", "x", "logits", "w_up", "b_up", "w_down", "b_down"), (y.detach(), *grads), (want.detach(), *wants)):
        if float(b.norm()) > 0:
            assert float((a.double() - b).norm() / b.norm()) < 6 * 2 ** -8, name
        else:
            assert float(a.double().norm()) < 1e-6, name
    default_status(cuda).check()


def test_expert_mlp_in_graphs(cuda):
    """Two captured training steps of different sizes, replayed in turn on new inputs, give what eager calls give."""
    def make(T):
        torch.manual_seed(T)
        x, lg = torch.randn(T, 64, device=cuda).to(BF16), torch.randn(T, 6, device=cuda).to(BF16)
        ws = [torch.randn(6, 64, 256, device=cuda).mul(0.1).to(BF16), torch.randn(6, 256, device=cuda).to(BF16),
              torch.randn(6, 128, 64, device=cuda).mul(0.1).to(BF16), torch.randn(6, 64, device=cuda).to(BF16)]
        return [t.requires_grad_(True) for t in (x, lg, *ws)], torch.randn(T, 64, device=cuda).to(BF16)

    def step(leaves, dy):
        y = expert_mlp(*leaves, top_k=2, checkpoint="e4m3")
        return (y, *torch.autograd.grad(y, leaves, dy))

    def copies(leaves):
        return [t.detach().clone().requires_grad_(True) for t in leaves]

    held = []
    for T in (40, 900):
        leaves, dy = make(T)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(leaves, dy)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(leaves, dy)
        held.append((graph, leaves, dy, out))
    for _ in range(2):
        for graph, leaves, dy, out in held:
            with torch.no_grad():
                for t in leaves[:2]:
                    t.copy_(torch.randn_like(t))
            graph.replay()
        for graph, leaves, dy, out in held:
            for a, b in zip(out, step(copies(leaves), dy)):
                assert torch.equal(a, b)
    default_status(cuda).check()


def test_another_stream(cuda):
    x, w = torch.randn(300, 64, device=cuda).to(BF16), torch.randn(4, 64, 96, device=cuda).to(BF16)
    lg = torch.randn(300, 4, device=cuda)
    want = grouped_linear(x, w, route=route_topk(lg, 2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = grouped_linear(x, w, route=route_topk(lg, 2))
    side.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_routed_layer_trains_on_flat_buffers(cuda, checkpoint):
    """A token mixer of routed experts bound to the flat fused optimizer: its flat gradients against 64-bit autograd."""
    from flare_b200.training.flat import DenseOptimizerConfig
    from flare_b200.training.fused_module import FusedDenseParameters

    torch.manual_seed(0)
    layer = BatchedExpertMoE(2, 64, 2, 4, True, 2, residual_norm=False, routed=True, checkpoint=checkpoint).to(cuda)
    flat = FusedDenseParameters(layer, DenseOptimizerConfig(learning_rate=0.1), device=cuda)
    x, dy = torch.randn(2, 200, 64, device=cuda).to(BF16), torch.randn(2, 200, 64, device=cuda).to(BF16)
    layer(x).backward(dy)
    ref = {n: p.detach().double().requires_grad_(True) for n, p in layer.named_parameters()}
    lg = (torch.einsum("dbi,dio->dbo", x, layer.w_gate) + layer.b_gate.unsqueeze(1)).detach().double().requires_grad_(True)
    want = plain_mlp(x.double(), lg, ref["w_up"], ref["b_up"], ref["w_down"], ref["b_down"], 2, checkpoint)
    want.backward(dy.double())
    for n in ("w_up", "b_up", "w_down", "b_down"):
        got = getattr(layer, n)._flare_grad.double()
        assert getattr(layer, n).grad is None
        assert float((got - ref[n].grad).norm() / ref[n].grad.norm()) < 6 * 2 ** -8, n  # as for the block
    before = layer.w_up.detach().clone()
    flat.step()
    assert not torch.equal(before, layer.w_up.detach())


def test_routed_mixer_runs_in_half_types(cuda):
    torch.manual_seed(1)
    mix = TokenMixLargeMoe(2, 4, 96, head_num=6, scale_size=2, num_experts=3, sparse=True, top_k=2, routed=True, checkpoint="e4m3").to(cuda)
    for dtype in (BF16, FP16):
        x = torch.randn(33, 4, 96, device=cuda).to(dtype).requires_grad_(True)
        y = mix(x)
        assert y.dtype == dtype and y.shape == (33, 96)
        y.float().square().mean().backward()
        assert torch.isfinite(x.grad).all() and all(torch.isfinite(p.grad).all() for p in mix.parameters())


@pytest.mark.parametrize("dtype,width", [(BF16, 64), (FP16, 64), (BF16, 12), (FP32, 12)])
@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_routed_layer_with_one_expert(cuda, checkpoint, dtype, width):
    """Nothing to route: any width and type, and the checkpoint is kept; outputs and gradients against 64 bits."""
    torch.manual_seed(2)
    layer = BatchedExpertMoE(2, width, 2, 1, True, 2, residual_norm=False, routed=True, checkpoint=checkpoint).to(cuda)
    h = 2 * width
    x, dy = torch.randn(2, 90, width, device=cuda).to(dtype).requires_grad_(True), torch.randn(2, 90, width, device=cuda).to(dtype)
    y = layer(x)
    assert y.dtype == dtype
    dx, dw = torch.autograd.grad(y, (x, layer.w_up), dy)
    wu, wd = (p.detach().to(dtype).double()[:, 0] for p in (layer.w_up, layer.w_down))
    u = torch.einsum("dbi,dih->dbh", x.detach().double(), wu)
    want = torch.einsum("dbh,dhi->dbi", u[..., :h] * torch.nn.functional.silu(u[..., h:]), wd)
    dz = torch.einsum("dbi,dhi->dbh", dy.double(), wd)
    if checkpoint:  # of the activation as the layer has it: one that lies on a border of e4m3 rounds to either side
        own = torch.einsum("dbi,deih->dbeh", x.detach(), layer.w_up.detach().to(dtype)) + layer.b_up.detach().to(dtype).unsqueeze(1)
        at = e4m3_checkpoint_reference(own.reshape(-1, 2 * h).cpu()).to(cuda).double().view_as(u)
    else:
        at = u
    s = torch.sigmoid(at[..., h:])
    du = torch.cat([dz * at[..., h:] * s, dz * at[..., :h] * s * (1 + at[..., h:] * (1 - s))], -1)
    # six roundings of half a step, as for the block; float32 sums of a few hundred products beside them
    tol = 6 * torch.finfo(dtype).eps / 2 + 512 * 2 ** -23
    for got, exact in ((y, want), (dx, torch.einsum("dbh,dih->dbi", du, wu)), (dw[:, 0], torch.einsum("dbi,dbh->dih", x.detach().double(), du))):
        assert float((got.detach().double() - exact).norm() / exact.norm()) < tol


# ------------------------------------------------------------------ refusals
def test_no_rows(cuda):
    w = torch.randn(3, 16, 24, device=cuda).to(BF16).requires_grad_(True)
    b = torch.randn(3, 24, device=cuda).to(BF16).requires_grad_(True)
    route = route_topk(torch.empty(0, 3, device=cuda), 2)
    assert route.offsets.tolist() == [0] * 4
    x = torch.empty(0, 16, device=cuda, dtype=BF16, requires_grad=True)
    for y in (grouped_linear(x, w, b, route=route), grouped_linear(x, w, b, offsets=route.offsets)):
        gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
        assert gx.shape == x.shape and not gw.any() and not gb.any()
    lg = torch.full((5, 3), -math.inf, device=cuda)  # tokens that go nowhere
    route = route_topk(lg, 2)
    x = torch.randn(5, 16, device=cuda).to(BF16).requires_grad_(True)
    y = grouped_linear(x, w, b, route=route)
    out = combine_rows(y, route, route.weights)
    assert not y.any() and not out.any()
    gx, gw, gb = torch.autograd.grad(out, (x, w, b), torch.ones_like(out))
    assert not gx.any() and not gw.any() and not gb.any()
    z, v = torch.empty(10, 0, device=cuda, requires_grad=True), torch.ones(5, 2, device=cuda, requires_grad=True)
    gz, gv = torch.autograd.grad(combine_rows(z, route, v), (z, v), torch.empty(5, 0, device=cuda))  # rows of no columns
    assert gz.shape == z.shape and not gv.any()
    for checkpoint in (None, "e4m3"):
        h = torch.empty(0, 8, device=cuda, dtype=BF16, requires_grad=True)
        assert torch.autograd.grad(swiglu(h, checkpoint=checkpoint), h, torch.empty(0, 4, device=cuda, dtype=BF16))[0].shape == (0, 8)


def test_refusals(cuda):
    lg = torch.randn(4, 3, device=cuda)
    route = route_topk(lg, 2)
    x, w = torch.randn(4, 16, device=cuda), torch.randn(3, 16, 24, device=cuda)
    with pytest.raises(TypeError, match="bfloat16"):
        grouped_linear(x, w, route=route)
    with pytest.raises(TypeError, match="weight"):
        grouped_linear(x.to(BF16), w.to(FP16), route=route)
    with pytest.raises(TypeError, match="bias"):
        grouped_linear(x.to(BF16), w, torch.zeros(3, 24, device=cuda, dtype=torch.float64), route=route)
    with pytest.raises(ValueError, match="multiples of 8"):
        grouped_linear(x[:, :12].to(BF16), w[:, :12].to(BF16), route=route)
    with pytest.raises(ValueError, match="multiples of 8"):
        grouped_linear(x.to(BF16), w[:, :, :20].to(BF16), route=route)
    with pytest.raises(ValueError, match="device"):
        grouped_linear(x.to(BF16), w.cpu(), route=route)
    many = MAX_GROUPS + 1
    with pytest.raises(ValueError, match="groups"):
        grouped_linear(x[:, :8].to(BF16), torch.zeros(many, 8, 8, device=cuda, dtype=BF16), offsets=torch.zeros(many + 1, dtype=torch.int32, device=cuda))
    with pytest.raises(ValueError, match="experts"):
        route_topk(torch.randn(2, MAX_EXPERTS + 1, device=cuda), 2)
    with pytest.raises(ValueError, match="top_k"):
        route_topk(torch.randn(2, 64, device=cuda), 33)
    with pytest.raises(ValueError, match="groups"):
        route_topk(torch.empty(8193, 0, 8, device=cuda), 2)
    with pytest.raises(TypeError, match="float32"):
        route_topk(lg.double(), 2)
    with pytest.raises(TypeError, match="float32"):
        swiglu(x.double())
    with pytest.raises(TypeError, match="float32"):
        combine_rows(torch.randn(8, 4, device=cuda).double(), route)
    leaf = x.to(BF16).requires_grad_(True)
    for y in (grouped_linear(leaf, w.to(BF16), route=route), swiglu(leaf), swiglu(leaf, checkpoint="e4m3")):
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(y.float().sum(), leaf, create_graph=True)


def test_tangents_are_refused(cuda):
    from torch.autograd import forward_ad

    lg, x, w = torch.randn(4, 3, device=cuda), torch.randn(4, 16, device=cuda).to(BF16), torch.randn(3, 16, 24, device=cuda).to(BF16)
    route = route_topk(lg, 2)
    z = torch.randn(8, 16, device=cuda)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for call in (lambda: route_topk(dual(lg), 2), lambda: swiglu(dual(x)), lambda: swiglu(dual(x), checkpoint="e4m3"),
                     lambda: grouped_linear(dual(x), w, route=route), lambda: grouped_linear(x, dual(w), offsets=torch.zeros(4, dtype=torch.int32, device=cuda)),
                     lambda: combine_rows(z, route, dual(route.weights)), lambda: combine_rows(dual(z), route)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
