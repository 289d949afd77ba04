"""Routed experts on the CPU: the plain forms against the definitions, the layers that use them, and the refusals
that need no device."""
import math

import pytest
import torch

from flare_b200.models.layers import BatchedExpertMoE, TokenMixLargeMoe, TokenMixLargePreGateNoPool
from flare_b200.ops.experts import (ExpertRoute, combine_rows, e4m3_checkpoint_reference, expert_mlp, grouped_linear, route_topk,
                                    swiglu)


def _loop_route(logits, k):
    """Token by token, in Python numbers."""
    S, B, E = logits.shape
    chosen, rows = {}, {}
    for s in range(S):
        for b in range(B):
            lg = [float(v) for v in logits[s, b]]
            order = sorted(range(E), key=lambda e: (-lg[e] if not math.isnan(lg[e]) else -math.inf, e))
            order = sorted(order, key=lambda e: 0 if math.isnan(lg[e]) else 1)
            chosen[s, b] = [e for e in order[:k] if lg[e] != -math.inf]
    r, offsets = 0, [0]
    for s in range(S):
        for e in range(E):
            for b in range(B):
                if e in chosen[s, b]:
                    rows[r] = (s * B + b, chosen[s, b].index(e))
                    r += 1
            offsets.append(r)
    return chosen, rows, offsets


def check_route(route, logits, k):
    """A route's whole numbers against the loop."""
    S, B, E = logits.shape
    chosen, rows, offsets = _loop_route(logits, k)
    experts, row_of = route.experts.view(S, B, k).tolist(), route.row_of.view(S * B, k).tolist()
    for (s, b), c in chosen.items():
        assert experts[s][b] == c + [-1] * (k - len(c))
    assert route.offsets.tolist() == offsets
    assert route.rows.tolist() == [rows[r][0] for r in range(len(rows))] + [-1] * (S * B * k - len(rows))
    for r, (t, j) in rows.items():
        assert row_of[t][j] == r
    assert sum(v >= 0 for line in row_of for v in line) == len(rows)


def hard_logits(S, B, E, seed, dtype=torch.float32):
    """Ties, masked experts, tokens with nothing left, signed zeros."""
    gen = torch.Generator().manual_seed(seed)
    lg = torch.randint(-3, 4, (S, B, E), generator=gen).float() * 0.5
    lg[torch.rand(S, B, E, generator=gen) < 0.3] = -math.inf
    lg[torch.rand(S, B, E, generator=gen) < 0.1] = -0.0
    lg[:, B // 2] = -math.inf
    return lg.to(dtype)


@pytest.mark.parametrize("S,B,E,k", [(1, 1, 1, 1), (1, 9, 4, 4), (3, 7, 5, 2), (2, 20, 33, 3)])
def test_route_reference(S, B, E, k):
    lg = hard_logits(S, B, E, S + B + E)
    route = route_topk(lg, k)
    check_route(route, lg, k)
    w = route.weights
    live = route.experts >= 0
    assert torch.equal(w == 0, ~live)
    torch.testing.assert_close(w.sum(-1), live.any(-1).float(), rtol=0, atol=k * 2 ** -23)
    assert torch.equal(route_topk(lg[0], k).experts, route_topk(lg[:1], k).experts[0])


def test_route_nan_is_largest():
    lg = torch.tensor([[[0.0, math.nan, 3.0, math.inf]]])
    route = route_topk(lg, 2)
    assert route.experts.tolist() == [[[1, 3]]] and route.weights.isnan().all()


def test_route_gradient_by_differences():
    torch.manual_seed(0)
    lg = torch.randn(2, 5, 6, dtype=torch.float64)
    lg[0, 1, 2] = -math.inf
    lg[1, 3] = -math.inf
    finite = torch.isfinite(lg)
    g = torch.randn(2, 5, 3, dtype=torch.float64)
    x = lg.clone().requires_grad_(True)
    (route_topk(x, 3).weights * g).sum().backward()
    h = 1e-6
    for i in finite.nonzero().tolist():
        up, dn = lg.clone(), lg.clone()
        up[tuple(i)] += h
        dn[tuple(i)] -= h
        d = ((route_topk(up, 3).weights - route_topk(dn, 3).weights) * g).sum() / (2 * h)
        assert abs(float(d) - float(x.grad[tuple(i)])) < 1e-7  # h^2 and 64-bit rounding over 2h
    assert torch.equal(x.grad[~finite], torch.zeros_like(x.grad[~finite]))


def test_grouped_linear_reference_rows_outside_groups():
    torch.manual_seed(1)
    x, w, b = torch.randn(10, 3), torch.randn(3, 3, 2), torch.randn(3, 2)
    y = grouped_linear(x, w, b, offsets=torch.tensor([2, 5, 5, 9], dtype=torch.int32))
    want = torch.zeros(10, 2)
    want[2:5] = x[2:5] @ w[0] + b[0]
    want[5:9] = x[5:9] @ w[2] + b[2]
    torch.testing.assert_close(y, want)


def test_checkpoint_values():
    """Every value of a group lands on an e4m3 value times the group's power of two, nearest to it."""
    grid = torch.tensor([m * 2.0 ** e / 8 for e in range(-6, 9) for m in range(8, 16)] + [m * 2.0 ** -9 for m in range(8)])
    grid = grid[grid <= 448]
    torch.manual_seed(2)
    x = torch.randn(6, 2 * 37) * torch.exp(3 * torch.randn(6, 1))
    q = e4m3_checkpoint_reference(x)
    for half in (slice(0, 37), slice(37, 74)):
        for c in (0, 32):
            v, got = x[:, half][:, c:c + 32], q[:, half][:, c:c + 32]
            top = v.abs().amax(1, keepdim=True)
            scale = 2.0 ** torch.ceil(torch.log2(top / 448))
            near = (v / scale).abs().unsqueeze(-1).sub(grid).abs().amin(-1)
            on_grid = (got / scale).abs().unsqueeze(-1).sub(grid).abs().amin(-1)
            assert torch.equal(on_grid, torch.zeros_like(on_grid))
            torch.testing.assert_close((got / scale - v / scale).abs(), near, rtol=0, atol=1e-4)


def test_checkpoint_keeps_other_values_beside_infinities():
    x = torch.ones(1, 64)
    x[0, 3], x[0, 40], x[0, 5] = math.inf, math.nan, 0.0
    q = e4m3_checkpoint_reference(x)
    assert q.isnan().nonzero().tolist() == [[0, 3], [0, 40]]
    ok = ~q.isnan()
    assert torch.equal(q[ok], x[ok])


def test_swiglu_gradient_is_the_formula_at_the_checkpoint():
    torch.manual_seed(3)
    x = torch.randn(5, 20, dtype=torch.float64)
    g = torch.randn(5, 10, dtype=torch.float64)
    for checkpoint in (None, "e4m3"):
        leaf = x.clone().requires_grad_(True)
        swiglu(leaf, checkpoint=checkpoint).backward(g)
        at = (e4m3_checkpoint_reference(x).double() if checkpoint else x.clone()).requires_grad_(True)
        (at[:, :10] * torch.nn.functional.silu(at[:, 10:])).backward(g)
        torch.testing.assert_close(leaf.grad, at.grad)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_swiglu_gates_whose_sigmoid_leaves_float32(dtype):
    gate = -torch.linspace(80, 110, 61)
    x = torch.cat([torch.full_like(gate, 1e36), gate]).view(1, -1).to(dtype)
    up, g = x[:, :61].double(), x[:, 61:].double()
    want = up * g * torch.exp(g)
    torch.testing.assert_close(swiglu(x).double(), want, rtol=torch.finfo(dtype).eps / 2 + 1e-12, atol=0)


@pytest.mark.parametrize("slots", [1, 3])
def test_expert_mlp_matches_all_experts_then_pick(slots):
    """The routed block against the sparse layer that computes every expert, outputs and gradients, in 64 bits."""
    torch.manual_seed(4)
    dense = BatchedExpertMoE(slots, 6, 2, 5, True, 2).double()
    routed = BatchedExpertMoE(slots, 6, 2, 5, True, 2, routed=True).double()
    with torch.no_grad():
        for p in dense.parameters():
            p.add_(0.1 * torch.randn_like(p))
    routed.load_state_dict(dense.state_dict())
    x = torch.randn(slots, 11, 6, dtype=torch.float64)
    xs = [x.clone().requires_grad_(True) for _ in range(2)]
    ys = [m(v) for m, v in zip((dense, routed), xs)]
    g = torch.randn_like(ys[0])
    for y in ys:
        y.backward(g)
    # the routed layer's norm is of the same formula; softmax weights are 32-bit in the dense layer
    torch.testing.assert_close(ys[1], ys[0], rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(xs[1].grad, xs[0].grad, rtol=1e-4, atol=1e-5)
    for (n, p), (_, q) in zip(routed.named_parameters(), dense.named_parameters()):
        torch.testing.assert_close(p.grad, q.grad, rtol=1e-4, atol=1e-5, msg=n)


def test_token_mixers_pass_the_option_on():
    torch.manual_seed(5)
    x = torch.randn(4, 4, 24)
    for cls in (TokenMixLargeMoe, TokenMixLargePreGateNoPool):
        a = cls(2, 4, 24, head_num=6, scale_size=2, num_experts=3, sparse=True, top_k=2)
        b = cls(2, 4, 24, head_num=6, scale_size=2, num_experts=3, sparse=True, top_k=2, routed=True, checkpoint="e4m3")
        b.load_state_dict(a.state_dict())
        assert all(m.routed and m.checkpoint == "e4m3" for m in b.modules() if isinstance(m, BatchedExpertMoE))
        torch.testing.assert_close(b(x), a(x), rtol=1e-4, atol=1e-5)


def test_routed_layer_decides_in_the_type_of_a_float32_gate():
    """Logits that are equal in 16 bits and not in float32, and gradients of the gate, with 16-bit rows."""
    layer = BatchedExpertMoE(1, 8, 1, 4, True, 1, residual_norm=False, routed=True)
    with torch.no_grad():
        for p in (layer.w_gate, layer.w_down):
            p.zero_()
        layer.b_gate.copy_(torch.tensor([[8.0, 8.01, 0.0, 8.005]]))
        layer.b_down.copy_(torch.arange(4.0).view(1, 4, 1).expand(1, 4, 8))
        assert torch.equal(layer(torch.randn(1, 3, 8).bfloat16()), torch.ones(1, 3, 8).bfloat16())  # expert 1
        layer.b_gate.zero_()
        layer.w_gate[0, :, 2], layer.w_gate[0, :, 0] = 1.0, 1.0 - 2.0 ** -10
        assert torch.equal(layer(torch.ones(1, 3, 8).bfloat16()), torch.full((1, 3, 8), 2.0).bfloat16())
    torch.manual_seed(8)
    layer = BatchedExpertMoE(2, 8, 2, 5, True, 2, residual_norm=False, routed=True)
    exact = BatchedExpertMoE(2, 8, 2, 5, True, 2, residual_norm=False, routed=True).double()
    exact.load_state_dict(layer.state_dict())
    x, dy = torch.randn(2, 40, 8).bfloat16(), torch.randn(2, 40, 8).bfloat16()
    layer(x).backward(dy)
    exact(x.double()).backward(dy.double())
    # the experts' rows come in bfloat16: six roundings of half a step in the norm, as for the block
    for n in ("w_gate", "b_gate"):
        got, want = getattr(layer, n).grad.double(), getattr(exact, n).grad
        assert float((got - want).norm() / want.norm()) < 6 * 2 ** -8, n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_routed_layer_with_one_expert(checkpoint, dtype):
    """Rows of x's type with float32 parameters are taken as with more experts, and the checkpoint is kept."""
    torch.manual_seed(6)
    layer = BatchedExpertMoE(2, 8, 2, 1, True, 2, residual_norm=False, routed=True, checkpoint=checkpoint)
    x = torch.randn(2, 5, 8).to(dtype).requires_grad_(True)
    y = layer(x)
    dy = torch.randn(2, 5, 8).to(dtype)
    dx, dw = torch.autograd.grad(y, (x, layer.w_up), dy)
    assert y.dtype == dtype and dx.dtype == dtype and dw.dtype == torch.float32
    ref = {n: p.detach().to(dtype).double() for n, p in layer.named_parameters()}
    xd = x.detach().double()
    h = torch.einsum("dbi,dih->dbh", xd, ref["w_up"][:, 0]) + ref["b_up"]
    z = h[..., :16] * torch.nn.functional.silu(h[..., 16:])
    want = torch.einsum("dbh,dhi->dbi", z, ref["w_down"][:, 0]) + ref["b_down"]
    dz = torch.einsum("dbi,dhi->dbh", dy.double(), ref["w_down"][:, 0])
    at = e4m3_checkpoint_reference(h.to(dtype).reshape(-1, 32)).double().view_as(h) if checkpoint else h
    s = torch.sigmoid(at[..., 16:])
    dh = torch.cat([dz * at[..., 16:] * s, dz * at[..., :16] * s * (1 + at[..., 16:] * (1 - s))], -1)
    # at most six roundings to x's type lie between input and output, as in the test of the block on CUDA
    tol = 6 * torch.finfo(dtype).eps / 2 + (1e-5 if dtype == torch.float32 else 0)
    for got, exact in ((y, want), (dx, torch.einsum("dbh,dih->dbi", dh, ref["w_up"][:, 0])), (dw[:, 0], torch.einsum("dbi,dbh->dih", xd, dh))):
        assert float((got.detach().double() - exact).norm() / exact.norm()) < tol
    full = BatchedExpertMoE(2, 8, 2, 1, True, 2, routed=True, checkpoint=checkpoint)  # with the norm: x's type as well
    assert full(x).dtype == dtype
    assert full(x[:, :0]).shape == (2, 0, 8)


def test_one_expert_keeps_the_checkpoint_and_not_the_activation():
    held = []

    def pack(t):
        held.append(t)
        return t

    layer = BatchedExpertMoE(1, 8, 2, 1, True, 2, residual_norm=False, routed=True, checkpoint="e4m3")
    x = torch.randn(1, 300, 8).bfloat16()
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        layer(x)
    up_gate = torch.einsum("dbi,deih->dbeh", x, layer.w_up.bfloat16()) + layer.b_up.bfloat16().unsqueeze(1)
    kept = e4m3_checkpoint_reference(up_gate.reshape(-1, 32))
    assert any(t.shape == kept.shape and torch.equal(t, kept) for t in held)  # on the CPU: the values that it stands for
    assert not any(t.numel() == up_gate.numel() and torch.equal(t.reshape(-1), up_gate.reshape(-1)) for t in held)


def test_routed_mixers_at_their_default_number_of_experts():
    torch.manual_seed(7)
    for cls in (TokenMixLargeMoe, TokenMixLargePreGateNoPool):
        mix = cls(1, 4, 24, head_num=6, scale_size=2, sparse=True, routed=True, checkpoint="e4m3")
        for dtype in (torch.bfloat16, torch.float32):
            y = mix(torch.randn(3, 4, 24).to(dtype))
            assert y.dtype == dtype and torch.isfinite(y).all()


def test_layers_pickled_without_the_options_still_run():
    import io

    torch.manual_seed(9)
    layer = BatchedExpertMoE(2, 8, 2, 3, True, 2)
    x = torch.randn(2, 5, 8)
    want = layer(x)
    for name in ("routed", "checkpoint"):
        layer.__dict__.pop(name, None)
    held = io.BytesIO()
    torch.save(layer, held)
    held.seek(0)
    assert torch.equal(torch.load(held, weights_only=False)(x), want)


def test_no_tokens():
    route = route_topk(torch.empty(2, 0, 3), 2)
    assert route.offsets.tolist() == [0] * 7 and route.rows.numel() == 0
    y = expert_mlp(torch.empty(2, 0, 4), torch.empty(2, 0, 3), torch.randn(2, 3, 4, 12), None, torch.randn(2, 3, 6, 4), None, top_k=2)
    assert y.shape == (2, 0, 4)


def test_refusals():
    lg = torch.randn(4, 3)
    with pytest.raises(ValueError, match="top_k"):
        route_topk(lg, 4)
    with pytest.raises(ValueError, match="top_k"):
        route_topk(lg, 0)
    with pytest.raises(ValueError, match="logits"):
        route_topk(lg[0], 1)
    route = route_topk(lg, 2)
    x, w = torch.randn(4, 6), torch.randn(3, 6, 5)
    with pytest.raises(ValueError, match="exactly one"):
        grouped_linear(x, w)
    with pytest.raises(ValueError, match="exactly one"):
        grouped_linear(x, w, offsets=route.offsets, route=route)
    with pytest.raises(ValueError, match="weight"):
        grouped_linear(x, w.transpose(1, 2), route=route)
    with pytest.raises(ValueError, match="offsets"):
        grouped_linear(x, w[:2], route=route)
    with pytest.raises(ValueError, match="offsets"):
        grouped_linear(x, w, offsets=route.offsets.long())
    with pytest.raises(ValueError, match="bias"):
        grouped_linear(x, w, torch.randn(3, 6), route=route)
    with pytest.raises(ValueError, match="tokens"):
        grouped_linear(torch.randn(3, 6), w, route=route)
    with pytest.raises(ValueError, match="2h"):
        swiglu(torch.randn(3, 5))
    with pytest.raises(ValueError, match="checkpoint"):
        swiglu(torch.randn(3, 4), checkpoint="int4")
    with pytest.raises(ValueError, match="route"):
        combine_rows(torch.randn(7, 2), route)
    with pytest.raises(ValueError, match="weights"):
        combine_rows(torch.randn(8, 2), route, torch.randn(4, 3))
    with pytest.raises(ValueError, match="same tokens"):
        expert_mlp(x, lg[:3], w, None, w, None, top_k=2)
    with pytest.raises(ValueError, match="sparse"):
        BatchedExpertMoE(1, 4, 2, 3, False, 2, routed=True)
    with pytest.raises(ValueError, match="routed"):
        BatchedExpertMoE(1, 4, 2, 3, True, 2, checkpoint="e4m3")
    assert ExpertRoute._fields == ("experts", "weights", "offsets", "rows", "row_of")


def test_native_refusals():
    """The native entry points check their arguments before they touch a device."""
    from flare_b200._native import available, native

    if not available():
        pytest.skip("the native extension is not built")
    C = native()
    x, w, off = torch.zeros(4, 16).bfloat16(), torch.zeros(3, 16, 24).bfloat16(), torch.zeros(4, dtype=torch.int32)

    def linear(x=x, w=w, bias=None, off=off, rows=None, row_of=None):
        return C.grouped_linear(x, w, bias, off, rows, row_of, None, None, 0, 0)

    row_of = torch.zeros(4, 2, dtype=torch.int32)
    for call, kind, words in (
            (lambda: linear(x=x[0]), ValueError, r"got \[16\]"), (lambda: linear(w=w[:, :8]), ValueError, r"\[3, 8, 24\]"),
            (lambda: linear(x=x.float()), TypeError, "got Float"), (lambda: linear(w=w.half()), TypeError, "Half"),
            (lambda: linear(w=w[:, :, :20]), ValueError, "got 16 and 20"), (lambda: linear(off=off[:2]), ValueError, "for 3 groups"),
            (lambda: linear(off=off.long()), ValueError, "int32"), (lambda: linear(bias=w[0]), ValueError, "bias"),
            (lambda: linear(bias=torch.zeros(3, 24).double()), TypeError, "bias"),
            (lambda: linear(rows=off, row_of=row_of), ValueError, "does not fit 4 tokens"),
            (lambda: linear(w=torch.zeros(2049, 16, 8).bfloat16()), ValueError, "groups, got 2049"),
            (lambda: C.route_topk(x[0], 1), ValueError, "logits"), (lambda: C.route_topk(x, 17), ValueError, "got 17"),
            (lambda: C.route_topk(torch.zeros(2, 513), 1), ValueError, "got 513"), (lambda: C.route_topk(x.double(), 1), TypeError, "Double"),
            (lambda: C.swiglu(x[:, :5], False), ValueError, r"got \[4, 5\]"), (lambda: C.swiglu(x.double(), False), TypeError, "Double"),
            (lambda: C.combine_rows(x, None, off, row_of), ValueError, r"must be \[8, n\]"),
            (lambda: C.combine_rows(x[:0], None, off, row_of[:, :0]), ValueError, "choices"),
            (lambda: linear(rows=off[:0], row_of=row_of[:, :0]), ValueError, "does not fit"),
            (lambda: C.combine_rows(torch.zeros(8, 3), torch.zeros(7), off, row_of), ValueError, "weights"),
            (lambda: C.combine_rows(torch.zeros(8, 3).double(), None, off, row_of), TypeError, "Double"),
            (lambda: linear(), RuntimeError, "CUDA device")):
        with pytest.raises(kind, match=words):
            call()


def test_combination_checks_the_offsets_of_a_route():
    """The gradient reads the last offset: a route whose offsets have none, or are of another type, is refused at the call."""
    from flare_b200._native import available, native

    route = route_topk(torch.randn(4, 3), 2)
    z = torch.randn(8, 2)
    for bad in (route.offsets[:0], route.offsets.long(), route.offsets.view(1, -1)):
        with pytest.raises(ValueError, match="offsets must be int32"):
            combine_rows(z, route._replace(offsets=bad), route.weights)
        if available():
            with pytest.raises(ValueError, match="offsets must be int32"):
                native().combine_rows(z, route.weights, bad, route.row_of)
    if available():
        with pytest.raises(ValueError, match="row_of must be int32"):
            native().combine_rows(z, route.weights, route.offsets, route.row_of.long())


def test_native_refusals_of_tangents():
    """A forward-mode tangent is refused, not dropped: with or without a gradient, on any operand."""
    from torch.autograd import forward_ad

    from flare_b200._native import available, native

    if not available():
        pytest.skip("the native extension is not built")
    C = native()
    x, w, b, off = torch.zeros(4, 16).bfloat16(), torch.zeros(3, 16, 24).bfloat16(), torch.zeros(3, 24).bfloat16(), torch.zeros(4, dtype=torch.int32)
    z, row_of, weights = torch.zeros(8, 16), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for leaf in (False, True):
            for call in (lambda t: C.route_topk(dual(t(x)), 2), lambda t: C.swiglu(dual(t(x)), False), lambda t: C.swiglu(dual(t(x)), True),
                         lambda t: C.combine_rows(dual(t(z)), weights, off, row_of), lambda t: C.combine_rows(z, dual(t(weights)), off, row_of),
                         lambda t: C.grouped_linear(dual(t(x)), w, b, off, None, None, None, None, 0, 0),
                         lambda t: C.grouped_linear(x, dual(t(w)), b, off, None, None, None, None, 0, 0),
                         lambda t: C.grouped_linear(x, w, dual(t(b)), off, None, None, None, None, 0, 0)):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(lambda v: v.clone().requires_grad_(leaf))


def test_combination_refuses_weights_of_another_layout():
    """As many values in another layout (choices first) are not the weights of these choices."""
    from flare_b200._native import available, native

    route = route_topk(torch.randn(2, 3, 4), 2)
    z, w = torch.randn(12, 5), route.weights
    assert torch.equal(combine_rows(z, route, w.reshape(6, 2)), combine_rows(z, route, w))
    for bad in (w.reshape(6, 2).t(), w.reshape(-1), w.reshape(2, 2, 3)):
        with pytest.raises(ValueError, match="weights must have the shape"):
            combine_rows(z, route, bad)
        if available():
            with pytest.raises(ValueError, match="weights must have the shape"):
                native().combine_rows(z, bad, route.offsets, route.row_of)


def test_combination_ignores_weights_where_there_is_no_choice():
    route = route_topk(torch.tensor([[0.0, 1.0, -math.inf], [-math.inf] * 3, [-math.inf, 2.0, -math.inf]]), 2)
    z = torch.ones(6, 4, requires_grad=True)
    for bad in (math.nan, math.inf):
        w = torch.where(route.experts < 0, bad, route.weights).requires_grad_(True)
        y = combine_rows(z, route, w)
        assert torch.equal(y, combine_rows(z, route, route.weights))
        dz, dw = torch.autograd.grad(y, (z, w), torch.ones_like(y))
        assert torch.isfinite(dz).all() and torch.isfinite(dw).all() and not dw[route.experts < 0].any()


def test_first_call_in_a_capture_is_refused(monkeypatch):
    from flare_b200 import _native
    from flare_b200.ops import experts

    monkeypatch.setattr(experts, "_STATUS", {})
    monkeypatch.setattr(_native, "_STATUS", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before the capture"):
        experts._status(torch.zeros(1))
    assert not experts._STATUS and not _native._STATUS
