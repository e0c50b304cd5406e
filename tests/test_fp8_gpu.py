"""Linear layers with 8-bit weights, routing to experts and the experts' products, against their formulas in 64 bits (plain_fp8.py)."""
from __future__ import annotations

import pytest
import torch

import plain_fp8 as plain

pytestmark = pytest.mark.gpu

BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
HALF_STEP = {BF: 2.0 ** -8, F32: 2.0 ** -24}


def _rand(seed, *shape, dtype=F32, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (std * torch.randn(*shape, generator=g, device="cuda")).to(dtype)


def _weight(seed, M, K):
    from stride_b200.kernels.linear import Fp8Weight
    return Fp8Weight.quantize(_rand(seed, M, K, std=K ** -0.5))


def _values(w):
    """What a plain (not stacked) weight stands for, in 64 bits."""
    return plain.weight_values(w.q[:, :w.shape[1]].to(F32), w.scales)


def _workspace(n):
    from stride_b200.parts.context import Workspace
    return Workspace(torch.device("cuda"), n)


def _quantize(x):
    from stride_b200.kernels import ops
    n, K = x.shape
    q = torch.zeros(n, -(-K // 16) * 16, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    s = torch.zeros(-(-K // 128), n, device="cuda")
    ops.quantize_fp8(x, q, s)
    return q, s


@pytest.mark.parametrize("n,K", [(1, 1), (1, 128), (3, 127), (5, 129), (17, 200), (2, 1000), (333, 2056), (64, 4096), (700, 260)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_quantised_rows(n, K, dtype):
    """Scales and values are exact: equal to the formula's, blocks of zeros, of tiny and of huge values and borders of the grid among them."""
    x = _rand(n * K, n, K, dtype=dtype)
    x[0, : K // 2] = 0
    x[-1] *= 2.0 ** 40
    if n > 2:
        x[1] *= 2.0 ** -120
        x[2] = 448.0
        x[2, ::3] = 26.0         # between two values: 448 has the scale 1, 26 is one of the grid's
        x[2, 1::3] = 25.0        # half way between 24 and 26: to even
    q, s = _quantize(x)
    want, scales = plain.quantised(x.to(F64))
    assert torch.equal(s.t().to(F64), scales)
    assert torch.equal(q[:, :K].to(F64), want)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_block_that_is_not_finite_poisons_its_token_only(bad):
    from stride_b200.kernels.linear import Linear
    x = _rand(1, 5, 300, dtype=BF)
    clean, out = torch.empty(5, 70, device="cuda"), torch.empty(5, 70, device="cuda")
    layer = Linear(_weight(2, 70, 300), BF)
    layer.forward(x, clean, workspace=_workspace(5))
    x[3, 170] = bad
    layer.forward(x, out, workspace=_workspace(5))
    assert torch.isnan(out[3]).all()
    assert torch.equal(out[[0, 1, 2, 4]], clean[[0, 1, 2, 4]])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_quantised_rows_at_the_ends_of_the_range(dtype):
    """The largest finite values, the smallest normal ones and below: the scale's exponent at both ends."""
    x = _rand(5, 6, 300, dtype=dtype)
    top = torch.finfo(dtype).max
    x[0], x[0, 1] = top, -top
    x[1], x[1, 200] = 1.0, top / 2
    x[2] = 2.0 ** -100 * 448
    x[3] = 2.0 ** -126
    x[4] = 0
    x[5, ::2] = 2.0 ** -133
    q, s = _quantize(x)
    want, scales = plain.quantised(x.to(F64))
    assert torch.equal(s.t().to(F64), scales)
    assert torch.equal(q[:, :300].to(F64), want)


SIZES = [(1, 1, 1), (1, 128, 128), (2, 130, 100), (16, 2048, 2048), (17, 500, 1000), (40, 128, 4096), (64, 1000, 900), (65, 300, 2056), (129, 256, 640),
         (333, 2500, 2056), (1000, 640, 384), (300, 12000, 256), (3000, 1300, 384), (200, 1000, 4096), (50, 20000, 256), (120, 19000, 130), (600, 1001, 4090)]


@pytest.mark.parametrize("n,M,K", SIZES)
@pytest.mark.parametrize("x_dtype,out_dtype", [(BF, F32), (F32, BF), (BF, BF), (F32, F32)])
def test_product(n, M, K, x_dtype, out_dtype):
    from stride_b200.kernels.linear import Linear
    x, w = _rand(n + M, n, K, dtype=x_dtype), _weight(K, M, K)
    out = torch.full((n, M), float("nan"), dtype=out_dtype, device="cuda")
    Linear(w, BF).forward(x, out, workspace=_workspace(n))
    xv, wv = plain.quantised_values(x.to(F64)), _values(w)
    want, bound = xv @ wv.t(), plain.product_bound(xv, wv)
    assert ((out.to(F64) - want).abs() <= bound + HALF_STEP[out_dtype] * (want.abs() + bound)).all()


@pytest.mark.parametrize("n,I,K", [(1, 1, 16), (1, 64, 128), (3, 100, 300), (8, 8192, 2048), (31, 65, 2048), (64, 1000, 520), (200, 200, 700), (333, 1408, 2056), (150, 200, 1100), (300, 1400, 2048)])
@pytest.mark.parametrize("out_dtype", [BF, F32])
def test_gated_product(n, I, K, out_dtype):
    """Gate and up matrices of any height, also where the up rows' scales do not begin at a multiple of 128."""
    from stride_b200.kernels.linear import Fp8Weight, Linear
    x, gate, up = _rand(n + I, n, K, dtype=BF), _weight(K, I, K), _weight(K + 1, I, K)
    out = torch.full((n, I), float("nan"), dtype=out_dtype, device="cuda")
    Linear(Fp8Weight.stack([gate, up]), BF).forward_swiglu(x, out, None, workspace=_workspace(n))
    want, bound = plain.gated(plain.quantised_values(x.to(F64)), _values(gate), _values(up))
    assert ((out.to(F64) - want).abs() <= bound + HALF_STEP[out_dtype] * (want.abs() + bound)).all()


@pytest.mark.parametrize("n", [1, 20, 300])
@pytest.mark.parametrize("activation,constants", [("gelu_tanh", ()), ("clamped", (1.5, 1.7))])
def test_other_gates(n, activation, constants):
    from stride_b200.kernels import ops
    from stride_b200.kernels.linear import Fp8Weight, Linear
    x, gate, up = _rand(n, n, 256, dtype=BF), _weight(5, 192, 256), _weight(6, 192, 256)
    out, ws = torch.empty(n, 192, dtype=BF, device="cuda"), _workspace(n)
    Linear(Fp8Weight.stack([gate, up]), BF).forward_swiglu(x, out, None, activation, constants, workspace=ws)
    g, u = torch.empty(n, 192, device="cuda"), torch.empty(n, 192, device="cuda")
    Linear(gate, BF).forward(x, g, workspace=ws)
    Linear(up, BF).forward(x, u, workspace=ws)
    g, u = g.to(F64), u.to(F64)
    if activation == "gelu_tanh":
        want = 0.5 * g * (1.0 + torch.tanh((2.0 / torch.pi) ** 0.5 * (g + 0.044715 * g ** 3))) * u
    else:
        want = g.clamp(max=1.5) * torch.sigmoid(1.7 * g.clamp(max=1.5)) * (u.clamp(-1.5, 1.5) + 1.0)
    assert ((out.to(F64) - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18 * (1.0 + u.abs())).all()


@pytest.mark.parametrize("n", [1, 30, 200])
def test_added_to_the_residual(n):
    from stride_b200.kernels import ops
    x, w, h = _rand(n, n, 512, dtype=BF), _weight(9, 384, 512), _rand(8, n, 384)
    q, s = _quantize(x)
    alone, out = torch.empty(n, 384, device="cuda"), h.clone()
    ops.gemm_fp8(q, s, w, alone)
    ops.gemm_fp8(q, s, w, out, ops.ADD)
    assert torch.equal(out, alone + h)


@pytest.mark.parametrize("M,K", [(128, 8192), (2048, 2048), (1500, 4104), (640, 260), (20000, 256), (12000, 384)])
def test_a_tokens_bits_do_not_depend_on_the_step(M, K):
    """Alone, in a few, in tiles of every size, the ranges of K on CTAs of their own and walked by one: the same bits."""
    from stride_b200.kernels.linear import Linear
    x, layer = _rand(M, 300, K, dtype=BF), Linear(_weight(K, M, K), BF)
    whole = torch.empty(300, M, device="cuda")
    layer.forward(x, whole, workspace=_workspace(300))
    for first, n in [(0, 1), (7, 16), (30, 17), (60, 33), (100, 65), (100, 128), (170, 129), (0, 257)]:
        part = torch.full((n, M), float("nan"), device="cuda")
        layer.forward(x[first:first + n], part, workspace=_workspace(300))
        assert torch.equal(part, whole[first:first + n]), (first, n)


@pytest.mark.parametrize("n,M,K,gated", [(600, 1001, 4090, False), (256, 4096, 1100, False), (300, 2816, 2048, True), (150, 400, 1100, True), (520, 1400, 4096, True)])
def test_bits_of_many_tokens_whose_ranges_are_shared_out(n, M, K, gated):
    """Weights of three and four ranges of K, a CTA of a cluster with one or two of them: the bits of a few tokens, where every range has a CTA; stored, gated
    and added to a residual."""
    from stride_b200.kernels import ops
    from stride_b200.kernels.linear import Fp8Weight, Linear
    x, W = _rand(M, n, K, dtype=BF), M // 2 if gated else M
    weight = Fp8Weight.stack([_weight(K, W, K), _weight(K + 1, W, K)]) if gated else _weight(K, M, K)
    layer, ws = Linear(weight, BF), _workspace(n)
    run = (lambda x, out: layer.forward_swiglu(x, out, None, workspace=ws)) if gated else (lambda x, out: layer.forward(x, out, workspace=ws))
    whole, part = torch.full((n, W), float("nan"), device="cuda"), torch.full((40, W), float("nan"), device="cuda")
    run(x, whole)
    for first in (0, 90, n - 40):
        run(x[first:first + 40], part)
        assert torch.equal(part, whole[first:first + 40]), first
    if not gated:
        h = _rand(3, n, M)
        added = h.clone()
        ops.gemm_fp8(*_quantize(x), weight, added, ops.ADD)
        assert torch.equal(added, whole + h)


@pytest.mark.parametrize("n", [1, 9, 16, 30, 50, 100, 300])
@pytest.mark.parametrize("columns,rows", [(257, 200), (256, 200), (256, 5000)])
def test_rows_of_larger_tensors_and_what_lies_around_them(n, columns, rows):
    """Input and result as column ranges of wider buffers, a slice that starts off a 16-byte border; what is around the result stays."""
    from stride_b200.kernels.linear import Linear
    wide, layer = _rand(3, n, 1003, dtype=BF), Linear(_weight(4, rows, columns), BF)
    x = wide[:, 5:5 + columns]
    want = torch.empty(n, rows, device="cuda")
    layer.forward(x.contiguous(), want, workspace=_workspace(n))
    for first in (100, 101):
        held = torch.full((n + 2, rows + 133), 7.0, device="cuda")
        layer.forward(x, held[1:n + 1, first:first + rows], workspace=_workspace(n))
        assert torch.equal(held[1:n + 1, first:first + rows], want)
        held[1:n + 1, first:first + rows] = 7.0
        assert (held == 7.0).all()


def test_calls_that_are_refused():
    """Shapes, types and layouts that the entry points do not take: an error, nothing is written."""
    from stride_b200.kernels import ops
    from stride_b200.kernels.linear import Fp8Weight, Linear
    x, w, ws = _rand(1, 4, 256, dtype=BF), _weight(2, 130, 256), _workspace(4)
    layer, out = Linear(w, BF), torch.full((4, 130), 7.0, device="cuda")
    with pytest.raises(ValueError):
        layer.forward(x[:, :255], out, workspace=ws)
    with pytest.raises(ValueError):
        layer.forward(x, out[:, :129], workspace=ws)
    with pytest.raises(ValueError):
        layer.forward(x.t().contiguous().t(), out, workspace=ws)
    with pytest.raises(ValueError):
        layer.forward(_rand(1, 5, 256, dtype=BF), torch.empty(5, 130, device="cuda"), workspace=ws)         # more rows than the workspace
    with pytest.raises(ValueError):
        layer.forward_swiglu(x, torch.empty(4, 65, device="cuda"), None, workspace=ws)                       # not stacked from two
    with pytest.raises(ValueError):
        Linear(Fp8Weight.stack([w, _weight(3, 130, 256)]), BF).forward(x, torch.empty(4, 260, device="cuda"), workspace=ws)
    with pytest.raises(TypeError):
        layer.forward(x.half(), out, workspace=ws)
    with pytest.raises(TypeError):
        layer.forward(x, out.half(), workspace=ws)
    q, s = _quantize(x)
    with pytest.raises(RuntimeError):
        ops.gemm_fp8(q, s, w, out.to(BF), ops.ADD)
    with pytest.raises(ValueError):
        ops.gemm_fp8(q, s[:1], w, out)
    with pytest.raises(TypeError):
        ops.gemm_fp8(q.view(torch.uint8), s, w, out)
    with pytest.raises(RuntimeError):
        ops.quantize_fp8(x, torch.zeros(4, 257, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn), s)      # rows off their 16-byte borders
    z, choice, weights = _rand(1, 4, 16), torch.full((4, 2), 7, dtype=torch.int32, device="cuda"), torch.full((2, 4), 7.0, device="cuda")
    for kw in ({"groups": 3}, {"groups": 0}, {"groups": 4, "top_groups": 5}, {"groups": 16, "top_groups": 1}, {"groups": 4, "top_groups": 2, "group_best": 3}):
        with pytest.raises(RuntimeError):
            ops.route_experts(z, choice, weights, **kw)
    for bad in ((z.double(), choice, weights), (z, choice.long(), weights), (z, choice, weights.t()), (z[:3], choice, weights), (z, choice, weights.to(BF))):
        with pytest.raises((TypeError, ValueError)):
            ops.route_experts(*bad)
    with pytest.raises(ValueError):
        ops.route_experts(z, choice, weights, score="relu")
    with pytest.raises(RuntimeError):
        ops.route_experts(_rand(1, 4, 1025), choice, weights)
    experts, _ = _experts(4, 256, 128)
    y = torch.full((4, 256), 7.0, device="cuda")
    good = experts.scratch(4, 2)
    with pytest.raises(RuntimeError):
        experts.forward(x, choice, weights, y, good[:-1])
    with pytest.raises(ValueError):
        experts.forward(x[:, :128], choice, weights, y, good)
    with pytest.raises(ValueError):
        experts.forward(x, choice, weights.t().contiguous(), y, good)
    with pytest.raises(TypeError):
        experts.forward(x, choice.long(), weights, y, good)
    assert (out == 7.0).all() and (choice == 7).all() and (weights == 7.0).all() and (y == 7.0).all()


def test_no_tokens():
    from stride_b200.kernels import ops
    from stride_b200.kernels.linear import Linear
    Linear(_weight(2, 130, 256), BF).forward(_rand(1, 0, 256, dtype=BF), torch.empty(0, 130, device="cuda"), workspace=_workspace(4))
    choice, weights = torch.empty(0, 2, dtype=torch.int32, device="cuda"), torch.empty(2, 0, device="cuda")
    ops.route_experts(torch.empty(0, 8, device="cuda"), choice, weights)
    experts, _ = _experts(4, 256, 128)
    experts.forward(torch.empty(0, 256, device="cuda"), choice, weights, torch.empty(0, 256, device="cuda"), experts.scratch(0, 2))
    torch.cuda.synchronize()


def test_product_in_a_graph_and_on_another_stream():
    from stride_b200.kernels.linear import Linear
    x, layer, ws = _rand(3, 9, 640, dtype=BF), Linear(_weight(4, 512, 640), BF), _workspace(9)
    out, want = torch.empty(9, 512, device="cuda"), torch.empty(9, 512, device="cuda")
    layer.forward(x, want, workspace=ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.forward(x, out, workspace=ws)
    side.synchronize()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.forward(x, out, workspace=ws)
    x.copy_(_rand(5, 9, 640, dtype=BF))
    layer.forward(x, want, workspace=ws)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


# ------------------------------------------------------------------ routing
ROUTES = [(1, 8, 2, {}), (5, 1, 1, {}), (33, 90, 6, {"score": "softmax", "renormalise": False}), (200, 256, 8, {"groups": 8, "top_groups": 4, "scale": 2.5}),
          (64, 160, 6, {"score": "softmax", "groups": 8, "top_groups": 3, "group_best": 1, "renormalise": False, "scale": 16.0}),
          (40, 1024, 32, {"groups": 32, "top_groups": 5}), (17, 33, 33 - 1, {}), (9, 12, 3, {"groups": 4, "top_groups": 1}), (100, 511, 9, {"score": "softmax"}),
          (7, 6, 2, {"groups": 6, "top_groups": 2})]


def _route(z, top, bias=None, **kw):
    from stride_b200.kernels import ops
    n = z.shape[0]
    choice = torch.full((n, top), -7, dtype=torch.int32, device="cuda")
    weights = torch.full((top, n), float("nan"), device="cuda")
    ops.route_experts(z, choice, weights, bias=bias, **kw)
    return choice.cpu(), weights.cpu()


def _close(weights, want):
    return ((weights.to(F64) - want).abs() <= 2.0 ** -20 * want.abs() + 1e-37).all()


@pytest.mark.parametrize("n,E,top,kw", ROUTES)
@pytest.mark.parametrize("biased", [False, True])
def test_routes(n, E, top, kw, biased):
    z = _rand(E, n, E, std=1.5)
    bias = _rand(E + 1, E, std=0.1) if biased else None
    choice, weights = _route(z, top, bias, **kw)
    want, want_weights = plain.route(z.cpu(), top, kw.get("score", "sigmoid"), None if bias is None else bias.cpu(), **{k: v for k, v in kw.items() if k != "score"})
    assert torch.equal(choice, want)
    assert _close(weights, want_weights)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("kw", [{}, {"groups": 4, "top_groups": 2}])
def test_routes_with_ties_masks_and_odd_logits(score, kw):
    """Equal logits, experts switched off by their logit or their bias, rows with fewer experts than places or none, infinities, NaN, the largest and
    the smallest floats."""
    z = _rand(3, 12, 32)
    z[0] = 0.25
    z[1] = torch.arange(32, device="cuda") // 5
    z[2] = float("-inf")
    z[3, 3:] = float("-inf")
    z[4] = float("nan")
    z[5, ::2] = float("nan")
    z[6, 7] = float("inf")
    z[7, 7], z[7, 20] = float("inf"), float("inf")
    z[8] = -3.0e38
    z[9] = 3.0e38
    z[10] = torch.linspace(30, 45, 32, device="cuda")
    z[11, 1:] = float("-inf")
    bias = _rand(4, 32, std=0.1)
    bias[5], bias[9] = float("-inf"), float("nan")
    for b in (None, bias):
        choice, weights = _route(z, 6, b, score=score, **kw)
        want, want_weights = plain.route(z.cpu(), 6, score, None if b is None else b.cpu(), **kw)
        assert torch.equal(choice, want)
        assert _close(weights, want_weights)


def test_routes_that_only_64_bits_tell_apart():
    """Scores plus bias that differ by less than half a 32-bit step of their size: the larger wins, whatever its place."""
    z = torch.zeros(64, 40, device="cuda")
    z += torch.arange(40, device="cuda") * 2.0 ** -26 * (1 - 2 * (torch.arange(64, device="cuda") % 2))[:, None]
    bias = torch.full((40,), 4.0, device="cuda")
    for kw in ({}, {"score": "softmax"}, {"groups": 4, "top_groups": 2}):
        choice, _ = _route(z, 7, bias, **kw)
        want, _ = plain.route(z.cpu(), 7, kw.get("score", "sigmoid"), bias.cpu(), **{k: v for k, v in kw.items() if k != "score"})
        assert torch.equal(choice, want), kw


@pytest.mark.parametrize("E,kw", [(256, {"groups": 8, "top_groups": 4}), (64, {"groups": 4, "top_groups": 1, "group_best": 1}), (160, {"groups": 5, "top_groups": 2}),
                                  (256, {}), (96, {"score": "softmax"}), (64, {"score": "softmax", "groups": 4, "top_groups": 2}), (512, {"groups": 2})])
@pytest.mark.parametrize("biased", [False, True])
def test_routes_whose_candidates_or_groups_are_next_to_equal(E, kw, biased):
    """Some logits one 32-bit step from one another, all over the row or a group's beside another's; few rows of them and whole rows."""
    n, groups = 48, kw.get("groups", 1)
    z = _rand(E, n, E, std=1.0)
    bias = (_rand(E + 1, E, std=0.1) if groups == 1 else _rand(E + 1, E // groups, std=0.1).repeat(groups)) if biased else None
    up = torch.tensor(float("inf"), device="cuda")
    size = E // groups
    for row in range(0, n, 3):                         # a group like its neighbour, one of its logits a step further on
        first = z[row, :size].clone() if groups > 1 else z[row, :E // 2].clone()
        z[row, size * (groups > 1) or E // 2:][:first.numel()] = first
        at = first.topk(2).indices[row % 2]
        z[row, at] = torch.nextafter(z[row, at], up)
    for row in range(1, n, 3):                         # the largest ones within a few steps
        at = z[row].topk(12 if row % 2 else 40).indices
        top = z[row].max()
        for i, a in enumerate(at.flip(0)):
            z[row, a] = top
            if i % 2:
                top = torch.nextafter(top, up)
    choice, weights = _route(z, 8, bias, **kw)
    want, want_weights = plain.route(z.cpu(), 8, kw.get("score", "sigmoid"), None if bias is None else bias.cpu(), **{k: v for k, v in kw.items() if k != "score"})
    assert torch.equal(choice, want)
    assert _close(weights, want_weights)


def test_routes_of_rows_of_a_wider_tensor():
    from stride_b200.kernels import ops
    wide = _rand(6, 21, 77)
    z = wide[:, 3:51]
    choice, weights = torch.empty(21, 4, dtype=torch.int32, device="cuda"), torch.full((4, 30), 7.0, device="cuda")
    ops.route_experts(z, choice, weights[:, 2:23])
    want, want_weights = plain.route(z.cpu(), 4, "sigmoid")
    assert torch.equal(choice.cpu(), want)
    assert _close(weights[:, 2:23].cpu(), want_weights)
    weights[:, 2:23] = 7.0
    assert (weights == 7.0).all()


# ------------------------------------------------------------------ experts
def _experts(E, W, F, seed=0):
    from stride_b200.kernels.linear import Fp8Experts
    gate, up, down = ([_weight(seed + 1000 * k + e, *shape) for e in range(E)] for k, shape in ((1, (F, W)), (2, (F, W)), (3, (W, F))))
    layer = Fp8Experts([w for pair in zip(gate, up) for w in pair], down)
    return layer, [[_values(w) for w in ws] for ws in (gate, up, down)]


def _choices(seed, n, E, top, missing=0.0):
    g = torch.Generator().manual_seed(seed)
    choice = torch.rand(n, E, generator=g).add(torch.linspace(0, 0.5, E)).argsort(dim=1, descending=True)[:, :top].to(torch.int32)
    choice[torch.rand(n, top, generator=g) < missing] = -1
    return choice.contiguous().cuda(), torch.rand(top, n, generator=g).cuda()


EXPERTS = [(1, 4, 2, 128, 128, 0.0), (1, 64, 6, 256, 200, 0.0), (3, 8, 3, 300, 100, 0.3), (32, 8, 2, 512, 384, 0.0), (64, 3, 3, 200, 70, 0.2),
           (257, 16, 4, 256, 520, 0.1), (1000, 4, 1, 384, 256, 0.5), (500, 40, 6, 640, 260, 0.0),
           (3000, 16, 6, 128, 128, 0.1)]


@pytest.mark.parametrize("n,E,top,W,F,missing", EXPERTS)
@pytest.mark.parametrize("x_dtype,out_dtype", [(BF, BF), (F32, F32)])
def test_experts(n, E, top, W, F, missing, x_dtype, out_dtype):
    """Ids that are no expert's have no term; a token without any gets zeros."""
    layer, (gate, up, down) = _experts(E, W, F)
    x = _rand(n, n, W, dtype=x_dtype)
    choice, weights = _choices(n, n, E, top, missing)
    if n > 2:
        choice[1], choice[2, 0] = -1, E
    out = torch.full((n, W), float("nan"), dtype=out_dtype, device="cuda")
    layer.forward(x, choice, weights, out, layer.scratch(n, top))
    want, bound = plain.experts(x.to(F64), choice, weights, gate, up, down)
    assert ((out.to(F64) - want).abs() <= bound + HALF_STEP[out_dtype] * (want.abs() + bound)).all()
    if n > 2:
        assert (out[1] == 0).all()


@pytest.mark.parametrize("n", [2, 40, 300])
def test_an_expert_chosen_twice_and_one_chosen_by_all(n):
    """The same id in several of a token's places counts as often; all tokens on one expert, the others idle."""
    layer, (gate, up, down) = _experts(3, 256, 160)
    x = _rand(n, n, 256, dtype=BF)
    choice = torch.full((n, 3), 1, dtype=torch.int32, device="cuda")
    choice[0] = torch.tensor([2, 2, 0], dtype=torch.int32)
    weights = _rand(4, 3, n).abs()
    out = torch.empty(n, 256, device="cuda")
    layer.forward(x, choice, weights, out, layer.scratch(n, 3))
    want, bound = plain.experts(x.to(F64), choice, weights, gate, up, down)
    assert ((out.to(F64) - want).abs() <= bound).all()


def test_two_streams_at_once():
    """Two layers' and two experts' calls side by side, each with buffers of its own."""
    from stride_b200.kernels.linear import Linear
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    linear = [Linear(_weight(20 + i, 2048, 1024), BF) for i in range(2)]
    experts = [_experts(8, 256, 264, seed=5000 * i)[0] for i in range(2)]
    x, rows = [_rand(30 + i, 70, 1024, dtype=BF) for i in range(2)], [_rand(40 + i, 70, 256, dtype=BF) for i in range(2)]
    routes = [_choices(50 + i, 70, 8, 2) for i in range(2)]
    work, scratch = [_workspace(70) for _ in range(2)], [experts[i].scratch(70, 2) for i in range(2)]
    alone, out = ([(torch.empty(70, 2048, device="cuda"), torch.empty(70, 256, device="cuda")) for _ in range(2)] for _ in range(2))
    for i in range(2):
        linear[i].forward(x[i], alone[i][0], workspace=work[i])
        experts[i].forward(rows[i], *routes[i], alone[i][1], scratch[i])
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                linear[i].forward(x[i], out[i][0], workspace=work[i])
                experts[i].forward(rows[i], *routes[i], out[i][1], scratch[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(out[i][0], alone[i][0]) and torch.equal(out[i][1], alone[i][1])


@pytest.mark.parametrize("n,E,top,offset", [(1, 1, 1, 0), (1, 64, 32, 0), (4, 5, 8, 0), (16, 2, 2, 0), (32, 70, 1, 0), (11, 5, 3, 0), (5, 6, 6, 1), (33, 40, 1, 0),
                                            (31, 2, 1, 0), (6, 200, 5, 0)])
def test_experts_of_few_choices(n, E, top, offset):
    """Around 32 choices in all, up to which no kernel puts them in order: an expert of more rows than a tile, ids that are no expert's, repeated ones, an
    input whose rows do not begin at 16 bytes; a call in a graph, replayed with other choices."""
    W, F = 256, 136
    layer, (gate, up, down) = _experts(E, W, F)
    x = _rand(n, n, W + offset, dtype=BF)[:, offset:]
    g = torch.Generator().manual_seed(n)
    choice, weights = torch.randint(0, E, (n, top), generator=g, dtype=torch.int32).cuda(), torch.rand(top, n, generator=g).cuda()
    scratch, out = layer.scratch(n, top), torch.empty(n, W, device="cuda")
    layer.forward(x, choice, weights, out, scratch)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.forward(x, choice, weights, out, scratch)
    for other in (choice.clone(), torch.zeros_like(choice), torch.full_like(choice, -1), torch.where(choice % 2 == 0, choice.flip(0), E + 3)):
        choice.copy_(other)
        out.fill_(float("nan"))
        graph.replay()
        want, bound = plain.experts(x.to(F64), choice, weights, gate, up, down)
        assert ((out.to(F64) - want).abs() <= bound + HALF_STEP[F32] * (want.abs() + bound)).all()


def test_experts_of_a_token_do_not_depend_on_the_step():
    """Alone, in a few and in many, whoever else chose the same experts; the same twice over the same scratch."""
    layer, _ = _experts(8, 384, 264)
    x = _rand(1, 400, 384, dtype=BF)
    choice, weights = _choices(2, 400, 8, 3)
    whole, again = torch.empty(400, 384, device="cuda"), torch.empty(400, 384, device="cuda")
    scratch = layer.scratch(400, 3)
    layer.forward(x, choice, weights, whole, scratch)
    layer.forward(x, choice, weights, again, scratch)
    assert torch.equal(whole, again)
    for first, n in [(0, 1), (9, 5), (100, 40), (200, 150), (0, 399)]:
        part = torch.full((n, 384), float("nan"), device="cuda")
        rows = slice(first, first + n)
        layer.forward(x[rows], choice[rows].contiguous(), weights[:, rows].contiguous(), part, scratch)
        assert torch.equal(part, whole[rows]), (first, n)


def test_router_and_experts_together():
    """As a feed-forward runs them: logits, choice and weights, the experts' products; in a captured graph, replayed with other inputs."""
    from stride_b200.kernels import ops
    E, W, F, n, top = 16, 256, 192, 37, 4
    layer, (gate, up, down) = _experts(E, W, F)
    router, bias = _rand(3, E, W, std=W ** -0.5), _rand(4, E, std=0.05)
    x = _rand(5, n, W, dtype=BF)
    logits, choice = torch.empty(n, E, device="cuda"), torch.empty(n, top, dtype=torch.int32, device="cuda")
    weights, out, scratch = torch.empty(top, n, device="cuda"), torch.empty(n, W, dtype=BF, device="cuda"), layer.scratch(n, top)

    def run():
        ops.gemm_f32(x, router, logits)
        ops.route_experts(logits, choice, weights, bias=bias, groups=4, top_groups=2, scale=2.0)
        layer.forward(x, choice, weights, out, scratch)

    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for seed in (6, 7):
        x.copy_(_rand(seed, n, W, dtype=BF))
        graph.replay()
        torch.cuda.synchronize()
        want_choice, want_weights = plain.route(logits.cpu(), top, "sigmoid", bias.cpu(), 4, 2, 2, True, 2.0)
        assert torch.equal(choice.cpu(), want_choice)
        want, bound = plain.experts(x.to(F64), choice, want_weights.cuda(), gate, up, down)
        bound = bound + 2.0 ** -20 * want.abs().amax()
        assert ((out.to(F64) - want).abs() <= bound + 2.0 ** -8 * (want.abs() + bound)).all()


@pytest.mark.parametrize("E,groups", [(8, 4), (12, 4), (64, 4), (160, 5), (256, 8)])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_groups_whose_best_two_sum_beyond_the_floats(E, groups, score):
    """Experts pushed down by biases of the lowest float, or up by the largest: groups judged by sums that 32 bits do not hold, beside groups in which
    every expert is switched off."""
    low, size = torch.finfo(F32).min, E // groups
    z = _rand(E, 5, E)
    for biases in ([None, low, None, None], [None, low, None, -3.0e38], [-3.2e38, low, None, -3.0e38], [0.0, None, -low, 3.0e38], [low, -low, low, low]):
        bias = torch.full((E,), float("-inf"), device="cuda")
        for g, value in enumerate(biases):
            if value is not None:
                bias[g * size:(g + 1) * size] = value
        for top_groups in (1, 2):
            kw = {"groups": groups, "top_groups": top_groups, "group_best": 2}
            choice, _ = _route(z, 2, bias, score=score, **kw)
            want, _ = plain.route(z.cpu(), 2, score, bias.cpu(), **kw)
            assert torch.equal(choice, want), (biases, top_groups)


@pytest.mark.parametrize("n", [1, 40, 100])
def test_a_lost_signal_can_be_read_and_the_products_run_again(n):
    """A caller without an engine: the word into which a wait that gave up reports (written by the host here) is read, and reset with that."""
    from stride_b200.kernels import ops
    from stride_b200.kernels.linear import Linear
    layer, x, work = Linear(_weight(1, 256, 2048), BF), _rand(2, n, 2048, dtype=BF), _workspace(n)
    want, out = torch.empty(n, 256, device="cuda"), torch.zeros(n, 256, device="cuda")
    layer.forward(x, want, workspace=work)
    assert ops.gemm_fp8_status() == 0
    ops.shared_status_word({"gemm_fp8"}).fill_(45)
    layer.forward(x, out, workspace=work)
    torch.cuda.synchronize()
    assert (out == 0).all()
    assert ops.gemm_fp8_status() == 45
    assert ops.gemm_fp8_status() == 0
    layer.forward(x, out, workspace=work)
    assert torch.equal(out, want)


@pytest.mark.parametrize("n,M,K", [(1100, 12000, 1300), (300, 20000, 2048)])
@pytest.mark.parametrize("gated", [False, True])
def test_wide_tiles_walked_in_several_rounds(n, M, K, gated):
    """CTAs and pairs that walk tiles of 256 weight rows, with waits for accumulators that are never there yet: the same bits every time, and a few
    tokens' in a step of their own."""
    from stride_b200.kernels.linear import Fp8Weight, Linear
    layer = Linear(Fp8Weight.stack([_weight(1, M // 2, K), _weight(2, M // 2, K)]) if gated else _weight(1, M, K), BF)
    x, work = _rand(3, n, K, dtype=BF), _workspace(n)
    call = (lambda x, out: layer.forward_swiglu(x, out, None, workspace=work)) if gated else (lambda x, out: layer.forward(x, out, workspace=work))
    want = torch.empty(n, M // 2 if gated else M, device="cuda")
    call(x, want)
    few = torch.empty(9, want.shape[1], device="cuda")
    call(x[n - 9:], few)
    assert torch.equal(few, want[n - 9:])
    for _ in range(10):
        out = torch.full_like(want, float("nan"))
        call(x, out)
        assert torch.equal(out, want)


@pytest.mark.parametrize("E,top", [(8, 4), (2, 2), (40, 8), (16, 8)])
def test_experts_keep_within_their_scratch(E, top):
    """Around the number of choices from which tiles of rows are walked (a mean of eight, or of sixteen and 256 in all), with scratch of just the bytes
    that are asked for and a border behind it; a buffer for more tokens serves fewer."""
    W, F = 256, 136
    layer, (gate, up, down) = _experts(E, W, F)
    border = max(8 * E, min(16 * E, 256)) // top
    sizes = [layer.scratch(n, top).numel() for n in range(0, 2 * border + 40)]
    assert sizes == sorted(sizes)
    for n in (1, border - 1, border, border + 1, border + 33):
        choice, weights = _choices(n, n, E, top)
        for offset in (0, 1):                      # (rows off 16-byte borders: quantised by a kernel of its own in either form)
            rows = _rand(n, n, W + offset, dtype=BF)[:, offset:]
            whole = torch.full((layer.scratch(n, top).numel() + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
            out = torch.empty(n, W, device="cuda")
            layer.forward(rows, choice, weights, out, whole[:-4096])
            assert (whole[-4096:] == 0xA5).all()
            want, bound = plain.experts(rows.to(F64), choice, weights, gate, up, down)
            assert ((out.to(F64) - want).abs() <= bound + HALF_STEP[F32] * (want.abs() + bound)).all()
            large = torch.empty(sizes[-1], dtype=torch.uint8, device="cuda")
            again = torch.empty(n, W, device="cuda")
            layer.forward(rows, choice, weights, again, large)
            assert torch.equal(again, out)


def test_scratch_of_many_tokens_has_no_room_for_what_few_need():
    """32-bit gated products are kept for few choices only: a long step's scratch is what its 8-bit rows, their scales and the results take."""
    from stride_b200.kernels import ops
    n, top, E, W, F = 8192, 8, 256, 7168, 2048
    pairs = n * top
    used = pairs * (W + 4 * (W // 128) + F + 4 * (F // 128) + 4 * W + 4 * 5)
    assert ops.experts_fp8_scratch(n, top, E, W, F) <= used + 2 * 8 * E * 4 * F + 4096


@pytest.mark.parametrize("E", [8, 40, 256])
def test_weights_below_the_smallest_normal_float(E):
    """Sigmoids of far negative logits, taken as they are: within the exponential's two units and the type's smallest step of e^z."""
    z = torch.linspace(-106.0, -70.0, E, device="cuda")[None].repeat(3, 1)
    z[1] = -95.0
    z[2, : E // 2] = float("-inf")
    choice, weights = _route(z, 4, renormalise=False, scale=0.5)
    want, want_weights = plain.route(z.cpu(), 4, "sigmoid", renormalise=False, scale=0.5)
    assert torch.equal(choice, want)
    # (s is off by 2 units of 2^-23 and a rounding to the smallest step, 2^-149; times the scale, rounded to that step again)
    assert ((weights.to(F64) - want_weights).abs() <= 2.0 ** -21 * want_weights + 2.0 ** -149).all()
    choice, weights = _route(z, 4, renormalise=True)
    assert _close(weights, plain.route(z.cpu(), 4, "sigmoid")[1])
    z = torch.full((1, E), -95.0, device="cuda")
    assert (_route(z, 2, renormalise=False)[1] > 0).all()


@pytest.mark.parametrize("E", [7, 32, 90, 256])
@pytest.mark.parametrize("renormalise", [False, True])
def test_softmax_weights_far_below_the_largest(E, renormalise):
    """Logits whose distance from the largest is no float: its rounding is made good again, so that a far weight is as exact as a near one."""
    n, top, per = 64, min(E, 6), 1 if E <= 32 else 4 if E <= 128 else 8
    z = _rand(E, n, E, std=2.0)
    z[:, :top] -= torch.rand(n, top, generator=torch.Generator("cuda").manual_seed(E), device="cuda") * 70.0 + 8.0
    bias = torch.zeros(E, device="cuda")
    bias[:top] = 4.0
    choice, weights = _route(z, top, bias, score="softmax", renormalise=renormalise)
    want, want_weights = plain.route(z.cpu(), top, "softmax", bias.cpu(), renormalise=renormalise)
    assert torch.equal(choice, want)
    # two units of the exponential and two roundings around it, above and below the line; up to 8 + per additions; two divisions, the scale
    assert ((weights.to(F64) - want_weights).abs() <= (2 * 6 + 8 + per + 3) * 2.0 ** -24 * want_weights + 2.0 ** -149).all()


@pytest.mark.parametrize("n,E,top", [(2100, 256, 8), (5000, 256, 8), (300, 1024, 8), (1200, 1024, 32)])
def test_many_experts_of_many_choices(n, E, top):
    """Hundreds of experts, few rows each and many, beyond the choices that are put in order from registers."""
    layer, (gate, up, down) = _experts(E, 144, 72)
    x = _rand(n, n, 144, dtype=BF)
    choice, weights = _choices(n, n, E, top, 0.02)
    out = torch.empty(n, 144, device="cuda")
    layer.forward(x, choice, weights, out, layer.scratch(n, top))
    want, bound = plain.experts(x.to(F64), choice, weights, gate, up, down)
    assert ((out.to(F64) - want).abs() <= bound + HALF_STEP[F32] * (want.abs() + bound)).all()
