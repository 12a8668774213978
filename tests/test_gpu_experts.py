"""Routed experts on the GPU: the router, the grouped int8 product, the combine, and the layer they make.

The router's integers and the grouped product (exact int32 sums, then one fp32 rounding per operation) have to
be equal bit for bit; the router's weights and the combine are held to bounds derived at their checks.
"""
from __future__ import annotations

import math

import pytest
import torch

from tilegen_b200 import _lib, ops
from tilegen_b200.quant import int8_expert_ffn, quantize_convrot_expert_weights

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _healthy_device(cuda):
    yield
    assert _lib.device_status(0) == 0


def _gen(seed, dev="cuda"):
    return torch.Generator(device=dev).manual_seed(seed)


# ---------------------------------------------------------------- router
def _route_ref(logits, top_k, renormalize):
    """The router in 64 bits, on the host."""
    x = logits.detach().cpu().double()
    t, e = x.shape
    value, ids = torch.sort(x, dim=1, descending=True, stable=True)
    value, ids = value[:, :top_k], ids[:, :top_k]
    top = torch.where(torch.isneginf(value[:, :1]), 0.0, value[:, :1])
    w = torch.exp(value - top)
    s = (w if renormalize else torch.exp(x - top)).sum(1, keepdim=True)
    live = ~torch.isneginf(value)
    w = torch.where(live, w / s, 0.0)
    place = torch.full((t, top_k), -1, dtype=torch.int64)
    groups = [[] for _ in range(e)]
    for i in range(t):
        for j in range(top_k):
            if live[i, j]:
                groups[ids[i, j]].append((i, j))
    rows, offsets = [], [0]
    for g in groups:
        for i, j in g:
            place[i, j] = len(rows)
            rows.append(i)
        offsets.append(len(rows))
    rows += [-1] * (t * top_k - len(rows))
    return w, torch.where(live, ids, -1), offsets, rows, place, value - top


def _check_route(logits, top_k, renormalize):
    got = ops.route_experts(logits, top_k, renormalize)
    w, ids, offsets, rows, place, d = _route_ref(logits, top_k, renormalize)
    assert torch.equal(got.ids.cpu().long(), ids)
    assert got.offsets.tolist() == offsets
    assert got.rows.tolist() == rows
    assert torch.equal(got.place.cpu().long(), place)
    # exp's argument is rounded once (|d| 2^-24 of exp), expf is within 2 ulp, the sum of up to E terms and the
    # division add E + 2 roundings; the terms' own errors weigh in the sum by their share (|d| exp(d) < 8 in all).
    # Where d is -inf the weight is exp(-inf) = 0 exactly, and |d| 2^-24 of it is 0 (not inf * 0).
    e = logits.shape[1]
    tol = 2.0 ** -24 * (torch.where(d.isinf(), 0.0, d.abs()) + e + 20) * w + 1e-37
    bad = ~((got.weights.cpu().double() - w).abs() <= tol) & ~(got.weights.cpu().isnan() & w.isnan())
    assert not bad.any(), f"weights off at {bad.nonzero()[:3].tolist()}"
    return got


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("t,e,top_k", [(1, 1, 1), (1, 64, 8), (2, 2, 2), (3, 33, 5), (31, 32, 32), (32, 8, 2), (33, 128, 8), (257, 31, 3),
                                       (1000, 64, 6), (700, 1024, 10), (1, 1024, 32), (4097, 16, 2)])
def test_route_shapes(cuda, t, e, top_k, renormalize):
    _check_route(torch.randn(t, e, generator=_gen(t + e), device=cuda), top_k, renormalize)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_route_ties_go_to_the_lower_index(cuda, dtype):
    g = _gen(4)
    x = torch.randint(-2, 3, (300, 48), generator=g, device=cuda).to(dtype)
    x[5] = 0
    x[6, ::2] = -0.0  # -0 and +0 are equal
    x[6, 1::2] = 0.0
    _check_route(x, 7, True)
    _check_route(x, 32, False)


@pytest.mark.parametrize("renormalize", [True, False])
def test_route_masks(cuda, renormalize):
    """Closed experts, padded tokens, fewer open experts than top_k, the lowest finite value, NaN and +inf."""
    x = torch.randn(200, 20, generator=_gen(7), device=cuda)
    x[::7] = -math.inf
    x[3, :18] = -math.inf
    x[4, 1:] = -math.inf
    x[:, 9] = -math.inf
    x[10] = torch.finfo(torch.float32).min
    x[11, 4:] = torch.finfo(torch.float32).min
    x[12, 3] = math.inf
    x[13, 5] = math.nan
    x[13, 2] = math.nan
    got = _check_route(x, 4, renormalize)
    live = int(got.offsets[-1])
    assert live < 800 and (got.rows[live:] == -1).all()


def test_route_every_token_masked(cuda):
    got = _check_route(torch.full((77, 6), -math.inf, device=cuda), 2, True)
    assert int(got.offsets[-1]) == 0 and (got.weights == 0).all()


def test_route_all_to_one_expert(cuda):
    x = torch.zeros(5000, 8, device=cuda)
    x[:, 6] = 1
    got = _check_route(x, 1, True)
    assert got.offsets.tolist() == [0] * 7 + [5000, 5000] and got.rows.tolist() == list(range(5000))


def test_route_no_tokens_strides_and_refusals(cuda):
    got = ops.route_experts(torch.empty(0, 5, device=cuda), 2)
    assert got.offsets.tolist() == [0] * 6 and got.rows.shape == (0,) and got.ids.shape == (0, 2)
    x = torch.randn(64, 40, generator=_gen(3), device=cuda)
    for a, b in zip(ops.route_experts(x[:, 4:20], 3), ops.route_experts(x[:, 4:20].clone(), 3)):
        assert torch.equal(a, b)
    for a, b in zip(ops.route_experts(x.t(), 3), ops.route_experts(x.t().contiguous(), 3)):
        assert torch.equal(a, b)
    for args, match in [((x, 0), "top_k"), ((x, 41), "top_k"), ((torch.zeros(2, 1025, device=cuda), 2), "experts"),
                        ((torch.zeros(2, 64, device=cuda), 33), "top_k"), ((x.double(), 2), "logits"), ((x[0], 2), "logits"),
                        ((x.clone().requires_grad_(), 2), "gradient")]:
        with pytest.raises(ValueError, match=match):
            ops.route_experts(*args)


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("e,top_k,dtype", [(1, 1, torch.float32), (2, 2, torch.float16), (31, 2, torch.float32), (32, 1, torch.bfloat16), (33, 4, torch.float32),
                                           (64, 3, torch.bfloat16), (128, 8, torch.float16)])
def test_route_many_tokens_few_experts(cuda, e, top_k, dtype, renormalize):
    """From 16384 tokens a thread takes a token: ties, closed experts, padded tokens, NaN, the last warp part-filled."""
    t = 16384 + 45
    x = (torch.randn(t, e, generator=_gen(e), device=cuda) * 4).round().mul(0.5).to(dtype)  # many equal logits
    x[::11] = -math.inf
    x[1::13, e // 2] = -math.inf
    x[5, 0] = math.nan
    x[6, e - 1] = math.inf
    x[t - 1] = 0
    _check_route(x, top_k, renormalize)


def test_route_many_tokens(cuda):
    """65521 tokens against torch's own sorts (integers only)."""
    t, e, top_k = 65521, 160, 6
    x = torch.randn(t, e, generator=_gen(8), device=cuda)
    got = ops.route_experts(x, top_k)
    ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top_k]
    assert torch.equal(got.ids.long(), ids)
    key, order = torch.sort(ids.reshape(-1), stable=True)
    assert torch.equal(got.rows.long(), order // top_k)
    assert torch.equal(got.place.view(-1).long()[order], torch.arange(t * top_k, device=cuda))
    assert torch.equal(got.offsets[1:].long(), torch.bincount(key, minlength=e).cumsum(0))


# ---------------------------------------------------------------- grouped product
def _group_case(counts, n, k, m=None, bias_dtype=None, scales="full", seed=0, dev="cuda"):
    """Groups of the given sizes; with ``m``, the rows are gathered from ``m`` activation rows."""
    g = _gen(seed)
    e, r = len(counts), sum(counts)
    xq = torch.randint(-128, 128, (r if m is None else m, k), generator=g, dtype=torch.int8, device=dev)
    wq = torch.randint(-128, 128, (e, n, k), generator=g, dtype=torch.int8, device=dev)
    xs = torch.rand(xq.shape[0], generator=g, device=dev) * 0.02 + 1e-4
    ws = torch.rand({"full": (e, n), "expert": (e,), "one": (1,)}[scales], generator=g, device=dev) * 0.01 + 1e-5
    bias = None if bias_dtype is None else torch.randn(e, n, generator=g, device=dev).to(bias_dtype)
    rows = None if m is None else torch.randint(0, m, (r,), generator=g, dtype=torch.int32, device=dev)
    offsets = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32, device=dev)
    return xq, xs, wq, ws, bias, offsets, rows


def _group_ref(xq, xs, wq, ws, bias, offsets, rows, dtype):
    """Expert by expert: int8 products summed exactly in fp64, then the fp32 sequence."""
    at = torch.arange(xq.shape[0], device=xq.device) if rows is None else rows.long()
    out = []
    bounds = offsets.tolist()
    for e in range(wq.shape[0]):
        a = at[bounds[e]:bounds[e + 1]]
        acc = (xq[a].double() @ wq[e].double().t()).float()
        scale = ws if ws.numel() == 1 else ws[e]
        y = acc * xs[a][:, None] * scale
        out.append((y if bias is None else y + bias[e].float()).to(dtype))
    return torch.cat(out)


def _check_group(case, dtype):
    xq, xs, wq, ws, bias, offsets, rows = case
    y = ops.int8_grouped_gemm_dequant(xq, xs, wq, ws, bias, offsets, dtype, rows=rows)
    ref = _group_ref(*case, dtype)
    live = int(offsets[-1])
    bad = (y[:live] != ref).nonzero()
    assert bad.numel() == 0, f"{len(bad)} of {ref.numel()} outputs differ, first at {bad[:3].tolist()}"


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("counts", [[1], [0, 1], [5, 0, 0, 3], [1, 1, 1, 1, 1, 1, 1, 1], [128], [127, 1, 129], [64, 65, 63], [300, 0, 7, 256, 257],
                                    [16, 17, 15, 33, 31], [0] * 30 + [3, 1], [1000, 24]])
def test_grouped_counts(cuda, counts, gather):
    _check_group(_group_case(counts, 200, 304, 50 if gather else None, seed=sum(counts)), torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bias_dtype", [None, torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scales", ["full", "expert", "one"])
@pytest.mark.parametrize("counts", [[3, 0, 2], [150, 20, 400]])
def test_grouped_types(cuda, dtype, bias_dtype, scales, counts):
    _check_group(_group_case(counts, 136, 512, 40, bias_dtype, scales, seed=5), dtype)


@pytest.mark.parametrize("n,k", [(8, 16), (16, 48), (520, 1040), (1536, 2048), (264, 5120), (5120, 176)])
@pytest.mark.parametrize("counts", [[2, 1, 0, 1], [70, 90, 20], [600, 520]])
def test_grouped_shapes(cuda, n, k, counts):
    for m in (None, 33):
        _check_group(_group_case(counts, n, k, m, seed=n + k), torch.bfloat16)


@pytest.mark.parametrize("e,most", [(128, 1), (1024, 3), (64, 40), (7, 900)])
def test_grouped_random_counts(cuda, e, most):
    counts = torch.randint(0, most + 1, (e,), generator=torch.Generator().manual_seed(e)).tolist()
    counts[0] += 1
    _check_group(_group_case(counts, 96, 256, 200, seed=e), torch.float16)


def test_grouped_rows_behind_the_last_group_stay(cuda):
    """Rows of out that no group covers -- behind the last, before the first -- keep what they held."""
    for counts in ([3, 0, 5], [200, 40]):
        xq, xs, wq, ws, bias, offsets, _ = _group_case(counts, 64, 128, seed=1)
        live = sum(counts)
        rows = torch.cat([torch.arange(live, device=cuda, dtype=torch.int32), torch.full((150,), -1, device=cuda, dtype=torch.int32)])
        out = torch.full((live + 150, 64), 7.0, device=cuda)
        y = ops.int8_grouped_gemm_dequant(xq, xs, wq, ws, bias, offsets, torch.float32, rows=rows, out=out)
        assert y is out and (out[live:] == 7).all()
        assert torch.equal(out[:live], _group_ref(xq, xs, wq, ws, bias, offsets, None, torch.float32))
        offsets = offsets.clone()
        offsets[0] = 2
        out.fill_(7)
        ops.int8_grouped_gemm_dequant(xq, xs, wq, ws, bias, offsets, torch.float32, rows=rows, out=out)
        assert (out[:2] == 7).all() and (out[live:] == 7).all()
        offsets.fill_(0)
        out.fill_(7)
        ops.int8_grouped_gemm_dequant(xq, xs, wq, ws, bias, offsets, torch.float32, rows=rows, out=out)
        assert (out == 7).all()


def test_grouped_bad_indices_are_zero_rows(cuda):
    """A row index outside [0, M) stands for a row of zeros; offsets are read as min(max(., 0), R)."""
    for counts in ([3, 4], [130, 200]):
        case = _group_case(counts, 64, 128, 20, torch.float32, seed=2)
        xq, xs, wq, ws, bias, offsets, rows = case
        rows[1], rows[4], rows[sum(counts) - 1] = -1, 20, 2 ** 31 - 1
        y = ops.int8_grouped_gemm_dequant(xq, xs, wq, ws, bias, offsets, torch.float32, rows=rows)
        ok = rows.clone()
        ok[(rows < 0) | (rows >= 20)] = 0
        ref = _group_ref(xq, xs, wq, ws, bias, offsets, ok, torch.float32)
        expert = torch.repeat_interleave(torch.arange(2, device=cuda), torch.tensor(counts, device=cuda))
        ref = torch.where(((rows < 0) | (rows >= 20))[:, None], bias[expert], ref)
        assert torch.equal(y, ref)
        wild = offsets.clone()
        wild[0], wild[2] = -5, 10 ** 6
        assert torch.equal(ops.int8_grouped_gemm_dequant(xq, xs, wq, ws, bias, wild, torch.float32, rows=rows), y)


def test_grouped_rows_gathered_first(cuda):
    """Products large enough that the rows are gathered by a pass of their own, bad row numbers among them."""
    counts, n, k, m = [2600, 0, 1500, 4000], 4096, 4096, 3000
    assert _lib.lib().tg_int8_grouped_gemm_dequant_workspace(sum(counts), 4, n, k) > 0
    case = _group_case(counts, n, k, m, torch.bfloat16, seed=4)
    xq, xs, wq, ws, bias, offsets, rows = case
    _check_group(case, torch.float16)
    rows[3], rows[2600], rows[-1] = -1, m, -2 ** 31
    y = ops.int8_grouped_gemm_dequant(xq, xs, wq, ws, bias, offsets, torch.float32, rows=rows)
    for r, e in ((3, 0), (2600, 2), (sum(counts) - 1, 3)):
        assert torch.equal(y[r], bias[e].float())
    live = torch.ones_like(rows, dtype=torch.bool)
    live[[3, 2600, -1]] = False
    rows[~live] = 0
    assert torch.equal(y[live], _group_ref(xq, xs, wq, ws, bias, offsets, rows, torch.float32)[live])


@pytest.mark.parametrize("m", [1, 9, 700])
def test_grouped_equals_the_single_linear(cuda, m):
    xq, xs, wq, ws, bias, offsets, _ = _group_case([m], 512, 1024, None, torch.float16, seed=m)
    a = ops.int8_grouped_gemm_dequant(xq, xs, wq, ws, bias, offsets, torch.float16)
    assert torch.equal(a, ops.int8_gemm_dequant(xq, xs, wq[0], ws[0], bias[0], torch.float16))


def test_grouped_past_32_bit_offsets(cuda):
    """Weights past 2^31 bytes: the last experts' rows are right, with few rows and with many."""
    e, n, k = 34, 13824, 5120
    wq = torch.zeros(e, n, k, dtype=torch.int8, device=cuda)
    g = _gen(11)
    wq[-1] = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8, device=cuda)
    for rows in (3, 300):
        xq = torch.randint(-128, 128, (rows, k), generator=g, dtype=torch.int8, device=cuda)
        xs, ws = torch.rand(rows, device=cuda), torch.rand(e, n, device=cuda)
        offsets = torch.zeros(e + 1, dtype=torch.int32, device=cuda)
        offsets[-1] = rows
        y = ops.int8_grouped_gemm_dequant(xq, xs, wq, ws, None, offsets, torch.float32)
        ref = (xq.double() @ wq[-1].double().t()).float() * xs[:, None] * ws[-1]
        assert torch.equal(y, ref)


def test_grouped_strides_and_refusals(cuda):
    xq, xs, wq, ws, bias, offsets, rows = _group_case([3, 4], 64, 128, 20, torch.float32, seed=2)
    f16 = torch.float16
    y = ops.int8_grouped_gemm_dequant(xq, xs, wq, ws, bias, offsets, f16, rows=rows)
    wide = torch.zeros(20, 200, dtype=torch.int8, device=cuda)
    wide[:, 5:133] = xq
    a = ops.int8_grouped_gemm_dequant(wide[:, 5:133], xs, wq.transpose(1, 2).contiguous().transpose(1, 2), ws, bias, offsets, f16,
                                      rows=rows.repeat_interleave(2)[::2])
    assert torch.equal(a, y)
    for args, kwargs, match in [((xq, xs, wq[0], ws, bias, offsets, f16), {}, "wq"), ((xq[:, :64], xs, wq, ws, bias, offsets, f16), {}, "match"),
                                ((xq, xs[:5], wq, ws, bias, offsets, f16), {}, "xscale"), ((xq, xs, wq, ws[:, :9], bias, offsets, f16), {}, "wscale"),
                                ((xq, xs, wq, ws, bias[:1], offsets, f16), {}, "bias"), ((xq, xs, wq, ws, bias, offsets[:2], f16), {}, "offsets"),
                                ((xq, xs, wq, ws, bias, offsets.long(), f16), {}, "offsets"), ((xq, xs, wq, ws, bias, offsets.cpu(), f16), {}, "offsets"),
                                ((xq, xs, wq, ws, bias, offsets, f16), {"rows": rows.long()}, "rows"), ((xq, xs, wq, ws, bias, offsets, torch.int8), {}, "out_dtype"),
                                ((xq, xs, wq, ws, bias, offsets, f16), {"out": torch.empty(3, 64, dtype=f16, device=cuda)}, "out"),
                                ((xq[:, :120], xs, wq[:, :, :120], ws, bias, offsets, f16), {}, "unsupported"),
                                ((xq, xs, wq[:, :60], ws[:, :60], bias[:, :60], offsets, f16), {}, "unsupported"),
                                ((xq, xs, wq, ws, bias.clone().requires_grad_(), offsets, f16), {}, "gradient")]:
        with pytest.raises(ValueError, match=match):
            ops.int8_grouped_gemm_dequant(*args, **kwargs)
    assert ops.int8_grouped_gemm_dequant(xq[:0], xs[:0], wq, ws, None, offsets, f16).shape == (0, 64)
    assert ops.int8_grouped_gemm_dequant(xq, xs, wq, ws, None, offsets, f16, rows=rows[:0]).shape == (0, 64)


def test_grouped_scale_shapes(cuda):
    """[E, N] scales by any of their unambiguous shapes; a transposed one, of as many elements, is refused."""
    xq, xs, wq, ws, bias, offsets, rows = _group_case([3, 4], 64, 128, 20, torch.float32, seed=2)
    y = ops.int8_grouped_gemm_dequant(xq, xs, wq, ws, bias, offsets, torch.float16, rows=rows)
    for same in (ws[..., None], ws.reshape(-1), ws.t().contiguous().t()):
        assert torch.equal(ops.int8_grouped_gemm_dequant(xq, xs, wq, same, bias, offsets, torch.float16, rows=rows), y)
    a = ops.int8_grouped_gemm_dequant(xq, xs, wq, ws[:, 0], bias, offsets, torch.float16, rows=rows)
    assert torch.equal(ops.int8_grouped_gemm_dequant(xq, xs, wq, ws[:, :1], bias, offsets, torch.float16, rows=rows), a)
    for bad in (ws.t(), ws.t().contiguous(), ws[0]):
        with pytest.raises(ValueError, match="wscale"):
            ops.int8_grouped_gemm_dequant(xq, xs, wq, bad, bias, offsets, torch.float16, rows=rows)


def test_deterministic_mode_fills_uncovered_rows(cuda):
    """torch's deterministic mode fills new memory: rows that no group covers are NaN, not what was there before."""
    xq, xs, wq, ws, bias, offsets, _ = _group_case([3, 4], 64, 128, seed=2)
    offsets[-1] = 5
    ref = ops.int8_grouped_gemm_dequant(xq, xs, wq, ws, bias, offsets, torch.float16)
    torch.use_deterministic_algorithms(True)
    try:
        y = ops.int8_grouped_gemm_dequant(xq, xs, wq, ws, bias, offsets, torch.float16)
    finally:
        torch.use_deterministic_algorithms(False)
    assert torch.equal(y[:5], ref[:5]) and y[5:].isnan().all()


# ---------------------------------------------------------------- combine
def _check_combine(y, place, weights, residual, out=None):
    got = ops.combine_experts(y, place, weights, residual=None if residual is None else residual.clone(), out=out)
    t, top_k = place.shape
    ref = torch.zeros(t, y.shape[1], dtype=torch.float64, device=y.device)
    mag = torch.zeros_like(ref)
    for j in range(top_k):
        at = place[:, j].long()
        ok = (at >= 0) & (at < y.shape[0])
        if y.shape[0]:
            term = torch.where(ok[:, None], weights[:, j].double()[:, None] * y[at.clamp(0, y.shape[0] - 1)].double(), 0.0)
            ref += term
            mag += term.abs()
    if residual is not None:
        ref += residual.double()
        mag += residual.double().abs()
    f = torch.finfo(y.dtype)
    # one fused multiply-add a term and one addition for the residual, each 2^-24 of a partial sum; one rounding to the type
    tol = (top_k + 1) * 2.0 ** -24 * mag + f.eps / 2 * ref.abs() * (1 + 2.0 ** -10) + f.tiny * f.eps
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} outputs off, first {bad.nonzero()[0].tolist()}"
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t,top_k,n", [(1, 1, 1), (1, 8, 5120), (3, 2, 7), (5, 32, 1000), (130, 4, 2049), (64, 3, 4096), (2, 5, 65537)])
def test_combine_shapes(cuda, dtype, t, top_k, n):
    g = _gen(t + n)
    r = t * top_k + 3
    y = torch.randn(r, n, generator=g, device=cuda).to(dtype)
    place = torch.randint(-1, r, (t, top_k), generator=g, dtype=torch.int32, device=cuda)
    w = torch.randn(t, top_k, generator=g, device=cuda)
    _check_combine(y, place, w, None)
    _check_combine(y, place, w, torch.randn(t, n, generator=g, device=cuda).to(dtype))


def test_combine_left_out_slots(cuda):
    """A slot left out adds nothing, whatever its weight and whatever the rows hold; the same row may come twice."""
    y = torch.randn(6, 40, generator=_gen(1), device=cuda)
    y[5] = math.nan
    w = torch.tensor([[0.5, math.nan], [math.inf, 2.0], [1.0, 1.0], [math.nan, math.inf]], device=cuda)
    place = torch.tensor([[3, -1], [6, 0], [2, 2], [2 ** 31 - 1, -2 ** 31]], dtype=torch.int32, device=cuda)
    got = ops.combine_experts(y, place, w)
    assert torch.equal(got[0], 0.5 * y[3]) and torch.equal(got[1], 2 * y[0]) and torch.equal(got[2], 2 * y[2])
    assert (got[3] == 0).all()
    res = torch.randn(4, 40, generator=_gen(2), device=cuda)
    assert torch.equal(ops.combine_experts(y, place, w, residual=res)[3], res[3])
    assert ops.combine_experts(y[:0], place, w, residual=res).equal(res)


def test_combine_in_place_strides_and_refusals(cuda):
    g = _gen(3)
    y, res = torch.randn(8, 96, generator=g, device=cuda).half(), torch.randn(4, 96, generator=g, device=cuda).half()
    place = torch.randint(0, 8, (4, 2), generator=g, dtype=torch.int32, device=cuda)
    w = torch.rand(4, 2, generator=g, device=cuda)
    ref = _check_combine(y, place, w, res)
    into = res.clone()
    assert ops.combine_experts(y, place, w, residual=into, out=into) is into and torch.equal(into, ref)
    # rows that start at odd addresses, a transposed y and place
    odd = torch.empty(4 * 96 + 1, dtype=torch.float16, device=cuda)[1:].view(4, 96)
    assert torch.equal(ops.combine_experts(y.t().contiguous().t(), place.t().contiguous().t(), w, residual=res, out=odd), ref)
    raw = torch.empty(8 * 96 + 1, dtype=torch.float16, device=cuda)[1:].view(8, 96)
    raw.copy_(y)
    assert torch.equal(ops.combine_experts(raw, place, w, residual=res), ref)
    for args, kwargs, match in [((y, place.long(), w), {}, "place"), ((y, place, w.half()), {}, "weights"), ((y, place, w[:, :1]), {}, "weights"),
                                ((y[0], place, w), {}, "y"), ((y, place, w), {"residual": res[:3]}, "residual"), ((y, place, w), {"residual": res.float()}, "residual"),
                                ((y, place.cpu(), w), {}, "place"), ((y, place, w), {"out": res[:, :90]}, "out"),
                                ((y, place.expand(4, 2).repeat(1, 17), w.repeat(1, 17)), {}, "32"), ((y.clone().requires_grad_(), place, w), {}, "gradient")]:
        with pytest.raises(ValueError, match=match):
            ops.combine_experts(*args, **kwargs)
    assert ops.combine_experts(y, place[:0], w[:0]).shape == (0, 96)


def test_combine_into_memory_of_an_input(cuda):
    g = _gen(4)
    whole = torch.randn(12, 96, generator=g, device=cuda)
    y, res = whole[:8], whole[8:].clone()
    place = torch.randint(0, 8, (4, 2), generator=g, dtype=torch.int32, device=cuda)
    w = torch.rand(4, 2, generator=g, device=cuda)
    for bad in (whole[:4], whole[4:8], whole[7:11]):
        with pytest.raises(ValueError, match="invalid argument"):
            ops.combine_experts(y, place, w, residual=res, out=bad)
    pair = torch.cat([res, res])
    with pytest.raises(ValueError, match="invalid argument"):
        ops.combine_experts(y, place, w, residual=pair[1:5], out=pair[:4])
    ref = ops.combine_experts(y, place, w, residual=res)
    assert torch.equal(ops.combine_experts(y, place, w, residual=res, out=whole[8:]), ref)  # right behind y


def test_combine_past_32_bit_offsets(cuda):
    y = torch.zeros(70000, 32768, dtype=torch.float16, device=cuda)
    y[-2:] = torch.randn(2, 32768, generator=_gen(5), device=cuda).half()
    place = torch.tensor([[69999, 69998], [0, 69999]], dtype=torch.int32, device=cuda)
    got = ops.combine_experts(y, place, torch.tensor([[1.0, 2.0], [1.0, 3.0]], device=cuda))
    assert torch.equal(got, torch.stack([y[-1].float() + 2 * y[-2].float(), 3 * y[-1].float()]).half())


# ---------------------------------------------------------------- the layer
def _layer(e, k, f, seed, dtype, dev):
    g = _gen(seed)
    up = quantize_convrot_expert_weights((torch.randn(e, f, k, generator=g, device=dev) * 0.02).to(dtype))
    down = quantize_convrot_expert_weights((torch.randn(e, k, f, generator=g, device=dev) * 0.02).to(dtype))
    b1, b2 = torch.randn(e, f, generator=g, device=dev) * 0.1, torch.randn(e, k, generator=g, device=dev) * 0.1
    return (*up, b1), (*down, b2)


def _layer_ref(x, logits, up, down, top_k, act, residual):
    """Token slots expert by expert on the framework's single-weight linear, joined in 64 bits."""
    value, ids = torch.sort(logits.double(), dim=1, descending=True, stable=True)
    value, ids = value[:, :top_k], ids[:, :top_k]
    w = torch.where(torch.isneginf(value), 0.0, torch.softmax(value, 1).nan_to_num())
    out = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(out)
    for e in range(up[0].shape[0]):
        t, j = ((ids == e) & ~torch.isneginf(value)).nonzero(as_tuple=True)
        if not len(t):
            continue
        q, s = ops.rotate_quant(x[t].contiguous(), 256)
        h = ops.int8_gemm_dequant(q, s, up[0][e], up[1][e], up[2][e], x.dtype)
        q, s = ops.quantize_act(h, 256, act)
        y = ops.int8_gemm_dequant(q, s, down[0][e], down[1][e], down[2][e], x.dtype)
        term = w[t, j][:, None] * y.double()
        out.index_add_(0, t, term)
        mag.index_add_(0, t, term.abs())
    return (out, mag) if residual is None else (out + residual.double(), mag + residual.double().abs())


@pytest.mark.parametrize("t,e,top_k", [(1, 8, 2), (37, 16, 4), (900, 4, 2)])
def test_layer(cuda, t, e, top_k):
    """Router, quantiser, grouped products and combine as a layer runs them, against expert-by-expert linears.
    All but the weights and the sum is bit-equal; the weights are within (|d| + E + 20) 2^-24 < 2^-17 and the sum
    within (top_k + 1) 2^-24 of the terms' magnitudes."""
    k, f, dtype = 512, 768, torch.bfloat16
    up, down = _layer(e, k, f, t, dtype, cuda)
    g = _gen(t)
    x = torch.randn(t, k, generator=g, device=cuda).to(dtype)
    logits = torch.randn(t, e, generator=g, device=cuda)
    if t > 1:
        logits[1] = -math.inf
    for act, residual in (("gelu_tanh", x), (None, None)):
        y = int8_expert_ffn(x, logits, up, down, top_k, act=act, residual=residual)
        ref, mag = _layer_ref(x, logits, up, down, top_k, act, residual)
        f32 = torch.finfo(dtype)
        tol = (2.0 ** -17 + (top_k + 1) * 2.0 ** -24) * mag + f32.eps / 2 * ref.abs() * (1 + 2.0 ** -7) + f32.tiny
        assert ((y.double() - ref).abs() <= tol).all()


def test_layer_in_a_graph_and_on_another_stream(cuda):
    t, e, top_k, k, f = 65, 8, 2, 256, 512
    up, down = _layer(e, k, f, 3, torch.float16, cuda)
    x, logits = torch.randn(t, k, device=cuda).half(), torch.randn(t, e, device=cuda)
    eager = int8_expert_ffn(x, logits, up, down, top_k)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = int8_expert_ffn(x, logits, up, down, top_k)
    s.synchronize()
    assert torch.equal(eager, other)
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = int8_expert_ffn(x, logits, up, down, top_k)
    with torch.cuda.graph(second):
        z = int8_expert_ffn(x, logits, up, down, 1)
    for i in range(3):
        x.copy_(torch.randn(t, k, device=cuda))
        logits.copy_(torch.randn(t, e, device=cuda) * (1 + i))
        graph.replay()
        second.replay()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, int8_expert_ffn(x, logits, up, down, top_k))
        assert torch.equal(z, int8_expert_ffn(x, logits, up, down, 1))
    del graph, second


def test_layer_empty_padded_and_refusals(cuda):
    e, k, f = 4, 256, 512
    up, down = _layer(e, k, f, 5, torch.float16, cuda)
    x, logits = torch.randn(2, 3, k, device=cuda).half(), torch.randn(2, 3, e, device=cuda)
    assert int8_expert_ffn(x[:0], logits[:0], up, down, 2).shape == (0, 3, k)
    closed = torch.full_like(logits, -math.inf)
    assert (int8_expert_ffn(x, closed, up, down, 2) == 0).all()
    assert torch.equal(int8_expert_ffn(x, closed, up, down, 2, residual=x), x)
    # a padded token leaves the others as they are
    y = int8_expert_ffn(x, logits, up, down, 2)
    logits[1, 1] = -math.inf
    z = int8_expert_ffn(x, logits, up, down, 2)
    assert (z[1, 1] == 0).all()
    keep = torch.ones(2, 3, dtype=torch.bool, device=cuda)
    keep[1, 1] = False
    assert torch.equal(y[keep], z[keep])
    for bad in ((x.clone().requires_grad_(), logits, None), (x, logits.clone().requires_grad_(), None), (x, logits, x.clone().requires_grad_())):
        with pytest.raises(ValueError, match="gradient"):
            int8_expert_ffn(bad[0], bad[1], up, down, 2, residual=bad[2])


def test_layers_on_two_streams_at_once(cuda):
    """Layers in flight together on two streams share nothing."""
    up, down = _layer(8, 512, 768, 6, torch.bfloat16, cuda)
    xs = [torch.randn(t, 512, generator=_gen(t), device=cuda).bfloat16() for t in (300, 7)]
    ls = [torch.randn(t, 8, generator=_gen(t + 1), device=cuda) for t in (300, 7)]
    want = [int8_expert_ffn(x, l, up, down, 2, residual=x) for x, l in zip(xs, ls)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(int8_expert_ffn(xs[i], ls[i], up, down, 2, residual=xs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


def test_first_calls_from_many_threads_at_once(cuda):
    """A fresh process whose first calls come from eight threads together, each on a stream of its own."""
    import subprocess
    import sys

    code = """
import threading, torch
from tilegen_b200 import ops
from tilegen_b200.quant import pack_int4
g = torch.Generator(device="cuda").manual_seed(1)
xq = torch.randint(-128, 128, (12, 512), generator=g, dtype=torch.int8, device="cuda")
codes = torch.randint(-8, 8, (96, 512), generator=g, dtype=torch.int8, device="cuda")
xs, ws = torch.rand(12, generator=g, device="cuda"), torch.rand(96, 4, generator=g, device="cuda")
wq, w4 = torch.randint(-128, 128, (2, 64, 512), generator=g, dtype=torch.int8, device="cuda"), pack_int4(codes)
logits, one = torch.randn(12, 2, generator=g, device="cuda"), torch.ones(1, device="cuda")
torch.cuda.synchronize()
start, out = threading.Barrier(8), [None] * 8
def work(i):
    with torch.cuda.stream(torch.cuda.Stream()):
        start.wait()
        a = [ops.int4_gemv_dequant(xq[:m], xs[:m], w4, ws, None, torch.float32) for m in (1, 12)]
        r = ops.route_experts(logits, 1)
        y = ops.int8_grouped_gemm_dequant(xq, xs, wq, one, None, r.offsets, torch.float32, rows=r.rows)
        out[i] = (*a, *r, y, ops.combine_experts(y, r.place, r.weights))
        torch.cuda.current_stream().synchronize()
threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
[t.start() for t in threads]
[t.join() for t in threads]
for i in range(8):
    assert all(torch.equal(p, q) for p, q in zip(out[i], out[0])), i
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, f"{done.returncode}: {done.stderr[-800:]}"


def test_grouped_with_few_sms(cuda):
    """The SM budget's smallest grids still cover every tile."""
    case = _group_case([300, 0, 5, 40], 520, 512, 60, seed=3)
    for sms in (1, 2, 3, 100):
        with ops.sm_budget(sms):
            _check_group(case, torch.float16)


def test_custom_ops(cuda):
    x = torch.randn(9, 8, generator=_gen(1), device=cuda)
    a, b = torch.ops.tilegen.route_experts(x, 2, True), ops.route_experts(x, 2)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    y = torch.randn(18, 16, device=cuda)
    assert torch.equal(torch.ops.tilegen.combine_experts(y, b.place, b.weights, None), ops.combine_experts(y, b.place, b.weights))
    xq, xs, wq, ws, _, offsets, rows = _group_case([3, 4], 64, 128, 20)
    assert torch.equal(torch.ops.tilegen.int8_grouped_gemm_dequant(xq, xs, wq, ws, None, offsets, torch.float16, rows),
                       ops.int8_grouped_gemm_dequant(xq, xs, wq, ws, None, offsets, torch.float16, rows=rows))
