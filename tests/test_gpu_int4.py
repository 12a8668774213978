"""Few-row products with a 4-bit weight (tg_int4_gemv_dequant) on the GPU, against the formula in 64 bits.

The sum inside a scale group is exact (int32); the groups are added in fp32, at most K/32 + 48 additions and
multiplications deep in any order the kernel may take, and the result is rounded once to the output type.  So an
output is off by at most (K/32 + 48) 2^-24 of the sum of the terms' magnitudes, and half a step of its type.
"""
from __future__ import annotations

import pytest
import torch

from tilegen_b200 import _lib, ops
from tilegen_b200.quant import int4_linear, pack_int4, quantize_convrot_weight_int4, unpack_int4

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _healthy_device(cuda):
    yield
    assert _lib.device_status(0) == 0


def _case(m, n, k, group, scale_dtype=torch.float16, bias_dtype=None, seed=0, dev="cuda"):
    g = torch.Generator(device=dev).manual_seed(seed)
    xq = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int8, device=dev)
    codes = torch.randint(-8, 8, (n, k), generator=g, dtype=torch.int8, device=dev)
    xs = torch.rand(m, generator=g, device=dev) * 0.02 + 1e-3
    ws = ((torch.rand(n, k // group, generator=g, device=dev) + 0.1) * 0.01).to(scale_dtype)
    bias = None if bias_dtype is None else torch.randn(n, generator=g, device=dev).to(bias_dtype)
    return xq, xs, codes, ws, bias


def _check(y, xq, xs, codes, ws, bias):
    """``y`` against the formula in 64 bits; ``codes`` unpacked."""
    (m, k), n, groups = xq.shape, codes.shape[0], ws.shape[1]
    x = xq.double().view(m, groups, -1)
    w = codes.double().view(n, groups, -1)
    ref = torch.zeros(m, n, dtype=torch.float64, device=xq.device)
    mag = torch.zeros_like(ref)
    for i in range(groups):
        t = (x[:, i] @ w[:, i].t()) * ws[:, i].double() * xs.double()[:, None]
        ref += t
        mag += t.abs()
    if bias is not None:
        ref += bias.double()
        mag += bias.double().abs()
    f = torch.finfo(y.dtype)
    tol = (k / 32 + 48) * 2.0 ** -24 * mag + f.eps / 2 * ref.abs() * (1 + 2.0 ** -10) + f.tiny * f.eps
    bad = (y.double() - ref).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outputs off, first {bad.nonzero()[0].tolist()}"


@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 7, 8, 9, 16, 17, 33, 64])
def test_rows_and_groups(cuda, m, group):
    xq, xs, codes, ws, bias = _case(m, 200, 768, group, seed=m)
    _check(ops.int4_gemv_dequant(xq, xs, pack_int4(codes), ws, bias, torch.float32), xq, xs, codes, ws, bias)


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scale_dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bias_dtype", [None, torch.float32, torch.float16, torch.bfloat16])
def test_types(cuda, out_dtype, scale_dtype, bias_dtype):
    for m in (1, 3, 12):
        xq, xs, codes, ws, bias = _case(m, 130, 512, 64, scale_dtype, bias_dtype, seed=3)
        _check(ops.int4_gemv_dequant(xq, xs, pack_int4(codes), ws, bias, out_dtype), xq, xs, codes, ws, bias)


@pytest.mark.parametrize("n,k,group", [(1, 128, 32), (1, 128, 128), (15, 128, 64), (16, 256, 256), (17, 1408, 128),
                                       (33, 14080, 128), (2000, 32768, 32), (70000, 256, 64), (1001, 5120, 32), (5120, 13824, 256), (13823, 5120, 128)])
def test_odd_and_block_shapes(cuda, n, k, group):
    for m in (1, 2, 4, 5, 40):
        xq, xs, codes, ws, bias = _case(m, n, k, group, torch.bfloat16, torch.float16, seed=n + k + m)
        _check(ops.int4_gemv_dequant(xq, xs, pack_int4(codes), ws, bias, torch.bfloat16), xq, xs, codes, ws, bias)


@pytest.mark.parametrize("m", [9, 12, 16])
def test_wide_weight_of_the_longest_rows_and_finest_scales(cuda, m):
    """Where 64 rows' scales do not fit an SM's shared memory (fp32 scales of 32 codes, K past 22000)."""
    for k in (22656, 22784, 32768):
        xq, xs, codes, ws, bias = _case(m, 7131, k, 32, torch.float32, torch.float32, seed=m)
        w4 = pack_int4(codes)
        y = ops.int4_gemv_dequant(xq, xs, w4, ws, bias, torch.float32)
        _check(y, xq, xs, codes, ws, bias)
        # the same rows in the other forms: a row's bits depend neither on M nor on the tile
        assert torch.equal(ops.int4_gemv_dequant(xq[:4], xs[:4], w4, ws, bias, torch.float32), y[:4])


@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("scale_dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_wide_weight_of_nine_to_sixteen_rows(cuda, scale_dtype, group):
    for m in (9, 14, 16):
        xq, xs, codes, ws, bias = _case(m, 7300, 1280, group, scale_dtype, torch.float16, seed=m)
        _check(ops.int4_gemv_dequant(xq, xs, pack_int4(codes), ws, bias, torch.float32), xq, xs, codes, ws, bias)


def test_extreme_codes_do_not_overflow(cuda):
    """-128 times -8 over the largest K the group allows: the int32 sums and 16-fold codes hold them."""
    k = 32768
    codes = torch.full((16, k), -8, dtype=torch.int8, device=cuda)
    ws = torch.full((16, k // 256), 1.0, device=cuda)
    for m in (1, 4, 5, 64):
        xq = torch.full((m, k), -128, dtype=torch.int8, device=cuda)
        y = ops.int4_gemv_dequant(xq, torch.ones(m, device=cuda), pack_int4(codes), ws, None, torch.float32)
        assert (y == 1024.0 * k).all()  # every partial sum is a multiple of 2^10, at most 2^25: exact


def test_a_row_does_not_depend_on_the_others(cuda):
    """Row i has the same bits in every batch of two rows or more, and one row alone the same wherever it comes from."""
    xq, xs, codes, ws, _ = _case(64, 333, 2048, 128, seed=5)
    w4 = pack_int4(codes)
    y = ops.int4_gemv_dequant(xq, xs, w4, ws, None, torch.float32)
    for i, j in ((0, 2), (1, 3), (3, 5), (3, 8), (10, 19), (40, 64), (31, 48), (0, 33)):
        assert torch.equal(ops.int4_gemv_dequant(xq[i:j], xs[i:j], w4, ws, None, torch.float32), y[i:j])
    one = [ops.int4_gemv_dequant(q[i:i + 1], xs[i:i + 1], w4, ws, None, torch.float32)
           for q, i in ((xq, 7), (xq.clone(), 7))]
    assert torch.equal(one[0], one[1])
    _check(one[0], xq[7:8], xs[7:8], codes, ws, None)


def test_infinite_and_nan_scales_stay_in_their_row(cuda):
    for m in (4, 8):
        xq, xs, codes, ws, _ = _case(m, 64, 512, 128, torch.float32, seed=6)
        ws[3, 1] = float("inf")
        ws[7, 0] = float("nan")
        xs[2] = float("nan")
        y = ops.int4_gemv_dequant(xq, xs, pack_int4(codes), ws, None, torch.float32)
        assert y[2].isnan().all() and y[:, 7].isnan().all() and not y[[0, 1, 3], 3].isfinite().any()
        keep = [i for i in range(64) if i not in (3, 7)]
        assert y[[0, 1, 3]][:, keep].isfinite().all()


def test_strided_and_unaligned_inputs(cuda):
    xq, xs, codes, ws, _ = _case(6, 40, 256, 64, seed=7)
    w4 = pack_int4(codes)
    y = ops.int4_gemv_dequant(xq, xs, w4, ws, None, torch.float32)
    wide = torch.zeros(6, 300, dtype=torch.int8, device=cuda)
    wide[:, 3:259] = xq
    raw = torch.zeros(w4.numel() + 1, dtype=torch.uint8, device=cuda)
    raw[1:] = w4.view(-1)
    a = ops.int4_gemv_dequant(wide[:, 3:259], xs.repeat_interleave(2)[::2], raw[1:].view_as(w4),
                              ws.t().contiguous().t(), None, torch.float32)
    assert torch.equal(a, y)
    out = torch.empty(6, 40, device=cuda)
    assert ops.int4_gemv_dequant(xq, xs, w4, ws, None, torch.float32, out=out) is out and torch.equal(out, y)


def test_refusals(cuda):
    xq, xs, codes, ws, _ = _case(4, 32, 256, 64)
    w4 = pack_int4(codes)
    f16 = torch.float16
    for args, match in [((xq.expand(17, 4, 256).reshape(68, 256), xs, w4, ws, None, f16), "at most"),
                        ((xq[:, :128], xs, w4, ws, None, f16), "match"), ((xq, xs[:3], w4, ws, None, f16), "xscale"),
                        ((xq, xs, w4, ws[:, :3], None, f16), "wscale"), ((xq, xs, w4, ws[:31], None, f16), "wscale"),
                        ((xq, xs.half(), w4, ws, None, f16), "xscale"), ((xq.float(), xs, w4, ws, None, f16), "xq"),
                        ((xq, xs, w4.to(torch.int8), ws, None, f16), "w4"), ((xq, xs, w4.cpu(), ws, None, f16), "w4"),
                        ((xq, xs, w4, ws, xs, f16), "bias"), ((xq, xs, w4, ws, None, torch.float64), "out_dtype"),
                        ((xq, xs, w4, ws.float().requires_grad_(), None, f16), "gradient")]:
        with pytest.raises(ValueError, match=match):
            ops.int4_gemv_dequant(*args)
    with pytest.raises(ValueError, match="out"):
        ops.int4_gemv_dequant(xq, xs, w4, ws, None, f16, out=torch.empty(4, 33, dtype=f16, device=cuda))
    assert ops.int4_gemv_dequant(xq[:0], xs[:0], w4, ws, None, f16).shape == (0, 32)


def test_weight_past_32_bit_offsets(cuda):
    """A weight of more than 2^32 codes and bytes past 2^31: its last rows are right."""
    n, k = 140000, 32768
    w4 = torch.zeros(n, k // 2, dtype=torch.uint8, device=cuda)
    xq, xs, codes, ws, _ = _case(3, 24, k, 256, seed=9)
    w4[-24:] = pack_int4(codes)
    scale = torch.ones(n, k // 256, dtype=torch.float16, device=cuda)
    scale[-24:] = ws
    for q, s in ((xq, xs), (xq.repeat(3, 1), xs.repeat(3))):  # each kernel
        y = ops.int4_gemv_dequant(q, s, w4, scale, None, torch.float32)
        _check(y[:, -24:], q, s, codes, ws, None)
        assert (y[:, :-24] == 0).all()


def test_other_stream_and_graph(cuda):
    """The quantiser and the product on another stream, then captured and replayed on new inputs."""
    k, n = 1024, 512
    w = torch.randn(n, k, generator=torch.Generator(device=cuda).manual_seed(1), device=cuda) * 0.02
    w4, ws = quantize_convrot_weight_int4(w)
    x = torch.randn(5, k, device=cuda).half()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a = int4_linear(x, w4, ws)
    s.synchronize()
    assert torch.equal(a, int4_linear(x, w4, ws))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = int4_linear(x, w4, ws)
    for i in range(3):
        x.copy_(torch.randn(5, k, device=cuda) * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, int4_linear(x, w4, ws))
    del graph


@pytest.mark.parametrize("m", [1, 64, 65, 150])
def test_linear_against_the_rotated_product(cuda, m):
    """int4_linear in one piece and in blocks: the formula on the quantiser's own codes."""
    k, n = 1024, 300
    g = torch.Generator(device=cuda).manual_seed(m)
    x = torch.randn(1, m, k, generator=g, device=cuda).to(torch.bfloat16)
    w4, ws = quantize_convrot_weight_int4(torch.randn(n, k, generator=g, device=cuda) * 0.02, scale_group=64)
    bias = torch.randn(n, generator=g, device=cuda)
    y = int4_linear(x, w4, ws, bias, input_act="gelu_tanh")
    assert y.shape == (1, m, n) and y.dtype == torch.bfloat16
    xq, xs = ops.quantize_act(x[0], 256, "gelu_tanh")
    _check(y[0], xq, xs, unpack_int4(w4), ws, bias)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_linear_rows_do_not_depend_on_their_number(cuda, dtype):
    k, n = 512, 77
    w4, ws = quantize_convrot_weight_int4(torch.randn(n, k, generator=torch.Generator(device=cuda).manual_seed(2), device=cuda))
    x = torch.randn(130, k, device=cuda).half()
    y = int4_linear(x, w4, ws, out_dtype=dtype)
    for m in (2, 64, 65, 66, 128, 129):
        assert torch.equal(int4_linear(x[:m], w4, ws, out_dtype=dtype), y[:m])


def test_out_at_any_address(cuda):
    """An out that starts at an odd element, for one row and for several."""
    for m in (1, 7, 40):
        xq, xs, codes, ws, _ = _case(m, 33, 256, 64, seed=7)
        w4 = pack_int4(codes)
        for dtype in (torch.float16, torch.float32):
            out = torch.full((m * 33 + 2,), 5.0, dtype=dtype, device=cuda)
            y = ops.int4_gemv_dequant(xq, xs, w4, ws, None, dtype, out=out[1:-1].view(m, 33))
            assert torch.equal(y, ops.int4_gemv_dequant(xq, xs, w4, ws, None, dtype))
            assert out[0] == 5 and out[-1] == 5


def test_linear_empty_and_refusals(cuda):
    w4, ws = quantize_convrot_weight_int4(torch.randn(64, 256, device=cuda))
    x = torch.randn(3, 256, device=cuda).half()
    assert int4_linear(x[:0], w4, ws).shape == (0, 64)
    with pytest.raises(ValueError, match="gradient"):
        int4_linear(x.clone().requires_grad_(), w4, ws)
    with torch.no_grad():
        assert torch.equal(int4_linear(x.clone().requires_grad_(), w4, ws), int4_linear(x, w4, ws))
    with pytest.raises(ValueError):
        int4_linear(x.float(), w4, ws)


@pytest.mark.parametrize("m", [1, 9, 17, 33, 40, 61, 64])
def test_short_rows_that_are_not_a_multiple_of_eight(cuda, m):
    """One block of K: the last slot's reads reach past the rows there are."""
    for n, group in ((5, 128), (200, 32)):
        xq, xs, codes, ws, bias = _case(m, n, 128, group, torch.float16, torch.float32, seed=m)
        _check(ops.int4_gemv_dequant(xq, xs, pack_int4(codes), ws, bias, torch.float32), xq, xs, codes, ws, bias)


def test_calls_on_two_streams_at_once(cuda):
    """Calls in flight together on two streams share nothing."""
    case = _case(12, 2000, 4096, 128, seed=8)
    other = _case(50, 1500, 4096, 64, seed=9)
    w4, o4 = pack_int4(case[2]), pack_int4(other[2])
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    ys, zs = [], []
    for _ in range(20):
        with torch.cuda.stream(a):
            ys.append(ops.int4_gemv_dequant(case[0], case[1], w4, case[3], None, torch.float32))
        with torch.cuda.stream(b):
            zs.append(ops.int4_gemv_dequant(other[0], other[1], o4, other[3], None, torch.float32))
    torch.cuda.synchronize()
    assert all(torch.equal(y, ys[0]) for y in ys) and all(torch.equal(z, zs[0]) for z in zs)
    _check(ys[0], *case[:4], None)
    _check(zs[0], *other[:4], None)


def test_custom_op(cuda):
    xq, xs, codes, ws, _ = _case(4, 32, 256, 64)
    w4 = pack_int4(codes)
    assert torch.equal(torch.ops.tilegen.int4_gemv_dequant(xq, xs, w4, ws, None, torch.float16),
                       ops.int4_gemv_dequant(xq, xs, w4, ws, None, torch.float16))
