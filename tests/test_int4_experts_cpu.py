"""4-bit weights and routed experts without a GPU: the packed layout, the weight quantiser, and every
argument check that returns before device work (Python and C ABI)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from tilegen_b200 import _lib, ops
from tilegen_b200.quant import (int4_linear, int8_expert_ffn, pack_int4, quantize_convrot_expert_weights,
                                quantize_convrot_weight, quantize_convrot_weight_int4, unpack_int4)

P = ctypes.c_void_p(256)
OK, ARG, UNS, MIS = _lib.TG_OK, _lib.TG_ERR_INVALID_ARG, _lib.TG_ERR_UNSUPPORTED, _lib.TG_ERR_MISALIGNED


# ---------------------------------------------------------------- layout and weight quantiser
@pytest.mark.parametrize("n,k", [(1, 128), (3, 256), (16, 640), (0, 128)])
def test_pack_roundtrip_and_layout(n, k):
    codes = torch.randint(-8, 8, (n, k), generator=torch.Generator().manual_seed(k), dtype=torch.int8)
    w4 = pack_int4(codes)
    assert w4.shape == (n, k // 2) and w4.dtype == torch.uint8
    assert torch.equal(unpack_int4(w4), codes)
    for row in range(n):
        for block in range(k // 128):
            for byte in (0, 3, 4, 17, 42, 63):
                t, j, b = byte // 16, byte % 16 // 4, byte % 4
                at = block * 128 + 32 * j + 8 * t + b
                v = int(w4[row, block * 64 + byte])
                assert v & 15 == int(codes[row, at]) & 15 and v >> 4 == int(codes[row, at + 4]) & 15


def test_pack_refusals():
    for bad in (torch.zeros(4, 120, dtype=torch.int8), torch.zeros(128, dtype=torch.int8), torch.zeros(4, 128)):
        with pytest.raises(ValueError):
            pack_int4(bad)
    for v in (-9, 8):
        with pytest.raises(ValueError, match="outside"):
            pack_int4(torch.full((1, 128), v, dtype=torch.int8))
    for bad in (torch.zeros(4, 60, dtype=torch.uint8), torch.zeros(4, 64, dtype=torch.int8)):
        with pytest.raises(ValueError):
            unpack_int4(bad)


@pytest.mark.parametrize("scale_group", [32, 64, 128, 256])
@pytest.mark.parametrize("scale_dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_weight_quantiser_error(scale_group, scale_dtype):
    """Each rotated value is within half a step of its code times the stored scale; at the clip (a scale
    rounded down) by at most 7 times the scale's own rounding more."""
    from tilegen_b200.kernels.hadamard import build_hadamard, rotate_by_group

    w = torch.randn(24, 512, generator=torch.Generator().manual_seed(1))
    w[3] = 0
    w4, ws = quantize_convrot_weight_int4(w, 256, scale_group, scale_dtype)
    assert ws.dtype == scale_dtype and ws.shape == (24, 512 // scale_group)
    rot = rotate_by_group(w.double(), build_hadamard(256, "cpu", torch.float64), 256).view(24, -1, scale_group)
    got = unpack_int4(w4).double().view(24, -1, scale_group) * ws.double()[..., None]
    step = ws.double()[..., None]
    slack = 7 * step * torch.finfo(scale_dtype).eps / 2 + 1e-5  # + the rotation in fp32
    assert ((got - rot).abs() <= step / 2 + slack).all()
    assert (got[3] == 0).all()


@pytest.mark.parametrize("scale_dtype,spread", [(dt, s) for dt in (torch.float32, torch.bfloat16) for s in (1e-4, 1e-6, 1e-9, 1e-30)]
                         + [(torch.float16, s) for s in (1e-4, 1e-5, 1e-6)])
def test_weight_quantiser_keeps_small_weights(scale_dtype, spread):
    """A value is off by at most half the step, and the step is the group's absmax/7 up to the division's rounding
    and its own (fp16 below 2^-14: up by less than 2^-24, with no code clipped)."""
    w = torch.randn(16, 512, generator=torch.Generator().manual_seed(5)) * spread
    w[2] = 0
    w4, ws = quantize_convrot_weight_int4(w, 1, 64, scale_dtype)
    got = unpack_int4(w4).double().view(16, 8, 64) * ws.double()[..., None]
    exact = w.double().view(16, 8, 64)
    half = torch.finfo(scale_dtype).eps / 2
    step = exact.abs().amax(-1, keepdim=True) / 7 * (1 + 2.0 ** -24) * (1 + half) + (2.0 ** -24 if scale_dtype == torch.float16 else 0)
    assert ((got - exact).abs() <= step / 2 + 7 * step * half + 2.0 ** -149).all()
    assert (got[2] == 0).all()


def test_weight_quantiser_fp16_scales_at_the_lower_end():
    w = torch.randn(4, 256, generator=torch.Generator().manual_seed(6))
    with pytest.raises(ValueError, match="too small"):
        quantize_convrot_weight_int4(w * 1e-9)
    quantize_convrot_weight_int4(w * 1e-9, scale_dtype=torch.bfloat16)
    w4, ws = quantize_convrot_weight_int4(torch.zeros(4, 256))
    assert (unpack_int4(w4) == 0).all() and (ws > 0).all()
    assert quantize_convrot_weight_int4(torch.zeros(0, 256))[1].shape == (0, 2)
    w[1] *= 1e-12  # one small row among others is not a reason to refuse: its values are below 2^-25
    w4, ws = quantize_convrot_weight_int4(w, 1)
    assert ((unpack_int4(w4).double().view(4, 2, 128)[1] * ws.double()[1, :, None]).abs() <= 2.0 ** -24).all()


def test_weight_quantiser_refusals():
    w = torch.zeros(4, 256)
    for kwargs in ({"scale_group": 16}, {"scale_group": 512}, {"scale_dtype": torch.float64}, {"group_size": 512}):
        with pytest.raises(ValueError):
            quantize_convrot_weight_int4(w, **kwargs)
    with pytest.raises(ValueError):
        quantize_convrot_weight_int4(torch.zeros(4, 2, 256))
    with pytest.raises(ValueError):
        quantize_convrot_weight_int4(torch.zeros(4, 64), scale_group=64)
    for v in (float("nan"), float("inf"), 1e9):
        w[1, 3] = v
        with pytest.raises(ValueError, match="cannot hold"):
            quantize_convrot_weight_int4(w)


def test_expert_weights_are_each_experts_weight():
    w = torch.randn(3, 16, 256, generator=torch.Generator().manual_seed(2))
    wq, ws = quantize_convrot_expert_weights(w)
    for e in range(3):
        q, s = quantize_convrot_weight(w[e])
        assert torch.equal(wq[e], q) and torch.equal(ws[e], s)
    with pytest.raises(ValueError):
        quantize_convrot_expert_weights(w[0])


@pytest.mark.parametrize("package", ["kernels", "quant", "runtime", "comfyui"])
def test_every_module_has_its_alias(package):
    """``tilegen.<package>.<module>`` is the ``tilegen_b200`` module, for every module file there is."""
    import importlib
    import pkgutil

    mine = importlib.import_module("tilegen_b200." + package)
    for info in pkgutil.iter_modules(mine.__path__):
        name = f"{package}.{info.name}"
        assert importlib.import_module("tilegen." + name) is importlib.import_module("tilegen_b200." + name)


# ---------------------------------------------------------------- Python refusals
def test_cpu_tensors_are_refused():
    i8, f = torch.zeros(2, 128, dtype=torch.int8), torch.zeros(2)
    with pytest.raises(ValueError, match="CUDA"):
        ops.int4_gemv_dequant(i8, f, torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 1), None, torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.route_experts(torch.zeros(2, 4), 2)
    with pytest.raises(ValueError, match="CUDA"):
        ops.int8_grouped_gemm_dequant(i8, f, torch.zeros(2, 8, 128, dtype=torch.int8), f, None,
                                      torch.zeros(3, dtype=torch.int32), torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.combine_experts(torch.zeros(2, 4), torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, 1))


def test_allocations_do_not_pass_modes_by(monkeypatch):
    """Outputs come from torch's own call where a dispatch mode or the deterministic fill has to see them, or the
    device is not the current one."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        count = 0

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            Seen.count += 1
            return func(*args, **(kwargs or {}))

    fast, meta = [], torch.device("meta", 0)

    def pretend(shape, stride, dtype):
        fast.append(shape)
        return torch.empty(shape, dtype=dtype)

    monkeypatch.setattr(ops, "_fast_empty", pretend)
    monkeypatch.setattr(ops, "_current_device", lambda: 0)

    def alloc(*shape):
        return ops._out("f", None, shape, torch.float16, meta)

    alloc(3, 4)
    assert fast == [(3, 4)]
    with Seen():
        assert alloc(3, 0).shape == (3, 0)
    assert Seen.count == 1 and fast == [(3, 4)]
    torch.use_deterministic_algorithms(True)
    try:
        assert alloc(5, 2).device.type == "meta" and len(fast) == 1
    finally:
        torch.use_deterministic_algorithms(False)
    monkeypatch.setattr(ops, "_current_device", lambda: 1)
    assert alloc(5, 2).device.type == "meta" and len(fast) == 1


def test_tangents_are_refused():
    """A forward-mode dual input is refused as one that wants a gradient is, not stripped of its tangent."""
    import torch.autograd.forward_ad as fwd

    x, up = torch.ones(2, 256), (torch.zeros(2, 512, 256, dtype=torch.int8), torch.zeros(2, 512), None)
    down = (torch.zeros(2, 256, 512, dtype=torch.int8), torch.zeros(2, 256), None)
    logits = torch.zeros(2, 2)
    ops.no_gradient("f", x, None)
    with fwd.dual_level():
        ops.no_gradient("f", x, None)
        dual = fwd.make_dual(x, torch.ones_like(x))
        for mode in (torch.enable_grad, torch.no_grad):
            with mode():
                with pytest.raises(ValueError, match="gradient"):
                    ops.no_gradient("f", None, x, dual)
                with pytest.raises(ValueError, match="gradient"):
                    int4_linear(dual, torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(4, 2))
                for args in ((dual, logits, None), (x, fwd.make_dual(logits, logits), None), (x, logits, dual)):
                    with pytest.raises(ValueError, match="gradient"):
                        int8_expert_ffn(args[0], args[1], up, down, 1, residual=args[2])
    with torch.no_grad():
        ops.no_gradient("f", x.clone().requires_grad_())
    with pytest.raises(ValueError, match="gradient"):
        ops.no_gradient("f", x.clone().requires_grad_())


@pytest.mark.parametrize("e,n", [(3, 8), (1, 16), (2, 4)])
def test_expert_scale_shapes(e, n):
    """A wscale of the right number of elements in the wrong order is refused."""
    cpu = torch.device("cpu")
    for shape in ((), (1,), (1, 1), (e,), (e, 1), (e, n), (e, n, 1), (e, 1, n), (e * n,)):
        ops._expert_scales("f", torch.zeros(shape), e, n, cpu)
    for bad in ((n,), (e + 1,), (e, n - 1), (2, e, n), (0,), (e, 0)) + (((n, e), (n, 1, e)) if e > 1 else ()):
        if (e == 1 and bad == (n,)):
            continue  # one expert's scales
        with pytest.raises(ValueError, match="wscale"):
            ops._expert_scales("f", torch.zeros(bad), e, n, cpu)
    for bad in (torch.zeros(e, n).double(), [1.0], torch.zeros(e, n, device="meta")):
        with pytest.raises(ValueError, match="wscale"):
            ops._expert_scales("f", bad, e, n, cpu)


def test_layer_functions_check_shapes():
    with pytest.raises(ValueError, match="differ"):
        int4_linear(torch.zeros(2, 256), torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 1))
    up = (torch.zeros(2, 512, 256, dtype=torch.int8), torch.zeros(2, 512), None)
    down = (torch.zeros(2, 256, 512, dtype=torch.int8), torch.zeros(2, 256), None)
    with pytest.raises(ValueError, match="logits"):
        int8_expert_ffn(torch.zeros(3, 256), torch.zeros(2, 2), up, down, 1)
    with pytest.raises(ValueError, match="channels"):
        int8_expert_ffn(torch.zeros(3, 256), torch.zeros(3, 2), up, up, 1)


def test_layer_checks_the_residuals_shape():
    up = (torch.zeros(2, 512, 256, dtype=torch.int8), torch.zeros(2, 512), None)
    down = (torch.zeros(2, 256, 512, dtype=torch.int8), torch.zeros(2, 256), None)
    x, logits = torch.zeros(3, 4, 256), torch.zeros(3, 4, 2)
    for shape in ((4, 3, 256), (3, 4, 255), (3, 256, 4), (1, 12, 256)):  # as many elements are not enough
        with pytest.raises(ValueError, match="residual"):
            int8_expert_ffn(x, logits, up, down, 1, residual=torch.zeros(shape))
    for shape in ((3, 4, 256), (12, 256)):  # the next check is the device's
        with pytest.raises(ValueError, match="CUDA"):
            int8_expert_ffn(x, logits, up, down, 1, residual=torch.zeros(shape))


@pytest.mark.parametrize("m", [1, 2, 63, 64, 65, 66, 127, 128, 129, 130, 193, 1025])
def test_linear_leaves_no_single_row_behind(monkeypatch, m):
    """The blocks cover every row once, and only a one-row input goes to the one-row kernel, which adds in an order
    of its own."""
    seen = []

    def product(xq, xs, w4, ws, bias, out_dtype, out=None):
        assert 1 <= xq.shape[0] <= ops.INT4_MAX_M and xs.shape[0] == xq.shape[0]
        seen.extend(xq[:, 0].tolist())
        assert xq.shape[0] > 1 or m == 1
        return torch.zeros(xq.shape[0], 5) if out is None else out.zero_()

    monkeypatch.setattr(ops, "quantize_act", lambda x, g, a: (x, x[:, 0]))
    monkeypatch.setattr(ops, "int4_gemv_dequant", product)
    x = torch.arange(m, dtype=torch.float32)[:, None].repeat(1, 128)
    assert int4_linear(x, torch.zeros(5, 64, dtype=torch.uint8), torch.zeros(5, 1)).shape == (m, 5)
    assert seen == list(range(m))


def test_custom_ops_trace_on_meta():
    m = torch.device("meta")
    y = torch.ops.tilegen.int4_gemv_dequant(torch.empty(3, 256, dtype=torch.int8, device=m), torch.empty(3, device=m),
                                            torch.empty(7, 128, dtype=torch.uint8, device=m),
                                            torch.empty(7, 2, device=m), None, torch.bfloat16)
    assert y.shape == (3, 7) and y.dtype == torch.bfloat16
    w, ids, offsets, rows, place = torch.ops.tilegen.route_experts(torch.empty(5, 8, device=m), 2, True)
    assert (w.shape, ids.shape, offsets.shape, rows.shape, place.shape) == ((5, 2), (5, 2), (9,), (10,), (5, 2))
    xq, wq = torch.empty(5, 64, dtype=torch.int8, device=m), torch.empty(8, 24, 64, dtype=torch.int8, device=m)
    y = torch.ops.tilegen.int8_grouped_gemm_dequant(xq, torch.empty(5, device=m), wq, torch.empty(8, 24, device=m), None,
                                                    offsets, torch.float16, rows)
    assert y.shape == (10, 24) and y.dtype == torch.float16
    assert torch.ops.tilegen.combine_experts(y, place, w, None).shape == (5, 24)


# ---------------------------------------------------------------- C ABI refusals
def _int4(xq=P, xs=P, w4=P, ws=P, wdt=1, group=128, bias=None, bdt=0, m=1, n=16, k=256, odt=1, out=P):
    return _lib.lib().tg_int4_gemv_dequant(xq, xs, w4, ws, wdt, group, bias, bdt, m, n, k, odt, out, None)


@pytest.mark.parametrize("kwargs,status", [
    ({"m": -1}, ARG), ({"n": 0}, ARG), ({"k": 0}, ARG), ({"odt": 3}, ARG), ({"wdt": 9}, ARG),
    ({"bias": P, "bdt": 5}, ARG), ({"group": 16}, UNS), ({"group": 512}, UNS), ({"m": 65}, UNS), ({"k": 192}, UNS),
    ({"k": 384, "group": 256}, UNS), ({"xq": None}, ARG), ({"xs": None}, ARG), ({"w4": None}, ARG), ({"ws": None}, ARG),
    ({"out": None}, ARG), ({"w4": ctypes.c_void_p(264)}, MIS), ({"xq": ctypes.c_void_p(8)}, MIS),
    ({"out": ctypes.c_void_p(257)}, MIS), ({"ws": ctypes.c_void_p(257)}, MIS), ({"m": 0, "xq": None, "out": None}, OK),
    ({"n": 1 << 31}, UNS), ({"n": (1 << 31) - 255}, UNS), ({"n": (1 << 31) - 256, "xq": None}, ARG),
])
def test_int4_entry_checks(kwargs, status):
    assert _int4(**kwargs) == status


def _route(logits=P, dt=0, t=4, e=8, k=2, w=P, ids=P, offsets=P, rows=P, place=P, ws=P, bytes=1 << 20):
    return _lib.lib().tg_route_experts(logits, dt, t, e, k, 1, w, ids, offsets, rows, place, ws, bytes, None)


@pytest.mark.parametrize("kwargs,status", [
    ({"t": -1}, ARG), ({"e": 0}, ARG), ({"k": 0}, ARG), ({"k": 9}, ARG), ({"dt": 4}, ARG), ({"e": 1025}, UNS),
    ({"e": 64, "k": 33}, UNS), ({"t": 1 << 30}, UNS), ({"offsets": None}, ARG), ({"logits": None}, ARG), ({"w": None}, ARG),
    ({"ids": None}, ARG), ({"rows": None}, ARG), ({"place": None}, ARG), ({"t": 257, "ws": None}, ARG), ({"t": 257, "bytes": 31}, ARG), ({"t": 257, "ws": ctypes.c_void_p(258)}, MIS),
    ({"logits": ctypes.c_void_p(258)}, MIS), ({"place": ctypes.c_void_p(258)}, MIS), ({"offsets": ctypes.c_void_p(258)}, MIS),
])
def test_route_entry_checks(kwargs, status):
    assert _lib.lib().tg_route_experts_workspace(257, 8) >= 9 * 8 * 4  # nine CTAs' counts
    assert _lib.lib().tg_route_experts_workspace(256, 8) == 0
    assert _lib.lib().tg_route_experts_workspace(0, 8) == 0
    assert _route(**kwargs) == status


def _grouped(xq=P, xs=P, m=4, wq=P, ws=P, wn=1, bias=None, bdt=0, rows=P, offsets=P, r=8, e=2, n=64, k=64, odt=1, out=P):
    return _lib.lib().tg_int8_grouped_gemm_dequant(xq, xs, m, wq, ws, wn, bias, bdt, rows, offsets, r, e, n, k, odt, out,
                                                   None, 0, None)


@pytest.mark.parametrize("kwargs,status", [
    ({"m": -1}, ARG), ({"r": -1}, ARG), ({"e": 0}, ARG), ({"n": 0}, ARG), ({"k": 0}, ARG), ({"odt": 7}, ARG),
    ({"bias": P, "bdt": 7}, ARG), ({"wn": 3}, ARG), ({"rows": None}, ARG), ({"k": 24}, UNS), ({"n": 12}, UNS),
    ({"n": 2, "odt": 0}, UNS), ({"e": 1025}, UNS), ({"e": 1000, "n": 1 << 22}, UNS), ({"xq": None}, ARG), ({"xs": None}, ARG), ({"wq": None}, ARG),
    ({"ws": None}, ARG), ({"offsets": None}, ARG), ({"out": None}, ARG), ({"xq": ctypes.c_void_p(8)}, MIS),
    ({"wq": ctypes.c_void_p(8)}, MIS), ({"out": ctypes.c_void_p(8)}, MIS), ({"rows": ctypes.c_void_p(2)}, MIS),
    ({"e": 1, "n": (1 << 31) - 248}, UNS), ({"e": 2, "n": (1 << 30) - 64}, UNS), ({"r": (1 << 31) - 255, "m": 1 << 30}, UNS),
    ({"m": (1 << 31) - 255}, UNS), ({"r": 0, "out": None}, OK), ({"m": 0, "r": 0, "xq": None}, OK),
])
def test_grouped_entry_checks(kwargs, status):
    need = _lib.lib().tg_int8_grouped_gemm_dequant_workspace
    assert need(8, 2, 64, 64) == 0 and need(4096, 8, 1024, 1024) == 0
    assert need(8192, 8, 13824, 5120) == 8192 * 5124
    assert _grouped(**kwargs) == status


def test_workspace_sizes_of_refused_calls():
    """Any 64-bit sizes: an answer, not the end of the process (in a child, which one division by zero would end)."""
    import subprocess
    import sys

    code = """
from tilegen_b200 import _lib
L, top = _lib.lib(), 2 ** 63 - 1
for t in (2 ** 30 + 1, 2 ** 40, 2 ** 62, top, -1, -top - 1):
    for e in (1, 1024, 1025, top, 0, -5):
        assert L.tg_route_experts_workspace(t, e) == 0, (t, e)
assert 0 < L.tg_route_experts_workspace(2 ** 30, 1024) <= 256 * 32 * 1024 * 4
sizes = (1, 2 ** 31, 2 ** 40, top, 0, -1)
for r in sizes:
    for e in sizes:
        for n in sizes:
            for k in sizes:
                assert L.tg_int8_grouped_gemm_dequant_workspace(r, e, n, k) == 0, (r, e, n, k)
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert done.returncode == 0, f"{done.returncode}: {done.stderr[-400:]}"


@pytest.mark.parametrize("kwargs", [{"e": 1 << 62, "n": 4}, {"e": 1 << 40, "n": 1 << 40}, {"n": (1 << 63) - 8}, {"r": 1 << 62},
                                    {"k": 1 << 62}, {"m": 1 << 62}])
def test_grouped_sizes_past_every_limit(kwargs):
    assert _grouped(**kwargs) == UNS


def _combine(y=P, dt=1, r=8, place=P, w=P, t=4, k=2, res=None, n=64, out=P):
    return _lib.lib().tg_combine_experts(y, dt, r, place, w, t, k, res, n, out, None)


@pytest.mark.parametrize("kwargs,status", [
    ({"t": -1}, ARG), ({"r": -1}, ARG), ({"n": 0}, ARG), ({"k": 0}, ARG), ({"dt": 3}, ARG), ({"k": 33}, UNS), ({"t": 1 << 31}, UNS),
    ({"y": None}, ARG), ({"place": None}, ARG), ({"w": None}, ARG), ({"out": None}, ARG), ({"y": ctypes.c_void_p(257)}, MIS),
    ({"out": ctypes.c_void_p(257)}, MIS), ({"res": ctypes.c_void_p(257)}, MIS), ({"place": ctypes.c_void_p(2)}, MIS),
    ({"t": 0, "y": None, "out": None}, OK),
])
def test_combine_entry_checks(kwargs, status):
    assert _combine(**kwargs) == status


@pytest.mark.parametrize("base,size", [("y", 8 * 64 * 2), ("place", 4 * 2 * 4), ("w", 4 * 2 * 4), ("res", 4 * 64 * 2)])
def test_combine_refuses_an_out_that_overlaps_an_input(base, size):
    """A fault of the call, not a race of its CTAs.  (What is in order gets as far as this machine's missing GPU, so
    only the refusals are looked at.)"""
    at = 1 << 20
    buffers = {"y": at << 1, "place": at << 2, "w": at << 3, "res": at << 4}
    pointers = {k: ctypes.c_void_p(v) for k, v in buffers.items()}
    first, out_bytes = buffers[base], 4 * 64 * 2
    for out in (first + 2, first + size - 2, first - out_bytes + 2) + (() if base == "res" else (first,)):
        assert _combine(**pointers, out=ctypes.c_void_p(out)) == ARG
    if torch.cuda.is_available():  # the others would be launched, on addresses that are not there
        return
    for out in (first + size, first - out_bytes) + ((first,) if base == "res" else ()):
        assert _combine(**pointers, out=ctypes.c_void_p(out)) != ARG
    assert _combine(**{**pointers, "y": None}, r=0, out=ctypes.c_void_p(1 << 26)) != ARG
