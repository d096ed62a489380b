"""The single compute backend: hand-written sm_100a kernels behind a C ABI.

Function names, keyword names, return types and error behaviour mirror the
reference's CUDA backend module (comfy_kitchen/backends/cuda/__init__.py:369-529,
1338-1498, 1681-1817) so the registry and the layout classes can call it
unchanged.  Differences, all additive: fp32 inputs to the block quantizers, fp32
bias in ``scaled_mm_*``, ``dequantize_mxfp8`` / ``scaled_mm_mxfp8`` on the device,
no zero-fill pass over the scale buffers (the kernels write the padding), and the
fused ``adaln_quantize_*`` / ``rmsnorm`` entry points, and the serving operators around a quantized linear
(``add_rmsnorm_quantize_*``, ``apply_rope_axes``, ``lora_add``).

Every output is allocated here with torch (caching allocator, CUDA-graph safe);
the native side only launches on the current stream.  Nothing synchronises.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from comfy_kitchen import _native
from comfy_kitchen._ops import refuse_derivatives as _no_grad
from comfy_kitchen.backends._modulation import adaln_prep_modulation
from comfy_kitchen.float_utils import roundup

DTYPE_CODE_TO_DTYPE = {
    0: torch.float32,
    1: torch.float16,
    2: torch.bfloat16,
    5: torch.float8_e4m3fn,
    6: torch.float8_e5m2,
}
DTYPE_TO_CODE = {v: k for k, v in DTYPE_CODE_TO_DTYPE.items()}

_native.load()  # fail at import when the library is absent: there is no other path


def _ptr(t: torch.Tensor | None):
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


def _stream(device) -> ctypes.c_void_p:
    # the raw handle: torch.cuda.current_stream builds a Stream object on the way to the same number (2.4 against 0.1 us)
    return ctypes.c_void_p(torch._C._cuda_getCurrentRawStream(torch.cuda.current_device() if device.index is None else device.index))


def _code(dtype: torch.dtype, what: str) -> int:
    try:
        return DTYPE_TO_CODE[dtype]
    except KeyError:
        raise TypeError(f"{what}: unsupported dtype {dtype}") from None


def _plain(t):
    if type(t) is torch.Tensor:   # (the instance check of Parameter is a Python call of its own, 0.7 us)
        return t
    return t.data if isinstance(t, torch.nn.Parameter) else t


# ------------------------------------------------------------------ FP8 per tensor


def quantize_per_tensor_fp8(
    x: torch.Tensor, scale: torch.Tensor, output_type: torch.dtype = torch.float8_e4m3fn
) -> torch.Tensor:
    if output_type not in (torch.float8_e4m3fn, torch.float8_e5m2):
        raise ValueError(
            f"Unsupported output_type: {output_type}. Expected torch.float8_e4m3fn or torch.float8_e5m2"
        )
    x = _plain(x)
    if not x.is_contiguous():
        x = x.contiguous()
    scale = _scalar_on(scale, x.device)
    out = torch.empty(x.shape, dtype=torch.uint8, device=x.device)
    _native.call(
        "launch_quantize_fp8_kernel", _ptr(x), _ptr(out), _ptr(scale), x.numel(),
        _code(x.dtype, "quantize_per_tensor_fp8"), DTYPE_TO_CODE[output_type], _stream(x.device),
    )
    return out.view(output_type)


def dequantize_per_tensor_fp8(
    x: torch.Tensor, scale: torch.Tensor, output_type: torch.dtype = torch.bfloat16
) -> torch.Tensor:
    assert scale.numel() == 1, "Scale must be a scalar tensor"
    x = _plain(x)
    if not x.is_contiguous():
        x = x.contiguous()
    scale = _scalar_on(scale, x.device)
    out = torch.empty(x.shape, dtype=output_type, device=x.device)
    _native.call(
        "launch_dequantize_fp8_kernel", _ptr(x), _ptr(out), _ptr(scale), x.numel(),
        _code(x.dtype, "dequantize_per_tensor_fp8"), _code(output_type, "dequantize_per_tensor_fp8"),
        _stream(x.device),
    )
    return out


def stochastic_rounding_fp8(
    x: torch.Tensor, rng: torch.Tensor, output_type: torch.dtype = torch.float8_e4m3fn
) -> torch.Tensor:
    """x.half() rounded to FP8 up or down according to one random byte per element (same bytes as the
    reference's eager function)."""
    if output_type not in (torch.float8_e4m3fn, torch.float8_e5m2):
        raise ValueError(f"Unsupported output_type: {output_type}. Expected torch.float8_e4m3fn or torch.float8_e5m2")
    x = _plain(x)
    assert rng.dtype == torch.uint8 and rng.shape == x.shape, "rng must be uint8 with x's shape"
    xc = x if x.is_contiguous() else x.contiguous()
    rc = rng if rng.is_contiguous() else rng.contiguous()
    out = torch.empty(x.shape, device=x.device, dtype=torch.uint8)
    _native.call("launch_stochastic_rounding_fp8_kernel", _ptr(xc), _ptr(rc), _ptr(out), xc.numel(),
                 _code(x.dtype, "stochastic_rounding_fp8"), DTYPE_TO_CODE[output_type], _stream(x.device))
    return out.view(output_type)


def _scalar_on(s, device) -> torch.Tensor:
    """fp32 one-element device tensor without a host round trip when it already is one."""
    s = _plain(s)
    if not isinstance(s, torch.Tensor):
        s = torch.tensor(float(s), dtype=torch.float32, device=device)
    if s.dtype != torch.float32 or s.device != device:
        s = s.to(device=device, dtype=torch.float32)
    return s.reshape(1) if s.dim() == 0 else s.contiguous()


def _bias_for(bias: torch.Tensor, n: int) -> torch.Tensor:
    """Bias vector for an output of n columns; a weight padded to the block multiple gets zero bias
    on its padding columns (they are cropped by the layout handlers afterwards)."""
    bias = bias.contiguous()
    if bias.numel() == n:
        return bias
    if bias.dim() != 1 or bias.numel() > n:
        raise RuntimeError(f"bias has {bias.numel()} elements, output has {n} columns")
    return torch.nn.functional.pad(bias, (0, n - bias.numel()))


# ------------------------------------------------------------------ NVFP4


def quantize_nvfp4(
    x: torch.Tensor,
    per_tensor_scale: torch.Tensor,
    epsilon: float = 0.0,
    pad_16x: bool = False,
    hi_first: bool = True,
) -> tuple[torch.Tensor, torch.Tensor]:
    x = _plain(x)
    assert x.dim() == 2, "Input must be 2D"
    assert x.is_contiguous(), "Input tensor must be contiguous"
    orig_rows, orig_cols = x.shape
    if pad_16x:
        num_rows, num_cols = roundup(orig_rows, 16), roundup(orig_cols, 16)
    else:
        num_rows, num_cols = orig_rows, orig_cols
        assert num_cols % 16 == 0, f"num_cols must be divisible by 16, got {num_cols}"
    qx = torch.empty((num_rows, num_cols // 2), device=x.device, dtype=torch.uint8)
    # the kernel writes every byte of the tiled scale buffer, padding included
    sx = torch.empty((roundup(num_rows, 128), roundup(num_cols // 16, 4)), device=x.device, dtype=torch.uint8)
    g = _scalar_on(per_tensor_scale, x.device)
    _native.call(
        "launch_quantize_nvfp4_kernel", _ptr(x), _ptr(g), _ptr(qx), _ptr(sx), num_rows, num_cols, orig_rows,
        orig_cols, float(epsilon), _code(x.dtype, "quantize_nvfp4"), bool(hi_first), _stream(x.device),
    )
    return qx, sx.view(torch.float8_e4m3fn)


def _segment(t: torch.Tensor, what: str):
    """(tensor, cols, group, group_stride, row_stride, rows) of one gather-quantizer segment."""
    if t.dim() == 2:      # [rows, cols], unit column stride, any row pitch
        assert t.stride(1) == 1, f"{what}: 2-D segments need unit column stride"
        return t, t.shape[1], t.shape[1], 0, t.stride(0), t.shape[0]
    if t.dim() == 3:      # [groups, rows, d] read as [rows, groups * d]  (attention's [heads, tokens, head_dim])
        assert t.stride(2) == 1, f"{what}: 3-D segments need unit stride in the last dim"
        return t, t.shape[0] * t.shape[2], t.shape[2], t.stride(0), t.stride(1), t.shape[1]
    raise ValueError(f"{what}: segments are 2-D [rows, cols] or 3-D [groups, rows, d]")


def quantize_nvfp4_gather(
    segments, per_tensor_scale: torch.Tensor, hi_first: bool = True
) -> tuple[torch.Tensor, torch.Tensor]:
    """quantize_nvfp4 of the column concatenation of one or two segments, without materialising it.

    segments: [(tensor, activation), ...] with activation None or "gelu_tanh"; a tensor is 2-D [rows, cols] with
    unit column stride (any row pitch: a column slice is fine) or 3-D [groups, rows, d], read as [rows, groups*d].
    Widths and strides must be multiples of 16 elements.  With no activation the result equals
    quantize_nvfp4(torch.cat(...)) byte for byte.
    """
    assert 1 <= len(segments) <= 2, "one or two segments"
    segs = []
    for t, act in segments:
        assert act in (None, "gelu_tanh"), f"unknown activation {act!r}"
        segs.append((*_segment(t, "quantize_nvfp4_gather"), 0 if act is None else 1))
    rows = segs[0][5]
    assert all(sg[5] == rows for sg in segs), "segments must have the same number of rows"
    dtype, device = segs[0][0].dtype, segs[0][0].device
    assert all(sg[0].dtype == dtype for sg in segs)
    cols = sum(sg[1] for sg in segs)
    qx = torch.empty((rows, cols // 2), device=device, dtype=torch.uint8)
    sx = torch.empty((roundup(rows, 128), roundup(cols // 16, 4)), device=device, dtype=torch.uint8)
    g = _scalar_on(per_tensor_scale, device)
    flat = []
    for i in range(2):
        if i < len(segs):
            t, c, grp, gs, rs, _, act = segs[i]
            flat += [_ptr(t), c, grp, gs, rs, act]
        else:
            flat += [None, 0, 16, 0, 16, 0]
    _native.call("launch_quantize_nvfp4_gather_kernel", *flat, _ptr(g), _ptr(qx), _ptr(sx), rows,
                 _code(dtype, "quantize_nvfp4_gather"), bool(hi_first), _stream(device))
    return qx, sx.view(torch.float8_e4m3fn)


def dequantize_nvfp4(
    qx: torch.Tensor,
    per_tensor_scale: torch.Tensor,
    block_scales: torch.Tensor,
    output_type: torch.dtype = torch.bfloat16,
    hi_first: bool = True,
) -> torch.Tensor:
    qx = _plain(qx)
    assert qx.is_contiguous(), "Input tensor must be contiguous"
    num_rows, packed = qx.shape
    num_cols = packed * 2
    out = torch.empty((num_rows, num_cols), device=qx.device, dtype=output_type)
    g = _scalar_on(per_tensor_scale, qx.device)
    sf = _plain(block_scales).contiguous().view(torch.uint8)
    _native.call(
        "launch_dequantize_nvfp4_kernel", _ptr(qx), _ptr(g), _ptr(sf), _ptr(out), num_rows, num_cols,
        _code(output_type, "dequantize_nvfp4"), bool(hi_first), _stream(qx.device),
    )
    return out


def scaled_mm_nvfp4(
    a: torch.Tensor,
    b: torch.Tensor,
    tensor_scale_a: torch.Tensor,
    tensor_scale_b: torch.Tensor,
    block_scale_a: torch.Tensor,
    block_scale_b: torch.Tensor,
    bias: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
    alpha: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    residual: torch.Tensor | None = None,
    gate: torch.Tensor | None = None,
    scatter=None,
) -> torch.Tensor:
    """``out`` (not in the reference's signature): a contiguous [M, N] tensor of ``out_dtype`` to write into,
    e.g. a row range of a larger buffer.  ``residual`` [M, N] and ``gate`` [N] (both of ``out_dtype``, bf16 or
    fp16; also additions): the kernel's epilogue returns ``residual + gate * y`` instead of ``y`` (bytes equal to
    the GEMM followed by ``torch.addcmul``); ``out`` may be ``residual`` itself.  ``scatter`` = (dests, bounds, world,
    row_offset) with ctypes arrays of peer-mapped destination pointers and row bounds (a tensor-parallel group's
    reduce-scatter fused into the epilogue, see ``launch_scaled_mm_nvfp4_scatter_kernel``): nothing is returned."""
    a, b = _plain(a), _plain(b)
    block_scale_a, block_scale_b = _plain(block_scale_a), _plain(block_scale_b)
    if alpha is None:
        alpha = _plain(tensor_scale_a) * _plain(tensor_scale_b)  # device op, no sync
    alpha = _scalar_on(alpha, a.device)
    assert alpha.numel() == 1, "alpha must be a scalar"
    m, k_a = a.shape
    n, k_b = b.shape
    assert k_a == k_b, "Matrix dimensions do not match"
    k = 2 * k_a
    assert n % 8 == 0, "B tensor must have 8 alignment in N dimension"
    assert block_scale_a.dtype == block_scale_b.dtype, "A and B scale dtype must match"
    if block_scale_a.dtype == torch.float8_e8m0fnu:
        raise ValueError("MXFP4 is not supported")
    if block_scale_a.dtype != torch.float8_e4m3fn:
        raise ValueError(f"Unsupported scale dtype: {block_scale_a.dtype}")
    sk = roundup(k // 16, 4)
    assert tuple(block_scale_a.shape) == (roundup(m, 128), sk), "Invalid A scale shape"
    assert tuple(block_scale_b.shape) == (roundup(n, 128), sk), "Invalid B scale shape"
    if out_dtype is None:
        out_dtype = torch.bfloat16
    bias_code = 0
    if bias is not None and bias.numel() > 0:
        bias = _bias_for(_plain(bias), n)
        assert bias.dtype in (torch.float16, torch.bfloat16, torch.float32), "bias must be fp16, bf16 or fp32"
        bias_code = DTYPE_TO_CODE[bias.dtype]
    else:
        bias = None
    if scatter is not None:
        dests, bounds, world, row_offset = scatter
        assert out is None and residual is None and out_dtype in (torch.bfloat16, torch.float16)
        _native.call(
            "launch_scaled_mm_nvfp4_scatter_kernel", _ptr(a.contiguous()), _ptr(block_scale_a.contiguous().view(torch.uint8)),
            _ptr(b.contiguous()), _ptr(block_scale_b.contiguous().view(torch.uint8)), dests, bounds, int(world), int(row_offset),
            _ptr(bias), bias_code, m, n, k, _ptr(alpha), _code(out_dtype, "scaled_mm_nvfp4"), _stream(a.device),
        )
        return None
    if out is None:
        out = torch.empty(m, n, dtype=out_dtype, device=a.device)
    else:
        assert out.shape == (m, n) and out.dtype == out_dtype and out.is_contiguous() and out.device == a.device
    if residual is not None:
        assert gate is not None, "residual needs a gate"
        gate = gate.reshape(-1)
        assert out_dtype in (torch.bfloat16, torch.float16), "the fused residual update needs a 16-bit output"
        assert residual.shape == (m, n) and residual.dtype == out_dtype and residual.is_contiguous()
        assert gate.numel() == n and gate.dtype == out_dtype and gate.is_contiguous()
        _native.call(
            "launch_scaled_mm_nvfp4_residual_kernel", _ptr(a.contiguous()), _ptr(block_scale_a.contiguous().view(torch.uint8)),
            _ptr(b.contiguous()), _ptr(block_scale_b.contiguous().view(torch.uint8)), _ptr(out), _ptr(bias), bias_code,
            _ptr(residual), _ptr(gate), m, n, k, _ptr(alpha), _code(out_dtype, "scaled_mm_nvfp4"), _stream(a.device),
        )
        return out
    _native.call(
        "launch_scaled_mm_nvfp4_kernel", _ptr(a.contiguous()), _ptr(block_scale_a.contiguous().view(torch.uint8)),
        _ptr(b.contiguous()), _ptr(block_scale_b.contiguous().view(torch.uint8)), _ptr(out), _ptr(bias), bias_code,
        m, n, k, _ptr(alpha), _code(out_dtype, "scaled_mm_nvfp4"), _stream(a.device),
    )
    return out


launch_residual_supported = True   # scaled_mm_nvfp4 accepts residual= / gate= (see its docstring)


# ------------------------------------------------------------------ MXFP8


def quantize_mxfp8(x: torch.Tensor, pad_32x: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    x = _plain(x)
    assert x.dim() == 2, "Input must be 2D"
    assert x.is_contiguous(), "Input tensor must be contiguous"
    orig_rows, orig_cols = x.shape
    if pad_32x:
        num_rows, num_cols = roundup(orig_rows, 32), roundup(orig_cols, 32)
    else:
        num_rows, num_cols = orig_rows, orig_cols
        assert num_cols % 32 == 0, f"num_cols must be divisible by 32, got {num_cols}"
    qx = torch.empty((num_rows, num_cols), device=x.device, dtype=torch.uint8)
    sx = torch.empty((roundup(num_rows, 128), roundup(num_cols // 32, 4)), device=x.device, dtype=torch.uint8)
    _native.call(
        "launch_quantize_mxfp8_kernel", _ptr(x), _ptr(qx), _ptr(sx), num_rows, num_cols, orig_rows, orig_cols,
        _code(x.dtype, "quantize_mxfp8"), _stream(x.device),
    )
    return qx.view(torch.float8_e4m3fn), sx.view(torch.float8_e8m0fnu)


def dequantize_mxfp8(
    qx: torch.Tensor, block_scales: torch.Tensor, output_type: torch.dtype = torch.bfloat16
) -> torch.Tensor:
    qx = _plain(qx)
    assert qx.is_contiguous(), "Input tensor must be contiguous"
    rows, cols = qx.shape
    out = torch.empty((rows, cols), device=qx.device, dtype=output_type)
    sf = _plain(block_scales).contiguous().view(torch.uint8)
    _native.call(
        "launch_dequantize_mxfp8_kernel", _ptr(qx), _ptr(sf), _ptr(out), rows, cols,
        _code(output_type, "dequantize_mxfp8"), _stream(qx.device),
    )
    return out


def scaled_mm_mxfp8(
    a: torch.Tensor,
    b: torch.Tensor,
    block_scale_a: torch.Tensor,
    block_scale_b: torch.Tensor,
    bias: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
) -> torch.Tensor:
    a, b = _plain(a), _plain(b)
    block_scale_a, block_scale_b = _plain(block_scale_a), _plain(block_scale_b)
    m, k = a.shape
    n, k_b = b.shape
    assert k == k_b, "Matrix dimensions do not match"
    assert n % 8 == 0, "B tensor must have 8 alignment in N dimension"
    sk = roundup(k // 32, 4)
    assert tuple(block_scale_a.shape) == (roundup(m, 128), sk), "Invalid A scale shape"
    assert tuple(block_scale_b.shape) == (roundup(n, 128), sk), "Invalid B scale shape"
    if out_dtype is None:
        out_dtype = torch.bfloat16
    bias_code = 0
    if bias is not None and bias.numel() > 0:
        bias = _bias_for(_plain(bias), n)
        bias_code = _code(bias.dtype, "scaled_mm_mxfp8")
    else:
        bias = None
    out = torch.empty(m, n, dtype=out_dtype, device=a.device)
    _native.call(
        "launch_scaled_mm_mxfp8_kernel", _ptr(a.contiguous()), _ptr(block_scale_a.contiguous().view(torch.uint8)),
        _ptr(b.contiguous()), _ptr(block_scale_b.contiguous().view(torch.uint8)), _ptr(out), _ptr(bias), bias_code,
        m, n, k, _code(out_dtype, "scaled_mm_mxfp8"), _stream(a.device),
    )
    return out


# ------------------------------------------------------------------ RoPE


def _rope(xq, xk, freqs_cis, split_half: bool):
    if xq.dim() != 4 or freqs_cis.dim() != 6:
        raise ValueError("apply_rope expects x [B, H, N, D] (or [B, N, H, D]) and freqs_cis [b, h, n, D/2, 2, 2]")
    xq = xq if xq.is_contiguous() else xq.contiguous()
    if xk is not None:
        xk = xk if xk.is_contiguous() else xk.contiguous()
    if not freqs_cis.is_contiguous():
        freqs_cis = freqs_cis.contiguous()
    oq = torch.empty_like(xq)
    ok = torch.empty_like(xk) if xk is not None else None
    sx, sf = xq.stride(), freqs_cis.stride()
    _native.call(
        "launch_apply_rope_kernel", _ptr(xq), _ptr(xk), _ptr(freqs_cis), _ptr(oq), _ptr(ok),
        *xq.shape, *freqs_cis.shape[:3], *sx, *sf,
        _code(xq.dtype, "apply_rope"), _code(freqs_cis.dtype, "apply_rope"), bool(split_half), _stream(xq.device),
    )
    return oq, ok


def apply_rope1(x: torch.Tensor, freqs_cis: torch.Tensor) -> torch.Tensor:
    return _rope(x, None, freqs_cis, False)[0]


def apply_rope(xq: torch.Tensor, xk: torch.Tensor, freqs_cis: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    if xq.shape != xk.shape:
        return apply_rope1(xq, freqs_cis), apply_rope1(xk, freqs_cis)
    return _rope(xq, xk, freqs_cis, False)


def apply_rope_split_half1(x: torch.Tensor, freqs_cis: torch.Tensor) -> torch.Tensor:
    return _rope(x, None, freqs_cis, True)[0]


def apply_rope_split_half(
    xq: torch.Tensor, xk: torch.Tensor, freqs_cis: torch.Tensor
) -> tuple[torch.Tensor, torch.Tensor]:
    if xq.shape != xk.shape:
        return apply_rope_split_half1(xq, freqs_cis), apply_rope_split_half1(xk, freqs_cis)
    return _rope(xq, xk, freqs_cis, True)


def qk_norm_rope(
    qkv: torch.Tensor,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor,
    freqs_cis: torch.Tensor,
    heads: int,
    q_out: torch.Tensor | None = None,
    k_out: torch.Tensor | None = None,
    v_out: torch.Tensor | None = None,
    token_offset: int = 0,
    eps: float = 1e-6,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Per-head RMSNorm of q and k, RoPE of both and the relayout of q, k, v for attention in one pass.

    qkv: [tokens, >= 3*heads*128], unit column stride (a column slice of a wider matrix is fine), columns
    [q heads | k heads | v heads].  freqs_cis: fp32 [1, 1, total_tokens, 64, 2, 2].  Outputs (allocated when
    not given): [1, heads, total_tokens, 128]; rows token_offset .. token_offset + tokens - 1 are written, so
    two calls can fill the text and the image part of one joint sequence.
    """
    assert qkv.dim() == 2 and qkv.stride(1) == 1 and qkv.shape[1] >= 3 * heads * 128, "qkv must be [tokens, 3*heads*128]"
    assert freqs_cis.dtype == torch.float32 and freqs_cis.is_contiguous() and freqs_cis.shape[-3:] == (64, 2, 2)
    assert freqs_cis.dim() == 6 and freqs_cis.shape[0] == freqs_cis.shape[1] == 1, "freqs_cis must be [1, 1, N, 64, 2, 2]"
    tokens, total = qkv.shape[0], freqs_cis.shape[2]
    outs = []
    for o in (q_out, k_out, v_out):
        if o is None:
            o = torch.empty((1, heads, total, 128), device=qkv.device, dtype=qkv.dtype)
        assert o.shape == (1, heads, total, 128) and o.is_contiguous() and o.dtype == qkv.dtype
        outs.append(o)
    qw = q_weight.to(qkv.dtype).contiguous()
    kw = k_weight.to(qkv.dtype).contiguous()
    _native.call(
        "launch_qk_norm_rope_kernel", _ptr(qkv), qkv.stride(0), _ptr(qw), _ptr(kw), _ptr(freqs_cis), _ptr(outs[0]),
        _ptr(outs[1]), _ptr(outs[2]), tokens, heads, int(token_offset), total, float(eps), _code(qkv.dtype, "qk_norm_rope"),
        _stream(qkv.device),
    )
    return outs[0], outs[1], outs[2]


# ------------------------------------------------------------------ AdaLN / RMSNorm


def _norm_inputs(x, scale, shift):
    d = x.shape[-1]
    n = x.numel() // d
    xf = x.reshape(n, d)
    if not xf.is_contiguous():
        xf = xf.contiguous()
    sc, sg = adaln_prep_modulation(scale.to(x.dtype), x, n, d)
    sh, hg = adaln_prep_modulation(shift.to(x.dtype), x, n, d)
    return xf, sc, sg, sh, hg, n, d


def adaln(x: torch.Tensor, scale: torch.Tensor, shift: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    xf, sc, sg, sh, hg, n, d = _norm_inputs(x, scale, shift)
    out = torch.empty_like(xf)
    _native.call(
        "launch_adaln_kernel", _ptr(xf), _ptr(sc), _ptr(sh), _ptr(out), n, d, sg, hg, float(eps),
        _code(x.dtype, "adaln"), _stream(x.device),
    )
    return out.reshape(x.shape)


def rmsnorm(x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-6) -> torch.Tensor:
    d = x.shape[-1]
    n = x.numel() // d
    xf = x.reshape(n, d)
    if not xf.is_contiguous():
        xf = xf.contiguous()
    w = None if weight is None else weight.to(x.dtype).contiguous()
    out = torch.empty_like(xf)
    _native.call(
        "launch_rmsnorm_kernel", _ptr(xf), _ptr(w), _ptr(out), n, d, float(eps), _code(x.dtype, "rmsnorm"),
        _stream(x.device),
    )
    return out.reshape(x.shape)


def adaln_quantize_nvfp4(
    x: torch.Tensor,
    scale: torch.Tensor,
    shift: torch.Tensor,
    per_tensor_scale: torch.Tensor,
    eps: float = 1e-6,
    hi_first: bool = True,
) -> tuple[torch.Tensor, torch.Tensor]:
    """quantize_nvfp4(adaln(x, scale, shift, eps), per_tensor_scale) in one pass over x."""
    xf, sc, sg, sh, hg, n, d = _norm_inputs(x, scale, shift)
    assert d % 16 == 0, f"last dim must be divisible by 16, got {d}"
    qx = torch.empty((n, d // 2), device=x.device, dtype=torch.uint8)
    sx = torch.empty((roundup(n, 128), roundup(d // 16, 4)), device=x.device, dtype=torch.uint8)
    g = _scalar_on(per_tensor_scale, x.device)
    _native.call(
        "launch_adaln_quantize_nvfp4_kernel", _ptr(xf), _ptr(sc), _ptr(sh), _ptr(g), _ptr(qx), _ptr(sx), n, d, sg, hg,
        float(eps), _code(x.dtype, "adaln_quantize_nvfp4"), bool(hi_first), 0, _stream(x.device),
    )
    return qx, sx.view(torch.float8_e4m3fn)


def adaln_quantize_nvfp4_rows(
    x: torch.Tensor,
    scale: torch.Tensor,
    shift: torch.Tensor,
    per_tensor_scale: torch.Tensor,
    qx: torch.Tensor,
    sx: torch.Tensor,
    row_begin: int,
    row_end: int,
    eps: float = 1e-6,
    hi_first: bool = True,
) -> None:
    """adaln_quantize_nvfp4 for rows [row_begin, row_end) of x only, written into the caller's whole-tensor buffers
    ``qx`` [N, D/2] uint8 and ``sx`` [roundup(N, 128), roundup(D/16, 4)] (the bytes of other rows are left alone).
    For sequence-parallel callers: each rank quantizes its rows of a shared activation."""
    xf, sc, sg, sh, hg, n, d = _norm_inputs(x, scale, shift)
    assert d % 16 == 0, f"last dim must be divisible by 16, got {d}"
    assert qx.shape == (n, d // 2) and qx.dtype == torch.uint8 and qx.is_contiguous()
    assert tuple(sx.shape) == (roundup(n, 128), roundup(d // 16, 4)) and sx.element_size() == 1 and sx.is_contiguous()
    g = _scalar_on(per_tensor_scale, x.device)
    _native.call(
        "launch_adaln_quantize_nvfp4_rows_kernel", _ptr(xf), _ptr(sc), _ptr(sh), _ptr(g), _ptr(qx), _ptr(sx), n, d, sg, hg,
        float(eps), _code(x.dtype, "adaln_quantize_nvfp4"), bool(hi_first), 0, int(row_begin), int(row_end), _stream(x.device),
    )


def adaln_quantize_mxfp8(
    x: torch.Tensor, scale: torch.Tensor, shift: torch.Tensor, eps: float = 1e-6
) -> tuple[torch.Tensor, torch.Tensor]:
    """quantize_mxfp8(adaln(x, scale, shift, eps)) in one pass over x."""
    xf, sc, sg, sh, hg, n, d = _norm_inputs(x, scale, shift)
    assert d % 32 == 0, f"last dim must be divisible by 32, got {d}"
    qx = torch.empty((n, d), device=x.device, dtype=torch.uint8)
    sx = torch.empty((roundup(n, 128), roundup(d // 32, 4)), device=x.device, dtype=torch.uint8)
    _native.call(
        "launch_adaln_quantize_mxfp8_kernel", _ptr(xf), _ptr(sc), _ptr(sh), _ptr(qx), _ptr(sx), n, d, sg, hg,
        float(eps), _code(x.dtype, "adaln_quantize_mxfp8"), 0, _stream(x.device),
    )
    return qx.view(torch.float8_e4m3fn), sx.view(torch.float8_e8m0fnu)


def rmsnorm_quantize_nvfp4(
    x: torch.Tensor, weight: torch.Tensor | None, per_tensor_scale: torch.Tensor, eps: float = 1e-6,
    hi_first: bool = True,
) -> tuple[torch.Tensor, torch.Tensor]:
    """quantize_nvfp4(rmsnorm(x, weight, eps), per_tensor_scale) in one pass over x."""
    d = x.shape[-1]
    n = x.numel() // d
    assert d % 16 == 0
    xf = x.reshape(n, d)
    if not xf.is_contiguous():
        xf = xf.contiguous()
    w = None if weight is None else weight.to(x.dtype).contiguous()
    qx = torch.empty((n, d // 2), device=x.device, dtype=torch.uint8)
    sx = torch.empty((roundup(n, 128), roundup(d // 16, 4)), device=x.device, dtype=torch.uint8)
    g = _scalar_on(per_tensor_scale, x.device)
    _native.call(
        "launch_adaln_quantize_nvfp4_kernel", _ptr(xf), _ptr(w), _ptr(None), _ptr(g), _ptr(qx), _ptr(sx), n, d, n, n,
        float(eps), _code(x.dtype, "rmsnorm_quantize_nvfp4"), bool(hi_first), 1, _stream(x.device),
    )
    return qx, sx.view(torch.float8_e4m3fn)


# ------------------------------------------------------------------ around a quantized linear, when serving


# A call of these runs for a few microseconds on the GPU when one token is served, so their host side is kept short: shapes
# are read once, addresses go to ctypes as plain integers, and the checks that format a message do so only when they fail.


def _same_device(what: str, device, *tensors) -> None:
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"{what}: tensors on {device} and {t.device}")


def _launch(device, name: str, *args) -> None:
    """_native.call with ``device`` current, on its current stream (appended as the last argument)."""
    index = device.index
    if index == torch._C._cuda_getDevice():   # (torch.cuda.current_device without its look at whether CUDA is up)
        _native.call(name, *args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            _native.call(name, *args, torch._C._cuda_getCurrentRawStream(index))


def _rows(t: torch.Tensor, width: int):
    """t as rows of `width` elements with unit column stride -> (the tensor that holds them, elements from row to row); a copy
    where it has no such view.  Of a contiguous tensor only the address matters."""
    if t.is_contiguous():
        return t, width
    if t.dim() != 2:
        try:
            t = t.view(-1, width)
        except RuntimeError:
            return t.reshape(-1, width).contiguous(), width
    rows, (apart, step) = t.shape[0], t.stride()
    if step != 1 or (rows > 1 and apart < width):
        return t.contiguous(), width
    return t, apart if rows > 1 else width


def _empty(like: torch.Tensor, shape, dtype) -> torch.Tensor:
    """A contiguous tensor on ``like``'s device; torch.empty_like is the cheapest way to one where it fits (1.4 against 2.6 us)."""
    if shape == like.shape and like.is_contiguous():
        return torch.empty_like(like, dtype=dtype)
    return like.new_empty(shape, dtype=dtype)


def _add_rmsnorm(what, x, residual, weight, eps, scale, output_type, return_norm, sum_out):
    _no_grad(what, x, residual, weight, sum_out)
    x, residual = _plain(x), _plain(residual)
    shape, dtype, device, stream_dtype = x.shape, x.dtype, x.device, residual.dtype
    if shape != residual.shape or not shape:
        raise ValueError(f"{what}: x {tuple(shape)} and residual {tuple(residual.shape)} must have the same shape")
    if stream_dtype != dtype and stream_dtype != torch.float32:
        raise ValueError(f"{what}: the residual has x's dtype or float32, got {stream_dtype}")
    d, mx = shape[-1], scale is None
    if d == 0 or (mx and d % 32):
        raise ValueError(f"{what}: last dim must be positive{' and divisible by 32' if mx else ''}, got {d}")
    n = x.numel() // d
    if weight is not None:
        weight = _plain(weight)
        if weight.shape != (d,):
            raise ValueError(f"{what}: weight must be [{d}], got {list(weight.shape)}")
        if weight.dtype != dtype or not weight.is_contiguous():
            weight = weight.to(dtype).contiguous()
    _same_device(what, device, residual, weight, sum_out)
    given = sum_out
    if given is None:
        sum_out = _empty(residual, shape, stream_dtype)
    elif sum_out.shape != shape or sum_out.dtype != stream_dtype or not sum_out.is_contiguous():
        raise ValueError(f"{what}: sum_out must be contiguous with the residual's shape and dtype")
    norm = _empty(x, shape, dtype) if return_norm else None
    q = _empty(x, (n, d) if mx and len(shape) != 2 else shape, output_type)
    sx = None
    if mx:
        cols = (d // 32 + 3) // 4 * 4
        sx = torch.empty_strided(((n + 127) // 128 * 128, cols), (cols, 1), dtype=torch.float8_e8m0fnu, device=device)
    if n:
        (xf, x_stride), (rf, r_stride) = _rows(x, d), _rows(residual, d)
        _launch(device, "launch_add_rmsnorm_quantize_kernel", xf.data_ptr(), rf.data_ptr(), 0 if weight is None else weight.data_ptr(),
                0 if mx else scale.data_ptr(), sum_out.data_ptr(), norm.data_ptr() if return_norm else 0, q.data_ptr(),
                sx.data_ptr() if mx else 0, n, d, x_stride, r_stride, eps, _code(dtype, what),
                _code(stream_dtype, what), DTYPE_TO_CODE[output_type])
        if given is not None:
            torch.autograd.graph.increment_version(given)   # (autograd is told, as by torch's in-place operators)
    return q, sx, sum_out, norm


def add_rmsnorm_quantize_mxfp8(
    x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-6,
    return_norm: bool = False, sum_out: torch.Tensor | None = None,
):
    """h = x + residual; quantize_mxfp8(rmsnorm(h, weight, eps)) in one pass -> (data, block scales, h), and with
    ``return_norm`` the normalised h behind them.

    ``residual`` (and h) has x's dtype or float32; ``weight`` is taken in x's dtype, whatever it has; the norm is taken of h as
    stored and rounded to x's dtype before it is quantized.  ``sum_out``: a contiguous tensor for h, which may be ``residual`` itself
    (or x, where it has h's dtype); any other overlap with an input is refused.
    """
    q, sx, h, norm = _add_rmsnorm("add_rmsnorm_quantize_mxfp8", x, residual, weight, eps, None, torch.float8_e4m3fn, return_norm, sum_out)
    return (q, sx, h, norm) if return_norm else (q, sx, h)


def add_rmsnorm_quantize_fp8(
    x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None, scale: torch.Tensor, eps: float = 1e-6,
    output_type: torch.dtype = torch.float8_e4m3fn, return_norm: bool = False, sum_out: torch.Tensor | None = None,
):
    """The same with quantize_per_tensor_fp8(normalised h, scale, output_type): -> (data in x's shape, h[, normalised h])."""
    if output_type not in (torch.float8_e4m3fn, torch.float8_e5m2):
        raise ValueError(f"Unsupported output_type: {output_type}. Expected torch.float8_e4m3fn or torch.float8_e5m2")
    if isinstance(scale, torch.Tensor):
        _no_grad("add_rmsnorm_quantize_fp8", scale)
    scale = _scalar_on(scale, x.device)
    if scale.numel() != 1:
        raise ValueError("add_rmsnorm_quantize_fp8: scale must be a scalar tensor")
    q, _, h, norm = _add_rmsnorm("add_rmsnorm_quantize_fp8", x, residual, weight, eps, scale, output_type, return_norm, sum_out)
    return (q, h, norm) if return_norm else (q, h)


_Strides, _Pairs = ctypes.c_int64 * 11, ctypes.c_int32 * 8


@functools.lru_cache(maxsize=256)
def _axes(axes_dim: tuple):
    """The C array of pairs per axis (read only), the elements that turn, the number of axes."""
    if not 1 <= len(axes_dim) <= 8 or any(int(a) != a or a <= 0 or a % 2 for a in axes_dim):
        raise ValueError
    return _Pairs(*[int(a) // 2 for a in axes_dim]), int(sum(axes_dim)), len(axes_dim)


_POSITION_CODES = {torch.float32: 0, torch.float64: 1, torch.int32: 2, torch.int64: 3}


def _rope_axes(what, xq, xk, positions, freqs, axes_dim, split_half, tokens_dim, inverse):
    _no_grad(what, xq, xk, positions, freqs)
    xq = _plain(xq)
    if tokens_dim != 1 and tokens_dim != 2:
        raise ValueError(f"{what}: tokens_dim is 2 for [B, H, N, D] or 1 for [B, N, H, D], got {tokens_dim}")
    heads_dim = 3 - tokens_dim
    q_shape, dtype, device = xq.shape, xq.dtype, xq.device
    if len(q_shape) != 4 or (xk is not None and xk.dim() != 4):
        raise ValueError(f"{what}: x must have four dimensions")
    b, n, d, heads_q, heads_k = q_shape[0], q_shape[tokens_dim], q_shape[3], q_shape[heads_dim], 0
    if xk is not None:
        xk = _plain(xk)
        k_shape = xk.shape
        heads_k = k_shape[heads_dim]
        if xk.dtype != dtype or k_shape[0] != b or k_shape[tokens_dim] != n or k_shape[3] != d:
            raise ValueError(f"{what}: q and k must agree in dtype and all dimensions but the heads")
    try:
        pairs, turned, count = _axes(tuple(axes_dim))
    except ValueError:
        turned = d + 1
    if turned > d or d % 2:
        raise ValueError(f"{what}: axes_dim {list(axes_dim)} must be 1 to 8 positive even sizes that add up to at most the (even) head dim {d}")
    if freqs.dtype != torch.float64 or freqs.shape != (turned // 2,):
        raise ValueError(f"{what}: freqs must be float64 [{turned // 2}], one per pair")
    p_shape = positions.shape
    if len(p_shape) == 2:
        p_shape = (1, *p_shape)
    if len(p_shape) != 3 or (p_shape[0] != 1 and p_shape[0] != b) or p_shape[1] != n or p_shape[2] != count:
        raise ValueError(f"{what}: positions must be [{n}, {count}], [1, {n}, {count}] or [{b}, {n}, {count}], got {list(positions.shape)}")
    code = _POSITION_CODES.get(positions.dtype)
    if code is None:
        raise ValueError(f"{what}: positions must be float32, float64, int32 or int64")
    _same_device(what, device, xk, positions, freqs)
    oq = _empty(xq, q_shape, dtype)
    ok = None if xk is None else _empty(xk, k_shape, dtype)
    if b == 0 or n == 0 or d == 0 or heads_q == 0 or (xk is not None and heads_k == 0):
        if oq.numel():
            oq, _ = _rope_axes(what, xq, None, positions, freqs, axes_dim, split_half, tokens_dim, inverse)
        elif ok is not None and ok.numel():
            ok, _ = _rope_axes(what, xk, None, positions, freqs, axes_dim, split_half, tokens_dim, inverse)
        return oq, ok
    if not freqs.is_contiguous():
        freqs = freqs.contiguous()
    sq, sp = xq.stride(), positions.stride()
    sk = sq if xk is None else xk.stride()
    strides = _Strides(sq[0], sq[tokens_dim], sq[heads_dim], sq[3], sk[0], sk[tokens_dim], sk[heads_dim], sk[3],
                       0 if p_shape[0] == 1 else sp[0], sp[-2], sp[-1])
    _launch(device, "launch_apply_rope_axes_kernel", xq.data_ptr(), 0 if xk is None else xk.data_ptr(), positions.data_ptr(), freqs.data_ptr(),
            oq.data_ptr(), 0 if xk is None else ok.data_ptr(), strides, b, n, heads_q, heads_k, d, pairs, count,
            _code(dtype, what), code, tokens_dim == 1, split_half, inverse)
    return oq, ok


def apply_rope_axes(
    xq: torch.Tensor, xk: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, axes_dim, split_half: bool = False,
    tokens_dim: int = 2, inverse: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Rotary embedding of q and k by positions of several axes, the angles computed in the kernel.

    xq, xk: [B, H, N, D] (``tokens_dim`` 2) or [B, N, H, D] (1), any strides; k may have fewer heads.  positions: [N, A],
    [1, N, A] or [B, N, A], integers or fractions.  axes_dim: how many elements of a head each of the A axes turns, in
    order; what is left of D passes through.  freqs: float64, one per pair, radians per unit of position
    (``rope_axes_freqs``).  ``inverse`` rotates back, which is also the gradient's rotation.  Outputs are contiguous.
    """
    return _rope_axes("apply_rope_axes", xq, xk, positions, freqs, axes_dim, split_half, tokens_dim, inverse)


def apply_rope_axes1(
    x: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, axes_dim, split_half: bool = False, tokens_dim: int = 2,
    inverse: bool = False,
) -> torch.Tensor:
    return _rope_axes("apply_rope_axes1", x, None, positions, freqs, axes_dim, split_half, tokens_dim, inverse)[0]


def lora_add(
    y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, adapter_ids: torch.Tensor,
    scales: torch.Tensor | None = None, out: torch.Tensor | None = None,
) -> torch.Tensor:
    """y + scales[i] * (x @ a[i].T) @ b[i].T, with i = adapter_ids of the row: the adapters of many requests beside a
    shared projection.

    y: [..., N], what the shared projection made of x: [..., K].  a: [L, R, K], b: [L, N, R] (adapters of a lower rank are
    padded with zeros).  adapter_ids: int32 or int64 in the shape of x's leading dimensions, or of the first of them
    (one per batch entry); an id outside [0, L) means no adapter, and the row of y is passed on.  scales: float32 [L].
    ``out``: where to write, in y's shape; may be y (or x) itself, any other overlap with an input is refused.
    K, N and R are multiples of 8, R at most 256.
    """
    what = "lora_add"
    _no_grad(what, y, x, a, b, scales, out)
    y, x, a, b = _plain(y), _plain(x), _plain(a), _plain(b)
    x_shape, y_shape, a_shape, b_shape, dtype, device = x.shape, y.shape, a.shape, b.shape, x.dtype, x.device
    if len(a_shape) != 3 or len(b_shape) != 3 or not x_shape:
        raise ValueError(f"{what}: a must be [L, R, K] and b [L, N, R]")
    (adapters, rank, k), n = a_shape, b_shape[1]
    if b_shape[0] != adapters or b_shape[2] != rank:
        raise ValueError(f"{what}: a {list(a_shape)} and b {list(b_shape)} do not match")
    if x_shape[-1] != k:
        raise ValueError(f"{what}: x has {x_shape[-1]} columns, a {k}")
    if y_shape[:-1] != x_shape[:-1] or y_shape[-1] != n:
        raise ValueError(f"{what}: y must be {[*x_shape[:-1], n]}, got {list(y_shape)}")
    if y.dtype != dtype or a.dtype != dtype or b.dtype != dtype:
        raise ValueError(f"{what}: y, x, a and b must have one dtype")
    if adapters == 0 or not 0 < rank <= 256 or rank % 8 or k == 0 or k % 8 or n == 0 or n % 8:
        raise ValueError(f"{what}: K, N and R must be multiples of 8 and R at most 256, got {k}, {n}, {rank} of {adapters} adapters")
    ids_dtype, ids_shape = adapter_ids.dtype, adapter_ids.shape
    if ids_dtype != torch.int32 and ids_dtype != torch.int64:
        raise ValueError(f"{what}: adapter_ids must be int32 or int64")
    if len(ids_shape) >= len(x_shape) or ids_shape != x_shape[:len(ids_shape)]:
        raise ValueError(f"{what}: adapter_ids {list(ids_shape)} must have the shape of x's leading dimensions {list(x_shape[:-1])} or of the first of them")
    if scales is not None and (scales.dtype != torch.float32 or scales.shape != (adapters,)):
        raise ValueError(f"{what}: scales must be float32 [{adapters}]")
    _same_device(what, device, y, a, b, adapter_ids, scales, out)
    given = out
    if given is None:
        out = _empty(y, y_shape, dtype)
    elif out.shape != y_shape or out.dtype != dtype:
        raise ValueError(f"{what}: out must have y's shape and dtype")
    rows = x.numel() // k
    if rows == 0:
        return out
    if device.index is not None and device.index != torch._C._cuda_getDevice():   # (the scratch's size goes by the device)
        with torch.cuda.device(device):
            return lora_add(y, x, a, b, adapter_ids, scales, given)
    # the kernels move 16 bytes at a time
    (xf, x_stride), (yf, y_stride), (of, o_stride) = _rows(x, k), _rows(y, n), _rows(out, n)
    px, py, po, pa, pb = xf.data_ptr(), yf.data_ptr(), of.data_ptr(), a.data_ptr(), b.data_ptr()
    if po != out.data_ptr() or po % 16 or o_stride % 8:
        raise ValueError(f"{what}: out must have unit column stride, rows of one stride and 16-byte alignment")
    if px % 16 or x_stride % 8:
        xf = xf.clone(memory_format=torch.contiguous_format)
        px, x_stride = xf.data_ptr(), k
    if py % 16 or y_stride % 8:
        yf = yf.clone(memory_format=torch.contiguous_format)
        py, y_stride = yf.data_ptr(), n
    if pa % 16 or not a.is_contiguous():
        a = a.clone(memory_format=torch.contiguous_format)
        pa = a.data_ptr()
    if pb % 16 or not b.is_contiguous():
        b = b.clone(memory_format=torch.contiguous_format)
        pb = b.data_ptr()
    ids = adapter_ids if adapter_ids.is_contiguous() else adapter_ids.contiguous()
    if scales is not None and not scales.is_contiguous():
        scales = scales.contiguous()
    # scratch of the tiled kernels; the allocator's, so that streams and captured graphs keep theirs apart
    need = _native.load().ck_lora_workspace_bytes(rows, k, n, rank)
    work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    _launch(device, "launch_lora_add_kernel", py, px, pa, pb, ids.data_ptr(), 0 if scales is None else scales.data_ptr(), po,
            0 if work is None else work.data_ptr(), rows, k, n, rank, adapters, y_stride, x_stride, o_stride, rows // ids.numel(),
            _code(dtype, what), ids_dtype == torch.int64)
    if given is not None:
        torch.autograd.graph.increment_version(given)
    return out


def build_constraints() -> dict:
    """What this backend accepts, per function (checked by the registry before dispatch)."""
    from comfy_kitchen.constraints import DivisibleBy, ExactDims, FunctionConstraints, ParamConstraint

    dev = frozenset({"cuda"})
    floats = frozenset({torch.float32, torch.float16, torch.bfloat16})
    fp8 = frozenset({torch.float8_e4m3fn, torch.float8_e5m2})
    sm100 = (10, 0)

    def fc(**params):
        return FunctionConstraints(params=params, default_devices=dev, min_compute_capability=sm100)

    two_d = (ExactDims(2),)
    rope = fc(x=ParamConstraint(dtypes=floats, shape_rules=(ExactDims(4),)),
              freqs_cis=ParamConstraint(dtypes=floats, shape_rules=(ExactDims(6),)))
    rope2 = fc(xq=ParamConstraint(dtypes=floats, shape_rules=(ExactDims(4),)),
               xk=ParamConstraint(dtypes=floats, shape_rules=(ExactDims(4),)),
               freqs_cis=ParamConstraint(dtypes=floats, shape_rules=(ExactDims(6),)))
    norm = dict(x=ParamConstraint(dtypes=floats), scale=ParamConstraint(dtypes=floats), shift=ParamConstraint(dtypes=floats))
    return {
        "quantize_per_tensor_fp8": fc(x=ParamConstraint(dtypes=floats), scale=ParamConstraint(dtypes=frozenset({torch.float32})),
                                      output_type=ParamConstraint(dtypes=fp8)),
        "dequantize_per_tensor_fp8": fc(x=ParamConstraint(dtypes=fp8), output_type=ParamConstraint(dtypes=floats)),
        "quantize_nvfp4": fc(x=ParamConstraint(dtypes=floats, shape_rules=two_d),
                             per_tensor_scale=ParamConstraint(dtypes=frozenset({torch.float32}))),
        "dequantize_nvfp4": fc(qx=ParamConstraint(dtypes=frozenset({torch.uint8}), shape_rules=two_d + (DivisibleBy(1, 8),)),
                               per_tensor_scale=ParamConstraint(dtypes=frozenset({torch.float32})),
                               block_scales=ParamConstraint(dtypes=frozenset({torch.float8_e4m3fn})),
                               output_type=ParamConstraint(dtypes=floats)),
        "scaled_mm_nvfp4": fc(a=ParamConstraint(dtypes=frozenset({torch.uint8}), shape_rules=two_d + (DivisibleBy(1, 16),)),
                              b=ParamConstraint(dtypes=frozenset({torch.uint8}), shape_rules=two_d + (DivisibleBy(1, 16), DivisibleBy(0, 8))),
                              block_scale_a=ParamConstraint(dtypes=frozenset({torch.float8_e4m3fn})),
                              block_scale_b=ParamConstraint(dtypes=frozenset({torch.float8_e4m3fn})),
                              bias=ParamConstraint(dtypes=floats), out_dtype=ParamConstraint(dtypes=floats)),
        "quantize_mxfp8": fc(x=ParamConstraint(dtypes=floats, shape_rules=two_d)),
        "dequantize_mxfp8": fc(qx=ParamConstraint(dtypes=frozenset({torch.float8_e4m3fn}), shape_rules=two_d + (DivisibleBy(1, 32),)),
                               block_scales=ParamConstraint(dtypes=frozenset({torch.float8_e8m0fnu})),
                               output_type=ParamConstraint(dtypes=floats)),
        "scaled_mm_mxfp8": fc(a=ParamConstraint(dtypes=frozenset({torch.float8_e4m3fn}), shape_rules=two_d + (DivisibleBy(1, 32),)),
                              b=ParamConstraint(dtypes=frozenset({torch.float8_e4m3fn}), shape_rules=two_d + (DivisibleBy(1, 32), DivisibleBy(0, 8))),
                              block_scale_a=ParamConstraint(dtypes=frozenset({torch.float8_e8m0fnu})),
                              block_scale_b=ParamConstraint(dtypes=frozenset({torch.float8_e8m0fnu})),
                              bias=ParamConstraint(dtypes=floats), out_dtype=ParamConstraint(dtypes=floats)),
        "apply_rope": rope2, "apply_rope1": rope, "apply_rope_split_half": rope2, "apply_rope_split_half1": rope,
        "adaln": fc(**norm),
        "rmsnorm": fc(x=ParamConstraint(dtypes=floats), weight=ParamConstraint(dtypes=floats)),
        "adaln_quantize_nvfp4": fc(**norm, per_tensor_scale=ParamConstraint(dtypes=frozenset({torch.float32}))),
        "adaln_quantize_mxfp8": fc(**norm),
        "stochastic_rounding_fp8": fc(x=ParamConstraint(dtypes=floats), rng=ParamConstraint(dtypes=frozenset({torch.uint8}))),
        "qk_norm_rope": fc(qkv=ParamConstraint(dtypes=frozenset({torch.bfloat16, torch.float16})),
                           freqs_cis=ParamConstraint(dtypes=frozenset({torch.float32}))),
        # (these check the rest of their arguments themselves, with messages that name the shapes)
        "add_rmsnorm_quantize_mxfp8": fc(x=ParamConstraint(dtypes=floats), weight=ParamConstraint(dtypes=floats)),
        "add_rmsnorm_quantize_fp8": fc(x=ParamConstraint(dtypes=floats), weight=ParamConstraint(dtypes=floats),
                                       scale=ParamConstraint(dtypes=frozenset({torch.float32}))),
        "apply_rope_axes": fc(xq=ParamConstraint(dtypes=floats)), "apply_rope_axes1": fc(x=ParamConstraint(dtypes=floats)),
        "lora_add": fc(x=ParamConstraint(dtypes=frozenset({torch.bfloat16, torch.float16}))),
        "quantize_nvfp4_gather": fc(per_tensor_scale=ParamConstraint(dtypes=frozenset({torch.float32}))),
    }


def set_option(name: str, value: int) -> None:
    """Process-wide library option (see ``ck_set_option`` in the C header)."""
    _native.call("ck_set_option", name.encode(), int(value))


def gemm_device_status() -> int:
    """Synchronise and return the GEMM kernels' device status word (0 = fine)."""
    return int(_native.load().ck_gemm_device_status())


def lora_device_status() -> int:
    """Synchronise and return (then clear) the adapter kernels' device-side status word; 0 = healthy."""
    return int(_native.load().ck_lora_device_status())


def norm_device_status() -> int:
    """Synchronise and return (then clear) the norm kernels' device-side status word; 0 = healthy."""
    return int(_native.load().ck_norm_device_status())
