"""8-bit experts: block quantisation to e4m3 and the grouped GEMM of such tensors.

A block of 128 values of a row (activations) or of 128 x 128 values (weights)
is held as float8_e4m3fn numbers and one power-of-two scale of type
float8_e8m0fnu, the smallest with which no value exceeds 448, the largest
e4m3 number. Dividing by it is exact, so quantising rounds a value once (at
most 2^-4 of it, or 2^-10 of the scale below the normal range), and the
tensor cores apply the scales themselves. Infinities and NaN become NaN.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence, Union

import torch

from . import _lib
from .ops import GroupedGemmPlan, _need_cuda, _need_dtype, _on, _p, _stream

__all__ = ["Fp8Tensor", "quantize_fp8", "quantize_fp8_weight", "dequantize_fp8", "permute_fp8",
           "grouped_gemm_fp8"]

BLOCK = 128


class Fp8Tensor(NamedTuple):
    """Rows: data [M,K] float8_e4m3fn, scale [M,ceil(K/128)] float8_e8m0fnu.
    Weights: data [G,N,K], scale [G,ceil(N/128),ceil(K/128)]."""
    data: torch.Tensor
    scale: torch.Tensor


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _empty(like: torch.Tensor, shape, scale_shape) -> Fp8Tensor:
    return Fp8Tensor(like.new_empty(shape, dtype=torch.float8_e4m3fn),
                     like.new_empty(scale_shape, dtype=torch.float8_e8m0fnu))


def _same_device(**tensors: Optional[torch.Tensor]) -> torch.device:
    dev = None
    for name, t in tensors.items():
        if t is None:
            continue
        _need_cuda(name, t)
        if dev is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, the other tensors on {dev}")
        dev = t.device
    return dev


def _need_k(name: str, k: int) -> None:
    if k < 16 or k % 16:
        raise ValueError(f"{name} must have a positive multiple of 16 columns, got {k}")


def _src_type(name: str, x: torch.Tensor) -> int:
    _need_dtype(name, x, torch.bfloat16, torch.float32)
    return 1 if x.dtype == torch.float32 else 0


def _need_fp8(name: str, q: Fp8Tensor, scale_shape) -> None:
    _need_dtype(f"{name}.data", q.data, torch.float8_e4m3fn)
    _need_dtype(f"{name}.scale", q.scale, torch.float8_e8m0fnu)
    if tuple(q.scale.shape) != tuple(scale_shape):
        raise ValueError(f"{name}.scale must be {tuple(scale_shape)}, got {tuple(q.scale.shape)}")


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t contiguous and 16-byte aligned (a view at an odd offset is copied)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def quantize_fp8(x: torch.Tensor) -> Fp8Tensor:
    """Rows x [M,K] (bf16 or fp32, K % 16 == 0) with one scale for 128 values."""
    dev = _same_device(x=x)
    if x.dim() != 2:
        raise ValueError(f"x must be [M,K], got {tuple(x.shape)}")
    src = _src_type("x", x)
    m, k = x.shape
    _need_k("x", k)
    xc = _aligned(x)
    out = _empty(xc, (m, k), (m, _blocks(k)))
    with _on(dev):
        _lib.call("moe_quantize_fp8", _p(xc), src, m, k, _p(out.data), _p(out.scale), _stream(dev))
    return out


def quantize_fp8_weight(w: torch.Tensor) -> Fp8Tensor:
    """Weights w [G,N,K] (bf16 or fp32, K % 16 == 0) with one scale for a block
    of 128 x 128, so that the result serves both layouts of grouped_gemm_fp8."""
    dev = _same_device(w=w)
    if w.dim() != 3 or w.shape[1] < 1:
        raise ValueError(f"w must be [G,N,K], got {tuple(w.shape)}")
    src = _src_type("w", w)
    g, n, k = w.shape
    _need_k("w", k)
    wc = _aligned(w)
    out = _empty(wc, (g, n, k), (g, _blocks(n), _blocks(k)))
    with _on(dev):
        _lib.call("moe_quantize_fp8_weight", _p(wc), src, g, n, k, _p(out.data), _p(out.scale),
                  _stream(dev))
    return out


def dequantize_fp8(q: Fp8Tensor) -> torch.Tensor:
    """bf16 rows of a quantised [M,K] tensor: e4m3 times a power of two, exact
    within bf16's range. Results below 2^-133 are rounded (under the smallest
    scales of fp32 rows alone); values from 1.9375 * 2^127 on were rounded to
    2^128, which reads back as infinity."""
    dev = _same_device(data=q.data, scale=q.scale)
    if q.data.dim() != 2:
        raise ValueError(f"q.data must be [M,K], got {tuple(q.data.shape)}")
    m, k = q.data.shape
    _need_fp8("q", q, (m, _blocks(k)))
    _need_k("q.data", k)
    data, scale = _aligned(q.data), q.scale.contiguous()
    out = data.new_empty((m, k), dtype=torch.bfloat16)
    with _on(dev):
        _lib.call("moe_dequantize_fp8", _p(data), _p(scale), m, k, _p(out), _stream(dev))
    return out


def permute_fp8(x: torch.Tensor, row_id_map: torch.Tensor, experts: torch.Tensor,
                num_out: int) -> Fp8Tensor:
    """ops.permute of the quantised rows of x [T,H] bf16, in one pass: row t is
    quantised once and written to rows row_id_map[t, experts[t,j]].

    row_id_map: the token-major [T,E] int64 map; experts [T,k] int64, k <= 32
    (RouterOutput.topk_idx). Rows of the result that nothing names stay
    uninitialised; experts outside [0,E) and rows outside [0,num_out) are
    skipped."""
    dev = _same_device(x=x, row_id_map=row_id_map, experts=experts)
    _need_dtype("x", x, torch.bfloat16)
    _need_dtype("row_id_map", row_id_map, torch.int64)
    _need_dtype("experts", experts, torch.int64)
    if x.dim() != 2 or row_id_map.dim() != 2 or row_id_map.shape[0] != x.shape[0]:
        raise ValueError(f"shapes x {tuple(x.shape)} row_id_map {tuple(row_id_map.shape)}")
    if experts.dim() != 2 or experts.shape[0] != x.shape[0]:
        raise ValueError(f"experts must be [{x.shape[0]},k], got {tuple(experts.shape)}")
    if num_out < 0:
        raise ValueError(f"num_out must not be negative, got {num_out}")
    t, h = x.shape
    _need_k("x", h)
    xc, mc, ec = _aligned(x), row_id_map.contiguous(), experts.contiguous()
    out = _empty(xc, (int(num_out), h), (int(num_out), _blocks(h)))
    with _on(dev):
        _lib.call("moe_permute_fp8", _p(xc), _p(mc), _p(ec), ec.shape[1], _p(out.data),
                  _p(out.scale), t, h, mc.shape[1], int(num_out), _stream(dev))
    return out


def grouped_gemm_fp8(x: Fp8Tensor, w: Fp8Tensor,
                     m_splits: Union[None, Sequence[int], torch.Tensor] = None,
                     epilogue: str = "none", plan: Optional[GroupedGemmPlan] = None,
                     w_layout: str = "NK", return_pre: bool = False):
    """out = cat_g(x[seg_g] @ w[g].T) of block-scaled e4m3 operands (fp32 accumulation).

    x: rows [R,K]; w: weights [G,N,K] ("[out,in]"), or with w_layout="KN"
    [G,K,N] and out = cat_g(x[seg_g] @ w[g]), the input gradient with the
    forward's weight tensor as it is. m_splits / plan: as ops.grouped_gemm.

    epilogue="none": bf16 [R,N] (N % 8 == 0; % 16 for "KN").
    epilogue="swiglu_fp8": w holds [gate|up] (N = 2F, F % 128 == 0) and the
    result is silu(gate)*up, quantised from fp32, as an Fp8Tensor of rows
    [R,F]; with return_pre (rows, gate|up bf16 [R,N]), for a backward pass.
    Rows in no group stay uninitialised.
    """
    dev = _same_device(x_data=x.data, x_scale=x.scale, w_data=w.data, w_scale=w.scale)
    if w_layout not in ("NK", "KN"):
        raise ValueError("w_layout must be 'NK' (w [G,N,K]) or 'KN' (w [G,K,N])")
    codes = {"none": 0, "swiglu_fp8": 1}
    if epilogue not in codes:
        raise ValueError("epilogue must be 'none' or 'swiglu_fp8'")
    if x.data.dim() != 2 or w.data.dim() != 3 or \
            x.data.shape[1] != w.data.shape[2 if w_layout == "NK" else 1]:
        raise ValueError(f"shapes x {tuple(x.data.shape)} w {tuple(w.data.shape)} ({w_layout})")
    rows, k = x.data.shape
    g, d1, d2 = w.data.shape
    n = d1 if w_layout == "NK" else d2
    if g < 1:
        raise ValueError("w holds no weight matrix")
    _need_k("x.data", k)
    _need_fp8("x", x, (rows, _blocks(k)))
    _need_fp8("w", w, (g, _blocks(d1), _blocks(d2)))
    if epilogue == "swiglu_fp8" and (w_layout == "KN" or n % 256):
        raise ValueError("the SwiGLU epilogue needs w_layout 'NK' and N = 2F with F % 128 == 0")
    if return_pre and epilogue != "swiglu_fp8":
        raise ValueError("return_pre needs epilogue='swiglu_fp8'")
    if n % (16 if w_layout == "KN" else 8):
        raise ValueError(f"N must be a multiple of {16 if w_layout == 'KN' else 8}, got {n}")
    if plan is None:
        if m_splits is None:
            base, rem = divmod(rows, g)
            m_splits = [base + (1 if i < rem else 0) for i in range(g)]
        if not isinstance(m_splits, torch.Tensor):
            if len(m_splits) != g:
                raise ValueError(f"m_splits has {len(m_splits)} entries for {g} groups")
            m_splits = [int(v) for v in m_splits]
            if min(m_splits) < 0:
                raise ValueError(f"m_splits must not be negative, got {min(m_splits)}")
            if sum(m_splits) > rows:
                raise ValueError("sum(m_splits) exceeds x rows")
            m_splits = torch.tensor(m_splits, dtype=torch.int32)
        with _on(dev):
            plan = GroupedGemmPlan(g, dev).from_splits(m_splits)
    if plan.num_w != g or plan.workspace.device != dev:
        raise ValueError(f"plan names {plan.num_w} weight matrices on {plan.workspace.device}, w has "
                         f"{g} on {dev}")
    xd, xs, wd, ws = _aligned(x.data), x.scale.contiguous(), _aligned(w.data), w.scale.contiguous()
    pre = None
    if epilogue == "none":
        out, out_scale = xd.new_empty((rows, n), dtype=torch.bfloat16), None
    else:
        out, out_scale = _empty(xd, (rows, n // 2), (rows, n // 2 // BLOCK))
        if return_pre:
            pre = xd.new_empty((rows, n), dtype=torch.bfloat16)
    with _on(dev):
        _lib.call("moe_grouped_gemm_fp8", _p(xd), _p(xs), _p(wd), _p(ws), _p(out), _p(out_scale),
                  _p(pre), rows, plan.num_groups, g, n, k, 1 if w_layout == "KN" else 0,
                  codes[epilogue], _p(plan.workspace), plan.nbytes, _stream(dev))
    if epilogue == "none":
        return out
    rows_out = Fp8Tensor(out, out_scale)
    return (rows_out, pre) if return_pre else rows_out
