"""``torch.library`` ops backed by the CUDA kernels in ``libdfb200.so``.

Every op of the reference's kernel package that sits on the decode path has a twin here with the same
argument list and the same error behaviour, registered under the ``dfb200::`` namespace:

====================================  ===========================================================
this package                          reference op (file:line of its definition)
====================================  ===========================================================
``dfb200::tiled_gemv_int4``           ``deltaforge::tiled_gemv_int4`` kernels/tiled_gemv.py:915
``dfb200::delta_rule_step``           ``deltaforge::delta_rule_step`` kernels/gated_delta_step.py:109
``dfb200::fused_causal_conv_step``    ``deltaforge::fused_causal_conv_step`` kernels/fused_causal_conv.py:136
``dfb200::gqa_decode_attention``      ``deltaforge::gqa_decode_attention`` kernels/gqa_decode.py:138
``dfb200::split_kv_decode_attention`` ``deltaforge::split_kv_decode_attention`` kernels/flash_decode_splitkv.py:177
``dfb200::add_rms_norm``              ``deltaforge::add_rms_norm`` kernels/fused_rmsnorm_residual.py:164
``dfb200::rms_norm``                  ``deltaforge::rms_norm`` kernels/fused_rmsnorm_residual.py:201
``dfb200::partial_rope``              ``deltaforge::partial_rope`` kernels/fused_rope.py:97
``dfb200::silu_mul``                  ``deltaforge::silu_mul`` kernels/fused_swiglu.py:51
====================================  ===========================================================

plus the fused forms the decode step is built from (``rmsnorm_int4_gemv``, ``int4_gemv_residual``,
``silu_mul_int4_gemv_residual``, ``deltanet_step``, ``attn_prep``, ``attn_decode_gated``), the two
bit-exactness probes ``int4_unpack`` / ``int4_dequant``, and the ops that take several new tokens of a
sequence at once, a prompt or a tree of drafted tokens: ``rotary_qk``, ``rotary_append`` (with
``rope_frequencies``), ``tree_attention``, ``delta_rule_chunk``, ``delta_rule_tree``.

Conventions kept from the reference: shape and dtype errors are ``ValueError`` and are raised before
the device check, so they surface on any machine; a CPU tensor raises ``RuntimeError`` because there is
no PyTorch fallback (kernels/_triton.py:56-69); outputs are allocated on the input's device; layouts
are coerced with ``.contiguous()``, shapes are not.
"""

from __future__ import annotations

import ctypes as C
import functools
import inspect
import math
import operator

import torch
from torch import Tensor

from . import _lib
from ._lib import AttnDesc, AttnPrepDesc, DeltaNetDesc, GemvDesc

MATH_FAST, MATH_EXACT, MATH_FAST_HALF2 = 0, 1, 2
PRO_NONE, PRO_RMSNORM, PRO_SILU_MUL = 0, 1, 2
EPI_STORE, EPI_RESIDUAL, EPI_CONV = 0, 1, 2

BF16 = torch.bfloat16

#: Arithmetic used by the int4 GEMV ops. FAST is the production setting; EXACT rounds each dequantised
#: weight to bf16 like the reference's expression (slower, for cross-checks).
default_math = MATH_FAST


def require_cuda(tensor: Tensor, op: str) -> None:
    if not tensor.is_cuda:
        raise RuntimeError(
            f"dfb200::{op} requires a CUDA tensor and has no PyTorch fallback, on purpose: falling back "
            "would run a different implementation than the one being measured."
        )


def _stream(t: Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _ptr(t: Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


_scratch: dict[tuple, Tensor] = {}


def _zeroed_scratch(device: torch.device, key: tuple, nbytes: int) -> Tensor | None:
    """A per-(device, problem) scratch buffer, zeroed once; the kernels leave their counters at zero."""
    if nbytes == 0:
        return None
    k = (device.index, *key)
    buf = _scratch.get(k)
    if buf is None or buf.numel() < nbytes:
        buf = torch.zeros(nbytes, dtype=torch.uint8, device=device)
        _scratch[k] = buf
    return buf


# --------------------------------------------------------------------------------------
# int4 GEMV family
# --------------------------------------------------------------------------------------


def _check_int4(x: Tensor, packed: Tensor, scale: Tensor, group_size: int, op: str) -> tuple[int, int]:
    if packed.dim() != 2 or packed.dtype != torch.uint8:
        raise ValueError(f"{op}: packed must be a 2-D uint8 tensor [K/2, N], got {tuple(packed.shape)} {packed.dtype}")
    half, n = packed.shape
    k = half * 2
    if x.shape[-1] != k:
        raise ValueError(f"{op}: activation has {x.shape[-1]} features, packed weight expects K={k}")
    if group_size <= 0 or half % group_size:
        raise ValueError(f"{op}: group size {group_size} does not divide K/2 = {half}")
    if tuple(scale.shape) != (k // group_size, n):
        raise ValueError(f"{op}: scale must be [K/group, N] = {(k // group_size, n)}, got {tuple(scale.shape)}")
    if scale.dtype not in (torch.float32, BF16):
        raise ValueError(f"{op}: scale must be float32 or bfloat16, got {scale.dtype}")
    if x.dtype != BF16:
        raise ValueError(f"{op}: activations must be bfloat16, got {x.dtype}")
    return k, n


def int4_gemv_fused(
    x: Tensor,
    packed: Tensor,
    scale: Tensor,
    group_size: int,
    *,
    prologue: int = PRO_NONE,
    norm_weight: Tensor | None = None,
    eps: float = 1e-6,
    up: Tensor | None = None,
    epilogue: int = EPI_STORE,
    residual: Tensor | None = None,
    conv_cache: Tensor | None = None,
    conv_weight: Tensor | None = None,
    math: int | None = None,
    force_tiled: bool = False,
    packed_k8: Tensor | None = None,
    packed_mma: Tensor | None = None,
    op: str = "int4_gemv",
) -> Tensor:
    """The general form behind every int4 linear op of this module. Returns ``[..., N]`` bf16.

    ``packed_k8`` is the optional re-packed copy of the weight (``int4_repack_k8``); with it, one
    activation row and the FAST arithmetic the streaming kernel runs instead of the register-tiled one.
    ``packed_mma`` is the optional copy of weight and scales made by ``int4_repack_mma`` (``pair=False``); with
    it, one activation row and the FAST arithmetic run on the integer tensor-core instruction.
    """
    k, n = _check_int4(x, packed, scale, group_size, op)
    if packed_k8 is not None and (packed_k8.dtype != torch.int32 or tuple(packed_k8.shape) != (k // 8, n)):
        raise ValueError(f"{op}: packed_k8 must be int32 [K/8, N] = {(k // 8, n)}, got {tuple(packed_k8.shape)} {packed_k8.dtype}")
    if prologue == PRO_RMSNORM:
        if norm_weight is None or norm_weight.shape != (k,):
            raise ValueError(f"{op}: RMSNorm weight must have {k} elements")
    if prologue == PRO_SILU_MUL and (up is None or up.shape != x.shape):
        raise ValueError(f"{op}: `up` must match the gate activation's shape {tuple(x.shape)}")
    lead = x.shape[:-1]
    rows = 1
    for s in lead:
        rows *= s
    if epilogue == EPI_RESIDUAL and (residual is None or residual.shape != (*lead, n)):
        raise ValueError(f"{op}: residual must have shape {(*lead, n)}")
    conv_dim = 0
    if epilogue == EPI_CONV:
        if conv_cache is None or conv_weight is None or conv_cache.dim() != 3 or conv_cache.shape[2] != 3:
            raise ValueError(f"{op}: conv epilogue needs a (B, C, 3) history and a (C, 4) weight")
        conv_dim = conv_cache.shape[1]
        if conv_cache.shape[0] != rows or conv_dim > n or conv_weight.numel() != conv_dim * 4:
            raise ValueError(f"{op}: conv history {tuple(conv_cache.shape)} does not match rows={rows}, N={n}")
        if not conv_cache.is_contiguous():
            raise ValueError(f"{op}: the conv history is updated in place and must be contiguous")
    require_cuda(x, op)
    flat = x.reshape(rows, k).contiguous()
    packed = packed.contiguous()
    scale = scale.contiguous()
    out = torch.empty((rows, n), device=x.device, dtype=BF16)
    if rows == 0:
        return out.reshape(*lead, n)
    lib = _lib.load()
    nbytes = lib.dfb_int4_gemv_scratch_bytes(rows, k, n, group_size)
    scratch = _zeroed_scratch(x.device, ("gemv", rows, k, n), nbytes)
    d = GemvDesc()
    d.x, d.x_stride, d.rows = flat.data_ptr(), k, rows
    d.packed, d.scale, d.scale_is_bf16 = packed.data_ptr(), scale.data_ptr(), int(scale.dtype == BF16)
    d.K, d.N, d.group = k, n, group_size
    d.prologue, d.eps = prologue, eps
    keep = [flat, packed, scale, out, scratch]
    if prologue == PRO_RMSNORM:
        nw = norm_weight.to(BF16).contiguous()
        keep.append(nw)
        d.norm_w = nw.data_ptr()
    if prologue == PRO_SILU_MUL:
        upc = up.reshape(rows, k).contiguous()
        keep.append(upc)
        d.up, d.up_stride = upc.data_ptr(), k
    d.epilogue, d.out, d.out_stride = epilogue, out.data_ptr(), n
    if epilogue == EPI_RESIDUAL:
        res = residual.reshape(rows, n).contiguous()
        keep.append(res)
        d.residual, d.residual_stride = res.data_ptr(), n
    if epilogue == EPI_CONV:
        cw = conv_weight.reshape(conv_dim, 4).to(BF16).contiguous()
        keep.append(cw)
        d.conv_state, d.conv_w, d.conv_dim = conv_cache.data_ptr(), cw.data_ptr(), conv_dim
    d.scratch, d.scratch_bytes = _ptr(scratch), nbytes
    d.math = default_math if math is None else math
    d.force_tiled = int(force_tiled)
    if packed_k8 is not None:
        packed_k8 = packed_k8.contiguous()
        keep.append(packed_k8)
        d.packed_k8 = packed_k8.data_ptr()
    if packed_mma is not None:
        want = _lib.load().dfb_int4_repack_mma_bytes(k, n, 0, int(scale.dtype == BF16))
        if packed_mma.dtype != torch.uint8 or packed_mma.numel() != want or not packed_mma.is_contiguous():
            raise ValueError(f"{op}: packed_mma must be the {want} contiguous bytes int4_repack_mma(pair=False) returns for this weight")
        keep.append(packed_mma)
        d.packed_mma = packed_mma.data_ptr()
    _lib.check(lib.dfb_int4_gemv(C.byref(d), _stream(x)), f"dfb200::{op}")
    return out.reshape(*lead, n)


@torch.library.custom_op("dfb200::tiled_gemv_int4", mutates_args=())
def tiled_gemv_int4(x: Tensor, packed: Tensor, scale: Tensor, group_size: int) -> Tensor:
    """Group-wise int4 GEMV. ``packed`` is ``[K // 2, N]``, ``scale`` ``[K // group, N]``."""
    return int4_gemv_fused(x, packed, scale, group_size, op="tiled_gemv_int4")


@tiled_gemv_int4.register_fake
def _(x, packed, scale, group_size):
    return x.new_empty((*x.shape[:-1], packed.shape[1]))


@torch.library.custom_op("dfb200::rmsnorm_int4_gemv", mutates_args=())
def rmsnorm_int4_gemv(x: Tensor, norm_weight: Tensor, eps: float, packed: Tensor, scale: Tensor, group_size: int) -> Tensor:
    """``tiled_gemv_int4(rms_norm(x, norm_weight, eps), ...)`` in one kernel."""
    return int4_gemv_fused(x, packed, scale, group_size, prologue=PRO_RMSNORM, norm_weight=norm_weight, eps=eps, op="rmsnorm_int4_gemv")


@rmsnorm_int4_gemv.register_fake
def _(x, norm_weight, eps, packed, scale, group_size):
    return x.new_empty((*x.shape[:-1], packed.shape[1]))


@torch.library.custom_op("dfb200::int4_gemv_residual", mutates_args=())
def int4_gemv_residual(x: Tensor, packed: Tensor, scale: Tensor, group_size: int, residual: Tensor) -> Tensor:
    """``residual + tiled_gemv_int4(x, ...)`` in one kernel (the sum is rounded to bf16 once more)."""
    return int4_gemv_fused(x, packed, scale, group_size, epilogue=EPI_RESIDUAL, residual=residual, op="int4_gemv_residual")


@int4_gemv_residual.register_fake
def _(x, packed, scale, group_size, residual):
    return torch.empty_like(residual)


@torch.library.custom_op("dfb200::silu_mul_int4_gemv_residual", mutates_args=())
def silu_mul_int4_gemv_residual(gate: Tensor, up: Tensor, packed: Tensor, scale: Tensor, group_size: int, residual: Tensor) -> Tensor:
    """``residual + tiled_gemv_int4(silu(gate) * up, ...)``: the MLP's down projection in one kernel."""
    return int4_gemv_fused(
        gate, packed, scale, group_size, prologue=PRO_SILU_MUL, up=up, epilogue=EPI_RESIDUAL, residual=residual,
        op="silu_mul_int4_gemv_residual",
    )  # fmt: skip


@silu_mul_int4_gemv_residual.register_fake
def _(gate, up, packed, scale, group_size, residual):
    return torch.empty_like(residual)


@torch.library.custom_op("dfb200::rmsnorm_int4_gemv_conv", mutates_args=("conv_cache",))
def rmsnorm_int4_gemv_conv(
    x: Tensor, norm_weight: Tensor, eps: float, packed: Tensor, scale: Tensor, group_size: int, conv_cache: Tensor, conv_weight: Tensor
) -> Tensor:
    """DeltaNet input projections: RMSNorm, GEMV over qkv|z|b|a, conv step + SiLU on the first C columns."""
    return int4_gemv_fused(
        x, packed, scale, group_size, prologue=PRO_RMSNORM, norm_weight=norm_weight, eps=eps, epilogue=EPI_CONV,
        conv_cache=conv_cache, conv_weight=conv_weight, op="rmsnorm_int4_gemv_conv",
    )  # fmt: skip


@rmsnorm_int4_gemv_conv.register_fake
def _(x, norm_weight, eps, packed, scale, group_size, conv_cache, conv_weight):
    return x.new_empty((*x.shape[:-1], packed.shape[1]))


@torch.library.custom_op("dfb200::int4_repack_k8", mutates_args=())
def int4_repack_k8(packed: Tensor) -> Tensor:
    """``packed [K/2, N]`` uint8 -> int32 ``[K/8, N]``: word ``(kb, n)`` holds the eight nibbles of column
    ``n`` for rows ``8kb .. 8kb+7`` (nibble ``i`` = row ``8kb + i``). The layout the streaming GEMV reads."""
    if packed.dim() != 2 or packed.dtype != torch.uint8 or (packed.shape[0] * 2) % 8:
        raise ValueError(f"int4_repack_k8: expected uint8 [K/2, N] with K a multiple of 8, got {tuple(packed.shape)} {packed.dtype}")
    require_cuda(packed, "int4_repack_k8")
    packed = packed.contiguous()
    half, n = packed.shape
    out = torch.empty((half // 4, n), dtype=torch.int32, device=packed.device)
    if out.numel():
        _lib.check(_lib.load().dfb_int4_repack_k8(packed.data_ptr(), 2 * half, n, out.data_ptr(), _stream(packed)), "dfb200::int4_repack_k8")
    return out


@int4_repack_k8.register_fake
def _(packed):
    return packed.new_empty((packed.shape[0] // 4, packed.shape[1]), dtype=torch.int32)


def int4_repack_mma(packed: Tensor, scale: Tensor, *, pair: bool = False) -> Tensor:
    """``packed [K/2, N]`` uint8 and ``scale [K/128, N]`` (fp32 or bf16) -> the bytes the integer tensor-core GEMV
    streams (``dfb_int4_repack_mma``): one contiguous unit per (column tile, 128-row group) with the group's words in
    operand-fragment order followed by its scales. ``pair=True`` lays a ``gate_proj|up_proj`` matrix out with each
    tile holding 128 gate columns and the matching up columns. K must be a multiple of 128."""
    if packed.dim() != 2 or packed.dtype != torch.uint8:
        raise ValueError(f"int4_repack_mma: expected uint8 [K/2, N], got {tuple(packed.shape)} {packed.dtype}")
    half, n = packed.shape
    k = 2 * half
    if k % 128 or scale.shape != (k // 128, n) or scale.dtype not in (torch.float32, BF16):
        raise ValueError(f"int4_repack_mma: K = {k} must be a multiple of 128 with scales [K/128, N] in fp32 or bf16, got {tuple(scale.shape)} {scale.dtype}")
    if pair and n % 2:
        raise ValueError("int4_repack_mma: a gate|up pair has an even number of columns")
    require_cuda(packed, "int4_repack_mma")
    packed, scale = packed.contiguous(), scale.contiguous()
    lib = _lib.load()
    is_bf16 = int(scale.dtype == BF16)
    out = torch.empty(lib.dfb_int4_repack_mma_bytes(k, n, int(pair), is_bf16), dtype=torch.uint8, device=packed.device)
    _lib.check(lib.dfb_int4_repack_mma(packed.data_ptr(), scale.data_ptr(), is_bf16, k, n, int(pair), out.data_ptr(), _stream(packed)),
               "dfb200::int4_repack_mma")  # fmt: skip
    return out


@torch.library.custom_op("dfb200::int4_unpack", mutates_args=())
def int4_unpack(packed: Tensor) -> Tensor:
    """``packed [K/2, N]`` -> signed int8 values ``[K, N]`` (low nibbles are rows 0..K/2)."""
    if packed.dim() != 2 or packed.dtype != torch.uint8:
        raise ValueError(f"int4_unpack: expected a 2-D uint8 tensor, got {tuple(packed.shape)} {packed.dtype}")
    require_cuda(packed, "int4_unpack")
    packed = packed.contiguous()
    half, n = packed.shape
    out = torch.empty((2 * half, n), dtype=torch.int8, device=packed.device)
    if out.numel():
        _lib.check(_lib.load().dfb_int4_unpack(packed.data_ptr(), 2 * half, n, out.data_ptr(), _stream(packed)), "dfb200::int4_unpack")
    return out


@int4_unpack.register_fake
def _(packed):
    return packed.new_empty((packed.shape[0] * 2, packed.shape[1]), dtype=torch.int8)


@torch.library.custom_op("dfb200::int4_dequant", mutates_args=())
def int4_dequant(packed: Tensor, scale: Tensor, group_size: int) -> Tensor:
    """bf16 weight ``[K, N]`` = bf16(value * scale): the tensor the reference's expression multiplies by."""
    if packed.dim() != 2 or packed.dtype != torch.uint8:
        raise ValueError(f"int4_dequant: expected a 2-D uint8 tensor, got {tuple(packed.shape)} {packed.dtype}")
    half, n = packed.shape
    if group_size <= 0 or half % group_size or tuple(scale.shape) != (2 * half // group_size, n):
        raise ValueError(f"int4_dequant: scale {tuple(scale.shape)} does not match K={2 * half}, N={n}, group={group_size}")
    if scale.dtype not in (torch.float32, BF16):
        raise ValueError(f"int4_dequant: scale must be float32 or bfloat16, got {scale.dtype}")
    require_cuda(packed, "int4_dequant")
    packed, scale = packed.contiguous(), scale.contiguous()
    out = torch.empty((2 * half, n), dtype=BF16, device=packed.device)
    if out.numel():
        rc = _lib.load().dfb_int4_dequant(
            packed.data_ptr(), scale.data_ptr(), int(scale.dtype == BF16), 2 * half, n, group_size, out.data_ptr(), _stream(packed)
        )
        _lib.check(rc, "dfb200::int4_dequant")
    return out


@int4_dequant.register_fake
def _(packed, scale, group_size):
    return packed.new_empty((packed.shape[0] * 2, packed.shape[1]), dtype=BF16)


# --------------------------------------------------------------------------------------
# Norms and elementwise
# --------------------------------------------------------------------------------------


def _check_norm(x: Tensor, weight: Tensor, name: str, residual: Tensor | None = None) -> None:
    if weight.dim() != 1 or not weight.is_contiguous():
        raise ValueError("norm weight must be a contiguous 1-D tensor; the kernel indexes it by column")
    if x.shape[-1] != weight.shape[0]:
        raise ValueError(f"weight has {weight.shape[0]} elements, activation row is {x.shape[-1]}")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"residual shape {tuple(residual.shape)} != activation shape {tuple(x.shape)}")
        if residual.dtype != x.dtype:
            raise ValueError(f"residual dtype {residual.dtype} != activation dtype {x.dtype}")
    if x.dtype != BF16:
        raise ValueError(f"{name}: activations must be bfloat16, got {x.dtype}")
    require_cuda(x, name)


@torch.library.custom_op("dfb200::rms_norm", mutates_args=())
def rms_norm(x: Tensor, weight: Tensor, eps: float) -> Tensor:
    """RMSNorm with the ``1 + weight`` scale."""
    _check_norm(x, weight, "rms_norm")
    x = x.contiguous()
    w = weight.to(BF16)
    n = x.shape[-1]
    out = torch.empty_like(x)
    if x.numel():
        _lib.check(_lib.load().dfb_rms_norm(x.data_ptr(), w.data_ptr(), eps, x.numel() // n, n, out.data_ptr(), _stream(x)), "dfb200::rms_norm")
    return out


@rms_norm.register_fake
def _(x, weight, eps):
    return torch.empty_like(x)


@torch.library.custom_op("dfb200::add_rms_norm", mutates_args=())
def add_rms_norm(x: Tensor, residual: Tensor, weight: Tensor, eps: float) -> tuple[Tensor, Tensor]:
    """``(residual + x, rms_norm(residual + x))`` in one pass."""
    _check_norm(x, weight, "add_rms_norm", residual=residual)
    x, residual = x.contiguous(), residual.contiguous()
    w = weight.to(BF16)
    n = x.shape[-1]
    resid_out, out = torch.empty_like(x), torch.empty_like(x)
    if x.numel():
        rc = _lib.load().dfb_add_rms_norm(
            x.data_ptr(), residual.data_ptr(), w.data_ptr(), eps, x.numel() // n, n, resid_out.data_ptr(), out.data_ptr(), _stream(x)
        )
        _lib.check(rc, "dfb200::add_rms_norm")
    return resid_out, out


@add_rms_norm.register_fake
def _(x, residual, weight, eps):
    return torch.empty_like(x), torch.empty_like(x)


@torch.library.custom_op("dfb200::silu_mul", mutates_args=())
def silu_mul(gate: Tensor, up: Tensor) -> Tensor:
    """``F.silu(gate) * up`` in one pass."""
    if gate.shape != up.shape:
        raise ValueError(f"gate shape {tuple(gate.shape)} != up shape {tuple(up.shape)}")
    if gate.dtype != up.dtype:
        raise ValueError(f"gate dtype {gate.dtype} != up dtype {up.dtype}")
    if gate.dtype != BF16:
        raise ValueError(f"silu_mul: activations must be bfloat16, got {gate.dtype}")
    require_cuda(gate, "silu_mul")
    gate, up = gate.contiguous(), up.contiguous()
    out = torch.empty_like(up)
    if out.numel():
        _lib.check(_lib.load().dfb_silu_mul(gate.data_ptr(), up.data_ptr(), out.numel(), out.data_ptr(), _stream(gate)), "dfb200::silu_mul")
    return out


@silu_mul.register_fake
def _(gate, up):
    return torch.empty_like(up)


@torch.library.custom_op("dfb200::partial_rope", mutates_args=())
def partial_rope(x: Tensor, cos: Tensor, sin: Tensor) -> Tensor:
    """Rotate the leading ``rotary_dim`` dims of ``x (batch, heads, seq, head_dim)``."""
    if x.dim() != 4:
        raise ValueError(f"expected (batch, heads, seq, head_dim), got {tuple(x.shape)}")
    if cos.shape != sin.shape:
        raise ValueError(f"cos shape {tuple(cos.shape)} != sin shape {tuple(sin.shape)}")
    if cos.dim() != 3:
        raise ValueError(f"expected cos as (batch, seq, rotary_dim), got {tuple(cos.shape)}")
    batch, heads, seq_len, head_dim = x.shape
    rotary_dim = cos.shape[-1]
    if cos.shape[0] != batch or cos.shape[1] != seq_len:
        raise ValueError(f"cos {tuple(cos.shape)} does not match x {tuple(x.shape)} on batch/seq")
    if rotary_dim > head_dim:
        raise ValueError(f"rotary_dim {rotary_dim} exceeds head_dim {head_dim}")
    if rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even to rotate in halves, got {rotary_dim}")
    if x.dtype != BF16:
        raise ValueError(f"partial_rope: activations must be bfloat16, got {x.dtype}")
    require_cuda(x, "partial_rope")
    x = x.contiguous()
    cos, sin = cos.to(BF16).contiguous(), sin.to(BF16).contiguous()
    out = torch.empty_like(x)
    if out.numel():
        rc = _lib.load().dfb_partial_rope(
            x.data_ptr(), cos.data_ptr(), sin.data_ptr(), batch, heads, seq_len, head_dim, rotary_dim, out.data_ptr(), _stream(x)
        )
        _lib.check(rc, "dfb200::partial_rope")
    return out


@partial_rope.register_fake
def _(x, cos, sin):
    return torch.empty_like(x)


@torch.library.custom_op("dfb200::fused_causal_conv_step", mutates_args=("conv_cache",))
def fused_causal_conv_step(x: Tensor, conv_cache: Tensor, weight: Tensor) -> Tensor:
    """``x (B, C, 1)``, ``conv_cache (B, C, 3)`` advanced in place, ``weight (C, 1, 4)`` -> ``(B, C, 1)``."""
    batch, channels, steps = x.shape
    if steps != 1:
        raise ValueError(f"fused_causal_conv_step is the decode step; got seq_len {steps}")
    if conv_cache.shape != (batch, channels, 3):
        raise ValueError(f"expected a (B, C, 3) history, got {tuple(conv_cache.shape)}")
    w = weight.reshape(channels, -1)
    if w.shape[1] != 4:
        raise ValueError(f"this kernel is the four-tap case; got {w.shape[1]} taps")
    if x.dtype != BF16 or conv_cache.dtype != BF16:
        raise ValueError("fused_causal_conv_step: activations and history must be bfloat16")
    if not conv_cache.is_contiguous():
        raise ValueError("the conv history is updated in place and must be contiguous")
    require_cuda(x, "fused_causal_conv_step")
    xc = x.contiguous()
    w = w.to(BF16).contiguous()
    out = torch.empty_like(xc)
    if out.numel():
        rc = _lib.load().dfb_causal_conv_step(xc.data_ptr(), conv_cache.data_ptr(), w.data_ptr(), batch, channels, out.data_ptr(), _stream(x))
        _lib.check(rc, "dfb200::fused_causal_conv_step")
    return out


@fused_causal_conv_step.register_fake
def _(x, conv_cache, weight):
    return torch.empty_like(x)


# --------------------------------------------------------------------------------------
# Gated DeltaNet
# --------------------------------------------------------------------------------------


@torch.library.custom_op("dfb200::delta_rule_step", mutates_args=())
def delta_rule_step(state: Tensor, query: Tensor, key: Tensor, value: Tensor, g: Tensor, beta: Tensor) -> tuple[Tensor, Tensor]:
    """One delta-rule step on pre-normalised q, k. Returns ``(output fp32, new_state)``."""
    if state.dim() != 4:
        raise ValueError(f"expected state (batch, heads, key_dim, value_dim), got {tuple(state.shape)}")
    batch, heads, key_dim, value_dim = state.shape
    for name, t, shape in (
        ("query", query, (batch, heads, key_dim)),
        ("key", key, (batch, heads, key_dim)),
        ("value", value, (batch, heads, value_dim)),
        ("g", g, (batch, heads)),
        ("beta", beta, (batch, heads)),
    ):
        if tuple(t.shape) != shape:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {shape}")
    if state.dtype != torch.float32:
        raise ValueError(
            f"the recurrent state is fp32 by config (mamba_ssm_dtype), got {state.dtype}. "
            "Running it in bf16 would change the model, not just the kernel."
        )
    require_cuda(state, "delta_rule_step")
    state = state.contiguous()
    q, k, v, gg, bb = (t.float().contiguous() for t in (query, key, value, g, beta))
    out = torch.empty((batch, heads, value_dim), device=state.device, dtype=torch.float32)
    state_out = torch.empty_like(state)
    if state.numel():
        rc = _lib.load().dfb_delta_rule_step(
            state.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), gg.data_ptr(), bb.data_ptr(),
            batch, heads, key_dim, value_dim, out.data_ptr(), state_out.data_ptr(), _stream(state),
        )  # fmt: skip
        _lib.check(rc, "dfb200::delta_rule_step")
    return out, state_out


@delta_rule_step.register_fake
def _(state, query, key, value, g, beta):
    b, h, _, dv = state.shape
    return torch.empty((b, h, dv), device=state.device, dtype=torch.float32), torch.empty_like(state)


@torch.library.custom_op("dfb200::deltanet_step", mutates_args=("state",))
def deltanet_step(
    q: Tensor, k: Tensor, v: Tensor, z: Tensor, b: Tensor, a: Tensor, a_log: Tensor, dt_bias: Tensor, norm_weight: Tensor,
    eps: float, state: Tensor,
) -> Tensor:  # fmt: skip
    """DeltaNet core for one token: ``q,k (B,Hk,dk)``, ``v,z (B,Hv,dv)``, ``b,a (B,Hv)`` post-conv bf16;
    ``state (B,Hv,dk,dv)`` fp32 updated in place. Returns the gated-normed output ``(B, Hv*dv)`` bf16."""
    if state.dim() != 4 or state.dtype != torch.float32:
        raise ValueError(f"state must be fp32 (batch, heads, key_dim, value_dim), got {tuple(state.shape)} {state.dtype}")
    batch, hv, dk, dv = state.shape
    if q.dim() != 3 or q.shape != k.shape or q.shape[0] != batch or q.shape[2] != dk:
        raise ValueError(f"q/k must be (batch, key_heads, {dk}), got {tuple(q.shape)} and {tuple(k.shape)}")
    hk = q.shape[1]
    if hk == 0 or hv % hk:
        raise ValueError(f"{hv} value heads do not divide into {hk} key heads")
    for name, t, shape in (("v", v, (batch, hv, dv)), ("z", z, (batch, hv, dv)), ("b", b, (batch, hv)), ("a", a, (batch, hv))):
        if tuple(t.shape) != shape:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {shape}")
    if a_log.shape != (hv,) or dt_bias.shape != (hv,) or norm_weight.shape != (dv,):
        raise ValueError("A_log and dt_bias must have one entry per value head, the norm weight one per value dim")
    if not state.is_contiguous():
        raise ValueError("the recurrent state is updated in place and must be contiguous")
    require_cuda(state, "deltanet_step")
    # one row per sequence: [q | k | v | z | b | a]
    row = torch.cat([t.reshape(batch, -1).to(BF16) for t in (q, k, v, z, b, a)], dim=1).contiguous()
    kd, vd = hk * dk, hv * dv
    out = torch.empty((batch, vd), device=state.device, dtype=BF16)
    al, dtb, nw = a_log.float().contiguous(), dt_bias.float().contiguous(), norm_weight.float().contiguous()
    d = DeltaNetDesc()
    d.batch, d.num_k_heads, d.num_v_heads, d.dk, d.dv = batch, hk, hv, dk, dv
    es = row.element_size()
    base = row.data_ptr()
    d.q, d.k, d.v = base, base + kd * es, base + 2 * kd * es
    d.z, d.b, d.a = base + (2 * kd + vd) * es, base + (2 * kd + 2 * vd) * es, base + (2 * kd + 2 * vd + hv) * es
    d.row_stride = row.shape[1]
    d.a_log, d.dt_bias, d.norm_w = al.data_ptr(), dtb.data_ptr(), nw.data_ptr()
    d.norm_w_is_bf16 = int(norm_weight.dtype == BF16)
    d.eps = eps
    d.state, d.out, d.out_stride = state.data_ptr(), out.data_ptr(), vd
    if batch:
        _lib.check(_lib.load().dfb_deltanet_step(C.byref(d), _stream(state)), "dfb200::deltanet_step")
    return out


@deltanet_step.register_fake
def _(q, k, v, z, b, a, a_log, dt_bias, norm_weight, eps, state):
    return state.new_empty((state.shape[0], state.shape[1] * state.shape[3]), dtype=BF16)


# --------------------------------------------------------------------------------------
# Decode attention
# --------------------------------------------------------------------------------------


def _check_attn(query: Tensor, key: Tensor, value: Tensor) -> tuple[int, int, int, int, int]:
    if query.dim() != 3:
        raise ValueError(f"expected query (batch, heads_q, head_dim), got {tuple(query.shape)}")
    if key.dim() != 4 or value.dim() != 4:
        raise ValueError(f"expected key/value (batch, heads_kv, key_len, head_dim), got {tuple(key.shape)} and {tuple(value.shape)}")
    if key.shape != value.shape:
        raise ValueError(f"key {tuple(key.shape)} and value {tuple(value.shape)} must match")
    batch, heads_q, head_dim = query.shape
    kv_batch, heads_kv, key_len, kv_dim = key.shape
    if kv_batch != batch or kv_dim != head_dim:
        raise ValueError(f"key {tuple(key.shape)} does not match query {tuple(query.shape)}")
    if heads_kv == 0 or heads_q % heads_kv:
        raise ValueError(f"{heads_q} query heads do not divide into {heads_kv} KV heads")
    if key_len < 1:
        raise ValueError("cannot attend over an empty KV cache")
    for name, t in (("query", query), ("key", key), ("value", value)):
        if t.stride(-1) != 1:
            raise ValueError(f"{name} must have the head dimension innermost and contiguous")
        if t.dtype != BF16:
            raise ValueError(f"{name} must be bfloat16, got {t.dtype}")
    return batch, heads_q, heads_kv, key_len, head_dim


def _attention(query: Tensor, key: Tensor, value: Tensor, scale: float, splits: int, gate: Tensor | None, swish: bool, op: str) -> Tensor:
    batch, hq, hkv, key_len, d = _check_attn(query, key, value)
    if gate is not None and gate.shape != query.shape:
        raise ValueError(f"gate shape {tuple(gate.shape)} != query shape {tuple(query.shape)}")
    require_cuda(query, op)
    query = query.contiguous()
    # Key and value may be views of a longer cache: rows stay where they are as long as a head's rows
    # are `head_dim` apart; anything else is copied.
    def rows_dense(t: Tensor) -> bool:
        return t.stride(2) == d and t.stride(3) == 1

    if not (rows_dense(key) and rows_dense(value) and key.stride() == value.stride()):
        key, value = key.contiguous(), value.contiguous()
    out = torch.empty((batch, hq * d), device=query.device, dtype=BF16)
    lib = _lib.load()
    nbytes = lib.dfb_attn_scratch_bytes(batch, hq, hkv, d, splits)
    scratch = _zeroed_scratch(query.device, ("attn", batch, hq, hkv, d, splits), nbytes)
    a = AttnDesc()
    a.batch, a.hq, a.hkv, a.d = batch, hq, hkv, d
    a.q, a.q_stride, a.qh_stride = query.data_ptr(), hq * d, d
    a.kcache, a.vcache = key.data_ptr(), value.data_ptr()
    a.kv_batch_stride, a.kv_head_stride = key.stride(0), key.stride(1)
    a.key_len, a.pos, a.scale, a.splits = key_len, None, scale, splits
    a.scratch, a.scratch_bytes = _ptr(scratch), nbytes
    if gate is not None:
        gate = gate.to(BF16).contiguous()
        a.gate, a.gate_stride, a.gateh_stride, a.gate_is_swish = gate.data_ptr(), hq * d, d, int(swish)
    a.out, a.out_stride = out.data_ptr(), hq * d
    _lib.check(lib.dfb_attn_decode(C.byref(a), _stream(query)), f"dfb200::{op}")
    return out.reshape(batch, hq, d)


@torch.library.custom_op("dfb200::gqa_decode_attention", mutates_args=())
def gqa_decode_attention(query: Tensor, key: Tensor, value: Tensor, scale: float) -> Tensor:
    """Single-token GQA attention against an unexpanded KV cache, one pass over the keys."""
    return _attention(query, key, value, scale, 1, None, False, "gqa_decode_attention")


@gqa_decode_attention.register_fake
def _(query, key, value, scale):
    return torch.empty_like(query)


@torch.library.custom_op("dfb200::split_kv_decode_attention", mutates_args=())
def split_kv_decode_attention(query: Tensor, key: Tensor, value: Tensor, scale: float, splits: int) -> Tensor:
    """Same result with the key scan cut into ``splits`` slices merged by log-sum-exp."""
    if splits < 1 or splits & (splits - 1):
        raise ValueError(f"splits must be a power of two so the merge can index it, got {splits}")
    if splits > 128:
        raise ValueError(f"at most 128 splits are supported, got {splits}")
    return _attention(query, key, value, scale, splits, None, False, "split_kv_decode_attention")


@split_kv_decode_attention.register_fake
def _(query, key, value, scale, splits):
    return torch.empty_like(query)


@torch.library.custom_op("dfb200::attn_decode_gated", mutates_args=())
def attn_decode_gated(query: Tensor, key: Tensor, value: Tensor, scale: float, splits: int, gate: Tensor, swish: bool) -> Tensor:
    """Split-KV decode attention times the output gate (sigmoid, or SiLU when ``swish``)."""
    if splits < 1 or splits > 128:
        raise ValueError(f"splits must be in 1..128, got {splits}")
    return _attention(query, key, value, scale, splits, gate, swish, "attn_decode_gated")


@attn_decode_gated.register_fake
def _(query, key, value, scale, splits, gate, swish):
    return torch.empty_like(query)


@torch.library.custom_op("dfb200::attn_prep", mutates_args=("key_cache", "value_cache"))
def attn_prep(
    proj: Tensor, q_norm_weight: Tensor, k_norm_weight: Tensor, eps: float, inv_freq: Tensor, pos: Tensor,
    key_cache: Tensor, value_cache: Tensor, num_heads: int, output_gate: bool,
) -> Tensor:  # fmt: skip
    """q/k RMSNorm, partial RoPE at device position ``pos`` and the KV-cache write, from the fused
    ``q(|gate)|k|v`` projection row ``proj (B, width)``. Returns the rotated query ``(B, Hq, D)``."""
    if key_cache.dim() != 4 or key_cache.shape != value_cache.shape:
        raise ValueError(f"caches must both be (batch, kv_heads, max_seq, head_dim), got {tuple(key_cache.shape)}")
    batch, hkv, max_seq, d = key_cache.shape
    width = num_heads * d * (2 if output_gate else 1) + 2 * hkv * d
    if proj.shape != (batch, width):
        raise ValueError(f"proj must be {(batch, width)}, got {tuple(proj.shape)}")
    if q_norm_weight.shape != (d,) or k_norm_weight.shape != (d,):
        raise ValueError(f"q/k norm weights must have {d} elements")
    rd = 2 * inv_freq.numel()
    if rd > d:
        raise ValueError(f"rotary_dim {rd} exceeds head_dim {d}")
    if pos.dtype != torch.int32 or pos.numel() != 1:
        raise ValueError("pos must be a single int32 on the device")
    if not (key_cache.is_contiguous() and value_cache.is_contiguous()):
        raise ValueError("the KV caches are written in place and must be contiguous")
    require_cuda(proj, "attn_prep")
    proj = proj.contiguous()
    qw, kw = q_norm_weight.to(BF16).contiguous(), k_norm_weight.to(BF16).contiguous()
    inv = inv_freq.float().contiguous()
    q_out = torch.empty((batch, num_heads, d), device=proj.device, dtype=BF16)
    p = AttnPrepDesc()
    p.batch, p.hq, p.hkv, p.d, p.rotary_dim = batch, num_heads, hkv, d, rd
    p.proj, p.proj_stride = proj.data_ptr(), width
    p.q_norm_w, p.k_norm_w, p.eps = qw.data_ptr(), kw.data_ptr(), eps
    p.inv_freq, p.pos, p.q_out = inv.data_ptr(), pos.data_ptr(), q_out.data_ptr()
    p.kcache, p.vcache = key_cache.data_ptr(), value_cache.data_ptr()
    p.kv_batch_stride, p.kv_head_stride = hkv * max_seq * d, max_seq * d
    p.attn_output_gate, p.max_seq = int(output_gate), max_seq
    _lib.check(_lib.load().dfb_attn_prep(C.byref(p), _stream(proj)), "dfb200::attn_prep")
    return q_out


@attn_prep.register_fake
def _(proj, q_norm_weight, k_norm_weight, eps, inv_freq, pos, key_cache, value_cache, num_heads, output_gate):
    return proj.new_empty((proj.shape[0], num_heads, key_cache.shape[3]))


@torch.library.custom_op("dfb200::attn_step", mutates_args=("key_cache", "value_cache"))
def attn_step(
    proj: Tensor, q_norm_weight: Tensor, k_norm_weight: Tensor, eps: float, inv_freq: Tensor, pos: Tensor,
    key_cache: Tensor, value_cache: Tensor, num_heads: int, output_gate: bool, swish: bool, splits: int, cluster_size: int,
) -> Tensor:  # fmt: skip
    """``attn_prep`` + gated split-KV decode attention in one launch, for one new token per sequence.

    ``proj (B, width)`` is the fused ``q(|gate)|k|v`` projection row, ``pos`` the device-side number of
    cached tokens (the new token becomes row ``pos`` of the caches). Returns ``(B, Hq * D)`` bf16.
    ``splits`` is a power of two with ``ceil(max_seq / splits) <= 160``; ``cluster_size`` 0 picks min(splits, 4).
    """
    if key_cache.dim() != 4 or key_cache.shape != value_cache.shape:
        raise ValueError(f"caches must both be (batch, kv_heads, max_seq, head_dim), got {tuple(key_cache.shape)}")
    batch, hkv, max_seq, d = key_cache.shape
    width = num_heads * d * (2 if output_gate else 1) + 2 * hkv * d
    if proj.shape != (batch, width):
        raise ValueError(f"proj must be {(batch, width)}, got {tuple(proj.shape)}")
    if q_norm_weight.shape != (d,) or k_norm_weight.shape != (d,):
        raise ValueError(f"q/k norm weights must have {d} elements")
    if splits < 1 or splits & (splits - 1):
        raise ValueError(f"splits must be a power of two, got {splits}")
    if -(-max_seq // splits) > 160:
        raise ValueError(f"{splits} slices of a {max_seq}-row cache exceed 160 keys per slice")
    if pos.dtype != torch.int32 or pos.numel() != 1:
        raise ValueError("pos must be a single int32 on the device")
    if not (key_cache.is_contiguous() and value_cache.is_contiguous()):
        raise ValueError("the KV caches are written in place and must be contiguous")
    if proj.dtype != BF16 or key_cache.dtype != BF16:
        raise ValueError("attn_step: activations and caches must be bfloat16")
    require_cuda(proj, "attn_step")
    proj = proj.contiguous()
    qw, kw = q_norm_weight.to(BF16).contiguous(), k_norm_weight.to(BF16).contiguous()
    inv = inv_freq.float().contiguous()
    out = torch.empty((batch, num_heads * d), device=proj.device, dtype=BF16)
    lib = _lib.load()
    nbytes = lib.dfb_attn_scratch_bytes(batch, num_heads, hkv, d, splits)
    scratch = _zeroed_scratch(proj.device, ("attn", batch, num_heads, hkv, d, splits), nbytes)
    a = _lib.AttnStepDesc()
    a.batch, a.hq, a.hkv, a.d, a.rotary_dim = batch, num_heads, hkv, d, 2 * inv.numel()
    a.proj, a.proj_stride = proj.data_ptr(), width
    a.q_norm_w, a.k_norm_w, a.eps = qw.data_ptr(), kw.data_ptr(), eps
    a.inv_freq, a.pos = inv.data_ptr(), pos.data_ptr()
    a.kcache, a.vcache = key_cache.data_ptr(), value_cache.data_ptr()
    a.kv_batch_stride, a.kv_head_stride, a.max_seq = hkv * max_seq * d, max_seq * d, max_seq
    a.attn_output_gate, a.gate_is_swish, a.scale = int(output_gate), int(swish), d**-0.5
    a.splits, a.cluster_size = splits, cluster_size
    a.scratch, a.scratch_bytes = _ptr(scratch), nbytes
    a.out, a.out_stride, a.status = out.data_ptr(), num_heads * d, None
    _lib.check(lib.dfb_attn_step(C.byref(a), _stream(proj)), "dfb200::attn_step")
    return out


@attn_step.register_fake
def _(proj, q_norm_weight, k_norm_weight, eps, inv_freq, pos, key_cache, value_cache, num_heads, output_gate, swish, splits, cluster_size):
    return proj.new_empty((proj.shape[0], num_heads * key_cache.shape[3]))


# --------------------------------------------------------------------------------------
# Several new tokens of a sequence at once: prompts, and trees of drafted tokens
# --------------------------------------------------------------------------------------
#
# Layout of all four: activations are (batch, tokens, heads, dim), which is what a projection's rows are; any strides with
# the last dim contiguous are read in place (so a fused projection's row can be passed as views of it, and a
# (batch, heads, seq, dim) tensor as its transpose). Outputs are new and contiguous.

MAX_TREE_NODES = 64
_DTYPES = {BF16: 0, torch.float16: 1, torch.float32: 2}
_ROTARY, _TREE, _DELTA = (_lib.packer(d) for d in (_lib.RotaryDesc, _lib.TreeAttnDesc, _lib.DeltaChunkDesc))


_dispatch_modes, _function_modes = torch._C._len_torch_dispatch_stack, torch._C._len_torch_function_stack
_transforms, _tracing = torch._C._functorch.peek_interpreter_stack, torch._C._is_tracing
_current_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


@functools.lru_cache(maxsize=4096)
def _scratch_bytes(query: str, *sizes: int) -> int:
    """What a scratch-size query of the library says; it depends on the sizes alone. (Bounded: a server meets prompts of every
    length.)"""
    return getattr(_lib.load(), query)(*sizes)


def _eager(op):
    """The function of a custom op, called directly where the dispatcher has nothing to add: plain tensors whose memory holds
    their values, nothing that compiles, traces or transforms, no dispatch or function mode, no gradient asked for. The
    dispatcher's 20 us are more than the smallest of these calls takes. Everything else goes through the op (and meets its
    errors there)."""
    run, mutates = op._init_fn, op._opoverload._schema.is_mutable
    params = list(inspect.signature(run).parameters.values())
    count = len(params)
    # activations, states and caches; and whole numbers, which have no gradients and no negative views
    counts = ("positions", "cache_len", "parents", "lengths")
    tensors = [i for i, x in enumerate(params) if "Tensor" in str(x.annotation)]
    values = operator.itemgetter(*(i for i in tensors if params[i].name not in counts))
    numbers = tuple(i for i in tensors if params[i].name in counts)
    caches = operator.itemgetter(*(i for i, x in enumerate(params) if x.name in ("key_cache", "value_cache"))) if mutates else None

    @functools.wraps(run)
    def call(*args, **kwargs):
        # (compiling first: the compiler follows this function, and stops at the other questions)
        if torch.compiler.is_dynamo_compiling() or kwargs or len(args) != count:
            return op(*args, **kwargs)
        if _dispatch_modes() or _function_modes() or _transforms() is not None or _tracing():
            return op(*args)
        grad = torch.is_grad_enabled()
        for x in values(args):
            kind = type(x)
            if kind is not Tensor and kind is not torch.nn.Parameter:
                return op(*args)
            if x.is_neg() or (grad and x.requires_grad):  # (a negative view's memory holds the opposite of its values)
                return op(*args)
        for i in numbers:
            x = args[i]
            if type(x) is not Tensor and x is not None:
                return op(*args)
        if args[0].is_meta:
            return op(*args)
        out = run(*args)
        if mutates:
            written = caches(args)
            if written[0].is_inference() or written[1].is_inference():  # (inference tensors have no version)
                written = tuple(x for x in written if not x.is_inference())
            torch._C._increment_version(written)
        return out

    call.op = op
    return call


def _launch(fn, desc, index: int, op: str) -> None:
    """Call a C entry point on the current stream of device `index`, whichever device is current."""
    if index == _current_device():
        rc = fn(desc, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(desc, _raw_stream(index))
    if rc:
        _lib.check(rc, f"dfb200::{op}")


def _same_device(op: str, first: Tensor, *rest: Tensor | None) -> None:
    require_cuda(first, op)
    index = first.get_device()
    for t in rest:
        if t is not None and t.get_device() != index:
            raise ValueError(f"{op}: all tensors must be on {first.device}, got one on {t.device}")


def _new_like(t: Tensor) -> Tensor:
    """A new contiguous tensor of `t`'s shape and type (a third of the host time of ``torch.empty(t.shape, ...)``)."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _fresh(t: Tensor) -> Tensor:
    """A contiguous copy (``contiguous`` would return a tensor that only starts at an odd offset as it is)."""
    return t.clone(memory_format=torch.contiguous_format)


def _rows(op: str, name: str, t: Tensor) -> tuple[int, int, int]:
    """Strides of the three leading dimensions; the last one must be contiguous."""
    s = t.stride()
    if s[3] != 1 and t.shape[3] > 1:
        raise ValueError(f"{op}: {name} must have its last dimension contiguous")
    return s[:3]


def _steps(t: Tensor) -> tuple[int, int, int]:
    """Strides of the three leading dimensions, 0 for one of size one: no address depends on it, and it may be anything."""
    return tuple(s if n > 1 else 0 for s, n in zip(t.stride()[:3], t.shape))


def _check_cache(op: str, batch: int, heads: int, dim: int, dtype: torch.dtype, key_cache: Tensor, value_cache: Tensor, cache_len: Tensor) -> int:
    shape = key_cache.shape
    if len(shape) != 4 or shape != value_cache.shape:
        raise ValueError(f"{op}: caches must both be (batch, kv_heads, max_seq, head_dim), got {tuple(shape)} and {tuple(value_cache.shape)}")
    if shape[0] != batch or shape[1] != heads or shape[3] != dim:
        raise ValueError(f"{op}: caches {tuple(shape)} do not match batch {batch}, {heads} KV heads, head dim {dim}")
    if key_cache.dtype != dtype or value_cache.dtype != dtype:
        raise ValueError(f"{op}: caches must be {dtype}, got {key_cache.dtype} and {value_cache.dtype}")
    if cache_len.shape != (batch,) or cache_len.dtype != torch.int32 or not cache_len.is_contiguous():
        raise ValueError(f"{op}: cache_len must be a contiguous int32 tensor of {batch} entries, got {tuple(cache_len.shape)} {cache_len.dtype}")
    return shape[2]


def rope_frequencies(
    rotary_dim: int, theta: float, *, stretch: float = 1.0, method: str = "by_parts", trained_len: int = 32768, slow_turns: float = 1.0,
    fast_turns: float = 32.0, device: torch.device | str = "cuda",
) -> tuple[Tensor, float]:  # fmt: skip
    """Inverse frequencies (fp64, ``rotary_dim / 2``) and the factor on cos and sin for ``rotary_qk`` / ``rotary_append``.

    ``stretch`` > 1 scales them for a context that many times ``trained_len``: ``"linear"`` divides every frequency by
    it; ``"base"`` raises ``theta`` so that the slowest frequency is divided by it and the fastest stays; ``"by_parts"``
    divides those that turn less than ``slow_turns`` times over ``trained_len``, keeps those that turn more than ``fast_turns``
    times, goes linearly in between, and scales cos and sin by ``0.1 ln(stretch) + 1``. The ramp is linear in the number of turns.
    Checkpoints whose configuration means a ramp that is linear in the index of the frequency, between two rounded indices, want
    other frequencies (64 dims, theta 1e7, stretch 4: six of 32 differ, by up to 41 %): compute those and pass them.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and at least 2, got {rotary_dim}")
    if not stretch >= 1.0:
        raise ValueError(f"stretch must be at least 1, got {stretch}")
    if method not in ("linear", "base", "by_parts"):
        raise ValueError(f"unknown method {method!r}: linear, base or by_parts")
    if fast_turns <= slow_turns:
        raise ValueError("fast_turns must be above slow_turns")
    if method == "base" and rotary_dim > 2:
        theta = theta * stretch ** (rotary_dim / (rotary_dim - 2))
    f = theta ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    factor = 1.0
    if stretch != 1.0 and method == "linear":
        f = f / stretch
    elif stretch != 1.0 and method == "by_parts":
        keep = ((trained_len * f / (2 * math.pi) - slow_turns) / (fast_turns - slow_turns)).clamp(0, 1)
        f = f * keep + f / stretch * (1 - keep)
        factor = 0.1 * math.log(stretch) + 1.0
    return f.to(device), factor


def _check_rotary(op: str, query: Tensor, key: Tensor, positions: Tensor, inv_freq: Tensor) -> int:
    """Checks what both rotary ops share; the number of dims that turn."""
    qs, ks = query.shape, key.shape
    if len(qs) != 4 or len(ks) != 4:
        raise ValueError(f"{op}: expected query and key (batch, tokens, heads, head_dim), got {tuple(qs)} and {tuple(ks)}")
    if ks[0] != qs[0] or ks[1] != qs[1] or ks[3] != qs[3]:
        raise ValueError(f"{op}: key {tuple(ks)} does not match query {tuple(qs)}")
    if qs[2] < 1 or ks[2] < 1:
        raise ValueError(f"{op}: query and key need at least one head")
    if query.dtype not in _DTYPES or key.dtype != query.dtype:
        raise ValueError(f"{op}: query and key must both be bfloat16, float16 or float32, got {query.dtype} and {key.dtype}")
    if positions.shape != qs[:2] or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{op}: positions must be int32 or int64 {tuple(qs[:2])}, got {tuple(positions.shape)} {positions.dtype}")
    if inv_freq.dim() != 1 or inv_freq.dtype not in (torch.float64, torch.float32) or not inv_freq.is_contiguous():
        raise ValueError(f"{op}: inv_freq must be a contiguous 1-D float64 or float32 tensor, got {tuple(inv_freq.shape)} {inv_freq.dtype}")
    rd = 2 * inv_freq.shape[0]
    if rd < 2 or rd > qs[3] or rd > 512:
        raise ValueError(f"{op}: rotary_dim {rd} must be at least 2 and at most the head dim {qs[3]} and 512")
    if qs[1] > 1 and positions.stride(1) != 1:
        raise ValueError(f"{op}: positions of a sequence must be contiguous")
    return rd


_NO_ROWS = (0, 0, 0)


@_eager
@torch.library.custom_op("dfb200::rotary_qk", mutates_args=())
def rotary_qk(query: Tensor, key: Tensor, positions: Tensor, inv_freq: Tensor, factor: float, interleaved: bool) -> tuple[Tensor, Tensor]:
    """Rotate the leading ``2 * len(inv_freq)`` dims of ``query (batch, tokens, heads, head_dim)`` and ``key`` by
    ``positions (batch, tokens)``: pairs ``(i, i + r/2)``, or ``(2i, 2i + 1)`` when ``interleaved``. Angles are formed in 64
    bits; cos and sin, times ``factor``, in fp32; the result is rounded once. bf16, fp16 or fp32."""
    op = "rotary_qk"
    rd = _check_rotary(op, query, key, positions, inv_freq)
    q_rows, k_rows = _rows(op, "query", query), _rows(op, "key", key)
    _same_device(op, query, key, positions, inv_freq)
    dtype, (batch, tokens, hq, d) = query.dtype, query.shape
    q_out, k_out = _new_like(query), _new_like(key)
    if batch and tokens:
        p = _lib.RotaryDesc()
        _ROTARY.pack_into(
            p, 0, batch, tokens, hq, key.shape[2], d, rd, interleaved, _DTYPES[dtype], query.data_ptr(), key.data_ptr(), 0, *q_rows, *k_rows, *_NO_ROWS,
            positions.data_ptr(), positions.stride(0), positions.dtype == torch.int64, inv_freq.data_ptr(), inv_freq.dtype == torch.float64, factor,
            q_out.data_ptr(), k_out.data_ptr(), 0, 0, *_NO_ROWS, *_NO_ROWS, 0, 0,
        )  # fmt: skip
        _launch(_lib.load().dfb_rotary, p, query.get_device(), op)
    return q_out, k_out


@rotary_qk.op.register_fake
def _(query, key, positions, inv_freq, factor, interleaved):
    return query.new_empty(query.shape), key.new_empty(key.shape)


@_eager
@torch.library.custom_op("dfb200::rotary_append", mutates_args=("key_cache", "value_cache"))
def rotary_append(
    query: Tensor, key: Tensor, value: Tensor, positions: Tensor, inv_freq: Tensor, factor: float, interleaved: bool,
    key_cache: Tensor, value_cache: Tensor, cache_len: Tensor,
) -> Tensor:  # fmt: skip
    """``rotary_qk``, with the rotated keys and the values written into the caches ``(batch, kv_heads, max_seq, head_dim)``
    instead of returned: token ``t`` of sequence ``b`` becomes row ``cache_len[b] + t`` (int32, on the device). Rows below 0 or
    from ``max_seq`` on are not written. The inputs must not overlap the rows that are. Returns the rotated query."""
    op = "rotary_append"
    rd = _check_rotary(op, query, key, positions, inv_freq)
    dtype, (batch, tokens, hq, d) = query.dtype, query.shape
    if value.shape != key.shape or value.dtype != dtype:
        raise ValueError(f"{op}: value {tuple(value.shape)} {value.dtype} must match key {tuple(key.shape)} {key.dtype}")
    max_seq = _check_cache(op, batch, key.shape[2], d, dtype, key_cache, value_cache, cache_len)
    q_rows, k_rows, v_rows = _rows(op, "query", query), _rows(op, "key", key), _rows(op, "value", value)
    kc_rows, vc_rows = _rows(op, "key_cache", key_cache), _rows(op, "value_cache", value_cache)
    if 0 in kc_rows or 0 in vc_rows:
        for t in (key_cache, value_cache):
            if any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
                raise ValueError(f"{op}: the caches are written in place and must not be expanded views")
    _same_device(op, query, key, value, positions, inv_freq, key_cache, value_cache, cache_len)
    if not max_seq:  # a cache without rows
        return rotary_qk.op._init_fn(query, key, positions, inv_freq, factor, interleaved)[0]
    q_out = _new_like(query)
    if batch and tokens:
        p = _lib.RotaryDesc()
        _ROTARY.pack_into(
            p, 0, batch, tokens, hq, key.shape[2], d, rd, interleaved, _DTYPES[dtype], query.data_ptr(), key.data_ptr(), value.data_ptr(),
            *q_rows, *k_rows, *v_rows, positions.data_ptr(), positions.stride(0), positions.dtype == torch.int64,
            inv_freq.data_ptr(), inv_freq.dtype == torch.float64, factor, q_out.data_ptr(), 0,
            key_cache.data_ptr(), value_cache.data_ptr(), *kc_rows, *vc_rows, cache_len.data_ptr(), max_seq,
        )  # fmt: skip
        _launch(_lib.load().dfb_rotary, p, query.get_device(), op)
    return q_out


@rotary_append.op.register_fake
def _(query, key, value, positions, inv_freq, factor, interleaved, key_cache, value_cache, cache_len):
    return query.new_empty(query.shape)


def _check_parents(op: str, parents: Tensor, batch: int, nodes: int) -> int:
    """Elements between two sequences' parents, 0 for one tree for all."""
    if nodes > MAX_TREE_NODES:
        raise ValueError(f"{op}: a tree has at most {MAX_TREE_NODES} nodes, got {nodes}")
    if parents.shape not in ((batch, nodes), (nodes,)) or parents.dtype != torch.int32:
        raise ValueError(f"{op}: parents must be int32 {(batch, nodes)} or {(nodes,)}, got {tuple(parents.shape)} {parents.dtype}")
    if nodes > 1 and parents.stride(-1) != 1:
        raise ValueError(f"{op}: parents of a sequence must be contiguous")
    return parents.stride(0) if parents.dim() == 2 else 0


@_eager
@torch.library.custom_op("dfb200::tree_attention", mutates_args=())
def tree_attention(query: Tensor, key_cache: Tensor, value_cache: Tensor, cache_len: Tensor, parents: Tensor, scale: float) -> Tensor:
    """Attention of a tree of up to 64 drafted tokens over an unexpanded KV cache ``(batch, kv_heads, max_seq, head_dim)``.

    ``query`` is ``(batch, nodes, heads, head_dim)``; node ``i`` of sequence ``b`` holds cache row ``cache_len[b] + i`` and sees
    the rows before ``cache_len[b]``, its ancestors' and its own. ``parents (batch, nodes)``, or ``(nodes,)`` for one tree for
    all: the index of a node's parent, which comes before it; -1 where the parent is the last cached token. Any other
    value marks a row without a node (a padded batch): its output is zero and no node sees it. Rows from ``max_seq`` on do
    not exist: a node that reaches no other row gives zeros too. One node is the decode
    attention, a chain (``parents = [-1, 0, 1, ...]``) causal attention. bf16 or fp16, head dim 32, 64, 128 or 256."""
    op = "tree_attention"
    if query.dim() != 4:
        raise ValueError(f"{op}: expected query (batch, nodes, heads, head_dim), got {tuple(query.shape)}")
    dtype, (batch, nodes, hq, d) = query.dtype, query.shape
    if dtype is not BF16 and dtype is not torch.float16:
        raise ValueError(f"{op}: query must be bfloat16 or float16, got {dtype}")
    hkv = key_cache.shape[1] if key_cache.dim() == 4 else 0
    if hkv and hq % hkv:
        raise ValueError(f"{op}: {hq} query heads do not divide into {hkv} KV heads")
    if d not in (32, 64, 128, 256):
        raise ValueError(f"{op}: head dim {d} is not 32, 64, 128 or 256")
    max_seq = _check_cache(op, batch, hkv, d, dtype, key_cache, value_cache, cache_len)
    if hkv < 1 or hq < 1 or max_seq < 1:
        raise ValueError(f"{op}: need at least one head and one cache row, got {hq} / {hkv} heads, {max_seq} rows")
    tree_stride = _check_parents(op, parents, batch, nodes)
    q_rows, k_rows, v_rows = _rows(op, "query", query), _rows(op, "key_cache", key_cache), _rows(op, "value_cache", value_cache)
    kp, vp = key_cache.data_ptr(), value_cache.data_ptr()
    if (k_rows[0] | k_rows[1] | k_rows[2] | v_rows[0] | v_rows[1] | v_rows[2]) % 8 or (kp | vp) % 16:
        k_rows, v_rows = _steps(key_cache), _steps(value_cache)
        if (k_rows[0] | k_rows[1] | k_rows[2] | v_rows[0] | v_rows[1] | v_rows[2]) % 8 or (kp | vp) % 16:
            raise ValueError(f"{op}: cache rows must start on 16-byte boundaries")
    _same_device(op, query, key_cache, value_cache, cache_len, parents)
    if (q_rows[0] | q_rows[1] | q_rows[2]) % 8 or query.data_ptr() % 16:
        query = _aligned_rows(query)
        q_rows = _steps(query)
    out = _new_like(query)
    if batch == 0 or nodes == 0:
        return out
    nbytes = _scratch_bytes("dfb_tree_attn_scratch_bytes", batch, nodes, hq, hkv, d, max_seq)
    # from the allocator, not kept: calls on two streams, or two captured graphs, never share it
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=query.device) if nbytes else None
    a = _lib.TreeAttnDesc()
    _TREE.pack_into(
        a, 0, batch, nodes, hq, hkv, d, max_seq, dtype is torch.float16, query.data_ptr(), kp, vp, *q_rows, *k_rows, *v_rows,
        cache_len.data_ptr(), parents.data_ptr(), tree_stride, scale, out.data_ptr(), scratch.data_ptr() if nbytes else 0, nbytes,
    )  # fmt: skip
    _launch(_lib.load().dfb_tree_attention, a, query.get_device(), op)
    return out


@tree_attention.op.register_fake
def _(query, key_cache, value_cache, cache_len, parents, scale):
    return query.new_empty(query.shape)


def _aligned_rows(t: Tensor, expanded: bool = True) -> Tensor:
    """`t`, copied if its rows do not start on 16-byte boundaries, or if it may not be `expanded` and is."""
    s = _steps(t)
    return _fresh(t) if (s[0] | s[1] | s[2]) % 8 or t.data_ptr() % 16 or not (expanded or all(x for x, n in zip(s, t.shape) if n > 1)) else t


def _delta_tokens(
    op: str, state: Tensor, query: Tensor, key: Tensor, value: Tensor, g: Tensor, beta: Tensor, lengths: Tensor | None, parents: Tensor | None, l2norm: bool
) -> tuple[Tensor, Tensor | None]:
    if state.dim() != 4 or state.dtype != torch.float32:
        raise ValueError(f"{op}: state must be fp32 (batch, heads, key_dim, value_dim), got {tuple(state.shape)} {state.dtype}")
    batch, hv, dk, dv = state.shape
    shape, per_head = query.shape, (batch, query.shape[1] if query.dim() == 4 else -1, hv)
    if len(shape) != 4 or shape != key.shape or shape[0] != batch or shape[3] != dk:
        raise ValueError(f"{op}: query and key must be (batch, tokens, key_heads, {dk}), got {tuple(shape)} and {tuple(key.shape)}")
    _, tokens, hk, _ = shape
    if hk == 0 or hv == 0 or hv % hk:
        raise ValueError(f"{op}: {hv} value heads do not divide into {hk} key heads")
    if value.shape != (*per_head, dv):
        raise ValueError(f"{op}: value has shape {tuple(value.shape)}, expected {(*per_head, dv)}")
    if g.shape != per_head or not g.is_floating_point():
        raise ValueError(f"{op}: g must be a floating tensor {per_head}, got {tuple(g.shape)} {g.dtype}")
    if beta.shape != per_head or not beta.is_floating_point():
        raise ValueError(f"{op}: beta must be a floating tensor {per_head}, got {tuple(beta.shape)} {beta.dtype}")
    if not query.dtype == key.dtype == value.dtype == BF16:
        raise ValueError(f"{op}: query, key and value must be bfloat16, got {query.dtype}, {key.dtype} and {value.dtype}")
    if dk % 8 or dv % 8 or dk < 8 or dk > 128 or dv < 8:
        raise ValueError(f"{op}: key dim {dk} (a multiple of 8, at most 128) or value dim {dv} (a multiple of 8) unsupported")
    if lengths is not None and (lengths.shape != (batch,) or lengths.dtype != torch.int32 or not lengths.is_contiguous()):
        raise ValueError(f"{op}: lengths must be a contiguous int32 tensor of {batch} entries, got {tuple(lengths.shape)} {lengths.dtype}")
    tree = parents is not None
    tree_stride = _check_parents(op, parents, batch, tokens) if tree else 0
    q_rows, k_rows, v_rows = _rows(op, "query", query), _rows(op, "key", key), _rows(op, "value", value)
    _same_device(op, state, query, key, value, g, beta, lengths, parents)
    qp, kp, vp = query.data_ptr(), key.data_ptr(), value.data_ptr()
    if 0 in v_rows or (q_rows[0] | q_rows[1] | q_rows[2] | k_rows[0] | k_rows[1] | k_rows[2] | v_rows[0] | v_rows[1] | v_rows[2]) % 8 or (qp | kp | vp) % 16:
        query, key, value = _aligned_rows(query), _aligned_rows(key), _aligned_rows(value, expanded=False)
        q_rows, k_rows, v_rows = _steps(query), _steps(key), _steps(value)
        qp, kp, vp = query.data_ptr(), key.data_ptr(), value.data_ptr()
    if not state.is_contiguous():
        state = state.contiguous()
    if g.dtype != torch.float32 or not g.is_contiguous():
        g = g.float().contiguous()
    if beta.dtype != torch.float32 or not beta.is_contiguous():
        beta = beta.float().contiguous()
    out = _new_like(value)
    if batch == 0 or tokens == 0:
        return out, None if tree else state.clone()
    new_state = None if tree else torch.empty_like(state)
    nbytes = _scratch_bytes("dfb_delta_chunk_scratch_bytes", batch, tokens, hk, hv, dk, dv, tree)
    # from the allocator, not kept, as in tree_attention
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=state.device) if nbytes else None
    p = _lib.DeltaChunkDesc()
    _DELTA.pack_into(
        p, 0, batch, tokens, hk, hv, dk, dv, qp, kp, vp, *q_rows, *k_rows, *v_rows,
        g.data_ptr(), beta.data_ptr(), 0 if lengths is None else lengths.data_ptr(), parents.data_ptr() if tree else 0, tree_stride, l2norm,
        state.data_ptr(), 0 if tree else new_state.data_ptr(), out.data_ptr(), scratch.data_ptr() if nbytes else 0, nbytes,
    )  # fmt: skip
    _launch(_lib.load().dfb_delta_chunk, p, state.get_device(), op)
    return out, new_state


@_eager
@torch.library.custom_op("dfb200::delta_rule_chunk", mutates_args=())
def delta_rule_chunk(
    state: Tensor, query: Tensor, key: Tensor, value: Tensor, g: Tensor, beta: Tensor, lengths: Tensor | None, qk_l2norm: bool
) -> tuple[Tensor, Tensor]:
    """The delta rule over several tokens of each sequence, in chunks of 64: ``delta_rule_step`` token after token.

    ``state (batch, heads, key_dim, value_dim)`` fp32; ``query, key (batch, tokens, key_heads, key_dim)`` and ``value (batch,
    tokens, heads, value_dim)`` bf16; ``g`` (log decay) and ``beta (batch, tokens, heads)``. ``qk_l2norm`` normalises q and k
    over the key dim and scales q by ``key_dim ** -0.5``; without it they are used as they are. With ``lengths (batch,)``
    int32, only the first ``lengths[b]`` tokens of a sequence count: later rows give zeros and leave its state as it is
    (a padded batch of prompts, or the accepted tokens of a draft). Returns ``(output bf16, new_state)``. Inputs that
    count are finite: a NaN or an infinity reaches the outputs of its chunk, and so does, with ``qk_l2norm``, a query or key whose
    sum of squares is beyond fp32."""
    return _delta_tokens("delta_rule_chunk", state, query, key, value, g, beta, lengths, None, qk_l2norm)


@delta_rule_chunk.op.register_fake
def _(state, query, key, value, g, beta, lengths, qk_l2norm):
    return value.new_empty(value.shape), state.new_empty(state.shape)


@_eager
@torch.library.custom_op("dfb200::delta_rule_tree", mutates_args=())
def delta_rule_tree(state: Tensor, query: Tensor, key: Tensor, value: Tensor, g: Tensor, beta: Tensor, parents: Tensor, qk_l2norm: bool) -> Tensor:
    """The delta rule over a tree of up to 64 drafted tokens: node ``i`` continues from the state that the path from the root
    to its parent leaves. Arguments as in ``delta_rule_chunk``, ``parents`` as in ``tree_attention``. Returns the nodes' outputs
    (zero for rows without a node); ``state`` stays as it is: once a path is accepted, run its tokens through
    ``delta_rule_chunk``."""
    return _delta_tokens("delta_rule_tree", state, query, key, value, g, beta, None, parents, qk_l2norm)[0]


@delta_rule_tree.op.register_fake
def _(state, query, key, value, g, beta, parents, qk_l2norm):
    return value.new_empty(value.shape)
