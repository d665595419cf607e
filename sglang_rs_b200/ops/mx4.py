"""Matrices in the microscaled four-bit format, products with them, and the router whose experts they are.

The format is MXFP4 of the OCP Microscaling Formats specification: 32 consecutive entries of a row share a scale 2^(s - 127), one
byte s (255: not a number), and an entry is a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6.  17 bits hold four entries, so a step with
few rows reads a quarter of the bytes that bfloat16 weights are, and two operands in it multiply at four times bfloat16's rate.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional

import torch

from ..csrc.build import load_library
from . import (GEMM_MODES, KernelError, ROUTER_SCORING, _check, _need, _need_rows, _ptr, _stream, activation_code, dtype_code)
from .trace import traced

#: entries of a row that share a scale
MX4_BLOCK = 32
#: up to this many rows a product runs on the kernel that has the weights on the M side (csrc/gemm_mx4.cu), above it on pairs of CTAs
MX4_FEW_ROWS = 64
#: experts' products run on pairs of CTAs where a step has more choices per expert than this
MX4_FEW_CHOICES = 16


def _tiles(n: int) -> int:
    return -(-n // 128)


@dataclass(frozen=True)
class Mx4:
    """A matrix [rows, width] (or several [matrices, rows, width]) in four bits, laid out for the kernels (csrc/mx4.cuh).

    ``codes`` uint8 [..., rows, 64 * ceil(width / 128)], two entries to a byte, the first in the low half, zero behind a row's
    last; ``scales`` uint8 [..., ceil(rows / 128), ceil(width / 128), 512], the scales of 128 rows x 128 entries side by side.
    Made by :func:`quantize_mx4` or :func:`mx4_from_rows`."""
    codes: torch.Tensor
    scales: torch.Tensor
    width: int

    @property
    def rows(self) -> int:
        return self.codes.shape[-2]

    @property
    def matrices(self) -> Optional[int]:
        """How many matrices there are; None for one that is not in a stack."""
        return self.codes.shape[0] if self.codes.dim() == 3 else None

    @property
    def shape(self) -> tuple:
        return (*self.codes.shape[:-1], self.width)

    @property
    def device(self) -> torch.device:
        return self.codes.device


def _here(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """The kernels run on the current device's stream: what they read and write has to be there."""
    here = torch.cuda.current_device()
    for tensor in tensors:
        if tensor is not None and tensor.device.index != here:
            raise KernelError(f"{what}: a tensor lies on {tensor.device}, the current device is cuda:{here}")


def _need_mx4(q: Mx4, name: str, stacked: Optional[bool]) -> None:
    """``q``'s tensors as the kernels take them (``stacked``: several matrices, one, or either)."""
    if not isinstance(q, Mx4):
        raise KernelError(f"{name} must be an Mx4, found {type(q).__name__}")
    _need(q.codes, f"{name}.codes", torch.uint8); _need(q.scales, f"{name}.scales", torch.uint8)
    if stacked is not None and (q.codes.dim() == 3) != stacked:
        raise KernelError(f"{name} must be {'a stack of matrices' if stacked else 'one matrix'}, found {q.shape}")
    lead = q.codes.shape[:-2]
    if (q.codes.dim() not in (2, 3) or q.width <= 0 or q.codes.shape[-1] != 64 * _tiles(q.width)
            or q.scales.shape != (*lead, _tiles(q.rows), _tiles(q.width), 512) or q.codes.data_ptr() % 32 or q.scales.data_ptr() % 16):
        raise KernelError(f"{name}: codes {tuple(q.codes.shape)} and scales {tuple(q.scales.shape)} do not hold rows of {q.width}")


def mx4_from_rows(codes: torch.Tensor, scales: torch.Tensor, width: Optional[int] = None) -> Mx4:
    """A matrix that a checkpoint holds row by row: ``codes`` uint8 [..., rows, ceil(width / 2)], two entries to a byte, the
    first in the low half, and ``scales`` uint8 [..., rows, ceil(width / 32)] (``width``: 2 * bytes of a row unless given).
    Laid out once, at load, by copies on the tensors' device; codes behind the last entry of a row count as zero."""
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.dim() not in (2, 3) or scales.dim() != codes.dim():
        raise KernelError("mx4_from_rows: codes and scales must be uint8 [rows, bytes] or [matrices, rows, bytes]")
    if not codes.is_cuda or scales.device != codes.device:
        raise KernelError("mx4_from_rows: codes and scales must be CUDA tensors of one device; this engine has no host path")
    width = 2 * codes.shape[-1] if width is None else int(width)
    *lead, rows, held = codes.shape
    blocks, k_tiles, row_tiles = -(-width // MX4_BLOCK), _tiles(width), _tiles(rows)
    if width <= 0 or held != -(-width // 2) or tuple(scales.shape) != (*lead, rows, blocks):
        raise KernelError(f"mx4_from_rows: codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not hold rows of {width}")
    laid = torch.zeros((*lead, rows, 64 * k_tiles), dtype=torch.uint8, device=codes.device)
    laid[..., :held] = codes
    if width % 2:
        laid[..., held - 1] &= 15
    padded = torch.full((*lead, row_tiles * 128, k_tiles * 4), 127, dtype=torch.uint8, device=codes.device)
    padded[..., :rows, :blocks] = scales
    # [row tile, quarter, row of it, column tile, block] -> [row tile, column tile, row of a quarter, quarter, block]
    tiles = padded.view(*lead, row_tiles, 4, 32, k_tiles, 4)
    at = len(lead)
    order = (*range(at), at, at + 3, at + 2, at + 1, at + 4)
    return Mx4(laid, tiles.permute(order).contiguous().view(*lead, row_tiles, k_tiles, 512), width)


@traced("quantize")
def quantize_mx4(x: torch.Tensor) -> Mx4:
    """``x`` [rows, width] (dense rows, any pitch) or [matrices, rows, width] (contiguous), float32 or bfloat16, in four bits.

    Per block of 32 entries the scale is 2^(floor(log2(largest magnitude)) - 2), at least 2^-127; entries go to the nearest
    value of the format, ties to the even mantissa, magnitudes above 6 scales to 6 (the specification's conversion).  A block
    with an infinity or something that is not a number becomes a block of such."""
    if x.dim() == 3:
        _need(x, "x")
    else:
        _need_rows(x, "x")
    code = dtype_code(x.dtype)
    _here("quantize_mx4", x)
    *lead, rows, width = x.shape
    if width == 0:
        raise KernelError("quantize_mx4: rows without entries")
    q = Mx4(torch.empty((*lead, rows, 64 * _tiles(width)), dtype=torch.uint8, device=x.device),
            torch.empty((*lead, _tiles(rows), _tiles(width), 512), dtype=torch.uint8, device=x.device), width)
    if rows and (not lead or lead[0]):
        lib = load_library("mx4")
        _check(lib, lib.srb_mx4_quantize(_ptr(x), ctypes.c_longlong(x.stride(-2)), ctypes.c_longlong(x.stride(0) if lead else 0),
                                         lead[0] if lead else 1, rows, width, _ptr(q.codes), _ptr(q.scales), code, _stream()))
    return q


@traced("quantize")
def dequantize_mx4(q: Mx4, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that ``q`` stands for, in bfloat16 (exact: a code times a power of two) or float32."""
    _need_mx4(q, "q", None)
    code = dtype_code(dtype)
    _here("dequantize_mx4", q.codes, q.scales)
    out = torch.empty(q.shape, dtype=dtype, device=q.device)
    if out.numel():
        lib = load_library("mx4")
        _check(lib, lib.srb_mx4_dequantize(_ptr(q.codes), _ptr(q.scales), q.matrices or 1, q.rows, q.width, _ptr(out), code, _stream()))
    return out


def _parts(x: torch.Tensor):
    """bfloat16 rows as eight rows of four bits each, and their scales (csrc/mx4.cuh)."""
    rows, width = x.shape
    codes = torch.empty((8 * rows, 64 * _tiles(width)), dtype=torch.uint8, device=x.device)
    scales = torch.empty((_tiles(8 * rows), _tiles(width), 512), dtype=torch.uint8, device=x.device)
    lib = load_library("mx4")
    _check(lib, lib.srb_mx4_parts(_ptr(x), ctypes.c_longlong(x.stride(0)), rows, width, _ptr(codes), _ptr(scales), _stream()))
    return codes, scales


def _split(x: torch.Tensor):
    """bfloat16 rows as the two eight-bit parts (and their scales) that multiply four-bit entries (csrc/mx4.cuh)."""
    rows, width = x.shape
    parts = torch.empty((2, rows, 128 * _tiles(width)), dtype=torch.uint8, device=x.device)
    scales = torch.empty((2, _tiles(rows), _tiles(width), 512), dtype=torch.uint8, device=x.device)
    lib = load_library("mx4")
    _check(lib, lib.srb_mx4_split(_ptr(x), ctypes.c_longlong(x.stride(0)), rows, width, _ptr(parts), _ptr(scales), _stream()))
    return parts, scales


@traced("gemm")
def linear_mx4(x, weight: Mx4, error_word: torch.Tensor, *, bias: Optional[torch.Tensor] = None,
               out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """y = x @ weight^T (+ bias), sums in 32 bits; bfloat16, or float32 with ``out_dtype``.

    ``x``: bfloat16 [rows, width] (dense rows, any pitch), or an :class:`Mx4` of rows: both operands are then multiplied in four
    bits.  ``weight``: one matrix [features, width]; ``bias`` float32 [features]."""
    four = isinstance(x, Mx4)
    if four:
        _need_mx4(x, "x", False)
        rows, width = x.shape
    else:
        if x.dtype == torch.float32:
            raise KernelError("linear_mx4: float32 rows are not taken; multiply dequantize_mx4(weight, torch.float32) by linear")
        _need_rows(x, "x", torch.bfloat16)
        rows, width = x.shape
    _need_mx4(weight, "weight", False)
    _need(error_word, "error_word", torch.int32)
    out_dtype = torch.bfloat16 if out_dtype is None else out_dtype
    dtype_code(out_dtype)
    if weight.width != width:
        raise KernelError(f"linear_mx4: rows of {width} and a weight {weight.shape} do not fit")
    if bias is not None:
        _need(bias, "bias", torch.float32)
        if bias.shape != (weight.rows,):
            raise KernelError("linear_mx4: one bias per feature is needed")
    _here("linear_mx4", x.codes if four else x, weight.codes, weight.scales, bias, error_word)
    many = rows > MX4_FEW_ROWS
    # the kernel for many rows stores rows that start on 16-byte borders
    pitch = -(-weight.rows // 8) * 8 if many else weight.rows
    out = torch.empty((rows, pitch), dtype=out_dtype, device=weight.device)
    if out.numel():
        lib = load_library("gemm_mx4_pair" if many else "gemm_mx4")
        product = lib.srb_mx4_linear_pair if many else lib.srb_mx4_linear
        held, scales = (x.codes, x.scales) if four else _split(x) if many else _parts(x)
        _check(lib, product(_ptr(held), _ptr(scales), int(four if many else not four), _ptr(weight.codes), _ptr(weight.scales), _ptr(bias), _ptr(out),
                            ctypes.c_longlong(out.stride(0)), rows, weight.rows, width, int(out_dtype == torch.float32),
                            _ptr(error_word), _stream()))
    return out if pitch == weight.rows else out[:, :weight.rows]


@traced("routed_experts")
def choose_experts(logits: torch.Tensor, top: int, renormalize: bool = False, *, scoring: str = "softmax",
                   choice_bias: Optional[torch.Tensor] = None, groups: int = 1, top_groups: int = 1, group_best: int = 1,
                   weight_scale: float = 1.0, norm_eps: float = 0.0):
    """A router's choice from its logits, the experts in groups: (chosen experts int32 [rows, top], weights float32 [rows, top]).

    ``logits`` float32 [rows, experts] (dense rows, any pitch).  Scores are a softmax over all experts or (``scoring`` ``sigmoid``)
    the sigmoid of each logit; ``choice_bias`` (float32 [experts]) is added to them for the choice alone.  The experts are
    ``groups`` runs of equal length; a group's score is the sum of its ``group_best`` (1 or 2) largest biased scores, and experts
    are chosen from the ``top_groups`` groups with the largest ones.  The ``top`` largest biased scores are chosen, largest first,
    ties to the lower index.  The weights are the chosen scores, with ``renormalize`` divided by (their sum + ``norm_eps``), times
    ``weight_scale``.  The choice is that of 64-bit scores: rows whose 32-bit scores lie too close are chosen again."""
    _need_rows(logits, "logits", torch.float32)
    rows, experts = logits.shape
    if scoring not in ROUTER_SCORING:
        raise KernelError(f"choose_experts: unknown scoring {scoring!r}; the kernel has {sorted(ROUTER_SCORING)}")
    if choice_bias is not None:
        _need(choice_bias, "choice_bias", torch.float32)
        if choice_bias.shape != (experts,):
            raise KernelError("choose_experts: one choice bias per expert is needed")
    if top < 0 or top > 2**31 - 1 or rows * max(top, 1) >= 2**31:
        raise KernelError(f"choose_experts: {rows} rows of {top} choices")
    _here("choose_experts", logits, choice_bias)
    chosen = torch.empty((rows, top), dtype=torch.int32, device=logits.device)
    weights = torch.empty((rows, top), dtype=torch.float32, device=logits.device)
    lib = load_library("route_groups")
    _check(lib, lib.srb_route_groups(_ptr(logits), ctypes.c_longlong(logits.stride(0)), rows, experts, _ptr(choice_bias), int(top), int(groups),
                                     int(top_groups), int(group_best), ROUTER_SCORING[scoring], int(renormalize), ctypes.c_float(weight_scale),
                                     ctypes.c_float(norm_eps), _ptr(chosen), _ptr(weights), _stream()))
    return chosen, weights


@traced("routed_experts")
def chosen_experts_mx4(h: torch.Tensor, chosen: torch.Tensor, weights: torch.Tensor, w_gate_up: Mx4, w_down: Mx4, activation: str,
                       error_word: torch.Tensor, *, gated: bool = True, activation_param: float = 0.0) -> torch.Tensor:
    """sum over a row's choices of weight * expert(h), bfloat16 [rows, width], the experts' matrices in four bits.

    ``h`` bfloat16 [rows, width]; ``chosen`` int32 and ``weights`` float32 [rows, top] (of :func:`choose_experts` or
    :func:`~sglang_rs_b200.ops.route`); a choice outside the experts adds nothing, one made twice counts twice.
    ``w_gate_up``: a stack [experts, 2 * inner, width], an expert's gate rows over its up rows (``gated`` False: the up matrices
    alone [experts, inner, width], an expert being W_down act(W_up h)); ``w_down`` a stack [experts, width, inner].  Sums are
    taken in 32 bits; act(gate) * up is rounded once between the two products.  Nothing is decided on the host."""
    _need(h, "h", torch.bfloat16); _need(chosen, "chosen", torch.int32); _need(weights, "weights", torch.float32)
    _need_mx4(w_gate_up, "w_gate_up", True); _need_mx4(w_down, "w_down", True); _need(error_word, "error_word", torch.int32)
    act_code = activation_code(activation, parametric=True)
    if h.dim() != 2 or chosen.dim() != 2 or chosen.shape[0] != h.shape[0] or weights.shape != chosen.shape:
        raise KernelError("chosen_experts_mx4: h must be [rows, width], chosen and weights [rows, top]")
    (rows, width), top = h.shape, chosen.shape[1]
    experts, inner = w_down.matrices, w_down.width
    if (w_gate_up.shape != (experts, (2 if gated else 1) * inner, width) or w_down.rows != width or experts < 1 or experts > 1024):
        raise KernelError(f"chosen_experts_mx4: h {tuple(h.shape)}, w_gate_up {w_gate_up.shape} and w_down {w_down.shape} do not fit "
                          "(at most 1024 experts)")
    if rows * max(top, 1) >= 2**31:
        raise KernelError(f"chosen_experts_mx4: {rows} rows of {top} choices")
    _here("chosen_experts_mx4", h, chosen, weights, w_gate_up.codes, w_gate_up.scales, w_down.codes, w_down.scales, error_word)
    if rows == 0 or top == 0:
        return torch.zeros((rows, width), dtype=torch.bfloat16, device=h.device)
    out = torch.empty((rows, width), dtype=torch.bfloat16, device=h.device)
    device, entries, stream = h.device, rows * top, _stream()
    # (the pairs' result rows start on 16-byte borders)
    many = entries > MX4_FEW_CHOICES * experts and width % 4 == 0
    tile = 256 if many else 8
    moe, lib, split = load_library("moe"), load_library("gemm_mx4"), load_library("mx4")
    plan = torch.empty(moe.srb_moe_plan_ints_of(rows, top, experts, tile), dtype=torch.int32, device=device)
    slot_row = torch.empty(entries, dtype=torch.int32, device=device)
    entry_slot = torch.empty(entries, dtype=torch.int32, device=device)
    y = torch.empty((entries, width), dtype=torch.float32, device=device)
    _check(moe, moe.srb_moe_plan_of(_ptr(chosen), rows, top, experts, tile, _ptr(plan), _ptr(slot_row), _ptr(entry_slot), None, None,
                                    _ptr(error_word), stream))
    # a tile has a slot at least
    tiles = min(entries, moe.srb_moe_max_tiles_of(rows, top, experts, tile))

    def held(size):
        """Room for every tile's rows of ``size`` entries, and for their scales: two eight-bit parts of 256 rows, or eight four-bit ones of 8."""
        if many:
            return (torch.empty((2, 256 * tiles, 128 * _tiles(size)), dtype=torch.uint8, device=device),
                    torch.empty((2, 2 * tiles, _tiles(size), 512), dtype=torch.uint8, device=device))
        return (torch.empty((64 * tiles, 64 * _tiles(size)), dtype=torch.uint8, device=device),
                torch.empty((_tiles(64 * tiles), _tiles(size), 512), dtype=torch.uint8, device=device))
    (parts, scales), (act, act_scales) = held(width), held(inner)
    up_scales, scale_rows, up_row = w_gate_up.scales, w_gate_up.rows, inner
    if gated and (many or inner % 128):
        # a tile's gate and up rows side by side: 96 of each for the pairs; otherwise all of them, the up rows on the border of a tile
        group = 96 if many else 128 * _tiles(inner)
        group_room, groups = (256, -(-128 * _tiles(inner) // 96)) if many else (2 * group, 1)
        scale_rows, up_row = groups * group_room, group
        up_scales = torch.empty((experts, scale_rows // 128, _tiles(width), 512), dtype=torch.uint8, device=device)
        _check(split, split.srb_mx4_gated_scales(_ptr(w_gate_up.scales), experts, inner, width, group, group_room, groups, _ptr(plan),
                                                 _ptr(up_scales), stream))
    # (last ahead of the products: those for few rows read what is older than it before it is done)
    in_slots = split.srb_mx4_split_slots if many else split.srb_mx4_parts_slots
    _check(split, in_slots(_ptr(h), width, _ptr(plan), _ptr(slot_row), experts, tiles, _ptr(parts), _ptr(scales), stream))
    mode, param = GEMM_MODES["gated" if gated else "act"], ctypes.c_float(activation_param)
    if many:
        pair = load_library("gemm_mx4_pair")
        _check(pair, pair.srb_mx4_experts_pair(_ptr(parts), _ptr(scales), _ptr(w_gate_up.codes), _ptr(up_scales), _ptr(act),
                                               _ptr(act_scales), _ptr(plan), tiles, entries, experts, inner, width, mode, act_code, param,
                                               _ptr(error_word), stream))
        _check(pair, pair.srb_mx4_experts_pair(_ptr(act), _ptr(act_scales), _ptr(w_down.codes), _ptr(w_down.scales), _ptr(y), None, _ptr(plan),
                                               tiles, entries, experts, width, inner, GEMM_MODES["f32"], 0, param, _ptr(error_word), stream))
    else:
        _check(lib, lib.srb_mx4_experts(_ptr(parts), _ptr(scales), _ptr(w_gate_up.codes), _ptr(up_scales), scale_rows, up_row if gated else 0,
                                        _ptr(act), _ptr(act_scales), _ptr(plan), tiles, experts, inner, width, mode, act_code, param,
                                        _ptr(error_word), stream))
        _check(lib, lib.srb_mx4_experts(_ptr(act), _ptr(act_scales), _ptr(w_down.codes), _ptr(w_down.scales), width, 0, _ptr(y), None,
                                        _ptr(plan), tiles, experts, width, inner, GEMM_MODES["f32"], 0, param, _ptr(error_word), stream))
    _check(lib, lib.srb_mx4_combine(_ptr(y), _ptr(entry_slot), _ptr(weights), rows, top, width, _ptr(out), stream))
    return out
