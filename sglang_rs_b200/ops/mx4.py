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
from .. import ops as _ops
from . import KernelError, ROUTER_SCORING, _check, _need, _need_rows, activation_code, dtype_code
from .trace import traced

#: entries of a row that share a scale
MX4_BLOCK = 32
#: the largest size of a matrix: the kernels count rows and entries in 32 bits, in whole tiles
MX4_MOST = 2**31 - 2**16
#: Up to this many rows a product runs on the kernel that has the weights on the M side (csrc/gemm_mx4.cu), above it on pairs of CTAs (us, that kernel and
#: pairs, 4,096 x 24,576: 64 rows 30 and 37, 96 rows 39 and 37; both operands in four bits, without the quantising of the rows, 64 rows 15.7 and 16.0, 96 rows
#: 19 and 17, 4,096 x 4,096: 64 rows 8.3 and 8.6, 96 rows 9.8 and 8.7) ...
MX4_FEW_ROWS = 64
#: ... and rows of bfloat16 up to this many there too, where the pairs' tiles would leave half of the pairs idle (4,096 x 4,096: 128 rows 14 and
#: 20, 192 rows 20 and 21, 256 rows 22 and 21; 12,288 x 4,096: 192 rows 48 and 49; 2,048 x 2,048: 192 rows 9 and 13)
MX4_FEW_ROWS_OF_SMALL = 192
#: The experts' products run on the kernel for few rows while choices per expert * bytes of an expert's codes stay below this.  That kernel reads an expert's
#: matrices, from L2, for every 8 of its rows, and holds what is between the products more finely; it is left where it is clearly the slower one (us, it
#: and the best of the others: 64 experts of 2,048 x 1,408 with 24 choices each 126 and 136, 32 156 and 144, 40 186 and 157; 32 of 1,024 x 1,024 with 64
#: 80 and 76, 96 107 and 79; 8 of 1,024 x 512 with 96 30 and 32, 144 36 and 35, 192 43 and 34)
MX4_FEW_BYTES = 136 << 20
#: above it, from this many experts on, they are divided on the device, those with up to MX4_FEW_SLOTS rows going to the kernel for few rows all the same: a tile
#: of 256 rows costs the pairs as much with one row.  That pays where some experts have many more rows than others, as routers choose them, and
#: costs three launches where all have as many (us, all on pairs and divided, from a graph: 64 of 2,048 x 1,408 with 192 choices each 340 and 319,
#: evenly 271 and 281; 64 of 1,024 x 1,024 with 187 165 and 165, evenly 144 and 155; 128 of 2,048 x 768 with 96 281 and 251, evenly 303 and 321; 256 of
#: 1,024 x 512 with 256 483 and 458, evenly 473 and 497).  Fewer experts do not gain: 48 of 1,024 x 1,024 with 192 131 and 140; 32 of 1,024 x 1,024
#: with 96 79 and 86.  How even the load is, only the device knows
MX4_DIVIDE_EXPERTS = 64
MX4_FEW_SLOTS = 48

_P, _I, _L, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float
_LINEAR = (_P, _L, _P, _P, _P, _P, _P, _L, _I, _I, _I, _I, _P, _P, _P)
_EXPERTS = (_P,) * 8 + (_I,) * 7 + (_F, _P, _P, _P)
_EXPERTS_PAIR = (_P,) * 8 + (_I,) * 9 + (_F, _P, _P, _P)
#: entry points by library and their arguments, declared once: a small call costs as long on the host as on the device
_SIGNATURES = {
    "mx4": {"srb_mx4_quantize": (_P, _L, _L, _I, _I, _I, _P, _P, _I, _P), "srb_mx4_dequantize": (_P, _P, _I, _I, _I, _P, _I, _P)},
    "gemm_mx4": {"srb_mx4_linear": _LINEAR, "srb_mx4_experts": _EXPERTS, "srb_mx4_linear_scratch": (_I,) * 2,
                 "srb_mx4_experts_scratch": (_I,) * 5, "srb_mx4_experts_tile": (), "srb_mx4_combine": (_P, _P, _P, _I, _I, _I, _P, _P)},
    "gemm_mx4_pair": {"srb_mx4_linear_pair": _LINEAR, "srb_mx4_experts_pair": _EXPERTS_PAIR, "srb_mx4_linear_pair_scratch": (_I,) * 2,
                      "srb_mx4_experts_pair_scratch": (_I,) * 5, "srb_mx4_experts_pair_tile": (),
                      "srb_mx4_divide_plan": (_P, _I, _I, _I, _I, _I, _P, _P, _P, _P)},
    "route_groups": {"srb_route_groups": (_P, _L, _I, _I, _P, _I, _I, _I, _I, _I, _I, _F, _F, _P, _P, _P)},
}
_declared: dict = {}


def _library(name: str):
    library = _declared.get(name)
    if library is None:
        library = load_library(name)
        for function, arguments in _SIGNATURES[name].items():
            getattr(library, function).argtypes = arguments
            if function.endswith("_scratch"):
                getattr(library, function).restype = _L
        _declared[name] = library
    return library


def _stream(device: int):
    """The handle of torch's current stream there (of the scope's, inside one), without the object that torch makes around it: that
    costs as much as a launch."""
    scoped = _ops._scoped_stream
    return scoped if scoped is not None else torch._C._cuda_getCurrentRawStream(device)


def _few_rows(rows: int, features: int, four: bool) -> bool:
    """True if a product goes to the kernel for few rows."""
    return rows <= MX4_FEW_ROWS or (not four and rows <= MX4_FEW_ROWS_OF_SMALL and -(-features // 192) * 4 <= _ops.sm_count())


def _tiles(n: int) -> int:
    return -(-n // 128)


def _room(n: int) -> int:
    """Bytes of a piece of scratch memory: pieces start on 256-byte borders."""
    return (n + 255) & ~255


@dataclass(frozen=True, eq=False)
class Mx4:
    """A matrix [rows, width] (or several [matrices, rows, width]) in four bits, laid out for the kernels (csrc/mx4.cuh).

    ``codes`` uint8 [..., rows, 64 * ceil(width / 128)], two entries to a byte, the first in the low half, zero behind a row's
    last; ``scales`` uint8 [..., ceil(rows / 128), ceil(width / 128), 512], the scales of 128 rows x 128 entries side by side.
    Made by :func:`quantize_mx4` or :func:`mx4_from_rows`."""
    codes: torch.Tensor
    scales: torch.Tensor
    width: int

    @classmethod
    def _made(cls, codes: torch.Tensor, scales: torch.Tensor, width: int) -> "Mx4":
        """One whose tensors were allocated here, without looking at them again."""
        q = object.__new__(cls)
        q.__dict__.update(codes=codes, scales=scales, width=width)
        return q

    def __post_init__(self):
        codes, scales = self.codes, self.scales
        if (not isinstance(codes, torch.Tensor) or not isinstance(scales, torch.Tensor) or codes.dtype != torch.uint8 or scales.dtype != torch.uint8
                or codes.dim() not in (2, 3) or self.width <= 0 or codes.shape[-1] != 64 * _tiles(self.width) or scales.device != codes.device
                or scales.shape != (*codes.shape[:-2], _tiles(codes.shape[-2]), _tiles(self.width), 512)
                or not codes.is_contiguous() or not scales.is_contiguous() or codes.data_ptr() % 32 or scales.data_ptr() % 16):
            raise KernelError(f"Mx4: codes and scales do not hold rows of {self.width}: contiguous uint8 [..., rows, 64 * ceil(width / 128)] on a "
                              "32-byte border and [..., ceil(rows / 128), ceil(width / 128), 512] on a 16-byte border are needed")

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


def _here(what: str, *tensors: Optional[torch.Tensor]) -> int:
    """The current device.  The kernels run on its stream: what they read and write has to be there."""
    here = torch.cuda.current_device()
    for tensor in tensors:
        if tensor is not None and tensor.get_device() != here:
            raise KernelError(f"{what}: a tensor lies on {tensor.device}, the current device is cuda:{here}")
    return here


def _need_mx4(q: Mx4, name: str, stacked: Optional[bool]) -> None:
    """``q`` as the kernels take it (``stacked``: several matrices, one, or either)."""
    if not isinstance(q, Mx4):
        raise KernelError(f"{name} must be an Mx4, found {type(q).__name__}")
    if not q.codes.is_cuda:
        raise KernelError(f"{name} must be on a CUDA device; this engine has no host path")
    if stacked is not None and (q.codes.dim() == 3) != stacked:
        raise KernelError(f"{name} must be {'a stack of matrices' if stacked else 'one matrix'}, found {q.shape}")


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
    stacked = x.dim() == 3
    if stacked:
        _need(x, "x")
    else:
        _need_rows(x, "x")
    code = dtype_code(x.dtype)
    here = _here("quantize_mx4", x)
    matrices, (rows, width) = x.shape[0] if stacked else 1, x.shape[1:] if stacked else x.shape
    if width == 0:
        raise KernelError("quantize_mx4: rows without entries")
    if rows > MX4_MOST or width > MX4_MOST or matrices > MX4_MOST:
        raise KernelError(f"quantize_mx4: sizes {tuple(x.shape)} are too large")
    k_tiles, lead = -(-width // 128), (matrices,) if stacked else ()
    codes = x.new_empty((*lead, rows, 64 * k_tiles), dtype=torch.uint8)
    scales = x.new_empty((*lead, -(-rows // 128), k_tiles, 512), dtype=torch.uint8)
    if matrices and rows:
        lib = _library("mx4")
        _check(lib, lib.srb_mx4_quantize(x.data_ptr(), x.stride(-2), x.stride(0) if stacked else 0, matrices, rows, width, codes.data_ptr(),
                                         scales.data_ptr(), code, _stream(here)))
    return Mx4._made(codes, scales, width)


@traced("quantize")
def dequantize_mx4(q: Mx4, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that ``q`` stands for, in bfloat16 or float32: exact in both, a code times a power of two, but for those of 2^128 and above, which
    scales of 253 and 254 (:func:`quantize_mx4` makes none) can have and which become infinite."""
    _need_mx4(q, "q", None)
    code = dtype_code(dtype)
    codes, width = q.codes, q.width
    here = _here("dequantize_mx4", codes, q.scales)
    lead = codes.shape[:-1]
    rows, matrices = lead[-1], lead[0] if len(lead) == 2 else 1
    if rows > MX4_MOST or width > MX4_MOST or matrices > MX4_MOST:
        raise KernelError(f"dequantize_mx4: sizes {q.shape} are too large")
    out = codes.new_empty((*lead, width), dtype=dtype)
    if rows and matrices:
        lib = _library("mx4")
        _check(lib, lib.srb_mx4_dequantize(codes.data_ptr(), q.scales.data_ptr(), matrices, rows, width, out.data_ptr(), code, _stream(here)))
    return out


@traced("gemm")
def linear_mx4(x, weight: Mx4, error_word: torch.Tensor, *, bias: Optional[torch.Tensor] = None,
               out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """y = x @ weight^T (+ bias), sums in 32 bits; bfloat16, or float32 with ``out_dtype``.

    ``x``: bfloat16 [rows, width] (dense rows, any pitch), or an :class:`Mx4` of rows: both operands are then multiplied in four
    bits.  ``weight``: one matrix [features, width]; ``bias`` float32 [features].  The result is contiguous.

    Rows of bfloat16 go in as parts that add up to them: every entry exactly where it is at least 2^-14 of the largest of its 32
    neighbours, otherwise to 2^-22 of that one; a few rows, up to 192, also to no less than 2^-129.  A row with an infinity or something
    that is not a number gives rows that are not numbers.  The bits of a row's result do not depend on what the other rows hold, nor on
    timing; they do on how many rows there are, by which the kernel, the parts and the order of the sums are chosen."""
    four = isinstance(x, Mx4)
    if four:
        _need_mx4(x, "x", False)
        held, rows, width = x.codes, x.codes.shape[0], x.width
    else:
        if x.dtype == torch.float32:
            raise KernelError("linear_mx4: float32 rows are not taken; multiply dequantize_mx4(weight, torch.float32) by linear")
        _need_rows(x, "x", torch.bfloat16)
        held, (rows, width) = x, x.shape
    _need_mx4(weight, "weight", False)
    codes = weight.codes
    features = codes.shape[0]
    _need(error_word, "error_word", torch.int32)
    out_dtype = torch.bfloat16 if out_dtype is None else out_dtype
    dtype_code(out_dtype)
    if rows > MX4_MOST or features > MX4_MOST or width > MX4_MOST:
        raise KernelError(f"linear_mx4: {rows} rows of {width} and a weight {weight.shape} are too large")
    if weight.width != width:
        raise KernelError(f"linear_mx4: rows of {width} and a weight {weight.shape} do not fit")
    if bias is not None:
        _need(bias, "bias", torch.float32)
        if bias.shape != (features,):
            raise KernelError("linear_mx4: one bias per feature is needed")
    here = _here("linear_mx4", held, codes, weight.scales, bias, error_word)
    many = not _few_rows(rows, features, four)
    out = codes.new_empty((rows, features), dtype=out_dtype)
    if rows and features:
        lib = _library("gemm_mx4_pair" if many else "gemm_mx4")
        product, needed = (lib.srb_mx4_linear_pair, lib.srb_mx4_linear_pair_scratch) if many else (lib.srb_mx4_linear, lib.srb_mx4_linear_scratch)
        needed = 0 if four else needed(rows, width)
        scratch = codes.new_empty(needed) if needed else None
        _check(lib, product(held.data_ptr(), held.stride(0), x.scales.data_ptr() if four else None, codes.data_ptr(), weight.scales.data_ptr(),
                            None if bias is None else bias.data_ptr(), out.data_ptr(), features, rows, features, width,
                            out_dtype == torch.float32, scratch.data_ptr() if needed else None, error_word.data_ptr(), _stream(here)), 2 if needed else 1)
    return out


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
    # (what follows counts in 32 bits; the kernel has its own limits below these)
    if not 0 < top <= experts or rows * top >= 2**31 or max(rows, experts) > MX4_MOST:
        raise KernelError(f"choose_experts: {rows} rows of {top} choices of {experts} experts")
    if not (0 < top_groups <= groups <= experts) or group_best not in (1, 2):
        raise KernelError(f"choose_experts: {experts} experts in {groups} groups, {top_groups} of them open by their {group_best} best")
    here = _here("choose_experts", logits, choice_bias)
    chosen, weights = logits.new_empty((rows, top), dtype=torch.int32), logits.new_empty((rows, top))
    lib = _library("route_groups")
    _check(lib, lib.srb_route_groups(logits.data_ptr(), logits.stride(0), rows, experts, None if choice_bias is None else choice_bias.data_ptr(), top,
                                     groups, top_groups, group_best, ROUTER_SCORING[scoring], renormalize, weight_scale, norm_eps, chosen.data_ptr(),
                                     weights.data_ptr(), _stream(here)))
    return chosen, weights


@traced("routed_experts")
def chosen_experts_mx4(h: torch.Tensor, chosen: torch.Tensor, weights: torch.Tensor, w_gate_up: Mx4, w_down: Mx4, activation: str,
                       error_word: torch.Tensor, *, gated: bool = True, activation_param: float = 0.0) -> torch.Tensor:
    """sum over a row's choices of weight * expert(h), bfloat16 [rows, width], the experts' matrices in four bits.

    ``h`` bfloat16 [rows, width]; ``chosen`` int32 and ``weights`` float32 [rows, top] (of :func:`choose_experts` or
    :func:`~sglang_rs_b200.ops.route`); a choice outside the experts adds nothing, one made twice counts twice.
    ``w_gate_up``: a stack [experts, 2 * inner, width], an expert's gate rows over its up rows (``gated`` False: the up matrices
    alone [experts, inner, width], an expert being W_down act(W_up h)); ``w_down`` a stack [experts, width, inner].  Sums are
    taken in 32 bits; act(gate) * up is rounded once between the two products: where an expert's rows go through the kernel for many, to
    a relative 2^-9 (two parts of four significant bits; bfloat16 has 2^-8) or 2^-22 of the largest of 32 neighbours, and through the one for few to
    2^-23 of that (eight parts).  Which of the two depends on the number of rows and, from 64 experts on, on how many of them chose the
    expert.  Nothing is decided on the host.  A row with an infinity or
    something that is not a number, and one whose act(gate) * up is beyond 32 bits, gives a row that is not a number, whatever the
    activation makes of it."""
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
    if rows * max(top, 1) >= 2**31 or max(width, 2 * inner) > MX4_MOST:
        raise KernelError(f"chosen_experts_mx4: {rows} rows of {top} choices, width {width}, inner {inner} are too large")
    here = _here("chosen_experts_mx4", h, chosen, weights, w_gate_up.codes, w_gate_up.scales, w_down.codes, w_down.scales, error_word)
    if rows == 0 or top == 0:
        return torch.zeros((rows, width), dtype=torch.bfloat16, device=h.device)
    out = torch.empty_like(h)
    entries, stream, error = rows * top, _stream(here), error_word.data_ptr()
    # (the pairs' result rows start on 16-byte borders)
    many = entries * (w_gate_up.codes.numel() + w_down.codes.numel()) > MX4_FEW_BYTES * experts * experts and width % 4 == 0
    divided = many and experts >= MX4_DIVIDE_EXPERTS
    moe, lib, pair = load_library("moe"), _library("gemm_mx4"), _library("gemm_mx4_pair") if many else None
    few_tile = lib.srb_mx4_experts_tile()
    tile = pair.srb_mx4_experts_pair_tile() if many else few_tile
    # a tile has a slot at least; divided, an expert of the pairs has more than MX4_FEW_SLOTS, one of the others no more
    tiles = min(entries, entries // tile + (min(experts, entries // (MX4_FEW_SLOTS + 1)) if divided else experts))
    few_tiles = min(entries, entries // few_tile + experts, experts * -(-MX4_FEW_SLOTS // few_tile)) if divided else 0 if many else tiles
    # one piece of memory: the plan, the row of every slot, the slot of every choice, the slots' results, and what the products need
    memory = []

    def take(size: int) -> int:
        memory.append(_room(size))
        return sum(memory[:-1])
    plan_at, slot_row_at = take(4 * moe.srb_moe_plan_ints_of(rows, top, experts, tile)), take(4 * entries)
    entry_slot_at, y_at = take(4 * entries), take(4 * entries * width)
    few_at = take(lib.srb_mx4_experts_scratch(few_tiles, experts, width, inner, gated))
    if many:
        pair_at = take(pair.srb_mx4_experts_pair_scratch(tiles, experts, width, inner, gated))
    if divided:
        few_plan_at, pair_plan_at = take(4 * (experts + 2 + 2 * few_tiles)), take(4 * (experts + 2 + 2 * tiles))
    held = torch.empty(sum(memory), dtype=torch.uint8, device=h.device)
    at = held.data_ptr()
    plan, slot_row, entry_slot, y = at + plan_at, at + slot_row_at, at + entry_slot_at, at + y_at
    _check(moe, moe.srb_moe_plan_of(_P(chosen.data_ptr()), rows, top, experts, tile, _P(plan), _P(slot_row), _P(entry_slot), None, None, _P(error),
                                    stream if isinstance(stream, _P) else _P(stream)))
    matrices = (w_gate_up.codes.data_ptr(), w_gate_up.scales.data_ptr(), w_down.codes.data_ptr(), w_down.scales.data_ptr(), y)
    sizes = (experts, width, inner, gated, act_code, activation_param)
    few_plan = pair_plan = plan
    if divided:
        few_plan, pair_plan = at + few_plan_at, at + pair_plan_at
        _check(pair, pair.srb_mx4_divide_plan(plan, experts, MX4_FEW_SLOTS, few_tile, few_tiles, tiles, few_plan, pair_plan, error, stream))
    if few_tiles:
        _check(lib, lib.srb_mx4_experts(h.data_ptr(), few_plan, slot_row, *matrices, few_tiles, entries, *sizes, at + few_at, error, stream),
               3 + int(gated and inner % 128 != 0))
    if many:
        _check(pair, pair.srb_mx4_experts_pair(h.data_ptr(), pair_plan, entry_slot, *matrices, tiles, rows, top, MX4_FEW_SLOTS if divided else 0, *sizes,
                                               at + pair_at, error, stream), 3)
    _check(lib, lib.srb_mx4_combine(y, entry_slot, weights.data_ptr(), rows, top, width, out.data_ptr(), stream))
    return out
