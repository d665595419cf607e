"""The microscaled four-bit format and what is computed with it, in 64 bits, one function per formula, no shared code."""
import itertools
import math

import torch

MAGNITUDES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def nearest_code(v: float) -> int:
    """The code of |v|, ties to the even code (even codes are those with an even mantissa)."""
    v = abs(v)
    best = min(range(8), key=lambda c: (abs(MAGNITUDES[c] - v), c & 1))
    return 7 if v > 6.0 else best


def quantize(x: torch.Tensor):
    """Codes (one to a byte) [..., width] and scales [..., blocks] of x, on the host."""
    x = x.detach().cpu().double()
    width = x.shape[-1]
    rows = x.reshape(-1, width)
    blocks = -(-width // 32)
    codes = torch.zeros(rows.shape[0], width, dtype=torch.uint8)
    scales = torch.zeros(rows.shape[0], blocks, dtype=torch.uint8)
    for r, b in itertools.product(range(rows.shape[0]), range(blocks)):
        block = rows[r, 32 * b:32 * b + 32].tolist()
        if not all(math.isfinite(v) for v in block):
            scales[r, b] = 255
            continue
        largest = max(abs(v) for v in block)
        e = max(-127, math.frexp(largest)[1] - 1 - 2) if largest else -127
        scales[r, b] = e + 127
        for i, v in enumerate(block):
            codes[r, 32 * b + i] = nearest_code(math.ldexp(v, -e)) | (8 if math.copysign(1.0, v) < 0 else 0)
    return codes.view(*x.shape[:-1], width), scales.view(*x.shape[:-1], blocks)


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """float64 [..., width] from codes (one to a byte) and scales."""
    table = torch.tensor(MAGNITUDES + [-m for m in MAGNITUDES], dtype=torch.float64)
    scale = torch.exp2(scales.cpu().double() - 127)
    scale = torch.where(scales.cpu() == 255, math.nan, scale)
    return table[codes.cpu().long()] * scale.repeat_interleave(32, dim=-1)[..., :codes.shape[-1]]


def packed(codes: torch.Tensor) -> torch.Tensor:
    """Two codes to a byte, the first in the low half."""
    if codes.shape[-1] % 2:
        codes = torch.cat([codes, torch.zeros_like(codes[..., :1])], dim=-1)
    return codes[..., 0::2] + 16 * codes[..., 1::2]


def scale_rows(scales: torch.Tensor, rows: int, width: int) -> torch.Tensor:
    """[..., rows, blocks] from tiles [..., row tiles, column tiles, 512]: byte (r % 32) * 16 + (r / 32) * 4 + b of a tile."""
    scales = scales.cpu()
    out = torch.zeros((*scales.shape[:-3], rows, -(-width // 32)), dtype=torch.uint8)
    for r in range(rows):
        for b in range(out.shape[-1]):
            out[..., r, b] = scales[..., r // 128, b // 4, (r % 32) * 16 + (r % 128) // 32 * 4 + b % 4]
    return out


def activation(name: str, g: torch.Tensor, u, param: float = 0.0) -> torch.Tensor:
    if name == "silu":
        return g / (1 + torch.exp(-g)) * u
    if name == "gelu_tanh":
        return g / 2 * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))) * u
    if name == "relu2":
        return g.clamp(min=0) ** 2 * u
    g = g.clamp(max=param)
    u = u if not isinstance(u, torch.Tensor) else u.clamp(-param, param)
    return g / (1 + torch.exp(-1.702 * g)) * (u + 1)


def choose(logits, top, groups=1, top_groups=1, group_best=1, scoring="softmax", bias=None, renormalize=False, scale=1.0, eps=0.0):
    """Row by row with sorted lists: (chosen, weights)."""
    logits = logits.detach().cpu().double()
    bias = None if bias is None else bias.detach().cpu().double()
    chosen, weights = [], []
    for z in logits:
        scores = torch.sigmoid(z) if scoring == "sigmoid" else torch.softmax(z, -1)
        picks = scores if bias is None else scores + bias
        picks = [p if p == p else -math.inf for p in picks.tolist()]
        length = len(picks) // groups
        of_group = [sum(sorted(picks[g * length:(g + 1) * length])[-group_best:]) for g in range(groups)]
        open_ = sorted(range(groups), key=lambda g: (-of_group[g], g))[:top_groups]
        order = sorted((e for e in range(len(picks)) if e // length in open_), key=lambda e: (-picks[e], e))[:top]
        w = scores[order]
        if renormalize:
            w = w / (w.sum() + eps)
        chosen.append(order)
        weights.append(w * scale)
    return torch.tensor(chosen, dtype=torch.int32).view(len(logits), top), torch.stack(weights) if weights else torch.zeros(0, top, dtype=torch.float64)


def experts(h, chosen, weights, up, down, name, gated=True, param=0.0):
    """(result, room): ``room`` is how far a result may be off whose act(gate) * up is rounded to bfloat16 once, whose sums run in
    32 bits (every product and partial sum off by at most 2^-20 of the magnitudes that went in) and which is rounded to bfloat16 at the end."""
    h, weights = h.detach().cpu().double(), weights.detach().cpu().double()
    out, room = torch.zeros(h.shape, dtype=torch.float64), torch.zeros(h.shape, dtype=torch.float64)
    for r, row in enumerate(chosen.cpu().tolist()):
        for c, e in enumerate(row):
            if not 0 <= e < up.shape[0]:
                continue
            z, around = up[e] @ h[r], up[e].abs() @ h[r].abs()
            inner = down.shape[-1]
            g, u = (z[:inner], z[inner:]) if gated else (z, 1.0)
            act = activation(name, g, u, param)
            # the sums' errors through the activation: slopes of all of them are below 2 in g (relu2: 2 |g|)
            slope = 2.0 + (2 * g.abs() if name == "relu2" else 0.0)
            second = (u.abs() + 1) if gated else 1.0
            off = 2.0 ** -20 * (around[:inner] * slope * second + (around[inner:] * (g.abs() + 1) if gated else 0.0))
            off = off + 2.0 ** -8 * act.abs() + 2.0 ** -18 * act.abs()
            out[r] += weights[r, c] * (down[e] @ act)
            room[r] += weights[r, c].abs() * (down[e].abs() @ (off + 2.0 ** -20 * act.abs()))
    return out, room + 2.0 ** -8 * (out.abs() + room)
