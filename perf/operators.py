"""Four-bit weights: the operators by which their speed is measured, and what they must compute.

Weights (and, where asked, rows) are held in the microscaled four-bit format of the OCP Microscaling Formats specification: blocks
of 32 entries of a row share a scale 2^(s - 127) held in one byte s (255: not a number), and an entry is one of 0, 0.5, 1, 1.5, 2,
3, 4, 6 with a sign, two to a byte, the first of a pair in the low half.  A block's scale is 2^(floor(log2(largest magnitude)) - 2),
its entries go to the nearest value, ties to the even mantissa, magnitudes above 6 to 6.

Kinds of cases:

* ``quantize``: rows of activations into that form, and the values that the result stands for.
* ``linear``: rows through a matrix held in that form; ``four``: the rows are quantised too, on the way.
* ``choose``: a router's logits to the chosen experts and their weights, the experts in groups of which only the best are open.
* ``experts``: rows through their chosen experts, whose matrices are held in that form.

Sizes: the projections of a layer of width 4,096 with a feed-forward of 12,288, the routed experts of the Gegepel bench (64 of
2,048 x 1,408, 6 chosen), a router over 256 experts in 8 groups, and odd ones.
"""
from __future__ import annotations

import math
import random

import torch

own = False

VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
EXPERT_SIZES = dict(width=2048, experts=64, inner=1408, top=6)
ROUTER = dict(experts=256, top=8, groups=8, top_groups=4, group_best=2, scoring="sigmoid", bias=True, renormalize=True, scale=2.5)
LARGEST_FLOPS = 2 * 2048 * 4096 * 24576


# ---------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # eight users' rows on their way into a product of two four-bit operands
        dict(name="quantize-b8", kind="quantize", rows=8, width=4096, dtype="bfloat16"),
        # the rows of a prompt portion ahead of the second product of a feed-forward
        dict(name="quantize-p2048", kind="quantize", rows=2048, width=12288, dtype="bfloat16"),
        # 32-bit weights of an odd size, as they are quantised at load
        dict(name="quantize-f32-odd", kind="quantize", rows=5171, width=2891, dtype="float32"),
        # one user: the gate/up matrix is streamed once
        dict(name="linear-b1", kind="linear", rows=1, width=4096, features=24576, four=False, bias=False),
        # a decode batch through a projection with a bias, no size a multiple of anything
        dict(name="linear-b33-odd", kind="linear", rows=33, width=4095, features=6145, four=False, bias=True),
        # a prompt portion, rows kept in bfloat16
        dict(name="linear-p2048", kind="linear", rows=2048, width=4096, features=24576, four=False, bias=False),
        # a prompt portion with both operands in four bits
        dict(name="linear-four-p2048", kind="linear", rows=2048, width=4096, features=24576, four=True, bias=False),
        # a decode batch with both operands in four bits
        dict(name="linear-four-b48", kind="linear", rows=48, width=4096, features=4096, four=True, bias=False),
        # the router of a decode batch, and of a long prompt
        dict(name="choose-b64", kind="choose", rows=64, **ROUTER),
        dict(name="choose-p8192", kind="choose", rows=8192, **ROUTER),
        # eight users' tokens through a layer of routed experts: most experts that are touched see one row
        dict(name="experts-b8", kind="experts", rows=8, **EXPERT_SIZES),
        # a prompt portion through it, experts of very different load
        dict(name="experts-p2048", kind="experts", rows=2048, **EXPERT_SIZES),
    ]


def _log(rng: random.Random, low: int, high: int) -> int:
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng: random.Random):
    kind = rng.choice(["quantize", "linear", "linear", "linear", "choose", "experts", "experts"])
    if kind == "quantize":
        rows = _log(rng, 1, 8192)
        return dict(kind="quantize", rows=rows, width=_log(rng, 16, min(16384, 2048 * 12288 // rows)), dtype=rng.choice(["bfloat16", "bfloat16", "float32"]))
    if kind == "linear":
        rows, width = _log(rng, 1, 2048), _log(rng, 64, 8192)
        if rng.random() < 0.7:
            width = -(-width // 64) * 64
        features = _log(rng, 16, 24576)
        if rng.random() < 0.7:
            features = -(-features // 16) * 16
        features = min(features, LARGEST_FLOPS // (2 * rows * width))
        return dict(kind="linear", rows=rows, width=width, features=features, four=rng.random() < 0.4, bias=rng.random() < 0.3)
    if kind == "choose":
        groups = rng.choice([1, 2, 4, 8])
        per_group = rng.randint(2, 256 // groups)
        top_groups = rng.randint(1, groups)
        return dict(kind="choose", rows=_log(rng, 1, 8192), experts=groups * per_group, top=rng.randint(1, min(8, top_groups * per_group)),
                    groups=groups, top_groups=top_groups, group_best=rng.choice([1, 2]), scoring=rng.choice(["softmax", "sigmoid"]),
                    bias=rng.random() < 0.6, renormalize=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]))
    experts = rng.randint(4, 64)
    return dict(kind="experts", rows=_log(rng, 1, 2048), width=32 * rng.randint(8, 64), experts=experts, inner=16 * rng.randint(8, 88),
                top=rng.randint(1, min(6, experts)))


# ---------------------------------------------------------------------------------------------- inputs from the seed
def _normal(g, *shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda") * std


def _activations(g, rows: int, width: int, dtype: str = "bfloat16"):
    """Rows as they stand ahead of a product: normal entries, channels of different size, a few of them large."""
    x = _normal(g, rows, width) * torch.exp(0.5 * _normal(g, width))
    x = x * torch.where(torch.rand(width, generator=g, device="cuda") < 0.004, 20.0, 1.0)
    return x.to(DTYPES[dtype])


def _four_bit_matrix(g, *shape):
    """A matrix [..., rows, width] as a checkpoint holds it: codes two to a byte [..., ceil(width / 2)], scales [..., ceil(width / 32)]."""
    codes, scales = _plain_quantize(_normal(g, *shape, std=0.02))
    if codes.shape[-1] % 2:
        codes = torch.nn.functional.pad(codes, (0, 1))
    return codes[..., 0::2] | (codes[..., 1::2] << 4), scales


def _choices(g, case):
    """Every row's experts, a few of them chosen far more often than others, and their weights."""
    rows, experts, top = case["rows"], case["experts"], case["top"]
    logits = _normal(g, rows, experts) + _normal(g, experts)
    best = torch.topk(logits, top, dim=-1)
    return best.indices.to(torch.int32), torch.softmax(best.values, dim=-1)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    kind = case["kind"]
    if kind == "quantize":
        x = _activations(g, case["rows"], case["width"], case["dtype"])
        return dict(x=x * (torch.rand((case["rows"], 1), generator=g, device="cuda") > 0.02).to(x.dtype))      # padded rows are zero
    if kind == "linear":
        codes, scales = _four_bit_matrix(g, case["features"], case["width"])
        return dict(x=_activations(g, case["rows"], case["width"]), codes=codes, scales=scales,
                    bias=_normal(g, case["features"]) if case["bias"] else None)
    if kind == "choose":
        return dict(logits=_normal(g, case["rows"], case["experts"], std=2.0),
                    bias=_normal(g, case["experts"], std=0.1) if case["bias"] else None)
    chosen, weights = _choices(g, case)
    up = _four_bit_matrix(g, case["experts"], 2 * case["inner"], case["width"])
    down = _four_bit_matrix(g, case["experts"], case["width"], case["inner"])
    return dict(h=_activations(g, case["rows"], case["width"]), chosen=chosen, weights=weights, up=up, down=down,
                most=int(torch.bincount(chosen.reshape(-1).long(), minlength=case["experts"]).max()))


def prepare(case, seed):
    state = dict(case=case, **_inputs(case, seed))
    if own:
        from sglang_rs_b200 import ops
        state["ops"], state["error"] = ops, ops.new_error_word("cuda")
        if case["kind"] == "linear":
            state["matrix"] = ops.mx4_from_rows(state["codes"], state["scales"], case["width"])
        if case["kind"] == "experts":
            state["up_matrix"] = ops.mx4_from_rows(*state["up"], case["width"])
            state["down_matrix"] = ops.mx4_from_rows(*state["down"], case["inner"])
    return state


# ---------------------------------------------------------------------------------------------- the plain forms
def _plain_quantize(x):
    """Codes (one to a byte) and scales of the last axis of x."""
    width = x.shape[-1]
    blocks = torch.nn.functional.pad(x.float(), (0, -width % 32)).unflatten(-1, (-1, 32))
    largest = blocks.abs().amax(-1)
    exponent = torch.where(largest > 0, torch.frexp(largest).exponent - 1 - 2, -127).clamp(-127, 125)
    scaled = torch.ldexp(blocks.double(), -exponent[..., None]).float().abs()
    step = torch.where(scaled < 2, 0.5, torch.where(scaled < 4, 1.0, 2.0))
    rounded = (torch.round(scaled / step) * step).clamp(max=6.0)          # round: halves to the even neighbour
    low = (rounded * 2).to(torch.uint8)                                   # below 2 the code is twice the value
    high = torch.where(rounded < 4, (rounded + 2).to(torch.uint8), torch.where(rounded < 6, 6, 7).to(torch.uint8))
    codes = torch.where(rounded < 2, low, high) | (torch.signbit(blocks).to(torch.uint8) << 3)
    return codes.flatten(-2)[..., :width], (exponent + 127).to(torch.uint8)


def _plain_values(codes, scales):
    """What codes (one to a byte) and scales stand for, in 32 bits."""
    width = codes.shape[-1]
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), device=codes.device)
    blocks = torch.nn.functional.pad(table[codes.int()], (0, -width % 32)).unflatten(-1, (-1, 32))
    return torch.ldexp(blocks, scales.int()[..., None] - 127).flatten(-2)[..., :width]


def _plain_matrix(packed, scales, width: int):
    return _plain_values(torch.stack([packed & 15, packed >> 4], dim=-1).flatten(-2)[..., :width], scales)


def _plain_linear(state):
    case, x = state["case"], state["x"]
    if case["four"]:
        x = _plain_values(*_plain_quantize(x))
    y = x.float() @ _plain_matrix(state["codes"], state["scales"], case["width"]).T
    return (y if state["bias"] is None else y + state["bias"]).to(torch.bfloat16)


def _plain_choose(state):
    """In 64 bits: which of two scores is larger may hang on their last bits."""
    case, z = state["case"], state["logits"].double()
    rows, experts = z.shape
    scores = torch.sigmoid(z) if case["scoring"] == "sigmoid" else torch.exp(z - torch.logsumexp(z, -1, keepdim=True))
    picks = scores if state["bias"] is None else scores + state["bias"].double()
    grouped = picks.view(rows, case["groups"], -1)
    of_groups = torch.sort(grouped, dim=-1, descending=True).values[..., :case["group_best"]].sum(-1)
    order = torch.sort(of_groups, dim=-1, descending=True, stable=True).indices[:, :case["top_groups"]]
    open_ = torch.zeros_like(of_groups, dtype=torch.bool).scatter_(1, order, True)
    picks = torch.where(open_[..., None], grouped, -math.inf).view(rows, experts)
    chosen = torch.sort(picks, dim=-1, descending=True, stable=True).indices[:, :case["top"]]
    weights = scores.gather(1, chosen)
    if case["renormalize"]:
        weights = weights / weights.sum(-1, keepdim=True)
    return chosen.to(torch.int32), (weights * case["scale"]).float()


def _plain_experts(state):
    """Every expert's rows side by side, padded to the fullest expert's, through one product per matrix for all experts."""
    case, chosen = state["case"], state["chosen"].long()
    rows, top = chosen.shape
    order = torch.sort(chosen.reshape(-1), stable=True).indices
    expert = chosen.reshape(-1)[order]
    counts = torch.bincount(expert, minlength=case["experts"])
    place = torch.arange(rows * top, device=order.device) - (torch.cumsum(counts, 0) - counts)[expert]
    x = torch.zeros((case["experts"], state["most"], case["width"]), device=order.device)
    x[expert, place] = state["h"].float()[order // top]
    gate, up = (x @ _plain_matrix(*state["up"], case["width"]).transpose(1, 2)).chunk(2, dim=-1)
    y = (gate / (1 + torch.exp(-gate)) * up) @ _plain_matrix(*state["down"], case["inner"]).transpose(1, 2)
    terms = torch.empty((rows * top, case["width"]), device=order.device)
    terms[order] = y[expert, place]
    return (terms.view(rows, top, -1) * state["weights"][..., None]).sum(1).to(torch.bfloat16)


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        ops, error = state["ops"], state["error"]
        if kind == "quantize":
            return ops.dequantize_mx4(ops.quantize_mx4(state["x"]), DTYPES[case["dtype"]])
        if kind == "linear":
            rows = ops.quantize_mx4(state["x"]) if case["four"] else state["x"]
            return ops.linear_mx4(rows, state["matrix"], error, bias=state["bias"])
        if kind == "choose":
            return ops.choose_experts(state["logits"], case["top"], case["renormalize"], scoring=case["scoring"], choice_bias=state["bias"],
                                      groups=case["groups"], top_groups=case["top_groups"], group_best=case["group_best"],
                                      weight_scale=case["scale"])
        return ops.chosen_experts_mx4(state["h"], state["chosen"], state["weights"], state["up_matrix"], state["down_matrix"], "silu", error)
    if kind == "quantize":
        return _plain_values(*_plain_quantize(state["x"])).to(DTYPES[case["dtype"]])
    return {"linear": _plain_linear, "choose": _plain_choose, "experts": _plain_experts}[kind](state)


# ---------------------------------------------------------------------------------------------- what a pass cannot do without
def _four_bit_bytes(rows: int, width: int) -> int:
    return rows * (-(-width // 2) + -(-width // 32))


def work(case):
    rows, kind = case["rows"], case["kind"]
    if kind == "quantize":
        # the rows in, their four-bit form out and in again, the values out
        wide = 2 if case["dtype"] == "bfloat16" else 4
        return {"bytes": 2 * rows * case["width"] * wide + 2 * _four_bit_bytes(rows, case["width"]), "flops": 2 * rows * case["width"]}
    if kind == "linear":
        n, k = case["features"], case["width"]
        return {"bytes": _four_bit_bytes(n, k) + 2 * rows * (k + n) + (4 * n if case["bias"] else 0), "flops": 2 * rows * n * k}
    if kind == "choose":
        return {"bytes": rows * (4 * case["experts"] + 8 * case["top"]) + (4 * case["experts"] if case["bias"] else 0), "flops": 4 * rows * case["experts"]}
    entries, inner, width = rows * case["top"], case["inner"], case["width"]
    # experts that are touched, if the choices were even
    touched = case["experts"] * (1 - (1 - 1 / case["experts"]) ** entries)
    matrices = touched * (_four_bit_bytes(2 * inner, width) + _four_bit_bytes(width, inner))
    return {"bytes": int(matrices) + 4 * rows * width + 8 * entries, "flops": 6 * entries * inner * width}


# ---------------------------------------------------------------------------------------------- the definitions in 64 bits
def _exact_values_of(x):
    """Nearest of the format's values by comparison with the borders between them; a border belongs to the neighbour with the even code."""
    x = x.double()
    *lead, width = x.shape
    padded = torch.zeros((*lead, -(-width // 32) * 32), dtype=torch.float64, device=x.device)
    padded[..., :width] = x
    blocks = padded.view(*lead, -1, 32)
    largest = blocks.abs().amax(-1, keepdim=True)
    # 2^floor(log2(largest)) from the powers of two themselves: log2 may round up to the next whole number
    power = torch.exp2(torch.floor(torch.log2(largest.clamp(min=2.0 ** -125))))
    power = torch.where(power > largest, power / 2, power)
    power = torch.where(power * 2 <= largest, power * 2, power)
    scale = (power / 4).clamp(min=2.0 ** -127)
    magnitude = blocks.abs() / scale
    code = torch.zeros_like(magnitude)
    for i in range(7):
        border = (VALUES[i] + VALUES[i + 1]) / 2
        code += (magnitude >= border if i % 2 else magnitude > border)
    table = torch.tensor(VALUES, dtype=torch.float64, device=x.device)
    return (table[code.long()] * scale * torch.where(blocks < 0, -1.0, 1.0)).reshape(*lead, -1)[..., :width]


def _exact_matrix(packed, scales, width: int):
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), dtype=torch.float64, device=packed.device)
    values = torch.empty((*packed.shape[:-1], 2 * packed.shape[-1]), dtype=torch.float64, device=packed.device)
    values[..., 0::2] = table[(packed % 16).long()]
    values[..., 1::2] = table[(packed // 16).long()]
    return values[..., :width] * torch.exp2(scales.double() - 127).repeat_interleave(32, dim=-1)[..., :width]


def _exact_choose(case, given):
    z = given["logits"].double()
    scores = 1 / (1 + torch.exp(-z)) if case["scoring"] == "sigmoid" else torch.softmax(z, -1)
    picks = scores + (given["bias"].double() if given["bias"] is not None else 0)
    per_group = case["experts"] // case["groups"]
    best = picks.unflatten(-1, (case["groups"], per_group)).topk(min(case["group_best"], per_group), dim=-1).values.sum(-1)
    # a group is open if fewer than top_groups groups are ahead of it; equal ones with a lower index are ahead
    index = torch.arange(case["groups"], device=z.device)
    ahead = (best[:, None, :] > best[:, :, None]) | ((best[:, None, :] == best[:, :, None]) & (index[None, None, :] < index[None, :, None]))
    closed = (ahead.sum(-1) >= case["top_groups"]).repeat_interleave(per_group, dim=-1)
    left = picks.masked_fill(closed, -math.inf)
    chosen = []
    for _ in range(case["top"]):
        chosen.append(left.argmax(-1, keepdim=True))
        left = left.scatter(1, chosen[-1], -math.inf)
    chosen = torch.cat(chosen, dim=-1)
    weights = scores.gather(1, chosen)
    if case["renormalize"]:
        weights = weights / weights.sum(-1, keepdim=True)
    return chosen.to(torch.int32), weights * case["scale"]


def exact(case, seed):
    given = _inputs(case, seed)
    if case["kind"] == "quantize":
        return _exact_values_of(given["x"])
    if case["kind"] == "linear":
        x = _exact_values_of(given["x"]) if case["four"] else given["x"].double()
        y = x @ _exact_matrix(given["codes"], given["scales"], case["width"]).T
        return y if given["bias"] is None else y + given["bias"].double()
    if case["kind"] == "choose":
        return _exact_choose(case, given)
    out = torch.zeros((case["rows"], case["width"]), dtype=torch.float64, device="cuda")
    h, weights = given["h"].double(), given["weights"].double()
    for e in range(case["experts"]):
        row, choice = torch.nonzero(given["chosen"] == e, as_tuple=True)
        up = _exact_matrix(given["up"][0][e], given["up"][1][e], case["width"])
        down = _exact_matrix(given["down"][0][e], given["down"][1][e], case["inner"])
        gate, value = (h[row] @ up.T).split(case["inner"], dim=-1)
        out.index_add_(0, row, (torch.sigmoid(gate) * gate * value) @ down.T * weights[row, choice][:, None])
    return out
