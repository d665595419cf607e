"""Matrices in four bits, the products with them and the router in groups, each against a plain implementation in 64 bits."""
import math

import pytest
import torch

import plain_mx4 as pm
from sglang_rs_b200 import ops
from sglang_rs_b200.ops import mx4

pytestmark = pytest.mark.gpu


def generator(seed):
    return torch.Generator().manual_seed(seed)


def rows_of(seed, *shape, dtype=torch.bfloat16, spread=0.5):
    g = generator(seed)
    x = torch.randn(shape, generator=g) * torch.exp(spread * torch.randn(shape[-1], generator=g))
    return x.to(dtype).cuda()


def random_matrix(seed, *shape, low=110, high=124):
    """(Mx4, its values in 64 bits on the host): random codes, scales 2^(low - 127) .. 2^(high - 127)."""
    g = generator(seed)
    codes = torch.randint(0, 16, shape, generator=g, dtype=torch.uint8)
    scales = torch.randint(low, high + 1, (*shape[:-1], -(-shape[-1] // 32)), generator=g, dtype=torch.uint8)
    return ops.mx4_from_rows(pm.packed(codes).cuda(), scales.cuda(), shape[-1]), pm.values(codes, scales)


def word():
    return ops.new_error_word("cuda")


# ------------------------------------------------------------------------------------------- the format
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 32), (3, 31), (2, 33), (5, 128), (4, 129), (1, 500), (130, 160), (33, 264)])
def test_quantized_rows(rows, width, dtype):
    x = rows_of(rows * 1000 + width, rows, width, dtype=dtype)
    q = ops.quantize_mx4(x)
    codes, scales = pm.quantize(x)
    assert q.shape == (rows, width)
    assert torch.equal(pm.scale_rows(q.scales, rows, width), scales)
    held = pm.packed(codes)
    assert torch.equal(q.codes[:, :held.shape[1]].cpu(), held)
    assert not q.codes[:, held.shape[1]:].any()
    for out in (torch.bfloat16, torch.float32):
        assert torch.equal(ops.dequantize_mx4(q, out).cpu().double(), pm.values(codes, scales))


def test_every_tie_and_every_border():
    eighths = torch.arange(-256, 257).float() / 32
    blocks = torch.zeros(len(eighths), 32)
    blocks[:, 0], blocks[:, 5] = 4.0, eighths                 # the 4 makes the scale 1, but for magnitudes of 8
    for x in (blocks, blocks * 2.0 ** -60, blocks.roll(9, dims=1) * 2.0 ** 70):
        codes, scales = pm.quantize(x)
        assert torch.equal(ops.dequantize_mx4(ops.quantize_mx4(x.cuda()), torch.float32).cpu().double(), pm.values(codes, scales))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_zero_tiny_and_huge_blocks(dtype):
    least = 2.0 ** -133 if dtype == torch.bfloat16 else 2.0 ** -149
    x = torch.zeros(6, 64, dtype=dtype)
    x[1, 3], x[1, 40] = least, -least
    x[2, :] = torch.finfo(dtype).max
    x[3, :] = torch.finfo(dtype).tiny
    x[4, 0], x[4, 1] = 2.0 ** -126, 2.0 ** -128
    x[5, 7], x[5, 8] = -0.0, 1.0
    codes, scales = pm.quantize(x)
    q = ops.quantize_mx4(x.cuda())
    assert torch.equal(pm.scale_rows(q.scales, 6, 64), scales)
    assert torch.equal(q.codes[:, :32].cpu(), pm.packed(codes))
    assert torch.equal(ops.dequantize_mx4(q, torch.float32).cpu().double(), pm.values(codes, scales))


def test_blocks_that_are_not_finite():
    x = rows_of(1, 4, 96)
    x[1, 40], x[2, 5], x[2, 95] = math.inf, math.nan, -math.inf
    got = ops.dequantize_mx4(ops.quantize_mx4(x)).cpu().double()
    codes, scales = pm.quantize(x)
    want = pm.values(codes, scales)
    assert torch.equal(got.isnan(), want.isnan()) and want.isnan().sum() == 96
    assert torch.equal(got.nan_to_num(), want.nan_to_num())


def test_stacks_pitches_and_borders_of_rows():
    wide = rows_of(2, 40, 300)
    for x in (wide[:, 3:170], wide[:, 8:136], wide[1:, :], wide[::2, 16:48]):
        codes, scales = pm.quantize(x)
        q = ops.quantize_mx4(x)
        assert torch.equal(q.codes[:, :pm.packed(codes).shape[1]].cpu(), pm.packed(codes))
        assert torch.equal(pm.scale_rows(q.scales, *x.shape), scales)
    stack = rows_of(3, 3, 70, 130)
    q = ops.quantize_mx4(stack)
    codes, scales = pm.quantize(stack)
    assert q.shape == (3, 70, 130) and torch.equal(pm.scale_rows(q.scales, 70, 130), scales)
    assert torch.equal(ops.dequantize_mx4(q).cpu().double(), pm.values(codes, scales))
    again = ops.mx4_from_rows(pm.packed(codes).cuda(), scales.cuda(), 130)
    assert torch.equal(again.codes, q.codes) and torch.equal(again.scales, q.scales)


def test_rows_behind_the_last_have_a_scale_of_one():
    q = ops.quantize_mx4(rows_of(4, 130, 160))
    padded = pm.scale_rows(q.scales, 256, 256)
    assert (padded[130:] == 127).all() and (padded[:130, 5:] == 127).all()


def test_nothing_to_quantize():
    q = ops.quantize_mx4(torch.empty(0, 40, device="cuda"))
    assert q.shape == (0, 40) and ops.dequantize_mx4(q).shape == (0, 40)
    assert ops.linear_mx4(q, random_matrix(1, 9, 40)[0], word()).shape == (0, 9)
    assert ops.linear_mx4(torch.empty(0, 40, device="cuda", dtype=torch.bfloat16), random_matrix(1, 9, 40)[0], word()).shape == (0, 9)


# ------------------------------------------------------------------------------------------- products
def room_of(x, w, y, out_dtype):
    """How far a product may be off: sums of ceil(width / 32) + 8 terms in 32 bits, each off by at most 2^-23 of the magnitudes; rows held as
    parts to 2^-22 of a block's largest entry or, since the format's least scale is 2^-127 and its least step 0.5, to half of 2^-128; one
    rounding of the result."""
    width = x.shape[1]
    around = x.abs() @ w.abs().T
    padded = torch.nn.functional.pad(x.abs(), (0, -width % 32)).view(x.shape[0], -1, 32).amax(-1)
    blocks = torch.nn.functional.pad(w.abs(), (0, -width % 32)).view(w.shape[0], -1, 32).sum(-1)
    room = (-(-width // 32) + 8) * 2.0 ** -23 * around + 2.0 ** -22 * (padded @ blocks.T) + 2.0 ** -129 * w.abs().sum(1)
    return room + torch.finfo(out_dtype).eps / 2 * (y.abs() + room) + torch.finfo(out_dtype).smallest_normal


def check_linear(x, matrix, w, bias=None, out_dtype=torch.bfloat16):
    error = word()
    got = ops.linear_mx4(x, matrix, error, bias=bias, out_dtype=out_dtype)
    ops.raise_on_error_word(error)
    rows = (ops.dequantize_mx4(x, torch.float32) if isinstance(x, ops.Mx4) else x).cpu().double()
    want = rows @ w.T
    if bias is not None:
        want = want + bias.cpu().double()
    assert got.dtype == out_dtype and got.shape == want.shape
    room = room_of(rows, w, want, out_dtype)
    if bias is not None:
        room = room + 2.0 ** -23 * bias.cpu().double().abs()
    excess = ((got.cpu().double() - want).abs() - room).max()
    assert excess <= 0, float(excess)
    return got


SHAPES = [(1, 32, 1), (1, 128, 128), (2, 1, 3), (3, 33, 130), (5, 256, 16), (7, 1000, 129), (8, 384, 300), (9, 2050, 96), (16, 130, 257),
          (17, 640, 128), (31, 96, 511), (33, 4095, 100), (48, 512, 384), (64, 160, 640), (65, 288, 127), (100, 257, 130), (128, 512, 256),
          (129, 130, 513), (200, 1024, 520), (257, 320, 260), (300, 72, 1030), (513, 200, 300),
          (1025, 328, 6150), (700, 1300, 9601)]


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("rows,width,features", SHAPES)
def test_products(rows, width, features, four):
    x = rows_of(rows + width, rows, width)
    matrix, w = random_matrix(features, features, width)
    check_linear(ops.quantize_mx4(x) if four else x, matrix, w)


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("rows,width,features", [(1, 200, 70), (20, 512, 256), (70, 300, 200), (300, 640, 258)])
def test_products_with_a_bias_and_in_32_bits(rows, width, features, four):
    x = rows_of(rows, rows, width)
    x = ops.quantize_mx4(x) if four else x
    matrix, w = random_matrix(features, features, width)
    bias = torch.randn(features, generator=generator(5)).cuda()
    check_linear(x, matrix, w, bias)
    check_linear(x, matrix, w, None, torch.float32)
    check_linear(x, matrix, w, bias, torch.float32)


@pytest.mark.parametrize("rows,four", [(1, False), (1, True), (2, False), (20, False), (64, True)])
def test_more_tiles_than_blocks(rows, four):
    """A head's many features: every block takes several tiles, the sums of one stored while the next one's are taken."""
    x = rows_of(rows, rows, 264)
    matrix, w = random_matrix(91, 79 * 1024 + 3, 264)
    check_linear(ops.quantize_mx4(x) if four else x, matrix, w)


@pytest.mark.parametrize("rows", [3, 40, 200])
def test_rows_of_a_wider_matrix(rows):
    wide = rows_of(6, rows, 700)
    for first, width in ((0, 640), (8, 512), (1, 320), (5, 333)):
        matrix, w = random_matrix(width, 140, width)
        check_linear(wide[:, first:first + width], matrix, w)


@pytest.mark.parametrize("rows", [1, 24, 200])
@pytest.mark.parametrize("four", [False, True])
def test_zero_rows_and_rows_that_are_not_finite_stay_by_themselves(rows, four):
    x = rows_of(7, rows + 3, 256)
    x[0] = 0
    x[1, 200], x[2, 3] = math.inf, math.nan
    matrix, w = random_matrix(8, 200, 256)
    held = ops.quantize_mx4(x) if four else x
    got = ops.linear_mx4(held, matrix, word())
    assert (got[0] == 0).all()
    assert not got[1].isfinite().any() and not got[2].isfinite().any()
    rest = ops.quantize_mx4(x[3:].contiguous()) if four else x[3:].contiguous()
    alone = check_linear(rest, matrix, w)
    assert torch.equal(got[3:], alone)


@pytest.mark.parametrize("rows", [2, 150])
@pytest.mark.parametrize("four", [False, True])
def test_a_weight_block_that_is_not_a_number_spoils_its_feature_alone(rows, four):
    codes = torch.randint(0, 16, (130, 256), generator=generator(9), dtype=torch.uint8)
    scales = torch.full((130, 8), 120, dtype=torch.uint8)
    scales[77, 6] = 255
    matrix = ops.mx4_from_rows(pm.packed(codes).cuda(), scales.cuda())
    x = rows_of(10, rows, 256)
    got = ops.linear_mx4(ops.quantize_mx4(x) if four else x, matrix, word())
    assert got[:, 77].isnan().all() and got[:, :77].isfinite().all() and got[:, 78:].isfinite().all()


@pytest.mark.parametrize("rows", [2, 150])
@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("size,low,high", [(2.0 ** -100, 200, 220), (2.0 ** 100, 30, 50), (1.0, 0, 12), (2.0 ** -120, 240, 252), (2.0 ** 120, 1, 9)])
def test_scales_at_the_ends_of_their_range(rows, four, size, low, high):
    x = (rows_of(11, rows, 192).float() * size).to(torch.bfloat16)
    matrix, w = random_matrix(12, 100, 192, low=low, high=high)
    check_linear(ops.quantize_mx4(x) if four else x, matrix, w, None, torch.float32)


@pytest.mark.parametrize("rows", [4, 140])
def test_entries_far_below_the_largest_of_their_block(rows):
    # powers of two down to 2^-14 of the block's largest entry are held exactly, with all eight bits of a bfloat16
    g = generator(13)
    x = torch.exp2(-torch.randint(0, 14, (rows, 256), generator=g).double()) * (1 + torch.randint(0, 128, (rows, 256), generator=g) / 128)
    x = x.to(torch.bfloat16).cuda()
    codes = torch.full((64, 256), 0, dtype=torch.uint8)
    for f in range(64):
        codes[f, (f * 37) % 256] = 2                          # one entry of the row, times one
    matrix = ops.mx4_from_rows(pm.packed(codes).cuda(), torch.full((64, 8), 127, dtype=torch.uint8).cuda())
    got = ops.linear_mx4(x, matrix, word())
    assert torch.equal(got, x[:, [(f * 37) % 256 for f in range(64)]])


@pytest.mark.parametrize("rows,width,features", [(1, 2048, 512), (40, 1024, 384), (300, 512, 512)])
@pytest.mark.parametrize("four", [False, True])
def test_the_same_bits_again_and_beside_other_work(rows, width, features, four):
    x = rows_of(14, rows, width)
    x = ops.quantize_mx4(x) if four else x
    matrix, _ = random_matrix(15, features, width)
    first = ops.linear_mx4(x, matrix, word())
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    results = []
    for stream in streams:
        with torch.cuda.stream(stream):
            results += [ops.linear_mx4(x, matrix, word()) for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(first, r) for r in results)


def test_products_in_a_captured_graph_follow_their_inputs():
    error = word()
    for rows in (1, 20, 200):
        x, (matrix, w) = rows_of(16, rows, 512), random_matrix(17, 256, 512)
        four, other = x.clone(), x.clone()
        for warm in range(2):
            ops.linear_mx4(other, matrix, error), ops.linear_mx4(ops.quantize_mx4(four), matrix, error)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a = ops.linear_mx4(other, matrix, error)
            b = ops.linear_mx4(ops.quantize_mx4(four), matrix, error)
        for seed in (18, 19):
            new = rows_of(seed, rows, 512)
            other.copy_(new), four.copy_(new)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(a, ops.linear_mx4(new, matrix, error)) and torch.equal(b, ops.linear_mx4(ops.quantize_mx4(new), matrix, error))
    ops.raise_on_error_word(error)


def test_refusals():
    matrix, _ = random_matrix(20, 64, 128)
    stack, _ = random_matrix(21, 2, 64, 128)
    x, error = rows_of(22, 4, 128), word()
    for call in (lambda: ops.linear_mx4(x.float(), matrix, error), lambda: ops.linear_mx4(x[:, :64], matrix, error),
                 lambda: ops.linear_mx4(x, stack, error), lambda: ops.linear_mx4(x.t(), matrix, error),
                 lambda: ops.linear_mx4(x, matrix, error, bias=torch.zeros(63, device="cuda")),
                 lambda: ops.linear_mx4(x, matrix, error, out_dtype=torch.float16), lambda: ops.linear_mx4(x, matrix.codes, error),
                 lambda: ops.linear_mx4(x, ops.Mx4(matrix.codes, matrix.scales, 200), error),
                 lambda: ops.quantize_mx4(x.half()), lambda: ops.quantize_mx4(x.t()), lambda: ops.dequantize_mx4(matrix, torch.int8),
                 lambda: ops.mx4_from_rows(matrix.codes, matrix.scales), lambda: ops.mx4_from_rows(matrix.codes.cpu(), matrix.scales.cpu())):
        with pytest.raises(ops.KernelError):
            call()


def test_more_rows_than_the_kernels_count_are_refused():
    x = torch.empty(2 ** 31 - 1, 1, dtype=torch.bfloat16, device="cuda")
    matrix, _ = random_matrix(20, 64, 1)
    for call in (lambda: ops.quantize_mx4(x), lambda: ops.linear_mx4(x, matrix, word())):
        with pytest.raises(ops.KernelError, match="too large"):
            call()


# ------------------------------------------------------------------------------------------- the router in groups
CHOICES = [dict(experts=8, top=2), dict(experts=1, top=1), dict(experts=64, top=6, renormalize=True),
           dict(experts=256, top=8, groups=8, top_groups=4, group_best=2, scoring="sigmoid", bias=0.1, renormalize=True, scale=2.5),
           dict(experts=160, top=6, groups=8, top_groups=3, group_best=1, scale=16.0), dict(experts=30, top=4, groups=3, top_groups=1, group_best=2, bias=0.02),
           dict(experts=1024, top=32, groups=32, top_groups=8, group_best=2, scoring="sigmoid", bias=1.0), dict(experts=257, top=9, scoring="sigmoid"),
           dict(experts=12, top=12, scoring="sigmoid", renormalize=True, eps=1e-20), dict(experts=20, top=10, groups=4, top_groups=2, bias=3.0)]


def check_choice(logits, case, bias):
    got, weights = ops.choose_experts(logits, case["top"], case.get("renormalize", False), scoring=case.get("scoring", "softmax"), choice_bias=bias,
                                      groups=case.get("groups", 1), top_groups=case.get("top_groups", 1), group_best=case.get("group_best", 1),
                                      weight_scale=case.get("scale", 1.0), norm_eps=case.get("eps", 0.0))
    want, w = pm.choose(logits, case["top"], case.get("groups", 1), case.get("top_groups", 1), case.get("group_best", 1), case.get("scoring", "softmax"),
                        bias, case.get("renormalize", False), case.get("scale", 1.0), case.get("eps", 0.0))
    assert torch.equal(got.cpu(), want)
    # a score: an exponential of an argument off by 2^-24 of its size (below 64 here), a sum and two divisions; a sum of scores; a product
    assert ((weights.cpu().double() - w).abs() <= 2.0 ** -17 * w.abs() + 1e-37).all()


@pytest.mark.parametrize("case", CHOICES)
@pytest.mark.parametrize("rows", [1, 5, 130])
def test_choices(case, rows):
    logits = torch.randn(rows, case["experts"], generator=generator(rows)).cuda() * 2
    bias = torch.randn(case["experts"], generator=generator(3)).cuda() * case["bias"] if "bias" in case else None
    check_choice(logits, case, bias)


@pytest.mark.parametrize("case", [c for c in CHOICES if c["experts"] <= 257])
def test_choices_of_more_rows_than_warps(case):
    """Many rows: the same as in small calls."""
    rows = 44 * torch.cuda.get_device_properties(0).multi_processor_count + 1
    logits = torch.randn(rows, case["experts"], generator=generator(92)).cuda() * 2
    logits[::97] = 0.5
    logits[5, ::2], logits[6, 1::2] = math.nan, -math.inf
    bias = torch.randn(case["experts"], generator=generator(3)).cuda() * case["bias"] if "bias" in case else None
    options = dict(scoring=case.get("scoring", "softmax"), choice_bias=bias, groups=case.get("groups", 1), top_groups=case.get("top_groups", 1),
                   group_best=case.get("group_best", 1))
    chosen, weights = ops.choose_experts(logits, case["top"], True, **options)
    for first in range(0, rows, 1024):
        few, same = ops.choose_experts(logits[first:first + 1024], case["top"], True, **options)
        assert torch.equal(chosen[first:first + 1024], few)
        assert torch.equal(weights[first:first + 1024].nan_to_num(7.0), same.nan_to_num(7.0))
    check_choice(logits[-300:], case, bias)


@pytest.mark.parametrize("case", CHOICES)
def test_choices_between_equals_and_all_but_equals(case):
    experts = case["experts"]
    g = generator(23)
    logits = torch.randint(-2, 3, (60, experts), generator=g).float()
    logits[:20] = 0.25                                        # all alike
    logits[20:40] += 2.0 ** -20 * torch.randint(-3, 4, (20, experts), generator=g).float()
    bias = torch.randint(-1, 2, (experts,), generator=g).float().cuda() * case["bias"] if "bias" in case else None
    check_choice(logits.cuda(), case, bias)


@pytest.mark.parametrize("groups,top_groups", [(1, 1), (8, 3)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("top", [1, 6, 24])
def test_choices_where_scores_of_unlike_logits_are_alike(scoring, groups, top_groups, top):
    """Sigmoids of 1 and of 0, exponentials of 1 and of 0: the lower index goes first, as it does between equal logits."""
    g = generator(41)
    levels = [torch.tensor([17.0, 30.5, 36.0, 37.0, 38.5, 40.0, 100.0]), torch.tensor([0.0, 1e-20, -1e-20, 3e-25, 1e-39, 0.0, -0.0]),
              torch.tensor([-720.0, -750.0, -800.0, -900.0, -750.0, -1e4, -math.inf]), torch.tensor([40.0, 38.5, 0.0, 1e-20, -800.0, -900.0, 3.0])]
    logits = torch.cat([level[torch.randint(0, 7, (40, 64), generator=g)] for level in levels])
    logits[-3:] = 0.0
    if scoring == "softmax":
        logits[80:120, 5] = 1.0                               # a row of minus infinities has no softmax
    check_choice(logits.cuda(), dict(experts=64, top=top, groups=groups, top_groups=top_groups, scoring=scoring), None)


@pytest.mark.parametrize("top", [1, 7, 8, 31, 32])
def test_choices_in_runs_of_all_but_equals(top):
    """Runs of five experts whose biased sigmoids are some 2^-24 apart: inside the chosen ones, over their end, and behind the 32nd."""
    g = generator(42)
    steps = (torch.arange(64) // 5 * 0.4 - 2.5).double()
    bias = 0.2 * torch.randn(64, generator=g)
    logits = torch.empty(200, 64)
    for row in logits:
        score = torch.sigmoid(steps[torch.randperm(64, generator=g)]) - bias.double() + 0.3
        row.copy_(torch.logit(score.clamp(0.01, 0.99)).float())
    check_choice(logits.cuda(), dict(experts=64, top=top, scoring="sigmoid"), bias.cuda())


def test_choices_among_masked_experts():
    logits = torch.randn(40, 64, generator=generator(24))
    logits[:, 1::2] = -math.inf
    logits[3, :] = -math.inf
    logits[4, 8:] = -math.inf
    logits[5, 6:] = torch.finfo(torch.float32).min
    case = dict(experts=64, top=6, groups=8, top_groups=4, group_best=2)
    for scoring in ("softmax", "sigmoid"):
        got, weights = ops.choose_experts(logits.cuda(), 6, scoring=scoring, groups=8, top_groups=4, group_best=2)
        want, w = pm.choose(logits, 6, 8, 4, 2, scoring)
        assert torch.equal(got.cpu(), want)
        assert torch.equal(weights.cpu().isnan(), w.isnan())
        assert ((weights.cpu().double() - w).abs().nan_to_num() <= 2.0 ** -17 * w.abs().nan_to_num() + 1e-37).all()


def test_logits_that_are_not_numbers_are_chosen_last():
    logits = torch.randn(4, 16, generator=generator(25))
    logits[1, 3], logits[2, :] = math.nan, math.nan
    got, weights = ops.choose_experts(logits.cuda(), 5, scoring="sigmoid")
    want, _ = pm.choose(logits, 5, scoring="sigmoid")
    assert torch.equal(got.cpu(), want) and 3 not in got[1].tolist() and got[2].tolist() == [0, 1, 2, 3, 4]


def test_choices_from_rows_of_a_wider_matrix_and_of_nothing():
    wide = torch.randn(30, 100, generator=generator(26)).cuda()
    check_choice(wide[:, 7:71], dict(experts=64, top=4, groups=4, top_groups=2), None)
    chosen, weights = ops.choose_experts(wide[:0], 3)
    assert chosen.shape == weights.shape == (0, 3)


@pytest.mark.parametrize("options", [dict(top=0), dict(top=33), dict(top=9), dict(top=2, groups=3), dict(top=2, groups=2, top_groups=3), dict(top=2, group_best=3),
                                     dict(top=5, groups=2, top_groups=1), dict(top=2, groups=8, top_groups=8, group_best=2), dict(top=-1),
                                     dict(top=2, scoring="none"), dict(top=2, choice_bias="short")])
def test_choices_that_are_refused(options):
    options = dict(options)
    if "choice_bias" in options:
        options["choice_bias"] = torch.zeros(7, device="cuda")
    with pytest.raises(ops.KernelError):
        ops.choose_experts(torch.zeros(3, 8, device="cuda"), options.pop("top"), **options)
    with pytest.raises(ops.KernelError):
        ops.choose_experts(torch.zeros(3, 1025, device="cuda"), 2)


# ------------------------------------------------------------------------------------------- experts
def check_experts(h, chosen, weights, up, down, name="silu", gated=True, param=0.0):
    (up_matrix, up_values), (down_matrix, down_values) = up, down
    error = word()
    got = ops.chosen_experts_mx4(h, chosen, weights, up_matrix, down_matrix, name, error, gated=gated, activation_param=param)
    ops.raise_on_error_word(error)
    want, room = pm.experts(h, chosen, weights, up_values, down_values, name, gated, param)
    assert got.dtype == torch.bfloat16 and got.shape == want.shape
    excess = ((got.cpu().double() - want).abs() - room).max() if want.numel() else torch.tensor(0.0)
    assert excess <= 1e-37, float(excess)
    return got


def expert_case(seed, rows, experts, width, inner, top, gated=True):
    g = generator(seed)
    h = torch.randn(rows, width, generator=g).to(torch.bfloat16).cuda()
    chosen = torch.stack([torch.randperm(experts, generator=g)[:top] for _ in range(rows)]).int().cuda() if rows else torch.zeros(0, top).int().cuda()
    weights = torch.rand(rows, top, generator=g).cuda()
    return h, chosen, weights, random_matrix(seed + 1, experts, (2 if gated else 1) * inner, width, low=116, high=122), random_matrix(seed + 2, experts, width, inner, low=116, high=122)


@pytest.mark.parametrize("rows,experts,width,inner,top", [(1, 4, 64, 32, 1), (1, 8, 256, 128, 3), (3, 5, 130, 70, 2), (8, 16, 256, 192, 4), (20, 3, 320, 96, 3),
                                                          (40, 2, 128, 256, 1), (70, 4, 96, 144, 2), (150, 3, 264, 136, 2), (33, 7, 257, 33, 5), (200, 8, 1540, 48, 4),
                                                          (90, 2, 192, 192, 1), (90, 2, 192, 224, 1)])
def test_experts(rows, experts, width, inner, top):
    check_experts(*expert_case(30 + rows, rows, experts, width, inner, top))


KERNELS = dict(few=dict(MX4_FEW_BYTES=1 << 62), pairs=dict(MX4_FEW_BYTES=0, MX4_DIVIDE_EXPERTS=1 << 20),
               divided=dict(MX4_FEW_BYTES=0, MX4_DIVIDE_EXPERTS=1, MX4_FEW_SLOTS=20))


@pytest.mark.parametrize("kernels", KERNELS)
@pytest.mark.parametrize("rows,experts,width,inner,top", [(1, 4, 64, 32, 1), (70, 4, 96, 144, 2), (130, 12, 264, 136, 2), (200, 8, 1540, 48, 4), (90, 2, 192, 224, 1),
                                                          (200, 9, 256, 640, 4)])
def test_experts_on_each_kernel(rows, experts, width, inner, top, kernels, monkeypatch):
    for name, value in KERNELS[kernels].items():
        monkeypatch.setattr(mx4, name, value)
    h, chosen, weights, up, down = expert_case(80 + rows, rows, experts, width, inner, top)
    if experts > top:
        chosen[: rows * 3 // 4][chosen[: rows * 3 // 4] == experts - 1] = 0      # few rows for one of them
    check_experts(h, chosen, weights, up, down)
    check_experts(*expert_case(81 + rows, rows, experts, width, inner, top, gated=False), "gelu_tanh", gated=False)


@pytest.mark.parametrize("rows,four", [(3, False), (3, True), (200, False), (200, True)])
def test_products_on_the_other_kernel(rows, four, monkeypatch):
    monkeypatch.setattr(mx4, "MX4_FEW_ROWS", 1000 if rows > 64 else 0)
    monkeypatch.setattr(mx4, "MX4_FEW_ROWS_OF_SMALL", 0)
    x, (matrix, w) = rows_of(rows, rows, 520), random_matrix(90, 330, 520)
    check_linear(ops.quantize_mx4(x) if four else x, matrix, w)


@pytest.mark.parametrize("rows", [5, 100])
@pytest.mark.parametrize("name,gated,param", [("silu", True, 0.0), ("gelu_tanh", True, 0.0), ("swiglu_clamp", True, 1.5), ("relu2", False, 0.0), ("gelu_tanh", False, 0.0)])
def test_activations_of_experts(rows, name, gated, param):
    check_experts(*expert_case(50, rows, 4, 160, 96, 2, gated), name, gated, param)


@pytest.mark.parametrize("rows", [6, 200])
def test_experts_chosen_twice_by_nobody_and_outside(rows):
    h, chosen, weights, up, down = expert_case(60, rows, 6, 128, 64, 3)
    chosen[0] = 2                                             # three times the same
    chosen[1] = torch.tensor([-1, 6, 1000], dtype=torch.int32)
    chosen[2:, 0] = 5
    chosen[chosen == 4] = -1                                  # nobody's
    got = check_experts(h, chosen, weights, up, down)
    assert (got[1] == 0).all()
    everywhere = torch.full_like(chosen, -1)
    assert (check_experts(h, everywhere, weights, up, down) == 0).all()


@pytest.mark.parametrize("kernels", KERNELS)
@pytest.mark.parametrize("rows,experts,width,inner,top", [(40, 24, 136, 72, 20), (90, 5, 192, 96, 17), (300, 3, 256, 128, 33)])
def test_many_choices_on_each_kernel_some_outside_and_some_twice(rows, experts, width, inner, top, kernels, monkeypatch):
    for name, value in KERNELS[kernels].items():
        monkeypatch.setattr(mx4, name, value)
    g = generator(71)
    h, weights = torch.randn(rows, width, generator=g).bfloat16().cuda(), torch.rand(rows, top, generator=g).cuda()
    chosen = torch.randint(-2, experts + 2, (rows, top), generator=g, dtype=torch.int32).cuda()
    chosen[rows // 2] = -1
    check_experts(h, chosen, weights, random_matrix(72, experts, 2 * inner, width, low=116, high=122), random_matrix(73, experts, width, inner, low=116, high=122))


def test_more_tiles_of_experts_than_a_grid_is_high():
    rows, experts, width, inner = 270_000, 64, 128, 64
    h = torch.randn(rows, width, generator=generator(61)).bfloat16().cuda()
    chosen = torch.randint(0, experts, (rows, 2), generator=generator(62), dtype=torch.int32).cuda()
    weights = torch.rand(rows, 2, generator=generator(63)).cuda()
    (up, _), (down, _), error = random_matrix(64, experts, 2 * inner, width), random_matrix(65, experts, width, inner), word()
    got = ops.chosen_experts_mx4(h, chosen, weights, up, down, "silu", error)
    for some in (slice(0, 500), slice(rows // 2, rows // 2 + 500), slice(rows - 500, rows)):
        assert torch.equal(got[some], ops.chosen_experts_mx4(h[some], chosen[some], weights[some], up, down, "silu", error))
    ops.raise_on_error_word(error)


def test_experts_of_no_rows_and_of_no_choice():
    h, chosen, weights, up, down = expert_case(61, 0, 4, 64, 32, 2)
    assert ops.chosen_experts_mx4(h, chosen, weights, up[0], down[0], "silu", word()).shape == (0, 64)
    h, chosen, weights, up, down = expert_case(62, 5, 4, 64, 32, 2)
    assert (ops.chosen_experts_mx4(h, chosen[:, :0].contiguous(), weights[:, :0].contiguous(), up[0], down[0], "silu", word()) == 0).all()


@pytest.mark.parametrize("rows", [7, 180])
def test_a_row_that_is_not_finite_spoils_itself_alone(rows):
    h, chosen, weights, up, down = expert_case(63, rows, 4, 128, 64, 2)
    clean = ops.chosen_experts_mx4(h, chosen, weights, up[0], down[0], "silu", word())
    h[3, 9] = math.nan
    got = ops.chosen_experts_mx4(h, chosen, weights, up[0], down[0], "silu", word())
    assert got[3].isnan().all()
    keep = torch.arange(rows, device="cuda") != 3
    assert torch.equal(got[keep], clean[keep])


def test_what_experts_refuse():
    h, chosen, weights, up, down = expert_case(64, 5, 4, 128, 64, 2)
    call = lambda **o: ops.chosen_experts_mx4(*[o.get(k, v) for k, v in dict(h=h, chosen=chosen, weights=weights, up=up[0], down=down[0], name="silu").items()], word(),
                                              gated=o.get("gated", True))
    for wrong in (dict(h=h.float()), dict(chosen=chosen.long()), dict(weights=weights.double()), dict(weights=weights[:, :1].contiguous()), dict(chosen=chosen[:4]),
                  dict(up=down[0]), dict(gated=False), dict(name="none"), dict(h=h[:, :64].contiguous()), dict(up=random_matrix(1, 128, 128)[0])):
        with pytest.raises(ops.KernelError):
            call(**wrong)


# ------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("rows", [2, 90])
def test_a_layer_of_experts_in_four_bits(rows):
    """Weights quantised at load, a router in groups, the chosen experts, a shared product of two four-bit operands; eager and captured."""
    width, inner, experts = 192, 96, 16
    up_weights, down_weights = rows_of(70, experts, 2 * inner, width) * 0.1, rows_of(71, experts, width, inner) * 0.1
    shared_weight, router, bias = rows_of(72, width, width) * 0.1, rows_of(73, experts, width) * 0.3, torch.randn(experts, generator=generator(74)).cuda() * 0.1
    up, down, shared = (ops.quantize_mx4(w.contiguous()) for w in (up_weights, down_weights, shared_weight))
    error, h = word(), rows_of(75, rows, width)

    def layer():
        logits = ops.linear(h, router, out_dtype=torch.float32, error_word=error)
        chosen, weights = ops.choose_experts(logits, 4, True, scoring="sigmoid", choice_bias=bias, groups=4, top_groups=2, group_best=2)
        out = ops.chosen_experts_mx4(h, chosen, weights, up, down, "silu", error)
        return logits, chosen, weights, out, ops.linear_mx4(ops.quantize_mx4(h), shared, error, out_dtype=torch.float32)

    def check(results):
        logits, chosen, weights, out, side = results
        ops.raise_on_error_word(error)
        want, w = pm.choose(logits, 4, 4, 2, 2, "sigmoid", bias, True)
        assert torch.equal(chosen.cpu(), want)
        result, room = pm.experts(h, chosen, weights, pm.values(*pm.quantize(up_weights)), pm.values(*pm.quantize(down_weights)), "silu")
        assert ((out.cpu().double() - result).abs() <= room + 1e-37).all()
        x, y = pm.values(*pm.quantize(h)), pm.values(*pm.quantize(shared_weight))
        assert ((side.cpu().double() - x @ y.T).abs() <= room_of(x, y, x @ y.T, torch.float32)).all()

    check(layer())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = layer()
    for seed in (76, 77):
        h.copy_(rows_of(seed, rows, width))
        graph.replay()
        torch.cuda.synchronize()
        check(results)


# ------------------------------------------------------------------------------------------- many steps on pairs
@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("rows,width,features", [(300, 4225, 15400), (257, 8192, 7700)])
def test_many_steps_and_more_tiles_than_pairs(rows, width, features, four):
    """Every stage and every place for scales is taken again many times, within a tile and from one to the next: the values, and the same bits
    beside other work."""
    g = torch.Generator("cuda").manual_seed(rows)
    x = (torch.randn(rows, width, generator=g, device="cuda") * torch.exp(torch.randn(width, generator=g, device="cuda"))).bfloat16()
    # every block with a scale of its own: one that is taken for another is off by powers of two
    size = torch.exp2(torch.randint(-8, 9, (features, -(-width // 32)), generator=g, device="cuda").float()).repeat_interleave(32, dim=1)[:, :width]
    matrix = ops.quantize_mx4(torch.randn(features, width, generator=g, device="cuda") * size)
    x = ops.quantize_mx4(x) if four else x
    error = word()
    got = ops.linear_mx4(x, matrix, error, out_dtype=torch.float32)
    rows_in_64, w = (ops.dequantize_mx4(x, torch.float32) if four else x).double(), ops.dequantize_mx4(matrix, torch.float32).double()
    want = rows_in_64 @ w.T
    assert ((got.double() - want).abs() <= room_of(rows_in_64, w, want, torch.float32)).all()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    results = []
    for stream in streams:
        with torch.cuda.stream(stream):
            results += [ops.linear_mx4(x, matrix, error, out_dtype=torch.float32) for _ in range(5)]
    torch.cuda.synchronize()
    ops.raise_on_error_word(error)
    assert all(torch.equal(got, r) for r in results)


# ------------------------------------------------------------------------------------------- what is not finite, through every activation
ACTIVATIONS = [("silu", True, 0.0), ("gelu_tanh", True, 0.0), ("swiglu_clamp", True, 1.5), ("relu2", True, 0.0), ("relu2", False, 0.0), ("silu", False, 0.0),
               ("gelu_tanh", False, 0.0), ("swiglu_clamp", False, 1.5)]


@pytest.mark.parametrize("kernels", KERNELS)
@pytest.mark.parametrize("name,gated,param", ACTIVATIONS)
def test_rows_that_are_not_finite_spoil_themselves_through_every_activation(name, gated, param, kernels, monkeypatch):
    for setting, value in KERNELS[kernels].items():
        monkeypatch.setattr(mx4, setting, value)
    h, chosen, weights, up, down = expert_case(66, 70, 4, 160, 96, 2, gated)
    call = lambda: ops.chosen_experts_mx4(h, chosen, weights, up[0], down[0], name, word(), gated=gated, activation_param=param)
    clean = call()
    spoilt = {3: math.nan, 11: math.inf, 40: -math.inf, 69: math.nan}
    for row, value in spoilt.items():
        h[row, 9 + row] = value
    got = call()
    rows = torch.zeros(70, dtype=torch.bool, device="cuda")
    rows[list(spoilt)] = True
    assert got[rows].isnan().all() and torch.equal(got[~rows], clean[~rows])


@pytest.mark.parametrize("kernels", KERNELS)
@pytest.mark.parametrize("name,gated,param", ACTIVATIONS)
def test_weights_that_are_not_numbers_spoil_the_rows_of_their_expert(name, gated, param, kernels, monkeypatch):
    for setting, value in KERNELS[kernels].items():
        monkeypatch.setattr(mx4, setting, value)
    h, chosen, weights, up, down = expert_case(67, 70, 4, 160, 96, 2, gated)
    call = lambda matrix: ops.chosen_experts_mx4(h, chosen, weights, matrix, down[0], name, word(), gated=gated, activation_param=param)
    clean = call(up[0])
    for row in ((5, 96 + 70) if gated else (5,)):             # a gate row, an up row
        scales = up[0].scales.clone()
        scales[2, row // 128, 0, (row % 32) * 16 + row % 128 // 32 * 4 + 1] = 255
        got, theirs = call(ops.Mx4(up[0].codes, scales, 160)), (chosen == 2).any(1)
        assert got[theirs].isnan().all() and torch.equal(got[~theirs], clean[~theirs])


# ------------------------------------------------------------------------------------------- scores where 32 bits say little
def test_choices_between_small_scores_that_a_small_bias_puts_in_order():
    """One logit 66 above two others: their scores, some 2e-29, are off by up to 7e-6 of themselves in 32 bits, and biases of 2e-6 of them decide."""
    g = generator(51)
    step = 2.0 ** -19
    most = 46 + torch.randint(0, 256, (600,), generator=g) * 2.0 ** -18
    second = -20 + torch.randint(0, 16, (600,), generator=g) * step
    third = second - torch.randint(0, 3, (600,), generator=g) * step
    logits = torch.stack([most, second, third, torch.full((600,), -40.0)], dim=1)
    bias = torch.tensor([0.0, 0.0, 2.2e-6 * math.exp(-66.0), 0.0])
    check_choice(logits.cuda(), dict(experts=4, top=3), bias.cuda())


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_groups_whose_scores_32_bits_do_not_hold(scoring):
    """A group's two best scores below the least 32-bit number add up to more than another's one above it."""
    logits = torch.full((40, 16), -200.0)
    logits[:, 4] = -88.71 + 0.001 * torch.arange(40)
    logits[:, 9], logits[:, 10] = -88.8, -88.9
    if scoring == "softmax":
        logits[:, 0] = 0.0
        logits[:, 4:12] -= 15.0
    check_choice(logits.cuda(), dict(experts=16, top=3, groups=4, top_groups=1 if scoring == "sigmoid" else 2, group_best=2, scoring=scoring), None)


@pytest.mark.parametrize("eps", [0.0, 1e-20])
@pytest.mark.parametrize("low", [-80.0, -88.0, -100.0, -300.0, -600.0])
def test_renormalised_weights_of_scores_that_32_bits_do_not_hold(low, eps):
    g = generator(53)
    logits = low + 2 * torch.randn(50, 32, generator=g)
    logits[25:, 7] = 1.0
    check_choice(logits.cuda(), dict(experts=32, top=4, renormalize=True, scoring="sigmoid", eps=eps, scale=2.5), None)
    # a bias that closes the one expert with a score to speak of
    bias = torch.zeros(32)
    bias[7] = -4.0
    logits[:, 7] = 1.0
    for scoring in ("softmax", "sigmoid"):
        check_choice(logits.cuda(), dict(experts=32, top=4, renormalize=True, scoring=scoring, eps=eps), bias.cuda())


@pytest.mark.parametrize("options", [dict(groups=2 ** 32 + 1), dict(groups=2 ** 32 + 2, top_groups=2 ** 32 + 1), dict(top_groups=2 ** 32 + 1), dict(group_best=2 ** 32 + 1),
                                     dict(top=2 ** 32 + 1), dict(top=2 ** 30), dict(groups=0), dict(top_groups=0), dict(groups=-1), dict(group_best=0)])
def test_numbers_that_32_bits_do_not_hold_are_refused(options):
    with pytest.raises(ops.KernelError):
        ops.choose_experts(torch.zeros(1, 8, device="cuda"), **{"top": 2, **options})


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("rows,width,features", [(1, 4096, 512), (16, 4096, 512), (17, 4096, 512), (48, 2100, 300), (64, 8192, 130), (65, 4096, 512), (200, 2048, 300)])
def test_a_row_does_not_depend_on_what_the_others_hold(rows, width, features, four):
    """K is cut into parts here; the same number of rows, all but one of them others (of other sizes, and not finite)."""
    x, matrix = rows_of(55, rows, width), random_matrix(56, features, width)[0]
    call = lambda x: ops.linear_mx4(ops.quantize_mx4(x) if four else x, matrix, word(), out_dtype=torch.float32)
    all_of_them = call(x)
    for keep in {0, rows // 2, rows - 1}:
        other = rows_of(57, rows, width) * 2.0 ** 30
        other[::3, 5], other[1::7, 9] = math.inf, math.nan
        other[keep] = x[keep]
        assert torch.equal(call(other)[keep], all_of_them[keep])


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,features", [(3, 129), (65, 7), (70, 33), (200, 129), (257, 199), (300, 1030), (290, 20001), (260, 196)])
def test_results_are_contiguous_whatever_their_sizes(rows, features, out_dtype, four):
    x, (matrix, w) = rows_of(58, rows, 200), random_matrix(59, features, 200)
    bias = torch.randn(features, generator=generator(60)).cuda()
    assert check_linear(ops.quantize_mx4(x) if four else x, matrix, w, bias, out_dtype).is_contiguous()


def test_a_product_feeds_the_experts_however_many_rows_there_are():
    _, chosen, weights, up, down = expert_case(68, 70, 4, 130, 64, 2)
    matrix, _ = random_matrix(69, 130, 96)
    for rows in (8, 70):
        h = ops.linear_mx4(rows_of(70, rows, 96) * 2.0 ** -8, matrix, word())
        check_experts(h, chosen[:rows], weights[:rows], up, down)


@pytest.mark.parametrize("kernels", KERNELS)
def test_a_thousand_experts_unevenly_loaded_on_each_kernel(kernels, monkeypatch):
    for setting, value in KERNELS[kernels].items():
        monkeypatch.setattr(mx4, setting, value)
    h, _, weights, up, down = expert_case(90, 700, 1000, 64, 32, 3)
    chosen = (torch.rand(700, 3, generator=generator(91)) ** 6 * 1000).int().cuda()        # some have a hundred rows, most none
    chosen[:5] = 999
    check_experts(h, chosen, weights, up, down)


@pytest.mark.parametrize("kernels", KERNELS)
def test_experts_give_the_same_bits_again_and_beside_other_work(kernels, monkeypatch):
    for setting, value in KERNELS[kernels].items():
        monkeypatch.setattr(mx4, setting, value)
    h, chosen, weights, up, down = expert_case(92, 300, 12, 264, 200, 3)
    error = word()
    call = lambda: ops.chosen_experts_mx4(h, chosen, weights, up[0], down[0], "silu", error)
    first = call()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    results = []
    for stream in streams:
        with torch.cuda.stream(stream):
            results += [call() for _ in range(4)]
    torch.cuda.synchronize()
    ops.raise_on_error_word(error)
    assert all(torch.equal(first, r) for r in results)


def test_a_matrix_quantised_right_ahead_of_its_product():
    """The product's early reads of the matrix come behind the kernel that makes it, eager and captured."""
    error = word()
    for rows in (1, 5, 40, 90):
        x, weights = rows_of(93, rows, 512), [rows_of(94 + i, 3000, 512) for i in range(3)]
        want = [ops.linear_mx4(x, ops.quantize_mx4(w), error) for w in weights]
        torch.cuda.synchronize()
        weight = weights[0].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            result = ops.linear_mx4(x, ops.quantize_mx4(weight), error)
        for _ in range(3):
            for w, y in zip(weights, want):
                weight.copy_(w)
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(result, y)
                matrix = ops.quantize_mx4(w)
                assert torch.equal(ops.linear_mx4(x, matrix, error), y)
                del matrix
    ops.raise_on_error_word(error)


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_every_scale_and_code_as_values(out):
    codes = torch.arange(16, dtype=torch.uint8).repeat(256, 2)
    scales = torch.arange(256, dtype=torch.uint8)[:, None].contiguous()
    want = pm.values(codes, scales)
    want = torch.where(want.abs() >= 2.0 ** 128, want.sign() * math.inf, want)
    got = ops.dequantize_mx4(ops.mx4_from_rows(pm.packed(codes).cuda(), scales.cuda()), out).cpu().double()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))
