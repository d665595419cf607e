"""Matrices in four bits: what is refused, and the plain implementation against itself (no GPU)."""
import pytest
import torch

import plain_mx4 as pm
from sglang_rs_b200 import ops


def host_mx4(rows=4, width=64, stack=None):
    lead = () if stack is None else (stack,)
    return ops.Mx4(torch.zeros((*lead, rows, 64 * -(-width // 128)), dtype=torch.uint8),
                   torch.zeros((*lead, -(-rows // 128), -(-width // 128), 512), dtype=torch.uint8), width)


def test_an_mx4_tells_its_sizes():
    q = host_mx4(130, 200, 3)
    assert q.shape == (3, 130, 200) and q.rows == 130 and q.matrices == 3
    assert host_mx4(5, 32).matrices is None and host_mx4(5, 32).shape == (5, 32)


@pytest.mark.parametrize("call", [
    lambda: ops.quantize_mx4(torch.zeros(2, 32)),
    lambda: ops.quantize_mx4(torch.zeros(1, 2, 32)),
    lambda: ops.dequantize_mx4(host_mx4()),
    lambda: ops.dequantize_mx4(torch.zeros(2, 2)),
    lambda: ops.linear_mx4(torch.zeros(2, 64, dtype=torch.bfloat16), host_mx4(), torch.zeros(1, dtype=torch.int32)),
    lambda: ops.linear_mx4(host_mx4(), host_mx4(), torch.zeros(1, dtype=torch.int32)),
    lambda: ops.choose_experts(torch.zeros(2, 8), 2),
    lambda: ops.chosen_experts_mx4(torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, 1),
                                   host_mx4(stack=2), host_mx4(stack=2), "silu", torch.zeros(1, dtype=torch.int32)),
    lambda: ops.mx4_from_rows(torch.zeros(2, 16, dtype=torch.uint8), torch.zeros(2, 1, dtype=torch.uint8)),
])
def test_host_tensors_are_refused(call):
    with pytest.raises(ops.KernelError):
        call()


def test_float32_rows_and_unknown_activations_are_refused_by_name():
    word = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ops.KernelError, match="float32 rows"):
        ops.linear_mx4(torch.zeros(2, 64), host_mx4(), word)
    with pytest.raises(ops.KernelError, match="float32 or bfloat16"):
        ops.dtype_code(torch.float16)


def test_plain_quantization_keeps_what_the_format_holds():
    codes = torch.arange(16, dtype=torch.uint8).repeat(4)[None]
    scales = torch.tensor([[120, 131]], dtype=torch.uint8)
    again, same = pm.quantize(pm.values(codes, scales))
    assert torch.equal(same, scales) and torch.equal(pm.values(again, same), pm.values(codes, scales))


def test_plain_quantization_rounds_ties_to_the_even_mantissa():
    # with 4 in the block the scale is 1
    block = torch.zeros(32)
    block[:9] = torch.tensor([4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.75])
    codes, scales = pm.quantize(block[None])
    assert scales.item() == 127
    assert pm.values(codes, scales)[0, :9].tolist() == [4.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, -1.0]
