"""The serving operators at the edges of what they take, and with values that are not finite where a query sees them."""
import math

import numpy as np
import pytest
import torch

from tensorlisp_b200 import device_ops as ops

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def room(n):
    return torch.full((max(int(n), 16),), 0xCD, dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("dtype,first", [(torch.float32, 0), (torch.bfloat16, 0), (torch.float16, 3)], ids=["f32", "bf16", "f16"])
def test_the_largest_vocabulary(native, dtype, first):
    """All but four logits are 60 below or more: their part in the sums, 2^31 e^-60 < 2^-55, is nothing, so the results are those of the four
    alone, to the accuracy of a sum of four (exponents and logarithm: 2^-20)."""
    vocab = 2 ** 31 - 2048
    memory = torch.full((vocab + first,), -57.0, dtype=dtype, device="cuda")
    x = memory[first:].unsqueeze(0)
    at, value = [5, 2 ** 30 + 1, vocab - 600, vocab - 1], [3.0, 2.5, 2.0, 3.0]
    for i, y in zip(at, value):
        x[0, i] = y
    lp, ent, ids, top = torch.zeros(1, device="cuda"), torch.zeros(1, device="cuda"), torch.zeros((1, 4), dtype=torch.int32, device="cuda"), torch.zeros((1, 4), device="cuda")
    ops.token_logprobs(native, x, i32([vocab - 1]), lp, ent, ids, top, workspace=room(ops.token_logprobs_workspace(native, x, 4)), stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    lse = math.log(sum(math.exp(y) for y in value))
    want = sorted((lse - y, i) for i, y in zip(at, value))
    assert ids.tolist() == [[i for _, i in want]]
    assert abs(lp.item() - (3.0 - lse)) < 2.0 ** -20 and abs(ent.item() - sum(math.exp(-d) * d for d, _ in want)) < 2.0 ** -19
    assert np.abs(top.cpu().numpy()[0] + [d for d, _ in want]).max() < 2.0 ** -20
