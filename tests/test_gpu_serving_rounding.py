"""Attention of packed prompts and of drafts where rounding and values that are not finite show: the weights' rounding in numerator and
sum, rows that are cut between CTAs, rows whose scores are all infinite."""
import numpy as np
import pytest
import torch

from tensorlisp_b200 import device_ops as ops

pytestmark = pytest.mark.gpu
LN2 = 0.6931471805599453


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def room(n):
    return torch.full((max(int(n), 16),), 0xCD, dtype=torch.uint8, device="cuda")


def randn(shape, seed, dtype=torch.float16):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def packed(native, q, k, v, q_at, kv_at=None, scale=None):
    out = torch.full_like(q, 77.0)
    ws = room(ops.packed_attention_workspace(native, q, k, len(q_at) - 1))
    ops.packed_attention(native, q, k, v, i32(q_at), out, scale, kv_offsets=None if kv_at is None else i32(kv_at), workspace=ws, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    return out


def tree(native, q, k_pool, v_pool, tables, context, counts, parents, scale=None):
    out = torch.full_like(q, 77.0)
    ws = room(ops.tree_attention_workspace(native, q, k_pool, tables))
    ops.tree_attention(native, q, k_pool, v_pool, tables, context, counts, parents, out, scale, workspace=ws, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    return out


# ------------------------------------------------------------------------------------------------ weights of sum one
# With values of 1 a result is sum P / sum P of the same rounded weights: 1 up to the two sums' own errors. n <= 1000 weights in f32, either
# order: relative 2 n 2^-24 < 2^-13; a product's accumulator and 1 / l add a few 2^-23. The nearest values beside 1 lie 2^-11 (f16) and 2^-8 (bf16)
# below, so every result is 1 to the last bit. A sum of unrounded weights is off by up to 2^-8 in bf16.
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows,keys", [(1, 700), (16, 1000), (256, 900)])
def test_one_key_outweighs_the_others(native, rows, keys, D, dtype):
    """Every 64th key scores 0, one key up to 7.9 (base 2: less than the step at which the reference moves), the others -30."""
    H = 4
    q, k = torch.zeros((rows, H, D)), torch.zeros((keys, 1, D))
    x = torch.arange(rows * H).reshape(rows, H) % 253 if rows * H > 253 else (torch.arange(rows * H).reshape(rows, H) * 67 + 186) % 253
    q[:, :, 0], q[:, :, 1] = x / 32, 1
    k[:, 0, 1] = -30
    k[::64, 0, 1] = 0
    k[130, 0, 0], k[130, 0, 1] = 1, 0
    out = packed(native, q.to(dtype).cuda(), k.to(dtype).cuda(), torch.ones((keys, 1, D), dtype=dtype, device="cuda"), [0, rows], [0, keys], LN2)
    assert torch.equal(out, torch.ones_like(out)), "%d of %d values are not 1, the farthest %g" % ((out != 1).sum(), out.numel(), (out.float() - 1).abs().max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("spread", [1.0, 3.0, 8.0])
def test_weights_of_a_row_sum_to_one(native, spread, D, dtype):
    lens = [3, 40, 300, 657]
    q, k = randn((1000, 8, D), 1, torch.float32) * spread, randn((1000, 2, D), 2, torch.float32)
    out = packed(native, q.to(dtype), k.to(dtype), torch.ones((1000, 2, D), dtype=dtype, device="cuda"), [0] + list(np.cumsum(lens)))
    assert torch.equal(out, torch.ones_like(out)), "%d of %d values are not 1, the farthest %g" % ((out != 1).sum(), out.numel(), (out.float() - 1).abs().max())


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("spread", [1.0, 3.0, 8.0])
def test_weights_of_a_draft_sum_to_one(native, spread, D):
    ctx = [900, 17, 300]
    pages = 3 * 60
    q, kp = randn((3, 12, 8, D), 3, torch.float32) * spread, randn((pages, 2, 16, D), 4)
    parents = i32(np.arange(12)[None, :].repeat(3, 0) - 1)
    out = tree(native, q.half(), kp, torch.ones_like(kp), i32(np.random.default_rng(5).permutation(pages).reshape(3, 60)), i32(ctx), i32([12, 12, 12]), parents)
    assert torch.equal(out, torch.ones_like(out)), "%d of %d values are not 1, the farthest %g" % ((out != 1).sum(), out.numel(), (out.float() - 1).abs().max())
