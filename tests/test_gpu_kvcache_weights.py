"""Attention over the 8-bit cache against the formula in 64 bits, to the bits that its weights keep.

Tolerance, from the arithmetic, for an output sum_j w_j v_j / l:
* a weight is rounded to 11 bits, 2^-11 of it at most (below 2^-21 of the largest weight the step is fixed,
  2^-32 of the largest: nothing beside it), so 2^-11 sum |w_j v_j| / l;
* scores are fp32 sums of up to 128 exact products: off by some 2^-22 of sum |scale q k|, here below 2^8, which is
  2^-14 of a weight; the sums over keys in fp32 are off by less;
* the output's own rounding: 2^-11 (fp16) or 2^-8 (bf16) of it, 2^-25 where it is subnormal."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

kv = pytest.importorskip("mlbricks_b200.kvcache")


@pytest.fixture(autouse=True)
def _cuda(cuda_ok):
    torch.manual_seed(1)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype,half", [(torch.float16, 2.0**-11), (torch.bfloat16, 2.0**-8)])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("new", [1, 5, 130])  # both kernels
def test_weights_keep_eleven_bits(new, dim, dtype, half):
    heads, group, block, scale = 2, 4, 32, dim**-0.5
    lengths = [new, new + 1, new + 3, 200, 1500]
    counts = [-(-n // block) for n in lengths]
    blocks = sum(counts)
    order = torch.randperm(blocks, device="cuda").int()
    tables = torch.full((len(lengths), max(counts)), -1, dtype=torch.int32, device="cuda")
    for i, n in enumerate(counts):
        tables[i, :n] = order[sum(counts[:i]):sum(counts[:i]) + n]
    codes = [torch.randint(-127, 128, (blocks, heads, block, dim), dtype=torch.int8, device="cuda") for _ in "kv"]
    scales = [0.01 * torch.exp(0.5 * torch.randn(blocks, heads, device="cuda")) for _ in "kv"]
    pool = kv.KVPool(codes[0], scales[0], codes[1], scales[1])
    q = torch.randn(new * len(lengths), heads * group, dim, device="cuda").to(dtype)
    out = kv.attention(q, pool, tables, i32(lengths), i32([i * new for i in range(len(lengths) + 1)]))
    for i, n in enumerate(lengths):
        ids = tables[i, :counts[i]].long()
        k, v = ((c[ids].double() * s[ids].double()[..., None, None]).transpose(0, 1).reshape(heads, -1, dim)[:, :n]
                .repeat_interleave(group, 0) for c, s in zip(codes, scales))
        rows = q[i * new:(i + 1) * new].double().transpose(0, 1)
        assert (scale * rows.abs() @ k.abs().transpose(1, 2)).max() < 2.0**8
        score = scale * rows @ k.transpose(1, 2)
        hidden = torch.arange(n, device="cuda")[None] > torch.arange(n - new, n, device="cuda")[:, None]
        w = torch.softmax(score.masked_fill(hidden, -torch.inf), 2)
        want, size = w @ v, w @ v.abs()
        got = out[i * new:(i + 1) * new].double().transpose(0, 1)
        tol = (2.0**-11 + 2.0**-14) * size + 1.001 * half * want.abs() + 2.0**-25
        assert ((got - want).abs() <= tol).all(), (i, ((got - want).abs() / tol).max())
