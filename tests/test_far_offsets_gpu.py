"""Offsets past 32 bits: pools and rows of more than 4 GiB, of which the calls touch the ends."""
import math

import pytest
import torch

import int4_common as ic
from speech_serving import native

pytestmark = pytest.mark.gpu
D = 64
SCALE = 1 / math.sqrt(D)


def rows(n, h, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(n, h, D, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_far_blocks_of_a_4_bit_pool(cuda, dtype):
    h, bs = 64, 64
    blocks = (1 << 32) // (h * bs * 40) + 5
    pools = [torch.zeros(native.int4_pool_shape(blocks, bs, h, D), dtype=torch.uint8, device="cuda") for _ in range(2)]
    assert pools[0].numel() > 1 << 32
    n = 70
    k, v, q = rows(n, h, dtype, 1), rows(n, h, dtype, 2), rows(1, h, dtype, 3)
    table = torch.tensor([[blocks - 1, blocks - 2]], dtype=torch.int32, device="cuda")
    pos = torch.arange(n, device="cuda")
    native.append_int4(k, v, *pools, table.long()[0, pos // bs] * bs + pos % bs)
    near = [torch.zeros(native.int4_pool_shape(2, bs, h, D), dtype=torch.uint8, device="cuda") for _ in range(2)]
    native.append_int4(k, v, *near, pos)
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    near_table = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    for a, b in zip(native.gather_int4(*pools, table, lens, n, dtype), native.gather_int4(*near, near_table, lens, n, dtype)):
        assert torch.equal(a, b) and bool((a != 0).any())
    got = native.paged_attention_int4(q, *pools, table, lens, 128, SCALE)
    assert torch.equal(got, native.paged_attention_int4(q, *near, near_table, lens, 128, SCALE))
    assert int(torch.count_nonzero(pools[0][:blocks - 2])) == 0


def test_far_slots_of_a_16_bit_pool(cuda):
    h, bs, dtype = 64, 64, torch.bfloat16
    blocks = (1 << 32) // (h * bs * D * 2) + 3
    pools = [torch.zeros(blocks, bs, h, D, dtype=dtype, device="cuda") for _ in range(2)]
    table = native.rotary_table(64, D)
    k, v = rows(5, h, dtype, 1), rows(5, h, dtype, 2)
    k_out = torch.empty_like(k)
    at = torch.arange(blocks * bs - 5, blocks * bs, device="cuda")
    native.append_rotary(k, v, *pools, at, torch.arange(5, device="cuda"), table, k_out=k_out)
    assert torch.equal(pools[0].view(-1, h, D)[-5:], k_out) and torch.equal(pools[1].view(-1, h, D)[-5:], v)
    assert int(torch.count_nonzero(pools[0].view(-1, h, D)[:-5])) == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_far_rows_of_a_prompt(cuda, dtype):
    """Rows 256 KiB apart: the last sequence starts past 4 GiB."""
    lens = [16000, 700]
    n, wide = sum(lens), (256 << 10) // torch.finfo(dtype).bits * 8
    base = torch.zeros(n, wide, dtype=dtype, device="cuda")
    q, k, v = (base[:, i * D:(i + 1) * D].unflatten(1, (1, D)) for i in range(3))
    for i, x in enumerate((q, k, v)):
        x.copy_(rows(n, 1, dtype, i))
    cu = torch.tensor([0, lens[0], n], dtype=torch.int32, device="cuda")
    out = base[:, 4 * D:5 * D].unflatten(1, (1, D))
    native.prompt_attention(q, k, v, cu, SCALE, out=out)
    want = native.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), cu, SCALE)
    assert torch.equal(out, want)
    vis = torch.arange(1, lens[1] + 1, device="cuda")
    ref = ic.attention64(*(x[lens[0]:, 0].double() for x in (q, k, v)), vis, SCALE)[0]
    # Values below 8: fp16 weights and result are half a step (2^-11) each; fp32 sums of 700 products, 2^-24 each.
    assert (out[lens[0]:, 0].double() - ref).abs().max() <= 8 * (2.0 ** -10 if dtype == torch.float16 else 700 * 2.0 ** -24)


def test_far_rows_of_an_append(cuda):
    """k, v and q rows 1 MiB apart, past 4 GiB in all."""
    n, h, dtype = 4200, 2, torch.float16
    base = torch.zeros(n, 1 << 19, dtype=dtype, device="cuda")
    q, k, v = (base[:, 2 * i * D:2 * (i + 1) * D].unflatten(1, (h, D)) for i in range(3))
    for i, x in enumerate((q, k, v)):
        x.copy_(rows(n, h, dtype, i))
    table = native.rotary_table(n, D)
    pos = torch.arange(n, device="cuda")
    shape = native.int4_pool_shape(-(-n // 16), 16, h, D)
    pools = [torch.zeros(shape, dtype=torch.uint8, device="cuda") for _ in range(4)]
    got = native.append_int4(k, v, pools[0], pools[1], pos, pos, table, q=q)
    want = native.append_int4(k.contiguous(), v.contiguous(), pools[2], pools[3], pos, pos, table, q=q.contiguous())
    assert torch.equal(got, want) and torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])
    p16 = [torch.zeros(-(-n // 16), 16, h, D, dtype=dtype, device="cuda") for _ in range(4)]
    got = native.append_rotary(k, v, p16[0], p16[1], pos, pos, table, q=q)
    want = native.append_rotary(k.contiguous(), v.contiguous(), p16[2], p16[3], pos, pos, table, q=q.contiguous())
    assert torch.equal(got, want) and torch.equal(p16[0], p16[2]) and torch.equal(p16[1], p16[3])
