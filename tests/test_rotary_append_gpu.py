"""append_rotary against float64: rotation to half a step, stored rows, skipped rows, layouts, in place."""
import numpy as np
import pytest
import torch

from int4_common import half_step, rotate64
from speech_serving import native

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
_TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def case(n, h, hkv, d, dtype, seed=0, positions=512, slots=None, fused=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, h + 2 * hkv, d, generator=g, device="cuda").to(dtype)
    q, k, v = x[:, :h], x[:, h:h + hkv], x[:, h + hkv:]
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    pos = torch.randint(0, positions, (n,), generator=g, device="cuda")
    slots = slots or n + 5
    at = torch.randperm(slots, generator=g, device="cuda")[:n].contiguous()
    return q, k, v, pos, at


def check_rows(got, x, table, pos, interleaved, dtype):
    """Each element is the float64 rotation rounded: half a step of the type, plus three fp32 roundings (2^-24 each) of the
    products and their sum."""
    ref, mag = rotate64(x, table, pos, interleaved)
    bound = half_step(dtype) * ref.abs() + 4 * 2.0 ** -24 * mag + _TINY[dtype]
    assert ((got.double() - ref).abs() <= bound).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,h,hkv,d,rot,inter", [
    (1, 4, 4, 64, 64, False), (7, 8, 2, 128, 128, False), (64, 12, 4, 64, 32, True), (33, 3, 1, 32, 16, False),
    (5, 2, 2, 16, 16, True), (130, 20, 20, 64, 64, True), (19, 4, 2, 96, 48, False), (3, 2, 1, 256, 64, False)])
def test_rotated_rows(cuda, dtype, n, h, hkv, d, rot, inter):
    q, k, v, pos, at = case(n, h, hkv, d, dtype)
    table = native.rotary_table(512, rot)
    bs = 3
    blocks = -(-(n + 5) // bs)
    kp, vp = (torch.full((blocks, bs, hkv, d), 7.0, device="cuda", dtype=dtype) for _ in range(2))
    k_out = torch.empty(n, hkv, d, device="cuda", dtype=dtype)
    q_out = native.append_rotary(k, v, kp, vp, at, pos, table, q=q, k_out=k_out, interleaved=inter)
    check_rows(q_out, q, table, pos, inter, dtype)
    check_rows(k_out, k, table, pos, inter, dtype)
    flat_k, flat_v = kp.view(-1, hkv, d), vp.view(-1, hkv, d)
    assert torch.equal(flat_k[at], k_out) and torch.equal(flat_v[at], v)
    rest = torch.ones(flat_k.shape[0], dtype=torch.bool, device="cuda")
    rest[at] = False
    assert (flat_k[rest] == 7).all() and (flat_v[rest] == 7).all()  # slots that no row names


@pytest.mark.parametrize("dtype", DTYPES)
def test_in_place_and_without_q(cuda, dtype):
    n, h, hkv, d = 50, 6, 3, 64
    table = native.rotary_table(512, d)
    q, k, v, pos, at = case(n, h, hkv, d, dtype)
    pools = [torch.zeros(4, 16, hkv, d, device="cuda", dtype=dtype) for _ in range(4)]
    want_k = torch.empty(n, hkv, d, device="cuda", dtype=dtype)
    want_q = native.append_rotary(k, v, pools[0], pools[1], at, pos, table, q=q, k_out=want_k)
    got = native.append_rotary(k, v, pools[2], pools[3], at, pos, table, q=q, q_out=q, k_out=k)
    assert got is q and torch.equal(q, want_q) and torch.equal(k, want_k)
    assert torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])
    q, k, v, pos, at = case(n, h, hkv, d, dtype)
    pools[2].zero_(), pools[3].zero_()
    assert native.append_rotary(k, v, pools[2], pools[3], at, pos, table) is None
    assert torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])


def test_skipped_rows(cuda):
    """A slot outside the pool skips the store, a position outside the table as well and leaves zeros."""
    n, h, hkv, d, dtype = 6, 2, 2, 64, torch.float16
    q, k, v, pos, at = case(n, h, hkv, d, dtype)
    table = native.rotary_table(100, d)
    pos = torch.tensor([0, 99, 100, -1, 5, 6], device="cuda")
    at = torch.tensor([0, 1, 2, 3, -1, 64], device="cuda")
    kp, vp = (torch.full((4, 16, hkv, d), 9.0, device="cuda", dtype=dtype) for _ in range(2))
    k_out = torch.full((n, hkv, d), 5.0, device="cuda", dtype=dtype)
    q_out = native.append_rotary(k, v, kp, vp, at, pos, table, q=q, k_out=k_out)
    ok = torch.tensor([0, 1, 4, 5], device="cuda")
    check_rows(q_out[ok], q[ok], table, pos[ok], False, dtype)
    check_rows(k_out[ok], k[ok], table, pos[ok], False, dtype)
    assert (q_out[2:4] == 0).all() and (k_out[2:4] == 0).all()
    flat_k, flat_v = kp.view(-1, hkv, d), vp.view(-1, hkv, d)
    assert torch.equal(flat_k[:2], k_out[:2]) and torch.equal(flat_v[:2], v[:2])
    assert (flat_k[2:] == 9).all() and (flat_v[2:] == 9).all()


def test_layouts(cuda):
    """Head-major rows, rows broadcast from one, an unaligned view (copied) and outputs at strides of their own."""
    n, h, hkv, d, dtype = 11, 4, 2, 64, torch.bfloat16
    q, k, v, pos, at = case(n, h, hkv, d, dtype)
    table = native.rotary_table(512, d)
    pools = [torch.zeros(1, 16, hkv, d, device="cuda", dtype=dtype) for _ in range(4)]
    want = native.append_rotary(k, v, pools[0], pools[1], at, pos, table, q=q)
    qh = q.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.empty(n * hkv * d + 1, device="cuda", dtype=dtype)[1:].view(n, hkv, d).copy_(k)
    wide = torch.zeros(n, 2 * h, d, device="cuda", dtype=dtype)
    got = native.append_rotary(odd, v, pools[2], pools[3], at, pos, table, q=qh, q_out=wide[:, ::2])
    assert torch.equal(got, want) and (wide[:, 1::2] == 0).all()
    assert torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])
    one = k[:1].expand(n, hkv, d)
    native.append_rotary(one, v, pools[2], pools[3], at, pos, table)
    native.append_rotary(one.contiguous(), v, pools[0], pools[1], at, pos, table)
    assert torch.equal(pools[0], pools[2])


def test_far_positions(cuda):
    """The table's angles are those of float64: at position 131071 a float32 angle would be off by 4e-3."""
    table = native.rotary_table(131072, 64)
    freq = 10000.0 ** (-np.arange(0, 64, 2) / 64.0)
    for p in (0, 1, 4095, 131071):
        ang = p * freq
        want = np.concatenate([np.cos(ang), np.sin(ang)])
        # one rounding to float32, and 131071 * 2^-52 of the product before the cosine
        assert np.abs(table[p].cpu().numpy() - want).max() <= 2.0 ** -24 + 131071 * 2.0 ** -51


@pytest.mark.parametrize("int4", [False, True])
def test_no_tokens(cuda, int4):
    e = torch.empty(0, 2, 64, device="cuda", dtype=torch.float16)
    i = torch.empty(0, dtype=torch.int64, device="cuda")
    table = native.rotary_table(8, 64)
    if int4:
        pools = [torch.zeros(native.int4_pool_shape(1, 16, 2, 64), dtype=torch.uint8, device="cuda") for _ in range(2)]
        assert native.append_int4(e, e, *pools, i, i, table, q=e).shape == (0, 2, 64)
        native.append_int4(e, e, *pools, i)
    else:
        pools = [torch.zeros(1, 16, 2, 64, dtype=torch.float16, device="cuda") for _ in range(2)]
        assert native.append_rotary(e, e, *pools, i, i, table, q=e).shape == (0, 2, 64)
    torch.cuda.synchronize()
