"""The 4-bit cache: appended bytes and gathered values against numpy bit for bit, attention against float64 within the
bounds that its roundings give."""
import itertools
import math

import numpy as np
import pytest
import torch

import int4_common as ic
from speech_serving import native

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def pools(blocks, bs, h, d, fill=0):
    return [torch.full(native.int4_pool_shape(blocks, bs, h, d), fill, dtype=torch.uint8, device="cuda") for _ in range(2)]


def rows(n, h, d, dtype, seed=0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(n, h, d, generator=g, device="cuda") * spread).to(dtype)


def written(k, v, at, blocks, bs, fill=0):
    """numpy pools after rows k, v went to the slots."""
    h, d = k.shape[1:]
    out = []
    for is_v, x in ((False, k), (True, v)):
        pool = np.full((blocks, h, bs // 16, 10 * d), fill, np.uint8)
        code, scale, low = ic.quantise(x.float().cpu().numpy())
        for i, slot in enumerate(at):
            if 0 <= slot < blocks * bs:
                for hh in range(h):
                    ic.write_row(pool, is_v, slot, hh, code[i, hh], scale[i, hh], low[i, hh])
        out.append(pool)
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,h,d,bs", [(1, 1, 32, 16), (40, 2, 64, 16), (21, 3, 128, 48), (65, 1, 128, 64)])
def test_append_bytes(cuda, dtype, n, h, d, bs):
    blocks = -(-(n + 9) // bs)
    k, v = rows(n, h, d, dtype, 1), rows(n, h, d, dtype, 2, 3.0)
    at = torch.randperm(blocks * bs, generator=torch.Generator().manual_seed(3))[:n].tolist()
    if n > 2:
        at[1], at[2] = -1, blocks * bs  # skipped
    kp, vp = pools(blocks, bs, h, d, 0xa5)
    native.append_int4(k, v, kp, vp, torch.tensor(at, device="cuda"))
    for got, want in zip((kp, vp), written(k, v, at, blocks, bs, 0xa5)):
        assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_order(cuda, dtype):
    """Consecutive slots (a prompt), one aligned quad, and the same rows in reverse order leave the same bytes."""
    n, h, d, bs = 53, 2, 64, 32
    k, v = rows(n, h, d, dtype, 1), rows(n, h, d, dtype, 2)
    at = list(range(3, 3 + n))
    want = written(k, v, at, 2, bs)
    for order in (list(range(n)), list(reversed(range(n))), list(range(1, n, 2)) + list(range(0, n, 2))):
        kp, vp = pools(2, bs, h, d)
        native.append_int4(k[order].contiguous(), v[order].contiguous(), kp, vp, torch.tensor(at, device="cuda")[order])
        assert np.array_equal(kp.cpu().numpy(), want[0]) and np.array_equal(vp.cpu().numpy(), want[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
def test_append_quads(cuda, dtype, d):
    """Four consecutive rows, each at its own place of one quad, at that place or another one of a quad elsewhere, or skipped, in
    all combinations (where one prompt ends and the next begins, some of them)."""
    at = []
    for i, kinds in enumerate(itertools.product(range(4), repeat=4)):
        for k, kind in enumerate(kinds):
            far = 1024 + 4 * (4 * i + k)
            at.append((4 * i + k, far + k, far + (k + 1) % 4, -1)[kind])
    n, bs, blocks = len(at), 64, 80
    k, v = rows(n, 1, d, dtype, 1), rows(n, 1, d, dtype, 2)
    kp, vp = pools(blocks, bs, 1, d, 0x5a)
    native.append_int4(k, v, kp, vp, torch.tensor(at, device="cuda"))
    for got, want in zip((kp, vp), written(k, v, at, blocks, bs, 0x5a)):
        assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("lens", [[55, 55, 55], [3, 3, 2, 7], [1, 2, 3, 1], [18, 21, 47]])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_append_prompts_side_by_side(cuda, d, lens):
    """Packed prompts of any length, each from position 0 of its own blocks on."""
    bs, width = 16, -(-max(lens) // 16)
    at = [(i * width) * bs + t for i, n in enumerate(lens) for t in range(n)]
    blocks = width * len(lens)
    k, v = rows(len(at), 2, d, torch.bfloat16, 1), rows(len(at), 2, d, torch.bfloat16, 2)
    kp, vp = pools(blocks, bs, 2, d)
    native.append_int4(k, v, kp, vp, torch.tensor(at, device="cuda"))
    for got, want in zip((kp, vp), written(k, v, at, blocks, bs)):
        assert np.array_equal(got.cpu().numpy(), want)


def test_append_extremes(cuda):
    """Constant groups, groups whose values tie between codes, tiny and huge ranges, infinities and NaN."""
    d = 64
    x = torch.zeros(8, 1, d)
    x[0] = 1.0001
    x[1, 0] = torch.arange(d) / 2.0
    x[2] = torch.rand(1, d) * 1e-7
    x[3] = torch.randn(1, d) * 1e30
    x[4, 0, 5], x[4, 0, 40] = math.inf, -math.inf
    x[5, 0, 7] = math.nan
    x[6] = -16384.0
    x[7, 0, ::2], x[7, 0, 1::2] = 16384.0, -16384.0
    for dtype in DTYPES:
        k = x.to("cuda", dtype)
        kp, vp = pools(1, 16, 1, d)
        at = list(range(8))
        native.append_int4(k, k, kp, vp, torch.tensor(at, device="cuda"))
        want = written(k, k, at, 1, 16)
        assert np.array_equal(kp.cpu().numpy(), want[0]) and np.array_equal(vp.cpu().numpy(), want[1])
        gk, gv = native.gather_int4(kp, vp, torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                                    torch.tensor([8], dtype=torch.int32, device="cuda"), 8, torch.float32)
        assert torch.isfinite(gk).all() and torch.isfinite(gv).all()


def test_append_every_scale(cuda):
    """Groups of every fp16 scale up to the greatest the cache takes, its codes' borders among the elements: what the kernel's
    reciprocal gives is what division gives."""
    scales = np.arange(1, 0x7c00, dtype=np.uint16).view(np.float16).astype(np.float32)
    scales = scales[scales <= 2184]
    n = -(-len(scales) // 8)
    scales = np.concatenate([scales, np.ones(n * 8 - len(scales), np.float32)])
    rng = np.random.default_rng(0)
    x = (rng.random((n * 8, 32), np.float32) * 15).astype(np.float32)
    x[:, 2:18] = np.arange(16) + np.where(np.arange(16) < 15, 0.5, 0)  # the borders between codes
    x[:, 0], x[:, 1] = 0, 15
    x = (x * scales[:, None] + rng.integers(-1, 2, (n * 8, 1)) * scales[:, None]).astype(np.float32).reshape(n, 8, 32)
    k = torch.from_numpy(x).cuda()
    blocks = -(-n // 16)
    kp, vp = pools(blocks, 16, 8, 32)
    native.append_int4(k, k, kp, vp, torch.arange(n, device="cuda"))
    code, scale, low = ic.quantise(x)
    want = torch.from_numpy(ic.values(code, scale, low)).float()
    table = torch.arange(blocks, dtype=torch.int32, device="cuda").view(1, -1)
    for got in native.gather_int4(kp, vp, table, torch.tensor([n], dtype=torch.int32, device="cuda"), n, torch.float32):
        assert torch.equal(got[0].transpose(0, 1).cpu(), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_many_groups(cuda, dtype):
    """262144 groups, enough for ranges next to a border between two fp16 scales: the product with 1 / 15 decides there."""
    n, h, d, bs = 16384, 8, 64, 64
    k, v = rows(n, h, d, dtype, 1), rows(n, h, d, dtype, 2, 30.0)
    kp, vp = pools(n // bs, bs, h, d)
    native.append_int4(k, v, kp, vp, torch.arange(n, device="cuda"))
    table = torch.arange(n // bs, dtype=torch.int32, device="cuda").view(1, -1)
    got = native.gather_int4(kp, vp, table, torch.tensor([n], dtype=torch.int32, device="cuda"), n, torch.float32)
    for x, y in zip(got, (k, v)):
        want = torch.from_numpy(ic.values(*ic.quantise(y.float().cpu().numpy()))).float()
        assert torch.equal(x[0].transpose(0, 1).cpu(), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("inter,rot", [(False, 128), (True, 128), (False, 32), (True, 16)])
def test_append_rotated(cuda, dtype, inter, rot):
    """The codes of rotated keys are those of append_rotary's rows; q and k come back as from it."""
    n, h, hkv, d, bs = 37, 4, 2, 128, 16
    q, k, v = rows(n, h, d, dtype, 1), rows(n, hkv, d, dtype, 2), rows(n, hkv, d, dtype, 3)
    table = native.rotary_table(300, rot)
    pos = torch.randint(0, 300, (n,), generator=torch.Generator().manual_seed(4)).cuda()
    at = torch.randperm(48, generator=torch.Generator().manual_seed(5))[:n].cuda()
    p16 = [torch.zeros(3, 16, hkv, d, device="cuda", dtype=dtype) for _ in range(2)]
    k16 = torch.empty_like(k)
    q16 = native.append_rotary(k, v, *p16, at, pos, table, q=q, k_out=k16, interleaved=inter)
    kp, vp = pools(3, bs, hkv, d)
    k4 = torch.empty_like(k)
    q4 = native.append_int4(k, v, kp, vp, at, pos, table, q=q, k_out=k4, interleaved=inter)
    assert torch.equal(q4, q16) and torch.equal(k4, k16)
    want = written(k16, v, at.tolist(), 3, bs)
    assert np.array_equal(kp.cpu().numpy(), want[0]) and np.array_equal(vp.cpu().numpy(), want[1])
    # in place, with a position outside the table
    pos[3] = 300
    native.append_int4(k, v, *pools(3, bs, hkv, d), at, pos, table, q=q, q_out=q, k_out=k, interleaved=inter)
    keep = torch.arange(n, device="cuda") != 3
    assert torch.equal(q[keep], q16[keep]) and torch.equal(k[keep], k16[keep])
    assert (q[3] == 0).all() and (k[3] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,bs,max_len", [(32, 16, 37), (64, 48, 96), (128, 16, 1), (64, 16, 30)])
def test_gather(cuda, dtype, d, bs, max_len):
    h, b = 2, 4
    width = -(-max_len // bs)
    blocks = b * width + 2
    g = torch.Generator().manual_seed(7)
    table = torch.randperm(blocks, generator=g)[:b * width].view(b, width).to(torch.int32)
    if width > 1:
        table[1, 0], table[2, 1] = -1, blocks
    lens = torch.tensor([max_len, max(1, max_len - 3), max_len // 2, 0], dtype=torch.int32)
    k, v = rows(blocks * bs, h, d, torch.float32, 8), rows(blocks * bs, h, d, torch.float32, 9)
    kp, vp = pools(blocks, bs, h, d)
    native.append_int4(k, v, kp, vp, torch.arange(blocks * bs, device="cuda"))
    gk, gv = native.gather_int4(kp, vp, table.cuda(), lens.cuda(), max_len, dtype)
    for got, x in ((gk, k), (gv, v)):
        val = torch.from_numpy(ic.values(*ic.quantise(x.cpu().numpy()))).to(torch.float32).to(dtype)  # [slots, h, d]
        want = torch.zeros(b, h, max_len, d, dtype=dtype)
        for r in range(b):
            for t in range(int(lens[r])):
                blk = int(table[r, t // bs])
                if 0 <= blk < blocks:
                    want[r, :, t] = val[blk * bs + t % bs]
        assert torch.equal(got.cpu(), want)


# ---------------------------------------------------------------------------
# Attention.
# ---------------------------------------------------------------------------
def filled(blocks, bs, h, d, seed=0, k_shift=0.0):
    """Random pools, and what they hold as float64 [slots, h, d] with scales and lows [slots, h, d / 32]."""
    n = blocks * bs
    k, v = rows(n, h, d, torch.float32, seed) + k_shift, rows(n, h, d, torch.float32, seed + 1, 2.0)
    kp, vp = pools(blocks, bs, h, d)
    native.append_int4(k, v, kp, vp, torch.arange(n, device="cuda"))
    held = []
    for x in (k, v):
        code, scale, low = ic.quantise(x.cpu().numpy())
        held.append([torch.from_numpy(a.astype(np.float64)).cuda() for a in (ic.values(code, scale, low), scale, low)])
    return kp, vp, held


def run_attention(b, qlen, heads, hkv, d, bs, lens, dtype, causal, chunk=0, scale=None, q_scale=1.0, bad=False, max_ctx=None,
                  trows=False):
    width = max(1, -(-max(lens + [1]) // bs))
    blocks = b * width + 2
    kp, vp, held = filled(blocks, bs, hkv, d)
    g = torch.Generator().manual_seed(11)
    table = torch.randperm(blocks, generator=g)[:b * width].view(b, width).to(torch.int32).cuda()
    if bad and width > 1:
        table[0, 1] = blocks + 3
        table[b - 1, 0] = -5
    q = rows(b * qlen, heads, d, dtype, 12, q_scale).view(b, qlen, heads, d)
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    cl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    order = torch.arange(b - 1, -1, -1, dtype=torch.int32, device="cuda") if trows else None
    max_ctx = width * bs if max_ctx is None else max_ctx
    out = native.paged_attention_int4(q if qlen > 1 else q[:, 0], kp, vp, table, cl, max_ctx, scale, causal=causal,
                                      table_rows=order, chunk_tokens=chunk).view(b, qlen, heads, d)
    for r in range(b):
        vis = torch.tensor([min(max(lens[r] - (qlen - 1 - i if causal else 0), 0), max_ctx) for i in range(qlen)],
                           device="cuda")
        ref, bound = ic.reference(q[r], held, table[b - 1 - r if trows else r], vis, bs, blocks, scale)
        err = (out[r].double() - ref).abs()
        assert (err <= bound).all(), (r, float((err - bound).max()), float(err.max()))
        assert (out[r][vis <= 0] == 0).all()
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,hkv,d,bs", [(4, 4, 64, 16), (8, 2, 128, 16), (3, 1, 32, 48), (20, 1, 64, 32), (32, 8, 128, 64)])
def test_attention_decode(cuda, dtype, heads, hkv, d, bs):
    run_attention(6, 1, heads, hkv, d, bs, [1, 0, 15, 16, 33, 250], dtype, False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("qlen,heads,hkv,d", [(2, 4, 4, 64), (5, 8, 2, 128), (17, 6, 2, 32), (40, 2, 2, 64)])
def test_attention_several_queries(cuda, dtype, causal, qlen, heads, hkv, d):
    run_attention(4, qlen, heads, hkv, d, 16, [qlen, 3, 100, 0], dtype, causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("chunk", [64, 128, 320])
def test_attention_split_keys(cuda, dtype, chunk):
    """Rows of one, several and partly filled chunks in one call."""
    run_attention(4, 3, 8, 4, 64, 16, [700, 64, 65, 1], dtype, True, chunk=chunk)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_invalid_blocks_and_table_rows(cuda, dtype):
    run_attention(3, 2, 4, 2, 64, 16, [100, 40, 33], dtype, True, bad=True)
    run_attention(3, 1, 4, 2, 128, 32, [100, 40, 70], dtype, False, bad=True, chunk=64, trows=True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_lengths_past_the_table(cuda, dtype):
    """Lengths beyond max_ctx count as max_ctx."""
    run_attention(2, 1, 4, 4, 64, 16, [50, 20], dtype, False, max_ctx=30)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, -0.125, 1.0])
def test_attention_scales(cuda, dtype, scale):
    run_attention(2, 2, 4, 2, 64, 16, [90, 31], dtype, True, scale=scale)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("q_scale", [0.0, 1e-4, 3000.0])
def test_attention_query_sizes(cuda, dtype, q_scale):
    run_attention(2, 1, 4, 2, 64, 16, [90, 31], dtype, False, q_scale=q_scale, scale=1.0 / (8 * max(q_scale, 1.0)))


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_scale_zero_and_tiny_queries(cuda, dtype):
    """Keys past a row's end stay out when scale and queries together leave fp32's range below: the mean of the values."""
    tiny = 2.0 ** -100 if dtype == torch.bfloat16 else 2.0 ** -14
    run_attention(3, 2, 4, 2, 64, 16, [90, 31, 1], dtype, True, scale=0.0, q_scale=tiny)
    run_attention(3, 1, 4, 2, 64, 16, [90, 31, 0], dtype, False, scale=1e-30, q_scale=tiny)


def test_attention_long_row(cuda):
    run_attention(1, 1, 8, 2, 128, 16, [9001], torch.bfloat16, False)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_ignores_what_no_query_sees(cuda, dtype):
    """Slots past a row's end and blocks that no table names may hold anything, NaN scales among it."""
    bs, h, d = 16, 2, 64
    kp, vp, held = filled(4, bs, h, d)
    table = torch.tensor([[2, 1]], dtype=torch.int32, device="cuda")
    q = rows(1, 4, d, dtype, 3)
    lens = torch.tensor([21], dtype=torch.int32, device="cuda")
    want = native.paged_attention_int4(q, kp, vp, table, lens, 32, 0.125)
    keep = {(2, t) for t in range(16)} | {(1, t) for t in range(5)}
    k_np, v_np = kp.cpu().numpy(), vp.cpu().numpy()
    wild = [np.full_like(k_np, 0xff), np.full_like(v_np, 0xff)]  # scales and lows of NaN
    for is_v, src, dst in ((False, k_np, wild[0]), (True, v_np, wild[1])):
        for blk, t in keep:
            for hh in range(h):
                ic.write_row(dst, is_v, blk * bs + t, hh, *ic.read_row(src, is_v, blk * bs + t, hh))
    got = native.paged_attention_int4(q, *(torch.from_numpy(w).cuda() for w in wild), table, lens, 32, 0.125)
    assert torch.equal(got, want)


def test_attention_strides_and_out(cuda):
    """Slices of a fused projection as q, an out of its own strides, and a call repeated bit for bit."""
    b, h, hkv, d, bs = 5, 8, 2, 128, 16
    kp, vp, _ = filled(20, bs, hkv, d)
    table = torch.randperm(20)[:b * 4].view(b, 4).to(torch.int32).cuda()
    lens = torch.tensor([64, 1, 17, 50, 33], dtype=torch.int32, device="cuda")
    fused = rows(b, h + 2 * hkv, d, torch.bfloat16, 3)
    want = native.paged_attention_int4(fused[:, :h].contiguous(), kp, vp, table, lens, 64, 0.1)
    wide = torch.full((b, h, 2 * d), 3.0, device="cuda", dtype=torch.bfloat16)
    got = native.paged_attention_int4(fused[:, :h], kp, vp, table, lens, 64, 0.1, out=wide[..., :d])
    assert torch.equal(got, want) and (wide[..., d:] == 3).all()
    wide_table = torch.zeros(b, 9, dtype=torch.int32, device="cuda")
    wide_table[:, :4] = table
    assert torch.equal(native.paged_attention_int4(fused[:, :h], kp, vp, wide_table, lens, 64, 0.1), want)
