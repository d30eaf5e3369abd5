"""prompt_attention against float64: packed lengths, grouped heads, types, layouts, and what later keys may hold."""
import math

import pytest
import torch

import int4_common as ic
from speech_serving import native

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def inputs(n, h, hkv, d, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, h + 2 * hkv, d, generator=g, device="cuda").to(dtype)
    return x[:, :h], x[:, h:h + hkv], x[:, h + hkv:]


def cumulative(lens):
    return torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)


def reference(q, k, v, lens, scale):
    """(out, bound) float64 [N, H, D]. Bound: the weights' rounding to the rows' type (half a step of each, none in fp32), the
    result's, and fp32 sums of D products in the scores."""
    out, bound = (torch.zeros(q.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    half = ic.half_step(q.dtype)
    group = q.shape[1] // k.shape[1]
    at, d = 0, q.shape[2]
    for n in lens:
        vis = torch.arange(1, n + 1, device="cuda")
        for h in range(q.shape[1] if n else 0):
            qq, kk, vv = (x[at:at + n, hh].double() for x, hh in ((q, h), (k, h // group), (v, h // group)))
            o, w, s = ic.attention64(qq, kk, vv, vis, scale)
            ds = abs(scale) * (d + 8) * 2.0 ** -24 * (qq.abs() @ kk.abs().T) + 2.0 ** -21 * s.abs() + 2.0 ** -21
            ds = torch.where(w > 0, ds, torch.zeros_like(ds)).amax(-1, keepdim=True)
            absw = w @ vv.abs()
            weights = 0.0 if q.dtype == torch.float32 else half
            out[at:at + n, h] = o
            bound[at:at + n, h] = (weights + torch.expm1(2 * ds) + 2.0 ** -20) * (absw + o.abs()) + half * o.abs() + 2.0 ** -25
        at += n
    return out, bound


def check(got, q, k, v, lens, scale):
    ref, bound = reference(q, k, v, lens, scale)
    n = sum(lens)
    err = (got[:n].double() - ref[:n]).abs()
    assert (err <= bound[:n]).all(), (float((err - bound[:n]).max()), float(err.max()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens", [[1], [0, 5, 0], [64], [65, 63, 128, 1], [300, 2, 129], [31, 33, 32, 95, 97]])
@pytest.mark.parametrize("h,hkv,d", [(4, 4, 64), (8, 2, 128), (3, 1, 32), (2, 2, 16)])
def test_lengths_and_heads(cuda, dtype, lens, h, hkv, d):
    q, k, v = inputs(sum(lens), h, hkv, d, dtype)
    out = native.prompt_attention(q, k, v, cumulative(lens), 1 / math.sqrt(d))
    check(out, q, k, v, lens, 1 / math.sqrt(d))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
def test_long(cuda, dtype, d):
    lens = [1500, 777] if dtype == torch.float32 else [2500, 1030]
    q, k, v = inputs(sum(lens), 2, 1, d, dtype)
    out = native.prompt_attention(q, k, v, cumulative(lens), 1 / math.sqrt(d))
    check(out, q, k, v, lens, 1 / math.sqrt(d))


def test_many_sequences(cuda):
    """More sequences than a wave has lanes, empty ones among them, 8 heads over the dies."""
    lens = [(7 * i) % 23 for i in range(150)] + [0, 0, 200]
    q, k, v = inputs(sum(lens), 8, 8, 64, torch.bfloat16)
    out = native.prompt_attention(q, k, v, cumulative(lens), 0.125)
    check(out, q, k, v, lens, 0.125)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("lens,h,hkv", [([1500, 417, 70], 40, 8), ([900, 417, 70], 32, 8), ([700, 30], 4, 2), ([20] * 70 + [333, 65], 4, 2)])
def test_forms(cuda, dtype, d, lens, h, hkv):
    """Many workgroups of long sequences, fewer, few, and short sequences beside a long one; then the same with a NaN row in the
    first long sequence, which only its later queries may see."""
    q, k, v = inputs(sum(lens), h, hkv, d, dtype)
    scale = 1 / math.sqrt(d)
    out = native.prompt_attention(q, k, v, cumulative(lens), scale)
    check(out, q, k, v, lens, scale)
    i = lens.index(max(lens))
    at, n, bad = sum(lens[:i]), lens[i], 3 * lens[i] // 5
    k2, v2 = k.clone(), v.clone()
    k2[at + bad, 0], v2[at + bad, -1, 5] = math.nan, math.inf
    got = native.prompt_attention(q, k2, v2, cumulative(lens), scale)
    first = slice(at, at + bad)
    check(got[first], q[first], k[first], v[first], [bad], scale)
    assert torch.equal(got[:at], out[:at]) and torch.equal(got[at + n:], out[at + n:])
    group = h // hkv
    assert torch.isnan(got[at + bad:at + n, :group]).all() and not torch.isfinite(got[at + bad:at + n, -group:, 5]).any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_thousands_of_sequences(cuda, dtype):
    """More groups of 64 sequences than a wave has lanes, empty sequences among them, long ones first, in between and last;
    against one float64 softmax under the sequences' mask, with reference()'s bound."""
    lens = [500] + [(7 * i) % 4 for i in range(2500)] + [260] + [(5 * i) % 3 for i in range(2500)] + [130]
    n, h, hkv, d, scale = sum(lens), 2, 1, 64, 0.125
    q, k, v = inputs(n, h, hkv, d, dtype)
    out = native.prompt_attention(q, k, v, cumulative(lens), scale)
    seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), torch.tensor(lens, device="cuda"))
    seen = (seq[:, None] == seq[None, :]).tril()
    kk, vv, half = k[:, 0].double(), v[:, 0].double(), ic.half_step(dtype)
    for i in range(h):
        qq = q[:, i].double()
        s = ((qq @ kk.T) * scale).masked_fill(~seen, -math.inf)
        w = torch.softmax(s, -1)
        ds = scale * (d + 8) * 2.0 ** -24 * (qq.abs() @ kk.abs().T) + 2.0 ** -21 * s.abs() + 2.0 ** -21
        ds = torch.where(seen, ds, torch.zeros_like(ds)).amax(-1, keepdim=True)
        o, absw = w @ vv, w @ vv.abs()
        weights = 0.0 if dtype == torch.float32 else half
        bound = (weights + torch.expm1(2 * ds) + 2.0 ** -20) * (absw + o.abs()) + half * o.abs() + 2.0 ** -25
        assert ((out[:, i].double() - o).abs() <= bound).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, -0.2, 2.0])
def test_scales(cuda, dtype, scale):
    q, k, v = inputs(150, 2, 2, 64, dtype)
    out = native.prompt_attention(q, k, v, cumulative([100, 50]), scale)
    check(out, q, k, v, [100, 50], scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_later_keys_may_hold_anything(cuda, dtype, d, bad):
    """A query's result depends on its own sequence's keys up to itself alone, whatever the others hold."""
    lens = [100, 90]
    q, k, v = inputs(sum(lens), 4, 2, d, dtype)
    want = native.prompt_attention(q, k, v, cumulative(lens), 0.1)
    k2, v2 = k.clone(), v.clone()
    k2[70], v2[70, :, 3] = bad, bad          # seen by queries 70.. of the first sequence
    v2[189, 0] = bad                         # the last row of all
    got = native.prompt_attention(q, k2, v2, cumulative(lens), 0.1)
    check(got[:70], q[:70], k[:70], v[:70], [70], 0.1)
    assert torch.equal(got[:32], want[:32])
    check(got[100:189], q[100:189], k[100:189], v[100:189], [89], 0.1)
    assert not torch.isfinite(got[70:100, :, 3].float()).any()
    assert not torch.isfinite(got[189, :2].float()).any() and torch.isfinite(got[189, 2:].float()).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_behind_the_last_sequence(cuda, dtype):
    """A padded batch: out keeps what it held there, and a NaN in padding reaches nobody."""
    lens = [40, 33]
    q, k, v = inputs(90, 2, 2, 64, dtype)
    k[73:], v[73:], q[73:] = math.nan, math.nan, math.nan
    out = torch.full((90, 2, 64), 7.0, device="cuda", dtype=dtype)
    got = native.prompt_attention(q, k, v, cumulative(lens), 0.125, out=out)
    assert got is out and (out[73:] == 7).all()
    check(out, q[:73], k[:73], v[:73], lens, 0.125)


def test_cumulative_lengths_out_of_range(cuda):
    """Ends past the rows and decreasing entries read and write nothing outside the rows."""
    q, k, v = inputs(64, 2, 2, 64, torch.float16)
    for cu in ([0, 64, 1000], [-5, 64], [0, 40, 20, 64]):
        out = torch.zeros(64, 2, 64, device="cuda", dtype=torch.float16)
        native.prompt_attention(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), 0.125, out=out)
        assert torch.isfinite(out).all()
    check(native.prompt_attention(q, k, v, torch.tensor([0, 64, 1000], dtype=torch.int32, device="cuda"), 0.125), q, k, v, [64],
          0.125)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(cuda, dtype):
    lens = [70, 33]
    q, k, v = inputs(103, 4, 2, 64, dtype)
    want = native.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), cumulative(lens), 0.125)
    assert torch.equal(native.prompt_attention(q, k, v, cumulative(lens), 0.125), want)
    head_major = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    wide = torch.full((103, 4, 128), 3.0, device="cuda", dtype=dtype)
    got = native.prompt_attention(*head_major, cumulative(lens), 0.125, out=wide[..., :64])
    assert torch.equal(got, want) and (wide[..., 64:] == 3).all()
    odd = torch.empty(103 * 2 * 64 + 1, device="cuda", dtype=dtype)[1:].view(103, 2, 64).copy_(k)
    assert torch.equal(native.prompt_attention(q, odd, v, cumulative(lens), 0.125), want)
    one = v[:1].expand(103, 2, 64)  # one row for every key: the result is that row, to its rounding
    got = native.prompt_attention(q, k, one, cumulative(lens), 0.125)
    check(got, q, k, one, lens, 0.125)


def test_no_rows(cuda):
    e = torch.empty(0, 2, 64, device="cuda", dtype=torch.float16)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert native.prompt_attention(e, e, e, zero, 1.0).shape == (0, 2, 64)
    q, k, v = inputs(10, 2, 2, 64, torch.float16)
    out = torch.full((10, 2, 64), 2.0, device="cuda", dtype=torch.float16)
    native.prompt_attention(q, k, v, zero, 1.0, out=out)
    native.prompt_attention(q, k, v, torch.zeros(4, dtype=torch.int32, device="cuda"), 1.0, out=out)
    assert (out == 2).all()
