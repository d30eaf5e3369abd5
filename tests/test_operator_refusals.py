"""What append_rotary, the 4-bit cache's calls and prompt_attention refuse: at the C entry before anything is launched (no GPU
needed, the pointers are never followed) and in the Python layer."""
import os

import pytest
import torch

from speech_serving import native
from speech_serving.block_manager import BlockManager

P = 1 << 20  # aligned, never dereferenced
F16 = native.SKV_F16
EINVAL, EDTYPE, EALIGN, EWORKSPACE = -1, -2, -3, -4


@pytest.fixture
def lib():
    if not os.path.exists(native.library_path()):
        pytest.skip("libspeechkv.so is not built")
    return native.lib()


ROTARY = dict(q=P, qn=512, qh=64, k=P, kn=256, kh=64, v=P, vn=256, vh=64, qo=P, qon=512, qoh=64, ko=P, kon=256, koh=64,
              kp=P, vp=P, slots=P, pos=P, cs=P, npos=100, rot=64, inter=0, n=4, heads=8, kv=4, d=64, num_slots=64, dtype=F16)


@pytest.mark.parametrize("change,code,word", [
    (dict(dtype=7), EDTYPE, b"dtype"), (dict(n=-1), EINVAL, b"sizes"), (dict(kv=0), EINVAL, b"sizes"),
    (dict(heads=0), EINVAL, b"sizes"), (dict(num_slots=-1), EINVAL, b"sizes"), (dict(npos=-1), EINVAL, b"sizes"),
    (dict(d=72), EINVAL, b"rot_dim"), (dict(rot=24), EINVAL, b"rot_dim"), (dict(rot=0), EINVAL, b"rot_dim"),
    (dict(rot=80), EINVAL, b"rot_dim"), (dict(k=None), EINVAL, b"null"), (dict(vp=None), EINVAL, b"null"),
    (dict(cs=None), EINVAL, b"null"), (dict(pos=None), EINVAL, b"null"), (dict(qo=None), EINVAL, b"null"),
    (dict(q=None), EINVAL, b"null"), (dict(ko=P + 8), EALIGN, b"align"), (dict(kn=252), EALIGN, b"stride"),
    (dict(qoh=68), EALIGN, b"stride"), (dict(kv=1 << 29), EINVAL, b"too large")])
def test_append_rotary_entry(lib, change, code, word):
    rc = lib.skv_append_rotary(*{**ROTARY, **change}.values(), None)
    assert rc == code and word in lib.skv_last_error(), lib.skv_last_error()


INT4 = {**{k: v for k, v in ROTARY.items() if k not in ("num_slots", "dtype")}, "bs": 16, "nb": 8, "dtype": F16}


@pytest.mark.parametrize("change,code,word", [
    (dict(dtype=-1), EDTYPE, b"dtype"), (dict(n=-1), EINVAL, b"sizes"), (dict(d=16), EINVAL, b"head_dim"),
    (dict(d=96), EINVAL, b"head_dim"), (dict(bs=8), EINVAL, b"block_size"), (dict(bs=24), EINVAL, b"block_size"),
    (dict(bs=0), EINVAL, b"block_size"), (dict(nb=-1), EINVAL, b"pool"), (dict(kv=0), EINVAL, b"pool"),
    (dict(kp=None), EINVAL, b"null"), (dict(kp=P + 4), EALIGN, b"align"), (dict(rot=8), EINVAL, b"rot_dim"),
    (dict(rot=128), EINVAL, b"rot_dim"), (dict(cs=None), EINVAL, b"null"), (dict(pos=None), EINVAL, b"null"),
    (dict(v=None), EINVAL, b"null"), (dict(q=None), EINVAL, b"null"), (dict(vh=4), EALIGN, b"stride"),
    (dict(k=P + 8), EALIGN, b"align")])
def test_append_int4_entry(lib, change, code, word):
    rc = lib.skv_append_int4(*{**INT4, **change}.values(), None)
    assert rc == code and word in lib.skv_last_error(), lib.skv_last_error()


GATHER = dict(kp=P, vp=P, tables=P, stride=4, lens=P, ko=P, vo=P, b=2, kv=4, d=64, bs=16, nb=8, max_len=64, dtype=F16)


@pytest.mark.parametrize("change,code,word", [
    (dict(dtype=3), EDTYPE, b"dtype"), (dict(b=-1), EINVAL, b"sizes"), (dict(max_len=-1), EINVAL, b"sizes"),
    (dict(max_len=65), EINVAL, b"past"), (dict(d=80), EINVAL, b"head_dim"), (dict(tables=None), EINVAL, b"null"),
    (dict(stride=0), EINVAL, b"table"), (dict(vo=None), EINVAL, b"null"), (dict(ko=P + 8), EALIGN, b"align"),
    (dict(vp=None), EINVAL, b"null")])
def test_gather_int4_entry(lib, change, code, word):
    rc = lib.skv_gather_int4(*{**GATHER, **change}.values(), None)
    assert rc == code and word in lib.skv_last_error(), lib.skv_last_error()


ATTN = dict(q=P, qb=512, qq=512, qh=64, kp=P, vp=P, tables=P, stride=40, rows=None, lens=P, o=P, ob=512, oq=512, oh=64, b=2,
            ql=1, heads=8, kv=4, d=64, bs=16, nb=8, max_ctx=640, scale=0.125, causal=0, dtype=F16, chunk=64, ws=P,
            ws_bytes=1 << 20)


@pytest.mark.parametrize("change,code,word", [
    (dict(dtype=9), EDTYPE, b"dtype"), (dict(d=48), EINVAL, b"head_dim"), (dict(heads=6), EINVAL, b"sizes"),
    (dict(ql=0), EINVAL, b"sizes"), (dict(ql=65536), EINVAL, b"sizes"), (dict(b=-1), EINVAL, b"sizes"),
    (dict(max_ctx=-1), EINVAL, b"sizes"), (dict(stride=0), EINVAL, b"sizes"), (dict(q=None), EINVAL, b"null"),
    (dict(lens=None), EINVAL, b"null"), (dict(tables=None), EINVAL, b"null"), (dict(o=P + 2), EALIGN, b"align"),
    (dict(qh=60), EALIGN, b"stride"), (dict(chunk=96), EINVAL, b"chunk"), (dict(ws=None), EWORKSPACE, b"workspace"),
    (dict(ws_bytes=100), EWORKSPACE, b"workspace"), (dict(ws=P + 8), EWORKSPACE, b"workspace"),
    (dict(b=1 << 22), EINVAL, b"too large"), (dict(nb=1 << 30), EINVAL, b"too large"),
    (dict(stride=1 << 27, max_ctx=(1 << 30) + 1), EINVAL, b"past"), (dict(chunk=(1 << 30) + 64), EINVAL, b"past")])
def test_paged_attention_int4_entry(lib, change, code, word):
    rc = lib.skv_paged_attention_int4(*{**ATTN, **change}.values(), None)
    assert rc == code and word in lib.skv_last_error(), lib.skv_last_error()


PROMPT = dict(q=P, qn=512, qh=64, k=P, kn=256, kh=64, v=P, vn=256, vh=64, cu=P, o=P, on=512, oh=64, n=10, seqs=2, heads=8, kv=4,
              d=64, scale=0.125, dtype=F16)


@pytest.mark.parametrize("change,code,word", [
    (dict(dtype=5), EDTYPE, b"dtype"), (dict(d=48), EINVAL, b"head_dim"), (dict(d=256), EINVAL, b"head_dim"),
    (dict(n=-1), EINVAL, b"sizes"), (dict(seqs=-1), EINVAL, b"sizes"), (dict(heads=6), EINVAL, b"sizes"),
    (dict(kv=0), EINVAL, b"sizes"), (dict(q=None), EINVAL, b"null"), (dict(cu=None), EINVAL, b"null"),
    (dict(o=P + 4), EALIGN, b"align"), (dict(vn=252), EALIGN, b"stride"), (dict(kn=-256), EINVAL, b"stride"),
    (dict(vn=1 << 23), EINVAL, b"stride"), (dict(n=1 << 30), EINVAL, b"too large"), (dict(seqs=1 << 22), EINVAL, b"too large")])
def test_prompt_attention_entry(lib, change, code, word):
    rc = lib.skv_prompt_attention(*{**PROMPT, **change}.values(), None)
    assert rc == code and word in lib.skv_last_error(), lib.skv_last_error()


def test_int4_blocks_past_2_gib(lib):
    """Blocks whose bytes pass 31 bits, which the attention counts in 32, are refused by every call of the cache."""
    big = dict(kv=256, d=128, bs=1 << 17, nb=1)  # 256 heads x 8192 tiles x 1280 bytes
    assert lib.skv_append_int4(*{**INT4, **big}.values(), None) == EINVAL and b"block of" in lib.skv_last_error()
    assert lib.skv_gather_int4(*{**GATHER, **big}.values(), None) == EINVAL and b"block of" in lib.skv_last_error()
    attn = {**ATTN, **big, "heads": 256}
    assert lib.skv_paged_attention_int4(*attn.values(), None) == EINVAL and b"block of" in lib.skv_last_error()


def test_workspace_sizes(lib):
    assert lib.skv_int4_workspace_bytes(2, 3, 8, 64, 640, 64) == 2 * 3 * 8 * 10 * (64 + 4) * 4
    assert lib.skv_int4_workspace_bytes(2, 3, 8, 64, 64, 64) == 0
    for args in ((0, 1, 8, 64, 640, 64), (2, 1, 8, 64, 0, 64), (2, 1, 8, 64, 640, 0)):
        assert lib.skv_int4_workspace_bytes(*args) == 0
    for dtype in (native.SKV_F32, native.SKV_F16, native.SKV_BF16):
        for b, q, h, kv, d, ctx in ((1, 1, 1, 1, 32, 1), (64, 1, 20, 20, 64, 452), (1, 1, 32, 8, 128, 1 << 20), (3, 5, 8, 2, 64, 9)):
            c = lib.skv_int4_chunk_tokens(b, q, h, kv, d, ctx, dtype)
            assert c > 0 and c % 64 == 0


# ---------------------------------------------------------------------------
# The Python layer, on CPU tensors: every refusal comes before a launch.
# ---------------------------------------------------------------------------
def rows(n=4, h=2, d=64, dtype=torch.float16):
    return torch.zeros(n, h, d, dtype=dtype)


def test_cpu_tensors_are_refused():
    i64, i32 = torch.zeros(4, dtype=torch.int64), torch.zeros(2, dtype=torch.int32)
    pool = torch.zeros(1, 16, 2, 64, dtype=torch.float16)
    pool4 = torch.zeros(native.int4_pool_shape(1, 16, 2, 64), dtype=torch.uint8)
    table = native.rotary_table(8, 64, device="cpu")
    calls = [lambda: native.append_rotary(rows(), rows(), pool, pool, i64, i64, table),
             lambda: native.append_int4(rows(), rows(), pool4, pool4, i64),
             lambda: native.gather_int4(pool4, pool4, torch.zeros(2, 1, dtype=torch.int32), i32, 4, torch.float16),
             lambda: native.paged_attention_int4(rows(), pool4, pool4, torch.zeros(4, 1, dtype=torch.int32), i32, 4, 1.0),
             lambda: native.prompt_attention(rows(), rows(), rows(), i32, 1.0)]
    for call in calls:
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_rotary_is_required():
    with pytest.raises(RuntimeError, match="required"):
        native.append_rotary(rows(), rows(), rows(), rows(), torch.zeros(4, dtype=torch.int64), None, None)


@pytest.mark.parametrize("args", [(8, 0), (8, 7), (-1, 8)])
def test_rotary_table_sizes(args):
    with pytest.raises(RuntimeError, match="rotary_table"):
        native.rotary_table(*args, device="cpu")


@pytest.mark.parametrize("args", [(1, 8, 2, 64), (1, 24, 2, 64), (1, 0, 2, 64), (1, 16, 2, 48), (1, 16, 2, 16)])
def test_int4_pool_shape_sizes(args):
    with pytest.raises(RuntimeError, match="int4_pool_shape"):
        native.int4_pool_shape(*args)


def test_block_manager_4_bits():
    bm = BlockManager(3, 2, 64, 32, num_blocks=5, dtype=torch.bfloat16, device="cpu", kv_bits=4)
    assert bm.key_pool[2].shape == native.int4_pool_shape(5, 32, 2, 64) and bm.value_pool[0].dtype == torch.uint8
    assert bm.block_bytes() * 5 == bm.arena.numel() and bm.get_stats()["pool_memory_mb"] == round(bm.arena.numel() / 2 ** 20, 2)
    assert bm.allocate_block() == 4 and bm.slot([4], 31) == 159
    for kw in (dict(block_size=8), dict(block_size=40), dict(head_dim=16), dict(kv_bits=8)):
        with pytest.raises(ValueError):
            BlockManager(**{**dict(num_layers=1, num_kv_heads=2, head_dim=64, block_size=16, num_blocks=2, device="cpu",
                                   kv_bits=4), **kw})
