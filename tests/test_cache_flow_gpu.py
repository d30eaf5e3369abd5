"""The operators together, as a serving loop uses them: ragged prompts rotated and appended and attended in packed form, then
decode steps over the cache they left, in 16 and in 4 bits; the same captured into graphs; calls on other streams."""
import math

import pytest
import torch

import int4_common as ic
from speech_serving import native
from speech_serving.block_manager import BlockManager
from test_packed_prompt_gpu import reference as prompt_reference

pytestmark = pytest.mark.gpu
H, HKV, D, BS = 8, 2, 64, 16
SCALE = 1 / math.sqrt(D)


def fused(n, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, H + 2 * HKV, D, generator=g, device="cuda").to(dtype)
    return x[:, :H], x[:, H:H + HKV], x[:, H + HKV:]


def serve(dtype, bits, lens, steps):
    """[(q, out, keys per row)] of the decode steps, after the prompts; pools, tables and each slot's stored rows."""
    table = native.rotary_table(512, D)
    width = -(-(max(lens) + steps) // BS)
    bm = BlockManager(1, HKV, D, BS, num_blocks=len(lens) * width + 1, dtype=dtype, kv_bits=4 if bits == 4 else None)
    tables = torch.tensor([[bm.allocate_block() for _ in range(width)] for _ in lens], dtype=torch.int32, device="cuda")
    kp, vp = bm.key_pool[0], bm.value_pool[0]
    stored = [torch.zeros(bm.num_blocks * BS, HKV, D, device="cuda", dtype=dtype) for _ in range(2)]

    def append(q, k, v, row, pos):
        at = tables.long()[row, pos // BS] * BS + pos % BS
        k_rot = torch.empty(k.shape, device="cuda", dtype=dtype)
        call = native.append_int4 if bits == 4 else native.append_rotary
        q = call(k, v, kp, vp, at, pos, table, q=q, k_out=k_rot)
        stored[0][at], stored[1][at] = k_rot, v
        return q, k_rot

    n = sum(lens)
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
    row = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), torch.tensor(lens, device="cuda"))
    pos = torch.arange(n, device="cuda") - cu.long()[row]
    q, k, v = fused(n, dtype, 1)
    q_rot, k_rot = append(q, k, v, row, pos)
    out = native.prompt_attention(q_rot, k_rot, v, cu, SCALE)
    ref, bound = prompt_reference(q_rot, k_rot, v, lens, SCALE)
    assert ((out.double() - ref).abs() <= bound).all()
    done = []
    rows = torch.arange(len(lens), device="cuda")
    for s in range(steps):
        q, k, v = fused(len(lens), dtype, 2 + s)
        pos = torch.tensor(lens, device="cuda") + s
        q, _ = append(q, k, v, rows, pos)
        ctx = (pos + 1).to(torch.int32)
        attend = native.paged_attention_int4 if bits == 4 else native.paged_attention
        done.append((q, attend(q, kp, vp, tables, ctx, width * BS, SCALE), ctx.tolist()))
    return done, bm, tables, stored


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [4, 16])
def test_prompts_then_decode(cuda, dtype, bits):
    lens = [33, 1, 70, 16]
    done, bm, tables, stored = serve(dtype, bits, lens, 3)
    if bits == 4:
        held = []
        for x in stored:
            code, scale, low = ic.quantise(x.float().cpu().numpy())
            held.append([torch.from_numpy(a.astype("float64")).cuda() for a in (ic.values(code, scale, low), scale, low)])
    for q, out, ctx in done:
        for b, n in enumerate(ctx):
            vis = torch.tensor([n], device="cuda")
            if bits == 4:
                ref, bound = ic.reference(q[b:b + 1], held, tables[b], vis, BS, bm.num_blocks, SCALE)
            else:
                slot = tables[b].long()[torch.arange(n, device="cuda") // BS] * BS + torch.arange(n, device="cuda") % BS
                ref = torch.stack([ic.attention64(q[b:b + 1, h].double(), stored[0][slot, h // 4].double(),
                                                  stored[1][slot, h // 4].double(), vis, SCALE)[0] for h in range(H)], 1)
                bound = torch.full_like(ref, 2e-3) + ic.half_step(dtype) * ref.abs()  # the 16-bit attention's own bar
            assert ((out[b:b + 1].double() - ref).abs() <= bound).all()
    if bits == 4:  # what the manager reads back is what the rows' codes stand for
        gk, gv = bm.gather(0, tables, torch.tensor(done[-1][2], dtype=torch.int32, device="cuda"), max(done[-1][2]))
        for b, n in enumerate(done[-1][2]):
            slot = tables[b].long()[torch.arange(n, device="cuda") // BS] * BS + torch.arange(n, device="cuda") % BS
            for got, x in ((gk, held[0][0]), (gv, held[1][0])):
                assert torch.equal(got[b, :, :n], x[slot].float().to(dtype).transpose(0, 1))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_captured_step(cuda, dtype):
    """A step (append with rotation, split attention over both caches, packed prompt) captured once and replayed with new
    inputs, eager work in between: every replay equals the eager calls bit for bit."""
    n, width = 4, 40
    table = native.rotary_table(1024, D)
    q, k, v = (x.contiguous() for x in fused(n, dtype, 0))
    blocks = n * width
    tables = torch.arange(blocks, dtype=torch.int32, device="cuda").view(n, width)
    kp, vp = (torch.randint(0, 60, native.int4_pool_shape(blocks, BS, HKV, D), dtype=torch.uint8, device="cuda") for _ in range(2))
    pos = torch.tensor([600, 10, 64, 300], device="cuda")
    cu = torch.tensor([0, 1, n], dtype=torch.int32, device="cuda")

    def step():
        at = tables.long().gather(1, (pos // BS)[:, None])[:, 0] * BS + pos % BS
        k_rot = torch.empty_like(k)
        q_rot = native.append_int4(k, v, kp, vp, at, pos, table, q=q, k_out=k_rot)
        a = native.paged_attention_int4(q_rot, kp, vp, tables, (pos + 1).to(torch.int32), width * BS, SCALE, chunk_tokens=64)
        return a, native.prompt_attention(q_rot, k_rot, v, cu, SCALE)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        for dst, src in zip((q, k, v), fused(n, dtype, 10 + i)):
            dst.copy_(src)
        pos += 1
        kp0, vp0 = kp.clone(), vp.clone()
        want = step()
        want_pools = kp.clone(), vp.clone()
        kp.copy_(kp0), vp.copy_(vp0)
        torch.cuda.synchronize()
        graph.replay()
        junk = torch.randn(1 << 20, device="cuda").sum()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]) and bool(torch.isfinite(junk))
        assert torch.equal(kp, want_pools[0]) and torch.equal(vp, want_pools[1])


def test_two_graphs_share_no_partials(cuda):
    """Two captured attention calls whose keys are split, replayed at once on two streams."""
    b, width = 2, 64
    blocks = b * width
    tables = torch.arange(blocks, dtype=torch.int32, device="cuda").view(b, width)
    lens = torch.tensor([1000, 700], dtype=torch.int32, device="cuda")
    runs = []
    for i in range(2):
        g = torch.Generator(device="cuda").manual_seed(i)
        n = blocks * BS
        pools = [torch.zeros(native.int4_pool_shape(blocks, BS, HKV, D), dtype=torch.uint8, device="cuda") for _ in range(2)]
        native.append_int4(*(torch.randn(n, HKV, D, generator=g, device="cuda", dtype=torch.float32).half() for _ in range(2)),
                           *pools, torch.arange(n, device="cuda"))
        q = torch.randn(b, H, D, generator=g, device="cuda").half()
        call = lambda q=q, pools=pools: native.paged_attention_int4(q, *pools, tables, lens, width * BS, SCALE, chunk_tokens=64)
        want = call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = [call() for _ in range(8)]
        runs.append((graph, out, want, torch.cuda.Stream(), (q, pools)))
    for _ in range(5):
        torch.cuda.synchronize()
        for graph, _, _, stream, _ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, out, want, _, _ in runs:
            assert all(torch.equal(o, want) for o in out)


def test_other_stream(cuda):
    """Calls run on the current stream, ordered behind what it already holds."""
    stream = torch.cuda.Stream()
    n = 300
    table = native.rotary_table(512, D)
    q, k, v = fused(n, torch.bfloat16, 5)
    pos = torch.arange(n, device="cuda")
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    pools = [torch.zeros(native.int4_pool_shape(20, BS, HKV, D), dtype=torch.uint8, device="cuda") for _ in range(4)]

    def work(kp, vp):
        k_rot = torch.empty(k.shape, device="cuda", dtype=k.dtype)
        q_rot = native.append_int4(k, v, kp, vp, pos, pos, table, q=q, k_out=k_rot)
        return native.prompt_attention(q_rot, k_rot, v, cu, SCALE)

    want = work(*pools[:2])
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        got = work(*pools[2:])
    stream.synchronize()
    assert torch.equal(got, want) and torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])
