"""Workspaces that the ops make for themselves: calls inside graph captures."""
import pytest
import torch

from speech_serving import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def decode_args(seed=0, ctx=5000, B=1, Hq=4, Hkv=2, D=64, bs=16):
    """One context long enough to be split over several CTAs, whose join needs arrival counters at zero."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    columns = -(-ctx // bs)
    pool = ops.kv_pool_int4(columns, Hkv, D, bs)
    pages = torch.rand(pool.shape, generator=g, device=DEV).mul_(255).to(torch.uint8)
    codes = D // 64 * bs * 32
    for part in (0, pool.shape[2] // 2):  # random codes; scale 0.25, zero -1
        pool[..., part : part + codes] = pages[..., part : part + codes]
        pool.view(torch.float16)[..., (part + codes) // 2 : part // 2 + pool.shape[2] // 4] = torch.tensor(
            [0.25, -1.0], dtype=torch.float16, device=DEV).repeat(D // 64 * bs)
    q = torch.randn(B, Hq, D, generator=g, device=DEV).half()
    table = torch.randperm(columns, generator=g, device=DEV).to(torch.int32)[None].expand(B, -1).contiguous()
    return q, pool, table, torch.full((B,), ctx, dtype=torch.int32, device=DEV)


def poisoned_pool(megabytes, stream=None):
    """A graph memory pool whose memory, free for captures on `stream`, holds ones; and the graph that fills
    it again."""
    pool, graph = torch.cuda.graph_pool_handle(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, pool=pool, stream=stream):
        # blocks of every size up to the whole: small requests come from segments of their own
        blocks = [torch.empty(n, dtype=torch.uint8, device=DEV) for n in [1 << 19] * 8 + [megabytes << 20]]
        for b in blocks:
            b.fill_(255)
    graph.replay()
    torch.cuda.synchronize()
    return pool, graph


def test_graphs_of_one_geometry_do_not_share_a_workspace():
    """Neither was warmed up, and the one captured last is replayed first, over memory full of ones."""
    args = decode_args(ctx=7000)
    ws = ops.decode_int4_workspace(1, 4, 2, 64, 16, args[2].shape[1], torch.float16, torch.device(DEV))
    want = ops.paged_decode_attention_int4(*args, workspace=ws)
    pool, poison = poisoned_pool(64)
    outs, graphs = [torch.zeros_like(want) for _ in range(3)], [torch.cuda.CUDAGraph() for _ in range(3)]
    for out, graph in zip(outs, graphs):
        with torch.cuda.graph(graph, pool=pool):
            ops.paged_decode_attention_int4(*args, out=out)
    for i in (2, 0, 1, 2):
        poison.replay()
        outs[i].fill_(7.0)
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[i], want)


def test_a_workspace_made_in_a_capture_serves_no_later_call():
    """A call on the capture's own stream before the graph has run."""
    args = decode_args(seed=1, ctx=9000)
    ws = ops.decode_int4_workspace(1, 4, 2, 64, 16, args[2].shape[1], torch.float16, torch.device(DEV))
    want = ops.paged_decode_attention_int4(*args, workspace=ws)
    side, graph, out = torch.cuda.Stream(), torch.cuda.CUDAGraph(), torch.zeros_like(want)
    pool, poison = poisoned_pool(64, side)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, pool=pool, stream=side):
        ops.paged_decode_attention_int4(*args, out=out)
    with torch.cuda.stream(side):
        poison.replay()
        got = ops.paged_decode_attention_int4(*args, out=torch.full_like(want, 7.0))
        assert torch.equal(got, want)
        graph.replay()
    side.synchronize()
    assert torch.equal(out, want)


def test_many_captures_keep_their_results():
    """More captures than are remembered; graphs of released ones still replay."""
    args = decode_args(seed=2, ctx=3000)
    want = ops.paged_decode_attention_int4(*args)
    held = []
    for _ in range(12):
        graph, out = torch.cuda.CUDAGraph(), torch.zeros_like(want)
        with torch.cuda.graph(graph):
            ops.paged_decode_attention_int4(*args, out=out)
        held.append((graph, out))
    for graph, out in held + held[::-1]:
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_the_kept_workspace_does_not_grow_with_the_geometries_seen():
    """Batches and tables of many sizes, back and forth: results stay, and no more memory than the largest needs."""
    cases = [(B, ctx, D, Hq) for B in (1, 2, 5) for ctx in (100, 1500, 6000, 20000, 33000) for D, Hq in ((64, 8), (128, 4))]
    args = {c: decode_args(seed=3, ctx=c[1], B=c[0], Hq=c[3], D=c[2]) for c in cases}
    sizes = {c: ops.decode_int4_workspace(c[0], c[3], 2, c[2], 16, args[c][2].shape[1], torch.float16,
                                          torch.device(DEV)).numel() for c in cases}
    want = {c: ops.paged_decode_attention_int4(*args[c], workspace=torch.zeros(sizes[c], dtype=torch.uint8, device=DEV))
            for c in cases}
    out = {c: torch.full_like(want[c], 7.0) for c in cases}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    with torch.cuda.stream(side):
        for c in cases + cases[::-1] + cases[::3]:
            ops.paged_decode_attention_int4(*args[c], out=out[c].fill_(7.0))
            assert torch.equal(out[c], want[c])
    assert torch.cuda.memory_allocated() - before <= 2 * max(sizes.values()) < sum(sizes.values())


@pytest.mark.parametrize("op", ["paged", "cross"])
def test_captured_calls_of_the_engine_ops_do_not_share_a_workspace(op):
    """The same for paged_decode_attention and cross_attention, over more captures than are remembered."""
    g = torch.Generator(device=DEV).manual_seed(4)
    B, H, D = 4, 12, 64
    q = torch.randn(B, H, D, generator=g, device=DEV).half()
    if op == "paged":
        pools = [torch.randn(128, 16, H, D, generator=g, device=DEV).half() for _ in range(2)]
        table = torch.randperm(128, generator=g, device=DEV).to(torch.int32)[: B * 28].view(B, 28)
        args = (q, *pools, table, torch.tensor([448, 100, 17, 300], dtype=torch.int32, device=DEV))
        call, make = ops.paged_decode_attention, ops.paged_attn_workspace(B, H, D, 28, torch.device(DEV))
    else:
        kv = [torch.randn(B, H, 1500, D, generator=g, device=DEV).half() for _ in range(2)]
        args = (q, *kv, torch.tensor([1500, 100, 17, 900], dtype=torch.int32, device=DEV))
        call, make = ops.cross_attention, ops.cross_attn_workspace(B, H, D, torch.device(DEV))
    want = call(*args, workspace=make)
    pool, poison = poisoned_pool(256)
    outs, graphs = [torch.zeros_like(want) for _ in range(10)], [torch.cuda.CUDAGraph() for _ in range(10)]
    for out, graph in zip(outs, graphs):
        with torch.cuda.graph(graph, pool=pool):
            call(*args, out=out)
    assert len({k[-1] for k in ops._WORKSPACES if k[-1]}) <= 8
    for i in (9, 0, 4, 9, 1):
        poison.replay()
        outs[i].fill_(7.0)
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[i], want)
