"""shared_prefix_decode_attention and cross_attention_packed where calls go wrong: no prefix, groups that do not cover the
batch, bad block and slot ids, lengths past the tables, what lies in masked places, strides, places of the
result, refusals, streams, graphs, workspaces, waits that run out, offsets past 32 bits."""
import math

import pytest
import torch

from int4_reference import cu
from speech_serving import _native as N
from speech_serving import ops
from test_candidates_gpu import DEV, Prefix, attend, near
from test_workspaces_gpu import poisoned_pool

pytestmark = pytest.mark.gpu
prefix = ops.shared_prefix_decode_attention


def word():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def case(seed=0, dtype=torch.float16, Hq=4, Hkv=2, D=64, **kw):
    return Prefix(seed, [3, 1, 5], [300, 40, 1000], [5, 0, 700, 1, 16, 17, 3, 64, 2], Hq, Hkv, D, dtype, **kw)


# ---- what takes part ---------------------------------------------------------------------------------
def test_calls_without_a_prefix():
    c = case()
    q, k, v, ptab, plens, cg, tab, lens = c.args()
    got = prefix(q, k, v, None, None, None, tab, lens)
    near(got, c.want(first=9))
    empty = torch.zeros(0, 7, dtype=torch.int32, device=DEV), lens[:0], torch.zeros(1, dtype=torch.int32, device=DEV)
    assert torch.equal(got, prefix(q, k, v, *empty, tab, lens))
    assert torch.equal(got, prefix(q, k, v, ptab[:, :0].contiguous(), plens * 0, cg, tab, lens))
    assert torch.equal(got, prefix(q, k, v, ptab, plens * 0 - 5, cg, tab, lens))


def test_sequences_outside_the_groups():
    c = case(1)
    a = c.args()
    a[5] = (a[5] + 2).clamp(max=9)
    near(prefix(*a), c.want(first=2))


def test_no_own_tokens_and_no_tokens_at_all():
    c = case(2)
    a = c.args()
    c.mine = [0] * 9
    none = torch.zeros(9, 0, dtype=torch.int32, device=DEV)
    want = c.want()
    near(prefix(*a[:6], none, a[7] * 0), want)
    near(prefix(*a[:6], a[6], a[7] * 0 - 3), want)
    out = torch.full_like(a[0], 7.0)
    prefix(*a[:3], None, None, None, none, a[7] * 0, out=out)
    assert (out == 0).all()
    prefix(*a[:4], a[4] * 0, *a[5:7], a[7] * 0, out=out.fill_(7.0))
    assert (out == 0).all()


def test_empty_batches():
    c = case()
    q, k, v, ptab, plens, cg, tab, lens = c.args()
    assert prefix(q[:0], k, v, ptab, plens, cg * 0, tab[:0], lens[:0]).shape == (0, 4, 64)
    kv = torch.zeros(2, 2, 8, 64, device=DEV).half()
    assert ops.cross_attention_packed(q[:0, :2], kv, kv, lens[:2], cg[:3] * 0).shape == (0, 2, 64)
    out = torch.full((9, 2, 64), 7.0, device=DEV).half()
    assert (ops.cross_attention_packed(q[:, :2], kv, kv, lens[:0], cg[:1] * 0, out=out) == 7).all()


@pytest.mark.parametrize("bs", [8, 16, 64])
def test_bad_block_ids_are_left_out_and_flagged(bs):
    c = case(3, bs=bs)
    lost = [int(c.ptab[0, 1]), int(c.ptab[2, 0]), int(c.ptab[2, (1000 - 1) // bs]), int(c.tab[2, 2]), int(c.tab[3, 0])]
    want = c.want(left_out=lost)
    a, e = c.args(), word()
    a[1][lost], a[2][lost] = math.nan, math.inf
    for table in (a[3], a[6]):
        bad = torch.isin(table, torch.tensor(lost, dtype=torch.int32, device=DEV))
        table[bad] = torch.tensor([-1, -2 ** 31, 2 ** 31 - 1, len(c.k), len(c.k) + 5], dtype=torch.int32, device=DEV)[: int(bad.sum())]
    got = prefix(*a, error_word=e)
    near(got, want)
    assert ops.read_error_word(e) == N.SPD_DEVERR_BLOCK_ID
    ws = ops.shared_prefix_workspace(9, 3, 4, 2, 64, bs, a[3].shape[1], a[6].shape[1], torch.device(DEV))
    assert torch.equal(got, prefix(*a, workspace=ws)) and ops.read_error_word(ws) == N.SPD_DEVERR_BLOCK_ID
    a[3].fill_(-1), a[6].fill_(-1)
    assert (prefix(*a) == 0).all()


def test_lengths_past_the_tables_are_cut_and_flagged():
    c = case(4)
    a, e = c.args(), word()
    a[4][0], a[7][2], a[7][4] = 10 ** 6, 2 ** 31 - 1, 2 ** 30
    c.prefix, c.mine = list(c.prefix), list(c.mine)
    c.prefix[0], c.mine[2], c.mine[4] = c.ptab.shape[1] * 16, c.tab.shape[1] * 16, c.tab.shape[1] * 16
    near(prefix(*a, error_word=e), c.want())
    assert ops.read_error_word(e) == N.SPD_DEVERR_LENGTH


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 65504.0])
def test_what_lies_behind_the_lengths_does_not_matter(bad):
    c = case(5)
    want = prefix(*c.args())
    used = torch.zeros(c.k.shape[0] * 16, dtype=torch.bool)
    for g, n in enumerate(c.prefix):
        used[c.rows(c.ptab[g], n)] = True
    for b, n in enumerate(c.mine):
        used[c.rows(c.tab[b], n)] = True
    for t in (c.k, c.v):
        t.flatten(0, 1)[~used] = bad
    assert torch.equal(prefix(*c.args()), want)


def test_infinite_and_nan_keys_stay_with_their_rows():
    """A NaN among one group's keys reaches no other group."""
    c = case(6)
    want = prefix(*c.args())
    c.k.flatten(0, 1)[c.rows(c.ptab[0], 300)[100]] = math.nan
    got = prefix(*c.args())
    assert torch.isnan(got[:3]).any(-1).any(-1).all() and torch.equal(got[3:], want[3:])


def test_large_scores():
    """Scores of thousands, of both signs: weights of zero and one."""
    for dtype in (torch.float16, torch.bfloat16):
        c = case(7, dtype, spread=300.0)
        near(prefix(*c.args()), c.want())
        near(prefix(*c.args(), scale=1e-4), c.want(scale=1e-4))


# ---- strides and places ----------------------------------------------------------------------------------
@pytest.mark.parametrize("D", [40, 64, 128])
def test_queries_of_any_strides(D):
    c = case(8, D=D)
    a = c.args()
    want = prefix(*a)
    packed = torch.randn(9, 8, D, device=DEV).half()
    packed[:, 2:6] = a[0]
    assert torch.equal(prefix(packed[:, 2:6], *a[1:]), want)
    turned = a[0].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(prefix(turned, *a[1:]), want)
    for view in (a[0][:1].expand(9, 4, D), a[0][:, :1].expand(9, 4, D)):
        assert torch.equal(prefix(view, *a[1:]), prefix(view.contiguous(), *a[1:]))


def test_cross_strides():
    B, T, H, D = 3, 333, 4, 64
    g = torch.Generator(device=DEV).manual_seed(0)
    kv = torch.randn(B, T, 2, H, D, device=DEV, generator=g).half()  # as a fused projection writes them
    q = torch.randn(9, 8, D, device=DEV, generator=g).half()[:, ::2]
    lens, cq = torch.tensor([333, 128, 1], dtype=torch.int32, device=DEV), cu([4, 0, 5]).to(DEV)
    k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    want = ops.cross_attention_packed(q.contiguous(), k.contiguous(), v.contiguous(), lens, cq)
    assert torch.equal(ops.cross_attention_packed(q, k, v, lens, cq), want)
    one = k[:, :1].expand(B, H, T, D), v[:, :1].expand(B, H, T, D)
    assert torch.equal(ops.cross_attention_packed(q, *one, lens, cq),
                       ops.cross_attention_packed(q, *(t.contiguous() for t in one), lens, cq))
    same = k[:1].expand(B, H, T, D), v[:1].expand(B, H, T, D)
    assert torch.equal(ops.cross_attention_packed(q, *same, lens, cq),
                       ops.cross_attention_packed(q, *(t.contiguous() for t in same), lens, cq))
    # heads in groups, and a slot of one head and one position
    grouped = ops.cross_attention_packed(q, k[:, :2], v[:, :2], lens, cq)
    wide = (t[:, :2].repeat_interleave(2, 1) for t in (k, v))
    assert (grouped.float() - ops.cross_attention_packed(q, *wide, lens, cq).float()).abs().max() <= 2 ** -9 * v.abs().max()
    tiny = ops.cross_attention_packed(q[:1, :1], k[:1, :1, :1], v[:1, :1, :1], lens[:1])
    assert torch.equal(tiny[0, 0], v[0, 0, 0])


def test_places_of_the_result():
    c = case(9)
    a = c.args()
    want = prefix(*a)
    q = a[0].clone()
    assert prefix(q, *a[1:], out=q) is not None and torch.equal(q, want)
    buf = torch.zeros(12, 4, 64, device=DEV).half()
    buf[:9] = a[0]
    for out in (buf[1:10], buf[:9].transpose(0, 1)[:, :9].transpose(0, 1)[1:]):
        with pytest.raises(RuntimeError, match="out must be"):
            prefix(buf[:9], *a[1:], out=out)
    with pytest.raises(RuntimeError, match="apart from the pools"):
        prefix(a[0], *a[1:], out=a[1].flatten(0, 2)[: 9 * 4].view(9, 4, 64))
    kv = torch.randn(3, 2, 4, 50, 64, device=DEV).half()
    lens, cq = torch.tensor([50, 0, 7], dtype=torch.int32, device=DEV), cu([2, 3, 4]).to(DEV)
    want = ops.cross_attention_packed(a[0], kv[:, 0], kv[:, 1], lens, cq)
    q = a[0].clone()
    ops.cross_attention_packed(q, kv[:, 0], kv[:, 1], lens, cq, out=q)
    assert torch.equal(q, want)
    with pytest.raises(RuntimeError, match="apart from k and v"):
        ops.cross_attention_packed(a[0], kv[:, 0], kv[:, 1], lens, cq, out=kv.flatten(0, 3)[:36].view(9, 4, 64))


def test_in_place_over_many_tiles_and_cut_items():
    g = torch.Generator(device=DEV).manual_seed(1)
    q = torch.randn(1500, 4, 64, device=DEV, generator=g).half()
    kv = torch.randn(5, 2, 4, 900, 64, device=DEV, generator=g).half()
    lens, cq = torch.tensor([900, 500, 0, 77, 900], dtype=torch.int32, device=DEV), cu([700, 1, 300, 0, 499]).to(DEV)
    want = ops.cross_attention_packed(q, kv[:, 0], kv[:, 1], lens, cq)
    for _ in range(5):
        again = q.clone()
        ops.cross_attention_packed(again, kv[:, 0], kv[:, 1], lens, cq, out=again)
        assert torch.equal(again, want)


# ---- requests over slots ---------------------------------------------------------------------------------
def test_slots_lengths_and_rows_of_no_request():
    g = torch.Generator().manual_seed(2)
    kv = torch.randn(4, 2, 2, 200, 64, generator=g).half()
    q = torch.randn(20, 4, 64, generator=g).half()
    beams, valid, slots = [3, 2, 4, 1, 2, 3], [200, 0, 10 ** 6, 64, -5, 50], [3, 0, 3, 4, 1, -1]  # a slot twice, two out of range
    d = kv.to(DEV)
    out, e = torch.full((20, 4, 64), 7.0, device=DEV).half(), word()
    ints = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (valid, slots))
    lens, ids = ints
    ops.cross_attention_packed(q.to(DEV), d[:, 0], d[:, 1], lens, (cu(beams) + 2).to(DEV), ids, out=out, error_word=e)
    assert ops.read_error_word(e) == N.SPD_DEVERR_BLOCK_ID | N.SPD_DEVERR_LENGTH
    parts, a = [], 2
    for n, t, s in zip(beams, valid, slots):
        t = max(0, min(200, t)) if 0 <= s < 4 else 0
        for i in range(n):
            parts.append(attend(q[a + i], kv[s % 4, 0, :, :t].transpose(0, 1), kv[s % 4, 1, :, :t].transpose(0, 1), 1 / 8))
        a += n
    near(out[2:17], parts)
    assert (out[:2] == 7).all() and (out[17:] == 7).all()
    ws = ops.cross_attn_packed_workspace(20, 4, 2, 64, torch.device(DEV))
    ops.cross_attention_packed(q.to(DEV), d[:, 0], d[:, 1], lens, (cu(beams) + 2).to(DEV), ids, out=out, workspace=ws)
    assert ops.read_error_word(ws) == N.SPD_DEVERR_BLOCK_ID | N.SPD_DEVERR_LENGTH
    d[:, :, :, 64:] = math.nan  # behind every length that follows
    lens = torch.tensor([64, 0, 1, 63, 33, 50], dtype=torch.int32, device=DEV)
    assert torch.isfinite(ops.cross_attention_packed(q.to(DEV), d[:, 0], d[:, 1], lens, cu([3, 2, 4, 5, 2, 4]).to(DEV), ids)).all()


def test_one_query_a_request():
    g = torch.Generator(device=DEV).manual_seed(3)
    kv = torch.randn(6, 2, 3, 150, 80, generator=g, device=DEV).bfloat16()
    q = torch.randn(5, 3, 80, generator=g, device=DEV).bfloat16()
    lens = torch.tensor([150, 1, 128, 129, 0], dtype=torch.int32, device=DEV)
    got = ops.cross_attention_packed(q, kv[:, 0], kv[:, 1], lens)
    assert torch.equal(got, ops.cross_attention_packed(q, kv[:, 0], kv[:, 1], lens, cu([1] * 5).to(DEV)))
    near(got, [attend(q[b].cpu(), *(kv[b, i, :, :t].transpose(0, 1).cpu() for i in (0, 1)), 80 ** -0.5) for b, t in enumerate(lens.tolist())])


def test_groups_out_of_order_stay_within_bounds():
    """Starts that overlap, fall or leave the batch are cut to it; groups that do not overlap are exact."""
    g = torch.Generator().manual_seed(4)
    kv, q = torch.randn(3, 2, 2, 100, 64, generator=g).half(), torch.randn(8, 2, 64, generator=g).half()
    d, lens = kv.to(DEV), torch.tensor([100, 100, 100], dtype=torch.int32, device=DEV)
    for starts, exact in (([0, 5, 3, 8], {0: range(3), 2: range(5, 8)}), ([-3, 2, 100, 100], {0: range(2), 1: range(2, 8)})):
        cq = torch.tensor(starts, dtype=torch.int32, device=DEV)
        got = ops.cross_attention_packed(q.to(DEV), d[:, 0], d[:, 1], lens, cq)
        for s, rows in exact.items():
            near(got[list(rows)], [attend(q[i], kv[s, 0].transpose(0, 1), kv[s, 1].transpose(0, 1), 1 / 8) for i in rows])


# ---- refusals ----------------------------------------------------------------------------------------------
def test_prefix_refuses():
    c = case()
    a = c.args()

    def with_(i, t):
        return [t if j == i else x for j, x in enumerate(a)]

    wrong = [
        with_(0, a[0].bfloat16()), with_(0, a[0].float()), with_(0, a[0][0]), with_(0, a[0][:, :3]), with_(0, a[0][:, :, :32]),
        with_(0, torch.zeros(9, 4, 65, device=DEV).half()[:, :, 1:]), with_(1, a[1][:, :, :, :32]), with_(1, a[1].float()),
        with_(2, a[2][:-1]), with_(1, a[1].transpose(1, 2)), with_(3, None), with_(4, None), with_(5, None), with_(3, a[3].long()),
        with_(3, a[3][:, ::2]), with_(4, a[4][:2]), with_(5, a[5][:3]), with_(5, a[5].float()), with_(6, a[6][:8]), with_(6, a[6].float()),
        with_(7, a[7][:8]), with_(7, a[7].long()), with_(7, a[7].cpu()), with_(1, a[1].cpu()),
    ]
    for args in wrong:
        with pytest.raises(RuntimeError):
            prefix(*args)
    for kw in (dict(scale=0.0), dict(scale="x"), dict(out=a[0][:8]), dict(out=torch.zeros_like(a[0]).float()),
               dict(workspace=torch.zeros(256, dtype=torch.uint8, device=DEV)), dict(workspace=torch.zeros(9, device=DEV)),
               dict(error_word=torch.zeros(1, device=DEV)), dict(out=torch.zeros(4, 9, 64, device=DEV).half().transpose(0, 1))):
        with pytest.raises(RuntimeError):
            prefix(*a, **kw)
    with pytest.raises(RuntimeError, match="unsupported geometry"):
        ops.shared_prefix_workspace(9, 3, 4, 2, 64, 24, 4, 4, torch.device(DEV))
    torch.cuda.synchronize()


def test_cross_refuses():
    q, kv = torch.zeros(6, 4, 64, device=DEV).half(), torch.zeros(3, 2, 2, 40, 64, device=DEV).half()
    lens, cq, ids = torch.ones(3, dtype=torch.int32, device=DEV), cu([2, 2, 2]).to(DEV), torch.arange(3, dtype=torch.int32, device=DEV)
    k, v = kv[:, 0], kv[:, 1]
    wrong = [
        (q.float(), k, v, lens, cq), (q, k.float(), v, lens, cq), (q, k, v[:, :1], lens, cq), (q[:, :3], k, v, lens, cq), (q, k, v, lens),
        (q, k, v, lens.long(), cq), (q, k, v, lens, cq[:3]), (q, k, v, lens, cq, ids[:2]), (q, k, v, lens, cq, ids.long()),
        (q, k, v.contiguous(), lens, cq), (q, k[:2], v[:2], lens, cq), (q, k[..., ::2], v[..., ::2], lens, cq), (q.cpu(), k, v, lens, cq),
        (q, k[:, :, :0], v[:, :, :0], lens, cq), (q, k, v, lens.view(3, 1), cq),
        (torch.zeros(6, 4, 68, device=DEV).half()[:, :, 2:66], k, v, lens, cq),
    ]
    for args in wrong:
        with pytest.raises(RuntimeError):
            ops.cross_attention_packed(*args)
    for kw in (dict(scale=-1.0), dict(out=q[:5]), dict(workspace=torch.zeros(512, dtype=torch.uint8, device=DEV)),
               dict(error_word=torch.zeros(0, dtype=torch.int32, device=DEV))):
        with pytest.raises(RuntimeError):
            ops.cross_attention_packed(q, k, v, lens, cq, **kw)
    with pytest.raises(RuntimeError, match="unsupported geometry"):
        ops.cross_attn_packed_workspace(6, 4, 3, 64, torch.device(DEV))
    torch.cuda.synchronize()


# ---- streams, graphs, workspaces ---------------------------------------------------------------------------
def long_case(seed):
    """Own tokens in several chunks, prefixes in several pieces."""
    return Prefix(seed, [4, 2], [5000, 900], [4000, 3, 0, 2500, 1, 600], 4, 2, 64, torch.bfloat16)


def test_two_streams_at_once():
    cases = [long_case(s).args() for s in range(4)]
    kv = torch.randn(2, 2, 2, 3000, 64, device=DEV).bfloat16()
    lens, cq = torch.tensor([3000, 1000], dtype=torch.int32, device=DEV), cu([4, 2]).to(DEV)

    def both(a):
        return prefix(*a), ops.cross_attention_packed(a[0], kv[:, 0], kv[:, 1], lens, cq)

    want = [both(a) for a in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    found = [[] for _ in cases]
    for _ in range(20):
        for s, a, f in zip(streams, cases, found):
            with torch.cuda.stream(s):
                f.append(both(a))
    torch.cuda.synchronize()
    for w, f in zip(want, found):
        assert all(torch.equal(x, y) for pair in f for x, y in zip(pair, w))


def test_graphs_of_one_geometry_do_not_share_a_workspace():
    a, b = long_case(0).args(), long_case(1).args()
    kv = torch.randn(2, 2, 2, 3000, 64, device=DEV).bfloat16()
    lens, cq = torch.tensor([3000, 1000], dtype=torch.int32, device=DEV), cu([4, 2]).to(DEV)

    def run(x, outs):
        prefix(*x, out=outs[0])
        ops.cross_attention_packed(x[0], kv[:, 0], kv[:, 1], lens, cq, out=outs[1])

    want = [[torch.empty_like(x[0]) for _ in range(2)] for x in (a, b)]
    for x, outs in zip((a, b), want):
        run(x, outs)
    pool, poison = poisoned_pool(64)
    found, graphs = [[torch.empty_like(x[0]) for _ in range(2)] for x in (a, b)], [torch.cuda.CUDAGraph() for _ in range(2)]
    for x, outs, graph in zip((a, b), found, graphs):
        with torch.cuda.graph(graph, pool=pool):
            run(x, outs)
    for i in (1, 0, 0, 1):
        poison.replay()
        for t in found[i]:
            t.fill_(7.0)
        graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(found[i], want[i]))


def test_one_workspace_for_calls_of_changing_lengths():
    """Counters are back at zero after every call, also beside other operators that keep theirs in the same memory."""
    c = long_case(2)
    a = c.args()
    ws = ops.shared_prefix_workspace(6, 2, 4, 2, 64, 16, a[3].shape[1], a[6].shape[1], torch.device(DEV))
    for seed in range(6):
        g = torch.Generator().manual_seed(seed)
        c.mine = [int(torch.randint(0, n + 1, (1,), generator=g)) for n in (4000, 3, 0, 2500, 1, 600)]
        c.prefix = [int(torch.randint(0, n + 1, (1,), generator=g)) for n in (5000, 900)]
        a[4].copy_(torch.tensor(c.prefix)), a[7].copy_(torch.tensor(c.mine))
        got = prefix(*a, workspace=ws)
        near(got, c.want())
        assert torch.equal(got, prefix(*a)) and ops.read_error_word(ws) == 0


# ---- waits that run out -----------------------------------------------------------------------------------
@pytest.mark.parametrize("members,prefix_len,D", [([3], 40000, 64), ([200], 9000, 128), ([5, 300, 40], 3000, 64), ([70, 2], 6000, 128)])
def test_waits_give_up_and_then_the_call_is_exact(members, prefix_len, D):
    """Under a bound of 1 ns any wait may give up: the launch records it and returns."""
    lib = N.load()
    B, G = sum(members), len(members)
    c = Prefix(0, members, [prefix_len] * G, [40] * B, 4, 2, D, torch.bfloat16)
    a, e = c.args(), word()
    kv = torch.randn(G, 2, 2, prefix_len, D, device=DEV).bfloat16()
    lens, cq = torch.full((G,), prefix_len, dtype=torch.int32, device=DEV), cu(members).to(DEV)

    def both():
        return prefix(*a, error_word=e), ops.cross_attention_packed(a[0], kv[:, 0], kv[:, 1], lens, cq, error_word=e)

    want = both()
    assert ops.read_error_word(e) == 0
    try:
        assert lib.spd_set_wait_timeout_ns(1) == N.SPD_OK
        for _ in range(3):
            both()
            torch.cuda.synchronize()
            assert ops.read_error_word(e) in (0, N.SPD_DEVERR_TIMEOUT)
    finally:
        assert lib.spd_set_wait_timeout_ns(0) == N.SPD_OK
    e.zero_()
    assert all(torch.equal(x, y) for x, y in zip(both(), want)) and ops.read_error_word(e) == 0


# ---- the largest ---------------------------------------------------------------------------------------------
def test_offsets_past_32_bits():
    """The blocks and slots that are read begin past 2^31 elements."""
    g = torch.Generator(device=DEV).manual_seed(5)
    blocks, near_end = 135_000, 134_900  # of 16 x 8 x 128 elements
    k, v = (torch.empty(blocks, 16, 8, 128, dtype=torch.float16, device=DEV) for _ in range(2))
    for t in (k, v):
        t[near_end:] = torch.randn(100, 16, 8, 128, device=DEV, generator=g).half()
    q = torch.randn(3, 8, 128, device=DEV, generator=g).half()
    ids = torch.randperm(100, device=DEV, generator=g).to(torch.int32) + near_end
    ptab, tab = ids[:40].view(1, 40), ids[40:100].view(3, 20).contiguous()
    plens, lens = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([640], [320, 1, 100]))
    args = (ptab, plens, cu([3]).to(DEV), tab, lens)
    got = prefix(q, k, v, *args)
    small = [x - near_end for x in (ptab, tab)]
    assert torch.equal(got, prefix(q, k[near_end:].clone(), v[near_end:].clone(), small[0], plens, args[2], small[1], lens))
    del k, v
    kv = torch.empty(1000, 20, 2000, 64, dtype=torch.float16, device=DEV)  # 2.56e9 elements
    kv[998:] = torch.randn(2, 20, 2000, 64, device=DEV, generator=g).half()
    q = torch.randn(6, 20, 64, device=DEV, generator=g).half()
    lens, cq = torch.tensor([2000, 1999], dtype=torch.int32, device=DEV), cu([5, 1]).to(DEV)
    got = ops.cross_attention_packed(q, kv, kv, lens, cq, lens * 0 + torch.tensor([999, 998], dtype=torch.int32, device=DEV))
    assert torch.equal(got, ops.cross_attention_packed(q, *[kv[998:].flip(0).contiguous()] * 2, lens, cq))


@pytest.mark.parametrize("groups", [31, 32, 33, 300, 1100])
def test_many_groups(groups):
    """More groups than a warp looks at at once, some of them empty, and sequences before, behind and in them."""
    g = torch.Generator().manual_seed(groups)
    members = torch.randint(0, 3, (groups,), generator=g).tolist()
    members[0], members[-1] = 1, 2
    pre = torch.randint(0, 40, (groups,), generator=g).tolist()
    mine = torch.randint(0, 4, (sum(members),), generator=g).tolist()
    c = Prefix(groups, members, pre, mine, 4, 2, 64, torch.float16, bs=8)
    near(prefix(*c.args()), c.want())
    a = c.args()
    a[5] = (a[5] + 1).clamp(max=sum(members))
    near(prefix(*a), c.want(first=1))
