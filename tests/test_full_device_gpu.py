"""The rotary, 4-bit and prompt operators at sizes that fill the device, where they take other ways through
the same kernels: prompt items that outnumber the SMs (ranked by length, taken over, steps of 64 keys at
head sizes up to 64), several tokens a CTA in the appends and the gather, contexts cut into chunks that
are dealt out.  Appends and gathers are compared whole and bit for bit, attention on sampled
sequences with the 64-bit form under the bounds of the operators' own tests."""
import pytest
import torch

import int4_reference as R
from speech_serving import ops
from test_decode_int4_gpu import UNIT as UNITS
from test_decode_int4_gpu import reference as decode_reference
from test_prompt_attention_gpu import UNIT
from test_prompt_attention_gpu import reference as prompt_reference
from test_rope_kv_gpu import Case

pytestmark = pytest.mark.gpu
DEV = "cuda"


def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


# ------------------------------------------------------------------------------- prompts
@pytest.mark.parametrize("Hq,Hkv,D", [(16, 16, 64), (16, 4, 64), (12, 2, 32), (20, 20, 40), (16, 16, 128), (32, 8, 128),
                                      (24, 4, 96)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal,prefixes", [(True, False), (True, True), (False, True)])
def test_more_prompt_items_than_ctas(Hq, Hkv, D, dtype, causal, prefixes):
    pack = (Hq // Hkv) & -(Hq // Hkv)
    tokens = 256 // pack
    g = torch.Generator().manual_seed(Hq * D + causal + 2 * prefixes)
    lens, items = [], 0
    while items <= 5 * sms():  # well above two for every slot of two CTAs an SM
        lens.append(int(torch.randint(0, 701, (1,), generator=g)) if len(lens) % 5 else [1, 0, 700, 257][len(lens) // 5 % 4])
        items += -(-lens[-1] // tokens) * (Hq // pack)
    keys = [n + int(torch.randint(0, 500, (1,), generator=g)) if prefixes and i % 3 else n for i, n in enumerate(lens)]
    n, m = sum(lens), sum(keys)
    gd = torch.Generator(device=DEV).manual_seed(1)
    q = torch.randn(n, Hq, D, generator=gd, device=DEV).to(dtype)
    k, v = (torch.randn(m, Hkv, D, generator=gd, device=DEV).to(dtype) for _ in range(2))
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = ops.prompt_attention(q, k, v, R.cu(lens).to(DEV), R.cu(keys).to(DEV), causal=causal, error_word=word)
    assert ops.read_error_word(word) == 0 and torch.isfinite(got).all()
    cq, ck = R.cu(lens).tolist(), R.cu(keys).tolist()
    order = sorted(range(len(lens)), key=lambda i: keys[i])
    for i in {0, 1, 2, 10, len(lens) - 1, order[-1], order[-2], order[len(order) // 2]} - {i for i, x in enumerate(lens) if not x}:
        a, b = slice(cq[i], cq[i + 1]), slice(ck[i], ck[i + 1])
        out, A, slack = prompt_reference(q[a].cpu(), k[b].cpu(), v[b].cpu(), [lens[i]], [keys[i]], causal, D ** -0.5)
        bound = UNIT[dtype] * (A + out.abs() * 1.001) + slack
        assert ((got[a].cpu().double() - out).abs() <= bound).all(), i


def test_each_prompt_item_is_done_once():
    """An integer pattern: with one key a sequence, every row is that key's value, exactly."""
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 600, (6 * sms(),), generator=g).tolist()
    for heads, D in ((2, 64), (1, 128)):
        v = torch.randint(-100, 100, (len(lens), heads, D), generator=g).half().to(DEV)
        q = torch.randn(sum(lens), heads, D, device=DEV).half()
        out = torch.full_like(q, float("nan"))
        ops.prompt_attention(q, torch.randn_like(v), v, R.cu(lens).to(DEV), R.cu([1] * len(lens)).to(DEV), causal=False, out=out)
        assert torch.equal(out, v.repeat_interleave(torch.tensor(lens, device=DEV), 0))


# ------------------------------------------------------------------------------- appends, gather
@pytest.mark.parametrize("tokens", [2, 5, 8])  # of a CTA
@pytest.mark.parametrize("Hq,Hkv,D,rot,bs", [(2, 1, 64, 64, 16), (1, 2, 128, 128, 8), (1, 1, 256, 128, 32)])
@pytest.mark.parametrize("dtype,interleaved", [(torch.float16, False), (torch.bfloat16, True), (torch.float32, False)])
def test_appends_and_gather_of_many_tokens(tokens, Hq, Hkv, D, rot, bs, dtype, interleaved):
    g = torch.Generator().manual_seed(tokens)
    want, lens = tokens * 16 * sms() + 3, []
    while sum(lens) < want:  # short, empty and a few longer ones, so that many end inside a CTA's tokens
        lens.append(int(torch.randint(0, 12, (1,), generator=g)) if len(lens) % 50 else int(torch.randint(100, 300, (1,), generator=g)))
    lens[-1] -= sum(lens) - want
    starts = [-1 if i % 17 == 5 else int(torch.randint(0, 40, (1,), generator=g)) for i in range(len(lens))]
    c = Case(lens, starts, Hq, Hkv, D, rot, bs, dtype, interleaved, seed=tokens)
    cu, err = c.cu.to(DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    want_q = c.rotated(c.q, torch.float32).to(dtype)
    want_q[~c.live] = 0
    at = (c.block[c.live], c.row[c.live])

    k0, v0 = (torch.randn(c.blocks, bs, Hkv, D, generator=g).to(dtype) for _ in range(2))
    kp, vp = k0.to(DEV), v0.to(DEV)
    q = ops.rope_kv_append(c.dq, c.dk, c.dv, *c.args, kp, vp, *c.where, cu_seqlens=cu, interleaved=interleaved, error_word=err)
    k0[at], v0[at] = c.rotated(c.k, torch.float32).to(dtype)[c.live], c.v[c.live]
    assert torch.equal(q.cpu(), want_q) and torch.equal(kp.cpu(), k0) and torch.equal(vp.cpu(), v0)

    pool = ops.kv_pool_int4(c.blocks, Hkv, D, bs)
    kc, kparam, vc, vparam = R.unpack(pool.cpu(), D, bs)
    q = ops.rope_kv_append_int4(c.dq, c.dk, c.dv, *c.args, pool, *c.where, cu_seqlens=cu, interleaved=interleaved, error_word=err)
    k_new, v_new = R.quantise(c.rotated(c.k, torch.float32)), R.quantise(c.v.float())
    kc[at], kparam[at], vc[at], vparam[at] = k_new[0][c.live], k_new[1][c.live], v_new[0][c.live], v_new[1][c.live]
    assert torch.equal(q.cpu(), want_q) and torch.equal(pool.cpu(), R.pack(kc, kparam, vc, vparam))

    k, v = ops.kv_gather_int4(pool, c.where[0], cu, sum(lens), D, dtype, starts=c.where[1], error_word=err)
    for got, new in ((k, k_new), (v, v_new)):
        values = R.values(*new).to(torch.float32).to(dtype)
        values[~c.live] = 0
        assert torch.equal(got.cpu(), values)
    assert ops.read_error_word(err) == 0


# ------------------------------------------------------------------------------- decode
@pytest.mark.parametrize("Hq,Hkv,D,bs", [(12, 12, 64, 16), (16, 2, 64, 8), (32, 8, 128, 16), (12, 2, 128, 32), (8, 8, 256, 16),
                                         (16, 1, 256, 8)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_decode_of_long_contexts_for_the_whole_device(Hq, Hkv, D, bs, dtype):
    """Tables that hold more than 4096 tokens for every CTA slot: chunks of 2048 to 4096, dealt out and joined."""
    slots, heads = sms() * {64: 4, 128: 3, 256: 2}[D], 4 if dtype == torch.float32 or Hq // Hkv <= 4 else 8
    tiles = Hkv * -(-(Hq // Hkv) // heads)
    longest = 9000
    B = 4100 * slots // (longest * tiles) + 2
    g = torch.Generator().manual_seed(Hq + D)
    columns = -(-longest // bs)
    assert columns * bs * B * tiles // slots > 4096
    pool, *_ = R.random_pool(g, 700, bs, Hkv, D)
    tables = torch.randint(0, 700, (B, columns), generator=g, dtype=torch.int32)
    lens = torch.randint(0, longest, (B,), generator=g)
    lens[:6] = torch.tensor([longest, 2048, 2049, 0, 1, 4097])
    q = torch.randn(B, Hq, D, generator=g).to(dtype)
    args = [t.to(DEV) for t in (q, pool, tables, lens.int())]
    ws = ops.decode_int4_workspace(B, Hq, Hkv, D, bs, columns, dtype, torch.device(DEV))
    got = ops.paged_decode_attention_int4(*args, workspace=ws)
    assert torch.isfinite(got).all() and ops.read_error_word(ws) == 0 and not ws[256 : 256 + 4 * B * Hq].any()
    assert torch.equal(got, ops.paged_decode_attention_int4(*args))
    u = 2.0 ** -22 if heads == 4 else 2.0 ** -11
    for b in (0, 1, 2, 3, 4, 5, B - 1):
        out, C, A, ds = decode_reference(q[b : b + 1], pool, tables[b : b + 1], [int(lens[b])], D, bs, D ** -0.5)
        bound = u * C + UNITS[dtype] * out.abs() * 1.001 + 2 * ds * A + 1e-6 * A
        assert ((got[b : b + 1].cpu().double() - out).abs() <= bound).all(), b
