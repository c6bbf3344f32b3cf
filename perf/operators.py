"""Cases, inputs and plain forms of the rotary, grouped-head and 4-bit-cache operators.

Five operators of ``speech_serving.ops`` that a decoder with rotary positions, grouped
key/value heads and a paged cache needs:

  prompt_attention             attention of whole packed prompts (causal or not, grouped heads,
                               keys longer than the queries where a prefix is cached)
  rope_kv_append               rotation of q and k, and k/v written to the paged 16/32-bit pools
  rope_kv_append_int4          the same into a paged 4-bit pool
  kv_gather_int4               tokens of a 4-bit pool back as packed k and v
  paged_decode_attention_int4  single-token attention over a 4-bit pool

``listed()`` names the measured cases, ``draw(rng)`` makes more of the same ranges,
``prepare(case, seed)`` makes a case's inputs on the GPU, ``run(state)`` is one pass (the
plain torch form, or with ``own`` the library's kernels), ``work(case)`` its bytes and
operations, ``exact(case, seed)`` the definition in 64 bits.

The 4-bit pool is uint8 [num_blocks][kv_heads][page bytes].  A page holds one block's tokens of
one head; with P = head_dim / 64 planes of 64 dimensions and bs tokens a block:
  K codes [P][bs][32 bytes], K (scale, zero) [P][bs][2 fp16], then V the same.
Byte b of a row holds dimension 2b in its low and 2b + 1 in its high half; the value of a code
c is c * scale + zero.
"""
import math
import random
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"fp16": 2, "bf16": 2, "fp32": 4}
PLANE = 64          # dimensions that share one scale and zero
ROW = PLANE // 2    # bytes of a token's codes in one plane


def _ops():
    if "inference-speech-model_b200" not in sys.path:
        sys.path.insert(0, "inference-speech-model_b200")
    from speech_serving import ops

    return ops


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # prompts of the decoder the benchmark serves (12 heads of 64, up to 448 positions):
        # a few short requests admitted together, where the launch counts
        dict(name="prompt short packed", op="prompt", B=6, lo=4, hi=224, cached=0, Hq=12, Hkv=12, D=64, dtype="fp16",
             causal=True, mix=1),
        # audio positions of 1500 each through 20 heads of 64, every position seeing all others
        dict(name="prompt audio 1500", op="prompt", B=8, lo=1500, hi=1500, cached=0, Hq=20, Hkv=20, D=64, dtype="fp16",
             causal=False, mix=2),
        # a ragged mix of grouped-head prompts, some continuing a cached prefix
        dict(name="prompt grouped ragged", op="prompt", B=13, lo=1, hi=2047, cached=1000, Hq=24, Hkv=4, D=128,
             dtype="bf16", causal=True, mix=3),
        # one long grouped-head prompt: the largest
        dict(name="prompt grouped 8192", op="prompt", B=1, lo=8192, hi=8192, cached=0, Hq=32, Hkv=8, D=128, dtype="bf16",
             causal=True, mix=4),
        # a decode step's new tokens into 16-bit pools: 64 requests, 12 heads of 64
        dict(name="append step 64", op="append", B=64, lo=1, hi=1, start=447, Hq=12, Hkv=12, D=64, rot=64, bs=16,
             dtype="fp16", interleaved=False, mix=5),
        # prompts admitted at once: 16 ragged ones, grouped heads, part of each head rotated
        dict(name="append prompts", op="append", B=16, lo=200, hi=2000, start=0, Hq=32, Hkv=8, D=128, rot=64, bs=16,
             dtype="bf16", interleaved=True, mix=6),
        # a decode step's new tokens into a 4-bit pool, and back: 48 requests
        dict(name="append4 step 48", op="append4", B=48, lo=1, hi=1, start=4000, Hq=32, Hkv=8, D=128, rot=128, bs=16,
             dtype="bf16", interleaved=False, mix=7),
        # long prompts into a 4-bit pool, and back
        dict(name="append4 prompts", op="append4", B=7, lo=500, hi=4001, start=100, Hq=16, Hkv=8, D=128, rot=128, bs=32,
             dtype="fp16", interleaved=False, mix=8),
        # one short cached prefix read back
        dict(name="gather4 prefix 448", op="gather4", B=2, lo=100, hi=448, start=0, Hkv=12, D=64, bs=16, dtype="fp16",
             mix=9),
        # the cached prefixes of a batch read back for its next prompt chunk
        dict(name="gather4 batch", op="gather4", B=16, lo=1000, hi=8000, start=0, Hkv=8, D=128, bs=16, dtype="bf16",
             mix=10),
        # one request's decode step over at most 448 positions: latency
        dict(name="decode4 one 448", op="decode4", B=1, lo=448, hi=448, Hq=12, Hkv=12, D=64, bs=16, dtype="fp16", mix=11),
        # a batch of long ragged contexts with grouped heads
        dict(name="decode4 long ragged", op="decode4", B=32, lo=1000, hi=32000, Hq=32, Hkv=8, D=128, bs=16, dtype="bf16",
             mix=12),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(12, 12), (20, 20), (6, 6), (32, 8), (16, 2), (24, 4), (8, 1), (10, 5)]  # query and key/value heads


def draw(rng):
    op = rng.choice(["prompt", "append", "append4", "gather4", "decode4"])
    Hq, Hkv = rng.choice(HEADS)
    c = dict(op=op, Hq=Hq, Hkv=Hkv, D=rng.choice([64, 128]), dtype=rng.choice(["fp16", "bf16"]), mix=rng.randrange(1 << 20))
    if op == "prompt":
        c["D"] = rng.choice([64, 64, 128, 128, 32, 80])
        c["B"] = _log(rng, 1, 24)
        c["hi"] = _log(rng, 8, max(8, int(8192 / math.sqrt(c["B"]))))
        c["lo"] = rng.randint(1, c["hi"])
        c["cached"] = rng.choice([0, 0, rng.randint(1, 2000)]) if c["hi"] <= 2048 else 0
        c["causal"] = rng.random() < 0.75
        return c
    c["bs"] = rng.choice([8, 16, 16, 32])
    if op in ("append", "append4"):
        if op == "append" and rng.random() < 0.25:
            c["dtype"] = "fp32"
        c["interleaved"] = rng.random() < 0.4
        c["rot"] = rng.choice([c["D"], c["D"], c["D"] // 2])
        c["start"] = _log(rng, 1, 4000) - 1
        c["B"] = _log(rng, 1, 256)
        step = rng.random() < 0.5
        c["hi"] = 1 if step else _log(rng, 2, max(2, min(4000, 20000 // c["B"])))
        c["lo"] = 1 if step else rng.randint(1, c["hi"])
        return c
    if op == "gather4":
        del c["Hq"]
        c["B"] = _log(rng, 1, 64)
        c["hi"] = _log(rng, 16, min(8000, 64000 // c["B"]))
        c["start"] = rng.choice([0, rng.randint(1, 100)])
    else:
        if rng.random() < 0.15:
            c["dtype"] = "fp32"
        c["B"] = _log(rng, 1, 128)
        c["hi"] = _log(rng, 16, min(32000, 500000 // c["B"]))
    c["lo"] = rng.randint(1, c["hi"])
    return c


def _lens(c):
    """The lengths of a case's sequences, and for prompts the cached tokens before each."""
    r = random.Random(c["mix"])
    lens = [r.randint(c["lo"], c["hi"]) for _ in range(c["B"])]
    lens[0] = c["hi"]
    cached = [r.randint(0, c["cached"]) if c.get("cached") else 0 for _ in lens]
    starts = [r.randint(0, c["start"]) if c.get("start") else 0 for _ in lens]
    return lens, cached, starts


def work(c):
    e = SIZE[c["dtype"]]
    lens, cached, starts = _lens(c)
    n, D, Hkv = sum(lens), c["D"], c["Hkv"]
    page_token = D // PLANE * 2 * (ROW + 4)  # bytes of one token of one head in a 4-bit pool, K and V
    if c["op"] == "prompt":
        Hq = c["Hq"]
        pairs = sum(q * p + (q * (q + 1) // 2 if c["causal"] else q * q) for q, p in zip(lens, cached))
        return dict(bytes=(2 * n * Hq + 2 * (n + sum(cached)) * Hkv) * D * e, flops=4 * pairs * Hq * D)
    if c["op"] == "append":
        return dict(bytes=(2 * c["Hq"] + 4 * Hkv) * n * D * e + n * c["rot"] * 4, flops=3 * n * (c["Hq"] + Hkv) * c["rot"])
    if c["op"] == "append4":  # rotated, quantised and written; then read and written as k and v
        return dict(bytes=(2 * c["Hq"] + 4 * Hkv) * n * D * e + 2 * n * Hkv * page_token + n * c["rot"] * 4,
                    flops=3 * n * (c["Hq"] + Hkv) * c["rot"] + 12 * n * Hkv * D)
    if c["op"] == "gather4":
        return dict(bytes=n * Hkv * (page_token + 2 * D * e), flops=4 * n * Hkv * D)
    return dict(bytes=n * Hkv * page_token + 2 * c["B"] * c["Hq"] * D * e, flops=4 * n * c["Hq"] * D)


# ------------------------------------------------------------------------------- inputs
def _cu(lens):
    return torch.tensor([0] + lens, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(DEV)


def _tables(g, ends, bs):
    """Block tables of sequences of `ends` tokens over a pool with a few blocks to spare."""
    most = max(1, -(-max(ends) // bs))
    blocks = len(ends) * most + 3
    perm = torch.randperm(blocks, generator=g, device=DEV)[: len(ends) * most]
    return perm.view(len(ends), most).to(torch.int32), blocks


def _angles(positions, rot):
    inv = 10000.0 ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
    a = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * inv
    return a.cos().float(), a.sin().float()


def _quantise(x):
    """fp32 [..., D] -> codes uint8 [..., D], scale and zero fp16 [..., D / 64]."""
    x = x.unflatten(-1, (-1, PLANE))
    least, most = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = ((most - least) / 15.0).clamp(max=65504.0).half()
    zero = least.clamp(-65504.0, 65504.0).half()
    steps = (x - zero.float()) / scale.float()
    codes = torch.where(scale > 0, steps.round().clamp(0.0, 15.0), 0.0).to(torch.uint8)
    return codes.flatten(-2), scale[..., 0], zero[..., 0]


def _pages(k, v):
    """fp32 k, v [blocks, bs, heads, D] -> the 4-bit pool that holds them."""
    parts = []
    for x in (k, v):
        codes, scale, zero = _quantise(x)
        codes = codes[..., 0::2] | (codes[..., 1::2] << 4)
        codes = codes.unflatten(-1, (-1, ROW)).permute(0, 2, 3, 1, 4)     # [blocks, heads, P, bs, 32]
        sz = torch.stack((scale, zero), -1).permute(0, 2, 3, 1, 4)        # [blocks, heads, P, bs, 2]
        parts += [codes.flatten(2), sz.contiguous().view(torch.uint8).flatten(2)]
    return torch.cat(parts, 2).contiguous()


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    lens, cached, starts = _lens(c)
    n, D, Hkv, Hq = sum(lens), c["D"], c["Hkv"], c.get("Hq", 0)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    s = dict(c, lens=lens, n=n, dt=dt)
    if c["op"] == "prompt":
        s["cu_q"] = _cu(lens)
        if any(cached):  # keys and values of the prefix and the prompt, packed; queries of the prompt alone
            keys = [a + b for a, b in zip(lens, cached)]
            s["cu_k"] = _cu(keys)
            s["q"] = rand(n, Hq, D).to(dt)
            s["k"], s["v"] = rand(sum(keys), Hkv, D).to(dt), rand(sum(keys), Hkv, D).to(dt)
        else:            # views of one packed projection, as a q|k|v weight gives
            keys = lens
            s["cu_k"] = s["cu_q"]
            qkv = rand(n, Hq + 2 * Hkv, D).to(dt)
            s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq : Hq + Hkv], qkv[:, Hq + Hkv :]
        s["most_q"], s["most_k"] = max(lens), max(keys)
        return s
    if c["op"] == "decode4":
        s["tables"], blocks = _tables(g, lens, c["bs"])
        # new inputs are made block by block of the pool from a smaller set of random rows
        few = min(blocks, 512)
        pool = _pages(rand(few, c["bs"], Hkv, D), rand(few, c["bs"], Hkv, D))
        s["pool"] = pool[torch.randint(few, (blocks,), generator=g, device=DEV)]
        s["q"] = rand(c["B"], Hq, D).to(dt)
        s["ctx"] = torch.tensor(lens, dtype=torch.int32).to(DEV)
        return s
    s["starts"] = torch.tensor(starts, dtype=torch.int32).to(DEV)
    s["cu"] = _cu(lens)
    s["step"] = c["op"] != "gather4" and c["hi"] == 1  # one token a sequence: no packed lengths
    ends = [a + b for a, b in zip(starts, lens)]
    if c["op"] == "gather4":
        s["tables"], blocks = _tables(g, ends, c["bs"])
        few = min(blocks, 512)
        pool = _pages(rand(few, c["bs"], Hkv, D), rand(few, c["bs"], Hkv, D))
        s["pool"] = pool[torch.randint(few, (blocks,), generator=g, device=DEV)]
        return s
    # for a step only the blocks that hold the new tokens are in use; the tables have all columns
    s["tables"], blocks = _tables(g, ends, c["bs"])
    s["cos"], s["sin"] = _angles(max(ends), c["rot"])
    qkv = rand(n, Hq + 2 * Hkv, D).to(dt)
    s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq : Hq + Hkv], qkv[:, Hq + Hkv :]
    if c["op"] == "append":
        # a step's pool: one block a sequence, since the pools come back whole
        if s["step"]:
            blocks = c["B"] + 3
            s["tables"] = (torch.randperm(blocks, generator=g, device=DEV)[: c["B"], None]
                           .expand(-1, s["tables"].shape[1]).to(torch.int32).contiguous())
        s["k_pool"] = rand(blocks, c["bs"], Hkv, D).to(dt)
        s["v_pool"] = rand(blocks, c["bs"], Hkv, D).to(dt)
    else:
        s["pool"] = torch.zeros(blocks, Hkv, D // PLANE * c["bs"] * 2 * (ROW + 4), dtype=torch.uint8, device=DEV)
    return s


# ------------------------------------------------------------------------------- plain forms
def _prompt(s):
    B, Tq, Tk, Hq, Hkv, D = s["B"], s["most_q"], s["most_k"], s["Hq"], s["Hkv"], s["D"]
    cq, ck = s["cu_q"].long(), s["cu_k"].long()
    nq, nk = cq.diff()[:, None], ck.diff()[:, None]
    iq, ik = torch.arange(Tq, device=DEV), torch.arange(Tk, device=DEV)
    # padded [B, heads, tokens, D] in 32 bits
    rows_q = (cq[:-1, None] + iq).clamp(max=s["q"].shape[0] - 1)
    rows_k = (ck[:-1, None] + ik).clamp(max=s["k"].shape[0] - 1)
    q = s["q"][rows_q].float().permute(0, 2, 1, 3).reshape(B, Hkv, Hq // Hkv * Tq, D)
    k = s["k"][rows_k].float().permute(0, 2, 3, 1)
    v = s["v"][rows_k].float().permute(0, 2, 1, 3)
    w = (q @ k).mul_(1.0 / math.sqrt(D)).view(B, Hkv, Hq // Hkv, Tq, Tk)
    seen = (ik < nk)[:, None, :].expand(B, Tq, Tk)
    if s["causal"]:
        seen = seen & (ik <= (iq + nk - nq)[:, :, None])
    w.masked_fill_(~seen[:, None, None], -math.inf)
    w.sub_(w.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = w.sum(-1, keepdim=True)
    out = (w.view(B, Hkv, -1, Tk) @ v).view(B, Hkv, Hq // Hkv, Tq, D) / total.clamp(min=1e-30)
    out = out.flatten(1, 2).permute(0, 2, 1, 3)  # [B, Tq, Hq, D]
    return out[iq < nq].to(s["dt"])


def _token_places(s):
    """For each packed token its sequence, its position, and the block and row that hold it."""
    cu = s["cu"].long()
    i = torch.arange(s["n"], device=DEV)
    b = torch.searchsorted(cu[1:], i, right=True)
    pos = s["starts"].long()[b] + i - cu[b]
    block = s["tables"].long()[b, pos // s["bs"]]
    return pos, block, pos % s["bs"]


def _rotate(x, cos, sin, interleaved):
    rot = 2 * cos.shape[-1]
    x, c, d = x.float(), cos[:, None], sin[:, None]
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack((a * c - b * d, b * c + a * d), -1).flatten(-2)
    else:
        a, b = x[..., : rot // 2], x[..., rot // 2 : rot]
        y = torch.cat((a * c - b * d, b * c + a * d), -1)
    return torch.cat((y, x[..., rot:]), -1)


def _page_views(s):
    """The pool as codes [blocks, heads, P, bs, 32] and scale/zero [blocks, heads, P, bs, 2], for K and V."""
    pool, bs, P = s["pool"], s["bs"], s["D"] // PLANE
    codes, sz = P * bs * ROW, P * bs * 4
    found = []
    at = [0, codes + sz]
    for o in (0, 1):
        found.append(pool[..., at[o] : at[o] + codes].unflatten(-1, (P, bs, ROW)))
        found.append(pool.view(torch.float16)[..., (at[o] + codes) // 2 : (at[o] + codes + sz) // 2].unflatten(-1, (P, bs, 2)))
    return found


def _values(codes, sz):
    """[..., P, 32] codes and [..., P, 2] scale/zero -> fp32 [..., D]."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
    return (c * sz[..., :1].float() + sz[..., 1:].float()).flatten(-2)


def _gather(s):
    _, block, row = _token_places(s)
    kc, ks, vc, vs = (x.transpose(1, 3)[block, row].transpose(1, 2) for x in _page_views(s))  # [n, heads, P, ...]
    return [_values(kc, ks).to(s["dt"]), _values(vc, vs).to(s["dt"])]


def _append(s):
    pos, block, row = _token_places(s)
    cos, sin = s["cos"][pos], s["sin"][pos]
    q = _rotate(s["q"], cos, sin, s["interleaved"]).to(s["dt"])
    k = _rotate(s["k"], cos, sin, s["interleaved"])
    if s["op"] == "append":
        s["k_pool"][block, row] = k.to(s["dt"])
        s["v_pool"][block, row] = s["v"]
        return [q, s["k_pool"], s["v_pool"]]
    kc, ks, vc, vs = _page_views(s)
    for x, codes_at, sz_at in ((k, kc, ks), (s["v"].float(), vc, vs)):
        codes, scale, zero = _quantise(x)
        codes = (codes[..., 0::2] | (codes[..., 1::2] << 4)).unflatten(-1, (-1, ROW))     # [n, heads, P, 32]
        codes_at.transpose(1, 3)[block, row] = codes.transpose(1, 2)
        sz_at.transpose(1, 3)[block, row] = torch.stack((scale, zero), -1).transpose(1, 2)
    return [q] + _gather(s)


def _decode(s):
    B, Hq, Hkv, D = s["B"], s["Hq"], s["Hkv"], s["D"]
    tables = s["tables"].long()
    # [B, blocks, heads, P, bs, ...] -> [B, heads, blocks * bs, D]
    kc, ks, vc, vs = (x[tables].permute(0, 2, 1, 4, 3, 5) for x in _page_views(s))
    k = _values(kc, ks).flatten(2, 3)
    v = _values(vc, vs).flatten(2, 3)
    q = s["q"].float().view(B, Hkv, Hq // Hkv, D)
    w = (q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(D))
    seen = torch.arange(k.shape[2], device=DEV) < s["ctx"][:, None]
    w = w.masked_fill(~seen[:, None, None], -math.inf)
    w = (w - w.amax(-1, keepdim=True).clamp(min=-1e30)).exp()
    out = (w @ v.masked_fill(~seen[:, None, :, None], 0.0)) / w.sum(-1, keepdim=True).clamp(min=1e-30)
    return out.view(B, Hq, D).to(s["dt"])


def run(s):
    if not own:
        return {"prompt": _prompt, "append": _append, "append4": _append, "gather4": _gather, "decode4": _decode}[s["op"]](s)
    ops = _ops()
    if s["op"] == "prompt":
        return ops.prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=s["causal"])
    if s["op"] == "decode4":
        return ops.paged_decode_attention_int4(s["q"], s["pool"], s["tables"], s["ctx"])
    if s["op"] == "gather4":
        return list(ops.kv_gather_int4(s["pool"], s["tables"], s["cu"], s["n"], s["D"], s["dt"], starts=s["starts"]))
    cu = None if s["step"] else s["cu"]
    if s["op"] == "append":
        q = ops.rope_kv_append(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["k_pool"], s["v_pool"], s["tables"],
                               s["starts"], cu_seqlens=cu, interleaved=s["interleaved"])
        return [q, s["k_pool"], s["v_pool"]]
    q = ops.rope_kv_append_int4(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["pool"], s["tables"], s["starts"],
                                cu_seqlens=cu, interleaved=s["interleaved"])
    return [q] + list(ops.kv_gather_int4(s["pool"], s["tables"], s["cu"], s["n"], s["D"], s["dt"], starts=s["starts"]))


# ------------------------------------------------------------------------------- 64 bits
def _softmax_rows(scores, v):
    p = torch.softmax(scores, -1)
    return torch.nan_to_num(p, nan=0.0) @ v


def _decode_words(pool, P, bs, second):
    """float64 [blocks, heads, bs, D] of the K (second = 0) or V (1) half of every page, word by word."""
    half = pool.view(torch.int32).flatten(2)
    words = P * bs * ROW // 4
    at = second * (words + P * bs)
    w = half[..., at : at + words].unflatten(-1, (P, bs, ROW // 4)).long() & 0xFFFFFFFF
    codes = torch.stack([(w >> (4 * j)) & 15 for j in range(8)], -1).flatten(-2).double()
    sz = half[..., at + words : at + words + P * bs].contiguous().view(torch.float16).unflatten(-1, (P, bs, 2)).double()
    return (codes * sz[..., :1] + sz[..., 1:]).permute(0, 1, 3, 2, 4).flatten(-2)


def exact(c, seed):
    s = prepare(c, seed)
    lens, cached, starts = _lens(c)
    D, Hkv = c["D"], c["Hkv"]
    if c["op"] == "prompt":
        G, outs, a, b = c["Hq"] // Hkv, [], 0, 0
        for n, p in zip(lens, cached):
            q, k, v = s["q"][a : a + n].double(), s["k"][b : b + n + p].double(), s["v"][b : b + n + p].double()
            heads = []
            for h in range(c["Hq"]):
                w = q[:, h] @ k[:, h // G].T / math.sqrt(D)
                if c["causal"]:
                    w = w.masked_fill(torch.ones(n, n + p, device=DEV, dtype=torch.bool).triu(p + 1), -math.inf)
                heads.append(_softmax_rows(w, v[:, h // G]))
            outs.append(torch.stack(heads, 1))
            a, b = a + n, b + n + p
        return torch.cat(outs)
    P, bs = D // PLANE, c["bs"]
    if c["op"] == "decode4":
        outs = []
        for i, n in enumerate(lens):
            pages = s["pool"][s["tables"][i].long()]
            k, v = (_decode_words(pages, P, bs, o).transpose(1, 2).flatten(0, 1)[:n].transpose(0, 1) for o in (0, 1))
            q = s["q"][i].double().view(Hkv, -1, D)
            outs.append(_softmax_rows(q @ k.transpose(1, 2) / math.sqrt(D), v).reshape(-1, D))
        return torch.stack(outs)
    if c["op"] == "gather4":
        both = []
        for o in (0, 1):
            rows = []
            for i, n in enumerate(lens):
                x = _decode_words(s["pool"][s["tables"][i].long()], P, bs, o).transpose(1, 2).flatten(0, 1)
                rows.append(x[starts[i] : starts[i] + n])
            both.append(torch.cat(rows))
        return both
    # the rotation as a product of complex numbers
    pos = torch.cat([torch.arange(a, a + n, device=DEV) for a, n in zip(starts, lens)])
    turn = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
    half = c["rot"] // 2

    def rotated(x):
        x = x.double()
        r, rest = x[..., : c["rot"]], x[..., c["rot"] :]
        if c["interleaved"]:
            y = torch.view_as_real(torch.view_as_complex(r.unflatten(-1, (half, 2)).contiguous()) * turn).flatten(-2)
        else:
            z = torch.complex(r[..., :half].contiguous(), r[..., half:].contiguous()) * turn
            y = torch.cat((z.real, z.imag), -1)
        return torch.cat((y, rest), -1)

    q, k, v = rotated(s["q"]), rotated(s["k"]), s["v"].double()
    if c["op"] == "append":
        k_pool, v_pool = s["k_pool"].double(), s["v_pool"].double()
        a = 0
        for i, n in enumerate(lens):
            p = torch.arange(starts[i], starts[i] + n, device=DEV)
            block = s["tables"][i].long()[p // bs]
            k_pool[block, p % bs], v_pool[block, p % bs] = k[a : a + n], v[a : a + n]
            a += n
        return [q, k_pool, v_pool]

    def kept(x):  # through 4 bits: 15 steps between the least and the largest of each 64 values
        x = x.unflatten(-1, (P, PLANE))
        least = x.amin(-1, keepdim=True)
        step = ((x.amax(-1, keepdim=True) - least) / 15).half().double()
        least = least.half().double()
        return (((x - least) / step).round().clamp(0, 15) * step + least).flatten(-2)

    return [q, kept(k), kept(v)]
