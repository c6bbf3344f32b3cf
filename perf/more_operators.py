"""Cases, inputs and plain forms of the operators that decode several candidates of one request.

Three operators of ``speech_serving.ops`` for candidates (samples, beams) that share a prompt or an
encoder's output:

  shared_prefix_decode_attention  single-token attention with grouped heads over a paged 16-bit cache:
                                  the keys of a prefix that a group of sequences shares, and each
                                  sequence's own
  cross_attention_packed          any number of queries a request (beams, prompt tokens) over the
                                  encoder keys and values of the request's slot, each of its own length
  sample_rows                     a token a row by temperature, top-k, top-p and min-p from a given
                                  random number, and its log-probability

``listed()`` names the measured cases, ``draw(rng)`` makes more of the same ranges,
``prepare(case, seed)`` makes a case's inputs on the GPU, ``run(state)`` is one pass (the
plain torch form, or with ``own`` the library's kernels), ``work(case)`` its bytes and
operations, ``exact(case, seed)`` the definition in 64 bits.

A row of sample_rows with the values x of its columns (those of ``skip`` count as -inf), their largest
m, a temperature t and a random number u:
  t <= 0, or m not finite: the first largest column, as argmax_rows picks it;
  otherwise, with w = exp((x - m) / t) and the columns sorted by x (the largest first, equal ones by
  their place): top_k > 0 leaves the first top_k; of these top_p < 1 leaves those before which less than
  top_p of their weight lies (at least one); of these min_p > 0 leaves those with x >= m + t log(min_p)
  (at least one).  The token is the first column, by its place, at which the weight of what is left so
  far passes u times all of it.  The log-probability is that of the token under softmax(x).
"""
import math
import random
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"fp16": 2, "bf16": 2, "fp32": 4}


def _ops():
    if "inference-speech-model_b200" not in sys.path:
        sys.path.insert(0, "inference-speech-model_b200")
    from speech_serving import ops

    return ops


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # eight candidates of one short request of the decoder the benchmark serves (12 heads of 64, up to
        # 448 positions): latency
        dict(name="prefix one request", op="prefix", G=1, least=8, most=8, plo=400, phi=400, lo=1, hi=48, Hq=12, Hkv=12,
             D=64, bs=16, dtype="fp16", mix=1),
        # four audio prompts of 1500 positions, five candidates each, up to 224 tokens of their own
        dict(name="prefix audio 1500", op="prefix", G=4, least=5, most=5, plo=1500, phi=1500, lo=20, hi=224, Hq=20, Hkv=20,
             D=64, bs=16, dtype="fp16", mix=2),
        # a ragged mix of prompts and of candidates a prompt, grouped heads
        dict(name="prefix grouped ragged", op="prefix", G=12, least=1, most=24, plo=100, phi=6000, lo=1, hi=700, Hq=24, Hkv=4,
             D=128, bs=16, dtype="bf16", mix=3),
        # two long prompts with 64 candidates each: the largest
        dict(name="prefix long 32000", op="prefix", G=2, least=64, most=64, plo=30000, phi=32000, lo=100, hi=1000, Hq=32,
             Hkv=8, D=128, bs=32, dtype="bf16", mix=4),
        # five beams of one request over its audio: latency
        dict(name="cross one request", op="cross", B=1, least=5, most=5, vlo=1500, vhi=1500, T=1500, H=12, Hkv=12, D=64,
             dtype="fp16", mix=5),
        # five beams of each of 32 requests, ragged audio
        dict(name="cross beams 32", op="cross", B=32, least=5, most=5, vlo=100, vhi=1500, T=1500, H=20, Hkv=20, D=64,
             dtype="bf16", mix=6),
        # prompts of 24 requests (text so far, up to 448 tokens) over their audio
        dict(name="cross prompts 24", op="cross", B=24, least=1, most=448, vlo=100, vhi=1500, T=1500, H=20, Hkv=20, D=64,
             dtype="fp16", mix=7),
        # one request's next token, top-p alone: latency
        dict(name="sample one 51865", op="sample", rows=1, cols=51865, ld=51865, dtype="fp32", how="p", spread=3.0, skip=90,
             mix=8),
        # a decode step of 64 requests, each with settings of its own
        dict(name="sample step 64", op="sample", rows=64, cols=51865, ld=51872, dtype="fp16", how="mixed", spread=3.0,
             skip=90, mix=9),
        # candidates of 192 sequences over a large vocabulary: top-k with top-p
        dict(name="sample 192 top-k", op="sample", rows=192, cols=128257, ld=128264, dtype="bf16", how="k", spread=2.5, skip=0,
             mix=10),
        # a large vocabulary in fp32: top-p and min-p alone, flatter rows
        dict(name="sample 96 top-p", op="sample", rows=96, cols=200019, ld=200019, dtype="fp32", how="mixed p", spread=1.5,
             skip=7, mix=11),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(12, 12), (20, 20), (6, 6), (32, 8), (16, 2), (24, 4), (8, 1), (10, 5)]  # query and key/value heads


def draw(rng):
    op = rng.choice(["prefix", "prefix", "cross", "sample", "sample"])
    c = dict(op=op, dtype=rng.choice(["fp16", "bf16"]), mix=rng.randrange(1 << 20))
    if op == "prefix":
        c["Hq"], c["Hkv"] = rng.choice(HEADS)
        c["D"], c["bs"] = rng.choice([64, 64, 128, 128, 32, 80]), rng.choice([8, 16, 16, 32])
        c["G"] = _log(rng, 1, 16)
        c["most"] = _log(rng, 1, max(1, 128 // c["G"]))
        c["least"] = rng.randint(1, c["most"])
        c["phi"] = _log(rng, 16, 48000 // c["G"])
        c["plo"] = rng.choice([rng.randint(0, c["phi"]), c["phi"]])
        c["hi"] = _log(rng, 1, min(1500, 60000 // (c["G"] * c["most"])))
        c["lo"] = rng.randint(0, c["hi"])
    elif op == "cross":
        c["H"], c["Hkv"] = rng.choice([(12, 12), (20, 20), (6, 6), (16, 4), (8, 8)])
        c["D"] = rng.choice([64, 64, 64, 128, 32, 80])
        c["T"] = rng.choice([1500, 1500, rng.randint(10, 3000)])
        c["vhi"] = c["T"]
        c["vlo"] = rng.choice([c["T"], rng.randint(0, c["T"])])
        c["B"] = _log(rng, 1, 48)
        c["most"] = _log(rng, 1, max(8, min(448, 6000 // c["B"])))
        c["least"] = rng.choice([c["most"], rng.randint(0, c["most"])])
    else:
        c["dtype"] = rng.choice(["fp16", "bf16", "fp32"])
        c["cols"] = _log(rng, 1000, 200000)
        c["ld"] = c["cols"] + rng.choice([0, 0, rng.randint(1, 100), -c["cols"] % 8])
        c["rows"] = _log(rng, 1, max(2, min(256, 19000000 // c["cols"])))
        c["how"] = rng.choice(["p", "k", "mixed", "mixed p", "plain"])
        c["spread"] = rng.uniform(1.0, 4.0)
        c["skip"] = rng.choice([0, rng.randint(1, 200)])
    return c


def _lens(c):
    """Prefix: members of each group, prefix lengths, own lengths.  Cross: queries and valid lengths."""
    r = random.Random(c["mix"])
    if c["op"] == "prefix":
        members = [r.randint(c["least"], c["most"]) for _ in range(c["G"])]
        members[0] = c["most"]
        prefix = [r.randint(c["plo"], c["phi"]) for _ in members]
        prefix[0] = c["phi"]
        mine = [r.randint(c["lo"], c["hi"]) for _ in range(sum(members))]
        mine[0] = c["hi"]
        return members, prefix, mine
    queries = [r.randint(c["least"], c["most"]) for _ in range(c["B"])]
    queries[0] = c["most"]
    valid = [r.randint(c["vlo"], c["vhi"]) for _ in queries]
    valid[0] = c["vhi"]
    return queries, valid


def work(c):
    e = SIZE[c["dtype"]]
    if c["op"] == "sample":
        return dict(bytes=c["rows"] * (c["cols"] * e + 32) + (c["cols"] if c["skip"] else 0), flops=6 * c["rows"] * c["cols"])
    if c["op"] == "prefix":
        members, prefix, mine = _lens(c)
        B, keys = len(mine), sum(prefix) + sum(mine)
        pairs = sum(m * p for m, p in zip(members, prefix)) + sum(mine)
        return dict(bytes=(2 * B * c["Hq"] + 2 * keys * c["Hkv"]) * c["D"] * e, flops=4 * pairs * c["Hq"] * c["D"])
    queries, valid = _lens(c)
    keys = sum(v for q, v in zip(queries, valid) if q)
    return dict(bytes=(2 * sum(queries) * c["H"] + 2 * keys * c["Hkv"]) * c["D"] * e,
                flops=4 * sum(q * v for q, v in zip(queries, valid)) * c["H"] * c["D"])


# ------------------------------------------------------------------------------- inputs
def _cu(lens):
    return torch.tensor([0] + lens, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(DEV)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32).to(DEV)


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[c["dtype"]]

    def rand(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    s = dict(c, dt=dt)
    if c["op"] == "prefix":
        members, prefix, mine = _lens(c)
        B, bs = len(mine), c["bs"]
        s["B"], s["most_members"] = B, max(members)
        cols_p, cols_o = max(1, -(-max(prefix) // bs)), max(1, -(-max(mine) // bs))
        blocks = c["G"] * cols_p + B * cols_o + 3  # one pool: a few blocks to spare
        perm = torch.randperm(blocks, generator=g, device=DEV).to(torch.int32)
        s["ptab"] = perm[: c["G"] * cols_p].view(c["G"], cols_p).contiguous()
        s["tab"] = perm[c["G"] * cols_p : c["G"] * cols_p + B * cols_o].view(B, cols_o).contiguous()
        s["k_pool"], s["v_pool"] = (rand(blocks, bs, c["Hkv"], c["D"]).to(dt) for _ in range(2))
        s["q"] = rand(B, c["Hq"], c["D"]).to(dt)
        s["plens"], s["lens"], s["cu"] = _ints(prefix), _ints(mine), _cu(members)
        return s
    if c["op"] == "cross":
        queries, valid = _lens(c)
        slots = c["B"] + 2  # the slot layout of one layer, [slots, 2, heads, T, D]; requests lie in any order
        kv = rand(slots, 2, c["Hkv"], c["T"], c["D"]).to(dt)
        s["k"], s["v"] = kv[:, 0], kv[:, 1]
        s["slots"] = torch.randperm(slots, generator=g, device=DEV)[: c["B"]].to(torch.int32)
        s["q"] = rand(sum(queries), c["H"], c["D"]).to(dt)
        s["cu"], s["valid"] = _cu(queries), _ints(valid)
        s["most_q"] = max(queries)
        return s
    rows, cols = c["rows"], c["cols"]
    # rows as a language model's: a broad mass of columns, a few dozen that stand out by more or less
    x = rand(rows, c["ld"]).mul_(c["spread"])
    at = torch.randint(cols, (rows, 40), generator=g, device=DEV)
    x.scatter_add_(1, at, torch.rand(rows, 40, generator=g, device=DEV) * (torch.rand(rows, 1, generator=g, device=DEV) * 18))
    s["x"] = x.to(dt)
    s["u"] = torch.rand(rows, generator=g, device=DEV)
    s["skip"] = None
    if c["skip"]:
        s["skip"] = torch.zeros(cols, dtype=torch.bool, device=DEV)
        s["skip"][torch.randint(cols, (c["skip"],), generator=g, device=DEV)] = True

    def between(lo, hi):
        return torch.rand(rows, generator=g, device=DEV) * (hi - lo) + lo

    def some(share, values, other):
        return torch.where(torch.rand(rows, generator=g, device=DEV) < share, values, torch.full_like(values, other))

    how = c["how"]
    s["t"] = between(0.5, 1.3)
    k = between(0.0, 1.0).mul_(math.log(400.0)).exp_().to(torch.int32)  # 1 to 400
    p, least = between(0.7, 0.99), between(0.01, 0.2)
    zero = torch.zeros(rows, device=DEV)
    s["k"] = {"k": k, "mixed": some(0.5, k, 0)}.get(how, zero.to(torch.int32))
    s["p"] = {"p": p, "k": some(0.7, p, 1.0), "mixed": some(0.6, p, 1.0), "mixed p": some(0.7, p, 1.0)}.get(how, zero + 1.0)
    s["least"] = {"mixed": some(0.3, least, 0.0), "mixed p": some(0.4, least, 0.0)}.get(how, zero)
    if how == "mixed":
        s["t"] = some(0.9, s["t"], 0.0)  # a few greedy rows
    return s


# ------------------------------------------------------------------------------- plain forms
def _pages(pool, tables):
    """The blocks of each table's row, side by side, [rows, heads, tokens, D] in 32 bits."""
    return pool[tables.long()].flatten(1, 2).permute(0, 2, 1, 3).float()


def _prefix(s):
    B, G, Hq, Hkv, D, M = s["B"], s["G"], s["Hq"], s["Hkv"], s["D"], s["most_members"]
    cu = s["cu"].long()
    b = torch.arange(B, device=DEV)
    group = torch.searchsorted(cu[1:], b, right=True)
    place = group * M + b - cu[group]                       # in the groups padded to M members
    q = s["q"].float().mul(1.0 / math.sqrt(D)).view(B, Hkv, Hq // Hkv, D)
    kp, vp = _pages(s["k_pool"], s["ptab"]), _pages(s["v_pool"], s["ptab"])
    ko, vo = _pages(s["k_pool"], s["tab"]), _pages(s["v_pool"], s["tab"])
    qp = torch.zeros(G * M, Hkv, Hq // Hkv, D, device=DEV)
    qp[place] = q
    qp = qp.view(G, M, Hkv, -1, D).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [G, Hkv, M * heads, D]
    wp = qp @ kp.transpose(-1, -2)
    wp.masked_fill_((torch.arange(kp.shape[2], device=DEV) >= s["plens"][:, None])[:, None, None], -math.inf)
    wo = q @ ko.transpose(-1, -2)                           # [B, Hkv, heads, own keys]
    wo.masked_fill_((torch.arange(ko.shape[2], device=DEV) >= s["lens"][:, None])[:, None, None], -math.inf)

    def of_groups(x):  # [G, Hkv, M * heads, n] -> [B, Hkv, heads, n]
        return x.unflatten(2, (M, -1)).transpose(1, 2).flatten(0, 1)[place]

    def to_groups(x):
        y = torch.zeros(G * M, *x.shape[1:], device=DEV)
        y[place] = x
        return y.view(G, M, *x.shape[1:]).transpose(1, 2).flatten(2, 3)

    m = torch.maximum(of_groups(wp.amax(-1, keepdim=True)), wo.amax(-1, keepdim=True)).clamp(min=-1e30)
    wp.sub_(to_groups(m)).exp_()
    wo.sub_(m).exp_()
    total = of_groups(wp.sum(-1, keepdim=True)) + wo.sum(-1, keepdim=True)
    out = (of_groups(wp @ vp) + wo @ vo) / total.clamp(min=1e-30)
    return out.reshape(B, Hq, D).to(s["dt"])


def _cross(s):
    B, Tq, H, Hkv, D = s["B"], s["most_q"], s["H"], s["Hkv"], s["D"]
    cu = s["cu"].long()
    i = torch.arange(Tq, device=DEV)
    there = i < cu.diff()[:, None]
    rows = (cu[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][rows].float().mul(1.0 / math.sqrt(D)).permute(0, 2, 1, 3).reshape(B, Hkv, H // Hkv * Tq, D)
    k, v = s["k"][s["slots"].long()].float(), s["v"][s["slots"].long()].float()
    w = q @ k.transpose(-1, -2)
    w.masked_fill_((torch.arange(s["T"], device=DEV) >= s["valid"][:, None])[:, None, None], -math.inf)
    w.sub_(w.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    out = (w @ v) / w.sum(-1, keepdim=True).clamp(min=1e-30)
    return out.view(B, H, Tq, D).transpose(1, 2)[there].to(s["dt"])


def _sample(s):
    x = s["x"][:, : s["cols"]].float()
    if s["skip"] is not None:
        x = x.masked_fill(s["skip"], -math.inf)
    m = x.amax(-1, keepdim=True).double()
    t = s["t"].double()[:, None]
    greedy = (t <= 0)[:, 0]
    t = torch.where(t > 0, t, 1.0)
    ranked, order = torch.sort(x, dim=-1, descending=True, stable=True)
    ranked = ranked.double()
    w = ((ranked - m) / t).exp()
    place = torch.arange(s["cols"], device=DEV)
    k = s["k"].long()[:, None]
    kept = (k <= 0) | (place < k)
    w = w * kept
    cum = w.cumsum(-1)
    p = s["p"].double()[:, None]
    kept = kept & ((p >= 1) | (cum - w < p * cum[:, -1:]) | (place == 0))
    least = s["least"].double()[:, None]
    kept = kept & ((least <= 0) | (ranked >= m + t * least.clamp(min=1e-300).log()) | (place == 0))
    # back to the columns' own places
    w = torch.zeros_like(w).scatter_(1, order, w * kept)
    kept = torch.zeros_like(kept).scatter_(1, order, kept)
    cum = w.cumsum(-1)
    passed = kept & (cum > s["u"].double()[:, None] * cum[:, -1:])
    first = torch.where(passed, place, s["cols"]).amin(-1)
    last = torch.where(kept, place, -1).amax(-1)
    token = torch.where(first < s["cols"], first, last)
    token = torch.where(greedy, order[:, 0], token)
    x = x.double()
    logprob = (x.gather(1, token[:, None]) - m - (x - m).exp().sum(-1, keepdim=True).log())[:, 0].float()
    return [token, logprob]


def run(s):
    if not own:
        return {"prefix": _prefix, "cross": _cross, "sample": _sample}[s["op"]](s)
    ops = _ops()
    if s["op"] == "prefix":
        return ops.shared_prefix_decode_attention(s["q"], s["k_pool"], s["v_pool"], s["ptab"], s["plens"], s["cu"], s["tab"],
                                                  s["lens"])
    if s["op"] == "cross":
        return ops.cross_attention_packed(s["q"], s["k"], s["v"], s["valid"], s["cu"], slot_ids=s["slots"])
    logprobs = torch.empty(s["rows"], dtype=torch.float32, device=DEV)
    token = ops.sample_rows(s["x"], s["u"], temperature=s["t"], top_k=s["k"], top_p=s["p"], min_p=s["least"], cols=s["cols"],
                            skip=s["skip"], logprobs=logprobs)
    return [token, logprobs]


# ------------------------------------------------------------------------------- 64 bits
def _attend(q, k, v):
    """q [n, Hq, D], k and v [keys, Hkv, D] in 64 bits, every query over every key."""
    n, Hq, D = q.shape
    Hkv = k.shape[1]
    if k.shape[0] == 0:
        return torch.zeros_like(q)
    heads = []
    for h in range(Hq):
        kv = h // (Hq // Hkv)
        heads.append(torch.softmax(q[:, h] @ k[:, kv].T / math.sqrt(D), -1) @ v[:, kv])
    return torch.stack(heads, 1)


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "prefix":
        members, prefix, mine = _lens(c)
        if sum(mine) + sum(m * p for m, p in zip(members, prefix)) > 8_000_000:
            return None
        kr, vr = s["k_pool"].flatten(0, 1), s["v_pool"].flatten(0, 1)

        def rows(table, n):  # the pool's rows of a table's first n tokens
            i = torch.arange(n, device=DEV)
            return table.long()[i // c["bs"]] * c["bs"] + i % c["bs"]

        outs, b = [], 0
        for gi, (m, p) in enumerate(zip(members, prefix)):
            shared = rows(s["ptab"][gi], p)
            ks, vs = kr[shared].double(), vr[shared].double()
            for _ in range(m):
                r = rows(s["tab"][b], mine[b])
                outs.append(_attend(s["q"][b : b + 1].double(), torch.cat((ks, kr[r].double())), torch.cat((vs, vr[r].double()))))
                b += 1
        return torch.cat(outs)
    if c["op"] == "cross":
        queries, valid = _lens(c)
        outs, a = [], 0
        for i, (n, t) in enumerate(zip(queries, valid)):
            slot = int(s["slots"][i])
            k, v = (x[slot, :, :t].transpose(0, 1).double() for x in (s["k"], s["v"]))
            outs.append(_attend(s["q"][a : a + n].double(), k, v))
            a += n
        return torch.cat(outs)
    # row by row, by the definition, on sorted columns of the host's choice: numbers of 64 bits throughout
    tokens, logs = [], []
    for r in range(c["rows"]):
        x = s["x"][r, : c["cols"]].double()
        if s["skip"] is not None:
            x[s["skip"]] = -math.inf
        t, k, p, least, u = (float(s[n][r]) for n in ("t", "k", "p", "least", "u"))
        m = x.max()
        top = int((x == m).nonzero()[0])
        if t <= 0:
            token = top
        else:
            # columns by value, equal ones by place: two stable sorts of the negated values give their rank
            order = torch.argsort(-x, stable=True)
            if k > 0:
                order = order[: int(k)]
            w = torch.exp((x[order] - m) / t)
            if p < 1:
                before = torch.cat((w.new_zeros(1), w.cumsum(0)[:-1]))
                order = order[: max(1, int((before < p * w.sum()).sum()))]
            if least > 0:
                order = order[: max(1, int((x[order] >= m + t * math.log(least)).sum()))]
            left = order.sort().values
            cum = torch.exp((x[left] - m) / t).cumsum(0)
            at = int((cum <= u * cum[-1]).sum())
            token = int(left[min(at, len(left) - 1)])
        tokens.append(token)
        logs.append(x[token] - m - torch.exp(x - m).sum().log())
    return [torch.tensor(tokens, device=DEV), torch.stack(logs)]
