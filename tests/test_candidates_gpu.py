"""shared_prefix_decode_attention and cross_attention_packed against plain 64-bit CPU forms.

Tolerance per output (u half a step of the input type: 2^-8 for bf16, 2^-11 for fp16):
  |off| <= (u + 2 e) A + u |out| + 2 ds A + n 2^-25 V
with A = sum p |v| (a weight is rounded at most once to the input type), e the relative error of an
exponential (polynomial of degree 3 for bf16, 7.6e-5, of degree 4 for fp16, 2.8e-6; met by
numerator and sum), ds the error of a score (2^-21 of scale * sum |q k|, for the fp32 sum of up to 128
products), and the last term the weights that fp16 holds as subnormals (n keys, V the largest |v|;
the largest weight is >= 1)."""
import math

import pytest
import torch

from int4_reference import cu
from speech_serving import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
EXPONENTIAL = {torch.float16: 2.8e-6, torch.bfloat16: 7.6e-5}


def attend(q, k, v, scale):
    """q [Hq, D], k and v [n, Hkv, D] -> the result and its bound, in 64 bits."""
    if k.shape[0] == 0:
        return torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    G, u = q.shape[0] // k.shape[1], UNIT[q.dtype]
    x, y, z = q.double(), k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1)
    s = torch.einsum("hd,jhd->hj", x, y) * scale
    size = torch.einsum("hd,jhd->hj", x.abs(), y.abs()) * scale
    p = torch.softmax(s, -1)
    out, A = torch.einsum("hj,jhd->hd", p, z), torch.einsum("hj,jhd->hd", p, z.abs())
    ds = 2.0 ** -21 * size.amax(-1, keepdim=True)
    return out, (u + 2 * EXPONENTIAL[q.dtype]) * A + u * out.abs() * 1.001 + 2 * ds * A + len(k) * 2.0 ** -25 * z.abs().max()


def near(got, parts):
    out, bound = (torch.stack(x) for x in zip(*parts))
    off = (got.cpu().double() - out).abs()
    assert (off <= bound).all(), (off / bound.clamp(min=1e-300)).max()


class Prefix:
    """Groups of `members` sequences with prefixes of `prefix` tokens, and own tokens."""

    def __init__(self, seed, members, prefix, mine, Hq, Hkv, D, dtype, bs=16, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        B, G = sum(members), len(members)
        assert len(mine) == B
        cols_p, cols = (max(1, -(-max(x, default=0) // bs)) for x in (prefix, mine))
        blocks = G * cols_p + B * cols + 2
        perm = torch.randperm(blocks, generator=g).to(torch.int32)
        self.ptab, self.tab = perm[: G * cols_p].view(G, cols_p), perm[G * cols_p : G * cols_p + B * cols].view(B, cols)
        self.k, self.v = (torch.randn(blocks, bs, Hkv, D, generator=g).to(dtype) for _ in range(2))
        self.q = (torch.randn(B, Hq, D, generator=g) * spread).to(dtype)
        self.members, self.prefix, self.mine, self.bs = members, prefix, mine, bs
        self.cu = cu(members)

    def rows(self, table, n):
        i = torch.arange(n)
        return table.long()[i // self.bs] * self.bs + i % self.bs

    def want(self, scale=None, first=0, left_out=()):
        """By sequence; `first`: sequences before the first group; `left_out`: blocks whose tokens do not count."""
        kr, vr = self.k.flatten(0, 1), self.v.flatten(0, 1)
        group = [-1] * first + [g for g, m in enumerate(self.members) for _ in range(m)]
        parts = []
        for b in range(len(self.q)):
            g = group[b] if b < len(group) else -1
            r = torch.cat((self.rows(self.ptab[g], self.prefix[g]) if g >= 0 else torch.zeros(0, dtype=torch.long),
                           self.rows(self.tab[b], self.mine[b])))
            r = r[~torch.isin(r // self.bs, torch.tensor(list(left_out), dtype=torch.long))]
            parts.append(attend(self.q[b], kr[r], vr[r], scale or 1 / math.sqrt(self.q.shape[2])))
        return parts

    def args(self):
        ints = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (self.prefix, self.mine))
        plens, lens = ints
        return [self.q.to(DEV), self.k.to(DEV), self.v.to(DEV), self.ptab.to(DEV).contiguous(), plens, self.cu.to(DEV),
                self.tab.to(DEV).contiguous(), lens]


SHAPES = [
    ([4], [100], [5, 1, 40, 17]),
    ([1], [1], [1]),
    ([3, 1, 2], [0, 130, 128], [0, 3, 16, 0, 33, 129]),
    ([2, 0, 5], [257, 50, 1500], [1, 2, 3, 4, 5, 6, 700]),
    ([40], [640], [i * 7 % 60 for i in range(40)]),
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: str((s[0], s[1])))
@pytest.mark.parametrize("Hq,Hkv,D", [(2, 2, 64), (4, 1, 128), (12, 2, 64), (8, 8, 128), (20, 1, 64)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prefix_matches_64_bits(shape, Hq, Hkv, D, dtype):
    c = Prefix(Hq + D, *shape, Hq, Hkv, D, dtype)
    near(ops.shared_prefix_decode_attention(*c.args()), c.want())


@pytest.mark.parametrize("D", [8, 16, 32, 40, 72, 80, 120])
@pytest.mark.parametrize("bs", [8, 16, 32, 64, 128])
def test_prefix_head_and_block_sizes(D, bs):
    c = Prefix(D + bs, [3, 2], [300, 77], [5, 200, 0, 31, 64], 4, 2, D, torch.float16, bs=bs)
    near(ops.shared_prefix_decode_attention(*c.args()), c.want())


@pytest.mark.parametrize("members,Hq,Hkv", [(200, 2, 2), (70, 8, 2), (130, 8, 2), (3, 128, 1), (5, 96, 1), (300, 3, 1)])
def test_prefix_of_more_rows_than_a_tile(members, Hq, Hkv):
    c = Prefix(members, [members, 2], [700, 90], [3] * (members + 2), Hq, Hkv, 64, torch.bfloat16)
    near(ops.shared_prefix_decode_attention(*c.args()), c.want())


def test_prefix_cut_into_many_pieces():
    """One key/value head and a long prefix: the item is shared by many CTAs."""
    c = Prefix(3, [5], [20000], [9000, 0, 1, 300, 2000], 4, 1, 128, torch.bfloat16, bs=32)
    near(ops.shared_prefix_decode_attention(*c.args()), c.want())


@pytest.mark.parametrize("beams,Hq,Hkv,D", [([5], 2, 2, 64), ([1, 0, 300, 17], 2, 2, 64), ([129, 1], 4, 2, 128),
                                            ([257, 3, 64], 6, 1, 64), ([1, 1, 1], 20, 20, 64), ([40, 70], 3, 3, 80)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_cross_matches_64_bits(beams, Hq, Hkv, D, dtype):
    g = torch.Generator().manual_seed(sum(beams) + D)
    B, T = len(beams), 700
    valid = [700, 1, 129, 640][:B]
    kv = torch.randn(B + 2, 2, Hkv, T, D, generator=g).to(dtype)
    q = torch.randn(sum(beams), Hq, D, generator=g).to(dtype)
    slots = torch.randperm(B + 2, generator=g)[:B]
    d = kv.to(DEV)
    got = ops.cross_attention_packed(q.to(DEV), d[:, 0], d[:, 1], torch.tensor(valid, dtype=torch.int32, device=DEV),
                                     cu(beams).to(DEV), slot_ids=slots.to(torch.int32).to(DEV))
    parts, a = [], 0
    for n, t, s in zip(beams, valid, slots):
        for i in range(n):
            parts.append(attend(q[a + i], kv[s, 0, :, :t].transpose(0, 1), kv[s, 1, :, :t].transpose(0, 1), D ** -0.5))
        a += n
    near(got, parts)
