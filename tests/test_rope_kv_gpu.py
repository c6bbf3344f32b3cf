"""rope_kv_append, rope_kv_append_int4 and kv_gather_int4 against plain CPU forms.

Tolerances.  The kernel rounds each product and sum of the rotation to fp32 and the result
once to the output type, as the fp32 CPU form does, so the two are equal bit for bit.
Against the 64-bit form a rotated value may be off by the fp32 roundings of two products and
a sum, 2^-23 (|x_i| + |x_j|), and by the output's own half unit: 2^-8 (bf16), 2^-11 (fp16)
or 2^-24 (fp32) of its size.  A stored 4-bit value is off by at most half a step, plus what
the fp16 roundings of zero (2^-11 of it) and scale (15 steps at 2^-11 each) move the ends by."""
import pytest
import torch

import int4_reference as R
from speech_serving import _native as N
from speech_serving import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


class Case:
    """Packed tokens of ragged sequences and what an append of them must leave behind."""

    def __init__(self, lens, starts, Hq, Hkv, D, rot, bs, dtype, interleaved, seed=0, packed=True):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.starts, self.D, self.bs, self.dtype, self.interleaved = lens, starts, D, bs, dtype, interleaved
        ends = [max(0, s) + n for s, n in zip(starts, lens)]
        self.tables, self.blocks = R.tables(g, ends, bs)
        self.cos, self.sin = R.angles(max(ends) + 1, rot)
        n = sum(lens)
        qkv = torch.randn(n, Hq + 2 * Hkv, D, generator=g).to(dtype)
        self.q, self.k, self.v = qkv[:, :Hq], qkv[:, Hq : Hq + Hkv], qkv[:, Hq + Hkv :]
        d = qkv.to(DEV)
        self.dq, self.dk, self.dv = (d[:, :Hq], d[:, Hq : Hq + Hkv], d[:, Hq + Hkv :]) if packed else (
            d[:, :Hq].contiguous(), d[:, Hq : Hq + Hkv].contiguous(), d[:, Hq + Hkv :].contiguous())
        self.cu = R.cu(lens)
        self.b = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
        self.pos = torch.cat([torch.arange(s, s + m) for s, m in zip(starts, lens)]) if n else torch.zeros(0, dtype=torch.long)
        self.live = torch.tensor(starts)[self.b] >= 0
        at = self.pos.clamp(min=0)
        self.block, self.row = self.tables.long()[self.b, at // bs], at % bs
        self.c, self.s = self.cos[at], self.sin[at]
        self.args = [t.to(DEV) for t in (self.cos, self.sin)]
        self.where = [self.tables.to(DEV), torch.tensor(starts, dtype=torch.int32, device=DEV)]

    def rotated(self, x, dtype):
        return R.rotate(x.to(dtype), self.c, self.s, self.interleaved)


CASES = [  # lens, starts, Hq, Hkv, D, rot, bs
    ([1], [0], 1, 1, 64, 64, 16),
    ([1, 1, 1, 1, 1], [0, 7, 8, 31, 447], 12, 12, 64, 64, 8),
    ([5, 0, 33, 1, 16], [0, 3, 15, 16, 100], 8, 2, 128, 128, 16),
    ([40, 3, 17], [31, -1, 0], 6, 3, 64, 32, 32),
    ([9, 70], [1, 0], 5, 1, 256, 64, 16),
    ([3, 4], [2, 6], 3, 1, 72, 48, 5),           # 16-bit pools alone: odd head and block sizes
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"B{len(c[0])}_H{c[2]}_{c[3]}_D{c[4]}_r{c[5]}_bs{c[6]}")
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_append_16_bit(case, interleaved, dtype):
    c = Case(*case, dtype, interleaved, seed=len(case[0]))
    shape = (c.blocks, c.bs, case[3], c.D)
    k0, v0 = torch.randn(shape).to(dtype), torch.randn(shape).to(dtype)
    kp, vp = k0.to(DEV), v0.to(DEV)
    q = ops.rope_kv_append(c.dq, c.dk, c.dv, *c.args, kp, vp, *c.where, cu_seqlens=c.cu.to(DEV), interleaved=interleaved)
    want_q = c.rotated(c.q, torch.float32).to(dtype)
    want_q[~c.live] = 0
    assert torch.equal(q.cpu(), want_q)
    k0[c.block[c.live], c.row[c.live]] = c.rotated(c.k, torch.float32).to(dtype)[c.live]
    v0[c.block[c.live], c.row[c.live]] = c.v[c.live]
    assert torch.equal(kp.cpu(), k0) and torch.equal(vp.cpu(), v0)  # and nothing else changed
    exact = c.rotated(c.q, torch.float64)[c.live]
    size = R.rotate(c.q.double(), torch.ones_like(c.c), -torch.ones_like(c.s), interleaved).abs()[c.live]
    size = torch.maximum(size, 2 * c.q.double().abs().amax(-1, keepdim=True)[c.live])  # >= |x_i| + |x_j|
    off = (q.cpu().double()[c.live] - exact).abs()
    assert (off <= 2.0 ** -23 * size + UNIT[dtype] * exact.abs() * 1.001).all()


@pytest.mark.parametrize("case", CASES[:5], ids=lambda c: f"B{len(c[0])}_H{c[2]}_{c[3]}_D{c[4]}_r{c[5]}_bs{c[6]}")
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_append_and_gather_4_bit(case, interleaved, dtype):
    c = Case(*case, dtype, interleaved, seed=10 + len(case[0]))
    Hkv = case[3]
    pool0, *_ = R.random_pool(torch.Generator().manual_seed(1), c.blocks, c.bs, Hkv, c.D)
    pool = pool0.to(DEV)
    assert pool.shape == ops.kv_pool_int4(c.blocks, Hkv, c.D, c.bs).shape
    q = ops.rope_kv_append_int4(c.dq, c.dk, c.dv, *c.args, pool, *c.where, cu_seqlens=c.cu.to(DEV), interleaved=interleaved)
    want_q = c.rotated(c.q, torch.float32).to(dtype)
    want_q[~c.live] = 0
    assert torch.equal(q.cpu(), want_q)
    kc, kp, vc, vp = R.unpack(pool0, c.D, c.bs)
    k_new, v_new = R.quantise(c.rotated(c.k, torch.float32)), R.quantise(c.v.float())
    at = (c.block[c.live], c.row[c.live])
    kc[at], kp[at], vc[at], vp[at] = k_new[0][c.live], k_new[1][c.live], v_new[0][c.live], v_new[1][c.live]
    assert torch.equal(pool.cpu(), R.pack(kc, kp, vc, vp))
    # read back: rows of skipped sequences (their start is negative) come back as zeros
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    k, v = ops.kv_gather_int4(pool, c.where[0], c.cu.to(DEV), sum(c.lens), c.D, dtype, starts=c.where[1], error_word=err)
    for got, new, exact in ((k, k_new, c.rotated(c.k, torch.float64)), (v, v_new, c.v.double())):
        want = R.values(*new).to(torch.float32).to(dtype)
        want[~c.live] = 0
        assert torch.equal(got.cpu(), want)
        step = new[1][..., :1].double()
        ends = (0.5 + 15 * 2.0 ** -11) * step + 2.0 ** -10 * new[1][..., 1:].double().abs() + 1e-6
        off = (R.values(*new) - exact).unflatten(-1, (-1, 64)).abs()
        assert (off <= ends).all()
    assert ops.read_error_word(err) == 0


@pytest.mark.parametrize("D,rot", [(128, 64), (128, 96), (128, 112), (256, 128), (256, 192), (256, 256)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotations_that_pair_groups(D, rot, interleaved):
    """Halves of a rotation in the same group of 64 dimensions, in two, and across their borders."""
    c = Case([19, 1, 4], [5, 0, 60], 3, 3, D, rot, 8, torch.float16, interleaved, seed=rot)
    pool = ops.kv_pool_int4(c.blocks, 3, D, 8)
    ops.rope_kv_append_int4(c.dq, c.dk, c.dv, *c.args, pool, *c.where, cu_seqlens=c.cu.to(DEV), interleaved=interleaved)
    kc, kp, vc, vp = R.unpack(pool.cpu(), D, 8)
    for codes, params, x in ((kc, kp, c.rotated(c.k, torch.float32)), (vc, vp, c.v.float())):
        want = R.quantise(x)
        assert torch.equal(codes[c.block, c.row], want[0]) and torch.equal(params[c.block, c.row], want[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_codes_of_all_kinds_of_groups(dtype):
    """Groups far from zero, wide, narrow to scales below fp16's normal numbers, and quotients that lie
    halfway between two codes: the same codes as the plain form's, bit for bit."""
    D, bs, g = 64, 32, torch.Generator().manual_seed(2)
    rows = []
    for offset in (0.0, -0.3, 3.0, -40.0, 1000.0, -6e4, 9e4):
        for spread in (1e-7, 1e-4, 1e-2, 1.0, 50.0, 2e4, 1e6):
            rows += [offset + spread * torch.randn(D, generator=g), offset + spread * torch.rand(D, generator=g)]
    for scale in (2.0 ** -20, 2.0 ** -14, 2.0 ** -3, 1.0, 512.0):
        ties = torch.randint(0, 31, (D,), generator=g) / 2  # 0, 1/2, ..., 15
        ties[:2] = torch.tensor([0.0, 15.0])
        rows += [scale * ties, scale * (ties - 7), scale * (ties - 900)]
    x = torch.stack(rows)[:, None]
    x = x if dtype == torch.float32 else x.clamp(-65504.0, 65504.0).to(dtype)
    n = x.shape[0]
    blocks = -(-n // bs)
    cos, sin = torch.ones(blocks * bs, 8), torch.zeros(blocks * bs, 8)
    pool = ops.kv_pool_int4(blocks, 1, D, bs)
    ops.rope_kv_append_int4(None, x.to(DEV), x.to(DEV), cos.to(DEV), sin.to(DEV), pool,
                            torch.arange(blocks, dtype=torch.int32, device=DEV)[None],
                            torch.zeros(1, dtype=torch.int32, device=DEV), cu_seqlens=R.cu([n]).to(DEV))
    want = R.quantise(x.float())
    for codes, params in (R.unpack(pool.cpu(), D, bs)[:2], R.unpack(pool.cpu(), D, bs)[2:]):
        assert torch.equal(params.flatten(0, 1)[:n], want[1])
        assert torch.equal(codes.flatten(0, 1)[:n], want[0])


def test_decode_form_without_cu_seqlens_and_without_q():
    c = Case([1] * 7, [0, 15, 16, 3, -1, 99, 40], 8, 2, 64, 64, 16, torch.float16, False, packed=False)
    one, two = (ops.kv_pool_int4(c.blocks, 2, 64, 16) for _ in range(2))
    a = ops.rope_kv_append_int4(c.dq, c.dk, c.dv, *c.args, one, *c.where)
    assert ops.rope_kv_append_int4(None, c.dk, c.dv, *c.args, two, *c.where, cu_seqlens=c.cu.to(DEV)) is None
    assert torch.equal(one, two) and not a[4].any() and a[0].any()


def test_special_values_in_4_bits():
    """Constant rows (scale 0), saturation beyond fp16, and a NaN that stays in its 64 values."""
    D, bs = 128, 16
    k = torch.zeros(6, 1, D)
    k[0] = 3.0
    k[1, :, :64] = torch.linspace(-1e6, 1e6, 64)
    k[2, 0, 70] = float("nan")
    k[3, 0, 5] = float("inf")
    k[4, 0, 9] = -float("inf")
    k[5] = torch.linspace(1.0, 1.0 + 2.0 ** -20, D)
    v = k.flip(0).contiguous()
    cos, sin = R.angles(16, 16)
    pool = ops.kv_pool_int4(1, 1, D, bs)
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    cu = R.cu([6]).to(DEV)
    one, nil = torch.ones_like(cos), torch.zeros_like(sin)
    ops.rope_kv_append_int4(None, k.to(DEV), v.to(DEV), one.to(DEV), nil.to(DEV), pool, table, zero, cu_seqlens=cu)
    got = ops.kv_gather_int4(pool, table, cu, 6, D, torch.float32)
    for x, y in ((k, got[0]), (v, got[1])):
        rot = R.rotate(x, one[:6], nil[:6], False) if x is k else x
        want = R.values(*R.quantise(rot)).float()
        y = y.cpu()
        assert torch.equal(torch.isnan(want), torch.isnan(y))
        assert torch.equal(want.nan_to_num(0.0), y.nan_to_num(0.0))
    assert torch.isnan(got[0][2, 0, 64:]).all() and torch.isfinite(got[0][2, 0, :64]).all()


def test_bad_positions_and_blocks_are_flagged_and_nothing_is_written():
    c = Case([1, 1, 1], [0, 0, 0], 2, 2, 64, 64, 16, torch.bfloat16, False)
    for change, flag in ((lambda t, p: t[1].fill_(c.blocks), N.SPD_DEVERR_BLOCK_ID), (lambda t, p: t[1].fill_(-3), N.SPD_DEVERR_BLOCK_ID),
                         (lambda t, p: p[1].fill_(16 * t.shape[1]), N.SPD_DEVERR_LENGTH)):
        t, p = c.where[0].clone(), c.where[1].clone()
        change(t, p)
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        pool, ref = ops.kv_pool_int4(c.blocks, 2, 64, 16), ops.kv_pool_int4(c.blocks, 2, 64, 16)
        q = ops.rope_kv_append_int4(c.dq, c.dk, c.dv, *c.args, pool, t, p, error_word=err)
        assert ops.read_error_word(err) == flag
        p[1] = -1
        ops.rope_kv_append_int4(c.dq, c.dk, c.dv, *c.args, ref, c.where[0], p)
        assert torch.equal(pool, ref) and not q[1].any() and q[0].any()
        kp, vp = (torch.zeros(c.blocks, 16, 2, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        t, p = c.where[0].clone(), c.where[1].clone()
        change(t, p)
        err.zero_()
        ops.rope_kv_append(c.dq, c.dk, c.dv, *c.args, kp, vp, t, p, error_word=err)
        assert ops.read_error_word(err) == flag


def test_tokens_past_the_last_sequence_are_left_alone():
    c = Case([3, 2], [0, 0], 2, 1, 64, 64, 16, torch.float16, False)
    cu = torch.tensor([1, 3, 4], dtype=torch.int32, device=DEV)  # token 0 and token 4 belong to nobody
    pool = ops.kv_pool_int4(c.blocks, 1, 64, 16)
    q = ops.rope_kv_append_int4(c.dq, c.dk, c.dv, *c.args, pool, *c.where, cu_seqlens=cu)
    assert not q[0].any() and not q[4].any() and q[1:4].any(-1).all()
    k, v = (torch.full((5, 1, 64), 7.0, dtype=torch.float16, device=DEV) for _ in range(2))
    ops.kv_gather_int4(pool, c.where[0], cu, 5, 64, torch.float16, k_out=k, v_out=v)
    assert (k[[0, 4]] == 7).all() and (v[[0, 4]] == 7).all() and (k[1:4] != 7).any()


def test_gather_into_outputs_aligned_to_16_bytes_only():
    c = Case([5, 40], [0, 3], 2, 2, 128, 128, 16, torch.bfloat16, False)
    pool = ops.kv_pool_int4(c.blocks, 2, 128, 16)
    cu = c.cu.to(DEV)
    ops.rope_kv_append_int4(None, c.dk, c.dv, *c.args, pool, *c.where, cu_seqlens=cu)
    want = ops.kv_gather_int4(pool, c.where[0], cu, 45, 128, torch.bfloat16, starts=c.where[1])
    n = 45 * 2 * 128
    k, v = (torch.empty(n + 8, dtype=torch.bfloat16, device=DEV)[8:].view(45, 2, 128) for _ in range(2))
    ops.kv_gather_int4(pool, c.where[0], cu, 45, 128, torch.bfloat16, starts=c.where[1], k_out=k, v_out=v)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_pool_beyond_two_gigabytes():
    """Offsets past 2^31 bytes: the last block of a large pool."""
    D, bs, H = 128, 32, 8
    blocks = (1 << 32) // (ops.kv_pool_int4(1, H, D, bs).numel()) + 2
    pool = ops.kv_pool_int4(blocks, H, D, bs)
    table = torch.tensor([[blocks - 1]], dtype=torch.int32, device=DEV)
    k = torch.randn(1, H, D, device=DEV).half()
    cos, sin = (t.to(DEV) for t in R.angles(32, 128))
    ops.rope_kv_append_int4(None, k, k, cos, sin, pool, table, torch.tensor([31], dtype=torch.int32, device=DEV))
    got = ops.kv_gather_int4(pool, table, R.cu([1]).to(DEV), 1, D, torch.float32,
                             starts=torch.tensor([31], dtype=torch.int32, device=DEV))[1]
    assert torch.equal(got.cpu(), R.values(*R.quantise(k.cpu().float())).float())
    q = torch.zeros(1, 16, D, dtype=torch.float16, device=DEV)  # even weights over the one written and 31 zero rows
    out = ops.paged_decode_attention_int4(q, pool, table, torch.tensor([32], dtype=torch.int32, device=DEV))
    want = got.cpu().double().repeat_interleave(2, 1) / 32
    assert (out.cpu().double() - want).abs().max() <= 2.0 ** -10 * want.abs().max()


def test_refusals():
    c = Case([2, 1], [0, 0], 2, 1, 64, 64, 16, torch.float16, False)
    pool = ops.kv_pool_int4(c.blocks, 1, 64, 16)
    cu = c.cu.to(DEV)
    good = dict(q=c.dq, k=c.dk, v=c.dv, cos=c.args[0], sin=c.args[1], pool=pool, block_tables=c.where[0], positions=c.where[1],
                cu_seqlens=cu)
    ops.rope_kv_append_int4(**good)
    for change, match in ((dict(cu_seqlens=None), "one token per sequence"), (dict(v=c.dv.float()), "one shape and dtype"),
                          (dict(q=c.dq.float()), "does not match"), (dict(pool=pool.view(torch.int8)), "uint8"),
                          (dict(pool=pool[:, :, :-16].contiguous()), "fit no block size"),
                          (dict(positions=c.where[1].long()), "positions"), (dict(cos=c.args[0].half()), "float32"),
                          (dict(cos=c.args[0][:, :4].contiguous(), sin=c.args[1][:, :4].contiguous()), "multiple of 16"),
                          (dict(q_out=c.dq), "apart from q"), (dict(block_tables=c.where[0][:1]), "block_tables"),
                          (dict(k=c.dk.cpu()), "CUDA tensors")):
        with pytest.raises(RuntimeError, match=match):
            ops.rope_kv_append_int4(**{**good, **change})
    with pytest.raises(RuntimeError, match="16 bytes"):  # a token stride that is no multiple of 16 bytes
        odd = torch.zeros(3, 68, dtype=torch.float16, device=DEV)[:, :64].unflatten(1, (1, 64))
        ops.rope_kv_append_int4(**{**good, "q": None, "k": odd, "v": odd})
    with pytest.raises(RuntimeError, match="not supported"):
        ops.kv_pool_int4(4, 1, 96, 16)
    with pytest.raises(RuntimeError, match="outputs must be"):
        ops.kv_gather_int4(pool, c.where[0], cu, 3, 64, torch.float16, k_out=torch.empty(2, 1, 64, device=DEV).half())
    kp = torch.zeros(4, 16, 1, 64, dtype=torch.float16, device=DEV)
    with pytest.raises(RuntimeError, match="pools must be"):
        ops.rope_kv_append(c.dq, c.dk, c.dv, *c.args, kp, kp.float(), *c.where, cu_seqlens=cu)
    wide = torch.zeros(3, 1, 1032, dtype=torch.float16, device=DEV)
    pools = [torch.zeros(c.blocks, 16, 1, 1032, dtype=torch.float16, device=DEV) for _ in range(2)]
    with pytest.raises(RuntimeError, match="up to 1024"):
        ops.rope_kv_append(None, wide, wide, *c.args, *pools, *c.where, cu_seqlens=cu)


def test_the_widest_heads():
    c = Case([3, 1], [2, 0], 2, 1, 1024, 1024, 16, torch.bfloat16, False)
    kp, vp = (torch.zeros(c.blocks, 16, 1, 1024, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    q = ops.rope_kv_append(c.dq, c.dk, c.dv, *c.args, kp, vp, *c.where, cu_seqlens=c.cu.to(DEV))
    assert torch.equal(q.cpu(), c.rotated(c.q, torch.float32).bfloat16())
    assert torch.equal(kp.cpu()[c.block, c.row], c.rotated(c.k, torch.float32).bfloat16())
    assert torch.equal(vp.cpu()[c.block, c.row], c.v)
