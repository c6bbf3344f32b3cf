"""The bounded waits of 4-bit decode attention and prompt attention run out, on the GPU, without a fault.

Under a 1 ns bound a wait gives up after two suspended tries of 4 us each: in prompt attention the warp
that asks for a CTA's next item waits for all keys of the present one, and any other wait may run out
too, with copies and products in flight.  The launch records SPD_DEVERR_TIMEOUT, lets what is in
flight land, and returns; the next launch under the default bound is exact.  Nothing here traps,
faults or hangs."""
import pytest
import torch

from speech_serving import _native as N
from speech_serving import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture
def short_waits():
    """Restores the default bound after a test that shortened it."""
    lib = N.load()
    yield lib
    assert lib.spd_set_wait_timeout_ns(0) == N.SPD_OK


@pytest.mark.parametrize("keys", [200_000, 200_001])
@pytest.mark.parametrize("heads,kv_heads,D,queries", [(4, 1, 128, 1), (2, 2, 64, 300), (8, 8, 64, 10_500), (8, 4, 128, 10_500), (8, 8, 64, 30_000)])
def test_prompt_attention_gives_up_and_then_is_exact(short_waits, keys, heads, kv_heads, D, queries):
    lib = short_waits
    g = torch.Generator(device=DEV).manual_seed(keys)
    keys = keys if queries < 1000 else keys // 8  # several items for every CTA slot
    q = torch.randn(queries, heads, D, generator=g, device=DEV).half()
    k, v = (torch.randn(keys, kv_heads, D, generator=g, device=DEV).half() for _ in range(2))
    cq, ck = (torch.tensor([0, n], dtype=torch.int32, device=DEV) for n in (queries, keys))
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    want = ops.prompt_attention(q, k, v, cq, ck, causal=False, error_word=word)
    assert ops.read_error_word(word) == 0
    assert lib.spd_set_wait_timeout_ns(1) == N.SPD_OK
    ops.prompt_attention(q, k, v, cq, ck, causal=False, error_word=word)
    torch.cuda.synchronize()
    given_up = ops.read_error_word(word)
    assert given_up in (0, N.SPD_DEVERR_TIMEOUT)
    if queries < 1000:  # one item of milliseconds
        assert given_up == N.SPD_DEVERR_TIMEOUT
    assert lib.spd_set_wait_timeout_ns(0) == N.SPD_OK
    word.zero_()
    assert torch.equal(ops.prompt_attention(q, k, v, cq, ck, causal=False, error_word=word), want)
    assert ops.read_error_word(word) == 0


@pytest.mark.parametrize("D,heads", [(64, 12), (128, 16)])
def test_int4_decode_under_a_tiny_bound_then_exact(short_waits, D, heads):
    """Its waits are for one copy each: the call is exact or gives up."""
    lib = short_waits
    g = torch.Generator(device=DEV).manual_seed(D)
    B, columns = 16, 512
    pool = torch.randint(0, 256, ops.kv_pool_int4(2048, 2, D, 16).shape, generator=g, device=DEV, dtype=torch.uint8)
    codes, half = D // 64 * 16 * 32, pool.shape[2] // 2
    for at in (codes, half + codes):  # scale 0.25, zero -1
        pool.view(torch.float16)[..., at // 2 : (at + D // 64 * 16 * 4) // 2] = torch.tensor(
            [0.25, -1.0], dtype=torch.float16, device=DEV).repeat(D // 64 * 16)
    q = torch.randn(B, heads, D, generator=g, device=DEV).half()
    tables = torch.randint(0, 2048, (B, columns), generator=g, device=DEV, dtype=torch.int32)
    lens = torch.randint(1, columns * 16, (B,), generator=g, device=DEV, dtype=torch.int32)
    ws = ops.decode_int4_workspace(B, heads, 2, D, 16, columns, torch.float16, torch.device(DEV))
    want = ops.paged_decode_attention_int4(q, pool, tables, lens, workspace=ws)
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert lib.spd_set_wait_timeout_ns(1) == N.SPD_OK
    got = ops.paged_decode_attention_int4(q, pool, tables, lens, workspace=ws, error_word=word)
    torch.cuda.synchronize()
    given_up = ops.read_error_word(word)
    assert given_up in (0, N.SPD_DEVERR_TIMEOUT)
    if given_up == 0:
        assert torch.equal(got, want)
    assert lib.spd_set_wait_timeout_ns(0) == N.SPD_OK
    assert not ws[256 : 256 + 4 * B * heads].any()  # the arrival counters came back to zero
    assert torch.equal(ops.paged_decode_attention_int4(q, pool, tables, lens, workspace=ws), want)
