"""Device flags reach the caller of 4-bit decode attention, with and without a workspace of its own."""
import sys

import pytest
import torch

import int4_reference as R
from conftest import REPO
from speech_serving import _native as N
from speech_serving import ops

sys.path.insert(0, str(REPO / "examples"))
from rotary_decoder import Config, RotaryDecoder  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"


def case():
    g = torch.Generator().manual_seed(0)
    lens = [40, 10]
    tables, blocks = R.tables(g, lens, 16)
    pool, *_ = R.random_pool(g, blocks, 16, 2, 64)
    return (torch.randn(2, 4, 64, generator=g).half().to(DEV), pool.to(DEV), tables.to(DEV),
            torch.tensor(lens, dtype=torch.int32, device=DEV))


def test_error_word_of_the_caller():
    q, pool, tables, lens = case()
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    want = ops.paged_decode_attention_int4(q, pool, tables, lens)
    assert torch.equal(want, ops.paged_decode_attention_int4(q, pool, tables, lens, error_word=word))
    assert ops.read_error_word(word) == 0
    wild = tables.clone()
    wild[0, 0] = -7
    ops.paged_decode_attention_int4(q, pool, wild, lens, error_word=word)
    assert ops.read_error_word(word) == N.SPD_DEVERR_BLOCK_ID
    ops.paged_decode_attention_int4(q, pool, tables, lens + 1000, error_word=word)  # flags add up
    assert ops.read_error_word(word) == N.SPD_DEVERR_BLOCK_ID | N.SPD_DEVERR_LENGTH
    # with both, the flags go to the word, and the workspace's own stays clear
    word.zero_()
    ws = ops.decode_int4_workspace(2, 4, 2, 64, 16, tables.shape[1], torch.float16, torch.device(DEV))
    ops.paged_decode_attention_int4(q, pool, wild, lens, workspace=ws, error_word=word)
    assert ops.read_error_word(word) == N.SPD_DEVERR_BLOCK_ID and ops.read_error_word(ws) == 0
    for bad in (torch.zeros(1, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV)):
        with pytest.raises(RuntimeError, match="error_word"):
            ops.paged_decode_attention_int4(q, pool, tables, lens, error_word=bad)


@pytest.mark.parametrize("bits,kv_heads", [(4, 2), (16, 4)])
def test_example_reports_what_decode_attention_flags(bits, kv_heads):
    """A wild id in a block that no append of the decode steps touches: only the attention can see it."""
    model = RotaryDecoder(Config(layers=2, heads=4, kv_heads=kv_heads, vocab=100, num_blocks=16, bits=bits, max_positions=100))
    logits = model.prefill([list(range(40))])
    model.decode(logits, 3)
    model.check_errors()
    whole = model._device_tables
    model._device_tables = lambda: whole().index_fill_(1, torch.zeros(1, dtype=torch.long, device=DEV), 10 ** 6)
    model.decode(logits, 3)
    with pytest.raises(RuntimeError, match="block id"):
        model.check_errors()
