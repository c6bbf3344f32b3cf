"""The spans' kernel under a wait limit of 1 ns: with a few hundred steps a CTA some wait takes longer than the two tries (some
4 us each) that any limit allows, so each operator has to report that it gave up, and the call after it is exact again."""
import pytest
import torch

from int4_reference import cu
from speech_serving import _native as N
from speech_serving import ops
from test_candidates_gpu import DEV

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def limits():
    yield
    assert N.load().spd_set_wait_timeout_ns(0) == N.SPD_OK


def gives_up(call):
    """`call(error_word)` as usual, ten times under the short limit, and as usual again."""
    lib, results = N.load(), []
    for limit, repeats in ((0, 1), (1, 10), (0, 1)):
        assert lib.spd_set_wait_timeout_ns(limit) == N.SPD_OK
        found = set()
        for _ in range(repeats):
            word = torch.zeros(1, dtype=torch.int32, device=DEV)
            out = call(word)
            torch.cuda.synchronize()
            found.add(ops.read_error_word(word))
        if limit:
            assert N.SPD_DEVERR_TIMEOUT in found and found <= {0, N.SPD_DEVERR_TIMEOUT}
        else:
            assert found == {0}
            results.append(out)
    assert torch.equal(*results)


def inputs(groups=40, members=300, tokens=4096, D=128):
    g = torch.Generator(device=DEV).manual_seed(0)
    kv = torch.randn(2, groups, 2, tokens, D, device=DEV, generator=g).bfloat16()
    q = torch.randn(groups * members, 4, D, device=DEV, generator=g).bfloat16()
    lens = torch.full((groups,), tokens, dtype=torch.int32, device=DEV)
    return q, kv, lens, cu([members] * groups).to(DEV)


def test_cross_attention_gives_up():
    q, kv, lens, cq = inputs()
    gives_up(lambda e: ops.cross_attention_packed(q, kv[0], kv[1], lens, cq, error_word=e))


def test_shared_prefixes_give_up():
    q, kv, lens, cq = inputs()
    pool = kv.permute(0, 1, 3, 2, 4).reshape(2, -1, 16, 2, 128).contiguous()
    table = torch.arange(pool.shape[1], dtype=torch.int32, device=DEV).view(len(lens), -1)
    own = torch.zeros(len(q), 1, dtype=torch.int32, device=DEV), torch.full((len(q),), 5, dtype=torch.int32, device=DEV)
    gives_up(lambda e: ops.shared_prefix_decode_attention(q, pool[0], pool[1], table, lens, cq, *own, error_word=e))
