"""examples/rotary_decoder.py against a plain 64-bit CPU form of the same network.

The network in fp16 rounds about ten times per layer to 2^-11 of values of order one, each carried
on by random weights of gain one: a logit (of order one, largest about four) is within 2^-6 of the
largest.  In the 4-bit form the plain network quantises its own keys and values; the fp16
values that differ by 2^-11 land on another code for about one value in a hundred, which moves it by a
sixteenth of its group's range: 2^-4 of the largest."""
import sys

import pytest
import torch
import torch.nn.functional as F

from conftest import REPO
from int4_reference import angles, quantise, rotate, values

sys.path.insert(0, str(REPO / "examples"))
from rotary_decoder import Config, RotaryDecoder  # noqa: E402

pytestmark = pytest.mark.gpu
TOLERANCE = {4: 2.0 ** -4, 16: 2.0 ** -6}


def plain_logits(model, tokens):
    """Logits of every position of one request [n, vocab], all positions at once."""
    c = model.cfg
    cos, sin = (t.double()[: len(tokens)] for t in angles(c.max_positions, c.head_dim))
    x = model.embed.cpu().double()[torch.tensor(tokens)]
    hidden = torch.ones(len(tokens), len(tokens), dtype=torch.bool).triu(1)
    for layer in model.layers:
        w = {k: t.cpu().double() for k, t in layer.items()}
        y = (F.layer_norm(x, (c.width,)) @ w["qkv"].T).view(-1, c.heads + 2 * c.kv_heads, c.head_dim)
        q, k, v = y.split((c.heads, c.kv_heads, c.kv_heads), 1)
        q, k = rotate(q, cos, sin, False), rotate(k, cos, sin, False)
        if c.bits == 4:
            k, v = (values(*quantise(t.float())) for t in (k, v))
        k, v = (t.repeat_interleave(c.heads // c.kv_heads, 1) for t in (k, v))
        s = torch.einsum("ihd,jhd->hij", q, k) * c.head_dim ** -0.5
        o = torch.einsum("hij,jhd->ihd", s.masked_fill(hidden, float("-inf")).softmax(-1), v)
        x = x + o.flatten(1) @ w["out"].T
        x = x + F.gelu(F.layer_norm(x, (c.width,)) @ w["up"].T) @ w["down"].T
    return F.layer_norm(x, (c.width,)) @ model.head.cpu().double().T


@pytest.mark.parametrize("bits,heads,kv_heads,head_dim", [(4, 8, 2, 64), (4, 4, 4, 128), (16, 4, 4, 64)])
def test_prompts_and_decode_match_the_plain_network(bits, heads, kv_heads, head_dim):
    cfg = Config(layers=2, heads=heads, kv_heads=kv_heads, head_dim=head_dim, vocab=500, num_blocks=64, bits=bits,
                 max_positions=200)
    model = RotaryDecoder(cfg)
    g = torch.Generator().manual_seed(bits)
    prompts = [torch.randint(0, cfg.vocab, (n,), generator=g).tolist() for n in (1, 150, 37, 64)]
    for chunk in (48, 500):
        logits = model.prefill(prompts, chunk)
        tokens = model.decode(logits, 6)
        assert model.lengths == [len(p) + 5 for p in prompts]
        model.check_errors()
        for r, p in enumerate(prompts):
            own = tokens[r].tolist()
            want = plain_logits(model, p + own)
            bound = TOLERANCE[bits] * want.abs().max().item()
            assert (logits[r].cpu().double() - want[len(p) - 1]).abs().max().item() <= bound
            for i, t in enumerate(own):  # greedy, up to the logits' error
                at = want[len(p) - 1 + i]
                assert at[t].item() >= at.max().item() - 2 * bound
        model.release()
        assert model.blocks.check_no_leaks()


def test_refusals():
    with pytest.raises(ValueError, match="4 or 16"):
        RotaryDecoder(Config(bits=8))
    with pytest.raises(ValueError, match="as many key/value heads"):
        RotaryDecoder(Config(bits=16))
    model = RotaryDecoder(Config(layers=1, num_blocks=4, max_positions=32))
    with pytest.raises(ValueError, match="one token or more"):
        model.prefill([[1], []])
    with pytest.raises(ValueError, match="positions reach 32"):
        model.prefill([[1] * 33])
    model.release()
    with pytest.raises(RuntimeError, match="out of physical blocks"):
        model.prefill([[1] * 32] * 3)
