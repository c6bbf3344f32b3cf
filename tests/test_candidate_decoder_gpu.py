"""examples/candidates.py: the operators for several candidates of a request as one decoder, against a plain 64-bit CPU form
of the same network.  A logit's bound is that of the rotary decoder with a third more roundings for the cross-attention,
2^-5 of the largest; a token's log-probability (a logit less a logarithm of a sum of exponentials of logits) is within twice
that."""
import sys

import pytest
import torch
import torch.nn.functional as F

from conftest import REPO
from int4_reference import angles, rotate

sys.path.insert(0, str(REPO / "examples"))
from candidates import CandidateDecoder  # noqa: E402
from rotary_decoder import Config  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"


def plain_logits(model, states, tokens):
    """Logits of every position of one request [n, vocab]; `states`: the encoder states that count."""
    c = model.cfg
    cos, sin = (t.double()[: len(tokens)] for t in angles(c.max_positions, c.head_dim))
    x, states = model.embed.cpu().double()[torch.tensor(tokens)], states.cpu().double()
    hidden = torch.ones(len(tokens), len(tokens), dtype=torch.bool).triu(1)
    wide = c.heads // c.kv_heads

    def attend(q, k, v, mask=None):
        k, v = (t.repeat_interleave(wide, 1) for t in (k, v))
        s = torch.einsum("ihd,jhd->hij", q, k) * c.head_dim ** -0.5
        if mask is not None:
            s = s.masked_fill(mask, float("-inf"))
        return torch.einsum("hij,jhd->ihd", s.softmax(-1), v).flatten(1)

    for layer in model.layers:
        w = {k: t.cpu().double() for k, t in layer.items()}
        y = (F.layer_norm(x, (c.width,)) @ w["qkv"].T).view(-1, c.heads + 2 * c.kv_heads, c.head_dim)
        q, k, v = y.split((c.heads, c.kv_heads, c.kv_heads), 1)
        q, k = rotate(q, cos, sin, False), rotate(k, cos, sin, False)
        x = x + attend(q, k, v, hidden) @ w["out"].T
        q = (F.layer_norm(x, (c.width,)) @ w["cross_q"].T).view(-1, c.heads, c.head_dim)
        k, v = (states @ w["cross_kv"].T).view(len(states), 2, c.kv_heads, c.head_dim).unbind(1)
        if len(states):
            x = x + attend(q, k, v) @ w["cross_out"].T
        x = x + F.gelu(F.layer_norm(x, (c.width,)) @ w["up"].T) @ w["down"].T
    return F.layer_norm(x, (c.width,)) @ model.head.cpu().double().T


def model_of(heads, kv_heads, head_dim, audio, seed=0):
    cfg = Config(layers=2, heads=heads, kv_heads=kv_heads, head_dim=head_dim, vocab=500, num_blocks=160, bits=16, max_positions=200,
                 seed=seed)
    model = CandidateDecoder(cfg)
    g = torch.Generator().manual_seed(seed)
    states = torch.randn(len(audio), max(audio), cfg.width, generator=g).to(DEV, cfg.dtype)
    model.encode(states, audio)
    return model, states, g


@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 2, 64), (4, 4, 128)])
def test_candidates_match_the_plain_network(heads, kv_heads, head_dim):
    audio = [150, 1, 0, 64]
    model, states, g = model_of(heads, kv_heads, head_dim, audio)
    prompts = [torch.randint(0, 500, (n,), generator=g).tolist() for n in (1, 150, 32, 75)]
    logits = model.prefill(prompts, 48)
    n, steps = 5, 6
    held = model.blocks.allocated_block_count
    tokens, scores = model.sample(logits, n, steps, 0.9, 40, 0.95, seed=3)
    again, same = model.sample(logits, n, steps, 0.9, 40, 0.95, seed=3)
    model.check_errors()
    assert torch.equal(tokens, again) and torch.equal(scores, same) and model.blocks.allocated_block_count == held
    first, _ = model.sample(logits, 2, steps, 0.0)
    model.check_errors()
    assert torch.equal(first[:, 0], first[:, 1])
    for r, p in enumerate(prompts):
        for i in range(n + 1):
            own = (tokens[r, i] if i < n else first[r, 0]).tolist()
            want = plain_logits(model, states[r, : audio[r]], p + own)[len(p) - 1 : len(p) - 1 + steps]
            bound = 2.0 ** -5 * want.abs().max().item()
            if i == 0:
                assert (logits[r].cpu().double() - want[0]).abs().max().item() <= bound
            if i < n:
                exact = F.log_softmax(want, -1)[range(steps), own].sum().item()
                assert abs(scores[r, i].item() - exact) <= 2 * bound * steps
                # no token below the 40 largest
                assert all(row[t] >= row.topk(40).values[-1] - 2 * bound for row, t in zip(want, own))
            else:
                assert all(row[t] >= row.max() - 2 * bound for row, t in zip(want, own))
    assert len({tuple(t) for t in tokens[1].tolist()}) > 1
    model.release()
    assert model.blocks.check_no_leaks()


def test_many_candidates_of_one_request():
    """More rows than a tile, and one candidate of its own: the same continuation either way, up to the logits' error."""
    model, _, g = model_of(4, 1, 64, [100], seed=1)
    logits = model.prefill([torch.randint(0, 500, (130,), generator=g).tolist()])
    model.sample(logits, 40, 4, 1.0, seed=1)
    assert model.sample(logits, 1, 1, 0.0)[0].item() == logits.argmax().item()
    model.check_errors()
    model.release()
    assert model.blocks.check_no_leaks()


def test_refusals():
    with pytest.raises(ValueError, match="16 bits"):
        CandidateDecoder(Config(bits=4))
    model, _, _ = model_of(4, 1, 64, [10])
    logits = model.prefill([[1] * 190])
    with pytest.raises(ValueError, match="positions reach 200"):
        model.sample(logits, 2, 11)
    with pytest.raises(ValueError, match="at least"):
        model.sample(logits, 0, 5)
    held = model.blocks.allocated_block_count
    with pytest.raises(RuntimeError, match="out of physical blocks"):
        model.sample(logits, 300, 5)
    assert model.blocks.allocated_block_count == held
    model.release()
