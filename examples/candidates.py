"""Several sampled continuations of each request, over its audio and its prompt: a decoder with rotary positions, grouped
heads, a 16-bit paged cache and cross-attention, random weights.

    python examples/candidates.py
    python examples/candidates.py --requests 1 --candidates 64 --longest 1500 --top-p 0.9

Prompt chunk, per layer:   rope_kv_append -> prompt_attention -> cross_attention_packed (its tokens a request)
Decode step, per layer:    rope_kv_append -> shared_prefix_decode_attention -> cross_attention_packed (its candidates)
             at its end:   sample_rows
A request's prompt stays in the cache once.  Its full blocks are the prefix that all its candidates share; each
candidate has blocks of its own from there on, the first with a copy of the tokens that the last full block
left over.  A decode step is captured once and replayed; the random numbers are drawn before.
"""
from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path
from typing import Sequence, Tuple

import torch
import torch.nn.functional as F

sys.path.insert(0, str(Path(__file__).resolve().parent))
from rotary_decoder import Config, RotaryDecoder  # noqa: E402
from speech_serving import ops  # noqa: E402


class CandidateDecoder(RotaryDecoder):
    grouped_16_bit = True  # both of its attentions take grouped heads

    def __init__(self, cfg: Config, device: str = "cuda"):
        if cfg.bits != 16:
            raise ValueError("candidates share a cache of 16 bits")
        super().__init__(cfg, device)
        g = torch.Generator().manual_seed(cfg.seed + 1)
        for layer in self.layers:
            for name, rows in (("cross_q", cfg.width), ("cross_kv", 2 * cfg.kv_heads * cfg.head_dim), ("cross_out", cfg.width)):
                layer[name] = (torch.randn(rows, cfg.width, generator=g) * cfg.width ** -0.5).to(device, cfg.dtype)

    # ---- audio ------------------------------------------------------------------------------
    def encode(self, states: torch.Tensor, lengths: Sequence[int]) -> None:
        """Cross-attention keys and values of encoder states [requests, T, width], of which lengths[r] count."""
        c = self.cfg
        self.audio_lens = self._ints(lengths)
        self.planes = []
        for layer in self.layers:
            kv = F.linear(states, layer["cross_kv"]).view(*states.shape[:2], 2, c.kv_heads, c.head_dim)
            self.planes.append(kv.permute(2, 0, 3, 1, 4))  # k, v [requests, kv_heads, T, head_dim], strided

    def _chunk(self, packed, starts, news):
        self.rows = F.pad(self._ints(news).cumsum(0, dtype=torch.int32), (1, 0))  # of each request
        return super()._chunk(packed, starts, news)

    def _rest(self, layer, x, attended):
        c = self.cfg
        x = x + F.linear(attended.flatten(1), layer["out"])
        k, v = self.planes[next(i for i, other in enumerate(self.layers) if other is layer)]
        q = F.linear(F.layer_norm(x, (c.width,)), layer["cross_q"]).view(-1, c.heads, c.head_dim)
        heard = ops.cross_attention_packed(q, k, v, self.audio_lens, self.rows, error_word=self.errors)
        x = x + F.linear(heard.flatten(1), layer["cross_out"])
        return x + F.linear(F.gelu(F.linear(F.layer_norm(x, (c.width,)), layer["up"])), layer["down"])

    # ---- candidates -------------------------------------------------------------------------
    def _fork(self, n: int, steps: int):
        """Blocks for n candidates of each request: the tables that the append indexes by position, those of the
        candidates' own blocks, and the tokens of the shared ones."""
        bs = self.cfg.block_size
        if n < 1 or steps < 1 or not self.tables:
            raise ValueError("a request, a candidate and a step at least")
        if max(self.lengths) + steps > self.cfg.max_positions:
            raise ValueError(f"request of {max(self.lengths) + steps} tokens; positions reach {self.cfg.max_positions}")
        shared = [length // bs for length in self.lengths]
        need = [-(-(length + steps) // bs) - full for length, full in zip(self.lengths, shared)]
        if n * sum(need) > self.blocks.num_free_blocks:
            raise RuntimeError(f"out of physical blocks: candidates need {n * sum(need)}")
        tables, own, copies = [], [], []
        for table, full, length, blocks in zip(self.tables, shared, self.lengths, need):
            for _ in range(n):
                mine = [self.blocks.allocate_block() for _ in range(blocks)]
                if length % bs:
                    copies.append((table[full], mine[0]))
                tables.append(table[:full] + mine)
                own.append(mine)
        if copies:
            old, new = torch.tensor(copies, device=self.device).T
            for i in range(self.cfg.layers):
                for pool in (self.blocks.key_pool[i], self.blocks.value_pool[i]):
                    pool[new] = pool[old]
        device_tables = [self.blocks.block_tables(t, max(len(x) for x in t), device=self.device) for t in (tables, own)]
        return own, *device_tables, self._ints(full * bs for full in shared)

    def sample(self, logits: torch.Tensor, n: int, steps: int, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0,
               min_p: float = 0.0, seed: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
        """n continuations of `steps` tokens for each request, from the logits of its last token: tokens [requests, n,
        steps] and each continuation's log-probability [requests, n].  The requests themselves stay as they are."""
        c, requests = self.cfg, len(self.tables)
        B = n * requests
        own, tables, own_tables, prefix_lens = self._fork(n, steps)
        prefix_tables = self._device_tables()
        self.rows = torch.arange(0, B + 1, n, dtype=torch.int32, device=self.device)
        positions = self._ints(length for length in self.lengths for _ in range(n))
        own_lens = positions - prefix_lens.repeat_interleave(n) + 1
        self.workspace = workspace = ops.shared_prefix_workspace(B, requests, c.heads, c.kv_heads, c.head_dim, c.block_size,
                                                                 prefix_tables.shape[1], own_tables.shape[1], torch.device(self.device))
        draws = torch.rand(steps, B, generator=torch.Generator().manual_seed(seed)).to(self.device)
        u, tokens = draws[0].clone(), torch.zeros(B, dtype=torch.long, device=self.device)
        logprobs, total = torch.zeros(B, device=self.device), torch.zeros(B, device=self.device)
        out = torch.empty(steps, B, dtype=torch.long, device=self.device)

        def draw(rows):
            ops.sample_rows(rows, u, temperature, top_k, top_p, min_p, out=tokens, logprobs=logprobs)
            total.add_(logprobs)

        def network():
            x = self.embed[tokens]
            for i, layer in enumerate(self.layers):
                q, k, v = self._qkv(layer, x)
                q = self._append(i, q, k, v, tables, positions, None)
                attended = ops.shared_prefix_decode_attention(
                    q, self.blocks.key_pool[i], self.blocks.value_pool[i], prefix_tables, prefix_lens, self.rows, own_tables,
                    own_lens, workspace=workspace, error_word=self.errors)
                x = self._rest(layer, x, attended)
            return self._logits(x)

        def step():
            draw(network())
            positions.add_(1)
            own_lens.add_(1)

        draw(logits.repeat_interleave(n, 0))
        if steps > 1:
            # once before the capture, for torch's own workspaces: the same token is written again later
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                network()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=side):
                    step()
            torch.cuda.current_stream().wait_stream(side)
        for s in range(steps):
            out[s] = tokens
            if s + 1 < steps:
                u.copy_(draws[s + 1])
                graph.replay()
        for blocks in own:
            self.blocks.free_blocks(blocks)
        return out.T.reshape(requests, n, steps), total.view(requests, n)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--heads", type=int, default=16)
    ap.add_argument("--kv-heads", type=int, default=4)
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--candidates", type=int, default=16)
    ap.add_argument("--audio", type=int, default=1500)
    ap.add_argument("--longest", type=int, default=400)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--temperature", type=float, default=0.8)
    ap.add_argument("--top-k", type=int, default=0)
    ap.add_argument("--top-p", type=float, default=0.95)
    a = ap.parse_args()
    cfg = Config(heads=a.heads, kv_heads=a.kv_heads, bits=16, max_positions=a.longest + a.steps)
    g = torch.Generator().manual_seed(1)
    lengths = torch.randint(1, a.longest + 1, (a.requests,), generator=g).tolist()
    cfg.num_blocks = sum(-(-n // cfg.block_size) + a.candidates * (-(-a.steps // cfg.block_size) + 1) for n in lengths)
    prompts = [torch.randint(0, cfg.vocab, (n,), generator=g).tolist() for n in lengths]
    model = CandidateDecoder(cfg)
    model.encode(torch.randn(a.requests, a.audio, cfg.width, generator=g).to(model.device, cfg.dtype), [a.audio] * a.requests)
    logits = model.prefill(prompts)
    for timed in (False, True):  # the first pass warms up
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        tokens, scores = model.sample(logits, a.candidates, a.steps, a.temperature, a.top_k, a.top_p)
        torch.cuda.synchronize()
        t1 = time.perf_counter()
        model.check_errors()
        if timed:
            print(f"{a.requests} requests of {min(lengths)} to {max(lengths)} tokens, {a.candidates} candidates each: "
                  f"{tokens.numel() / (t1 - t0):,.0f} tokens/s (capture included)")
            best = scores[0].argmax()
            print(f"the likeliest of the first request ({scores[0, best]:.1f}) goes on with", tokens[0, best, :8].tolist())
    model.release()


if __name__ == "__main__":
    main()
