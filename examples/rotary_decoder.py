"""A decoder with rotary positions, grouped heads and a paged cache of 4 or 16 bits, random weights:
ragged prompts are read in chunks, then decoded one token at a time from a CUDA graph.

    python examples/rotary_decoder.py                 # 4-bit cache, 16 query and 4 key/value heads
    python examples/rotary_decoder.py --bits 16 --kv-heads 16

Prompt chunk, per layer:   rope_kv_append_int4 -> kv_gather_int4 -> prompt_attention
Decode step, per layer:    rope_kv_append_int4 -> paged_decode_attention_int4
With --bits 16 the same through rope_kv_append, the pool's rows and paged_decode_attention, whose
query and key/value heads are as many.  Prompts attend to what the cache holds (their own keys and
values rounded as decode steps will read them), so a token's logits do not depend on how its
context was split into chunks and steps, beyond rounding.
"""
from __future__ import annotations

import argparse
import sys
import time
from dataclasses import dataclass
from pathlib import Path
from typing import List, Sequence

import torch
import torch.nn.functional as F

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "inference-speech-model_b200"))
from speech_serving import ops  # noqa: E402
from speech_serving.block_manager import BlockManager  # noqa: E402


@dataclass
class Config:
    layers: int = 4
    heads: int = 16
    kv_heads: int = 4
    head_dim: int = 64
    vocab: int = 4096
    block_size: int = 16
    num_blocks: int = 2048
    max_positions: int = 2048
    bits: int = 4
    dtype: torch.dtype = torch.float16
    seed: int = 0

    @property
    def width(self) -> int:
        return self.heads * self.head_dim


class RotaryDecoder:
    """Weights, cache and the packed batch of requests of one decoder."""

    def __init__(self, cfg: Config, device: str = "cuda"):
        if cfg.bits not in (4, 16):
            raise ValueError(f"cache of {cfg.bits} bits: 4 or 16")
        if cfg.bits == 16 and cfg.heads != cfg.kv_heads:
            raise ValueError("a 16-bit cache needs as many key/value heads as query heads")
        self.cfg, self.device = cfg, device
        g = torch.Generator().manual_seed(cfg.seed)

        def weight(rows, cols):
            return (torch.randn(rows, cols, generator=g) * cols ** -0.5).to(device, cfg.dtype)

        W, rows = cfg.width, cfg.heads + 2 * cfg.kv_heads
        self.layers = [dict(qkv=weight(rows * cfg.head_dim, W), out=weight(W, W), up=weight(2 * W, W),
                            down=weight(W, 2 * W)) for _ in range(cfg.layers)]
        self.embed = weight(cfg.vocab, W) * W ** 0.5
        self.head = weight(cfg.vocab, W)
        inv = 10000.0 ** (-torch.arange(0, cfg.head_dim, 2, dtype=torch.float64) / cfg.head_dim)
        a = torch.arange(cfg.max_positions, dtype=torch.float64)[:, None] * inv
        self.cos, self.sin = a.cos().float().to(device), a.sin().float().to(device)
        # Block ids come from the manager; with 4 bits only its free list is used, with one id per block
        # for all layers' pools.
        if cfg.bits == 4:
            self.blocks = BlockManager(1, 1, 1, cfg.block_size, cfg.num_blocks, device="cpu")
            self.pools = [ops.kv_pool_int4(cfg.num_blocks, cfg.kv_heads, cfg.head_dim, cfg.block_size, device)
                          for _ in range(cfg.layers)]
        else:
            self.blocks = BlockManager(cfg.layers, cfg.kv_heads, cfg.head_dim, cfg.block_size, cfg.num_blocks, cfg.dtype,
                                       device)
        self.errors = torch.zeros(1, dtype=torch.int32, device=device)
        self.workspace = None  # of the last decode() call's attention
        self.tables: List[List[int]] = []
        self.lengths: List[int] = []

    # ---- requests ---------------------------------------------------------------------------
    def _reserve(self, request: int, tokens: int) -> None:
        if tokens > self.cfg.max_positions:
            raise ValueError(f"request of {tokens} tokens; positions reach {self.cfg.max_positions}")
        while len(self.tables[request]) * self.cfg.block_size < tokens:
            self.tables[request].append(self.blocks.allocate_block())

    def _device_tables(self) -> torch.Tensor:
        return self.blocks.block_tables(self.tables, max(1, max(len(t) for t in self.tables)), device=self.device)

    def _ints(self, values: Sequence[int]) -> torch.Tensor:
        return torch.tensor(list(values), dtype=torch.int32, device=self.device)

    def release(self) -> None:
        """Gives all blocks back."""
        for t in self.tables:
            self.blocks.free_blocks(t)
        self.tables, self.lengths = [], []

    def _decode_workspace(self, columns: int) -> torch.Tensor:
        c, n, device = self.cfg, len(self.tables), torch.device(self.device)
        if c.bits == 4:
            return ops.decode_int4_workspace(n, c.heads, c.kv_heads, c.head_dim, c.block_size, columns, c.dtype, device)
        return ops.paged_attn_workspace(n, c.heads, c.head_dim, columns, device)

    def check_errors(self) -> None:
        word = ops.read_error_word(self.errors)
        if self.workspace is not None:
            word |= ops.read_error_word(self.workspace)  # where paged_decode_attention leaves its flags
        if word:
            raise RuntimeError(f"a kernel refused a length or a block id, or gave up waiting: {word:#x}")

    # ---- the network ------------------------------------------------------------------------
    def _qkv(self, layer, x):
        """q, k, v as strided views of one packed projection."""
        c = self.cfg
        y = F.linear(F.layer_norm(x, (c.width,)), layer["qkv"]).view(-1, c.heads + 2 * c.kv_heads, c.head_dim)
        return y.split((c.heads, c.kv_heads, c.kv_heads), 1)

    def _append(self, i, q, k, v, tables, positions, cu):
        if self.cfg.bits == 4:
            return ops.rope_kv_append_int4(q, k, v, self.cos, self.sin, self.pools[i], tables, positions, cu,
                                           error_word=self.errors)
        return ops.rope_kv_append(q, k, v, self.cos, self.sin, self.blocks.key_pool[i], self.blocks.value_pool[i], tables,
                                  positions, cu, error_word=self.errors)

    def _rest(self, layer, x, attended):
        x = x + F.linear(attended.flatten(1), layer["out"])
        return x + F.linear(F.gelu(F.linear(F.layer_norm(x, (self.cfg.width,)), layer["up"])), layer["down"])

    def _logits(self, x):
        return F.linear(F.layer_norm(x, (self.cfg.width,)), self.head)

    # ---- prompts ----------------------------------------------------------------------------
    def prefill(self, prompts: Sequence[Sequence[int]], chunk: int = 512) -> torch.Tensor:
        """Reads new requests, at most `chunk` tokens of each at a time; the logits of every prompt's last
        token [requests, vocab]."""
        if self.tables or not prompts or any(len(p) == 0 for p in prompts):
            raise ValueError("prefill needs prompts of one token or more, and no request in the cache")
        self.tables, self.lengths = [[] for _ in prompts], [0] * len(prompts)
        last = torch.empty(len(prompts), self.cfg.vocab, dtype=self.cfg.dtype, device=self.device)
        while any(n < len(p) for n, p in zip(self.lengths, prompts)):
            starts = list(self.lengths)
            news = [min(chunk, len(p) - n) for n, p in zip(starts, prompts)]
            for r, n in enumerate(news):
                self.lengths[r] += n
                self._reserve(r, self.lengths[r])
            packed = [t for p, s, n in zip(prompts, starts, news) for t in p[s : s + n]]
            logits = self._chunk(packed, starts, news)
            ends = torch.tensor(news).cumsum(0) - 1
            done = [r for r, p in enumerate(prompts) if news[r] and self.lengths[r] == len(p)]
            last[done] = logits[ends[done].to(self.device)]
        return last

    def _chunk(self, packed, starts, news):
        tables, positions = self._device_tables(), self._ints(starts)
        cu_q = F.pad(self._ints(news).cumsum(0, dtype=torch.int32), (1, 0))
        # a request without new tokens takes no part: no keys either
        seen = [s + n if n else 0 for s, n in zip(starts, news)]
        cu_k = F.pad(self._ints(seen).cumsum(0, dtype=torch.int32), (1, 0))
        if self.cfg.bits == 16:  # the pool's row of each key
            bs = self.cfg.block_size
            rows = torch.tensor([t[p // bs] * bs + p % bs for t, n in zip(self.tables, seen) for p in range(n)],
                                device=self.device)
        x = self.embed[torch.tensor(packed, device=self.device)]
        for i, layer in enumerate(self.layers):
            q, k, v = self._qkv(layer, x)
            q = self._append(i, q, k, v, tables, positions, cu_q)
            if self.cfg.bits == 4:
                k, v = ops.kv_gather_int4(self.pools[i], tables, cu_k, sum(seen), self.cfg.head_dim, self.cfg.dtype,
                                          error_word=self.errors)
            else:
                k, v = (p.flatten(0, 1)[rows] for p in (self.blocks.key_pool[i], self.blocks.value_pool[i]))
            x = self._rest(layer, x, ops.prompt_attention(q, k, v, cu_q, cu_k, error_word=self.errors))
        return self._logits(x)

    # ---- decode -----------------------------------------------------------------------------
    def _step(self, tokens, positions, context, tables, workspace):
        x = self.embed[tokens]
        for i, layer in enumerate(self.layers):
            q, k, v = self._qkv(layer, x)
            q = self._append(i, q, k, v, tables, positions, None)
            if self.cfg.bits == 4:
                attended = ops.paged_decode_attention_int4(q, self.pools[i], tables, context, workspace=workspace,
                                                           error_word=self.errors)
            else:
                attended = ops.paged_decode_attention(q, self.blocks.key_pool[i], self.blocks.value_pool[i], tables, context,
                                                      workspace=workspace)
            x = self._rest(layer, x, attended)
        return self._logits(x)

    def decode(self, logits: torch.Tensor, steps: int) -> torch.Tensor:
        """Greedy continuation of every request by `steps` tokens [requests, steps], from the logits of its
        last token; the step is captured once and replayed."""
        for r, n in enumerate(self.lengths):
            self._reserve(r, n + steps)
        tables, positions = self._device_tables(), self._ints(self.lengths)
        context = positions + 1
        workspace = self.workspace = self._decode_workspace(tables.shape[1])
        tokens = ops.argmax_rows(logits)
        out = torch.empty(steps, len(self.tables), dtype=torch.long, device=self.device)

        def step():
            ops.argmax_rows(self._step(tokens, positions, context, tables, workspace), out=tokens)
            positions.add_(1)
            context.add_(1)

        if steps > 1:
            # once before the capture, for torch's own workspaces: the same token is written again later
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                self._step(tokens, positions, context, tables, workspace)
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=side):
                    step()
            torch.cuda.current_stream().wait_stream(side)
        for s in range(steps):
            out[s] = tokens
            if s + 1 < steps:
                graph.replay()
        self.lengths = [n + max(0, steps - 1) for n in self.lengths]  # the last token is not in the cache
        return out.T


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--bits", type=int, default=4)
    ap.add_argument("--heads", type=int, default=16)
    ap.add_argument("--kv-heads", type=int, default=4)
    ap.add_argument("--head-dim", type=int, default=64)
    ap.add_argument("--requests", type=int, default=16)
    ap.add_argument("--longest", type=int, default=1500)
    ap.add_argument("--chunk", type=int, default=512)
    ap.add_argument("--steps", type=int, default=64)
    a = ap.parse_args()
    cfg = Config(heads=a.heads, kv_heads=a.kv_heads, head_dim=a.head_dim, bits=a.bits,
                 max_positions=a.longest + a.steps)
    g = torch.Generator().manual_seed(1)
    lengths = torch.randint(1, a.longest + 1, (a.requests,), generator=g).tolist()
    cfg.num_blocks = sum(-(-(n + a.steps) // cfg.block_size) for n in lengths)
    prompts = [torch.randint(0, cfg.vocab, (n,), generator=g).tolist() for n in lengths]
    model = RotaryDecoder(cfg)
    for timed in (False, True):  # the first pass warms up
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        logits = model.prefill(prompts, a.chunk)
        torch.cuda.synchronize()
        t1 = time.perf_counter()
        tokens = model.decode(logits, a.steps)
        torch.cuda.synchronize()
        t2 = time.perf_counter()
        model.check_errors()
        if timed:
            print(f"{a.bits}-bit cache, {a.requests} requests of {min(lengths)} to {max(lengths)} tokens: "
                  f"prompts {sum(lengths) / (t1 - t0):,.0f} tokens/s, "
                  f"decode {a.requests * a.steps / (t2 - t1):,.0f} tokens/s (capture included)")
            print("first request continues with", tokens[0, :8].tolist())
        model.release()


if __name__ == "__main__":
    main()
