"""A serving loop on the decoder: a quantised paged cache, a prefix that the batch shares, long contexts, sampling.

The reference has no model code (see ``decoder``).  ``ServingDecoder`` is ``Decoder`` with

* ``PackedKVCache`` in place of the bf16 cache: half or a quarter of its bytes, in pages;
* any ``Rotary`` positions (layouts, partial heads, scaled frequencies) in place of the fixed ones;
* prompts of any length, in chunks of ``max_prompt`` tokens over what is cached of them;
* a common prefix: stored once, run through the model once, and read once per step for the whole batch;
* ``sample`` in place of the greedy choice.

``python -m tinygrad_mi355x.serving`` runs it on random weights.
"""

from __future__ import annotations

import argparse
import math
import time

import torch

from tinygrad_mi355x.decoder import Decoder, DecoderConfig, DecoderWeights, random_weights
from tinygrad_mi355x.kv_cache import PackedKVCache
from tinygrad_mi355x.rotary import Rotary
from tinygrad_mi355x.runtime import kernels as K
from tinygrad_mi355x.sampling import sample


class ServingDecoder(Decoder):
    """``batch`` sequences of up to ``max_seq`` positions, the first ``prefix`` of them common to all."""

    def __init__(self, weights: DecoderWeights, cfg: DecoderConfig, batch: int, max_seq: int, max_prompt: int, *,
                 prefix: int = 0, page_size: int = 64, k_format: str = "fp8_e4m3", v_format: str = "fp8_e4m3",
                 rotary: Rotary | None = None) -> None:
        if prefix < 0 or prefix % page_size or prefix >= max_seq:
            raise ValueError(f"prefix must be a multiple of {page_size} below {max_seq}, got {prefix}")
        self.prefix, self._cache_kw = prefix, dict(page_size=page_size, k_format=k_format, v_format=v_format)
        super().__init__(weights, cfg, batch, max_seq, max_prompt)
        if rotary is None:
            rotary = Rotary(cfg.head_dim, base=cfg.rope_base, device=self.device)
        rotary.check(self.qkv, cfg.head_dim)
        self.rotary = rotary
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=self.device)
        self.u = torch.zeros(batch, dtype=torch.float32, device=self.device)
        # written to and never replaced, as everything else that a step reads: a captured step holds their addresses
        self._filters = {name: torch.full((batch,), value, dtype=dtype, device=self.device) for name, value, dtype in (
            ("temperature", 1.0, torch.float32), ("top_k", 0, torch.int32), ("top_p", 1.0, torch.float32),
            ("min_p", 0.0, torch.float32))}
        self._prefix_loaded = prefix == 0

    def _allocate_cache(self) -> None:
        cfg, page = self.cfg, self._cache_kw["page_size"]
        cols, common = -(-self.max_seq // page), self.prefix // page
        pages = common + self.batch * (cols - common)
        self.caches = [PackedKVCache(pages, cfg.kv_heads, cfg.head_dim, device=self.device, **self._cache_kw)
                       for _ in range(cfg.layers)]
        # the common pages in front of every row, then each row's own
        table = torch.empty((self.batch, cols), dtype=torch.int32)
        table[:, :common] = torch.arange(common)
        table[:, common:] = torch.arange(common, pages).view(self.batch, cols - common)
        self.table = table.to(self.device)

    def _attention(self, li: int, rows: int, seq_rows: int, splits: int, stream: int) -> None:
        cfg, n = self.cfg, rows // seq_rows
        heads = self.qkv[:rows].view(n, seq_rows, cfg.heads + 2 * cfg.kv_heads, cfg.head_dim)
        q, k, v = heads.split((cfg.heads, cfg.kv_heads, cfg.kv_heads), 2)
        cache, table = self.caches[li], self.table[:n]
        q = cache.append(k, v, table, self.pos[:n], rotary=self.rotary, q=q).q
        out = cache.attend(q, table, self.lengths[:n], shared=self.prefix if n > 1 else 0)
        self.attn[:rows].copy_(out.view(rows, -1))

    def _pass(self, tokens: torch.Tensor | None, n: int, t: int) -> None:
        """``t`` tokens of each of the first ``n`` sequences (their last ones if ``tokens`` is None) through the layers,
        from position ``pos`` on."""
        stream = K.stream_of(self.h)
        if tokens is not None:
            self.tokens[:n * t].copy_(tokens.reshape(-1))
        torch.add(self.pos, t, out=self.lengths)
        K.call("tgm_dec_embed", self.w.embed.data_ptr(), self.cfg.vocab, self.cfg.hidden, self.tokens.data_ptr(), n * t,
               self.h.data_ptr(), stream)
        self._layers(n * t, t, 1, stream)
        self.pos[:n].add_(t)

    def _draw(self, first_row: int, row_stride: int) -> None:
        """Output head over one row per sequence, and a token from each."""
        cfg = self.cfg
        K.call("tgm_dec_gemv_bf16", self.w.lm_head.data_ptr(), cfg.vocab, cfg.hidden, self.xnb[first_row].data_ptr(),
               self.batch, row_stride * cfg.hidden, self.logits.data_ptr(), cfg.vocab, K.stream_of(self.h))
        sample(self.logits, self.u, out=self.tokens[:self.batch], **self._filters)

    def _check_prompt(self, tokens: torch.Tensor, rows: int, name: str) -> None:
        if tokens.dim() != 2 or tokens.shape[0] != rows or tokens.shape[1] < 1:
            raise ValueError(f"{name} must be [{rows}, tokens], got {tuple(tokens.shape)}")
        if int(tokens.min()) < 0 or int(tokens.max()) >= self.cfg.vocab:
            raise ValueError(f"{name} tokens out of range")

    def load_prefix(self, tokens: torch.Tensor) -> None:
        """Run the common prefix (int [prefix]) once, into the pages that every sequence reads."""
        if tokens.dim() != 1 or tokens.shape[0] != self.prefix:
            raise ValueError(f"the prefix must be {self.prefix} tokens, got {tuple(tokens.shape)}")
        if not self.prefix:
            return
        self._check_prompt(tokens[None], 1, "prefix")
        self._prefix_loaded = False
        self.pos.zero_()
        for t0 in range(0, self.prefix, self.max_prompt):
            chunk = tokens[t0:t0 + self.max_prompt]
            self._pass(chunk, 1, chunk.shape[0])
        self._prefix_loaded = True

    def prefill(self, prompts: torch.Tensor) -> torch.Tensor:
        """Run the prompts (int [batch, T], T of any length) behind the prefix, which has to be loaded; the first sampled
        tokens."""
        self._check_prompt(prompts, self.batch, "prompts")
        if self.prefix + prompts.shape[1] > self.max_seq:
            raise ValueError("prefix + prompt exceed max_seq")
        if not self._prefix_loaded:
            raise RuntimeError(f"the prefix of {self.prefix} positions is not loaded: call load_prefix first")
        self.pos.fill_(self.prefix)
        for t0 in range(0, prompts.shape[1], self.max_prompt):
            chunk = prompts[:, t0:t0 + self.max_prompt]
            self._pass(chunk, self.batch, chunk.shape[1])
        self._draw(chunk.shape[1] - 1, chunk.shape[1])
        return self.tokens[:self.batch].clone()

    def _decode_step(self) -> None:
        self._pass(None, self.batch, 1)
        self._draw(0, 1)

    def capture(self) -> torch.cuda.CUDAGraph:
        """One step as a graph, with the tensors it allocates in a pool of its own.  Replays step on from where the decoder
        is (``pos``, ``tokens``, ``u``), with the filters of the last ``generate``."""
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            self._decode_step()
        return graph

    def generate(self, prompts: torch.Tensor, new_tokens: int, u: torch.Tensor, *, temperature=1.0, top_k=0, top_p=1.0,
                 min_p=0.0, graph: bool = True) -> torch.Tensor:
        """[batch, new_tokens] sampled token ids; ``u`` float32 [batch, new_tokens] in [0, 1) are the random numbers,
        the filters (``sampling.sample``) one number or one per sequence."""
        if new_tokens < 1 or self.prefix + prompts.shape[1] + new_tokens - 1 > self.max_seq:
            raise ValueError("prefix + prompt + generated tokens exceed max_seq")
        if u.shape != (self.batch, new_tokens) or u.dtype is not torch.float32 or u.device != self.device:
            raise ValueError(f"u must be float32 [{self.batch}, {new_tokens}] on {self.device}")
        for name, value in (("temperature", temperature), ("top_k", top_k), ("top_p", top_p), ("min_p", min_p)):
            held = self._filters[name]
            held.copy_(torch.as_tensor(value, dtype=held.dtype, device=self.device).expand(self.batch))
        history = torch.empty((self.batch, new_tokens), dtype=torch.int32, device=self.device)
        self.u.copy_(u[:, 0])
        history[:, 0] = self.prefill(prompts)
        step = self._decode_step
        for i in range(1, new_tokens):
            # the first step runs eagerly: it also performs every kernel's one-time set-up
            if graph and i == 2:
                step = self.capture().replay
            self.u.copy_(u[:, i])
            step()
            history[:, i] = self.tokens[:self.batch]
        return history


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--batch", type=int, default=8)
    p.add_argument("--layers", type=int, default=2)
    p.add_argument("--prefix", type=int, default=2048, help="positions common to the batch")
    p.add_argument("--prompt", type=int, default=200)
    p.add_argument("--new", type=int, default=64)
    p.add_argument("--v-format", default="fp8_e4m3")
    a = p.parse_args()
    cfg = DecoderConfig(layers=a.layers)
    max_seq = 64 * math.ceil((a.prefix + a.prompt + a.new) / 64)
    rotary = Rotary(cfg.head_dim, base=cfg.rope_base, scaling=dict(kind="yarn", factor=4.0, trained=4096))
    d = ServingDecoder(random_weights(cfg), cfg, a.batch, max_seq, 512, prefix=a.prefix, v_format=a.v_format, rotary=rotary)
    g = torch.Generator(device="cuda").manual_seed(0)
    tokens = torch.randint(0, cfg.vocab, (a.prefix + a.batch * a.prompt,), device="cuda", generator=g)
    u = torch.rand((a.batch, a.new), device="cuda", generator=g)
    d.load_prefix(tokens[:a.prefix])
    for _ in range(2):  # the first one sets kernels up
        torch.cuda.synchronize()
        start = time.perf_counter()
        out = d.generate(tokens[a.prefix:].view(a.batch, a.prompt), a.new, u, temperature=0.8, top_k=50, top_p=0.95)
        torch.cuda.synchronize()
        took = time.perf_counter() - start
    print(f"{a.batch} sequences of {a.prompt} tokens behind {a.prefix} common ones, {a.new} sampled each: {took * 1e3:.1f} ms, "
          f"cache {sum(c.nbytes() for c in d.caches) / 2**20:.1f} MiB")
    print(out[:, :12].tolist())


if __name__ == "__main__":
    main()
