"""A Llama-shaped decoder served from a paged key-value cache that is kept within a budget, its answers scored.

The dense parts of a step are executables (one plan for all layers: norm, projections, rotation before the attention; output
projection and feed-forward block behind it), the attention between them, the eviction and the scoring are the backend's operators;
all of it works on the backend's buffers and stream. Sequences of a batch have lengths of their own and share one pool of
pages per layer.

    python -m pjrtx_b200.programs.paged_llama        # a toy decoder with random weights
"""
from __future__ import annotations

import dataclasses
from typing import Dict, List, Optional, Sequence

import numpy as np

from .. import plan as P
from ..plan import PlanBuilder
from . import llama

BEFORE = ("attn_norm", "wq", "wk", "wv")
BEHIND = ("wo", "mlp_norm", "w_gate", "w_up", "w_down")


def build_embed(cfg: llama.LlamaConfig, batch: int) -> PlanBuilder:
    """(token[B], embed[V, D]) -> x[B, D]"""
    b = PlanBuilder()
    token, table = b.parameter(P.S32, [batch]), b.parameter(cfg.dtype, [cfg.vocab, cfg.d_model])
    b.set_outputs([b.gather_rows(table, token)])
    return b


def build_before(cfg: llama.LlamaConfig, batch: int) -> PlanBuilder:
    """(x[B, D], position[B], attn_norm, wq, wk, wv) -> rotated q[B, H, hd], rotated k[B, G, hd], v[B, G, hd]"""
    b = PlanBuilder()
    e = llama._Emit(b, cfg)
    x, position = b.parameter(cfg.dtype, [batch, cfg.d_model]), b.parameter(P.S32, [batch])
    shapes = {"attn_norm": [cfg.d_model], "wq": [cfg.d_model, cfg.q_dim], "wk": [cfg.d_model, cfg.kv_dim], "wv": [cfg.d_model, cfg.kv_dim]}
    w = {name: b.parameter(cfg.dtype, shapes[name]) for name in BEFORE}
    cos, sin = e.rope_tables(position, [batch], [0])
    h = e.rms_norm(x, w["attn_norm"])
    q = e.rope(b.reshape(e.linear(h, w["wq"], None), [batch, cfg.heads, cfg.head_dim]), cos, sin)
    k = e.rope(b.reshape(e.linear(h, w["wk"], None), [batch, cfg.kv_heads, cfg.head_dim]), cos, sin)
    v = b.reshape(e.linear(h, w["wv"], None), [batch, cfg.kv_heads, cfg.head_dim])
    b.set_outputs([q, k, v])
    return b


def build_behind(cfg: llama.LlamaConfig, batch: int) -> PlanBuilder:
    """(x[B, D], context[B, H, hd], wo, mlp_norm, w_gate, w_up, w_down) -> x[B, D]"""
    b = PlanBuilder()
    e = llama._Emit(b, cfg)
    x, context = b.parameter(cfg.dtype, [batch, cfg.d_model]), b.parameter(cfg.dtype, [batch, cfg.heads, cfg.head_dim])
    shapes = {"wo": [cfg.q_dim, cfg.d_model], "mlp_norm": [cfg.d_model], "w_gate": [cfg.d_model, cfg.ffn], "w_up": [cfg.d_model, cfg.ffn],
              "w_down": [cfg.ffn, cfg.d_model]}
    w = {name: b.parameter(cfg.dtype, shapes[name]) for name in BEHIND}
    x = x + e.linear(b.reshape(context, [batch, cfg.q_dim]), w["wo"], None)
    h = e.rms_norm(x, w["mlp_norm"])
    gate = e.linear(h, w["w_gate"], None)
    x = x + e.linear(gate * b.unary("logistic", gate) * e.linear(h, w["w_up"], None), w["w_down"], None)
    b.set_outputs([x])
    return b


def build_head(cfg: llama.LlamaConfig, batch: int) -> PlanBuilder:
    """(x[B, D], final_norm, lm_head) -> next token[B], logits[B, V]"""
    b = PlanBuilder()
    e = llama._Emit(b, cfg)
    x, norm, head = (b.parameter(cfg.dtype, d) for d in ([batch, cfg.d_model], [cfg.d_model], [cfg.d_model, cfg.vocab]))
    logits = e.linear(e.rms_norm(x, norm), head, None)
    b.set_outputs([b.argmax(logits, 1)[1], logits])
    return b


@dataclasses.dataclass
class Step:
    """One decoded position of every sequence."""
    next_token: np.ndarray      # [batch], the likeliest one
    log_prob: np.ndarray        # [batch], of next_token
    entropy: np.ndarray         # [batch]
    top_ids: np.ndarray         # [batch, alternatives]
    top_log_probs: np.ndarray   # [batch, alternatives]
    logits: object              # device buffer [batch, vocabulary]


class PagedDecoder:
    """Decodes `batch` sequences of up to `max_pages * page_size` cached tokens each. `weights`: device buffers by the names of
    `llama.weight_shapes`. `keep`: the budget of rows a sequence is cut back to whenever it is full (None: it is an error to
    outgrow the pages); the first `sinks` and last `recent` tokens are never evicted."""

    def __init__(self, backend, cfg: llama.LlamaConfig, weights: Dict[str, object], batch: int, page_size: int, max_pages: int,
                 keep: Optional[int] = None, recent: int = 0, sinks: int = 0, alternatives: int = 4, device: int = 0):
        assert not cfg.int8_weights, "the decoder's plans take weights of its element type"
        self.backend, self.cfg, self.weights, self.batch, self.device = backend, cfg, weights, batch, device
        self.page_size, self.max_pages, self.keep, self.recent, self.sinks = page_size, max_pages, keep, recent, sinks
        self.capacity, self.alternatives = page_size * max_pages, alternatives
        track = keep is not None
        self.cache = backend.paged_cache(cfg.dtype, batch, cfg.heads, cfg.kv_heads, cfg.head_dim, page_size, max_pages, track=track, device=device)
        pages = batch * max_pages
        pool = [pages, page_size, cfg.kv_heads, cfg.head_dim]
        self.pools = [tuple(backend.allocate_buffer(cfg.dtype, pool, device) for _ in "kv") for _ in range(cfg.layers)]
        self.tracked: List[dict] = [{} for _ in range(cfg.layers)]
        if track:
            rows = [batch, cfg.kv_heads, self.capacity]
            self.tracked = [{"weights": backend.allocate_buffer(P.F32, rows, device), "positions": backend.allocate_buffer(P.S32, rows, device)}
                            for _ in range(cfg.layers)]
        self.free = list(range(pages - 1, -1, -1))
        self.table = np.full((batch, max_pages), -1, np.int32)
        self.lengths, self.tokens = np.zeros(batch, np.int32), np.zeros(batch, np.int32)
        self.cut_lengths = backend.allocate_buffer(P.S32, [batch], device)
        self.embed, self.before, self.behind, self.head = (backend.compile_executable(build(cfg, batch), [device]) for build in
                                                           (build_embed, build_before, build_behind, build_head))
        self.scores = {name: backend.allocate_buffer(P.F32, [batch], device) for name in ("log_probs", "entropy")}
        if alternatives:
            self.scores["top_ids"] = backend.allocate_buffer(P.S32, [batch, alternatives], device)
            self.scores["top_log_probs"] = backend.allocate_buffer(P.F32, [batch, alternatives], device)

    def _upload(self, array: np.ndarray):
        return self.backend.buffer_from_host(np.ascontiguousarray(array, np.int32), self.device)

    def _layer(self, index: int, names: Sequence[str]) -> list:
        return [self.weights[f"l{index}.{name}"] for name in names]

    def _grow(self, new: np.ndarray) -> None:
        """Rows for `new` more tokens of each sequence, and pages under them."""
        if np.any(self.lengths + new > self.capacity):
            raise ValueError(f"sequences of up to {int((self.lengths + new).max())} rows, the cache has {self.capacity} each")
        self.lengths += new.astype(np.int32)
        self.tokens += new.astype(np.int32)
        for b in range(self.batch):
            for column in range(-(-int(self.lengths[b]) // self.page_size)):
                if self.table[b, column] < 0:
                    self.table[b, column] = self.free.pop()

    def _evict(self) -> None:
        """Cuts every sequence to the budget and gives the pages behind it back."""
        table, lengths, tokens = self._upload(self.table), self._upload(self.lengths), self._upload(self.tokens)
        for (k, v), tracked in zip(self.pools, self.tracked):
            self.cache.evict(k, v, table, lengths, tokens, tracked["weights"], tracked["positions"], self.keep, recent=self.recent,
                             sinks=self.sinks, lengths_out=self.cut_lengths)
        self.lengths = np.minimum(self.lengths, self.keep).astype(np.int32)
        for b in range(self.batch):
            for column in range(-(-int(self.lengths[b]) // self.page_size), self.max_pages):
                if self.table[b, column] >= 0:
                    self.free.append(int(self.table[b, column]))
                    self.table[b, column] = -1

    def append(self, caches: Sequence[object], counts: Sequence[int]) -> None:
        """Takes the first counts[b] rows of contiguous caches [batch, rows, kv_heads, head_dim] in, keys and values of every
        layer in turn, as a prefill program returns them."""
        counts = np.asarray(counts, np.int32)
        shapes = {tuple(getattr(c, "dims", None) or c.shape) for c in caches}  # buffers, or a tensor library's arrays
        rows = max((s[1] for s in shapes if len(s) == 4), default=0)
        if len(caches) != 2 * self.cfg.layers or shapes != {(self.batch, rows, self.cfg.kv_heads, self.cfg.head_dim)}:
            raise ValueError(f"{2 * self.cfg.layers} caches [{self.batch}, rows, {self.cfg.kv_heads}, {self.cfg.head_dim}] are needed")
        if counts.shape != (self.batch,) or np.any(counts < 0) or np.any(counts > rows):
            raise ValueError(f"a count from 0 to {rows} for each of {self.batch} sequences is needed")
        self._grow(counts)
        table, lengths, tokens, new = (self._upload(a) for a in (self.table, self.lengths, self.tokens, counts))
        for i, ((k, v), tracked) in enumerate(zip(self.pools, self.tracked)):
            self.cache.append(k, v, table, lengths, caches[2 * i], caches[2 * i + 1], counts=new, tokens=tokens if tracked else None, **tracked)

    def step(self, tokens: Sequence[int]) -> Step:
        """Decodes one token of every sequence."""
        be, tokens = self.backend, np.asarray(tokens, np.int32)
        if tokens.shape != (self.batch,):
            raise ValueError(f"a token for each of {self.batch} sequences is needed")
        if self.keep is not None and np.any(self.lengths >= self.capacity):
            self._evict()
        position = self._upload(self.tokens)  # of the token that comes in now
        self._grow(np.ones(self.batch, np.int32))
        table, lengths, seen = self._upload(self.table), self._upload(self.lengths), self._upload(self.tokens)
        x = be.execute_executable(self.embed, [self._upload(tokens), self.weights["embed"]])[0]
        for i, ((k, v), tracked) in enumerate(zip(self.pools, self.tracked)):
            q, k_new, v_new = be.execute_executable(self.before, [x, position] + self._layer(i, BEFORE))
            context = be.allocate_buffer(self.cfg.dtype, [self.batch, self.cfg.heads, self.cfg.head_dim], self.device)
            self.cache.attend(q, k, v, table, lengths, context, k_new=k_new, v_new=v_new, tokens=seen if tracked else None, **tracked)
            x = be.execute_executable(self.behind, [x, context] + self._layer(i, BEHIND))[0]
        next_token, logits = be.execute_executable(self.head, [x, self.weights["final_norm"], self.weights["lm_head"]])
        be.token_log_probs(logits, next_token, **self.scores, device=self.device)
        read = {name: s.to_numpy() for name, s in self.scores.items()}
        none = np.zeros((self.batch, 0))
        return Step(next_token.to_numpy(), read["log_probs"], read["entropy"], read.get("top_ids", none), read.get("top_log_probs", none), logits)


def main() -> None:
    import pjrtx_b200

    be, cfg = pjrtx_b200.Backend(), llama.TINY
    weights = {name: be.buffer_from_host(w) for name, w in llama.make_weights(cfg, seed=0).items()}
    decoder = PagedDecoder(be, cfg, weights, batch=2, page_size=16, max_pages=4, keep=48, recent=16, sinks=4)
    tokens = np.array([3, 7], np.int32)
    for i in range(100):
        s = decoder.step(tokens)
        tokens = s.next_token
        if i % 20 == 19:
            print(f"{i + 1} tokens, {decoder.lengths[0]} rows: next {s.next_token.tolist()}, log probabilities "
                  f"{np.round(s.log_prob, 3).tolist()}, entropy {np.round(s.entropy, 3).tolist()}, alternatives {s.top_ids.tolist()}")
    be.synchronize()


if __name__ == "__main__":
    main()
