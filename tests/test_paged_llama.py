"""A decoder over a paged cache against the same decoder over contiguous caches, and with its cache cut back as it goes."""
import numpy as np
import pytest

from pjrtx_b200 import backend as be_mod
from pjrtx_b200.programs import llama, paged_llama
from tests.util import assert_close

pytestmark = pytest.mark.gpu


def _weights(be, cfg):
    host = llama.make_weights(cfg, seed=0)
    return host, {name: be.buffer_from_host(w) for name, w in host.items()}


@pytest.mark.parametrize("batch,page_size", [(1, 16), (3, 10)])
def test_paged_decoding_follows_contiguous_decoding(gpu_backend, batch, page_size):
    be, cfg, steps, seq = gpu_backend, llama.TINY, 6, 21
    host, weights = _weights(be, cfg)
    builder, _ = llama.build_prefill(cfg, batch, seq)
    prompt = np.random.default_rng(0).integers(0, cfg.vocab, (batch, seq)).astype(np.int32)
    prefilled = be.execute_executable(be.compile_executable(builder), [be.buffer_from_host(prompt)] + [weights[n] for n, _ in llama.weight_shapes(cfg)])
    max_len = seq + steps
    step_builder, names = llama.build_decode_step(cfg, batch, max_len, return_logits=True)
    step = be.compile_executable(step_builder)
    caches = []
    for c in prefilled[1:]:
        full = np.zeros((batch, max_len, cfg.kv_heads, cfg.head_dim), c.to_numpy().dtype)
        full[:, :seq] = c.to_numpy()
        caches.append(be.buffer_from_host(full))
    paged = paged_llama.PagedDecoder(be, cfg, weights, batch, page_size, -(-max_len // page_size))
    paged.append(prefilled[1:], [seq] * batch)
    token = prefilled[0].to_numpy()
    for i in range(steps):
        outs = be.execute_executable(step, [be.buffer_from_host(token), be.buffer_from_host(np.array(seq + i, np.int32))]
                                     + [weights[n] for n in names[2:2 + len(weights)]] + caches)
        caches = outs[2:]
        want = outs[1].to_numpy().astype(np.float64)
        got = paged.step(token)
        logits = got.logits.to_numpy().astype(np.float64)
        assert_close(logits, want, 2e-2, what=f"step {i} logits")
        log_p = logits - np.log(np.exp(logits - logits.max(1, keepdims=True)).sum(1, keepdims=True)) - logits.max(1, keepdims=True)
        assert np.array_equal(got.next_token, logits.argmax(1)) and np.array_equal(got.top_ids[:, 0], got.next_token)
        assert np.abs(got.log_prob - log_p[np.arange(batch), got.next_token]).max() < 1e-4
        assert np.abs(got.entropy + (np.exp(log_p) * log_p).sum(1)).max() < 1e-3
        token = outs[0].to_numpy()
    be.synchronize()


def test_a_refused_call_leaves_the_decoder_as_it_was(gpu_backend):
    be, cfg, batch, seq = gpu_backend, llama.TINY, 2, 9
    _, weights = _weights(be, cfg)
    caches = [be.allocate_buffer(cfg.dtype, [batch, seq, cfg.kv_heads, cfg.head_dim]) for _ in range(2 * cfg.layers)]
    decoder = paged_llama.PagedDecoder(be, cfg, weights, batch, 8, 4)
    decoder.append(caches, [seq, 4])
    state = lambda: (decoder.lengths.tolist(), decoder.tokens.tolist(), decoder.table.tolist(), list(decoder.free))
    before = state()
    short = [be.allocate_buffer(cfg.dtype, [batch, seq, cfg.kv_heads, cfg.head_dim - 8])] * (2 * cfg.layers)
    for refused in (lambda: decoder.append(caches, [3]), lambda: decoder.append(caches, [-1, 2]), lambda: decoder.append(caches, [1, seq + 1]),
                    lambda: decoder.append(caches[:-1], [1, 1]), lambda: decoder.append(short, [1, 1]), lambda: decoder.append(caches, [9, 30]),
                    lambda: decoder.step([1]), lambda: decoder.step([1, 2, 3])):
        with pytest.raises((ValueError, be_mod.BackendError)):
            refused()
        assert state() == before
    decoder.step([1, 2])
    assert decoder.lengths.tolist() == [seq + 1, 5]
    be.synchronize()


def test_a_cache_within_its_budget(gpu_backend):
    be, cfg, batch = gpu_backend, llama.TINY, 2
    _, weights = _weights(be, cfg)
    keep, recent, sinks, page, pages = 40, 12, 3, 8, 6
    bounded = paged_llama.PagedDecoder(be, cfg, weights, batch, page, pages, keep=keep, recent=recent, sinks=sinks)
    whole = paged_llama.PagedDecoder(be, cfg, weights, batch, page, 16)
    rng = np.random.default_rng(1)
    for i in range(100):
        token = rng.integers(0, cfg.vocab, batch).astype(np.int32)
        a, b = bounded.step(token), whole.step(token)
        if i < page * pages:  # nothing was evicted yet
            assert_close(a.logits.to_numpy(), b.logits.to_numpy(), 2e-2, what=f"step {i}")
        assert np.isfinite(a.log_prob).all() and np.isfinite(a.entropy).all()
        n = int(bounded.lengths[0])
        assert n <= page * pages and (i < page * pages or n >= keep + 1)
        assert len(bounded.free) == batch * (pages - -(-n // page))
    for layer in bounded.tracked:
        positions, seen = layer["positions"].to_numpy()[:, :, :n], layer["weights"].to_numpy()
        for p in positions.reshape(-1, n):
            assert len(set(p.tolist())) == n and set(range(sinks)) <= set(p.tolist()) and set(range(100 - recent, 100)) <= set(p.tolist())
        # every head of a step gives its weights to the rows: what is there is at most one unit a head and step
        assert (seen >= 0).all() and (seen.sum(-1) <= 100 * (cfg.heads // cfg.kv_heads) * 1.001).all()
        assert (seen[:, :, n:] == 0).all() and (layer["positions"].to_numpy()[:, :, n:] <= 0).all()
    be.synchronize()
    with pytest.raises(ValueError, match="the cache has 128"):
        for i in range(40):
            whole.step([1, 2])
