"""The operators around a paged key-value cache and a decoder's logits, as measurable cases and a way to draw more.

A cache is a pool of pages [pages, page, kv_heads, head_dim] for keys and one for values; row `t` of sequence `b` is row
`t % page` of page `page_table[b, t // page]`, and `lengths[b]` counts the rows, those that a call appends among them.

  append   writes the rows of new tokens behind those that the sequences have
  attend   attention of one new token per sequence over its pages. `append`: the token's own key and value come with the call
           and are stored too. `track`: every row's attention weight, summed over the query heads that share it, is added up
  evict    keeps `keep` rows of every (sequence, KV head): the first `sinks` and last `recent` tokens, then those with the
           most weight (ties: the lowest row). Kept rows beyond `keep` move into the places of dropped ones before it
  score    log probability of one given token per row of logits, the distribution's entropy and its `top` likeliest tokens
  grad     gradient of the logits from gradients of the log probabilities and entropies
"""
import math
import random

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODE = {"f32": 2, "f16": 7, "bf16": 8}  # element-type codes of the C ABI
ESIZE = {"f32": 4, "f16": 2, "bf16": 2}
MOST_CACHE = 540e6   # bytes of keys and values that a case may have
MOST_LOGITS = 1.06e9


def _attend(name, dtype, batch, heads, kv_heads, head_dim, page, longest, append=True, track=False):
    return {"name": name, "kind": "attend", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "longest": longest, "append": append, "track": track}


def _append(name, dtype, batch, kv_heads, head_dim, page, longest, new, track):
    return {"name": name, "kind": "append", "dtype": dtype, "batch": batch, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "longest": longest, "new": new, "track": track}


def _evict(name, dtype, batch, kv_heads, head_dim, page, longest, keep, recent, sinks):
    return {"name": name, "kind": "evict", "dtype": dtype, "batch": batch, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "longest": longest, "keep": keep, "recent": recent, "sinks": sinks}


def _score(name, dtype, rows, vocab, top, banned=0.0, scale=1.0):
    return {"name": name, "kind": "score", "dtype": dtype, "rows": rows, "vocab": vocab, "top": top, "banned": banned, "scale": scale}


def _grad(name, dtype, rows, vocab, entropy, scale=1.0):
    return {"name": name, "kind": "grad", "dtype": dtype, "rows": rows, "vocab": vocab, "entropy": entropy, "scale": scale}


def listed():
    return [
        # a single chat, one layer of an 8B-shaped decoder, a short odd length: latency
        _attend("attend_b1_517", "bf16", 1, 32, 8, 128, 16, 517),
        # batched serving on the same decoder, ragged lengths up to 2048, one slot of the batch idle
        _attend("attend_b32_2048", "bf16", 32, 32, 8, 128, 16, 2048),
        # two long documents, 70B-shaped heads, large pages, the rows already appended
        _attend("attend_long_65536", "f16", 2, 64, 8, 128, 64, 65536, append=False),
        # serving with a bounded cache: weights are added up for the eviction that follows
        _attend("attend_track_b16_4096", "bf16", 16, 32, 8, 128, 16, 4096, track=True),
        # the rows of one decode step
        _append("append_b32_step", "bf16", 32, 8, 128, 16, 2048, 1, False),
        # four prompts going into the cache
        _append("append_b4_prompts", "bf16", 4, 8, 128, 16, 2048, 2048, True),
        # one row over the budget: what a bounded cache does at every step
        _evict("evict_b1_step", "bf16", 1, 8, 128, 16, 2049, 2048, 256, 4),
        # a batch cut to half at once
        _evict("evict_b16_4096", "bf16", 16, 8, 128, 16, 4096, 2048, 512, 4),
        # a sampled token's log probability and alternatives, after a grammar has ruled most of the vocabulary out
        _score("score_n1_banned", "bf16", 1, 128256, 20, banned=0.9, scale=1.25),
        # scoring two prompts of 2048 tokens
        _score("score_n4096", "bf16", 4096, 128256, 5),
        # a small policy update: a few sequences of a smaller decoder with an odd vocabulary
        _grad("grad_n97_odd_vocab", "f16", 97, 32001, True, scale=0.8),
        # a training batch with f32 logits
        _grad("grad_n2048_f32", "f32", 2048, 128256, False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend"] * 5 + ["append"] * 2 + ["evict"] * 2 + ["score"] * 3 + ["grad"] * 2)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind in ("score", "grad"):
        vocab = rng.choice([1024, 32000, 32001, 128256, _log_int(rng, 40, 128256)])
        rows = max(1, min(_log_int(rng, 1, 4096), int(MOST_LOGITS / (vocab * ESIZE[dtype]))))
        scale = rng.choice([1.0, round(rng.uniform(0.5, 2.0), 3)])
        if kind == "score":
            case = _score("", dtype, rows, vocab, rng.choice([0, 1, 5, 20, rng.randint(2, 32)]), rng.choice([0.0, 0.0, 0.9]), scale)
        else:
            case = _grad("", dtype, rows, vocab, rng.random() < 0.5, scale)
    else:
        heads, kv_heads, head_dim = rng.choice([(32, 8, 128), (32, 8, 128), (64, 8, 128), (8, 1, 128), (16, 8, 128), (8, 8, 64), (4, 2, 64)])
        page = rng.choice([8, 16, 16, 20, 32, 64, 128])
        batch = _log_int(rng, 1, 64)
        row = 2 * kv_heads * head_dim * ESIZE[dtype]
        longest = min(_log_int(rng, 16, 65536), max(16, int(MOST_CACHE / (batch * row))))
        if kind == "attend":
            case = _attend("", dtype, batch, heads, kv_heads, head_dim, page, longest, rng.random() < 0.7, rng.random() < 0.3)
        elif kind == "append":
            longest = min(longest, 8192)
            case = _append("", dtype, batch, kv_heads, head_dim, page, longest, rng.choice([1, _log_int(rng, 1, longest)]), rng.random() < 0.5)
        else:
            longest = min(longest, 32768)
            keep = rng.choice([longest - 1, max(8, int(longest * rng.uniform(0.3, 0.95)))])
            case = _evict("", dtype, batch, kv_heads, head_dim, page, longest, keep, _log_int(rng, 1, max(1, keep // 2)), rng.choice([0, 4]))
    case.pop("name")
    return case


# ---- inputs --------------------------------------------------------------------------------------------------------


def _randn(gen, dtype, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)


def _lengths(case):
    """Lengths of the batch: from `longest` down to a third of it; of eight sequences and more the last slot is idle."""
    n, longest = case["batch"], case["longest"]
    out = [max(1, longest - (longest * 2 * i) // (3 * n)) for i in range(n)]
    if n >= 8:
        out[-1] = 0
    return out


def _news(case, lengths):
    """Rows that an append writes to each sequence."""
    return [min(case["new"], n) for n in lengths]


def _max_pages(case):
    return -(-case["longest"] // case["page"])


def _cache(case, gen):
    """The pools, the page table and the lengths: pages in a random order, -1 in the table beyond a sequence's own."""
    dtype, page, max_pages = TORCH[case["dtype"]], case["page"], _max_pages(case)
    lengths = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    lengths = lengths[torch.randperm(case["batch"], generator=gen, device="cuda")]
    count = (lengths.long() + page - 1) // page
    pages = int(sum(-(-n // page) for n in _lengths(case))) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").int()
    column = torch.arange(max_pages, device="cuda")
    first = torch.cumsum(count, 0) - count
    table = torch.where(column < count[:, None], order[(first[:, None] + column).clamp(max=pages - 1)], -1)
    shape = (pages, page, case["kv_heads"], case["head_dim"])
    return {"k_pages": _randn(gen, dtype, *shape), "v_pages": _randn(gen, dtype, *shape), "page_table": table.int().contiguous(),
            "lengths": lengths.contiguous()}


def _tracking(case, lengths, gen):
    """Weights and positions of a cache that was cut before: the rows are in no order and the middle half of the tokens is gone."""
    capacity = _max_pages(case) * case["page"]
    shape = (case["batch"], case["kv_heads"], capacity)
    slot = torch.arange(capacity, device="cuda")
    there = slot < lengths[:, None, None]
    weights = torch.exp(2 * torch.randn(shape, generator=gen, device="cuda")) * (torch.rand(shape, generator=gen, device="cuda") > 0.05)
    order = torch.where(there, torch.rand(shape, generator=gen, device="cuda"), 2.0).argsort(-1).argsort(-1)
    gap = (lengths // 2)[:, None, None]
    positions = torch.where(order < gap, order, order + gap)
    return {"tokens": (lengths + lengths // 2).int().contiguous(), "weights": torch.where(there, weights, 0.0).contiguous(),
            "positions": torch.where(there, positions, -1).int().contiguous()}


def _backend():
    import pjrtx_b200

    return pjrtx_b200.Backend()


def _paged_cache(case):
    """The handle that a program keeps for all layers of this shape."""
    return _backend().paged_cache(CODE[case["dtype"]], case["batch"], case.get("heads", case["kv_heads"]), case["kv_heads"],
                                            case["head_dim"], case["page"], _max_pages(case), track=case.get("track", True))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, kind = TORCH[case["dtype"]], case["kind"]
    if kind in ("score", "grad"):
        rows, vocab = case["rows"], case["vocab"]
        logits = _randn(gen, dtype, rows, vocab).mul_(3)
        tokens = torch.randint(0, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
        if rows >= 8:
            tokens[-1] = -1  # a padded position
        s = {"case": case, "logits": logits, "tokens": tokens}
        if kind == "score":
            if case["banned"]:
                given = logits.gather(1, tokens.clamp(min=0).long()[:, None])
                logits.masked_fill_(torch.rand(logits.shape, generator=gen, device="cuda") < case["banned"], -math.inf)
                logits.scatter_(1, tokens.clamp(min=0).long()[:, None], given)
            for name in ("log_probs", "entropy", "lse"):
                s[name] = torch.empty(rows, device="cuda")
            s["top_ids"] = torch.empty((rows, case["top"]), dtype=torch.int32, device="cuda")
            s["top_log_probs"] = torch.empty((rows, case["top"]), device="cuda")
        else:
            x = logits.float() * case["scale"]
            s["lse"] = torch.logsumexp(x, 1)
            s["entropy"] = s["lse"] - (torch.softmax(x, 1) * x).sum(1)
            s["grad_log_probs"] = _randn(gen, torch.float32, rows)
            s["grad_entropy"] = _randn(gen, torch.float32, rows).mul_(0.1) if case["entropy"] else None
            s["grad_logits"] = torch.empty_like(logits)
        s["backend"] = _backend() if own else None
        return s
    s = {"case": case, **_cache(case, gen)}
    batch, kv_heads, dim = case["batch"], case["kv_heads"], case["head_dim"]
    if kind == "evict" or case["track"]:
        s.update(_tracking(case, s["lengths"], gen))
    if kind == "append":
        s["counts"] = torch.minimum(s["lengths"], torch.tensor(case["new"], device="cuda")).int()
        s["k_new"], s["v_new"] = _randn(gen, dtype, batch, case["new"], kv_heads, dim), _randn(gen, dtype, batch, case["new"], kv_heads, dim)
    elif kind == "attend":
        s["q"] = _randn(gen, dtype, batch, case["heads"], dim).mul_(2)
        if case["append"]:
            s["k_new"], s["v_new"] = _randn(gen, dtype, batch, kv_heads, dim), _randn(gen, dtype, batch, kv_heads, dim)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty((batch, case["heads"]), device="cuda")
    else:
        for name in ("lengths", "weights", "positions"):
            s[name + "_out"] = torch.empty_like(s[name])
    s["cache"] = _paged_cache(case) if own else None
    return s


# ---- the plain forms -----------------------------------------------------------------------------------------------


def _places(s, slot):
    """Page and row of slot[b, ...] of every sequence; slots out of a sequence's pages give those of another one."""
    page, shape = s["case"]["page"], slot.shape
    flat = slot.reshape(shape[0], -1)
    pages = s["page_table"].long().gather(1, (flat // page).clamp(0, s["page_table"].shape[1] - 1)).clamp(min=0)
    return pages.reshape(shape), flat.reshape(shape) % page


def _plain_append(s):
    lengths, counts = s["lengths"].long()[:, None], s["counts"].long()[:, None]
    t = torch.arange(s["k_new"].shape[1], device="cuda")[None]
    slot = lengths - counts + t
    b, at = (t < counts).nonzero(as_tuple=True)
    page, row = _places(s, slot)
    page, row, slot = page[b, at], row[b, at], slot[b, at]
    s["k_pages"][page, row] = s["k_new"][b, at]
    s["v_pages"][page, row] = s["v_new"][b, at]
    if s["case"]["track"]:
        s["weights"][b, :, slot] = 0.0
        s["positions"][b, :, slot] = (s["tokens"].long()[:, None] - counts + t).int()[b, at][:, None]


def _plain_attend(s):
    case = s["case"]
    batch, kv_heads, dim = case["batch"], case["kv_heads"], case["head_dim"]
    rep = case["heads"] // kv_heads
    lengths = s["lengths"].long()
    if case["append"]:
        b = lengths.nonzero()[:, 0]
        page, row = _places(s, (lengths - 1).clamp(min=0)[:, None])
        s["k_pages"][page[b, 0], row[b, 0]] = s["k_new"][b]
        s["v_pages"][page[b, 0], row[b, 0]] = s["v_new"][b]
    table = s["page_table"].long().clamp(min=0)
    slot = torch.arange(table.shape[1] * case["page"], device="cuda")
    there = (slot < lengths[:, None])[:, None, None]
    k = s["k_pages"][table].reshape(batch, -1, kv_heads, dim).permute(0, 2, 3, 1).float()
    scores = torch.matmul(s["q"].reshape(batch, kv_heads, rep, dim).float(), k) * (1.0 / math.sqrt(dim))
    del k
    scores = torch.where(there, scores, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    e = torch.exp(scores - top)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total > 0, total, 1.0)
    v = s["v_pages"][table].reshape(batch, -1, kv_heads, dim).permute(0, 2, 1, 3).float()
    out = torch.matmul(p, v).reshape(batch, kv_heads * rep, dim).to(s["q"].dtype)
    lse = torch.where(total > 0, top + torch.log(total), -math.inf).reshape(batch, kv_heads * rep)
    if case["track"]:
        last = (lengths - 1).clamp(min=0)
        b = lengths.nonzero()[:, 0]
        if case["append"]:
            s["weights"][b, :, last[b]] = 0.0
            s["positions"][b, :, last[b]] = (s["tokens"] - 1)[b][:, None]
        s["weights"] += p.sum(2)
    return out, lse


def _plain_evict(s):
    case, weights, positions = s["case"], s["weights"], s["positions"]
    keep, capacity = case["keep"], weights.shape[-1]
    lengths, tokens = s["lengths"].long()[:, None, None], s["tokens"].long()[:, None, None]
    slot = torch.arange(capacity, device="cuda")
    there = slot < lengths
    protected = (positions < case["sinks"]) | (positions >= tokens - case["recent"])
    bits = torch.where(weights == 0, 0.0, weights).view(torch.int32).long()
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) + protected.long() * (1 << 33)
    key = torch.where(there, order * (1 << 20) + (capacity - 1 - slot), -(1 << 60))
    kept = torch.zeros_like(there.expand_as(key)).scatter(-1, key.topk(min(keep, capacity), -1).indices, True) & there
    left = lengths.clamp(max=keep)
    stays = kept & (slot < left)
    hole, source = (~kept & (slot < left)).nonzero(as_tuple=True), (kept & (slot >= left)).nonzero(as_tuple=True)
    weights_out, positions_out = torch.where(stays, weights, 0.0), torch.where(stays, positions, -1)
    weights_out[hole], positions_out[hole] = weights[source], positions[source]
    page, row = s["page_table"].long(), case["page"]
    to = page[hole[0], hole[2] // row], hole[2] % row, hole[1]
    at = page[source[0], source[2] // row], source[2] % row, source[1]
    s["k_pages"][to] = s["k_pages"][at]
    s["v_pages"][to] = s["v_pages"][at]
    return left[:, 0, 0].int(), weights_out, positions_out


def _plain_score(s):
    case, logits, tokens = s["case"], s["logits"], s["tokens"].long()
    x = logits.float()
    bits = torch.where(x == 0, 0.0, x).view(torch.int32).long()
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    key = order * (1 << 20) + (x.shape[1] - 1 - torch.arange(x.shape[1], device="cuda"))
    ids = (x.shape[1] - 1) - (key.topk(case["top"], 1).values & ((1 << 20) - 1))
    del bits, order, key
    x = x * case["scale"]
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    lse = top + torch.log(total)
    e *= torch.where(e > 0, x - top, 0.0)
    entropy = (torch.log(total) - e.sum(1, keepdim=True) / total)[:, 0]
    given = x.gather(1, tokens.clamp(min=0)[:, None]) - lse
    return {"log_probs": torch.where(tokens >= 0, given[:, 0], 0.0), "entropy": entropy, "lse": lse[:, 0],
            "top_ids": ids.int(), "top_log_probs": x.gather(1, ids) - lse}


def _plain_grad(s):
    case, tokens = s["case"], s["tokens"].long()
    log_p = s["logits"].float() * case["scale"] - s["lse"][:, None]
    p = torch.exp(log_p)
    given = torch.where(tokens >= 0, s["grad_log_probs"], 0.0)[:, None]
    grad = -given * p
    if case["entropy"]:
        grad -= s["grad_entropy"][:, None] * p * torch.where(p > 0, log_p + s["entropy"][:, None], 0.0)
    grad.scatter_add_(1, tokens.clamp(min=0)[:, None], given)
    return (grad * case["scale"]).to(s["logits"].dtype)


# ---- one pass ------------------------------------------------------------------------------------------------------


def _plain(s):
    kind = s["case"]["kind"]
    if kind == "score":
        return _plain_score(s)
    if kind == "grad":
        return {"grad_logits": _plain_grad(s)}
    if kind == "evict":
        lengths, weights, positions = _plain_evict(s)
        return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "lengths": lengths, "weights": weights, "positions": positions}
    out = {}
    if kind == "append":
        _plain_append(s)
    else:
        out["out"], out["lse"] = _plain_attend(s)
    return _state_of(s, out)


def _state_of(s, out):
    """`out` with what the call changed in the cache."""
    if s["case"]["kind"] == "append" or s["case"]["append"]:
        out["k_pages"], out["v_pages"] = s["k_pages"], s["v_pages"]
    if s["case"]["track"]:
        out["weights"], out["positions"] = s["weights"], s["positions"]
    return out


def run(state):
    s = state
    if not own:
        return _plain(s)
    case, stream = s["case"], torch.cuda.current_stream().cuda_stream
    kind = case["kind"]
    if kind == "score":
        s["backend"].token_log_probs(s["logits"], s["tokens"], s["log_probs"], entropy=s["entropy"], lse=s["lse"], top_ids=s["top_ids"],
                                     top_log_probs=s["top_log_probs"], scale=case["scale"], stream=stream)
        return {name: s[name] for name in ("log_probs", "entropy", "lse", "top_ids", "top_log_probs")}
    if kind == "grad":
        s["backend"].token_log_probs_backward(s["logits"], s["tokens"], s["lse"], s["grad_logits"], grad_log_probs=s["grad_log_probs"],
                                              entropy=s["entropy"], grad_entropy=s["grad_entropy"], scale=case["scale"], stream=stream)
        return {"grad_logits": s["grad_logits"]}
    cache = s["cache"]
    if kind == "evict":
        cache.evict(s["k_pages"], s["v_pages"], s["page_table"], s["lengths"], s["tokens"], s["weights"], s["positions"], case["keep"],
                    recent=case["recent"], sinks=case["sinks"], lengths_out=s["lengths_out"], weights_out=s["weights_out"],
                    positions_out=s["positions_out"], stream=stream)
        return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "lengths": s["lengths_out"], "weights": s["weights_out"],
                "positions": s["positions_out"]}
    tracked = {name: s[name] for name in ("tokens", "weights", "positions")} if case["track"] else {}
    if kind == "append":
        cache.append(s["k_pages"], s["v_pages"], s["page_table"], s["lengths"], s["k_new"], s["v_new"], counts=s["counts"], stream=stream, **tracked)
        return _state_of(s, {})
    cache.attend(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["lengths"], s["out"], lse=s["lse"], k_new=s.get("k_new"),
                 v_new=s.get("v_new"), stream=stream, **tracked)
    return _state_of(s, {"out": s["out"], "lse": s["lse"]})


# ---- what a pass cannot do without ---------------------------------------------------------------------------------


def work(case):
    es, kind = ESIZE[case["dtype"]], case["kind"]
    if kind in ("score", "grad"):
        n = case["rows"] * case["vocab"]
        if kind == "score":
            return {"bytes": n * es + case["rows"] * (16 + 8 * case["top"]), "flops": 6 * n}
        return {"bytes": 2 * n * es + 12 * case["rows"], "flops": (8 if case["entropy"] else 4) * n}
    lengths, heads, dim = _lengths(case), case["kv_heads"], case["head_dim"]
    row = 2 * heads * dim * es  # a token's key and value
    table = 4 * sum(-(-n // case["page"]) for n in lengths) + 4 * case["batch"]
    if kind == "append":
        new = sum(_news(case, lengths))
        return {"bytes": 2 * row * new + 4 * sum(-(-n // case["page"]) for n in _news(case, lengths)) + (8 * heads * new if case["track"] else 0), "flops": 0}
    if kind == "attend":
        total = sum(lengths)
        size = row * total + table + 2 * case["batch"] * case["heads"] * dim * es + 4 * case["batch"] * case["heads"]
        size += 2 * case["batch"] * row if case["append"] else 0
        size += 8 * heads * total if case["track"] else 0
        return {"bytes": size, "flops": 4 * total * case["heads"] * dim}
    capacity = _max_pages(case) * case["page"]
    size = 16 * case["batch"]
    for n in lengths:
        size += heads * 8 * (n + capacity)
        over = max(0, n - case["keep"])
        if over:
            free = case["recent"] + case["sinks"]  # of the rows beyond `keep`, a share is kept that goes by weight or is protected
            moved = over * (free / n + (1 - free / n) * max(0, case["keep"] - free) / max(1, n - free))
            size += int(moved) * 2 * row
    return {"bytes": size, "flops": 0}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------


def _exact_score(s):
    case, tokens = s["case"], s["tokens"]
    outs = []
    for r0 in range(0, case["rows"], 512):
        x = s["logits"][r0:r0 + 512].double() * case["scale"]
        t = tokens[r0:r0 + 512]
        lse = torch.logsumexp(x, 1)
        log_p = x - lse[:, None]
        entropy = -torch.special.xlogy(torch.exp(log_p), torch.exp(log_p)).sum(1)
        log_prob = torch.where(t < 0, 0.0, log_p.gather(1, t.long().clamp(min=0)[:, None])[:, 0])
        outs.append((log_prob, entropy, lse, torch.sort(log_p, 1, descending=True).values[:, :case["top"]]))
    log_probs, entropy, lse, top = (torch.cat(c) for c in zip(*outs))
    return {"log_probs": log_probs, "entropy": entropy, "lse": lse, "top_ids": None, "top_log_probs": top}


def _exact_grad(s):
    """Row by row blocks: the derivative of sum(g log p[token]) + sum(h H) by the logits, with lse and H as given."""
    case = s["case"]
    out = torch.empty(s["logits"].shape, dtype=torch.float64, device="cuda")
    for r0 in range(0, case["rows"], 512):
        r = slice(r0, r0 + 512)
        log_p = case["scale"] * s["logits"][r].double() - s["lse"][r].double()[:, None]
        given = torch.zeros_like(log_p)
        t = s["tokens"][r].long()
        i = (t >= 0).nonzero()[:, 0]
        given[i, t[i]] = 1.0
        g = torch.where(t >= 0, s["grad_log_probs"][r].double(), 0.0)
        d = g[:, None] * (given - torch.exp(log_p))
        if case["entropy"]:
            d = d - s["grad_entropy"][r].double()[:, None] * torch.exp(log_p) * (log_p + s["entropy"][r].double()[:, None])
        out[r] = case["scale"] * d
    return {"grad_logits": out}


def _rows_of(s, b, n):
    """Page and row of the first n slots of sequence b."""
    t = torch.arange(n, device="cuda")
    return s["page_table"][b].long()[t // s["case"]["page"]], t % s["case"]["page"]


def _exact_cache(s):
    case = s["case"]
    k, v = s["k_pages"].double(), s["v_pages"].double()
    lengths = s["lengths"].tolist()
    got = {}
    if case.get("track") or case["kind"] == "evict":
        weights, positions, tokens = s["weights"].double(), s["positions"], s["tokens"].tolist()
    if case["kind"] == "append":
        for b, (n, c) in enumerate(zip(lengths, s["counts"].tolist())):
            page, row = (x[n - c:] for x in _rows_of(s, b, n))
            k[page, row], v[page, row] = s["k_new"][b, :c].double(), s["v_new"][b, :c].double()
            if case["track"]:
                weights[b, :, n - c:n] = 0.0
    elif case["kind"] == "attend":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        lse = torch.full(s["lse"].shape, -math.inf, dtype=torch.float64, device="cuda")
        rep = case["heads"] // case["kv_heads"]
        for b, n in enumerate(lengths):
            if n == 0:
                continue
            page, row = _rows_of(s, b, n)
            if case["append"]:
                k[page[-1], row[-1]], v[page[-1], row[-1]] = s["k_new"][b].double(), s["v_new"][b].double()
            keys = k[page, row].repeat_interleave(rep, 1)
            scores = (s["q"][b].double()[None] * keys).sum(-1) / math.sqrt(case["head_dim"])
            p = torch.softmax(scores, 0)
            out[b] = (p[:, :, None] * v[page, row].repeat_interleave(rep, 1)).sum(0)
            lse[b] = torch.logsumexp(scores, 0)
            if case["track"]:
                if case["append"]:
                    weights[b, :, n - 1] = 0.0
                weights[b, :, :n] += p.reshape(n, case["kv_heads"], rep).sum(2).T
        got = {"out": out, "lse": lse}
    else:
        weights_out = torch.zeros_like(weights)
        for b, n in enumerate(lengths):
            page, row = _rows_of(s, b, n)
            for g in range(case["kv_heads"]):
                w, p = weights[b, g, :n].cpu().tolist(), positions[b, g, :n].cpu().tolist()
                rank = sorted(range(n), key=lambda t: (not (p[t] < case["sinks"] or p[t] >= tokens[b] - case["recent"]), -w[t], t))
                kept = set(rank[:case["keep"]])
                left = min(n, case["keep"])
                place = list(range(left))
                moved = iter(t for t in range(left, n) if t in kept)
                place = [t if t in kept else next(moved) for t in place]
                at = torch.tensor(place, dtype=torch.long, device="cuda")
                k[page[:left], row[:left], g] = k[page[at], row[at], g]
                v[page[:left], row[:left], g] = v[page[at], row[at], g]
                weights_out[b, g, :left] = weights[b, g, at]
        return {"k_pages": k, "v_pages": v, "lengths": None, "weights": weights_out, "positions": None}
    if case["kind"] == "append" or case["append"]:
        got["k_pages"], got["v_pages"] = k, v
    if case["track"]:
        got["weights"], got["positions"] = weights, None
    return got


def exact(case, seed):
    global own
    was, own = own, False  # the inputs alone: nothing of the package
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["kind"] == "score":
        return _exact_score(s)
    if case["kind"] == "grad":
        return _exact_grad(s)
    return _exact_cache(s)


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(i)) for i in range(6)]:
        print(c, work(c))
