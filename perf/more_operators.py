"""The operators that bring prompts and drafted tokens to a paged key-value cache, as measurable cases and a way to draw more.

A cache is a pool of pages [pages, page, kv_heads, head_dim] for keys and one for values; row `t` of sequence `b` is row
`t % page` of page `page_table[b, t // page]`. A row's slot is its page times the page size plus the row in it. Packed arrays hold
the tokens of all sequences one behind the other, those of sequence `b` from `starts[b]` to `starts[b + 1]`; rows behind the last
sequence belong to no one and stay as they were.

  prompt  causal attention of whole prompts, packed, each over its own tokens
  tree    attention of a tree of drafted tokens per sequence: every node sees the cached rows, its ancestors and itself
  assign  pages for the rows that sequences are to have, taken from a stack of free ones and given back to it, and the slots of
          the packed new tokens. Sequences are served in order; one that does not fit, and those behind it that want more, get none
  path    slots for the nodes on the path to an accepted leaf, as the next rows of each sequence; -1 for the others
  store   rows of packed keys and values into the slots of the cache, those of negative slots into none
"""
import math
import random

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODE = {"f32": 2, "f16": 7, "bf16": 8}  # element-type codes of the C ABI
ESIZE = {"f32": 4, "f16": 2, "bf16": 2}
MOST_BYTES = 280e6      # of keys and values, or of a packed batch, that a case may have
MOST_PRODUCTS = 5.5e11  # of queries and keys, masked ones among them; an eighth of it in f32
MOST_PAGES = 1 << 19


def _prompt(name, dtype, batch, heads, kv_heads, head_dim, longest, scale=None):
    return {"name": name, "kind": "prompt", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "longest": longest, "scale": scale or 0.0}


def _tree(name, dtype, batch, heads, kv_heads, head_dim, page, longest, nodes, chain=False):
    return {"name": name, "kind": "tree", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "longest": longest, "nodes": nodes, "chain": chain}


def _assign(name, batch, page, longest, turnover, short=False):
    return {"name": name, "kind": "assign", "batch": batch, "page": page, "longest": longest, "turnover": turnover, "short": short}


def _path(name, batch, page, longest, nodes):
    return {"name": name, "kind": "path", "batch": batch, "page": page, "longest": longest, "nodes": nodes}


def _store(name, dtype, batch, kv_heads, head_dim, page, longest, kept=1.0):
    return {"name": name, "kind": "store", "dtype": dtype, "batch": batch, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
            "longest": longest, "kept": kept}


def listed():
    return [
        # a single chat's prompt of an odd length, one layer of an 8B-shaped decoder: latency
        _prompt("prompt_b1_517", "bf16", 1, 32, 8, 128, 517),
        # two long documents on the same decoder
        _prompt("prompt_b2_8192", "f16", 2, 32, 8, 128, 8192),
        # many short questions at once on a small decoder in f32, one slot of the batch idle
        _prompt("prompt_b48_f32_200", "f32", 48, 4, 2, 64, 200),
        # a single chat, eight drafted tokens to verify: latency
        _tree("tree_b1_517_n8", "bf16", 1, 32, 8, 128, 16, 517, 8),
        # batched serving with drafts of sixteen tokens, ragged lengths, one slot idle
        _tree("tree_b16_4096_n16", "bf16", 16, 32, 8, 128, 16, 4096, 16),
        # a long document on 70B-shaped heads, a further piece of 64 tokens of its prompt behind the cached ones, large pages
        _tree("tree_b1_65536_n64", "f16", 1, 64, 8, 128, 64, 65536, 64, chain=True),
        # a decode step: a row more for every sequence, a page for those that have filled theirs
        _assign("assign_b32_step", 32, 16, 2048, 0.0),
        # a third of a large batch has ended, prompts come in their places, with slots for their tokens
        _assign("assign_b512_prompts", 512, 16, 4096, 0.33),
        # the tokens that a verification step has accepted
        _path("path_b1_n8", 1, 16, 517, 8),
        # the same for a large batch of large trees
        _path("path_b256_n64", 256, 16, 4096, 64),
        # rows of four packed prompts going into the cache
        _store("store_b4_2048", "bf16", 4, 8, 128, 16, 2048),
        # accepted tokens: a fifth of the drafted rows has a slot
        _store("store_b64_n16_some", "bf16", 64, 8, 128, 16, 16, kept=0.2),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(32, 8, 128), (32, 8, 128), (64, 8, 128), (8, 1, 128), (16, 8, 128), (8, 8, 64), (4, 2, 64), (12, 4, 96), (6, 3, 256)]


def draw(rng):
    kind = rng.choice(["prompt"] * 4 + ["tree"] * 4 + ["assign"] * 2 + ["path"] + ["store"] * 2)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    heads, kv_heads, head_dim = rng.choice(HEADS)
    page = rng.choice([8, 16, 16, 20, 32, 64, 128])
    if kind == "prompt":
        batch = _log_int(rng, 1, 256)
        products = MOST_PRODUCTS / (8 if dtype == "f32" else 1)
        longest = min(_log_int(rng, 1, 8192), int(math.sqrt(products / (batch * heads * head_dim))),
                      int(MOST_BYTES / (batch * 2 * (heads + kv_heads) * head_dim * ESIZE[dtype])))
        case = _prompt("", dtype, batch, heads, kv_heads, head_dim, longest, rng.choice([None, None, round(rng.uniform(0.05, 0.2), 4)]))
    elif kind == "tree":
        batch, nodes = _log_int(rng, 1, 64), _log_int(rng, 1, 64)
        products = MOST_PRODUCTS / (128 if dtype == "f32" else 16)
        longest = min(_log_int(rng, 1, 65536), int(MOST_BYTES / (batch * 2 * kv_heads * head_dim * ESIZE[dtype])),
                      max(16, int(products / (batch * heads * nodes * head_dim))))
        case = _tree("", dtype, batch, heads, kv_heads, head_dim, page, longest, nodes, rng.random() < 0.3)
    elif kind == "assign":
        batch = _log_int(rng, 1, 1024)
        longest = min(_log_int(rng, 1, 32768), MOST_PAGES * page // batch)
        case = _assign("", batch, page, longest, rng.choice([0.0, 0.1, 0.5, 1.0]), rng.random() < 0.25)
    elif kind == "path":
        case = _path("", _log_int(rng, 1, 1024), page, _log_int(rng, 1, 8192), _log_int(rng, 1, 64))
    else:
        batch = _log_int(rng, 1, 64)
        longest = min(_log_int(rng, 1, 8192), int(MOST_BYTES / 2 / (batch * 2 * kv_heads * head_dim * ESIZE[dtype])))
        case = _store("", dtype, batch, kv_heads, head_dim, page, longest, rng.choice([1.0, 1.0, round(rng.uniform(0.1, 0.9), 2)]))
    case.pop("name")
    return case


# ---- inputs --------------------------------------------------------------------------------------------------------


def _randn(gen, dtype, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)


def _rand(gen, *shape):
    return torch.rand(shape, generator=gen, device="cuda")


def _ints(x):
    return torch.as_tensor(x, device="cuda").to(torch.int32).contiguous()


def _lengths(case):
    """Lengths of the batch: from `longest` down to a third of it; of eight sequences and more the last slot is idle."""
    n, longest = case["batch"], case["longest"]
    out = [max(1, longest - (longest * 2 * i) // (3 * n)) for i in range(n)]
    if n >= 8:
        out[-1] = 0
    return out


def _mixed(case, gen):
    lengths = _ints(_lengths(case))
    return lengths[torch.randperm(case["batch"], generator=gen, device="cuda")]


def _starts(lengths):
    return _ints(torch.cat([torch.zeros_like(lengths[:1]), torch.cumsum(lengths, 0)]))


def _padded(total):
    """Rows of a packed array: a program that replays a graph has them in steps."""
    return -(-(total + 1) // 32) * 32


def _table(counts, page_count, max_pages, gen):
    """A page table with counts[b] pages for each sequence in a random order, -1 behind them, and the pages that are left over."""
    order = torch.randperm(page_count, generator=gen, device="cuda").int()
    column = torch.arange(max_pages, device="cuda")
    counts = counts.long()
    first = torch.cumsum(counts, 0) - counts
    table = torch.where(column < counts[:, None], order[(first[:, None] + column).clamp(max=page_count - 1)], -1)
    return table.int().contiguous(), order


def _pages(rows, page):
    return (rows + page - 1) // page


def _pools(case, pages, gen):
    shape = (pages, case["page"], case["kv_heads"], case["head_dim"])
    return {"k_pages": _randn(gen, TORCH[case["dtype"]], *shape), "v_pages": _randn(gen, TORCH[case["dtype"]], *shape)}


def _parents(case, gen):
    """Each node's parent among those before it, -1 for a root; a chain is what a further piece of a prompt is."""
    i = torch.arange(case["nodes"], device="cuda").expand(case["batch"], -1)
    if case.get("chain"):
        return _ints(i - 1)
    return _ints((_rand(gen, case["batch"], case["nodes"]) * (i + 1)).long().clamp(max=i) - 1)


def _backend():
    import pjrtx_b200

    return pjrtx_b200.Backend()


def _paged_cache(case):
    """The handle that a program keeps for all layers of this shape."""
    heads = case.get("heads", case.get("kv_heads", 1))
    return _backend().paged_cache(CODE[case.get("dtype", "bf16")], case["batch"], heads, case.get("kv_heads", 1), case.get("head_dim", 128),
                                  case["page"], _max_pages(case), tree=case.get("nodes", 0))


def _max_pages(case):
    return -(-(case["longest"] + case.get("nodes", 0) + 1) // case["page"])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case, **{"prompt": _prepare_prompt, "tree": _prepare_tree, "assign": _prepare_assign, "path": _prepare_path,
                          "store": _prepare_store}[case["kind"]](case, gen)}
    if own:
        if case["kind"] == "prompt":
            s["backend"] = _backend()
        else:
            s["cache"] = _paged_cache(case)
    return s


def _prepare_prompt(case, gen):
    dtype, heads, kv_heads, dim = TORCH[case["dtype"]], case["heads"], case["kv_heads"], case["head_dim"]
    starts, tokens = _starts(_mixed(case, gen)), _padded(sum(_lengths(case)))
    packed = _randn(gen, dtype, tokens, heads + 2 * kv_heads, dim)  # as one projection writes them
    packed[:, :heads] *= 2
    return {"q": packed[:, :heads], "k": packed[:, heads:heads + kv_heads], "v": packed[:, heads + kv_heads:], "starts": starts,
            "out": torch.zeros((tokens, heads, dim), dtype=dtype, device="cuda"), "lse": torch.zeros((tokens, heads), device="cuda")}


def _prepare_tree(case, gen):
    dtype, batch, nodes, heads, kv_heads, dim = TORCH[case["dtype"]], case["batch"], case["nodes"], case["heads"], case["kv_heads"], case["head_dim"]
    lengths, page = _mixed(case, gen), case["page"]
    pages = sum(-(-n // page) for n in _lengths(case)) + 3
    table, _ = _table(_pages(lengths, page), pages, _max_pages(case), gen)
    counts = (_rand(gen, batch) * nodes * 0.5).long() + (nodes + 1) // 2  # the upper half of what there is room for
    counts = torch.where(lengths > 0, counts.clamp(max=nodes), 0)
    packed = _randn(gen, dtype, batch, nodes, heads + 2 * kv_heads, dim)
    packed[:, :, :heads] *= 2
    return {**_pools(case, pages, gen), "page_table": table, "lengths": lengths, "q": packed[:, :, :heads],
            "k_new": packed[:, :, heads:heads + kv_heads], "v_new": packed[:, :, heads + kv_heads:], "parents": _parents(case, gen),
            "counts": _ints(counts), "out": torch.zeros((batch, nodes, heads, dim), dtype=dtype, device="cuda"),
            "lse": torch.zeros((batch, nodes, heads), device="cuda")}


def _turn(case):
    """Rows before, rows after and new tokens of every slot of the batch: some end, some of their places are taken by prompts, the
    rest grows by a row."""
    before, every = _lengths(case), max(1, round(1 / case["turnover"])) if case["turnover"] else 0
    after, new = [], []
    for i, n in enumerate(before):
        if every and i % every == 0:
            m = 0 if i % (3 * every) == 0 else max(1, case["longest"] - n // 2)
            after.append(m)
            new.append(m)
        else:
            after.append(n + 1 if n else 0)
            new.append(1 if n else 0)
    return before, after, new


def _prepare_assign(case, gen):
    batch, page = case["batch"], case["page"]
    before, after, new = _turn(case)
    order = torch.randperm(batch, generator=gen, device="cuda")
    before_t, lengths, new_t = (_ints(x)[order] for x in (before, after, new))
    held = _pages(before_t, page)
    used = sum(-(-n // page) for n in before)
    grown = sum(max(0, -(-m // page) - -(-n // page)) for n, m in zip(before, after))
    pages = used + (grown // 2 if case["short"] else grown) + 3
    table, order = _table(held, pages, _max_pages(case), gen)
    free = torch.cat([order[used:], torch.full((used,), -1, dtype=torch.int32, device="cuda")])
    s = {"lengths": lengths.contiguous(), "held": _ints(held), "page_table": table, "free_pages": free.contiguous(),
         "free_count": _ints([pages - used]), "starts": _starts(new_t), "slots": torch.zeros(_padded(sum(new)), dtype=torch.int32, device="cuda")}
    for name in ("held", "page_table", "free_pages", "free_count"):  # written apart: the step before may still be reading them
        s[name + "_out"] = torch.empty_like(s[name])
    return s


def _prepare_path(case, gen):
    batch, page, nodes = case["batch"], case["page"], case["nodes"]
    lengths = _mixed(case, gen)
    counts = _pages(lengths + nodes, page)
    table, _ = _table(counts, sum(-(-(n + nodes) // page) for n in _lengths(case)) + 3, _max_pages(case), gen)
    leaves = (_rand(gen, batch) * (nodes + 1)).long().clamp(max=nodes) - 1  # -1: nothing accepted
    return {"page_table": table, "lengths": lengths, "parents": _parents(case, gen), "leaves": _ints(torch.where(lengths > 0, leaves, -1)),
            "slots": torch.zeros((batch, nodes), dtype=torch.int32, device="cuda"), "lengths_out": torch.zeros_like(lengths)}


def _prepare_store(case, gen):
    dtype, page, kv_heads, dim = TORCH[case["dtype"]], case["page"], case["kv_heads"], case["head_dim"]
    lengths = _mixed(case, gen)
    pages = sum(-(-n // page) for n in _lengths(case)) + 3
    table, _ = _table(_pages(lengths, page), pages, _max_pages(case), gen)
    tokens = _padded(sum(_lengths(case)))
    token = torch.arange(tokens, device="cuda")
    starts = _starts(lengths).long()
    b = (torch.searchsorted(starts, token, right=True) - 1).clamp(max=case["batch"] - 1)
    row = token - starts[b]
    slots = table[b, (row // page).clamp(max=table.shape[1] - 1)] * page + row % page
    there = (token < starts[-1]) & (_rand(gen, tokens) < case["kept"])
    packed = _randn(gen, dtype, tokens, 2 * kv_heads, dim)
    return {**_pools(case, pages, gen), "k_new": packed[:, :kv_heads], "v_new": packed[:, kv_heads:], "slots": _ints(torch.where(there, slots, -1))}


# ---- the plain forms -----------------------------------------------------------------------------------------------


def _softmax_(scores, seen):
    """Scores [..., rows, keys] to probabilities, in place, and their log-sum-exp; rows that see nothing give zeros and -inf."""
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_(min=-3e38)
    total = scores.sub_(top).exp_().sum(-1, keepdim=True)
    scores.div_(torch.where(total > 0, total, 1.0))
    return torch.where(total > 0, top + torch.log(total), -math.inf)[..., 0]


def _plain_prompt(s):
    case = s["case"]
    batch, heads, kv_heads, dim, longest = (case[n] for n in ("batch", "heads", "kv_heads", "head_dim", "longest"))
    rep, starts, tokens = heads // kv_heads, s["starts"].long(), s["q"].shape[0]
    row = torch.arange(longest, device="cuda")
    at = (starts[:-1, None] + row).clamp(max=tokens - 1)
    there = row < (starts[1:] - starts[:-1])[:, None]
    q = s["q"].float()[at].reshape(batch, longest, kv_heads, rep, dim).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, rep * longest, dim)
    k = s["k"].float()[at].permute(0, 2, 3, 1)
    scores = torch.matmul(q, k).mul_(case["scale"] or 1.0 / math.sqrt(dim)).view(batch, kv_heads, rep, longest, longest)
    lse = _softmax_(scores, (row[:, None] >= row) & there[:, None, None, None])
    v = s["v"].float()[at].permute(0, 2, 1, 3)
    out = torch.matmul(scores.view(batch, kv_heads, rep * longest, longest), v).view(batch, kv_heads, rep, longest, dim)
    b, t = there.nonzero(as_tuple=True)
    to = at[b, t]
    s["out"][to] = out.permute(0, 3, 1, 2, 4).reshape(batch, longest, heads, dim)[b, t].to(s["out"].dtype)
    s["lse"][to] = lse.permute(0, 3, 1, 2).reshape(batch, longest, heads)[b, t]
    return {"out": s["out"], "lse": s["lse"]}


def _ancestors(parents):
    """[batch, nodes, nodes]: whether column j is node i or above it, by doubling the steps."""
    nodes = parents.shape[1]
    step = torch.eye(nodes, device="cuda") + (parents[:, :, None] == torch.arange(nodes, device="cuda")).float()
    for _ in range((nodes - 1).bit_length()):
        step = (torch.matmul(step, step) > 0).float()
    return step > 0


def _plain_tree(s):
    case = s["case"]
    batch, heads, kv_heads, dim, nodes, page = (case[n] for n in ("batch", "heads", "kv_heads", "head_dim", "nodes", "page"))
    rep, lengths, counts = heads // kv_heads, s["lengths"].long(), s["counts"].long()
    table = s["page_table"].long().clamp(min=0)
    slot = torch.arange(table.shape[1] * page, device="cuda")
    node = torch.arange(nodes, device="cuda")
    seen = torch.cat([(slot < lengths[:, None])[:, None].expand(-1, nodes, -1), _ancestors(s["parents"])], 2)
    k = torch.cat([s["k_pages"][table].reshape(batch, -1, kv_heads, dim), s["k_new"]], 1).permute(0, 2, 3, 1).float()
    q = s["q"].float().reshape(batch, nodes, kv_heads, rep, dim).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, rep * nodes, dim)
    scores = torch.matmul(q, k).mul_(1.0 / math.sqrt(dim)).view(batch, kv_heads, rep, nodes, -1)
    del k
    lse = _softmax_(scores, seen[:, None, None])
    v = torch.cat([s["v_pages"][table].reshape(batch, -1, kv_heads, dim), s["v_new"]], 1).permute(0, 2, 1, 3).float()
    out = torch.matmul(scores.view(batch, kv_heads, rep * nodes, -1), v).view(batch, kv_heads, rep, nodes, dim)
    there = node < counts[:, None]
    out, lse = out.permute(0, 3, 1, 2, 4).reshape(s["out"].shape).to(s["out"].dtype), lse.permute(0, 3, 1, 2).reshape(s["lse"].shape)
    s["out"].copy_(torch.where(there[..., None, None], out, s["out"]))
    s["lse"].copy_(torch.where(there[..., None], lse, s["lse"]))
    return {"out": s["out"], "lse": s["lse"]}


def _slots_of(table, page, b, row):
    return table[b, (row // page).clamp(0, table.shape[1] - 1)] * page + row % page


def _plain_assign(s):
    page, batch = s["case"]["page"], s["case"]["batch"]
    held, lengths, table = s["held"].long(), s["lengths"].long(), s["page_table"].long().clone()
    free, free_count = s["free_pages"].long().clone(), s["free_count"].long()
    need = _pages(lengths, page)
    give, take = (held - need).clamp(min=0), (need - held).clamp(min=0)
    column = torch.arange(table.shape[1], device="cuda")
    b, c = ((column >= need[:, None]) & (column < held[:, None])).nonzero(as_tuple=True)
    free[free_count + torch.arange(b.numel(), device="cuda")] = table[b, c]
    table[b, c] = -1
    there = free_count + give.sum()
    want = torch.cumsum(take, 0)
    served = want <= there
    take = torch.where(served, take, 0)
    held_out = torch.where(served, need, torch.minimum(held, need))
    b, c = ((column >= held[:, None]) & (column < held_out[:, None])).nonzero(as_tuple=True)
    place = (there - 1 - torch.arange(b.numel(), device="cuda")).clamp(min=0)
    table[b, c] = free[place]
    free[place] = -1
    token = torch.arange(s["slots"].numel(), device="cuda")
    starts = s["starts"].long()
    b = (torch.searchsorted(starts, token, right=True) - 1).clamp(max=batch - 1)
    row = lengths[b] - (starts[b + 1] - token)
    slots = torch.where((token < starts[-1]) & (held_out[b] >= need[b]), _slots_of(table, page, b, row), -1)
    return {"held": held_out.int(), "page_table": table.int(), "free_pages": free.int(), "free_count": (there - take.sum()).int(), "slots": slots.int()}


def _plain_path(s):
    batch, nodes, page = s["case"]["batch"], s["case"]["nodes"], s["case"]["page"]
    leaves, lengths, table = s["leaves"].long(), s["lengths"].long(), s["page_table"].long()
    b = torch.arange(batch, device="cuda")
    on = _ancestors(s["parents"])[b, leaves.clamp(min=0)] & (leaves >= 0)[:, None]
    row = lengths[:, None] + torch.cumsum(on, 1) - 1
    return {"slots": torch.where(on, _slots_of(table, page, b[:, None], row), -1).int(), "lengths": (lengths + on.sum(1)).int()}


def _plain_store(s):
    page, slots = s["case"]["page"], s["slots"].long()
    t = (slots >= 0).nonzero()[:, 0]
    to = slots[t] // page, slots[t] % page
    s["k_pages"][to] = s["k_new"][t]
    s["v_pages"][to] = s["v_new"][t]
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


# ---- one pass ------------------------------------------------------------------------------------------------------


def run(state):
    s = state
    case = s["case"]
    kind = case["kind"]
    if not own:
        return {"prompt": _plain_prompt, "tree": _plain_tree, "assign": _plain_assign, "path": _plain_path, "store": _plain_store}[kind](s)
    stream = torch.cuda.current_stream().cuda_stream
    if kind == "prompt":
        s["backend"].prompt_attention(s["q"], s["k"], s["v"], s["starts"], s["out"], lse=s["lse"], scale=case["scale"] or None, stream=stream)
        return {"out": s["out"], "lse": s["lse"]}
    cache = s["cache"]
    if kind == "tree":
        cache.attend_tree(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["lengths"], s["out"], s["k_new"], s["v_new"], s["parents"],
                          counts=s["counts"], lse=s["lse"], stream=stream)
        return {"out": s["out"], "lse": s["lse"]}
    if kind == "assign":
        cache.assign_pages(s["lengths"], s["held"], s["page_table"], s["free_pages"], s["free_count"], starts=s["starts"], slots=s["slots"],
                           held_out=s["held_out"], page_table_out=s["page_table_out"], free_pages_out=s["free_pages_out"],
                           free_count_out=s["free_count_out"], stream=stream)
        return {"held": s["held_out"], "page_table": s["page_table_out"], "free_pages": s["free_pages_out"], "free_count": s["free_count_out"],
                "slots": s["slots"]}
    if kind == "path":
        cache.path_slots(s["page_table"], s["lengths"], s["parents"], s["leaves"], s["slots"], lengths_out=s["lengths_out"], stream=stream)
        return {"slots": s["slots"], "lengths": s["lengths_out"]}
    cache.store(s["k_pages"], s["v_pages"], s["k_new"], s["v_new"], s["slots"], stream=stream)
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


# ---- what a pass cannot do without ---------------------------------------------------------------------------------


def work(case):
    kind, batch = case["kind"], case["batch"]
    if kind == "assign":
        before, after, new = _turn(case)
        page = case["page"]
        changed = sum(abs(-(-m // page) - -(-n // page)) for n, m in zip(before, after))
        pages = sum(-(-n // page) for n in before) + 3
        # the table and the stack go to other arrays: each entry read and written
        return {"bytes": 8 * batch * _max_pages(case) + 8 * (pages + changed) + 16 * batch + 4 * sum(new), "flops": 0}
    if kind == "path":
        return {"bytes": 8 * batch * case["nodes"] + 4 * (case["nodes"] // case["page"] + 1) * batch + 12 * batch, "flops": 0}
    es, kv_heads, dim, lengths = ESIZE[case["dtype"]], case["kv_heads"], case["head_dim"], _lengths(case)
    row = 2 * kv_heads * dim * es  # a token's key and value
    if kind == "store":
        kept = int(sum(lengths) * case["kept"])
        return {"bytes": 2 * row * kept + 4 * _padded(sum(lengths)), "flops": 0}
    heads, query = case["heads"], 2 * case["heads"] * dim * es + 4 * case["heads"]  # q in, out and lse out
    if kind == "prompt":
        return {"bytes": sum(lengths) * (row + query) + 4 * batch, "flops": 2 * dim * heads * sum(n * (n + 1) for n in lengths)}
    nodes = sum(-(-case["nodes"] * 3 // 4) for n in lengths if n)  # on average
    table = 4 * sum(-(-n // case["page"]) for n in lengths)
    return {"bytes": row * sum(lengths) + table + nodes * (row + query + 4) + 8 * batch,
            "flops": 4 * dim * heads * sum(n * (case["nodes"] * 3 / 4) for n in lengths)}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------


def _exact_rows(q, k, v, scale, seen):
    """q [n, rep, d], k and v [m, d] of one KV head, seen [n, m] or None: attention and log-sum-exp in 64 bits."""
    scores = torch.einsum("nrd,md->nrm", q.double(), k.double()) * scale
    if seen is not None:
        scores = torch.where(seen[:, None], scores, -math.inf)
    return torch.einsum("nrm,md->nrd", torch.softmax(scores, -1), v.double()), torch.logsumexp(scores, -1)


def _exact_prompt(s):
    case = s["case"]
    rep, scale = case["heads"] // case["kv_heads"], case["scale"] or case["head_dim"] ** -0.5
    out, lse, starts = s["out"].double(), s["lse"].double(), s["starts"].tolist()
    for a, z in zip(starts, starts[1:]):
        for r0 in range(a, z, 2048):  # some query rows at a time
            r1 = min(z, r0 + 2048)
            seen = torch.arange(r0, r1, device="cuda")[:, None] >= torch.arange(a, r1, device="cuda")
            for g in range(case["kv_heads"]):
                h = slice(g * rep, (g + 1) * rep)
                out[r0:r1, h], lse[r0:r1, h] = _exact_rows(s["q"][r0:r1, h], s["k"][a:r1, g], s["v"][a:r1, g], scale, seen)
    return {"out": out, "lse": lse}


def _exact_tree(s):
    case = s["case"]
    rep, page = case["heads"] // case["kv_heads"], case["page"]
    out, lse = s["out"].double(), s["lse"].double()
    parents = s["parents"].tolist()
    for b, (n, c) in enumerate(zip(s["lengths"].tolist(), s["counts"].tolist())):
        if c == 0:
            continue
        above = []
        for i in range(c):
            above.append([j == i or (parents[b][i] >= 0 and above[parents[b][i]][j]) for j in range(c)])
        seen = torch.cat([torch.ones((c, n), dtype=torch.bool), torch.tensor(above)], 1).cuda()
        t = torch.arange(n, device="cuda")
        at = s["page_table"][b].long()[t // page], t % page
        for g in range(case["kv_heads"]):
            k, v = (torch.cat([s[x + "_pages"][at[0], at[1], g], s[x + "_new"][b, :c, g]]) for x in "kv")
            h = slice(g * rep, (g + 1) * rep)
            out[b, :c, h], lse[b, :c, h] = _exact_rows(s["q"][b, :c, h], k, v, case["head_dim"] ** -0.5, seen)
    return {"out": out, "lse": lse}


def _exact_store(s):
    got = {}
    for x in "kv":
        pool = s[x + "_pages"].double()
        rows = pool.view(-1, *pool.shape[2:])
        for r0 in range(0, s["slots"].numel(), 1 << 14):
            slots = s["slots"][r0:r0 + (1 << 14)].long()
            rows.index_copy_(0, slots[slots >= 0], s[x + "_new"][r0:r0 + (1 << 14)][slots >= 0].double())
        got[x + "_pages"] = pool
    return got


def exact(case, seed):
    global own
    if case["kind"] in ("assign", "path"):  # whole numbers
        return None
    was, own = own, False  # the inputs alone: nothing of the package
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"prompt": _exact_prompt, "tree": _exact_tree, "store": _exact_store}[case["kind"]](s)


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(i)) for i in range(6)]:
        print(c, work(c))
