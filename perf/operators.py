"""Differential attention and the pages of a key-value cache: the workloads whose speed matters, with plain forms.

Differential attention takes q (.., heads, d) and k, v (.., heads_k, d); the halves of d of q and k give two softmax maps
over the same values, and the output is (A_1 - lam_h A_2) V with a learned weight per head.  ``train`` cases are dense training
steps, ``varlen`` ones packed training steps, ``serve`` ones a step against a key-value cache: one token or a chunk of a prompt.
The page cases keep the tables of a paged cache: ``copy`` pages, a serving ``round`` (reserve pages for the next tokens, fork
sequences, free the finished ones) and ``compact``.  All data are fp16, the type of the framework's attention.
"""
import math
import random

import torch

own = False


def _train(name, batch, seqlen_q, seqlen_k, heads, heads_k, head_dim, causal):
    return dict(name=name, kind="train", batch=batch, seqlen_q=seqlen_q, seqlen_k=seqlen_k, heads=heads, heads_k=heads_k,
                head_dim=head_dim, causal=causal)


def _varlen(name, batch, shortest, longest, lengths_seed, heads, heads_k, head_dim, causal):
    return dict(name=name, kind="varlen", batch=batch, shortest=shortest, longest=longest, lengths_seed=lengths_seed, heads=heads,
                heads_k=heads_k, head_dim=head_dim, causal=causal)


def _serve(name, batch, new_tokens, shortest, longest, lengths_seed, page, heads, heads_k, head_dim):
    return dict(name=name, kind="serve", batch=batch, new_tokens=new_tokens, shortest=shortest, longest=longest,
                lengths_seed=lengths_seed, page=page, heads=heads, heads_k=heads_k, head_dim=head_dim)


def _copy(name, layers, pages, page, heads_k, head_dim, pairs):
    return dict(name=name, kind="copy", layers=layers, pages=pages, page=page, heads_k=heads_k, head_dim=head_dim, pairs=pairs)


def _tables(kind, name, layers, pages, page, heads_k, head_dim, rows, lengths_seed):
    return dict(name=name, kind=kind, layers=layers, pages=pages, page=page, heads_k=heads_k, head_dim=head_dim, rows=rows,
                lengths_seed=lengths_seed)


def listed():
    return [
        # A training step of a small bidirectional encoder, odd length: launches and the host are most of it.
        _train("train_small_odd", 3, 197, 197, 6, 6, 64, False),
        # Pre-training at a long context, grouped heads.
        _train("train_8k_gqa", 1, 8192, 8192, 16, 4, 128, True),
        # Fine-tuning on texts of very different lengths, packed end to end.
        _varlen("train_texts", 14, 131, 1000, 1, 16, 8, 64, True),
        # One user's next token: a contiguous cache that is partly filled.
        _serve("decode_one", 1, 1, 1500, 1500, 3, 0, 16, 4, 128),
        # The next token of a serving batch: paged cache, lengths far apart.
        _serve("decode_batch_paged", 32, 1, 512, 8192, 4, 256, 16, 4, 128),
        # A chunk of four prompts on top of what the cache already holds.
        _serve("chunk_paged", 4, 256, 500, 4000, 5, 256, 16, 8, 128),
        # A few pages of a small model's cache.
        _copy("copy_few", 2, 40, 256, 2, 64, 3),
        # Pages of every layer of a larger model.
        _copy("copy_layers", 16, 64, 256, 8, 128, 24),
        # One step of a small beam search.
        _tables("round", "round_beams", 2, 64, 256, 2, 64, 8, 4),
        # One step of a full serving batch with parallel samples of its prompts.
        _tables("round", "round_batch", 8, 512, 256, 4, 128, 192, 7),
        # The pool of a small model after requests have come and gone.
        _tables("compact", "compact_small", 4, 96, 256, 2, 64, 12, 8),
        # The pool of a larger model, odd number of rows.
        _tables("compact", "compact_layers", 16, 127, 512, 4, 128, 33, 9),
    ]


MOST_PAIRS = 1 << 30  # (head, query, key): the plain form holds them all
MOST_POOL = 1.2e9     # bytes of a pool
MOST_GATHERED = 3e8   # cached elements of the sequences of a batch


def _log_between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    while True:
        kind = rng.choice(("train", "train", "varlen", "serve", "serve", "serve", "copy", "round", "compact"))
        d = rng.choice((64, 128))
        heads_k = rng.choice((1, 2, 4, 6, 8))
        heads = heads_k * rng.choice((1, 2, 4))
        if kind == "train":
            seqlen_q = _log_between(rng, 130, 8192)
            cross = rng.random() < 0.25
            seqlen_k = _log_between(rng, 130, 8192) if cross else seqlen_q
            case = _train("", _log_between(rng, 1, 8), seqlen_q, seqlen_k, heads, heads_k, d, not cross and rng.random() < 0.6)
        elif kind == "varlen":
            longest = _log_between(rng, 200, 4096)
            case = _varlen("", _log_between(rng, 2, 32), int(rng.uniform(130, longest)), longest, rng.randrange(1 << 30), heads, heads_k, d,
                           rng.random() < 0.6)
        elif kind == "serve":
            longest = _log_between(rng, 32, 16384)
            case = _serve("", _log_between(rng, 1, 64), rng.choice((1, 1, 1, 2, 3, _log_between(rng, 16, 512))),
                          max(1, int(longest * rng.uniform(0.05, 1.0))), longest, rng.randrange(1 << 30), rng.choice((0, 256, 512)), heads,
                          heads_k, d)
        elif kind == "copy":
            pages = _log_between(rng, 16, 1024)
            case = _copy("", _log_between(rng, 1, 32), pages, rng.choice((256, 512)), heads_k, d, rng.randint(1, pages // 2))
        else:
            case = _tables(kind, "", _log_between(rng, 1, 32), _log_between(rng, 32, 2048), rng.choice((256, 512)), heads_k, d,
                           _log_between(rng, 4, 256), rng.randrange(1 << 30))
        del case["name"]
        if _fits(case):
            return case


def _fits(case):
    kind, d = case["kind"], case["head_dim"]
    if kind == "train":
        return case["batch"] * case["heads"] * case["seqlen_q"] * case["seqlen_k"] <= MOST_PAIRS and work(case)["flops"] <= 1e12
    if kind == "varlen":
        return case["heads"] * sum(_lengths(case)) ** 2 <= MOST_PAIRS and work(case)["flops"] <= 1e12
    if kind == "serve":
        cached = case["batch"] * _capacity(case)
        return cached * case["heads_k"] * d <= MOST_GATHERED and cached * case["heads"] * case["new_tokens"] <= MOST_PAIRS
    pool = 2 * case["layers"] * case["pages"] * case["page"] * case["heads_k"] * d * 2
    return 1e6 <= pool <= MOST_POOL and (kind == "copy" or case["rows"] <= case["pages"] // 2)


def _lengths(case):
    rng = random.Random(case["lengths_seed"])
    return [rng.randint(case["shortest"], case["longest"]) for _ in range(case["batch"])]


def _capacity(case):
    step = case["page"] or 64
    return -(-(case["longest"] + case["new_tokens"]) // step) * step


def _normal(generator, *shape):
    return torch.randn(*shape, generator=generator, device="cuda", dtype=torch.float16)


def _values(generator, *shape):
    """Values and output gradients have channels whose mean is not zero."""
    return _normal(generator, *shape) + 0.5 * _normal(generator, *shape[-2:])


def _weights(generator, heads):
    return (0.2 + 0.6 * torch.rand(heads, generator=generator, device="cuda")).half()


def _page_plan(case):
    """The sequences of a paged pool whose requests came and went, from the case alone: lengths of the rows (0: empty) and the pages
    of each, spread over the pool; and what the next step does with them: new tokens, forks, finished rows."""
    rng = random.Random(case["lengths_seed"])
    rows, page, pages = case["rows"], case["page"], case["pages"]
    columns = max(4, 2 * pages // rows)
    live = max(1, (2 * rows) // 3)  # the rows behind them are empty
    order = rng.sample(range(pages), pages)
    budget = max(live, (3 * pages) // 5)
    lengths, table = [0] * rows, [[-1] * columns for _ in range(rows)]
    for r in range(live):
        most = min(columns - 1, max(1, budget - (live - 1 - r)))
        n = min(most, rng.randint(1, max(1, 2 * budget // (live - r))))
        lengths[r] = n * page - (rng.randrange(page) if rng.random() < 0.8 else 0)
        table[r][:n] = [order.pop() for _ in range(n)]
        budget -= n
    new = [rng.choice((0, 1, 1, 1, 8, page)) for _ in range(rows)]
    children = list(range(live, rows))[: max(1, rows // 4)]
    parents = [rng.randrange(live) for _ in children]
    finished = rng.sample(range(live), max(1, live // 5))
    return lengths, table, new, parents, children, finished


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, d, h_k = case["kind"], case["head_dim"], case["heads_k"]
    state = {"case": case}
    if kind in ("train", "varlen"):
        h = case["heads"]
        if kind == "train":
            rows_q, rows_k = (case["batch"], case["seqlen_q"]), (case["batch"], case["seqlen_k"])
        else:
            lengths = _lengths(case)
            rows_q = rows_k = (sum(lengths),)
            state["cu_seqlens"], state["longest"] = _int([0] + lengths).cumsum(0, dtype=torch.int32), max(lengths)
        state["inputs"] = (_normal(g, *rows_q, h, d), _normal(g, *rows_k, h_k, d), _values(g, *rows_k, h_k, d), _weights(g, h))
        for t in state["inputs"]:
            t.requires_grad_(True)
        state["dout"] = _values(g, *rows_q, h, d)
        return state
    if kind == "serve":
        b, h, new, page, capacity = case["batch"], case["heads"], case["new_tokens"], case["page"], _capacity(case)
        state["q"], state["lam"] = _normal(g, b, new, h, d), _weights(g, h)
        state["k"], state["v"] = _normal(g, b, new, h_k, d), _values(g, b, new, h_k, d)
        rows = (b * capacity // page, page) if page else (b, capacity)
        state["k_cache"], state["v_cache"] = _normal(g, *rows, h_k, d), _values(g, *rows, h_k, d)
        state["cache_seqlens"] = _int(_lengths(case))
        state["block_table"] = torch.randperm(rows[0], generator=g, device="cuda").int().view(b, -1) if page else None
        return state
    state["pool"] = _normal(g, 2 * case["layers"], case["pages"], case["page"], h_k, d)
    state["caches"] = list(state["pool"].unbind(0))  # k and v of every layer
    if kind == "copy":
        order = torch.randperm(case["pages"], generator=g, device="cuda").int()
        state["src"], state["dst"] = order[: case["pairs"]].contiguous(), order[-case["pairs"]:].contiguous()
        return state
    lengths, table, new, parents, children, finished = _page_plan(case)
    state["before"] = _int(table), _int(lengths), torch.zeros(case["pages"], dtype=torch.int32, device="cuda")
    held = state["before"][0]
    state["before"][2][held[held >= 0].long()] = 1
    state["tables"] = [t.clone() for t in state["before"]]
    state["new"], state["parents"], state["children"], state["finished"] = _int(new), _int(parents), _int(children), _int(finished)
    return state


# ---- plain forms ----
def _attend(q, k, v, lam, mask, dout=None):
    """q (b, sq, h, d), k, v (b, sk, h_k, d), lam (h), all fp32; mask (b, sq, sk): visible.  The output, and with dout the gradients."""
    b, sq, h, d = q.shape
    sk, h_k = k.shape[1:3]
    group, half = h // h_k, d // 2
    scale = half ** -0.5
    seen = mask[:, None, None]
    lam = lam.view(1, h_k, group, 1, 1)
    q = q.view(b, sq, h_k, group, d).permute(0, 2, 3, 1, 4).reshape(b, h_k, group * sq, d)
    k, v = k.permute(0, 2, 1, 3), v.permute(0, 2, 1, 3)

    def softmax(m):
        at = slice(m * half, (m + 1) * half)
        s = (q[..., at] @ k[..., at].transpose(-1, -2)).view(b, h_k, group, sq, sk).mul_(scale).masked_fill_(~seen, -math.inf)
        top = s.amax(-1, keepdim=True)
        s = s.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
        return s.div_(s.sum(-1, keepdim=True).clamp_min(1e-30))

    def rows(x):  # (b, h_k, group * sq, d) -> (b, sq, h, d)
        return x.view(b, h_k, group, sq, -1).permute(0, 3, 1, 2, 4).reshape(b, sq, h, -1)

    a_1, a_2 = softmax(0), softmax(1)
    out = rows((a_1 - lam * a_2).view(b, h_k, group * sq, sk) @ v)
    if dout is None:
        return out
    do = dout.view(b, sq, h_k, group, d).permute(0, 2, 3, 1, 4).reshape(b, h_k, group * sq, d)
    dv = (a_1 - lam * a_2).view(b, h_k, group * sq, sk).transpose(-1, -2) @ do
    dp = (do @ v.transpose(-1, -2)).view(b, h_k, group, sq, sk)
    delta_1, delta_2 = (a_1 * dp).sum(-1, keepdim=True), (a_2 * dp).sum(-1, keepdim=True)
    dlam = -delta_2.double().sum((0, 3, 4)).view(h).float()
    ds_1 = (a_1.mul_(dp - delta_1)).view(b, h_k, group * sq, sk)
    ds_2 = (a_2.mul_(dp - delta_2).mul_(-lam)).view(b, h_k, group * sq, sk)
    dq = rows(torch.cat((ds_1 @ k[..., :half], ds_2 @ k[..., half:]), -1)) * scale
    dk = torch.cat((ds_1.transpose(-1, -2) @ q[..., :half], ds_2.transpose(-1, -2) @ q[..., half:]), -1) * scale
    return out, dq, dk.permute(0, 2, 1, 3), dv.permute(0, 2, 1, 3), dlam


def _half(*tensors):
    return tuple(t.half() for t in tensors)


def _at_or_before(rows, keys, causal):
    """Visible pairs, the diagonal at the bottom right."""
    i, j = torch.arange(rows, device="cuda")[:, None], torch.arange(keys, device="cuda")[None]
    return j <= i + keys - rows if causal else torch.ones(rows, keys, dtype=torch.bool, device="cuda")


def _plain_train(state):
    case = state["case"]
    with torch.no_grad():
        q, k, v, lam = (t.float() for t in state["inputs"])
        dout = state["dout"].float()
        if case["kind"] == "train":
            mask = _at_or_before(case["seqlen_q"], case["seqlen_k"], case["causal"])[None].expand(case["batch"], -1, -1)
            return _half(*_attend(q, k, v, lam, mask, dout))
        at = torch.arange(q.shape[0], device="cuda")
        text = torch.searchsorted(state["cu_seqlens"].long(), at, right=True)
        mask = text[:, None] == text[None]
        if case["causal"]:
            mask = mask & (at[None] <= at[:, None])
        out, dq, dk, dv, dlam = _attend(q[None], k[None], v[None], lam, mask[None], dout[None])
        return _half(out[0], dq[0], dk[0], dv[0], dlam)


def _plain_serve(state):
    q, k, v, lens, table = (state[n] for n in ("q", "k", "v", "cache_seqlens", "block_table"))
    k_cache, v_cache = state["k_cache"], state["v_cache"]
    b, new = q.shape[:2]
    at = lens.long()[:, None] + torch.arange(new, device="cuda")
    if table is None:
        place = torch.arange(b, device="cuda")[:, None].expand_as(at), at
    else:
        page = k_cache.shape[1]
        place = table.long().gather(1, at // page), at % page
    k_cache[place], v_cache[place] = k, v

    def cached(x):
        return (x if table is None else x[table.long()].flatten(1, 2)).float()

    keys = cached(k_cache)
    mask = torch.arange(keys.shape[1], device="cuda") <= at[..., None]
    return _half(_attend(q.float(), keys, cached(v_cache), state["lam"].float(), mask)) + (k_cache, v_cache)


def _free_pages(refs):
    """The free pages in ascending order, the others behind them; how many are free."""
    free = refs == 0
    return torch.argsort((~free).to(torch.int8), stable=True), free.sum()


def _plain_reserve(table, lens, refs, new, page):
    columns = table.shape[1]
    held = (table >= 0).long().cumprod(1).sum(1)
    want = (lens.long() + new + page - 1) // page
    need = torch.where(want <= columns, (want - held).clamp_min(0), 0)
    upto = need.cumsum(0)
    free, n_free = _free_pages(refs)
    granted = (want <= columns) & ((need == 0) | (upto <= n_free))
    col = torch.arange(columns, device="cuda")
    gets = granted[:, None] & (col >= held[:, None]) & (col < (held + need)[:, None])
    page_of = free[((upto - need)[:, None] + col - held[:, None]).clamp(0, refs.numel() - 1)]
    table.copy_(torch.where(gets, page_of.int(), table))
    refs.index_add_(0, page_of.flatten(), gets.flatten().int())
    return granted


def _plain_fork(pool, table, lens, refs, parents, children, page):
    parents, children = parents.long(), children.long()
    n, rows, columns = parents.numel(), table.shape[0], table.shape[1]
    held = (table >= 0).long().cumprod(1).sum(1)
    inside = (parents >= 0) & (parents < rows) & (children >= 0) & (children < rows)
    p, c = parents.clamp(0, rows - 1), children.clamp(0, rows - 1)
    first = torch.full((rows,), n, device="cuda").scatter_reduce_(0, c, torch.where(inside, torch.arange(n, device="cuda"), n), "amin")
    length = lens[p].long()
    full, rest = length // page, length % page
    valid = inside & (held[c] == 0) & (held[p] > 0) & (held[p] >= full + (rest > 0)) & (first[c] == torch.arange(n, device="cuda"))
    need = (valid & (rest > 0)).long()
    upto = need.cumsum(0)
    free, n_free = _free_pages(refs)
    granted = valid & ((need == 0) | (upto <= n_free))
    col = torch.arange(columns, device="cuda")
    shared = granted[:, None] & (col < full[:, None])
    copied = granted & (need > 0)
    to = free[(upto - need).clamp(0, refs.numel() - 1)]
    old = table[p]
    row = torch.where(shared, old, torch.where(copied[:, None] & (col == full[:, None]), to[:, None].int(), -1))
    refs.index_add_(0, old.clamp_min(0).long().flatten(), shared.flatten().int())
    refs.index_add_(0, to, copied.int())
    table[c[granted]] = row[granted]
    lens[c[granted]] = length[granted].int()
    src = old.gather(1, full.clamp_max(columns - 1)[:, None])[copied, 0].long()
    used = torch.arange(page, device="cuda") < rest[copied][:, None]
    pool[:, to[copied]] = torch.where(used[..., None, None], pool[:, src], pool[:, to[copied]])
    return granted


def _plain_free(table, lens, refs, rows):
    rows = rows.long().unique()
    held = table[rows]
    refs.index_add_(0, held.clamp_min(0).long().flatten(), -(held >= 0).flatten().int())
    table[rows] = -1
    lens[rows] = 0


def _plain_compact(pool, table, refs):
    live = refs > 0
    n = live.sum()
    at = torch.arange(refs.numel(), device="cuda")
    src, dst = at[live & (at >= n)], at[~live & (at < n)]
    pool[:, dst] = pool[:, src]
    to = at.int()
    to[src] = dst.int()
    table.copy_(torch.where(table >= 0, to[table.clamp_min(0).long()], table))
    refs[dst] = refs[src]
    refs[src] = 0
    return n.int().view(1)


def _plain_copy(pool, src, dst):
    done = torch.ones(src.numel(), dtype=torch.bool, device="cuda")
    pool[:, dst.long()] = pool[:, src.long()]
    return done


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        import flash_attention_turing_b200 as fa
    if kind in ("train", "varlen"):
        if not own:
            return _plain_train(state)
        if kind == "train":
            out = fa.flash_diff_attn_func(*state["inputs"], causal=case["causal"])
        else:
            cu, longest = state["cu_seqlens"], state["longest"]
            out = fa.flash_diff_attn_varlen_func(*state["inputs"], cu, cu, longest, longest, causal=case["causal"])
        return (out.detach(), *torch.autograd.grad(out, state["inputs"], state["dout"]))
    if kind == "serve":
        if not own:
            return _plain_serve(state)
        out = fa.flash_diff_attn_with_kvcache(state["q"], state["k_cache"], state["v_cache"], state["lam"], state["k"], state["v"],
                                              cache_seqlens=state["cache_seqlens"], block_table=state["block_table"], causal=True)
        return out, state["k_cache"], state["v_cache"]
    pool, caches = state["pool"], state["caches"]
    if kind == "copy":
        if own:
            return fa.kvcache_copy_pages(caches, state["src"], state["dst"]), pool
        return _plain_copy(pool, state["src"], state["dst"]), pool
    for now, before in zip(state["tables"], state["before"]):  # every pass begins with the same tables
        now.copy_(before)
    table, lens, refs = state["tables"]
    if kind == "compact":
        n = fa.kvcache_compact(caches, table, refs) if own else _plain_compact(pool, table, refs)
        return n, table, refs, pool
    page = case["page"]
    if own:
        reserved = fa.kvcache_reserve(table, lens, refs, state["new"], page)
        forked = fa.kvcache_fork(caches, table, lens, refs, state["parents"], state["children"])
        fa.kvcache_free(table, lens, refs, state["finished"])
    else:
        reserved = _plain_reserve(table, lens, refs, state["new"], page)
        forked = _plain_fork(pool, table, lens, refs, state["parents"], state["children"], page)
        _plain_free(table, lens, refs, state["finished"])
    return reserved, forked, table, lens, refs, pool


# ---- the definition in 64 bits ----
def _one_head(q, k, v, weight, seen):
    """One head of one sequence by the definition."""
    maps = []
    for a, b in zip(q.chunk(2, -1), k.chunk(2, -1)):
        s = (a @ b.T) / math.sqrt(a.shape[-1])
        s = torch.where(seen, s, torch.full_like(s, -math.inf))
        maps.append(torch.softmax(s, -1).nan_to_num(0.0))
    return (maps[0] - weight * maps[1]) @ v


def exact(case, seed):
    if case["kind"] not in ("train", "varlen", "serve"):
        return None  # whole numbers and copies
    state = prepare(case, seed)
    group = case["heads"] // case["heads_k"]
    if case["kind"] == "serve":
        q, lam = state["q"].double(), state["lam"].double()
        out = torch.empty_like(q)
        for b, n in enumerate(_lengths(case)):
            stored = []
            for cache, more in ((state["k_cache"], state["k"]), (state["v_cache"], state["v"])):
                whole = cache[b] if state["block_table"] is None else cache[state["block_table"][b].long()].flatten(0, 1)
                stored.append(torch.cat((whole[:n], more[b])).double())
            seen = _at_or_before(q.shape[1], stored[0].shape[0], True)
            for h in range(case["heads"]):
                out[b, :, h] = _one_head(q[b, :, h], stored[0][:, h // group], stored[1][:, h // group], lam[h], seen)
        return out, None, None
    q, k, v, lam = (t.detach().double() for t in state["inputs"])
    dout = state["dout"].double()
    if case["kind"] == "train":
        parts = [(b, slice(0, case["seqlen_q"]), slice(0, case["seqlen_k"])) for b in range(case["batch"])]
    else:
        q, k, v, dout = q[None], k[None], v[None], dout[None]
        ends = state["cu_seqlens"].tolist()
        parts = [(0, slice(a, b), slice(a, b)) for a, b in zip(ends, ends[1:])]
    out, dq, dk, dv, dlam = (torch.zeros_like(t) for t in (q, q, k, v, lam))
    for b, rows, keys in parts:
        seen = _at_or_before(rows.stop - rows.start, keys.stop - keys.start, case["causal"])
        for h in range(case["heads"]):
            at = h // group
            leaves = [t.clone().requires_grad_(True) for t in (q[b, rows, h], k[b, keys, at], v[b, keys, at], lam[h])]
            o = _one_head(*leaves, seen)
            grads = torch.autograd.grad(o, leaves, dout[b, rows, h])
            out[b, rows, h], dq[b, rows, h] = o.detach(), grads[0]
            dk[b, keys, at] += grads[1]
            dv[b, keys, at] += grads[2]
            dlam[h] += grads[3]
    if case["kind"] == "varlen":
        out, dq, dk, dv = out[0], dq[0], dk[0], dv[0]
    return out, dq, dk, dv, dlam


# ---- what a pass cannot do without ----
def _pairs(rows, keys, causal):
    if not causal:
        return rows * keys
    return rows * keys - rows * (rows - 1) // 2 if keys >= rows else keys * (keys + 1) // 2


def work(case):
    """Products over the visible pairs: two in the forward (both maps: 2 d each), five in the backward."""
    kind, d, h_k = case["kind"], case["head_dim"], case["heads_k"]
    if kind in ("train", "varlen"):
        h = case["heads"]
        if kind == "train":
            pairs = case["batch"] * _pairs(case["seqlen_q"], case["seqlen_k"], case["causal"])
            tokens, tokens_k = case["batch"] * case["seqlen_q"], case["batch"] * case["seqlen_k"]
        else:
            pairs = sum(_pairs(n, n, case["causal"]) for n in _lengths(case))
            tokens = tokens_k = sum(_lengths(case))
        return {"bytes": 2 * d * (4 * tokens * h + 4 * tokens_k * h_k), "flops": 14.0 * pairs * h * d}
    if kind == "serve":
        h, new, lengths = case["heads"], case["new_tokens"], _lengths(case)
        moved = 2 * 2 * h_k * d * (sum(lengths) + 2 * case["batch"] * new) + 2 * 2 * case["batch"] * new * h * d
        return {"bytes": moved, "flops": 4.0 * h * d * sum(_pairs(new, n + new, True) for n in lengths)}
    token = 2 * 2 * case["layers"] * h_k * d  # bytes of a token in all caches
    if kind == "copy":
        return {"bytes": 2 * case["pairs"] * case["page"] * token, "flops": 0.0}
    lengths, table, _, parents, _, _ = _page_plan(case)
    tables = 4 * (case["pages"] + case["rows"] * (len(table[0]) + 1))
    if kind == "round":
        return {"bytes": 2 * token * sum(lengths[p] % case["page"] for p in parents) + 2 * tables, "flops": 0.0}
    live = {p for row in table for p in row if p >= 0}
    return {"bytes": 2 * token * case["page"] * sum(p >= len(live) for p in live) + 2 * tables, "flops": 0.0}
