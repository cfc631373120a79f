"""Reserving, forking, freeing, compacting and copying the pages of a KV cache: tables and pages are compared exactly with a model
of lists, which does one thing after the other."""
import random

import pytest
import torch

import flash_attention_turing_b200 as fa
from diff_oracle import check, sequence

pytestmark = pytest.mark.gpu


class Model:
    """The tables and the pages as Python lists; a page is one number per token."""

    def __init__(self, rows, columns, pages, page_size):
        self.table, self.lens, self.refs = [[] for _ in range(rows)], [0] * rows, [0] * pages
        self.columns, self.page = columns, page_size
        self.data = [[0] * page_size for _ in range(pages)]

    def free_pages(self):
        return [p for p, r in enumerate(self.refs) if r == 0]

    def reserve(self, new):
        free, used, granted = self.free_pages(), 0, []
        for r, more in enumerate(new):
            want = -(-(self.lens[r] + max(more, 0)) // self.page)
            need = max(0, want - len(self.table[r]))
            if want > self.columns:
                granted.append(False)
                continue
            granted.append(need == 0 or used + need <= len(free))
            if granted[-1]:
                for p in free[used:used + need]:
                    self.table[r].append(p)
                    self.refs[p] = 1
            used += need
        return granted

    def fork(self, parents, children):
        free, used, granted, named, before = self.free_pages(), 0, [], set(), [len(t) for t in self.table]
        rows = len(self.table)
        for p, c in zip(parents, children):
            ok = 0 <= p < rows and 0 <= c < rows
            if ok and c in named:
                ok = False
            elif ok:
                named.add(c)
            ok = ok and before[c] == 0 and before[p] > 0 and before[p] >= -(-self.lens[p] // self.page)
            full, rest = divmod(self.lens[p], self.page) if ok else (0, 0)
            if ok and rest:
                used += 1
                ok = used <= len(free)
            granted.append(ok)
            if not ok:
                continue
            self.table[c] = self.table[p][:full]
            for x in self.table[c]:
                self.refs[x] += 1
            if rest:
                x = free[used - 1]
                self.table[c].append(x)
                self.refs[x] = 1
                self.data[x][:rest] = self.data[self.table[p][full]][:rest]
            self.lens[c] = self.lens[p]
        return granted

    def free(self, rows):
        for r in rows:
            if 0 <= r < len(self.table):
                for p in self.table[r]:
                    self.refs[p] -= 1
                self.table[r], self.lens[r] = [], 0

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        dst = [p for p in range(live) if self.refs[p] == 0]
        src = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        to = dict(zip(src, dst))
        for a, b in to.items():
            self.data[b], self.refs[b], self.refs[a] = list(self.data[a]), self.refs[a], 0
        self.table = [[to.get(p, p) for p in t] for t in self.table]
        return live

    def copy(self, src, dst):
        n, done, before = len(self.refs), [], [list(d) for d in self.data]
        inside = [0 <= a < n and 0 <= b < n for a, b in zip(src, dst)]
        writes = {}
        for i, (a, b) in enumerate(zip(src, dst)):
            if inside[i] and a != b:
                writes[b] = i
        for i, (a, b) in enumerate(zip(src, dst)):
            done.append(inside[i] and a not in writes and (a == b or writes[b] == i))
            if done[-1]:
                self.data[b] = list(before[a])
        return done


class Cache:
    """The tensors of a model: every value of a token is the token's number plus its place in the layer."""

    def __init__(self, model, layers=2, heads=1, d=64, dtype=torch.float16, spare_columns=0):
        self.m, self.layers, self.shape = model, layers, (heads, d)
        rows, pages = len(model.table), len(model.refs)
        wide = torch.full((rows, model.columns + spare_columns), -7, dtype=torch.int32, device="cuda")
        self.table = wide[:, :model.columns]
        self.wide = wide
        self.table.fill_(-1)
        self.lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        self.pool = torch.zeros(pages, 2 * layers, model.page, heads, d, dtype=dtype, device="cuda")  # a page of all layers together
        self.caches = list(self.pool.unbind(1))
        self.offset = torch.arange(2 * layers * heads * d, device="cuda").view(1, 2 * layers, 1, heads, d) % 7
        self.write()

    def write(self):
        """New contents for all pages: tokens' numbers, as the model has them."""
        x = torch.tensor(self.m.data, device="cuda")[:, None, :, None, None]
        self.pool.copy_((x + self.offset).to(self.pool.dtype))

    def compare(self):
        m = self.m
        want = [t + [-1] * (m.columns - len(t)) for t in m.table]
        assert self.table.tolist() == want
        assert self.lens.tolist() == m.lens and self.refs.tolist() == m.refs
        assert (self.wide[:, m.columns:] == -7).all()
        x = torch.tensor(m.data, device="cuda")[:, None, :, None, None]
        assert torch.equal(self.pool, (x + self.offset).to(self.pool.dtype))


def _int(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


CACHES = [  # rows, columns, pages, page size, layers, heads, d, dtype
    (6, 5, 17, 256, 2, 1, 64, torch.float16),
    (3, 40, 20, 16, 1, 3, 8, torch.bfloat16),
    (40, 7, 90, 64, 3, 2, 128, torch.float32),
    (9, 6, 31, 48, 70, 1, 16, torch.uint8),        # 140 caches: more than one launch
    (1500, 4, 5000, 16, 1, 1, 16, torch.float16),  # more rows and pages than threads
]


@pytest.mark.parametrize("rows,columns,pages,page,layers,heads,d,dtype", CACHES)
def test_random_serving_steps(rows, columns, pages, page, layers, heads, d, dtype):
    rng = random.Random(rows)
    m = Model(rows, columns, pages, page)
    c = Cache(m, layers, heads, d, dtype, spare_columns=3)
    some = min(rows, 60)

    def fill():
        for p in range(pages):
            start = rng.randrange(100)
            m.data[p] = [(start + i) % 100 for i in range(page)]
        c.write()

    fill()
    for step in range(14):
        if rng.random() < 0.2:
            more = rng.choice((0, 1, page))
            got, new = fa.kvcache_reserve(c.table, c.lens, c.refs, more, page), [more] * rows
        else:
            new = [rng.choice((-3, 0, 1, page - 1, page, 2 * page, 3 * page + 1, columns * page + 1)) for _ in range(rows)]
            got = fa.kvcache_reserve(c.table, c.lens, c.refs, _int(new), page)
        granted = m.reserve(new)
        assert got.tolist() == granted
        c.compare()
        for r in range(rows):  # the attention would append now
            if granted[r]:
                m.lens[r] += max(new[r], 0)
        c.lens.copy_(_int(m.lens))
        parents = [rng.randrange(-2, rows + 2) for _ in range(some)]
        children = [rng.randrange(-2, rows + 2) for _ in range(some)]
        got = fa.kvcache_fork(c.caches, c.table, c.lens, c.refs, _int(parents), _int(children))
        assert got.tolist() == m.fork(parents, children)
        c.compare()
        gone = [rng.randrange(-2, rows + 2) for _ in range(rng.choice((1, some // 2 + 1, rows)))]
        gone += gone[:2]
        fa.kvcache_free(c.table, c.lens, c.refs, _int(gone))
        m.free(gone)
        c.compare()
        if step % 3 == 2:
            assert fa.kvcache_compact(c.caches, c.table, c.refs).tolist() == [m.compact()]
            c.compare()
            fill()
        src = [rng.randrange(-1, pages + 1) for _ in range(some)]
        dst = [rng.randrange(-1, pages + 1) for _ in range(some)]
        src += src[:3] + [2]
        dst += [0, 1, 0, 2]
        assert fa.kvcache_copy_pages(c.caches, _int(src), _int(dst)).tolist() == m.copy(src, dst)
        c.compare()


@pytest.mark.parametrize("n", [512, 513, 2500])
def test_copies_of_many_pages(n):
    """Up to 512 entries are looked at by every CTA, more by a kernel of their own."""
    rng, pages = random.Random(n), 3000
    m = Model(1, 1, pages, 2)
    m.data = [[p % 90] * 2 for p in range(pages)]
    c = Cache(m, 1, 1, 8)
    src, dst = ([rng.randrange(-1, pages + 1) for _ in range(n)] for _ in range(2))
    assert fa.kvcache_copy_pages(c.caches, _int(src), _int(dst)).tolist() == m.copy(src, dst)
    c.compare()
    order = rng.sample(range(pages), pages)  # none in another's way
    src, dst = order[:n // 2], order[-(n // 2):]
    assert fa.kvcache_copy_pages(c.caches, _int(src), _int(dst)).all() and all(m.copy(src, dst))
    c.compare()


@pytest.mark.parametrize("n", [1, 32, 33, 300])
def test_forks_of_many_rows(n):
    """Up to 32 entries are looked at by every CTA, more by a kernel of their own; in either case the free pages may not suffice."""
    rng, rows, page = random.Random(n), 350, 32
    m = Model(rows, 4, 160, page)
    c = Cache(m, 2, 2, 64)
    new = [rng.choice((0, 1, 40, 64, 100)) if r < 60 else 0 for r in range(rows)]
    got = fa.kvcache_reserve(c.table, c.lens, c.refs, _int(new), page)
    granted = m.reserve(new)
    assert got.tolist() == granted
    m.lens = [x * ok for x, ok in zip(new, granted)]
    c.lens.copy_(_int(m.lens))
    for p in range(160):
        m.data[p] = [(p + i) % 90 for i in range(page)]
    c.write()
    for _ in range(3):
        parents = [rng.randrange(-1, 70) for _ in range(n)]
        children = [rng.randrange(60, rows + 1) for _ in range(n)]
        got = fa.kvcache_fork(c.caches, c.table, c.lens, c.refs, _int(parents), _int(children))
        assert got.tolist() == m.fork(parents, children)
        c.compare()
        fa.kvcache_free(c.table, c.lens, c.refs, _int(children[::2]))
        m.free(children[::2])


def test_rows_behind_one_that_cannot_be_served():
    m = Model(5, 8, 6, 32)
    c = Cache(m)
    for new in ([32, 0, 0, 0, 1], [0, 64, 1000, 128, 1], [1, 0, 33, 0, 32], [0, 0, 0, 0, 32]):
        assert fa.kvcache_reserve(c.table, c.lens, c.refs, _int(new), 32).tolist() == m.reserve(new)
        c.compare()
    assert fa.kvcache_reserve(c.table, c.lens, c.refs, 0, 32).tolist() == [True] * 5


def test_forks_beyond_the_last_page():
    m = Model(8, 4, 4, 32)
    c = Cache(m)
    m.reserve([40, 32, 0, 0, 0, 0, 0, 0])
    fa.kvcache_reserve(c.table, c.lens, c.refs, _int([40, 32, 0, 0, 0, 0, 0, 0]), 32)
    m.lens[:2] = [40, 32]
    c.lens.copy_(_int(m.lens))
    m.data = [[p] * 32 for p in range(4)]
    c.write()
    parents, children = [0, 0, 1, 0, 1, 1], [2, 3, 4, 4, 5, 5]
    got = fa.kvcache_fork(c.caches, c.table, c.lens, c.refs, _int(parents), _int(children))
    assert got.tolist() == m.fork(parents, children) == [True, False, True, False, True, False]
    c.compare()
    fa.kvcache_free(c.table, c.lens, c.refs, _int([1, 4, 5]))
    m.free([1, 4, 5])
    c.compare()
    m.lens[0] = 200  # longer than its pages: nothing to fork
    c.lens[0] = 200
    assert fa.kvcache_fork(c.caches, c.table, c.lens, c.refs, _int([0]), _int([6])).tolist() == m.fork([0], [6]) == [False]
    c.compare()


def test_empty_lists_and_empty_pool():
    m = Model(3, 4, 5, 32)
    c = Cache(m)
    none = _int([])
    assert fa.kvcache_fork(c.caches, c.table, c.lens, c.refs, none, none).shape == (0,)
    fa.kvcache_free(c.table, c.lens, c.refs, none)
    assert fa.kvcache_copy_pages(c.caches, none, none).shape == (0,)
    assert fa.kvcache_compact(c.caches, c.table, c.refs).tolist() == [0]
    c.compare()
    empty = [torch.zeros(0, 32, 64, dtype=torch.float16, device="cuda")]
    assert fa.kvcache_copy_pages(empty, _int([0]), _int([1])).tolist() == [False]


def test_pages_beyond_four_gigabytes():
    pages, size = 2600, 2 << 20
    cache = torch.empty(pages, 256, size // 256, dtype=torch.uint8, device="cuda")
    cache[pages - 1], cache[0] = 7, 3
    cache[1, 0], cache[pages - 2] = 0, 0
    assert fa.kvcache_copy_pages([cache], _int([pages - 1, 0]), _int([1, pages - 2])).all()
    assert (cache[1] == 7).all() and (cache[pages - 2] == 3).all() and (cache[0] == 3).all()


def test_in_a_cuda_graph_and_on_another_stream():
    m = Model(4, 6, 20, 32)
    c = Cache(m)
    new, parents, children, gone = _int([33, 0, 64, 0]), _int([0, 2]), _int([1, 3]), _int([0])

    def step():
        a = fa.kvcache_reserve(c.table, c.lens, c.refs, new, 32)
        c.lens.add_(new * a)
        b = fa.kvcache_fork(c.caches, c.table, c.lens, c.refs, parents, children)
        fa.kvcache_free(c.table, c.lens, c.refs, gone)
        return a, b, fa.kvcache_compact(c.caches, c.table, c.refs)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step()  # outside a capture first
        for t, x in ((c.table, -1), (c.lens, 0), (c.refs, 0)):
            t.fill_(x)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        got = step()
    m.data = [[p] * 32 for p in range(20)]
    c.write()
    for _ in range(3):
        graph.replay()
        granted = m.reserve(new.tolist())
        for r, ok in enumerate(granted):
            m.lens[r] += ok * new.tolist()[r]
        forked = m.fork([0, 2], [1, 3])
        m.free([0])
        live = m.compact()
        assert [x.tolist() for x in got] == [granted, forked, [live]]
        c.compare()


@pytest.mark.parametrize("differential", [True, False])
def test_serving_loop(differential):
    """Prompts in chunks, single tokens, forks, sequences that end and a compaction, two layers on one block table; the attention of
    every step against the sequences kept as plain tensors."""
    gen, rng = torch.Generator().manual_seed(1), random.Random(1)
    rows, columns, pages, page, layers, h, hk, d = 6, 5, 14, 256, 2, 4, 2, 64
    table = torch.full((rows, columns), -1, dtype=torch.int32, device="cuda")
    lens, refs = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(pages, dtype=torch.int32, device="cuda")
    caches = [torch.full((pages, page, hk, d), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2 * layers)]
    lam = torch.tensor([0.3, 0.8, 0.5, 0.6], device="cuda")
    empty = torch.zeros(0, hk, d, dtype=torch.float16, device="cuda")
    kept = [[[empty, empty] for _ in range(layers)] for _ in range(rows)]

    def randn(*shape):
        return torch.randn(*shape, generator=gen).half().cuda()

    def attend(size, live):
        new = torch.zeros(rows, dtype=torch.int32)
        new[live] = size
        granted = fa.kvcache_reserve(table, lens, refs, new.cuda(), page)
        assert granted.all()
        at = torch.tensor(live, device="cuda")
        for layer in range(layers):
            q, k, v = randn(len(live), size, h, d), randn(len(live), size, hk, d), randn(len(live), size, hk, d)
            k_cache, v_cache = caches[2 * layer:2 * layer + 2]
            args = dict(cache_seqlens=lens[at], block_table=table[at], causal=True)
            if differential:
                out = fa.flash_diff_attn_with_kvcache(q, k_cache, v_cache, lam, k, v, **args)
            else:
                out = fa.flash_attn_with_kvcache(q, k_cache, v_cache, k, v, **args)
            for i, r in enumerate(live):
                kept[r][layer] = [torch.cat((a, b[i])) for a, b in zip(kept[r][layer], (k, v))]
                kk, vv = kept[r][layer]
                if differential:
                    check(out[i], sequence(q[i], kk, vv, lam, True)["out"], f"row {r}")
                else:
                    seen = torch.arange(kk.shape[0], device="cuda") <= torch.arange(size, device="cuda")[:, None] + kk.shape[0] - size
                    for head in range(h):
                        s = q[i, :, head].double() @ kk[:, head // 2].double().T * d ** -0.5
                        p = torch.softmax(s.masked_fill(~seen, -float("inf")), -1)
                        want, size_ = p @ vv[:, head // 2].double(), p @ vv[:, head // 2].double().abs()
                        # one rounding of P, one of the output, scores in 32 bits
                        assert ((out[i, :, head].double() - want).abs() <= 2 ** -11 * (1.1 * size_ + want.abs()) + 2 ** -20).all()
        lens[at] += size

    attend(200, [0, 1])
    attend(130, [0, 1])
    attend(1, [0, 1])
    parents, children = _int([0, 0, 1]), _int([2, 3, 4])
    assert fa.kvcache_fork(caches, table, lens, refs, parents, children).all()
    for p, c in ((0, 2), (0, 3), (1, 4)):
        kept[c] = [list(x) for x in kept[p]]
    attend(1, [0, 1, 2, 3, 4])
    attend(5, [2, 4])
    fa.kvcache_free(table, lens, refs, _int([0, 4, -1]))
    kept[0], kept[4] = ([[empty, empty] for _ in range(layers)] for _ in range(2))
    live = fa.kvcache_compact(caches, table, refs)
    used = {p for row in table.tolist() for p in row if p >= 0}
    assert used == set(range(live.item()))
    attend(60, [1, 2, 3])
    attend(300, [0, 5])
    assert fa.kvcache_fork(caches, table, lens, refs, _int([5]), _int([4])).all()
    kept[4] = [list(x) for x in kept[5]]
    attend(1, [rng.randrange(4), 4, 5])
    assert fa.device_status() == 0


def test_refusals():
    m = Model(3, 4, 5, 32)
    c = Cache(m)
    one = _int([0])
    for call, text in (
        (lambda: fa.kvcache_reserve(c.table, c.lens, c.refs.long(), 1, 32), "page_refs must be a torch.int32"),
        (lambda: fa.kvcache_reserve(c.table, c.lens[:2], c.refs, 1, 32), "cache_seqlens must have shape"),
        (lambda: fa.kvcache_reserve(c.table, c.lens, c.refs, -1, 32), "non-negative"),
        (lambda: fa.kvcache_reserve(c.table, c.lens, c.refs, 1, 0), "page_size"),
        (lambda: fa.kvcache_reserve(c.table, c.lens, c.refs, _int([1, 2]), 32), "new_tokens must have shape"),
        (lambda: fa.kvcache_reserve(c.table.t(), _int([0] * 4), c.refs, 1, 32), "contiguous last dimension"),
        (lambda: fa.kvcache_reserve(c.table.cpu(), c.lens, c.refs, 1, 32), "CUDA"),
        (lambda: fa.kvcache_fork(c.caches, c.table, c.lens, c.refs[:4], one, one), "number of pages"),
        (lambda: fa.kvcache_fork(c.caches, c.table, c.lens, c.refs, one, _int([1, 2])), "same length"),
        (lambda: fa.kvcache_fork(c.caches, c.table, c.lens, c.refs, one.cpu(), one), "parents must be a CUDA tensor"),
        (lambda: fa.kvcache_fork([c.caches[0], c.caches[1][:, :16]], c.table, c.lens, c.refs, one, one), "same device, shape"),
        (lambda: fa.kvcache_copy_pages([c.caches[0].transpose(1, 3)], one, one), "contiguous in every cache"),
        (lambda: fa.kvcache_copy_pages([torch.zeros(4, 3, 1, device="cuda").half()], one, one), "multiple of 16"),
        (lambda: fa.kvcache_copy_pages([torch.zeros(1 + 4 * 32, device="cuda").half()[1:].view(4, 32)], one, one), "aligned"),
        (lambda: fa.kvcache_copy_pages([torch.zeros(1, 32, 16, device="cuda").expand(4, 32, 16)], one, one), "overlap"),
        (lambda: fa.kvcache_copy_pages([], one, one), "at least one"),
        (lambda: fa.kvcache_free(c.table, c.lens, c.refs, one.long()), "rows must be a torch.int32"),
        (lambda: fa.kvcache_fork([torch.zeros(5, 32, 1, 4, device="cuda").half()], c.table, c.lens, c.refs, one, one), "token must be a multiple"),
    ):
        with pytest.raises(RuntimeError, match=text):
            call()
    c.compare()


@pytest.mark.parametrize("n", [1, 5, 40])
def test_a_parent_whose_row_has_a_hole_is_not_forked(n):
    """-1 before the last page, which no function leaves: refused, and nothing is counted in front of page_refs."""
    rows, pages, page = n + 3, 120, 16
    memory = torch.zeros(pages + 64, dtype=torch.int32, device="cuda")
    refs = memory[32:32 + pages]
    table = torch.full((rows, 4), -1, dtype=torch.int32, device="cuda")
    table[0], table[1], table[2] = _int([3, -1, 5, -1]), _int([0, 1, 2, -1]), _int([6, -1, 7, 8])
    for p in (3, 5, 0, 1, 2, 6, 7, 8):
        refs[p] = 1
    lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    lens[:3] = _int([3 * page, 2 * page + 5, 3 * page + 2])  # full pages; a last one to copy; and one behind a hole
    cache = torch.arange(pages, device="cuda").half()[:, None, None].expand(pages, page, 64).contiguous()
    before = table.clone()
    parents = [(0, 2, 1)[i % 3] for i in range(n)]
    got = fa.kvcache_fork([cache], table, lens, refs, _int(parents), _int(list(range(3, rows)))).tolist()
    assert got == [p == 1 for p in parents]
    assert not memory[:32].any() and not memory[32 + pages:].any() and torch.equal(table[:3], before[:3])
    copies = sum(got)
    assert refs[:3].tolist() == [1 + copies, 1 + copies, 1] and refs.sum().item() == 8 + 3 * copies
    for i, (p, ok) in enumerate(zip(parents, got)):
        row, length = table[3 + i].tolist(), lens[3 + i].item()
        assert (row[:2] == [0, 1] and row[3] == -1 and length == 2 * page + 5) if ok else (row == [-1] * 4 and length == 0)
        if ok:
            assert (cache[row[2], :5] == 2).all() and refs[row[2]] == 1
