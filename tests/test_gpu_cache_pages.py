"""GPU: the page operators against a model of them in Python integers; contents are compared bit for bit."""

from __future__ import annotations

import random

import pytest
import torch

from rows_helpers import i32

pytestmark = pytest.mark.gpu


def _ops():
    from specdec_b200.kernels import ops

    return ops


def _cache(B, pages, cap, *, v8=False, KV=2, D=128, layers=2, seed=0):
    from specdec_b200.engine.paged_cache import PagedKVCache

    c = PagedKVCache.allocate(layers, B, KV, D, cap, v_dtype="e4m3" if v8 else "bf16", num_pages=pages, on_demand=True)
    g = torch.Generator(device="cuda").manual_seed(seed)
    for p in c.pools:  # every page its own contents
        for t in (p.k, p.v, p.v_scale):
            if t is not None:
                t.view(torch.uint8).random_(0, 256, generator=g)
    return c


def _bytes(c):
    """Contents of every page: [num_pages] tuples of the layers' bytes, as one tensor a page."""
    parts = [t.reshape(c.num_pages, -1).view(torch.uint8) for p in c.pools for t in (p.k, p.v, p.v_scale) if t is not None]
    return torch.cat(parts, 1).cpu()


class Model:
    """What the operators do, on lists."""

    def __init__(self, c):
        self.pages, self.max = c.num_pages, c.max_pages
        self.rows = [[] for _ in range(c.num_seqs)]
        self.len = [0] * c.num_seqs
        self.refs = [0] * c.num_pages
        self.data = list(range(c.num_pages))  # whose contents a page has
        self.status = 0

    def free_pages(self):
        return [p for p in range(self.pages) if self.refs[p] <= 0]

    def free(self, seqs):
        from specdec_b200 import _lib

        for s in seqs:
            if not 0 <= s < len(self.rows):
                self.status |= _lib.STATUS_BAD_SEQUENCE
                continue
            for p in self.rows[s]:
                self.refs[p] -= 1
            self.rows[s], self.len[s] = [], 0

    def fork(self, src, dst, length):
        from specdec_b200 import _lib

        B, todo = len(self.rows), []
        real = [0 <= s < B and 0 <= d < B and s != d for s, d in zip(src, dst)]
        for i, (s, d, n) in enumerate(zip(src, dst, length)):
            bad = not real[i] or n < 0 or n > self.max * 16 or n > self.len[s]
            for k in range(len(src)):
                if real[i] and real[k]:
                    bad |= (dst[k] == d and k < i) or dst[k] == s
            if bad:
                self.status |= _lib.STATUS_BAD_SEQUENCE
            elif (n + 15) // 16 > len(self.rows[s]):
                self.status |= _lib.STATUS_BAD_PAGE
            else:
                todo.append((s, d, n))
        for s, d, n in todo:
            for p in self.rows[d]:
                self.refs[p] -= 1
        for s, d, n in todo:
            self.rows[d] = self.rows[s][:n // 16]
            self.len[d] = n
            for p in self.rows[d]:
                self.refs[p] += 1
        free = self.free_pages()
        for s, d, n in todo:
            if n % 16:
                if not free:
                    self.status |= _lib.STATUS_NO_PAGES
                    self.len[d] = n // 16 * 16
                    continue
                p = free.pop(0)
                self.refs[p] = 1
                self.data[p] = self.data[self.rows[s][n // 16]]
                self.rows[d].append(p)

    def reserve(self, tokens):
        from specdec_b200 import _lib

        free, given, out_of = self.free_pages(), [], False
        old = list(self.refs)
        moves = []
        for s, n in enumerate(tokens):
            if n < 0 or n > self.max * 16:
                self.status |= _lib.STATUS_PAGE_OVERFLOW
                continue
            row, want = self.rows[s], (n + 15) // 16
            swaps = [j for j in range(self.len[s] // 16, min(len(row), want)) if old[row[j]] > 1] if n > self.len[s] else []
            k = len(swaps) + max(want - len(row), 0)
            if k == 0:
                continue
            if out_of or k > len(free):
                out_of = True
                self.status |= _lib.STATUS_NO_PAGES
                continue
            for j in swaps:
                p = free.pop(0)
                given.append(row[j])
                if j == self.len[s] // 16 and self.len[s] % 16:
                    moves.append((p, row[j]))
                row[j] = p
                self.refs[p] = 1
            while len(row) < want:
                row.append(free.pop(0))
                self.refs[row[-1]] = 1
        for p in given:
            self.refs[p] -= 1
        before = list(self.data)
        for new, was in moves:
            self.data[new] = before[was]

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        holes = [p for p in range(live) if self.refs[p] <= 0]
        move = [p for p in range(live, self.pages) if self.refs[p] > 0]
        to = dict(zip(move, holes))
        for a, b in to.items():
            self.data[b], self.refs[b], self.refs[a] = self.data[a], self.refs[a], 0
        self.rows = [[to.get(p, p) for p in r] for r in self.rows]
        return live

    def check(self, c, first, status=None):
        table = c.page_table.cpu().tolist()
        assert table == [r + [-1] * (self.max - len(r)) for r in self.rows]
        assert c.lengths.cpu().tolist() == self.len
        assert c.page_refs.cpu().tolist() == self.refs
        now = _bytes(c)
        for p in range(self.pages):
            if self.refs[p] > 0:
                assert torch.equal(now[p], first[self.data[p]]), f"page {p}"
        if status is not None:
            assert int(status) == self.status, (int(status), self.status)


@pytest.mark.parametrize("v8,KV,D,layers", [(False, 2, 128, 2), (True, 2, 128, 2), (False, 1, 64, 1), (True, 3, 128, 65)])
@pytest.mark.parametrize("seed", range(4))
def test_random_calls(v8, KV, D, layers, seed):
    """Forks, reserves, frees and compactions in any order, pools that run out among them."""
    ops, rng = _ops(), random.Random(seed)
    B, cap = rng.choice([(5, 100), (17, 300), (40, 33)])
    pages = rng.choice([12, 60, B * (cap // 16 + 1)])
    if layers > 60:
        pages = min(pages, 60)
    c = _cache(B, pages, cap, v8=v8, KV=KV, D=D, layers=layers, seed=seed)
    first, m = _bytes(c), Model(c)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ws = ops.page_workspace(c, 2 * B)
    for step in range(40 if layers < 60 else 12):
        kind = rng.choice(["reserve", "reserve", "fork", "fork", "free", "compact"])
        kw = dict(status=status, workspace=rng.choice([None, ws]))
        if kind == "reserve":
            tokens = [rng.choice([0, m.len[b], m.len[b] + rng.randint(0, 40), rng.randint(0, c.capacity)])
                      for b in range(B)]
            tokens = [min(t, c.capacity) for t in tokens]
            if rng.random() < 0.1:
                tokens[rng.randrange(B)] = rng.choice([-1, c.capacity + 1, 2**31 - 1])
            ops.reserve_pages(c, i32(tokens), **kw)
            m.reserve(tokens)
            # the sequences go on writing: some of the reserved tokens become theirs
            for b in range(B):
                if m.len[b] < tokens[b] <= len(m.rows[b]) * 16 and rng.random() < 0.7:
                    m.len[b] = rng.randint(m.len[b], tokens[b])
            c.lengths.copy_(i32(m.len))
        elif kind == "fork":
            n = rng.randint(0, B)
            src = [rng.randrange(-1, B + 1) if rng.random() < 0.1 else rng.randrange(B) for _ in range(n)]
            dst = [rng.randrange(-1, B + 1) if rng.random() < 0.1 else rng.randrange(B) for _ in range(n)]
            length = [rng.randint(-1, m.len[s] + 1) if 0 <= s < B else 5 for s in src]
            ops.fork_sequences(c, i32(src), i32(dst), i32(length), **kw)
            m.fork(src, dst, length)
        elif kind == "free":
            seqs = [rng.randrange(-1, B + 1) for _ in range(rng.randint(0, B // 2))]
            ops.free_sequences(c, i32(seqs), **kw)
            m.free([s for i, s in enumerate(seqs)])
        else:
            n = ops.compact_pages(c, **kw)
            assert int(n) == m.compact()
        m.check(c, first, status)
        status.zero_()
        m.status = 0


def test_many_sequences_and_requests():
    """More sequences and requests than a CTA has threads; more pages than one pass of it."""
    ops = _ops()
    B = 2500
    c = _cache(B, 5000, 48, KV=1, D=64, layers=1)
    first, m = _bytes(c), Model(c)
    c.reserve([33] + [0] * (B - 1))
    m.reserve([33] + [0] * (B - 1))
    m.len[0] = 33
    c.lengths.copy_(i32(m.len))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    c.fork([0] * (B - 1), range(1, B), [33] * (B - 1), status=status)
    m.fork([0] * (B - 1), list(range(1, B)), [33] * (B - 1))
    m.check(c, first, status)
    assert c.page_refs[0] == B
    odd = list(range(1, B, 2))
    c.free(odd, status=status)
    m.free(odd)
    m.check(c, first, status)
    assert int(c.compact(status=status)) == m.compact()
    m.check(c, first, status)
    # everyone goes on writing into its own page, and past the pool's end nobody after the last that fits
    want = [48] * B
    c.reserve(want, status=status)
    m.reserve(want)
    m.check(c, first, status)


def test_writes_after_a_fork_stay_apart():
    """A sequence that was forked from, and its fork, both go on in the page that they shared."""
    ops = _ops()
    for at in (16, 24, 31, 32):
        c = _cache(2, 20, 80)
        first, m = _bytes(c), Model(c)
        m.reserve([48, 0]), c.reserve([48, 0])
        m.len[0] = 48
        c.lengths.copy_(i32(m.len))
        c.fork([0], [1], [32])
        m.fork([0], [1], [32])
        # rolled back into the shared pages, both of them
        m.len = [at, at]
        c.lengths.copy_(i32(m.len))
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        c.reserve([48, 48], status=status)
        m.reserve([48, 48])
        m.check(c, first, status)
        rows = c.page_table.cpu().tolist()
        assert not set(rows[0][at // 16:3]) & set(rows[1][at // 16:3]) and rows[0][:at // 16] == rows[1][:at // 16]


def test_no_page_left():
    from specdec_b200 import _lib

    c = _cache(3, 3, 64)
    first, m = _bytes(c), Model(c)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    c.reserve([40, 16, 0], status=status)
    m.reserve([40, 16, 0])
    assert m.status == _lib.STATUS_NO_PAGES  # three pages for the first, none for the second
    m.check(c, first, status)
    status.zero_()
    m.status, m.len[0] = 0, 40
    c.lengths.copy_(i32(m.len))
    c.fork([0], [2], [40], status=status)
    m.fork([0], [2], [40])
    assert m.len[2] == 32 and m.status == _lib.STATUS_NO_PAGES  # the full pages only
    m.check(c, first, status)


@pytest.mark.parametrize("v8", [False, True])
def test_copy_pages(v8):
    from specdec_b200 import _lib

    ops = _ops()
    c = _cache(1, 700, 64, v8=v8, KV=3, layers=3)
    first = _bytes(c)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    perm = torch.randperm(700).tolist()
    src, dst = perm[:300], perm[300:600]
    src[7], dst[9], src[11], dst[13] = -1, 700, 2**31 - 1, -2**31
    src[20] = dst[20]  # onto itself
    ops.copy_pages(c, i32(src), i32(dst), status=status)
    assert int(status) == _lib.STATUS_BAD_PAGE
    want = first.clone()
    for i, (s, d) in enumerate(zip(src, dst)):
        if i not in (7, 9, 11, 13):
            want[d] = first[s]
    assert torch.equal(_bytes(c), want)
    ops.copy_pages(c, i32([]), i32([]))
    assert torch.equal(_bytes(c), want)


def test_offsets_past_32_bits():
    ops = _ops()
    from specdec_b200.engine.paged_cache import PagedKVCache

    c = PagedKVCache.allocate(1, 1, 2, 128, 16, num_pages=560_000, on_demand=True)  # 4.6 GB a pool
    n = c.num_pages
    c.pools[0].k[n - 2], c.pools[0].v[n - 2] = 3.0, 5.0
    ops.copy_pages(c, i32([n - 2]), i32([n - 1]))
    assert (c.pools[0].k[n - 1] == 3).all() and (c.pools[0].v[n - 1] == 5).all()
    assert not c.pools[0].k[:n - 2].any()
    assert int(c.compact()) == 0


def test_captured_calls():
    """Fork, reserve, free and compact in one graph, replayed: the same tables as the calls one by one."""
    ops = _ops()
    made = []
    for captured in (False, True):
        c = _cache(4, 40, 120, seed=1)
        c.reserve([50, 20, 0, 0])
        c.lengths.copy_(i32([50, 20, 0, 0]))
        a = dict(src=i32([0, 1]), dst=i32([2, 3]), length=i32([41, 17]))
        tokens, seqs = i32([60, 60, 60, 60]), i32([0])
        ws = ops.page_workspace(c, 4)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")

        def calls():
            ops.fork_sequences(c, a["src"], a["dst"], a["length"], workspace=ws, status=status)
            ops.reserve_pages(c, tokens, workspace=ws, status=status)
            ops.free_sequences(c, seqs, workspace=ws, status=status)
            return ops.compact_pages(c, workspace=ws, status=status)

        if captured:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                live = calls()
            graph.replay()
        else:
            live = calls()
        torch.cuda.synchronize()
        made.append((c.page_table.cpu(), c.page_refs.cpu(), c.lengths.cpu(), int(live), int(status), _bytes(c)))
    for x, y in zip(*made):
        assert x == y if isinstance(x, int) else torch.equal(x, y)
    assert made[0][4] == 0


def test_refusals_on_the_device():
    ops = _ops()
    c = _cache(3, 10, 64)
    from specdec_b200.engine.paged_cache import PagedKVCache

    static = PagedKVCache.allocate(1, 3, 2, 128, 64)
    for bad in (lambda: ops.free_sequences(static, i32([0])), lambda: ops.reserve_pages(c, i32([1, 2])),
                lambda: ops.reserve_pages(c, torch.zeros(3, device="cuda")), lambda: ops.free_sequences(c, torch.zeros(1)),
                lambda: ops.fork_sequences(c, i32([0]), i32([1, 2]), i32([3])),
                lambda: ops.fork_sequences(c, i32([0]), i32([1]), i32([3]), workspace=i32([0])),
                lambda: ops.free_sequences(c, i32([0]), workspace=torch.zeros(16, dtype=torch.uint8, device="cuda")),
                lambda: ops.copy_pages(c, i32([0]), i32([1, 2])), lambda: ops.compact_pages(c, status=torch.zeros(1))):
        with pytest.raises((ValueError, RuntimeError)):
            bad()
    ops.copy_pages(static, i32([0]), i32([1]))  # pages of any cache can be copied
