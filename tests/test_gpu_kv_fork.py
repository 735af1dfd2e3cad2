"""The page table after a selection over beams, against the same steps in Python; every table, length and page is compared bit for bit."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
KINDS = ["f32", "bf16", "i8", "e4m3"]
SIZE = {"f32": 4, "bf16": 2, "i8": 1, "e4m3": 1}


def fork(table, lens, parents, grow, n_pages, page, max_len):
    """(new table, new lengths, copies as (from page, to page, rows), free pages left, whether an error is reported)"""
    n, width = table.shape
    new, new_lens, error, used, lack = np.full_like(table, -1), np.zeros(n, np.int32), False, set(), False
    plans = []
    for i in range(n):
        parent, more = int(parents[i]), 0 if grow is None else int(grow[i])
        if parent >= n:
            error, parent = True, -1
        if parent < 0:
            plans.append(None)
            continue
        length = min(max(int(lens[parent]), 0), max_len)
        error = error or length != lens[parent]
        if more < 0 or length + more > max_len:
            error, more = True, 0
        new_lens[i] = length + more
        full, part = divmod(length, page)
        for j in range(full + (part > 0)):
            there = 0 <= table[parent, j] < n_pages
            error = error or not there
            if j < full and there:
                new[i, j] = table[parent, j]
                used.add(int(new[i, j]))
        at = int(table[parent, full]) if part and 0 <= table[parent, full] < n_pages else -1
        plans.append([full, part, at, -(-int(new_lens[i]) // page), False])
    owners = {}
    for i, plan in enumerate(plans):
        if plan and plan[2] >= 0 and plan[2] not in used and plan[2] not in owners:
            owners[plan[2]] = i
            plan[4] = True
    used |= set(owners)
    free = [p for p in range(n_pages) if p not in used]
    copies = []
    for i, plan in enumerate(plans):
        if not plan:
            continue
        full, part, at, end, kept = plan
        j = full
        if part and (kept or at < 0):
            new[i, j] = at
            j += 1
        for j in range(j, end):
            if free:
                new[i, j] = free.pop(0)
                if j == full and part:
                    copies.append((at, int(new[i, j]), part))
            else:
                error = True
    return new, new_lens, copies, len(free), error


class Pages:
    """A cache of random bytes with a table of its own, and the same on the host."""

    def __init__(self, fdx, kind, n_pages, page, kv, dk, dv, block, seed=0, odd=0):
        r = np.random.default_rng(seed)
        self.fdx, self.kind, self.n_pages, self.page, self.kv, self.dk, self.dv, self.block = fdx, kind, n_pages, page, kv, dk, dv, block
        self.host = [r.integers(0, 256, (n_pages, page, kv * d * SIZE[kind])).astype(np.uint8) for d in (dk, dv)]
        self.scales = [r.standard_normal((n_pages, page // block, kv)).astype(np.float32) for _ in range(2)] if block else []
        self.odd = odd   # bytes that the pages are off 16-byte places
        self.dev = [fdx.DevBuf.from_host(np.concatenate([np.zeros(odd, np.uint8), h.ravel()]), np.uint8) for h in self.host]
        self.dev_scales = [fdx.DevBuf.from_host(s) for s in self.scales]

    def call(self, table, lens, parents, grow, max_len, free_pages=True):
        fdx, (n, width) = self.fdx, table.shape
        ints = lambda a: fdx.DevBuf.from_host(np.asarray(a, np.int32), np.int32)
        at = [type("At", (), dict(ptr=ctypes.c_void_p(d.ptr.value + self.odd))) for d in self.dev]
        dt, dl, dp, dg = ints(table), ints(lens), ints(parents), None if grow is None else ints(grow)
        args = (*at, self.kind, self.n_pages, self.page, self.kv, self.dk, self.dv, dt, width, dl, n, max_len)
        c = fdx.KvPages8(*args, *self.dev_scales, self.block) if self.block else fdx.KvPages(*args)
        call, need = (fdx.lib.fdx_kv8_fork, fdx.lib.fdx_kv8_fork_scratch_bytes) if self.block else (fdx.lib.fdx_kv_fork, fdx.lib.fdx_kv_fork_scratch_bytes)
        size = need(ctypes.byref(c))
        new_table, new_lens, free, flag = ints(np.full((n, width), 77)), ints(np.full(n, 77)), ints([77]), ints([0])
        scratch = fdx.DevBuf.from_host(np.random.default_rng(1).integers(0, 256, size + 16).astype(np.uint8), np.uint8)
        behind = scratch.to_host((size + 16,), np.uint8)[size:].copy()
        fdx.check(call(ctypes.byref(c), dp.ptr, dg and dg.ptr, new_table.ptr, new_lens.ptr, free.ptr if free_pages else None, scratch.ptr, flag.ptr))
        fdx.sync()
        assert np.array_equal(scratch.to_host((size + 16,), np.uint8)[size:], behind)
        assert np.array_equal(dt.to_host((n, width), np.int32), table) and np.array_equal(dl.to_host((n,), np.int32), lens)
        return new_table.to_host((n, width), np.int32), new_lens.to_host((n,), np.int32), int(free.to_host((1,), np.int32)[0]), int(flag.to_host((1,), np.int32)[0])

    def step(self, table, lens, parents, grow, max_len):
        table, lens = np.asarray(table, np.int32), np.asarray(lens, np.int32)
        want, want_lens, copies, left, error = fork(table, lens, parents, grow, self.n_pages, self.page, max_len)
        got, got_lens, free, flag = self.call(table, lens, parents, grow, max_len)
        assert np.array_equal(got_lens, want_lens), (got_lens, want_lens)
        assert np.array_equal(got, want), (got, want)
        assert free == left and flag == int(error), (free, left, flag, error)
        sources = [h.copy() for h in self.host], [s.copy() for s in self.scales]
        for a, b, rows in copies:
            for h, was in zip(self.host, sources[0]):
                h[b, :rows] = was[a, :rows]
            for s, was in zip(self.scales, sources[1]):
                s[b, :-(-rows // self.block)] = was[a, :-(-rows // self.block)]
        for h, d in zip(self.host, self.dev):
            assert np.array_equal(d.to_host((self.odd + h.size,), np.uint8)[self.odd:], h.ravel())
        for s, d in zip(self.scales, self.dev_scales):
            assert np.array_equal(d.to_host(s.shape), s)
        return got, got_lens


def beams(r, groups, beams, longest, page, spare):
    """a table whose groups share the full pages of a prompt, in a shuffled cache; (table, lens, n_pages)"""
    lens = np.repeat(r.integers(0, longest + 1, groups), beams)
    width = longest // page + 2
    table, at = np.full((len(lens), width), -1, np.int32), 0
    for g in range(groups):
        shared = int(r.integers(0, lens[g * beams] // page + 1))
        for b in range(beams):
            i = g * beams + b
            for j in range(-(-int(lens[i]) // page)):
                if j < shared and b > 0:
                    table[i, j] = table[g * beams, j]
                else:
                    table[i, j] = at
                    at += 1
    n_pages = at + spare
    order = r.permutation(n_pages).astype(np.int32)
    return np.where(table >= 0, order[table], -1), lens.astype(np.int32), n_pages


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("groups,width,longest,page,kv,dk,dv", [
    (1, 4, 60, 16, 2, 64, 64), (1, 1, 5, 3, 1, 13, 7), (7, 3, 40, 8, 3, 20, 12), (64, 8, 200, 16, 1, 32, 32), (3, 16, 300, 64, 8, 128, 128), (1, 2, 0, 4, 1, 4, 4),
    (150, 9, 30, 4, 1, 8, 8), (5, 5, 100, 1, 2, 4, 12)])
def test_fork(fdx, groups, width, longest, page, kv, dk, dv, kind):
    """Several steps behind one another, each from the table of the one before."""
    r = np.random.default_rng(groups + page)
    table, lens, n_pages = beams(r, groups, width, longest, page, 3 * groups * width + 5)
    max_len = table.shape[1] * page
    p = Pages(fdx, kind, n_pages, page, kv, dk, dv, 0 if kind in ("f32", "bf16") else {16: 8, 64: 16, 8: 8}.get(page, 1))
    n = groups * width
    for step in range(4):
        parents = np.arange(n) // width * width + r.integers(0, width, n)
        parents[r.random(n) < 0.1] = -1
        grow = [None, np.ones(n), r.integers(0, 4, n), np.zeros(n)][step]
        if grow is not None:
            grow = np.where(np.where(parents >= 0, lens[parents], 0) + grow > max_len, 0, grow).astype(np.int32)
        print("fork", kind, groups, width, longest, page, step, flush=True)
        table, lens = p.step(table, lens, parents.astype(np.int32), grow, max_len)


@pytest.mark.parametrize("kind,odd", [("f32", 4), ("bf16", 2), ("i8", 1), ("e4m3", 8), ("i8", 16)])
def test_fork_alignment(fdx, kind, odd):
    r = np.random.default_rng(3)
    table, lens, n_pages = beams(r, 3, 4, 50, 8, 40)
    p = Pages(fdx, kind, n_pages, 8, 3, 16, 24, 0 if kind in ("f32", "bf16") else 2, odd=odd)
    p.step(table, lens, r.integers(0, 12, 12), None, table.shape[1] * 8)


def test_fork_of_any_parents(fdx):
    """Sequences that go on from others of any length, shared last pages, and full pages of one that are another's last."""
    r = np.random.default_rng(4)
    for trial in range(20):
        page, n, width, n_pages = int(r.integers(1, 7)), int(r.integers(1, 30)), 6, 60
        table = r.integers(0, n_pages if trial % 2 else 12, (n, width)).astype(np.int32)   # many share pages anyhow
        lens = r.integers(0, width * page + 1, n).astype(np.int32)
        parents, grow = r.integers(-1, n, n).astype(np.int32), r.integers(0, 3, n).astype(np.int32)
        grow = np.where(np.where(parents >= 0, lens[parents], 0) + grow > width * page, 0, grow).astype(np.int32)
        print("fork any", trial, page, n, flush=True)
        Pages(fdx, "f32", n_pages + 4 * n * (trial % 3), page, 1, 4, 8, 0, seed=trial).step(table, lens, parents, grow, width * page)


def test_fork_reports(fdx):
    """Parents, lengths, growth and pages that are none, and a lack of pages: as documented, nothing outside the cache is touched."""
    table, lens = np.array([[0, 1, -1], [2, 3, -1], [4, -1, -1]], np.int32), np.array([6, 7, 2], np.int32)
    big, low = 2**31 - 1, -2**31
    for parents, grow, change in (([3, 0, 1], None, None), ([big, 0, 1], None, None), ([low, 0, 1], None, None), ([-1, -1, -1], [1, 1, 1], None),
                                  ([0, 1, 2], [-1, 1, 1], None), ([0, 1, 2], [7, 5, 1], None), ([0, 1, 2], [big, low, 10], None),
                                  ([0, 0, 1], None, dict(lens=[13, 7, 2])), ([0, 0, 1], None, dict(lens=[big, -1, low])),
                                  ([0, 0, 1], [1, 1, 1], dict(entry=(0, 0, -1))), ([0, 0, 1], [3, 3, 3], dict(entry=(0, 1, 9))),
                                  ([0, 0, 1], [3, 3, 3], dict(entry=(0, 1, big))), ([1, 1, 1], [5, 5, 5], dict(n_pages=5)), ([0, 0, 0], None, dict(n_pages=3))):
        t, ls, n_pages = table.copy(), lens.copy(), 9
        for key, value in (change or {}).items():
            if key == "lens":
                ls = np.array(value, np.int32)
            elif key == "entry":
                t[value[0], value[1]] = value[2]
            else:
                n_pages = value
                t[t >= n_pages] = 0
        print("fork reports", parents, grow, change, flush=True)
        Pages(fdx, "i8", n_pages, 4, 2, 8, 8, 2).step(t, ls, np.array(parents), None if grow is None else np.array(grow), 12)


@pytest.mark.parametrize("n_pages,n,width", [(31, 1, 4), (32, 2, 4), (33, 3, 4), (1000, 5, 100), (40_000, 1100, 20), (700_000, 40, 3000), (3_000_000, 3, 7)])
def test_fork_sizes(fdx, n_pages, n, width):
    """Numbers of pages beside the words of bits that stand for them, more sequences than a workgroup has threads, long tables, large caches."""
    r = np.random.default_rng(n)
    page = 2
    table = r.permutation(n_pages)[:n * width].reshape(n, width) if n * width <= n_pages else r.integers(0, n_pages, (n, width))
    lens = r.integers(0, (width - 1) * page, n).astype(np.int32)
    print("fork sizes", n_pages, n, width, flush=True)
    p = Pages(fdx, "i8", n_pages, page, 1, 4, 4, 1)
    for _ in range(2):
        table, lens = p.step(table.astype(np.int32), lens, r.integers(-1, n, n).astype(np.int32), np.ones(n, np.int32), width * page)


def test_fork_of_wide_tables(fdx):
    """Entries of the table whose positions would be beyond 32 bits: nobody has a page there."""
    page, width = 1 << 20, 4100
    table = np.full((3, width), -1)
    table[0, 0], table[1, 0], table[2, 0] = 1, 3, 4
    for more in (4095, 4096, 4097):
        table[:, more] = 2   # what it holds there is nothing to anyone
    for n in (1, 3):
        p = Pages(fdx, "i8", 6, page, 1, 1, 1, 1 << 10)
        p.step(table[:n], np.array([page - 5, 1 << 10, page])[:n], np.array([0, 0, 2])[:n] % n, np.array([5, 0, 0])[:n], page)


def test_release_after_a_fork(fdx):
    """Pages that sequences share stay theirs when one of them ends."""
    r = np.random.default_rng(8)
    kv, d, heads = 2, 16, 4
    c = fdx.PagedCache(8, 4, kv, d, d, 3, 24, "e4m3")
    k, v = (r.standard_normal((10, kv * d)).astype(np.float32) for _ in range(2))
    fdx.kv_append(c, k, v, [10, 0, 0])
    q = r.standard_normal((1, heads * d)).astype(np.float32)
    want = fdx.mha_paged(c, q, [1, 0, 0], heads)
    fdx.kv_fork(c, [0, 0, -1])
    c.release(0)
    assert len(set(c.free)) == len(c.free) == 5 and not set(c.free) & set(c.table.ravel().tolist())
    fdx.kv_append(c, np.ones((20, kv * d), np.float32), np.ones((20, kv * d), np.float32), [0, 0, 20])
    assert np.array_equal(fdx.mha_paged(c, q, [0, 1, 0], heads), want)


def test_python_fork(fdx):
    """kv_fork on a PagedCache: appended tokens go to each sequence's own pages, and attention sees what its ancestors wrote."""
    r = np.random.default_rng(6)
    for kind in KINDS:
        n, kv, d, heads = 4, 2, 16, 4
        c = fdx.PagedCache(30, 4, kv, d, d, n, 24, kind)
        rows = [[] for _ in range(n)]

        def add(new):
            k, v = (r.integers(-127, 128, (sum(new), kv * d)).astype(np.float32) for _ in range(2))
            k[:, ::d] = v[:, ::d] = 127   # codes of i8 are exact; bf16 holds them too
            if kind == "e4m3":
                k, v = np.sign(k), np.sign(v)
            fdx.kv_append(c, k, v, new)
            for s, at in zip(range(n), np.cumsum([0] + list(new))):
                rows[s] = rows[s] + [(k[at + j], v[at + j]) for j in range(new[s])]
        add([6, 9, 4, 1])
        for parents in ([1, 1, 0, 3], [0, 0, 0, 0], [3, -1, 2, 1], [0, 2, 2, 3]):
            fdx.kv_fork(c, parents)
            rows = [list(rows[p]) if p >= 0 else [] for p in parents]
            assert c.lens.tolist() == [len(x) for x in rows]
            assert sorted(set(c.table.ravel().tolist()) - {-1}) + sorted(c.free) == sorted(set(range(30)) - set(c.free)) + sorted(c.free)
            add([1, 2, 1, 0])
            new = [min(1, len(x)) for x in rows]
            q = 0.01 * r.standard_normal((sum(new), heads * d)).astype(np.float32)
            got, at = fdx.mha_paged(c, q, new, heads), 0
            for s in range(n):
                if not new[s]:
                    continue
                k, v = (np.array([x[w] for x in rows[s]], np.float64).reshape(-1, kv, d) for w in (0, 1))
                for h in range(heads):
                    x = k[:, h // 2] @ q[at].reshape(heads, d)[h].astype(np.float64) / np.sqrt(d)
                    e = np.exp(x - x.max())
                    want = e / e.sum() @ v[:, h // 2]
                    assert np.abs(got[at].reshape(heads, d)[h] - want).max() <= 1e-5 * np.abs(want).max(), (kind, parents, s, h)
                at += 1
    with pytest.raises(fdx.FdxError, match="free pages"):
        c = fdx.PagedCache(3, 4, 1, 4, 4, 3, 8)
        fdx.kv_append(c, np.zeros((6, 4), np.float32), np.zeros((6, 4), np.float32), [6, 0, 0])
        fdx.kv_fork(c, [0, 0, 0])
    assert c.lens.tolist() == [6, 0, 0] and len(c.free) == 1


@pytest.mark.parametrize("n,width", [(1024, 63), (1024, 64), (1024, 65), (512, 128), (513, 128), (512, 256), (1, 65536), (1, 65537)])
def test_fork_of_tables_beside_the_border_of_its_forms(fdx, n, width):
    """Tables of 64 512 to 131 072 entries, the most that one workgroup walks (65 536) among them; sequences of any length in them."""
    r = np.random.default_rng(width)
    page = 4
    lens = r.integers(0, np.where(r.random(n) < 0.9, min(width, 12), width) * page - 1).astype(np.int32)
    counts = -(-lens.astype(np.int64) // page)
    total = int(counts.sum())
    order, at = r.permutation(total + 3 * n + 5), np.cumsum(counts) - counts
    table = np.full((n, width), -1, np.int32)
    for i in range(n):
        table[i, :counts[i]] = order[at[i]:at[i] + counts[i]]
    p = Pages(fdx, "i8", len(order), page, 1, 4, 4, 2)
    print("fork border", n, width, len(order), flush=True)
    for _ in range(2):
        table, lens = p.step(table, lens, r.integers(-1, n, n).astype(np.int32), np.ones(n, np.int32), width * page)
