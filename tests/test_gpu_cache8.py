"""The cache in 8 bits: its codes and scales against their definition, bit for bit, and attention over them against plain sums in 64 bits
of the values that the codes stand for.

Bounds of attention.  Codes are exact; a query is held to 22 bits or more, so a product of a score is off by at most 2^-22 of its size, and sums in
fp32 add 2^-24 a step.  With independent signs a score of dk products of unit operands is off by about (0.64 * 2^-22 + 2^-24) sqrt(dk) / sqrt(dk) =
2e-7 absolute, which is the relative error of a probability.  Scores k times larger carry k times the error.  The tokens here differ in size by
e^(0.5 z), z normal: of 5000 keys the largest, which draw the weight and leave little to average over, are e^(0.5 * 4.1) = 8 times as large, so 1.6e-6;
exponentials and the second sum add 2e-7 each: 2e-6 in the 2-norm, and ten times that of the largest value for any single output."""
import ctypes

import numpy as np
import pytest

from cache8 import HostCache, decode, encode

pytestmark = pytest.mark.gpu
KINDS = ["i8", "e4m3"]
I64 = ctypes.c_int64


def attend(q, k, v, heads, kv_heads, sees):
    """q [n][heads*dk], k [keys][kv*dk], v [keys][kv*dv]; query i sees the keys that sees[i] marks, or the first sees[i]; in 64 bits"""
    n, keys = q.shape[0], k.shape[0]
    q = q.astype(np.float64).reshape(n, heads, q.shape[1] // heads)
    k, v = (a.reshape(keys, kv_heads, a.shape[1] // kv_heads) for a in (k, v))
    out = np.zeros((n, heads, v.shape[2]))
    for h in range(heads):
        kh, vh = k[:, h * kv_heads // heads], v[:, h * kv_heads // heads]
        with np.errstate(all="ignore"):
            x = q[:, h] @ kh.T / np.sqrt(q.shape[2])
            for i in range(n):
                seen = np.arange(keys) < sees[i] if np.ndim(sees[i]) == 0 else sees[i]
                if seen.any():
                    e = np.exp(x[i, seen] - x[i, seen].max())
                    out[i, h] = e / e.sum() @ vh[seen]
    return out.reshape(n, heads * v.shape[2])


def close(got, want, bound=2e-6):
    assert np.array_equal(np.isnan(got), np.isnan(want))
    got, want = got[~np.isnan(want)], want[~np.isnan(want)]
    if want.size == 0:
        return
    err, worst = np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-30), np.abs(got - want).max() / max(np.abs(want).max(), 1e-30)
    print("relative error %.2e, largest %.2e" % (err, worst), flush=True)
    assert err <= bound and worst <= 10 * bound, (err, worst)


class Filled:
    """A cache and its copy on the host, filled in steps; pages come in a shuffled order."""

    def __init__(self, fdx, context, kv, dk, dv, page, kind, block=None, steps=1, seed=0, change=None, spread=0.5):
        r = np.random.default_rng(seed)
        n_pages, width = sum(-(-n // page) for n in context) + 4, max(max(context), 1)
        self.fdx, self.page = fdx, page
        self.cache = fdx.PagedCache(n_pages, page, kv, dk, dv, len(context), width, kind, block)
        r.shuffle(self.cache.free)
        self.host = HostCache(n_pages, page, kv, dk, dv, kind, self.cache.block)
        left = np.array(context)
        for step in range(steps):
            new = left if step == steps - 1 else np.array([r.integers(0, n + 1) for n in left])
            left = left - new
            self.append(r, new, change, spread)

    def row_of(self, s):
        table = self.cache.table
        return lambda pos: int(table[s][pos // self.page]) * self.page + pos % self.page

    def append(self, r, new, change=None, spread=0.5):
        c, total = self.cache, int(np.sum(new))
        size = np.exp(spread * r.standard_normal((total, 1)))
        k, v = ((r.standard_normal((total, c.kv_heads * d)) * size).astype(np.float32) for d in (c.dk, c.dv))
        if change:
            change(k, v)
        first = c.lens.copy()
        self.fdx.kv_append(c, k, v, new)
        at = 0
        for s, n in enumerate(new):
            for which, x in enumerate((k, v)):
                self.host.append(self.row_of(s), int(first[s]), x[at:at + n].reshape(n, c.kv_heads, x.shape[1] // c.kv_heads), which)
            at += n

    def rows(self, s, length=None):
        return [self.row_of(s)(p) for p in range(self.cache.lens[s] if length is None else length)]

    def reference(self, q, new, heads):
        out, at = [], 0
        for s, n in enumerate(new):
            length, rows = int(self.cache.lens[s]), self.rows(s)
            out.append(attend(q[at:at + n], self.host.values(rows, 0), self.host.values(rows, 1), heads, self.cache.kv_heads,
                              np.arange(length - n, length) + 1))
            at += n
        return np.concatenate(out)

    def check(self):
        same(self.cache, self.host)


def same(cache, host):
    """every byte of the device's cache is the host's, and every scale"""
    for which, (codes, scales) in enumerate(((cache.k, cache.k_scale), (cache.v, cache.v_scale))):
        got = codes.to_host(host.codes[which].shape, np.uint8)
        assert np.array_equal(got, host.codes[which]), (which, np.argwhere(got != host.codes[which])[:5])
        got = scales.to_host(host.scales[which].shape)
        assert np.array_equal(got, host.scales[which], equal_nan=True), (which, np.argwhere(got != host.scales[which])[:5])


# ---------------------------------------------------------------- new tokens

SHAPES = [(2, 64, 64, 16, 16), (3, 128, 128, 20, 5), (1, 80, 80, 64, 32), (2, 13, 7, 3, 3), (2, 96, 64, 8, 1), (1, 32, 128, 200, 40), (2, 61, 45, 12, 4),
          (1, 300, 260, 6, 2), (12, 64, 64, 16, 16), (1, 4, 4, 128, 128), (1, 128, 128, 96, 96), (2, 128, 128, 64, 64), (1, 128, 64, 130, 65),
          (3, 128, 128, 40, 1), (1, 8, 8, 70, 1), (2, 100, 36, 24, 12)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("kv,dk,dv,page,block", SHAPES)
def test_append(fdx, kv, dk, dv, page, block, kind):
    """Prompts, pieces and single tokens: blocks are started, filled and their scales grow; other places of the cache stay as they are."""
    print("append8", kv, dk, dv, page, block, kind, flush=True)
    f = Filled(fdx, [1, 0, 77, 16, 130], kv, dk, dv, page, kind, block, steps=4, seed=dk)
    f.check()
    f.cache.max_len += 3 * page
    f.cache.table = np.concatenate([f.cache.table, np.full((5, 4), -1, np.int32)], 1)
    f.cache.max_len = min(f.cache.max_len, f.cache.table.shape[1] * page)
    r = np.random.default_rng(1)
    for _ in range(3):   # tokens one at a time
        new = r.integers(0, 2, 5)
        if sum(max(0, -(-int(a + b) // page) - int((t >= 0).sum())) for a, b, t in zip(f.cache.lens, new, f.cache.table)) <= len(f.cache.free):
            f.append(r, new)
            f.check()


@pytest.mark.parametrize("kind", KINDS)
def test_append_rounds(fdx, kind):
    """Values on and beside the middle between two codes, zeros, the largest and the smallest numbers."""
    base = [0.5, 1.5, 2.5, -0.5, -1.5, 126.5, 127, 0, -0.0, 1e-30, 2.0 ** -126, 3, 17, 18, 19, 20, 240, 248, 30.5, 0.0009765625, 0.0029296875, 0.001]
    base = np.array(base + [np.nextafter(np.float32(x), np.float32(9e9)) for x in base] + [np.nextafter(np.float32(x), np.float32(-9e9)) for x in base], np.float32)
    r = np.random.default_rng(0)
    many = np.concatenate([base, np.float32(448) * r.uniform(-1, 1, 62).astype(np.float32)])
    for most, by in ((448, 1), (127, 1), (448, 2.0 ** -120), (448, 7e35), (127, 2.6e36), (448, 1e-44), (0, 1), (1, 2.0 ** -149), (3.4e38, 1)):
        x = np.clip(many, -most, most).astype(np.float32) * np.float32(by)
        x[-1] = np.float32(min(most * float(by), 3.4e38))
        c = fdx.PagedCache(1, 1, 1, len(x), len(x), 1, 1, kind)
        host = HostCache(1, 1, 1, len(x), len(x), kind, 1)
        print("rounds", kind, most, by, flush=True)
        fdx.kv_append(c, x[None], -x[None], [1])
        for which, y in enumerate((x, -x)):
            host.append(lambda p: 0, 0, y[None, None], which)
        same(c, host)


def test_codes_of_e4m3(fdx):
    """Every code is reached from its own value, and nothing else."""
    codes = np.array([c for c in range(256) if c & 127 != 127], np.uint8)
    x = decode(codes, "e4m3")
    assert np.array_equal(encode(x, "e4m3"), codes)
    c = fdx.PagedCache(1, 1, 1, len(x), len(x), 1, 1, "e4m3")
    fdx.kv_append(c, x[None], x[None], [1])
    assert c.k_scale.to_host((1,))[0] == 1 and np.array_equal(c.k.to_host((len(x),), np.uint8), codes)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
def test_append_of_infinities_and_nan(fdx, what, kind):
    """They make their block and head NaN, also for tokens of earlier calls, until it is started anew; other heads and blocks stay as they are."""
    for steps in (1, 5):
        def change(k, v):
            if len(k) > 6:
                k[5, 3], v[6, 20] = what, what
        f = Filled(fdx, [30, 21], 2, 16, 16, 8, kind, 4, steps=steps, change=change)
        f.check()
        assert sum(np.isnan(s).sum() for s in f.host.scales) > 0
        f.cache.max_len = 32
        f.append(np.random.default_rng(1), [2, 3])
        f.check()
        for s in (0, 1):
            f.cache.release(s)
        f.append(np.random.default_rng(2), [30, 32])
        f.check()
        assert all(np.isfinite(s[[f.row_of(q)(p) // 4 for q in (0, 1) for p in range(28)]]).all() for s in f.host.scales)


def call_append(fdx, pages, k, ldk, v, ldv, starts, tokens):
    d_starts, flag = fdx.DevBuf.from_host(np.asarray(starts, np.int32), np.int32), fdx.DevBuf.from_host(np.zeros(1, np.int32), np.int32)
    fdx.check(fdx.lib.fdx_kv8_append_f32(k, I64(ldk), v, I64(ldv), d_starts.ptr, tokens, ctypes.byref(pages), flag.ptr))
    return int(flag.to_host((1,), np.int32)[0])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shift,pad", [(0, 4), (1, 0), (0, 3), (3, 1)])
def test_append_strides_and_alignment(fdx, shift, pad, kind):
    kv, d, page, block = 3, 32, 8, 4
    lens, new = [21, 9], [13, 9]
    r = np.random.default_rng(5)
    x = r.standard_normal((2 + 22 + 1, kv * d + pad)).astype(np.float32)
    dx = fdx.DevBuf.from_host(np.concatenate([np.zeros(shift, np.float32), x.ravel()]))
    c, host = fdx.PagedCache(8, page, kv, d, d, 2, 32, kind, block), HostCache(8, page, kv, d, d, kind, block)
    c.table[:, :3], c.lens = [[4, 1, 0], [7, 2, -1]], np.array(lens, np.int32)
    at = ctypes.c_void_p(dx.ptr.value + 4 * shift)
    print("append8 strides", shift, pad, kind, flush=True)
    assert call_append(fdx, c.pages(), at, kv * d + pad, at, kv * d + pad, [2, 15, 24], 25) == 0
    for s, first in ((0, 2), (1, 15)):
        for which in (0, 1):
            host.append(lambda p: int(c.table[s][p // page]) * page + p % page, lens[s] - new[s], x[first:first + new[s], :kv * d].reshape(new[s], kv, d), which)
    same(c, host)


def test_append_outside_the_cache(fdx):
    """Positions below zero, from max_len on and of pages that are none: not written, reported; the others are."""
    kv, d, page, block = 1, 8, 4, 2
    x = np.random.default_rng(1).standard_normal((6, 8)).astype(np.float32)
    for lens, table, want in (([2, 3], [[0, 1], [2, 3]], [(0, 0, 1, 2), (1, 0, 3, 3)]),       # (sequence, first position, row of x, rows)
                              ([9, 3], [[0, 1], [2, 3]], [(0, 6, 0, 2), (1, 0, 3, 3)]),
                              ([3, 5], [[0, 1], [2, 9]], [(0, 0, 0, 3), (1, 2, 3, 2)]),
                              ([3, 3], [[-1, 1], [2, 3]], [(1, 0, 3, 3)]),
                              ([-2**31, 2**31 - 1], [[0, 1], [2, 3]], []), ([2, 4], [[2**31 - 1, 1], [-2**31, 3]], [])):
        c, host = fdx.PagedCache(4, page, kv, d, d, 2, 8, "i8", block), HostCache(4, page, kv, d, d, "i8", block)
        c.table, c.lens = np.array(table, np.int32), np.array(lens, np.int32)
        dx = fdx.DevBuf.from_host(x)
        print("append8 outside", lens, table, flush=True)
        assert call_append(fdx, c.pages(), dx.ptr, 8, dx.ptr, 8, [0, 3, 6], 6) == 1
        for s, first, row, n in want:
            for which in (0, 1):
                host.append(lambda p: int(c.table[s][p // page]) * page + p % page, first, x[row:row + n].reshape(n, 1, 8), which)
        same(c, host)
    for starts in ([0, 2**31 - 1, 6], [-5, 2, 6], [3, 0, 6], [0, 3, -2**31]):
        c = fdx.PagedCache(4, page, kv, d, d, 2, 8, "i8", block)
        c.table, c.lens = np.array([[0, 1], [2, 3]], np.int32), np.array([8, 8], np.int32)
        dx = fdx.DevBuf.from_host(x)
        print("append8 starts", starts, flush=True)
        assert call_append(fdx, c.pages(), dx.ptr, 8, dx.ptr, 8, starts, 6) == 1


@pytest.mark.parametrize("n_seqs", [63, 64, 65, 300])
def test_many_sequences(fdx, n_seqs):
    r = np.random.default_rng(n_seqs)
    context = r.integers(0, 40, n_seqs)
    f = Filled(fdx, context.tolist(), 2, 16, 16, 8, "i8", 4, steps=3)
    f.check()
    new = [min(int(n), int(r.integers(0, 3))) for n in context]
    q = r.standard_normal((sum(new), 4 * 16)).astype(np.float32)
    close(fdx.mha_paged(f.cache, q, new, 4), f.reference(q, new, 4))


# ---------------------------------------------------------------- attention

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("context,new,heads,kv,dk,dv,page,block", [
    ([1], [1], 1, 1, 64, 64, 16, 16), ([201], [1], 12, 12, 64, 64, 16, 16), ([5, 300, 64, 17], [1, 1, 1, 1], 8, 2, 64, 64, 16, 4),
    ([700, 33, 1], [1, 1, 1], 32, 8, 128, 128, 16, 16), ([100, 260, 31], [1, 0, 1], 16, 1, 128, 128, 7, 7), ([100, 50], [1, 1], 32, 1, 64, 64, 32, 1),
    ([130, 90], [1, 1], 10, 5, 80, 80, 13, 1), ([60, 61, 62], [1, 1, 1], 6, 2, 13, 7, 3, 3), ([90], [1], 40, 1, 64, 64, 16, 8),
    ([70], [1], 4, 2, 96, 64, 1, 1), ([200, 77, 16], [3, 5, 16], 4, 4, 64, 64, 16, 16), ([400, 90, 2], [7, 1, 2], 8, 2, 128, 128, 16, 2),
    ([300, 200], [40, 1], 8, 2, 64, 64, 16, 16), ([500, 129, 40, 3], [129, 129, 1, 3], 8, 2, 64, 64, 24, 6), ([450, 260], [300, 17], 7, 1, 128, 128, 64, 32),
    ([140], [140], 3, 3, 32, 32, 200, 50), ([77, 190], [60, 33], 5, 1, 33, 127, 11, 11), ([2100, 1900], [1, 2], 4, 1, 64, 64, 16, 16),
    ([2300, 5, 1030], [70, 5, 1], 4, 2, 128, 128, 32, 32), ([300, 40], [20, 3], 9, 3, 61, 45, 20, 5), ([90, 700], [1, 1], 4, 2, 8, 16, 16, 16),
    ([260, 33], [33, 2], 32, 8, 128, 128, 16, 16), ([200], [35], 4, 4, 112, 72, 16, 16)])
def test_paged(fdx, context, new, heads, kv, dk, dv, page, block, kind):
    print("paged8", context, new, heads, kv, dk, dv, page, block, kind, flush=True)
    f = Filled(fdx, context, kv, dk, dv, page, kind, block, steps=2, seed=sum(context))
    f.check()
    q = np.random.default_rng(dk).standard_normal((sum(new), heads * dk)).astype(np.float32)
    close(fdx.mha_paged(f.cache, q, new, heads), f.reference(q, new, heads))


def call_paged(fdx, cache, q, ldq, starts, tokens, max_new, heads, out, ldo, **change):
    c = cache.pages()
    kept = []
    for key, value in change.items():
        if key in ("table", "lens"):
            kept.append(fdx.DevBuf.from_host(value, np.int32))
            value = kept[-1].ptr
        setattr(c.pages, key, value)
    d_starts, flag = fdx.DevBuf.from_host(np.asarray(starts, np.int32), np.int32), fdx.DevBuf.from_host(np.zeros(1, np.int32), np.int32)
    need = fdx.lib.fdx_mha_paged8_scratch_bytes(tokens, max_new, heads, ctypes.byref(c))
    scratch = fdx.DevBuf.from_host(np.full(need + 16, 0xff, np.uint8), np.uint8)   # NaN
    fdx.check(fdx.lib.fdx_mha_paged8_f32(q, I64(ldq), d_starts.ptr, tokens, max_new, heads, ctypes.byref(c), out, I64(ldo), scratch.ptr, flag.ptr))
    fdx.sync()
    assert (scratch.to_host((need + 16,), np.uint8)[need:] == 0xff).all()
    return int(flag.to_host((1,), np.int32)[0])


@pytest.mark.parametrize("new", [[1, 1, 1], [3, 1, 2], [40, 9, 70]])
def test_paged_tokens_that_see_nothing(fdx, new):
    """More new tokens than positions: the first ones see none and get zeros, none of it is an error."""
    f = Filled(fdx, [50, 2, 30], 2, 64, 64, 16, "i8", 4)
    lens = np.array([50, 0, min(30, new[2])], np.int32) if new[0] == 1 else np.array([50, 1, 1], np.int32)
    tokens, heads = sum(new), 4
    q = np.random.default_rng(1).standard_normal((tokens, heads * 64)).astype(np.float32)
    out, dq, starts = fdx.DevBuf.from_host(np.full((tokens, heads * 64), 9, np.float32)), fdx.DevBuf.from_host(q), np.concatenate([[0], np.cumsum(new)])
    print("paged8 empty", new, lens, flush=True)
    flag = call_paged(fdx, f.cache, dq.ptr, heads * 64, starts, tokens, max(new), heads, out.ptr, heads * 64, lens=lens)
    got = out.to_host((tokens, heads * 64))
    want = np.concatenate([attend(q[starts[s]:starts[s + 1]], f.host.values(f.rows(s), 0), f.host.values(f.rows(s), 1), heads, 2,
                                  np.arange(lens[s] - n, lens[s]) + 1) for s, n in enumerate(new)])
    assert flag == 0
    close(got, want)
    assert (got[want == 0] == 0).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shift,pad", [(0, 4), (1, 0), (0, 3)])
@pytest.mark.parametrize("new", [[1, 1], [2, 30]])
def test_paged_strides_and_alignment(fdx, shift, pad, kind, new):
    heads, kv, d = 4, 2, 64
    f = Filled(fdx, [90, 131], kv, d, d, 16, kind, 8)
    tokens = 2 + sum(new) + 3
    ld = heads * d + pad
    x = np.random.default_rng(4).standard_normal((tokens, ld)).astype(np.float32)
    dq, out = fdx.DevBuf.from_host(np.concatenate([np.zeros(shift, np.float32), x.ravel()])), fdx.DevBuf.from_host(np.full(shift + tokens * ld, 7, np.float32))
    at = lambda b: ctypes.c_void_p(b.ptr.value + 4 * shift)
    print("paged8 strides", shift, pad, kind, new, flush=True)
    assert call_paged(fdx, f.cache, at(dq), ld, [2, 2 + new[0], 2 + sum(new)], tokens, max(new), heads, at(out), ld) == 0
    got = out.to_host((shift + tokens * ld,))[shift:].reshape(tokens, ld)
    close(got[2:-3, :heads * d], f.reference(x[2:-3, :heads * d], new, heads))
    assert (got[:2] == 7).all() and (got[-3:] == 7).all() and (got[:, heads * d:] == 7).all()


@pytest.mark.parametrize("new", [[1, 1], [4, 3], [60, 9]])
def test_paged_pages_that_are_none(fdx, new):
    """Positions of pages that the cache does not have are left out and reported; so are lengths and tokens beyond what was said."""
    heads, kv, d, page = 4, 2, 64, 16
    f = Filled(fdx, [90, 131], kv, d, d, page, "i8", 16)
    q = np.random.default_rng(4).standard_normal((sum(new), heads * d)).astype(np.float32)
    dq, starts = fdx.DevBuf.from_host(q), [0, new[0], sum(new)]
    out = fdx.DevBuf.from_host(np.zeros((sum(new) + 50, heads * d), np.float32))
    k0, v0, k1, v1 = (f.host.values(f.rows(s), w) for s in (0, 1) for w in (0, 1))
    for bad in (-1, f.cache.n_pages, 2**31 - 1, -2**31):
        table = f.cache.table.copy()
        table[1, 2] = bad
        print("paged8 bad page", new, bad, flush=True)
        assert call_paged(fdx, f.cache, dq.ptr, heads * d, starts, sum(new), max(new), heads, out.ptr, heads * d, table=table) == 1
        got = out.to_host((sum(new), heads * d))
        keep = np.r_[0:32, 48:131]
        close(got[new[0]:], attend(q[new[0]:], k1[keep], v1[keep], heads, kv, [keep < 131 - new[1] + j + 1 for j in range(new[1])]))
        close(got[:new[0]], attend(q[:new[0]], k0, v0, heads, kv, np.arange(90 - new[0], 90) + 1))
    table = np.full_like(f.cache.table, -1)
    assert call_paged(fdx, f.cache, dq.ptr, heads * d, starts, sum(new), max(new), heads, out.ptr, heads * d, table=table) == 1
    assert (out.to_host((sum(new), heads * d)) == 0).all()
    for lens, flag in (([90, 132], 1), ([90, 2**31 - 1], 1), ([-1, 131], 1), ([-2**31, 131], 1), ([90, 131], 0)):
        print("paged8 lens", lens, flush=True)
        assert call_paged(fdx, f.cache, dq.ptr, heads * d, starts, sum(new), max(new), heads, out.ptr, heads * d, lens=lens) == flag
        got = out.to_host((sum(new), heads * d))
        close(got[new[0]:], attend(q[new[0]:], k1, v1, heads, kv, np.arange(131 - new[1], 131) + 1))
        if lens[0] < 0:
            assert (got[:new[0]] == 0).all()
    for starts in ([0, 2**31 - 1, 5], [-4, 1, sum(new)], [1, 0, 1]):
        print("paged8 starts", starts, flush=True)
        assert call_paged(fdx, f.cache, dq.ptr, heads * d, starts, sum(new), max(new), heads, out.ptr, heads * d) == 1
    assert (out.to_host((sum(new) + 50, heads * d))[sum(new):] == 0).all()


@pytest.mark.parametrize("heads", [4, 40])
def test_lengths_of_sequences_without_new_tokens(fdx, heads):
    """A length out of range is reported though nobody reads it."""
    f = Filled(fdx, [20, 30, 9], 2, 64, 64, 16, "i8", 8)
    q = np.random.default_rng(1).standard_normal((2, heads * 64)).astype(np.float32)
    dq, out = fdx.DevBuf.from_host(q), fdx.DevBuf.from_host(np.zeros((2, heads * 64), np.float32))
    for lens, flag in (([20, 30, 9], 0), ([20, -1, 9], 1), ([20, 31, 9], 1), ([20, 2**31 - 1, 9], 1)):
        assert call_paged(fdx, f.cache, dq.ptr, heads * 64, [0, 1, 1, 2], 2, 1, heads, out.ptr, heads * 64, lens=lens) == flag
        f.cache.lens = np.array([20, 30, 9], np.int32)
        close(out.to_host((2, heads * 64)), f.reference(q, [1, 0, 1], heads))


@pytest.mark.parametrize("n,new", [(40, 1), (130, 2), (40, 35)])
def test_shares_of_the_longest_cache(fdx, n, new):
    """A cache that says 2^30 positions: blocks are counted in sets."""
    page, kv, heads, d, width = 4096, 1, 2, 16, 1 << 18
    r = np.random.default_rng(n)
    context = np.where(r.random(n) < 0.2, r.integers(1000, 4000, n), r.integers(40, 200, n)).tolist()
    f = Filled(fdx, context, kv, d, d, page, "e4m3", 32)
    q = r.standard_normal((n * new, heads * d)).astype(np.float32)
    table = np.full((n, width), -1, np.int32)
    table[:, 0] = f.cache.table[:, 0]
    dq, out = fdx.DevBuf.from_host(q), fdx.DevBuf.from_host(np.zeros((n * new, heads * d), np.float32))
    print("paged8 longest cache", n, new, flush=True)
    assert call_paged(fdx, f.cache, dq.ptr, heads * d, np.arange(n + 1) * new, n * new, new, heads, out.ptr, heads * d, table=table, table_width=width,
                      max_len=1 << 30) == 0
    close(out.to_host((n * new, heads * d)), f.reference(q, [new] * n, heads))


@pytest.mark.parametrize("context,heads,kv", [([190, 150], 8, 8), ([190, 150, 30], 4, 2), ([300, 20], 4, 4), ([384], 4, 4), ([700, 700], 4, 4), ([190, 150], 600, 600)])
@pytest.mark.parametrize("new", [35, 1])
def test_whole_sequences_beside_tiles_in_ranges(fdx, context, heads, kv, new):
    """Tiles whose ranges are joined, and decode steps that nobody shares; a call that says more new tokens than any sequence has."""
    d = 8 if kv > 8 else 128
    f = Filled(fdx, context, kv, d, d, 16, "i8", 8)
    counts = [new] + [1] * (len(context) - 1)
    rows = sum(counts) + (0 if new > 1 else 40)   # rows behind the last sequence
    q = np.random.default_rng(3).standard_normal((rows, heads * d)).astype(np.float32)
    dq, out = fdx.DevBuf.from_host(q), fdx.DevBuf.from_host(np.full((rows, heads * d), 7, np.float32))
    print("paged8 whole sequences", context, heads, kv, new, flush=True)
    assert call_paged(fdx, f.cache, dq.ptr, heads * d, np.cumsum([0] + counts), rows, 35, heads, out.ptr, heads * d) == 0
    got, n = out.to_host((rows, heads * d)), sum(counts)
    close(got[:n], f.reference(q[:n], counts, heads))
    assert (got[n:] == 7).all()


@pytest.mark.parametrize("at", [0, 63, 64, 130, 299])
def test_lengths_out_of_range_among_many(fdx, at):
    n, heads = 300, 4
    f = Filled(fdx, [5] * n, 2, 32, 32, 16, "i8", 8)
    q = np.random.default_rng(1).standard_normal((n, heads * 32)).astype(np.float32)
    dq, out = fdx.DevBuf.from_host(q), fdx.DevBuf.from_host(np.zeros((n, heads * 32), np.float32))
    for bad, new in ((-1, 1), (6, 1), (5, 1), (6, 0)):
        lens = np.full(n, 5)
        lens[at] = bad
        starts = np.minimum(np.arange(n + 1), n) if new else np.arange(n + 1) - (np.arange(n + 1) > at)
        assert call_paged(fdx, f.cache, dq.ptr, heads * 32, starts, n, 1, heads, out.ptr, heads * 32, lens=lens) == (bad != 5), (bad, new)


@pytest.mark.parametrize("n_seqs", [65, 200, 1300, 4200])
@pytest.mark.parametrize("heads,kv", [(4, 2), (6, 6)])
def test_shares_over_many_sequences(fdx, n_seqs, heads, kv):
    """Long sequences beside short ones and ones without tokens, more than a wave has lanes: every key counts once, whoever has it."""
    r = np.random.default_rng(n_seqs)
    context = np.where(r.random(n_seqs) < 0.05, r.integers(500, 2500, n_seqs), r.integers(0, 30, n_seqs))
    f = Filled(fdx, context.tolist(), kv, 32, 32, 16, "i8", 8)
    new = np.where(context > 0, r.integers(0, 3, n_seqs), 0)
    new = np.minimum(new, context)
    q = r.standard_normal((int(new.sum()), heads * 32)).astype(np.float32)
    close(fdx.mha_paged(f.cache, q, new, heads), f.reference(q, new, heads))


def test_paged_more_new_tokens_than_said(fdx):
    f, heads = Filled(fdx, [90, 131], 2, 64, 64, 16, "i8"), 4
    q = np.random.default_rng(4).standard_normal((45, heads * 64)).astype(np.float32)
    dq, out = fdx.DevBuf.from_host(q), fdx.DevBuf.from_host(np.full((45, heads * 64), 5, np.float32))
    assert call_paged(fdx, f.cache, dq.ptr, heads * 64, [0, 5, 45], 45, 5, heads, out.ptr, heads * 64) == 1
    got = out.to_host((45, heads * 64))
    close(got[:5], attend(q[:5], f.host.values(f.rows(0), 0), f.host.values(f.rows(0), 1), heads, 2, np.arange(85, 90) + 1))
    close(got[5:10], attend(q[5:10], f.host.values(f.rows(1), 0), f.host.values(f.rows(1), 1), heads, 2, np.arange(131 - 40, 131 - 35) + 1))
    assert (got[10:] == 5).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [1, 4, 16, 50, 100])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("block,d", [(4, 64), (16, 64), (16, 128)])
def test_paged_blocks_of_nan(fdx, new, which, kind, block, d):
    """A block whose scale is NaN: NaN for the rows that see a token of it (of its key head), nothing for the others, whatever tile they share."""
    heads, kv = 4, 2
    f = Filled(fdx, [150, 40], kv, d, d, 16, kind, block)
    q = np.random.default_rng(2).standard_normal((new + 1, heads * d)).astype(np.float32)
    base = f.reference(q, [new, 1], heads)
    scales = (f.cache.k_scale, f.cache.v_scale)[which]
    for pos in (149, 148, 120, 51, 50, 0):
        changed = f.host.scales[which].copy()
        changed[f.row_of(0)(pos) // block, 1] = np.nan
        buf = fdx.DevBuf.from_host(changed)
        setattr(f.cache, ("k_scale", "v_scale")[which], buf)
        print("paged8 NaN", new, which, kind, pos, flush=True)
        got = fdx.mha_paged(f.cache, q, [new, 1], heads).reshape(new + 1, heads, d)
        hit = np.zeros((new + 1, heads), bool)
        hit[:new, 2:] = (np.arange(150 - new, 150) >= pos // block * block)[:, None]
        assert np.isnan(got[hit]).all()
        close(got[~hit], base.reshape(new + 1, heads, d)[~hit])
    setattr(f.cache, ("k_scale", "v_scale")[which], scales)


@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("new", [1, 5, 60])
def test_paged_queries_of_nan(fdx, new, what):
    heads, kv, d = 4, 2, 64
    f = Filled(fdx, [90, 100], kv, d, d, 16, "i8", 16)
    q = np.random.default_rng(2).standard_normal((new + 1, heads * d)).astype(np.float32)
    base = f.reference(q, [new, 1], heads).reshape(new + 1, heads, d)
    q[new // 2, 64 + 3] = what
    print("paged8 odd query", new, what, flush=True)
    got = fdx.mha_paged(f.cache, q, [new, 1], heads).reshape(new + 1, heads, d)
    assert np.isnan(got[new // 2, 1]).all()
    got[new // 2, 1] = base[new // 2, 1] = 0
    close(got, base)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [[1, 1], [3, 40], [140, 1]])
@pytest.mark.parametrize("eq,ek,ev", [(60, -60, 0), (-60, 60, 0), (-100, 100, 0), (0, 0, 100), (0, 0, -100), (-40, -80, 5), (110, -110, 110), (0, 0, 119), (-110, 98, -118), (-60, -100, 7), (-100, -110, -100)])
@pytest.mark.parametrize("block", [8, 16])
def test_paged_sizes_of_operands(fdx, new, eq, ek, ev, kind, block):
    """Operands far from one in size: the result scales."""
    def change(k, v):
        k *= np.float32(2.0 ** ek)
        v *= np.float32(2.0 ** ev)
    f, heads = Filled(fdx, [200, 141], 2, 64, 64, 16, kind, block, change=change), 4
    q = np.ldexp(np.random.default_rng(5).standard_normal((sum(new), heads * 64)).astype(np.float32), eq).astype(np.float32)
    print("paged8 sizes", new, eq, ek, ev, kind, flush=True)
    got = fdx.mha_paged(f.cache, q, new, heads)
    close(np.ldexp(got.astype(np.float64), -ev), np.ldexp(f.reference(q, new, heads), -ev))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [1, 12, 100])
@pytest.mark.parametrize("spread", [4.0, 12.0])
def test_paged_tokens_of_mixed_sizes(fdx, new, spread, kind):
    """Keys and values whose sizes differ from token to token by e^spread as a standard deviation.  Scores are large where keys are, so keys
    are of one size; a result is then as large as the largest value it averages."""
    def change(k, v):
        k /= np.abs(k).max(1, keepdims=True)
    f, heads = Filled(fdx, [160], 2, 64, 64, 16, kind, 2, change=change, spread=spread), 4
    q = np.random.default_rng(3).standard_normal((new, heads * 64)).astype(np.float32)
    print("paged8 mixed", new, spread, kind, flush=True)
    close(fdx.mha_paged(f.cache, q, [new], heads), f.reference(q, [new], heads))


@pytest.mark.parametrize("new", [1, 12, 100])
def test_paged_one_value_of_many_sizes(fdx, new):
    """Every query has one key's score 200 above all others', whose values are up to 2^60 larger: each result keeps the bound of its own size.
    The tenfold bound of a single output, as its errors do not average."""
    n, d = 160, 64
    power = np.random.default_rng(7).integers(-30, 31, (n, 1))
    places = np.stack([np.arange(n) % d, (np.arange(n) % d + 1 + np.arange(n) // d) % d], 1)   # a pair of depths for each key

    def change(k, v):
        k[:], v[:] = 0, np.ldexp(v / np.abs(v).max(1, keepdims=True), power)
        k[np.arange(n)[:, None], places] = 1
    f = Filled(fdx, [n], 1, d, d, 16, "i8", 1, change=change)
    q = np.zeros((new, d), np.float32)
    q[np.arange(new)[:, None], places[np.random.default_rng(8).integers(0, n - new, new)]] = 1600
    got, want = fdx.mha_paged(f.cache, q, [new], 1), f.reference(q, [new], 1)
    size = np.abs(want).max(1, keepdims=True)
    print("worst row", (np.abs(got - want) / size).max(), flush=True)
    assert (np.abs(got - want) <= 1e-5 * size).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [1, 9, 60, 300])
def test_paged_zeros(fdx, new, kind):
    """Keys or values of zeros: equal weights, zeros."""
    for which in (0, 1):
        def change(k, v):
            (k, v)[which][:] = 0
        f, heads = Filled(fdx, [333], 2, 64, 64, 16, kind, 16, change=change), 4
        q = np.random.default_rng(3).standard_normal((new, heads * 64)).astype(np.float32)
        got = fdx.mha_paged(f.cache, q, [new], heads)
        if which:
            assert (got == 0).all()
        else:
            close(got, f.reference(q, [new], heads))


@pytest.mark.parametrize("new", [1, 4, 60])
def test_paged_scores_of_a_few_hundred(fdx, new):
    """The running maximum moves from tile to tile; scores 40 times larger, errors too.  And scores that climb all the way, then fall."""
    f, heads = Filled(fdx, [333], 2, 64, 64, 16, "i8", 16), 4
    q = 40 * np.random.default_rng(3).standard_normal((new, heads * 64)).astype(np.float32)
    close(fdx.mha_paged(f.cache, q, [new], heads), f.reference(q, [new], heads), 4e-5)
    for sign in (1, -1):
        def climb(k, v):
            k[:] = 0
            k[:, ::64] = sign * np.arange(len(k))[:, None] * 8
        f = Filled(fdx, [333], 2, 64, 64, 16, "i8", 1, change=climb)
        q = np.zeros((new, heads * 64), np.float32)
        q[:, ::64] = 1
        # a score is one product, off by less than 2^-22 * 333 = 8e-5 where it is largest
        close(fdx.mha_paged(f.cache, q, [new], heads), f.reference(q, [new], heads), 8e-5)


@pytest.mark.parametrize("new", [1, 12, 100])
@pytest.mark.parametrize("up", [1, -1])
@pytest.mark.parametrize("block", [2, 16])
def test_paged_jumps_of_scores_and_values(fdx, new, up, block):
    """From one token to another scores rise by thousands and values shrink by 2^180, or the other way round: sums of the tokens that went before are
    gone, and nothing passes fp32's range on the way.

    Blocks of sixteen have both sorts of tokens in one, with the larger ones' scale s and the smaller ones' codes 0.  A probability times its value's scale
    is held to 2^-34 of the row's largest such product, which is s times the probability that all n tokens that count have in common: a sum of n
    products with codes up to 127, over n such probabilities, is off by up to 127 * 2^-34 s.  A step of the block itself is s."""
    n, first = 300, 150

    def jump(k, v):
        k[:] = 0
        k[:first, ::64] = -4000 * up
        k[first:, ::64] = 4000 * up
        v[:first] *= np.float32(2.0 ** (90 * up))
        v[first:] *= np.float32(2.0 ** (-90 * up))
    f, heads = Filled(fdx, [n], 2, 64, 64, 16, "i8", block, change=jump), 4
    q = np.zeros((new, heads * 64), np.float32)
    q[:, ::64] = 3
    want = f.reference(q, [new], heads)
    # all scores that count are the same number: what is left are the errors of means of values
    assert np.isfinite(want).all()
    got = fdx.mha_paged(f.cache, q, [new], heads).astype(np.float64)
    count = [p for p in range(n) if (p >= first) == (up > 0)]
    most = max(float(f.host.scales[1][f.row_of(0)(p) // block].max()) for p in count)
    off, step = np.abs(got - want), 127 * 2.0 ** -34 * most
    print("off %.2e of %.2e, step %.2e" % (off.max(), np.abs(want).max(), step), flush=True)
    assert off.max() <= step + 2e-5 * np.abs(want).max()
    assert np.linalg.norm(off * 2.0 ** (90 * up)) <= 2.0 ** (90 * up) * step * np.sqrt(off.size) + 2e-6 * np.linalg.norm(want * 2.0 ** (90 * up))


@pytest.mark.parametrize("new", [3, 100])
@pytest.mark.parametrize("eq,ek,ev", [(80, 80, 60), (80, 80, -60), (-80, 60, 110)])
def test_paged_products_that_are_zero(fdx, new, eq, ek, ev):
    """Queries and keys whose product would be far out of range, and has no terms; values near fp32's end beside ones near its beginning."""
    n, heads, kv, d = 300, 4, 2, 64

    def change(k, v):
        k[:] *= np.float32(2.0 ** ek)
        k[:, ::2] = 0
        v[::2] *= np.float32(2.0 ** ev)
        v[1::2] *= np.float32(2.0 ** -ev)
    f = Filled(fdx, [n], kv, d, d, 16, "i8", 16, change=change)
    q = (2.0 ** eq * np.random.default_rng(9).standard_normal((new, heads * d))).astype(np.float32)
    q[:, 1::2] = 0
    close(fdx.mha_paged(f.cache, q, [new], heads).astype(np.float64) * 2.0 ** -abs(ev), f.reference(q, [new], heads) * 2.0 ** -abs(ev))


@pytest.mark.parametrize("new", [1, 12, 100])
def test_paged_scores_far_below_zero(fdx, new):
    """Every score is far below zero, some rows' by hundreds: their sums are as exact as other rows'."""
    def change(k, v):
        k[:, 0] = k[:, 64] = 60
    f, heads = Filled(fdx, [250], 2, 64, 64, 16, "e4m3", 16, change=change), 4
    q = np.random.default_rng(3).standard_normal((new, heads * 64)).astype(np.float32)
    q[:, ::64] = -np.linspace(1, 40, new)[:, None]
    # scores of 60 * 40 / 8 = 300, a tenth of which is rounded 300 times as much as a score of one: 300 * 2e-7
    close(fdx.mha_paged(f.cache, q, [new], heads), f.reference(q, [new], heads), 6e-5)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("context,new,heads,kv,d", [([5000, 40], [1, 1], 4, 2, 64), ([3000, 2900, 700], [40, 1, 100], 8, 2, 128),
                                                    ([9000], [1], 32, 8, 128), ([4100, 4100], [3, 300], 4, 4, 64)])
def test_paged_long_contexts(fdx, context, new, heads, kv, d, kind):
    f = Filled(fdx, context, kv, d, d, 64, kind, 16)
    q = np.random.default_rng(5).standard_normal((sum(new), heads * d)).astype(np.float32)
    print("paged8 long", context, new, heads, kv, d, kind, flush=True)
    close(fdx.mha_paged(f.cache, q, new, heads), f.reference(q, new, heads))


@pytest.mark.parametrize("new", [1, 70])
def test_every_part_of_a_long_sequence_counts_once(fdx, new):
    """Equal scores and values that name their part: the mean tells how often each part was counted."""
    n, d, heads = 6000, 64, 2

    def change(k, v):
        k[:] = 0
        v[:] = 0
        v[np.arange(n), np.arange(n) // 100 % d] = 1
    f = Filled(fdx, [n], 1, d, d, 16, "i8", 16, change=change)
    q = np.random.default_rng(1).standard_normal((new, heads * d)).astype(np.float32)
    close(fdx.mha_paged(f.cache, q, [new], heads), f.reference(q, [new], heads))


@pytest.mark.parametrize("new", [1, 70])
def test_runs_are_equal(fdx, new):
    f = Filled(fdx, [3000, 500], 2, 64, 64, 16, "i8", 16)
    q = np.random.default_rng(1).standard_normal((new + 1, 8 * 64)).astype(np.float32)
    first = fdx.mha_paged(f.cache, q, [new, 1], 8)
    for _ in range(3):
        assert np.array_equal(first, fdx.mha_paged(f.cache, q, [new, 1], 8))


@pytest.mark.parametrize("kind", KINDS)
def test_offsets_beyond_32_bits(fdx, kind):
    """Pages whose first byte lies beyond 2^32 of the cache's."""
    kv, d, page = 64, 128, 64
    n_pages = (1 << 32) // (page * kv * d) + 6
    c = fdx.PagedCache(2, page, kv, d, d, 2, 3 * page, kind, 16)
    big = [fdx.DevBuf(n_pages * page * kv * d) for _ in range(2)]
    scales = [fdx.DevBuf(n_pages * page // 16 * kv * 4) for _ in range(2)]
    c.n_pages, c.k, c.v, c.k_scale, c.v_scale = n_pages, *big, *scales
    c.free = [n_pages - 1, n_pages - 2, 0, n_pages - 3, n_pages - 4, n_pages - 5]
    r = np.random.default_rng(9)
    k, v = (r.standard_normal((150, kv * d)).astype(np.float32) for _ in range(2))
    print("paged8 far pages", kind, flush=True)
    fdx.kv_append(c, k, v, [100, 50])
    host = HostCache(5, page, kv, d, d, kind, 16)   # the pages of the sequences in order
    for s, (a, b) in enumerate(((0, 100), (100, 150))):
        for which, x in enumerate((k, v)):
            host.append(lambda p: 2 * s * page + p, 0, x[a:b].reshape(b - a, kv, d), which)
    q = r.standard_normal((36, kv * d)).astype(np.float32)
    for new in ([1, 1], [35, 1]):
        got, at = fdx.mha_paged(c, q[:sum(new)], new, kv), 0
        for s, n in enumerate(new):
            length = (100, 50)[s]
            rows = 2 * s * page + np.arange(length)
            close(got[at:at + n], attend(q[at:at + n], host.values(rows, 0), host.values(rows, 1), kv, kv, np.arange(length - n, length) + 1))
            at += n


def test_two_threads(fdx):
    """Calls of two host threads, each with a cache of its own."""
    import threading
    heads, want, got, errors = 4, [None, None], [None, None], []
    r = np.random.default_rng(11)
    k, v, q = (r.standard_normal((2, n, w)).astype(np.float32) for n, w in ((500, 128), (500, 128), (2, heads * 64)))
    logits, scores = r.standard_normal((2, 3, 4, 3001)).astype(np.float32), -r.random((2, 3, 4)).astype(np.float32)

    def steps(i):
        c = fdx.PagedCache(60, 16, 2, 64, 64, 2, 400, ("i8", "e4m3")[i], 8)
        out = []
        for at in range(0, 500, 100):
            fdx.kv_append(c, k[i, at:at + 100], v[i, at:at + 100], [40 + i, 60 - i])
            out.append(fdx.mha_paged(c, q[i], [1, 1], heads))
            best = fdx.beam_select(logits[i], scores[i], 4)
            out += [best[key] for key in sorted(best)]
            fdx.kv_fork(c, [0, 1] if at % 200 else [1, 0])
        return out

    def work(i):
        try:
            for _ in range(5):
                got[i] = steps(i)
        except Exception as e:   # reported below, by the test's own thread
            errors.append(e)
    want = [steps(0), steps(1)]
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors, errors
    for a, b in zip(want, got):
        assert all(np.array_equal(x, y) for x, y in zip(a, b)) and len(a) == len(b)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [1, 12, 100])
@pytest.mark.parametrize("keys,rise", [(300, 7.9), (300, 3.9), (900, 7.9), (3000, 7.5)])
def test_paged_values_near_the_end_of_fp32(fdx, keys, rise, new, kind):
    """Values up to 3.2e38 behind scores that rise by less than a power of 2^8 on the way: sums are means, none passes fp32's range.  The keys of
    either half have one score, so its error is common to them: what is left are the errors of means of values."""
    def change(k, v):
        k[:] = 0
        k[keys // 2:, ::64] = rise * np.log(2) * 8
        v[:] = np.float32(3.2e38) * np.random.default_rng(2).uniform(-1, 1, v.shape).astype(np.float32)
    f, heads = Filled(fdx, [keys], 2, 64, 64, 16, kind, 16, change=change), 4
    q = np.zeros((new, heads * 64), np.float32)
    q[:, ::64] = 1
    print("paged8 largest values", keys, rise, new, kind, flush=True)
    got, want = fdx.mha_paged(f.cache, q, [new], heads), f.reference(q, [new], heads)
    close(np.ldexp(got.astype(np.float64), -127), np.ldexp(want, -127))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [1, 12, 100])
@pytest.mark.parametrize("block", [8, 16])
@pytest.mark.parametrize("eq,ek", [(16, 0), (20, 0), (24, 0), (30, 0), (0, 60), (60, 50), (-20, 90)])
def test_paged_scores_far_from_zero(fdx, eq, ek, block, new, kind):
    """Scores from 2^17 to 2^114, either sign, whose differences are thousands and more: the keys of the largest one, which are several and have the
    same codes, share the weight.  What is left are the errors of means of values."""
    n = 300

    def change(k, v):
        r = np.random.default_rng(4)
        k[:] = 0
        c = r.integers(-126, 127, (n, 1)) if kind == "i8" else 16 * r.integers(-27, 28, (n, 1))
        c[::8] = 127 if kind == "i8" else 448   # every block has the same scale, and codes are exact
        c[4::8] = -c[::8][:len(c[4::8])]
        k[:, ::64] = np.ldexp(c.astype(np.float32), ek)
    f, heads = Filled(fdx, [n], 2, 64, 64, 16, kind, block, change=change), 4
    r = np.random.default_rng(5)
    q = np.zeros((new, heads * 64), np.float32)
    q[:, ::64] = np.ldexp(r.uniform(0.5, 1.5, (new, heads)) * r.choice([-1, 1], (new, heads)), eq)
    print("paged8 far scores", eq, ek, block, new, kind, flush=True)
    close(fdx.mha_paged(f.cache, q, [new], heads), f.reference(q, [new], heads))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [[1, 1], [3, 40], [140, 1]])
@pytest.mark.parametrize("e", [108, 114, 118, 122, 124])
@pytest.mark.parametrize("d", [64, 128])
def test_paged_queries_near_the_end_of_fp32(fdx, new, e, kind, d):
    """Queries up to 2^126 and keys as small: scores of ordinary size, though a sum over codes alone passes fp32's range."""
    def change(k, v):
        k *= np.float32(2.0 ** -e)
    f, heads = Filled(fdx, [200, 141], 2, d, d, 16, kind, 16, change=change), 4
    q = np.random.default_rng(5).standard_normal((sum(new), heads * d)).astype(np.float32)
    q = np.ldexp(np.clip(q, -3.5, 3.5), e).astype(np.float32)
    q[-1, :d] = np.ldexp(q[-1, :d], -2 * e)   # a row of small ones beside them
    print("paged8 largest queries", new, e, kind, d, flush=True)
    close(fdx.mha_paged(f.cache, q, new, heads), f.reference(q, new, heads))


def test_two_threads_at_every_repetition(fdx):
    """As test_two_threads, all repetitions of either thread compared, and begun together."""
    import threading
    heads, times, errors = 4, 6, []
    r = np.random.default_rng(12)
    k, v, q = (r.standard_normal((2, n, w)).astype(np.float32) for n, w in ((500, 128), (500, 128), (42, heads * 64)))
    logits, scores = r.standard_normal((2, 3, 4, 3001)).astype(np.float32), -r.random((2, 3, 4)).astype(np.float32)

    def steps(i):
        c = fdx.PagedCache(70, 16, 2, 64, 64, 2, 400, ("e4m3", "i8")[i], 8)
        out = []
        for at in range(0, 500, 100):
            fdx.kv_append(c, k[i, at:at + 100], v[i, at:at + 100], [40 + i, 60 - i])
            out += [fdx.mha_paged(c, q[i, :2], [1, 1], heads), fdx.mha_paged(c, q[i], [41, 1], heads)]
            best = fdx.beam_select(logits[i], scores[i], 4)
            out += [best[key] for key in sorted(best)]
            fdx.kv_fork(c, [0, 1] if at % 200 else [1, 0])
            out += [c.table.copy(), c.lens.copy()]
        return out
    want, got, together = [steps(0), steps(1)], [[], []], threading.Barrier(2)

    def work(i):
        try:
            for _ in range(times):
                together.wait(60)
                got[i].append(steps(i))
        except Exception as e:   # reported below, by the test's own thread
            errors.append(e)
            together.abort()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors, errors
    for i in range(2):
        assert len(got[i]) == times
        for one in got[i]:
            assert len(one) == len(want[i]) and all(np.array_equal(x, y) for x, y in zip(one, want[i]))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 13])
def test_append_of_scales_beyond_each_other(fdx, d, kind):
    """A block whose scale grows so far that what was there in front has no size beside it: earlier codes are zeros of their own sign, as rounding makes
    them; and where a NaN joins them, zeros."""
    for first, then in ((-120, 60), (-149, 127), (-60, 100), (-126, 24), (-120, 28)):
        r = np.random.default_rng(-first)
        c, host = fdx.PagedCache(1, 8, 2, d, d, 1, 8, kind, 8), HostCache(1, 8, 2, d, d, kind, 8)
        for at, e in enumerate((first, then, first, None)):
            x = np.ldexp(r.uniform(-1.9, 1.9, (2, 2 * d)), 0 if e is None else e).astype(np.float32)
            if e is None:
                x[1, 3] = np.nan
            print("append8 scales", first, then, at, d, kind, flush=True)
            fdx.kv_append(c, x, -x, [2])
            for which, y in enumerate((x, -x)):
                host.append(lambda p: p, 2 * at, y.reshape(2, 2, d), which)
            same(c, host)
