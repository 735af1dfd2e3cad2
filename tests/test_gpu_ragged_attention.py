"""Attention over packed prompts and over paged caches, and the writing of such caches, against plain sums in 64 bits.

Bounds.  fp32 operands may be held as two fp16 numbers (22 bits) for the matrix instructions: a product is off by at most
3 * 2^-22 of its size, a score of dk products of unit operands by about 0.64 sqrt(dk) 2^-22 * 3 / sqrt(dk) (independent signs) = 5e-7
absolute, which is the relative error of a probability; the sums of the output add as much again, and both average out over the
keys.  1e-6 in the 2-norm, and 1e-5 of the largest value for any single output, leave a factor of two over that.  Scores k times
larger carry k times the error.  bf16 caches: the reference takes the rounded keys and values, so the bounds are the same."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def bf16(x):
    """fp32 values rounded to the nearest bf16, ties to even"""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((b + 0x7fff + ((b >> 16) & 1)) & 0xffff0000).astype(np.uint32).view(np.float32)


def attend(q, k, v, heads, kv_heads, sees):
    """q [n][heads*dk], k [keys][kv*dk], v [keys][kv*dv]; query i sees the first sees[i] keys; in 64 bits"""
    n, keys = q.shape[0], k.shape[0]
    q = q.astype(np.float64).reshape(n, heads, q.shape[1] // heads)
    k, v = (a.astype(np.float64).reshape(keys, kv_heads, a.shape[1] // kv_heads) for a in (k, v))
    out = np.zeros((n, heads, v.shape[2]))
    for h in range(heads):
        kh, vh = k[:, h * kv_heads // heads], v[:, h * kv_heads // heads]
        x = q[:, h] @ kh.T / np.sqrt(q.shape[2])
        for i in range(n):
            if sees[i] > 0:
                e = np.exp(x[i, :sees[i]] - x[i, :sees[i]].max())
                out[i, h] = e / e.sum() @ vh[:sees[i]]
    return out.reshape(n, heads * v.shape[2])


def close(got, want, bound=1e-6):
    norm = np.linalg.norm(want)
    err, worst = np.linalg.norm(got - want) / max(norm, 1e-30), np.abs(got - want).max() / max(np.abs(want).max(), 1e-30)
    print("relative error %.2e, largest %.2e" % (err, worst), flush=True)
    assert err <= bound and worst <= 10 * bound, (err, worst)


def packed_reference(q, k, v, lengths, heads, kv_heads, causal):
    out, at = [], 0
    for n in lengths:
        rows = slice(at, at + n)
        out.append(attend(q[rows], k[rows], v[rows], heads, kv_heads, np.arange(n) + 1 if causal else np.full(n, n)))
        at += n
    return np.concatenate(out)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,heads,kv_heads,dk,dv", [
    ([1], 1, 1, 64, 64), ([2, 1, 1], 3, 1, 64, 64), ([37], 12, 12, 64, 64), ([0, 5, 0, 0, 64, 65, 1, 0], 8, 2, 64, 64),
    ([129, 31, 200], 4, 4, 128, 128), ([300], 7, 1, 128, 128), ([127, 128, 129], 10, 5, 80, 80), ([63, 190], 6, 6, 32, 32),
    ([70, 11], 4, 2, 96, 64), ([70, 11], 4, 2, 40, 128), ([33, 90], 3, 1, 1, 1), ([33, 90], 6, 2, 13, 7), ([400], 2, 2, 127, 125),
    ([600, 10, 513], 2, 1, 64, 64)])
def test_packed(fdx, lengths, heads, kv_heads, dk, dv, causal):
    print("packed", lengths, heads, kv_heads, dk, dv, causal, flush=True)
    r, tokens = np.random.default_rng(sum(lengths) + dk), sum(lengths)
    q, k, v = (r.standard_normal((tokens, h * d)).astype(np.float32) for h, d in ((heads, dk), (kv_heads, dk), (kv_heads, dv)))
    close(fdx.mha_packed(q, k, v, lengths, heads, kv_heads, dk, dv, causal), packed_reference(q, k, v, lengths, heads, kv_heads, causal))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,heads,kv_heads,dk,dv", [
    ([513, 130], 4, 2, 128, 128), ([700], 5, 5, 80, 80), ([520, 1, 0, 300], 2, 1, 33, 127), ([64] * 9, 3, 3, 64, 64), ([512], 1, 1, 64, 64),
    ([33, 600, 95, 32, 31], 8, 1, 128, 128), ([1, 1200, 2], 6, 2, 32, 32), ([300, 300], 7, 7, 64, 40), ([900], 16, 2, 64, 64),
    # many rows a key head, from where on keys and values are split in a pass of their own
    ([300], 32, 4, 64, 64), ([200, 130], 32, 1, 128, 128), ([2, 300, 0, 129, 1], 32, 1, 64, 64), ([190, 65], 40, 2, 80, 96), ([129], 16, 1, 33, 127),
    ([2100], 1, 1, 32, 32)])
def test_packed_of_many_tokens(fdx, lengths, heads, kv_heads, dk, dv, causal):
    test_packed(fdx, lengths, heads, kv_heads, dk, dv, causal)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,heads,kv_heads,dk,dv", [
    ([1500], 4, 4, 64, 64), ([513], 1, 1, 64, 64), ([512, 512], 3, 3, 64, 64), ([2100, 0, 700], 4, 2, 64, 64), ([1024], 5, 1, 128, 128),
    ([700, 1, 1200], 2, 2, 33, 127), ([769, 770, 767], 6, 6, 32, 32), ([1, 0, 3000], 2, 1, 80, 96), ([1025], 12, 12, 64, 64), ([2047], 12, 12, 64, 64)])
def test_packed_few_long(fdx, lengths, heads, kv_heads, dk, dv, causal):
    """Fewer tiles than the GPU takes: keys in ranges."""
    print("packed few", lengths, heads, kv_heads, dk, dv, causal, flush=True)
    test_packed(fdx, lengths, heads, kv_heads, dk, dv, causal)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,heads,kv_heads,dk,dv", [
    ([400], 6, 1, 64, 64), ([511, 300, 0, 1], 16, 1, 64, 64), ([257, 128, 129], 16, 1, 128, 128), ([500, 31], 20, 2, 80, 80), ([450], 7, 1, 33, 127),
    ([1300, 900], 16, 16, 64, 64)])
def test_packed_split_once(fdx, lengths, heads, kv_heads, dk, dv, causal):
    """Many query rows a key head: a pass of its own splits keys and values."""
    print("packed once", lengths, heads, kv_heads, dk, dv, causal, flush=True)
    test_packed(fdx, lengths, heads, kv_heads, dk, dv, causal)


@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("name,row", [("v", 333), ("k", 333), ("k", 64), ("v", 399)])
def test_packed_split_once_infinities_and_nan(fdx, what, name, row):
    r, n, heads, kv = np.random.default_rng(9), 400, 8, 1
    q, k, v = (r.standard_normal((n, h * 64)).astype(np.float32) for h in (heads, kv, kv))
    base = packed_reference(q, k, v, [n], heads, kv, True)
    print("packed once odd", what, name, row, flush=True)
    dict(k=k, v=v)[name][row, 7] = what
    got = fdx.mha_packed(q, k, v, [n], heads, kv, 64, 64)
    close(got[:row], base[:row])
    with np.errstate(all="ignore"):
        want = packed_reference(q, k, v, [n], heads, kv, True)[row:]
    assert np.array_equal(np.isnan(got[row:]), np.isnan(want)) and np.array_equal(np.isinf(got[row:]), np.isinf(want))


@pytest.mark.parametrize("lengths,heads", [([90, 150, 40], 4), ([640, 200], 4), ([260, 150], 64)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("power", [12, 18, 30, 70, 124])
def test_packed_sizes_behind_the_mask(fdx, lengths, heads, d, power):
    """Keys and values of later tokens 2^power times larger: the tokens in front of them do not see them and keep their bound, also
    those that share a tile with them."""
    r, kv, total = np.random.default_rng(power), 2, sum(lengths)
    q, k, v = (r.standard_normal((total, h * d)).astype(np.float32) for h in (heads, kv, kv))
    base = packed_reference(q, k, v, lengths, heads, kv, True)
    for name, first in (("k", 41), ("v", 41), ("v", lengths[0] - 1), ("k", 2), ("v", 3)):
        print("packed behind the mask", lengths, d, power, name, first, flush=True)
        kk, vv = k.copy(), v.copy()
        dict(k=kk, v=vv)[name][first:lengths[0]] *= np.float32(2.0 ** power)
        got = fdx.mha_packed(q, kk, vv, lengths, heads, kv, d, d)
        keep = np.r_[0:first, lengths[0]:total]
        close(got[keep], base[keep])
        if name == "v":   # and the rows that see them: their result is as large as the largest they see
            with np.errstate(all="ignore"):
                want = packed_reference(q, kk, vv, lengths, heads, kv, True)[first:lengths[0]]
            # one probability with nothing to average over: its score is a chain of d sums of up to 3 sqrt(d) = 34, each off by up to
            # half of 2^-19 and by a quarter on average, 0.25 * 2^-19 * sqrt(d) / sqrt(d) = 5e-7 in all as a standard deviation, over a few rows
            close(got[first:lengths[0]].astype(np.float64), want, 2e-6)


def test_packed_many_tokens_infinities_and_nan(fdx):
    """A NaN or infinity in one of several ranges of keys."""
    r, n, heads, kv = np.random.default_rng(8), 700, 6, 1
    q, k, v = (r.standard_normal((n, h * 64)).astype(np.float32) for h in (heads, kv, kv))
    base = packed_reference(q, k, v, [n], heads, kv, True)
    for what in (np.nan, np.inf, -np.inf):
        for name, row in (("v", 333), ("k", 333), ("k", 640)):
            print("packed many odd", what, name, row, flush=True)
            kk, vv = k.copy(), v.copy()
            dict(k=kk, v=vv)[name][row, 7] = what
            got = fdx.mha_packed(q, kk, vv, [n], heads, kv, 64, 64)
            close(got[:row], base[:row])
            with np.errstate(all="ignore"):
                want = packed_reference(q, kk, vv, [n], heads, kv, True)[row:]
            assert np.array_equal(np.isnan(got[row:]), np.isnan(want)) and np.array_equal(np.isinf(got[row:]), np.isinf(want))
            ok = np.isfinite(want)
            if ok.any():
                close(got[row:][ok], want[ok])


def test_packed_scores_of_a_few_hundred(fdx):
    """The running maximum moves from tile to tile; scores 40 times larger, errors too."""
    r, lengths = np.random.default_rng(3), [333, 50]
    q, k, v = (r.standard_normal((383, h * 64)).astype(np.float32) for h in (8, 2, 2))
    close(fdx.mha_packed(40 * q, k, v, lengths, 8, 2, 64, 64), packed_reference(40 * q, k, v, lengths, 8, 2, True), 4e-5)
    # and one that climbs all the way: every key beats those in front of it
    k[:, :64] = q[:, :64] * 0 + 1
    k[:, 0] = np.arange(383) * 8
    q[:, ::64] = 1
    close(fdx.mha_packed(q, k, v, lengths, 8, 2, 64, 64), packed_reference(q, k, v, lengths, 8, 2, True), 4e-5)


@pytest.mark.parametrize("eq,ek,ev", [(0, 0, 0), (60, -60, 0), (-60, 60, 0), (-100, 100, 0), (0, 0, 100), (0, 0, -100), (-40, -80, 5), (110, -110, 110)])
def test_packed_sizes_of_operands(fdx, eq, ek, ev):
    """Operands far from one in size: scaled by powers of two, the result scales."""
    r, lengths = np.random.default_rng(5), [200, 41]
    q, k, v = (r.standard_normal((241, h * 64)).astype(np.float32) for h in (4, 2, 2))
    q, k, v = (np.ldexp(a, e).astype(np.float32) for a, e in ((q, eq), (k, ek), (v, ev)))
    got = fdx.mha_packed(q, k, v, lengths, 4, 2, 64, 64)
    close(np.ldexp(got.astype(np.float64), -ev), packed_reference(q, k, np.ldexp(v.astype(np.float64), -ev), lengths, 4, 2, True))


def test_packed_rows_of_mixed_sizes(fdx):
    """Keys and values whose sizes differ by 2^15 from row to row and by 2^12 from depth to depth keep the bound of their own size:
    every query sees its own key only (scores of +-200 apart), so a result is one row of values."""
    r, n = np.random.default_rng(6), 160
    q, k = np.zeros((n, 64), np.float32), np.zeros((n, 64), np.float32)
    angle = 2 * np.pi * np.arange(n) / n
    q[:, 0], q[:, 1] = np.cos(angle), np.sin(angle)
    k[:, :2], q = q[:, :2] * 1000, q * 10000
    v = (r.standard_normal((n, 64)) * 2.0 ** r.integers(-7, 8, (n, 1)) * 2.0 ** r.integers(-6, 7, (1, 64))).astype(np.float32)
    got, want = fdx.mha_packed(q, k, v, [n], 1, 1, 64, 64, False), packed_reference(q, k, v, [n], 1, 1, False)
    size = np.abs(want).max(1, keepdims=True)
    print("worst row", (np.abs(got - want) / size).max(), flush=True)
    assert (np.abs(got - want) <= 1e-6 * size).all()


def test_packed_infinities_and_nan(fdx):
    """A NaN or infinity reaches the queries that see it and no other, whatever tile they share."""
    r, lengths, heads, kv = np.random.default_rng(8), [90, 150, 40], 4, 2
    q, k, v = (r.standard_normal((280, h * 64)).astype(np.float32) for h in (heads, kv, kv))
    base = packed_reference(q, k, v, lengths, heads, kv, True)
    for what in (np.nan, np.inf, -np.inf):
        for name, row, first, last in (("v", 120, 120, 240), ("k", 120, 120, 240), ("q", 100, 100, 101), ("v", 279, 279, 280), ("k", 0, 0, 90)):
            print("packed odd", what, name, row, flush=True)
            qq, kk, vv = q.copy(), k.copy(), v.copy()
            dict(q=qq, k=kk, v=vv)[name][row, 64 + 3] = what   # query head 1 / key head 1
            got = fdx.mha_packed(qq, kk, vv, lengths, heads, kv, 64, 64).reshape(280, heads, 64)
            hit = np.zeros((280, heads, 64), bool)
            if name == "v":
                hit[first:last, 2:, 3] = True
            else:
                hit[first:last, (slice(1, 2) if name == "q" else slice(2, 4))] = True
            with np.errstate(all="ignore"):
                want = packed_reference(qq, kk, vv, lengths, heads, kv, True).reshape(280, heads, 64)
            close(got[~hit], base.reshape(280, heads, 64)[~hit])
            seen = want[hit]
            if name == "v":
                assert np.array_equal(np.isnan(got[hit]), np.isnan(seen)) and np.array_equal(got[hit][np.isinf(seen)], seen[np.isinf(seen)])
            else:   # scores of -infinity drop a key, those of +infinity and NaN leave nothing
                assert np.array_equal(np.isnan(got[hit]), np.isnan(seen))
                close(got[hit][~np.isnan(seen)], seen[~np.isnan(seen)]) if (~np.isnan(seen)).any() else None


def noise(fdx, size):
    """Memory whose contents mean nothing: NaN in every place."""
    return fdx.DevBuf.from_host(np.full(size + 16, 255, np.uint8), np.uint8)


def call_packed(fdx, q, ldq, k, ldk, v, ldv, starts, tokens, heads, kv, dk, dv, out, ldo, causal=True):
    """The entry point itself: byte offsets of 4 behind the buffers' starts are kept."""
    i64, n_seqs = ctypes.c_int64, len(starts) - 1
    d_starts, flag = fdx.DevBuf.from_host(np.asarray(starts, np.int32), np.int32), fdx.DevBuf.from_host(np.zeros(1, np.int32), np.int32)
    scratch = noise(fdx, fdx.lib.fdx_mha_packed_scratch_bytes(tokens, n_seqs, heads, kv, dk, dv))
    fdx.check(fdx.lib.fdx_mha_packed_f32(q, i64(ldq), k, i64(ldk), v, i64(ldv), d_starts.ptr, n_seqs, tokens, heads, kv, dk, dv, int(causal), out,
                                         i64(ldo), scratch.ptr, flag.ptr))
    fdx.sync()
    return int(flag.to_host((1,), np.int32)[0])


@pytest.mark.parametrize("shift,pad", [(0, 4), (1, 4), (0, 3), (2, 1), (3, 0)])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128)])
def test_packed_strides_and_alignment(fdx, shift, pad, dk, dv):
    """q, k and v as column blocks of one projection that starts `shift` floats behind an aligned address, rows `pad` floats apart;
    rows in front of and behind the sequences, and the gaps between rows of the output, stay as they were."""
    heads, kv, lengths, before, behind = 4, 2, [70, 0, 135], 3, 5
    r, tokens = np.random.default_rng(shift), before + 205 + behind
    width = (heads + kv) * dk + kv * dv + pad
    x = r.standard_normal((tokens, width)).astype(np.float32)
    buf = fdx.DevBuf.from_host(np.concatenate([np.zeros(shift, np.float32), x.ravel()]))
    ldo = heads * dv + pad
    out = fdx.DevBuf.from_host(np.full(shift + tokens * ldo, 7, np.float32))
    at = lambda b, floats: ctypes.c_void_p(b.ptr.value + 4 * floats)
    flag = call_packed(fdx, at(buf, shift), width, at(buf, shift + heads * dk), width, at(buf, shift + (heads + kv) * dk), width,
                       [before, before + 70, before + 70, before + 205], tokens, heads, kv, dk, dv, at(out, shift), ldo)
    got = out.to_host((shift + tokens * ldo,))[shift:].reshape(tokens, ldo)
    q, k, v = x[before:-behind, :heads * dk], x[before:-behind, heads * dk:(heads + kv) * dk], x[before:-behind, (heads + kv) * dk:(heads + kv) * dk + kv * dv]
    assert flag == 0
    close(got[before:-behind, :heads * dv], packed_reference(q, k, v, lengths, heads, kv, True))
    assert (got[:before] == 7).all() and (got[-behind:] == 7).all() and (got[:, heads * dv:] == 7).all()


@pytest.mark.parametrize("starts", [[0, 50, 20, 60], [0, 10, 61], [-5, 30], [0, 40, 2**31 - 1], [40, 20, 0], [-2**31, 2**31 - 1]])
def test_packed_starts_that_are_none(fdx, starts):
    """Reported, nothing outside the tensors touched: what lies behind the output stays."""
    r, tokens = np.random.default_rng(1), 60
    q, k, v = (fdx.DevBuf.from_host(r.standard_normal((tokens, 128)).astype(np.float32)) for _ in range(3))
    out = fdx.DevBuf.from_host(np.full((tokens + 100) * 128, 3, np.float32))
    print("packed starts", starts, flush=True)
    assert call_packed(fdx, q.ptr, 128, k.ptr, 128, v.ptr, 128, starts, tokens, 2, 2, 64, 64, out.ptr, 128) == 1
    assert (out.to_host(((tokens + 100) * 128,))[tokens * 128:] == 3).all()


def test_packed_runs_are_equal(fdx):
    r, lengths = np.random.default_rng(2), [300, 20, 1, 77]
    q, k, v = (r.standard_normal((398, h * 64)).astype(np.float32) for h in (8, 2, 2))
    first = fdx.mha_packed(q, k, v, lengths, 8, 2, 64, 64)
    for _ in range(3):
        assert np.array_equal(first, fdx.mha_packed(q, k, v, lengths, 8, 2, 64, 64))


# ---------------------------------------------------------------- paged caches

class Filled:
    """A cache with `context` positions per sequence written by kv_append in `steps` calls, and the rows that went in."""

    def __init__(self, fdx, context, kv, dk, dv, page, kind, seed=0, extra=4, steps=2, max_len=None):
        r = np.random.default_rng(seed)
        self.keys = [r.standard_normal((n, kv * dk)).astype(np.float32) for n in context]
        self.values = [r.standard_normal((n, kv * dv)).astype(np.float32) for n in context]
        n_pages = sum(-(-n // page) for n in context) + extra
        self.cache = fdx.PagedCache(n_pages, page, kv, dk, dv, len(context), max_len or max(max(context), 1), kind)
        r.shuffle(self.cache.free)   # pages of a sequence lie apart
        done = [0] * len(context)
        for step in range(steps):
            upto = [n if step == steps - 1 else n // 2 for n in context]
            part = [b - a for a, b in zip(done, upto)]
            if sum(part):
                fdx.kv_append(self.cache, *(np.concatenate([x[a:b] for x, a, b in zip(xs, done, upto)]) for xs in (self.keys, self.values)), part)
            done = upto
        if kind == "bf16":
            self.keys, self.values = [bf16(x) for x in self.keys], [bf16(x) for x in self.values]

    def reference(self, q, new, heads):
        out, at = [], 0
        for s, n in enumerate(new):
            length = len(self.keys[s])
            out.append(attend(q[at:at + n], self.keys[s], self.values[s], heads, self.cache.kv_heads, np.arange(length - n, length) + 1))
            at += n
        return np.concatenate(out)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("kv,dk,dv,page", [(2, 64, 64, 16), (3, 128, 128, 5), (1, 80, 80, 64), (2, 13, 7, 3), (2, 96, 64, 1), (1, 32, 128, 200)])
def test_append(fdx, kv, dk, dv, page, kind):
    """Every position holds its row, rounded to nearest in bf16, and no other place of the pages has changed."""
    context = [1, 0, 77, 16, 130]
    print("append", kv, dk, dv, page, kind, flush=True)
    f = Filled(fdx, context, kv, dk, dv, page, kind, steps=3)
    c, rows = f.cache, f.cache.n_pages * page
    for buf, d, want in ((c.k, dk, f.keys), (c.v, dv, f.values)):
        held = buf.to_host((rows, kv * d), np.float32) if kind == "f32" else \
            (buf.to_host((rows, kv * d), np.uint16).astype(np.uint32) << 16).view(np.float32)
        used = np.zeros(rows, bool)
        for s, n in enumerate(context):
            pos = np.arange(n)
            at = c.table[s][pos // page] * page + pos % page
            assert np.array_equal(held[at], want[s])
            used[at] = True
        assert (held[~used] == 0).all()


def test_append_rounds_to_nearest(fdx):
    x = np.array([1, 1 + 2**-8, 1 + 3 * 2**-8, 1 + 2**-8 + 2**-20, -1 - 2**-8, 3.4e38, -3.4e38, 1e-40, 2**-133, 0.0, -0.0, np.inf, -np.inf, np.nan,
                  65504, 1e-38], np.float32)
    c = fdx.PagedCache(1, 1, 1, 16, 16, 1, 1, "bf16")
    fdx.kv_append(c, x[None], x[None], [1])
    held = (c.k.to_host((16,), np.uint16).astype(np.uint32) << 16).view(np.float32)
    want = bf16(x)
    ok = ~np.isnan(x)
    assert np.array_equal(held[ok].view(np.uint32), want[ok].view(np.uint32)) and np.isnan(held[~ok]).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("context,new,heads,kv,dk,dv,page", [
    ([1], [1], 1, 1, 64, 64, 16), ([201], [1], 12, 12, 64, 64, 16), ([5, 300, 64, 17], [1, 1, 1, 1], 8, 2, 64, 64, 16),
    ([700, 33, 1], [1, 1, 1], 32, 8, 128, 128, 16), ([100, 260, 31], [1, 0, 1], 16, 1, 128, 128, 7), ([100, 50], [1, 1], 32, 1, 64, 64, 32),
    ([130, 90], [1, 1], 10, 5, 80, 80, 13), ([60, 61, 62], [1, 1, 1], 6, 2, 13, 7, 3), ([90], [1], 40, 1, 64, 64, 16), ([70], [1], 4, 2, 96, 64, 1),
    ([200, 77, 16], [3, 5, 16], 4, 4, 64, 64, 16), ([400, 90, 2], [7, 1, 2], 8, 2, 128, 128, 16), ([300, 200], [40, 1], 8, 2, 64, 64, 16),
    ([500, 129, 40, 3], [129, 129, 1, 3], 8, 2, 64, 64, 24), ([450, 260], [300, 17], 7, 1, 128, 128, 64), ([140], [140], 3, 3, 32, 32, 200),
    ([77, 190], [60, 33], 5, 1, 33, 127, 11), ([2100, 1900], [1, 2], 4, 1, 64, 64, 16), ([2300, 5, 1030], [70, 5, 1], 4, 2, 128, 128, 32)])
def test_paged(fdx, context, new, heads, kv, dk, dv, page, kind):
    print("paged", context, new, heads, kv, dk, dv, page, kind, flush=True)
    f = Filled(fdx, context, kv, dk, dv, page, kind, seed=sum(context))
    q = np.random.default_rng(dk).standard_normal((sum(new), heads * dk)).astype(np.float32)
    close(fdx.mha_paged(f.cache, q, new, heads), f.reference(q, new, heads))


def call_paged(fdx, cache, q, ldq, starts, tokens, max_new, heads, out, ldo, **change):
    c = cache.pages()
    for key, value in change.items():
        if key in ("table", "lens"):
            value = fdx.DevBuf.from_host(value, np.int32)
            c._kept += (value,)
            value = value.ptr
        setattr(c, key, value)
    d_starts, flag = fdx.DevBuf.from_host(np.asarray(starts, np.int32), np.int32), fdx.DevBuf.from_host(np.zeros(1, np.int32), np.int32)
    scratch = noise(fdx, fdx.lib.fdx_mha_paged_scratch_bytes(tokens, max_new, heads, ctypes.byref(c)))
    fdx.check(fdx.lib.fdx_mha_paged_f32(q, ctypes.c_int64(ldq), d_starts.ptr, tokens, max_new, heads, ctypes.byref(c), out, ctypes.c_int64(ldo),
                                        scratch.ptr, flag.ptr))
    fdx.sync()
    return int(flag.to_host((1,), np.int32)[0])


@pytest.mark.parametrize("new", [[1, 1, 1], [3, 1, 2], [40, 9, 70]])
def test_paged_tokens_that_see_nothing(fdx, new):
    """More new tokens than positions: the first ones see none and get zeros, none of it is an error."""
    f = Filled(fdx, [50, 2, 30], 2, 64, 64, 16, "f32")
    lens = np.array([50, 0, min(30, new[2])], np.int32) if new[0] == 1 else np.array([50, 1, 1], np.int32)
    tokens, heads = sum(new), 4
    q = np.random.default_rng(1).standard_normal((tokens, heads * 64)).astype(np.float32)
    out, dq, starts = fdx.DevBuf.from_host(np.full((tokens, heads * 64), 9, np.float32)), fdx.DevBuf.from_host(q), np.concatenate([[0], np.cumsum(new)])
    print("paged empty", new, lens, flush=True)
    flag = call_paged(fdx, f.cache, dq.ptr, heads * 64, starts, tokens, max(new), heads, out.ptr, heads * 64, lens=lens)
    got = out.to_host((tokens, heads * 64))
    want = np.concatenate([attend(q[starts[s]:starts[s + 1]], f.keys[s], f.values[s], heads, 2, np.arange(lens[s] - n, lens[s]) + 1)
                           for s, n in enumerate(new)])
    assert flag == 0
    close(got, want)
    assert (got[want == 0] == 0).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("shift,pad", [(0, 4), (1, 0), (0, 3)])
@pytest.mark.parametrize("new", [[1, 1], [2, 30]])
def test_paged_strides_and_alignment(fdx, shift, pad, kind, new):
    heads, kv, d = 4, 2, 64
    f = Filled(fdx, [90, 131], kv, d, d, 16, kind)
    tokens = 2 + sum(new) + 3
    ld = heads * d + pad
    x = np.random.default_rng(4).standard_normal((tokens, ld)).astype(np.float32)
    dq, out = fdx.DevBuf.from_host(np.concatenate([np.zeros(shift, np.float32), x.ravel()])), fdx.DevBuf.from_host(np.full(shift + tokens * ld, 7, np.float32))
    at = lambda b: ctypes.c_void_p(b.ptr.value + 4 * shift)
    print("paged strides", shift, pad, kind, new, flush=True)
    assert call_paged(fdx, f.cache, at(dq), ld, [2, 2 + new[0], 2 + sum(new)], tokens, max(new), heads, at(out), ld) == 0
    got = out.to_host((shift + tokens * ld,))[shift:].reshape(tokens, ld)
    close(got[2:-3, :heads * d], f.reference(x[2:-3, :heads * d], new, heads))
    assert (got[:2] == 7).all() and (got[-3:] == 7).all() and (got[:, heads * d:] == 7).all()


@pytest.mark.parametrize("new", [[1, 1], [4, 3], [60, 9]])
def test_paged_pages_that_are_none(fdx, new):
    """Positions of pages that the cache does not have are left out and reported; so are lengths and tokens beyond what was said."""
    heads, kv, d, page = 4, 2, 64, 16
    f = Filled(fdx, [90, 131], kv, d, d, page, "f32")
    q = np.random.default_rng(4).standard_normal((sum(new), heads * d)).astype(np.float32)
    dq, starts = fdx.DevBuf.from_host(q), [0, new[0], sum(new)]
    out = fdx.DevBuf.from_host(np.zeros((sum(new) + 50, heads * d), np.float32))
    for bad in (-1, f.cache.n_pages, 2**31 - 1, -2**31):
        table = f.cache.table.copy()
        table[1, 2] = bad
        print("paged bad page", new, bad, flush=True)
        assert call_paged(fdx, f.cache, dq.ptr, heads * d, starts, sum(new), max(new), heads, out.ptr, heads * d, table=table) == 1
        got = out.to_host((sum(new), heads * d))
        keep = np.r_[0:32, 48:131]
        sees = np.array([(keep < 131 - new[1] + j + 1).sum() for j in range(new[1])])
        close(got[new[0]:], attend(q[new[0]:], f.keys[1][keep], f.values[1][keep], heads, kv, sees))
        close(got[:new[0]], attend(q[:new[0]], f.keys[0], f.values[0], heads, kv, np.arange(90 - new[0], 90) + 1))
    for lens, flag in (([90, 132], 1), ([90, 2**31 - 1], 1), ([-1, 131], 1), ([-2**31, 131], 1), ([90, 131], 0)):
        print("paged lens", lens, flush=True)
        assert call_paged(fdx, f.cache, dq.ptr, heads * d, starts, sum(new), max(new), heads, out.ptr, heads * d, lens=lens) == flag
        got = out.to_host((sum(new), heads * d))
        close(got[new[0]:], attend(q[new[0]:], f.keys[1], f.values[1], heads, kv, np.arange(131 - new[1], 131) + 1))
        if lens[0] < 0:
            assert (got[:new[0]] == 0).all()
    for starts in ([0, 2**31 - 1, 5], [-4, 1, sum(new)], [1, 0, 1]):
        print("paged starts", starts, flush=True)
        assert call_paged(fdx, f.cache, dq.ptr, heads * d, starts, sum(new), max(new), heads, out.ptr, heads * d) == 1
    assert (out.to_host((sum(new) + 50, heads * d))[sum(new):] == 0).all()


def test_paged_more_new_tokens_than_said(fdx):
    f, heads = Filled(fdx, [90, 131], 2, 64, 64, 16, "f32"), 4
    q = np.random.default_rng(4).standard_normal((45, heads * 64)).astype(np.float32)
    dq, out = fdx.DevBuf.from_host(q), fdx.DevBuf.from_host(np.full((45, heads * 64), 5, np.float32))
    assert call_paged(fdx, f.cache, dq.ptr, heads * 64, [0, 5, 45], 45, 5, heads, out.ptr, heads * 64) == 1
    got = out.to_host((45, heads * 64))
    close(got[:5], attend(q[:5], f.keys[0], f.values[0], heads, 2, np.arange(85, 90) + 1))
    close(got[5:10], attend(q[5:10], f.keys[1], f.values[1], heads, 2, np.arange(131 - 40, 131 - 35) + 1))
    assert (got[10:] == 5).all()


def test_append_outside_the_cache(fdx):
    """Positions below zero, from max_len on and of pages that are none: not written, reported; the others are."""
    kv, d, page = 1, 8, 4
    x = np.arange(1, 6 * 8 + 1, dtype=np.float32).reshape(6, 8)
    for lens, table, want in (([2, 3], [[0, 1], [2, 3]], {8: 3, 9: 4, 10: 5, 0: 1, 1: 2}), ([9, 3], [[0, 1], [2, 3]], {6: 0, 7: 1, 8: 3, 9: 4, 10: 5}),
                              ([3, 5], [[0, 1], [2, 9]], {0: 0, 1: 1, 2: 2, 10: 3, 11: 4}), ([3, 3], [[-1, 1], [2, 3]], {8: 3, 9: 4, 10: 5})):
        c = fdx.PagedCache(4, page, kv, d, d, 2, 8)
        c.table, c.lens = np.array(table, np.int32), np.array(lens, np.int32)
        pages, dx, starts = c.pages(), fdx.DevBuf.from_host(x), fdx.DevBuf.from_host(np.array([0, 3, 6], np.int32), np.int32)
        flag = fdx.DevBuf.from_host(np.zeros(1, np.int32), np.int32)
        fdx.check(fdx.lib.fdx_kv_append_f32(dx.ptr, ctypes.c_int64(8), dx.ptr, ctypes.c_int64(8), starts.ptr, 6, ctypes.byref(pages), flag.ptr))
        assert flag.to_host((1,), np.int32)[0] == 1
        rows = np.zeros((16, 8), np.float32)
        for row, of in want.items():
            rows[row] = x[of]
        assert np.array_equal(c.k.to_host((16, 8)), rows) and np.array_equal(c.v.to_host((16, 8)), rows)


def test_paged_nan_that_only_later_tokens_see(fdx):
    """Keys and values that a chunk's later tokens see and its earlier ones do not: a NaN there stays with the later ones."""
    for new in ([4], [16], [50], [100]):
        f = Filled(fdx, [150], 2, 64, 64, 16, "f32")
        q = np.random.default_rng(4).standard_normal((new[0], 256)).astype(np.float32)
        base = f.reference(q, new, 4)
        for buf, name in ((f.cache.v, "v"), (f.cache.k, "k")):
            rows = buf.to_host((f.cache.n_pages * 16, 128))
            at = f.cache.table[0][148 // 16] * 16 + 148 % 16
            keep = rows[at, 64].copy()
            rows[at, 64] = np.nan
            odd = fdx.DevBuf.from_host(rows)
            setattr(f.cache, name, odd)
            got = fdx.mha_paged(f.cache, q, new, 4).reshape(new[0], 4, 64)
            setattr(f.cache, name, buf)
            print("paged nan", new, name, flush=True)
            hit = np.zeros(got.shape, bool)
            hit[-2:, 2:, (slice(0, 1) if name == "v" else slice(0, 64))] = True
            assert np.isnan(got[hit]).all()
            close(got[~hit], base.reshape(got.shape)[~hit])


@pytest.mark.parametrize("new", [[4], [60], [140]])
@pytest.mark.parametrize("power", [14, 40, 124])
def test_paged_sizes_behind_the_mask(fdx, new, power):
    """A chunk whose last tokens' keys and values are 2^power times larger than the others'."""
    for name in ("v", "k"):
        f = Filled(fdx, [150], 2, 64, 64, 16, "f32")
        q = np.random.default_rng(4).standard_normal((new[0], 256)).astype(np.float32)
        base = f.reference(q, new, 4)
        buf = f.cache.v if name == "v" else f.cache.k
        rows = buf.to_host((f.cache.n_pages * 16, 128))
        at = f.cache.table[0][np.arange(147, 150) // 16] * 16 + np.arange(147, 150) % 16
        rows[at] *= np.float32(2.0 ** power)
        setattr(f.cache, name, fdx.DevBuf.from_host(rows))
        print("paged behind the mask", new, power, name, flush=True)
        close(fdx.mha_paged(f.cache, q, new, 4)[:-3], base[:-3])


def test_prompts_then_tokens(fdx):
    """The operators as a serving program uses them: prompts at once, their keys and values into the cache, then steps of one token,
    a chunk for one sequence beside them, and the scores of the tokens: the same as one pass over each whole sequence."""
    heads, kv, d, vocab = 8, 2, 64, 501
    r = np.random.default_rng(11)
    prompts, steps = [40, 7, 1, 129], [[1, 1, 1, 1], [1, 30, 0, 1], [1, 1, 1, 1]]
    total = [p + sum(s[i] for s in steps) for i, p in enumerate(prompts)]
    q, k, v = ([r.standard_normal((n, h * d)).astype(np.float32) for n in total] for h in (heads, kv, kv))
    head = r.standard_normal((vocab, heads * d)).astype(np.float32) / 10
    whole = np.split(fdx.mha_packed(np.concatenate(q), np.concatenate(k), np.concatenate(v), total, heads, kv, d, d), np.cumsum(total)[:-1])
    for kind in ("f32", "bf16"):
        cache = fdx.PagedCache(40, 16, kv, d, d, 4, max(total), kind)
        done = [0] * 4
        for new in [prompts] + steps:
            part = lambda xs: np.concatenate([x[a:a + n] for x, a, n in zip(xs, done, new)])
            fdx.kv_append(cache, part(k), part(v), new)
            got = fdx.mha_paged(cache, part(q), new, heads)
            if new is prompts:
                close(got, fdx.mha_packed(part(q), part(k), part(v), new, heads, kv, d, d), 1e-6 if kind == "f32" else 1e-2)
            close(got, part(whole), 2e-6 if kind == "f32" else 1e-2)   # bf16: keys off by 2^-9 a score, values by 2^-9
            logits = fdx.gemm(got, head)
            scores = fdx.token_logprobs(logits, ids=np.arange(len(got)) % vocab, top=3)
            x = logits.astype(np.float64)
            lp = x - np.log(np.exp(x - x.max(1, keepdims=True)).sum(1, keepdims=True)) - x.max(1, keepdims=True)
            assert np.abs(scores["logprobs"] - lp[np.arange(len(got)), np.arange(len(got)) % vocab]).max() < 1e-5
            assert np.array_equal(scores["top_ids"][:, 0], fdx.argmax(logits)[0])
            done = [a + n for a, n in zip(done, new)]
        for s in range(4):
            cache.release(s)
        assert sorted(cache.free) == list(range(40))


@pytest.mark.parametrize("n_seqs", [63, 64, 65, 300])
def test_many_sequences(fdx, n_seqs):
    """Lengths of 0 to 9 and two longer ones somewhere, as prompts and as the newest tokens of caches."""
    r = np.random.default_rng(n_seqs)
    lengths = r.integers(0, 10, n_seqs).tolist()
    lengths[n_seqs // 3], lengths[n_seqs - 2] = 150, 70
    heads, kv, d = 4, 2, 64
    print("many sequences", n_seqs, flush=True)
    q, k, v = (r.standard_normal((sum(lengths), h * d)).astype(np.float32) for h in (heads, kv, kv))
    for causal in (True, False):
        close(fdx.mha_packed(q, k, v, lengths, heads, kv, d, d, causal), packed_reference(q, k, v, lengths, heads, kv, causal))
    new = [min(n, int(m)) for n, m in zip(lengths, r.integers(0, 12, n_seqs))]
    new[n_seqs // 3] = 90
    f = Filled(fdx, lengths, kv, d, d, 8, "f32", seed=1, max_len=2000)
    q = r.standard_normal((sum(new), heads * d)).astype(np.float32)
    close(fdx.mha_paged(f.cache, q, new, heads), f.reference(q, new, heads))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("context,new,heads,kv,d", [([5000, 40], [1, 1], 4, 2, 64), ([3000, 2900, 700], [40, 1, 100], 8, 2, 128),
                                                    ([2600, 1], [2, 1], 6, 6, 64), ([4500], [600], 2, 1, 128), ([1500, 0, 900], [33, 0, 3], 32, 1, 64)])
def test_paged_long_contexts(fdx, context, new, heads, kv, d, kind):
    """Keys in ranges over several workgroups; pages of sixteen, and of a size that divides nothing."""
    for page in (16, 37):
        print("paged long", context, new, heads, kv, d, page, kind, flush=True)
        f = Filled(fdx, context, kv, d, d, page, kind, seed=sum(context), steps=1)
        q = np.random.default_rng(d).standard_normal((sum(new), heads * d)).astype(np.float32)
        close(fdx.mha_paged(f.cache, q, new, heads), f.reference(q, new, heads))
        first = fdx.mha_paged(f.cache, q, new, heads)
        assert np.array_equal(first, fdx.mha_paged(f.cache, q, new, heads))


def test_scratch_holds_anything_before_a_call(fdx):
    """Key ranges and split prompts in memory full of NaN; a second call in the same memory right behind the first."""
    heads, kv, d = 16, 1, 64
    f = Filled(fdx, [2500, 700], kv, d, d, 16, "f32", steps=1)
    r = np.random.default_rng(3)
    q = r.standard_normal((41, heads * d)).astype(np.float32)
    dq, out, c = fdx.DevBuf.from_host(q), [fdx.DevBuf(q.nbytes) for _ in range(2)], f.cache.pages()
    starts = fdx.DevBuf.from_host(np.array([0, 1, 41], np.int32), np.int32)
    need = fdx.lib.fdx_mha_paged_scratch_bytes(41, 40, heads, ctypes.byref(c))
    assert need > 0
    scratch = noise(fdx, need)
    for o in out:
        fdx.check(fdx.lib.fdx_mha_paged_f32(dq.ptr, ctypes.c_int64(heads * d), starts.ptr, 41, 40, heads, ctypes.byref(c), o.ptr, ctypes.c_int64(heads * d),
                                            scratch.ptr, None))
    want = f.reference(q, [1, 40], heads)
    close(out[0].to_host(q.shape), want)
    assert np.array_equal(out[0].to_host(q.shape), out[1].to_host(q.shape))
    n = 300
    q, k, v = (r.standard_normal((n, h * d)).astype(np.float32) for h in (heads, kv, kv))
    assert fdx.lib.fdx_mha_packed_scratch_bytes(n, 1, heads, kv, d, d) > 0
    bufs, o = [fdx.DevBuf.from_host(x) for x in (q, k, v)], fdx.DevBuf(q.nbytes)
    assert call_packed(fdx, bufs[0].ptr, heads * d, bufs[1].ptr, d, bufs[2].ptr, d, [0, n], n, heads, kv, d, d, o.ptr, heads * d) == 0
    close(o.to_host(q.shape), packed_reference(q, k, v, [n], heads, kv, True))


def test_two_threads(fdx):
    """Calls of two host threads, each with memory of its own."""
    import threading
    f, heads = Filled(fdx, [1200, 90], 2, 64, 64, 16, "bf16", steps=1), 8
    r = np.random.default_rng(5)
    qs = [r.standard_normal((n, heads * 64)).astype(np.float32) for n in (2, 61)]
    new = [[1, 1], [60, 1]]
    want, got, wrong = [f.reference(q, n, heads) for q, n in zip(qs, new)], [[], []], []

    def work(i):
        try:
            for _ in range(10):
                got[i].append(fdx.mha_paged(f.cache, qs[i], new[i], heads))
        except Exception as e:   # reported below, by the test's own thread
            wrong.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong, wrong
    for i in range(2):
        close(got[i][0], want[i])
        assert all(np.array_equal(got[i][0], x) for x in got[i])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_offsets_beyond_32_bits(fdx, kind):
    """Pages whose rows start beyond 2^32 elements of the cache."""
    heads, kv, d, page, context, new = 16, 8, 128, 16, [90, 40], [1, 33]
    n_pages = (1 << 32) // (page * kv * d) + 20
    size = n_pages * page * kv * d * (4 if kind == "f32" else 2)
    c = fdx.PagedCache(1, page, kv, d, d, 2, 100, kind)
    c.n_pages, c.k, c.v, c.free = n_pages, fdx.DevBuf(size), fdx.DevBuf(size), [*range(n_pages - 8, n_pages), 3, n_pages // 2 + 1]
    r = np.random.default_rng(12)
    keys, values = ([r.standard_normal((n, kv * d)).astype(np.float32) for n in context] for _ in range(2))
    print("far pages", kind, flush=True)
    fdx.kv_append(c, np.concatenate(keys), np.concatenate(values), context)
    if kind == "bf16":
        keys, values = [bf16(x) for x in keys], [bf16(x) for x in values]
    q = r.standard_normal((sum(new), heads * d)).astype(np.float32)
    got = fdx.mha_paged(c, q, new, heads)
    c.k.free()
    c.v.free()
    close(got[:1], attend(q[:1], keys[0], values[0], heads, kv, np.array([90])))
    close(got[1:], attend(q[1:], keys[1], values[1], heads, kv, np.arange(40 - 33, 40) + 1))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("new", [1, 70])
def test_a_long_sequence(fdx, new, kind):
    """Three million positions, all of them in five pages: the row at position p is row p % 80, so the softmax over all positions is that
    over 80 rows, each with its number of times.  A range has 3e6 / 16 keys or fewer, a wave's accumulators take 2930 tiles of 64 of them in
    12 additions each, the sums of weights 16: at most (12 + 16) 2930 roundings of 2^-24 to sums of terms of one sign and size, 5e-3
    of the largest value."""
    length, heads, d, page = 3000000, 2, 64, 16
    r = np.random.default_rng(13)
    rows = [r.standard_normal((80, d)).astype(np.float32) for _ in range(2)]
    c = fdx.PagedCache(5, page, 1, d, d, 1, length, kind)
    fdx.kv_append(c, rows[0], rows[1], [80])
    first = c.table[0][:5].copy()
    c.table[0][:] = first[np.arange(c.table.shape[1]) % 5]
    c.lens[0] = length
    k, v = (x.astype(np.float64) if kind == "f32" else bf16(x).astype(np.float64) for x in rows)
    q = r.standard_normal((new, heads * d)).astype(np.float32)
    print("long", new, kind, flush=True)
    got = fdx.mha_paged(c, q, [new], heads).reshape(new, heads, d)
    sees = np.arange(length - new, length) + 1
    times = sees[:, None] // 80 + (np.arange(80)[None] < sees[:, None] % 80)
    s = q.reshape(new, heads, d).astype(np.float64) @ k.T / np.sqrt(d)
    p = np.exp(s - s.max(-1, keepdims=True)) * times[:, None]
    want = p @ v / p.sum(-1, keepdims=True)
    assert np.abs(got - want).max() <= 5e-3 * np.abs(v).max()


def test_shapes_that_do_not_fit(fdx):
    x = np.zeros((5, 128), np.float32)
    with pytest.raises(fdx.FdxError, match="k of shape"):
        fdx.mha_packed(x, x[:4], x, [5], 2, 2, 64, 64)
    c = fdx.PagedCache(4, 16, 2, 64, 64, 1, 40)
    with pytest.raises(fdx.FdxError, match="v of shape"):
        fdx.kv_append(c, x, x[:, :64], [5])
    with pytest.raises(fdx.FdxError, match="at most 40"):
        fdx.kv_append(c, np.zeros((41, 128), np.float32), np.zeros((41, 128), np.float32), [41])
    fdx.kv_append(c, x, x, [5])
    with pytest.raises(fdx.FdxError, match="q of shape"):
        fdx.mha_paged(c, x[:3], [5], 2)
    for lengths in ([5, 0], [], [-5], [[5]], 5):
        with pytest.raises(fdx.FdxError, match="1 sequences need"):
            fdx.mha_paged(c, x, lengths, 2)
        with pytest.raises(fdx.FdxError, match="1 sequences need"):
            fdx.kv_append(c, x, x, lengths)
    with pytest.raises(fdx.FdxError, match="lengths of the packed"):
        fdx.mha_packed(x, x, x, [7, -2], 2, 2, 64, 64)
    with pytest.raises(fdx.FdxError, match="free pages"):
        d = fdx.PagedCache(1, 16, 2, 64, 64, 2, 40)
        d.grow([16, 1])
    with pytest.raises(fdx.FdxError, match="overlap"):
        fdx.check(fdx.lib.fdx_kv_append_f32(c.k.ptr, ctypes.c_int64(3), c.v.ptr, ctypes.c_int64(128), c.k.ptr, 1, ctypes.byref(c.pages()), None))


def test_packed_rows_beyond_32_bits(fdx):
    """Rows of q, k, v and out so far apart that the last ones start beyond 2^32 floats."""
    n, heads, kv, d, ld = 150, 4, 2, 64, (1 << 32) // 140
    r = np.random.default_rng(14)
    q, k, v = (r.standard_normal((n, h * d)).astype(np.float32) for h in (heads, kv, kv))
    buf = fdx.DevBuf(4 * (ld * (n - 1) + 1024))   # columns: q, k, v, out
    at = [0, heads * d, (heads + kv) * d, (heads + 2 * kv) * d]
    print("packed far rows", flush=True)
    for i in range(n):
        row = np.concatenate([q[i], k[i], v[i]])
        fdx.check(fdx.lib.fdx_h2d(ctypes.c_void_p(buf.ptr.value + 4 * ld * i), row.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(row.nbytes)))
    p = [ctypes.c_void_p(buf.ptr.value + 4 * x) for x in at]
    for lengths in ([150], [10, 140]):
        starts = [0, *np.cumsum(lengths).tolist()]
        assert call_packed(fdx, p[0], ld, p[1], ld, p[2], ld, starts, n, heads, kv, d, d, p[3], ld) == 0
        got = np.zeros((n, heads * d), np.float32)
        for i in range(n):
            fdx.check(fdx.lib.fdx_d2h(got[i].ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(p[3].value + 4 * ld * i), ctypes.c_size_t(got[i].nbytes)))
        close(got, packed_reference(q, k, v, lengths, heads, kv, True))
    buf.free()


def far_scores(r, n, heads, kv, d, e=80):
    """Queries and keys whose largest elements, 2^80, meet zeros, so that a product's scale passes fp32's range (the sum of the exponents is more
    than 156) while its scores, products of 2^60 and -2^60, all equal and about -2^117, do not: with equal scores a row's result is the mean of the
    values it sees.  Powers of two, so that nothing is rounded."""
    q, k = np.zeros((n, heads, d), np.float32), np.zeros((n, kv, d), np.float32)
    q[:, :, 0], k[:, :, 1] = 2.0 ** e, 2.0 ** e
    q[:, :, 2], k[:, :, 2] = -2.0 ** 60, 2.0 ** 60
    return q.reshape(n, -1), k.reshape(n, -1), r.standard_normal((n, kv * d)).astype(np.float32)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,heads,kv_heads", [([40, 1, 150], 4, 2), ([300], 7, 1), ([1500], 4, 4), ([400], 6, 1), ([511, 300, 0, 1], 16, 1), ([2100], 1, 1)])
@pytest.mark.parametrize("d", [64, 128])
def test_packed_scores_far_below_zero(fdx, lengths, heads, kv_heads, d, causal):
    """No score is near zero: a row's sums are those of its largest scores, however small these are.  Sequences in tiles, in ranges of keys, and
    with keys that are split once.  The mean of n values that are added in a chain: 0.42 * 2^-24 of the partial sum, some sqrt(i), a step, so
    0.3 * 2^-24 sqrt(n) of the result, 8e-7 for 2100; twice the usual bound."""
    print("packed far below zero", lengths, heads, kv_heads, d, causal, flush=True)
    q, k, v = far_scores(np.random.default_rng(15), sum(lengths), heads, kv_heads, d)
    close(fdx.mha_packed(q, k, v, lengths, heads, kv_heads, d, d, causal), packed_reference(q, k, v, lengths, heads, kv_heads, causal), 2e-6)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("context,new", [([90], [1]), ([300, 17], [5, 1]), ([150], [60]), ([150, 700], [1, 140]), ([2500, 64], [70, 64])])
def test_paged_scores_far_below_zero(fdx, context, new, kind):
    heads, kv, d, page = 4, 2, 64, 16
    r, total = np.random.default_rng(16), sum(context)
    q, k, v = far_scores(r, total, heads, kv, d)
    q = q[:sum(new)]
    print("paged far below zero", context, new, kind, flush=True)
    cache = fdx.PagedCache(sum(-(-n // page) for n in context), page, kv, d, d, len(context), max(context), kind)
    fdx.kv_append(cache, k, v, context)
    if kind == "bf16":
        v = bf16(v)
    want, at, row = [], 0, 0
    for length, n in zip(context, new):
        want.append(attend(q[row:row + n], k[at:at + length], v[at:at + length], heads, kv, np.arange(length - n, length) + 1))
        at, row = at + length, row + n
    close(fdx.mha_paged(cache, q, new, heads), np.concatenate(want), 2e-6)


@pytest.mark.parametrize("new", [1, 4, 60])
def test_scores_far_below_zero_beside_others(fdx, new):
    """Scores of -2^110 / 8, and one of -2^102 / 8 in a tile whose keys' scale passes fp32's range: the row sees that one alone.  (2^42 beside
    2^80 is the last bit that a tile of keys holds.)"""
    heads, kv, d, n = 4, 2, 64, 192
    q, k, v = far_scores(np.random.default_rng(17), n, heads, kv, d)
    k = k.reshape(n, kv, d)
    k[:, :, 1], k[:, :, 2] = 2.0 ** 60, 2.0 ** 50
    k[64:128, :, 1] = 2.0 ** 68   # near enough to 2^80 for one scale
    k[70, :, 1], k[70, :, 2] = 2.0 ** 80, 2.0 ** 42
    k = k.reshape(n, -1)
    for lengths in ([n], [100, 92]):
        print("far below zero beside others", lengths, flush=True)
        close(fdx.mha_packed(q, k, v, lengths, heads, kv, d, d), packed_reference(q, k, v, lengths, heads, kv, True))
    cache = fdx.PagedCache(12, 16, kv, d, d, 1, n)
    fdx.kv_append(cache, k, v, [n])
    close(fdx.mha_paged(cache, q[-new:], [new], heads), attend(q[-new:], k, v, heads, kv, np.arange(n - new, n) + 1))


@pytest.mark.parametrize("sign", [1, -1])
def test_scores_past_the_range_of_fp32(fdx, sign):
    """Scores of +-2^160: infinite in fp32, all of them, so no row has a softmax; NaN whatever path takes it."""
    heads, kv, d = 4, 2, 64
    for lengths, h, g in (([40, 30], heads, kv), ([400], 6, 1), ([1500], 4, 4)):
        n = sum(lengths)
        q, k, v = np.full((n, h * d), sign * 2.0 ** 80, np.float32), np.full((n, g * d), 2.0 ** 80, np.float32), np.ones((n, g * d), np.float32)
        print("scores past fp32", sign, lengths, flush=True)
        assert np.isnan(fdx.mha_packed(q, k, v, lengths, h, g, d, d)).all()
    cache = fdx.PagedCache(10, 16, kv, d, d, 1, 160)
    fdx.kv_append(cache, np.full((150, kv * d), 2.0 ** 80, np.float32), np.ones((150, kv * d), np.float32), [150])
    for new in (1, 5, 60, 140):
        assert np.isnan(fdx.mha_paged(cache, np.full((new, heads * d), sign * 2.0 ** 80, np.float32), [new], heads)).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_paged_ranges_of_many_tokens(fdx, kind):
    """2000 tiles in a cache of up to 131 072 positions: eight ranges of 16 384 keys, no more than scratch memory of 1 GiB holds; a few rows of
    each sequence are looked at.  Bound: 5e-7 of the operands as above; an accumulator adds three products for 16 keys, 1880 in a range of 10 000 keys,
    each rounded by 0.29 of the last bit, some 0.42 * 2^-24 of a partial sum that grows with their root: 0.42 * 2^-24 sqrt(1880 / 2) = 8e-7 of the
    result; sqrt(5^2 + 8^2) e-7 = 9.4e-7 are to be expected, twice that allowed."""
    context, new, heads, kv, d = [20000, 16500, 300], [3900, 60, 40], 64, 8, 64
    print("paged ranges of many tokens", kind, flush=True)
    f = Filled(fdx, context, kv, d, d, 64, kind, seed=18, steps=1, max_len=131072)
    q = np.random.default_rng(19).standard_normal((sum(new), heads * d)).astype(np.float32)
    got, at = fdx.mha_paged(f.cache, q, new, heads), 0
    for s, n in enumerate(new):
        rows = np.unique([0, n // 3, n - 1])
        sees = context[s] - n + 1 + rows
        close(got[at + rows], attend(q[at + rows], f.keys[s], f.values[s], heads, kv, sees), 2e-6)
        at += n


@pytest.mark.parametrize("heads", [4, 40])
def test_paged_lengths_of_sequences_without_new_tokens(fdx, heads):
    """A length that is none is reported whether its sequence brings rows or not, also where many heads share a key head; the others' rows are right."""
    kv, d = 1, 64
    f = Filled(fdx, [90, 131, 20], kv, d, d, 16, "f32")
    for new in ([1, 0, 1], [50, 0, 1]):
        tokens = sum(new)
        q = np.random.default_rng(20).standard_normal((tokens, heads * d)).astype(np.float32)
        dq, out = fdx.DevBuf.from_host(q), fdx.DevBuf(q.nbytes)
        for length, flag in ((131, 0), (132, 1), (-1, 1), (0, 0), (2**31 - 1, 1), (-2**31, 1)):
            print("paged lengths without tokens", heads, new, length, flush=True)
            assert call_paged(fdx, f.cache, dq.ptr, heads * d, np.concatenate([[0], np.cumsum(new)]), tokens, max(new), heads, out.ptr, heads * d,
                              lens=[90, length, 20]) == flag
            close(out.to_host(q.shape), np.concatenate([attend(q[:new[0]], f.keys[0], f.values[0], heads, kv, np.arange(90 - new[0], 90) + 1),
                                                        attend(q[new[0]:], f.keys[2], f.values[2], heads, kv, np.array([20]))]))


def fastest(fdx, call):
    """Seconds of a call, the best of four."""
    import time
    best = 1e9
    for _ in range(4):
        fdx.sync()
        start = time.perf_counter()
        call()
        fdx.sync()
        best = min(best, time.perf_counter() - start)
    return best


ZEROS = [(0, 128), (64, 192), (256, 320), (0, 64), (300, 500), (0, 500), (37, 300)]


@pytest.mark.parametrize("first,last", ZEROS)
@pytest.mark.parametrize("lengths,heads,kv_heads,d", [([520, 30], 4, 2, 64), ([520, 30], 4, 2, 128), ([600], 6, 1, 64), ([600], 16, 1, 128), ([1500], 4, 4, 64)])
def test_packed_values_of_zeros(fdx, lengths, heads, kv_heads, d, first, last):
    """Whole tiles of values that are zeros, in front of, between and behind values of sizes that differ by 2^40."""
    for causal in (True, False):
        print("packed zeros", lengths, heads, kv_heads, d, first, last, causal, flush=True)
        r, n = np.random.default_rng(21), sum(lengths)
        q, k, v = (r.standard_normal((n, h * d)).astype(np.float32) for h in (heads, kv_heads, kv_heads))
        v[first:last] = 0
        close(fdx.mha_packed(q, k, v, lengths, heads, kv_heads, d, d, causal), packed_reference(q, k, v, lengths, heads, kv_heads, causal))
        v[last:] *= np.float32(2.0 ** -40)
        got, want = fdx.mha_packed(q, k, v, lengths, heads, kv_heads, d, d, causal), packed_reference(q, k, v, lengths, heads, kv_heads, causal)
        close(got, want)
        v[:] = 0
        assert (fdx.mha_packed(q, k, v, lengths, heads, kv_heads, d, d, causal) == 0).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("new", [1, 9, 60, 300])
def test_paged_values_of_zeros(fdx, new, kind):
    heads, kv, d, page, length = 4, 2, 64, 16, 1200
    for first, last in ZEROS + [(0, length)]:
        f = Filled(fdx, [length], kv, d, d, page, kind, steps=1)
        f.values[0][first:last] = 0
        f.cache.release(0)
        fdx.kv_append(f.cache, f.keys[0], f.values[0], [length])
        q = np.random.default_rng(22).standard_normal((new, heads * d)).astype(np.float32)
        print("paged zeros", new, kind, first, last, flush=True)
        close(fdx.mha_paged(f.cache, q, [new], heads), f.reference(q, [new], heads))


@pytest.mark.parametrize("n,heads,kv_heads", [(2048, 12, 12), (2048, 16, 4)])
def test_packed_values_of_zeros_take_no_longer(fdx, n, heads, kv_heads):
    """No row by row sums because of them, which take a hundred times as long; ten leaves room for a disturbed call."""
    d, r = 64, np.random.default_rng(23)
    q, k, v = (r.standard_normal((n, h * d)).astype(np.float32) for h in (heads, kv_heads, kv_heads))
    dq, dk, out, times = fdx.DevBuf.from_host(q), fdx.DevBuf.from_host(k), fdx.DevBuf(q.nbytes), []
    scratch, starts = fdx.DevBuf(fdx.lib.fdx_mha_packed_scratch_bytes(n, 1, heads, kv_heads, d, d)), fdx.DevBuf.from_host(np.array([0, n], np.int32), np.int32)
    i64 = ctypes.c_int64
    for first, last in ((0, 0), (0, 128), (1024, 1152)):
        v[first:last] = 0
        dv = fdx.DevBuf.from_host(v)
        times.append(fastest(fdx, lambda: fdx.check(fdx.lib.fdx_mha_packed_f32(dq.ptr, i64(heads * d), dk.ptr, i64(kv_heads * d), dv.ptr, i64(kv_heads * d),
                                                                              starts.ptr, 1, n, heads, kv_heads, d, d, 1, out.ptr, i64(heads * d),
                                                                              scratch.ptr, None))))
    print("times in us", [round(1e6 * t) for t in times], flush=True)
    assert max(times[1:]) < 10 * times[0]


def test_paged_values_of_zeros_take_no_longer(fdx):
    heads, kv, d, page, length, new = 12, 12, 64, 64, 2000, 300
    f, times = Filled(fdx, [length], kv, d, d, page, "f32", steps=1), []
    q = fdx.DevBuf.from_host(np.random.default_rng(24).standard_normal((new, heads * d)).astype(np.float32))
    out, starts = fdx.DevBuf(4 * new * heads * d), fdx.DevBuf.from_host(np.array([0, new], np.int32), np.int32)
    for first, last in ((0, 0), (1024, 1280)):
        f.values[0][first:last] = 0
        f.cache.release(0)
        fdx.kv_append(f.cache, f.keys[0], f.values[0], [length])
        c = f.cache.pages()
        scratch = fdx.DevBuf(fdx.lib.fdx_mha_paged_scratch_bytes(new, new, heads, ctypes.byref(c)))
        times.append(fastest(fdx, lambda: fdx.check(fdx.lib.fdx_mha_paged_f32(q.ptr, ctypes.c_int64(heads * d), starts.ptr, new, new, heads, ctypes.byref(c),
                                                                             out.ptr, ctypes.c_int64(heads * d), scratch.ptr, None))))
    print("times in us", [round(1e6 * t) for t in times], flush=True)
    assert times[1] < 10 * times[0]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("new", [1, 70])
def test_every_part_of_a_long_sequence_counts_once(fdx, new, kind):
    """Three million positions of which two pages decide: their keys score 40 above the rest, their values are their own.  A range of keys that were
    left out, summed twice or read from elsewhere would change the share of its page, wherever that lies, by a sixth or more of the values.
    Scores of 320 / 8 are chains of 64 sums (three products each in tiles) of up to 320, each off by up to 2^-24 * 320: at most 192 * 2.4e-6 = 5e-4 of a
    probability; 1e-3 of the largest value for that and the sums of the rest (e^-40 * 3e6 of the whole)."""
    length, heads, d, page = 3000000, 2, 64, 16
    r, n_pages = np.random.default_rng(25), 3000000 // 16
    keys, values = (r.standard_normal((7 * page, d)).astype(np.float32) for _ in range(2))   # pages 0 to 4 everywhere, 5 and 6 once each
    keys[:, 0] = 0
    keys[5 * page:, 0] = 40
    c = fdx.PagedCache(7, page, 1, d, d, 1, length, kind)
    fdx.kv_append(c, keys, values, [7 * page])
    first = c.table[0][:7].copy()
    c.lens[0] = length
    q = r.standard_normal((new, heads * d)).astype(np.float32)
    q[:, ::d] = 8
    k, v = (x[5 * page:].astype(np.float64) if kind == "f32" else bf16(x)[5 * page:].astype(np.float64) for x in (keys, values))
    s = q.reshape(new, heads, d).astype(np.float64) @ k.T / np.sqrt(d)
    p = np.exp(s - s.max(-1, keepdims=True))
    want = p @ v / p.sum(-1, keepdims=True)
    # the last pages hold keys that not every row sees
    last = n_pages - 6
    places = sorted({0, 1, last} | {last * i // 71 for i in range(72)} | {int(x) for x in r.integers(0, last, 20)})
    for at in places:
        other = (at + last // 2 + 1) % last
        c.table[0][:] = first[np.arange(n_pages) % 5]
        c.table[0][at], c.table[0][other] = first[5], first[6]
        got = fdx.mha_paged(c, q, [new], heads).reshape(new, heads, d)
        assert np.abs(got - want).max() <= 1e-3 * np.abs(v).max(), (at, np.abs(got - want).max())


@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("name,row", [("v", 333), ("v", 399), ("v", 0), ("k", 333)])
def test_packed_split_once_values_beside_infinities_and_nan(fdx, what, name, row):
    """The other depths of rows that see a NaN or an infinity among the values, and every depth behind a key of -infinity's score."""
    r, n, heads, kv = np.random.default_rng(9), 400, 8, 1
    q, k, v = (r.standard_normal((n, h * 64)).astype(np.float32) for h in (heads, kv, kv))
    print("packed once beside", what, name, row, flush=True)
    dict(k=k, v=v)[name][row, 7] = what
    got = fdx.mha_packed(q, k, v, [n], heads, kv, 64, 64)
    with np.errstate(all="ignore"):
        want = packed_reference(q, k, v, [n], heads, kv, True)
    ok = np.isfinite(want)
    assert np.array_equal(np.isfinite(got), ok)
    close(got[ok], want[ok])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("parts", [2, 3, 4, 5, 6, 7, 9, 12, 15, 16, 17, 18])
def test_paged_infinite_values_in_one_of_several_ranges(fdx, parts, kind):
    """One token over ranges of 256 keys, a value of one of them infinite: so is the mean of its depth, and nothing else, whichever range it is."""
    n, kv, d, heads = 256 * parts, 2, 64, 4
    r = np.random.default_rng(parts)
    k, v = (r.standard_normal((n, kv * d)).astype(np.float32) for _ in range(2))
    q = r.standard_normal((1, heads * d)).astype(np.float32)
    cache = fdx.PagedCache(-(-n // 64), 64, kv, d, d, 1, n, kind)
    base = attend(q, *((k, v) if kind == "f32" else (bf16(k), bf16(v))), heads, kv, [n]).reshape(heads, d)
    for part in range(parts):
        x, what = v.copy(), (-1) ** part * np.inf
        x[256 * part + 5, 7] = what
        cache.release(0)
        fdx.kv_append(cache, k, x, [n])
        print("paged infinity in a range", parts, part, kind, flush=True)
        got = fdx.mha_paged(cache, q, [1], heads).reshape(heads, d)
        assert (got[:2, 7] == what).all(), (part, got[:2, 7])   # heads of key head 0
        got[:2, 7] = base[:2, 7]
        close(got, base)


@pytest.mark.parametrize("n", [700, 1100, 2000])
def test_packed_infinite_values_in_one_of_several_ranges(fdx, n):
    """The same for a prompt whose tiles are cut in ranges."""
    r, heads = np.random.default_rng(8), 6
    q, k, v = (r.standard_normal((n, h * 64)).astype(np.float32) for h in (heads, 1, 1))
    base = packed_reference(q, k, v, [n], heads, 1, True).reshape(n, heads, 64)
    for row in range(5, n, 128):
        x = v.copy()
        x[row, 7] = np.inf
        print("packed infinity in a range", n, row, flush=True)
        got = fdx.mha_packed(q, k, x, [n], heads, 1, 64, 64).reshape(n, heads, 64)
        assert (got[row:, :, 7] == np.inf).all() and np.isfinite(got[:row]).all()
        got[row:, :, 7] = base[row:, :, 7]
        close(got, base)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("new", [1, 12, 100])
@pytest.mark.parametrize("keys,least", [(300, -1), (900, -1), (900, 0.99), (3000, 0.9)])
def test_paged_values_near_the_end_of_fp32(fdx, keys, least, new, kind):
    """Values up to 3.2e38, also all of one sign, over one range of keys and over several: results are means, none passes fp32's range.  The keys of
    either half have one score, so its error is common to them."""
    heads, kv, d = 4, 2, 64
    k, v = np.zeros((keys, kv * d), np.float32), (3.2e38 * np.random.default_rng(2).uniform(least, 1, (keys, kv * d))).astype(np.float32)
    k[keys // 2:, ::d] = 7.9 * np.log(2) * 8
    cache = fdx.PagedCache(-(-keys // 16), 16, kv, d, d, 1, keys, kind)
    fdx.kv_append(cache, k, v, [keys])
    q = np.zeros((new, heads * d), np.float32)
    q[:, ::d] = 1
    print("paged largest values", keys, least, new, kind, flush=True)
    got = fdx.mha_paged(cache, q, [new], heads).astype(np.float64)
    want = attend(q, *((k, v) if kind == "f32" else (bf16(k), bf16(v))), heads, kv, np.arange(keys - new, keys) + 1)
    close(np.ldexp(got, -127), np.ldexp(want, -127))


@pytest.mark.parametrize("n,heads", [(300, 6), (700, 6), (2000, 6), (2100, 1)])
@pytest.mark.parametrize("least", [-1, 0.99])
def test_packed_values_near_the_end_of_fp32(fdx, n, heads, least):
    """The same for prompts."""
    r = np.random.default_rng(3)
    q, k = (r.standard_normal((n, h * 64)).astype(np.float32) for h in (heads, 1))
    v = (3.2e38 * r.uniform(least, 1, (n, 64))).astype(np.float32)
    print("packed largest values", n, heads, least, flush=True)
    got = fdx.mha_packed(q, k, v, [n], heads, 1, 64, 64).astype(np.float64)
    close(np.ldexp(got, -127), np.ldexp(packed_reference(q, k, v, [n], heads, 1, True), -127))
