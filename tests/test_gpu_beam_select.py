"""The best continuations over beams and vocabulary, against totals in 64 bits.

The order is decided in 64 bits on sums that the kernel has to about 1e-7, so two candidates of different beams that are nearer than that may
change places: inputs are drawn so that no two of a sequence's totals near the cut are nearer than 4e-6.  Scores are rounded once to fp32, 2^-24 of
their size, and carry the error of a row's sum, about 2^-24 for each of a few terms that carry it: 4e-7 + 2^-23 of the size."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def totals_of(x, scores, done, end_id):
    """every continuation of a sequence as (total, beam, -logit, token), best first"""
    out = []
    for b in range(x.shape[0]):
        if not np.isfinite(scores[b]):
            continue
        if done is not None and done[b]:
            out.append((float(scores[b]), b, 0.0, end_id))
            continue
        row = x[b].astype(np.float64)
        if np.isnan(row).any() or (row == np.inf).any() or (row == -np.inf).all():
            continue
        lse = row.max() + np.log(np.exp(row - row.max()).sum())
        near = np.argsort(-row, kind="stable")[:40]
        out += [(float(scores[b]) + (row[t] - lse), b, -row[t], int(t)) for t in near if row[t] > -np.inf]
    return sorted(out, key=lambda c: (-c[0], c[1], c[2], c[3]))


def expect(x, scores, keep, done=None, end_id=-1, near_ok=False):
    n, beams, _ = x.shape
    parents, tokens, best = np.full((n, keep), -1), np.full((n, keep), -1), np.full((n, keep), -np.inf)
    ended = np.zeros((n, keep), int)
    for s in range(n):
        every = totals_of(x[s], scores[s], None if done is None else done[s], end_id)
        gaps = [a[0] - b[0] for a, b in zip(every, every[1:keep + 1]) if a[1] != b[1]]
        assert near_ok or not gaps or min(gaps) > 4e-6, "draw other inputs"
        for j, (total, b, _, t) in enumerate(every[:keep]):
            parents[s, j], tokens[s, j], best[s, j] = s * beams + b, t, total
            ended[s, j] = t == end_id or (done is not None and bool(done[s, b]))
    return parents, tokens, best, ended


def check(fdx, x, scores, keep, done=None, end_id=-1, near_ok=False):
    parents, tokens, best, ended = expect(x, scores, keep, done, end_id, near_ok)
    got = fdx.beam_select(x, scores, keep, done, end_id)
    assert np.array_equal(got["parents"], parents), (got["parents"], parents)
    assert np.array_equal(got["tokens"], tokens), (got["tokens"], tokens)
    there = best > -np.inf
    assert (got["scores"][~there] == -np.inf).all()
    off = np.abs(got["scores"][there].astype(np.float64) - best[there])
    assert (off <= 4e-7 + 2.0 ** -23 * np.abs(best[there])).all(), off.max()
    if end_id >= 0:
        assert np.array_equal(got["done"], ended)


def draw(seed, n, beams, vocab, size=2.5, keep=None, done=None, end_id=-1, **how):
    """logits and scores without two totals near each other: the first such draw from the seed on"""
    for more in range(20):
        r = np.random.default_rng(1000 * seed + more)
        x = (size * r.standard_normal((n, beams, vocab))).astype(np.float32)
        if how.get("masked"):
            x[r.random(x.shape) < how["masked"]] = -np.inf
        scores = -np.sort(r.uniform(0, 3, (n, beams)), 1).astype(np.float32) - 5
        try:
            expect(x, scores, keep or beams, done, end_id)
            return x, scores
        except AssertionError:
            pass
    raise AssertionError("no draw without near totals")


@pytest.mark.parametrize("n,beams,vocab,keep", [
    (1, 1, 1, 1), (1, 1, 5, 5), (1, 4, 50257, 4), (3, 2, 7, 14), (2, 5, 64, 10), (4, 3, 255, 6), (2, 3, 256, 1), (2, 3, 257, 32), (1, 32, 1000, 32), (5, 4, 4096, 8),
    (3, 4, 4097, 4), (2, 8, 8192, 16), (7, 5, 10007, 10), (1, 2, 131072, 4), (40, 4, 3001, 4), (1, 16, 40000, 31), (130, 2, 1025, 4), (300, 8, 2000, 8), (2, 31, 1500, 7)])
def test_select(fdx, n, beams, vocab, keep):
    print("beam", n, beams, vocab, keep, flush=True)
    x, scores = draw(vocab, n, beams, vocab, keep=keep)
    check(fdx, x, scores, keep)


@pytest.mark.parametrize("size", [0.01, 1.0, 30.0])
def test_sizes_of_logits(fdx, size):
    print("beam size", size, flush=True)
    x, scores = draw(5, 3, 4, 20000 if size > 0.1 else 300, size=size, keep=8)
    check(fdx, x, scores, 8)
    check(fdx, x + np.float32(1000), scores, 8, near_ok=True) if size == 30.0 else None


def test_first_step(fdx):
    """All beams equal, all but the first dead."""
    x, _ = draw(6, 4, 1, 5000, keep=8)
    x = np.repeat(x, 4, 1)
    scores = np.full((4, 4), -np.inf, np.float32)
    scores[:, 0] = 0
    check(fdx, x, scores, 4)
    check(fdx, x, scores, 8)
    # and with equal scores every total is there four times: the lowest beam first
    got = fdx.beam_select(x, np.zeros((4, 4), np.float32), 8)
    assert np.array_equal(got["parents"], np.tile(np.arange(4), 2)[None] + 4 * np.arange(4)[:, None])
    assert (got["tokens"][:, :4] == got["tokens"][:, :1]).all() and (got["tokens"][:, 4:] == got["tokens"][:, 4:5]).all()


@pytest.mark.parametrize("masked", [0.5, 0.99, 0.9995])
def test_ruled_out_tokens(fdx, masked):
    x, scores = draw(8, 5, 4, 9000, keep=16, masked=masked)
    check(fdx, x, scores, 16)


def test_nothing_left(fdx):
    """Rows of ruled-out tokens, dead beams, sequences without a continuation, fewer continuations than asked for."""
    x, scores = np.full((4, 3, 3000), -np.inf, np.float32), np.full((4, 3), -1, np.float32)
    x[0, 1, 77], x[0, 1, 2999], x[1, 2, 0] = 1, 2, 5
    x[2] = np.random.default_rng(1).standard_normal((3, 3000))
    scores[2] = -np.inf
    x[3, 0, 5] = -3.4e38
    check(fdx, x, scores, 8)


@pytest.mark.parametrize("end_id", [0, 17, 4999])
def test_ended_beams(fdx, end_id):
    done = np.random.default_rng(2).random((6, 5)) < 0.4
    done[0], done[1] = True, False
    x, scores = draw(9, 6, 5, 5000, keep=10, done=done, end_id=end_id)
    x[2, 1:, end_id] = 30   # an end that is likely
    check(fdx, x, scores, 10, done, end_id, near_ok=True)
    x[done] = np.nan        # rows of ended beams are not read
    check(fdx, x, scores, 10, done, end_id, near_ok=True)
    check(fdx, x[:2][1:], scores[1:2], 10, None, end_id, near_ok=True)


@pytest.mark.parametrize("vocab", [300, 20000])
def test_equal_logits(fdx, vocab):
    """Equal logits by id, -0 like 0, in whatever part of a row they lie; more of them than places."""
    for value in (0.0, -7.25, 3.4e38, -3.4e38):
        x = np.full((2, 2, vocab), np.float32(value))
        x[:, :, ::2] = -np.float32(0) if value == 0 else value
        got = fdx.beam_select(x, np.array([[0, -1], [-1, 0]], np.float32), 6)
        assert np.array_equal(got["tokens"], [[0, 1, 2, 3, 4, 5]] * 2) and np.array_equal(got["parents"], [[0] * 6, [3] * 6])
    r = np.random.default_rng(3)
    x = r.integers(0, 4, (3, 3, vocab)).astype(np.float32)
    scores = np.array([[0, -1.5, -9.25]] * 3, np.float32)
    check(fdx, x, scores, 32, near_ok=True)
    x[:, :, vocab // 2:] += 1   # the best lie behind
    check(fdx, x, scores, 32, near_ok=True)


@pytest.mark.parametrize("n,beams,vocab,keep", [(2, 32, 5000, 32), (1, 4, 70000, 32), (1, 16, 20000, 16), (3, 8, 4096, 32), (40, 16, 9000, 32), (1, 1, 131072, 32), (2, 2, 33, 31)])
@pytest.mark.parametrize("what", ["equal", "steps", "one beam"])
def test_lists_of_one_order(fdx, n, beams, vocab, keep, what):
    """All that is kept in one list, or as many from each, or all totals the same."""
    x, scores = np.zeros((n, beams, vocab), np.float32), np.zeros((n, beams), np.float32)
    if what == "steps":
        x[:, :, :] = -np.arange(vocab) % 7
    if what == "one beam":
        x[:, :, :] = np.random.default_rng(keep).permutation(vocab).astype(np.float32) / 64
        scores[:, :] = -1000 * ((np.arange(beams) + 1) % beams)
    got = fdx.beam_select(x, scores, keep)
    total = x[0].astype(np.float64) + scores[0][:, None]   # less the same number for every beam
    order = np.argsort(-total.ravel(), kind="stable")[:keep]   # equal ones by beam, then by token
    rows, tokens = order // vocab, order % vocab
    assert (got["parents"] - beams * np.arange(n)[:, None] == rows).all(), (got["parents"], rows)
    assert (got["tokens"] == tokens).all(), (got["tokens"], tokens)


def test_logits_near_each_other(fdx):
    """Logits of one row that differ in their last bit, whose totals are the same in fp32: the larger first."""
    vocab = 6000
    x = np.full((1, 2, vocab), -20, np.float32)
    at = np.random.default_rng(4).permutation(vocab)[:20]
    value = np.float32(3)
    for t in at:
        x[0, 0, t] = value
        value = np.nextafter(value, np.float32(9))
    check(fdx, x, np.array([[-100, -300]], np.float32), 20, near_ok=True)


def test_nan_and_infinities(fdx):
    x, scores = draw(11, 3, 3, 5000, keep=6)
    for what in (np.nan, np.inf):
        for row in (0, 2499, 4999):
            y = x.copy()
            y[1, 2, row] = what
            with pytest.raises(fdx.FdxError, match="NaN or infinite"):
                fdx.beam_select(y, scores, 6)
        for value in (np.nan, np.inf):
            bad = scores.copy()
            bad[2, 0] = value
            with pytest.raises(fdx.FdxError, match="NaN or infinite"):
                fdx.beam_select(x, bad, 6)
    got = {}

    def keep_out(flag, message):
        got["flag"] = int(flag.to_host((1,), np.int32)[0])
    y, bad = x.copy(), scores.copy()
    y[1, 2, 1234], bad[2, 0], bad[0, 1] = np.nan, np.inf, np.nan
    was, fdx._raise_if_set = fdx._raise_if_set, keep_out
    try:
        check(fdx, y, bad, 6, near_ok=True)
    finally:
        fdx._raise_if_set = was
    assert got["flag"] == 1


@pytest.mark.parametrize("shift,pad", [(1, 0), (0, 3), (2, 5), (0, 4)])
def test_strides_and_alignment(fdx, shift, pad):
    import ctypes
    n, beams, vocab, keep = 2, 3, 9001, 6
    x, scores = draw(12, n, beams, vocab, keep=keep)
    rows = np.full((n * beams, vocab + pad), 99, np.float32)
    rows[:, :vocab] = x.reshape(n * beams, vocab)
    dx, ds = fdx.DevBuf.from_host(np.concatenate([np.zeros(shift, np.float32), rows.ravel()])), fdx.DevBuf.from_host(scores)
    out = [fdx.DevBuf.from_host(np.full(n * keep + 3, 5, np.int32), np.int32) for _ in range(2)]
    new = fdx.DevBuf.from_host(np.full(n * keep + 3, 5, np.float32))
    need = fdx.lib.fdx_beam_select_scratch_bytes(n, beams, vocab, keep)
    scratch = fdx.DevBuf.from_host(np.full(need + 16, 0xff, np.uint8), np.uint8)
    fdx.check(fdx.lib.fdx_beam_select_f32(ctypes.c_void_p(dx.ptr.value + 4 * shift), ctypes.c_int64(vocab + pad), n, beams, vocab, ds.ptr, None, -1, keep,
                                          out[0].ptr, out[1].ptr, new.ptr, None, scratch.ptr, None))
    fdx.sync()
    parents, tokens, best, _ = expect(x, scores, keep)
    assert np.array_equal(out[0].to_host((n * keep + 3,), np.int32), np.append(parents.ravel(), [5, 5, 5]))
    assert np.array_equal(out[1].to_host((n * keep + 3,), np.int32), np.append(tokens.ravel(), [5, 5, 5]))
    assert (new.to_host((n * keep + 3,))[-3:] == 5).all() and (scratch.to_host((need + 16,), np.uint8)[need:] == 0xff).all()


@pytest.mark.parametrize("n,beams,vocab", [(3, 4, 5000), (300, 7, 300), (2, 32, 20000)])
def test_results_in_the_place_of_scores(fdx, n, beams, vocab):
    """Where as many are kept as there were, the new scores and ends may take the old ones' place."""
    import ctypes
    r = np.random.default_rng(n)
    done = (r.random((n, beams)) < 0.3).astype(np.int32)
    x, scores = r.standard_normal((n, beams, vocab)).astype(np.float32), -r.uniform(0, 3, (n, beams)).astype(np.float32)
    want = fdx.beam_select(x, scores, beams, done, 11)
    dx, ds, dd = fdx.DevBuf.from_host(x), fdx.DevBuf.from_host(scores), fdx.DevBuf.from_host(done, np.int32)
    out = [fdx.DevBuf(4 * n * beams) for _ in range(2)]
    scratch = fdx.DevBuf(fdx.lib.fdx_beam_select_scratch_bytes(n, beams, vocab, beams))
    fdx.check(fdx.lib.fdx_beam_select_f32(dx.ptr, ctypes.c_int64(vocab), n, beams, vocab, ds.ptr, dd.ptr, 11, beams, out[0].ptr, out[1].ptr, ds.ptr, dd.ptr,
                                          scratch.ptr, None))
    fdx.sync()
    assert np.array_equal(ds.to_host((n, beams)), want["scores"]) and np.array_equal(dd.to_host((n, beams), np.int32), want["done"])
    assert np.array_equal(out[0].to_host((n, beams), np.int32), want["parents"]) and np.array_equal(out[1].to_host((n, beams), np.int32), want["tokens"])


def test_runs_are_equal(fdx):
    r = np.random.default_rng(13)
    x, scores = r.standard_normal((16, 4, 50257)).astype(np.float32), -r.uniform(0, 3, (16, 4)).astype(np.float32)
    first = fdx.beam_select(x, scores, 8, None, 3)
    for _ in range(3):
        again = fdx.beam_select(x, scores, 8, None, 3)
        assert all(np.array_equal(first[key], again[key]) for key in first)


@pytest.mark.parametrize("vocab", [7, 300, 20000])
@pytest.mark.parametrize("value", [-3.4028235e38, 3.4028235e38, -1e30, 1e20, -1e13])
def test_rows_of_one_far_value(fdx, value, vocab):
    """Every token of a row has one logit of any size, as where a mask of fp32's lowest value leaves nothing: each has the probability 1 / vocab, which beams
    with ordinary logits are compared with."""
    far = np.full(vocab, value, np.float32)
    x, _ = draw(12, 2, 3, vocab, keep=4)
    x[0, 1], x[1, 0], x[1, 2] = far, far, far
    scores = np.array([[-4, -3, -5], [-1, -3, -1.5]], np.float32)
    got = fdx.beam_select(x, scores, 6)
    for s in range(2):
        every = []
        for b in range(3):
            row = x[s, b].astype(np.float64) - x[s, b].astype(np.float64).max()
            every += [(float(scores[s, b]) + total, b, t) for t, total in enumerate(row - np.log(np.exp(row).sum()))]
        every = sorted(every, key=lambda c: (-c[0], c[1], c[2]))[:6]
        want = np.array([c[0] for c in every])
        print("beam far value", value, vocab, got["scores"][s], want, flush=True)
        assert got["parents"][s].tolist() == [3 * s + c[1] for c in every] and got["tokens"][s].tolist() == [c[2] for c in every]
        assert (np.abs(got["scores"][s] - want) <= 4e-7 + 2.0 ** -23 * np.abs(want)).all()


@pytest.mark.parametrize("vocab", [300, 20000])
def test_masks_of_the_lowest_value(fdx, vocab):
    """Rows with some tokens at fp32's lowest value beside ones with -infinity there: the same selection, the same scores; a row of nothing else is as likely
    as any other of equal logits."""
    r = np.random.default_rng(13)
    x, scores = draw(14, 4, 3, vocab, keep=6)
    out = r.random(x.shape) < 0.9
    x[out] = -np.inf
    y = np.where(out, np.finfo(np.float32).min, x)
    a, b = fdx.beam_select(x, scores, 6), fdx.beam_select(y, scores, 6)
    assert all(np.array_equal(a[key], b[key]) for key in a)
