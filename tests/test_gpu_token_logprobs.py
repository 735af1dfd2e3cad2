"""Log probabilities, entropy and the likeliest tokens against 64 bits.

Bounds.  x - max is rounded once (2^-24 of itself), the exponential is good to a few units of 2^-23, the sum of n of them is added
in chains of at most a few hundred: relative error of Z below 64 * 2^-24 = 4e-6, which is the absolute error of log Z; a log
probability of size s carries s * 2^-23 beside it.  In the 2-norm over rows these average out: 2e-6."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def reference(x):
    x = x.astype(np.float64)
    with np.errstate(all="ignore"):
        m = x.max(1, keepdims=True)
        lp = x - m - np.log(np.exp(x - m).sum(1, keepdims=True))
        p = np.exp(lp)
        return lp, -(np.where(p > 0, p * lp, 0)).sum(1)


def order(row, top):
    """ids by descending logit, then ascending; NaN last"""
    return np.lexsort((np.arange(len(row)), -np.where(np.isnan(row), -np.inf, row.astype(np.float64)), np.isnan(row)))[:top]


def compare(fdx, x, ids, top):
    got = fdx.token_logprobs(x, ids, top)
    lp, entropy = reference(x)
    rows = np.arange(len(x))
    finite = np.isfinite(lp).any(1)
    bound = lambda want: 4e-6 + 2.0 ** -22 * np.abs(want)
    if ids is not None:
        want = np.where(ids < 0, 0, lp[rows, np.maximum(ids, 0)])
        ok = np.isfinite(want)
        assert (np.abs(got["logprobs"] - want)[ok] <= bound(want[ok])).all(), np.abs(got["logprobs"] - want)[ok].max()
        assert np.array_equal(got["logprobs"][~ok & finite], want[~ok & finite])
    print("entropy off by", np.abs(got["entropy"] - entropy)[finite].max() if finite.any() else 0, flush=True)
    # H = log Z - W / Z: W is a sum of e d, d up to the row's spread where e counts
    assert (np.abs(got["entropy"] - entropy)[finite] <= 1e-5 * (1 + entropy[finite])).all()
    if top:
        want = np.stack([order(r, top) for r in x])
        assert np.array_equal(got["top_ids"], want)
        w = np.take_along_axis(lp, want, 1)
        ok = np.isfinite(w)
        assert (np.abs(got["top_logprobs"] - w)[ok] <= bound(w[ok])).all()
        assert (got["top_logprobs"][finite][~ok[finite]] == -np.inf).all()
    return got


@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 1, 0), (3, 2, 2), (2, 7, 5), (5, 63, 32), (5, 64, 1), (4, 65, 3), (1, 1000, 20), (7, 4097, 32),
                                            (1, 50257, 5), (16, 50257, 20), (300, 1021, 8), (2, 131072, 32), (1, 262147, 32), (70, 32001, 0),
                                            (1100, 300, 2), (600, 5000, 32), (3, 33000, 31)])
def test_against_64_bits(fdx, rows, vocab, top):
    print("token logprobs", rows, vocab, top, flush=True)
    r = np.random.default_rng(rows + vocab)
    x = (3 * r.standard_normal((rows, vocab))).astype(np.float32)
    x[np.arange(rows), r.integers(0, vocab, rows)] += 9
    ids = r.integers(0, vocab, rows)
    ids[::3] = x[::3].argmax(1)
    ids[1::5] = -1
    compare(fdx, x, ids, top)
    compare(fdx, x, None, top)


@pytest.mark.parametrize("vocab", [40, 5003, 50257])
def test_equal_logits_in_the_order_of_their_ids(fdx, vocab):
    """Rows of few different values, of one value, of zeros of both signs, ascending and descending rows."""
    r = np.random.default_rng(1)
    x = np.stack([r.integers(0, 3, vocab), np.full(vocab, -2.5), np.where(np.arange(vocab) % 2, 0.0, -0.0), np.arange(vocab) / 64,
                  -np.arange(vocab) / 64, np.where(np.arange(vocab) >= vocab - 35, 1.0, 0.0), np.arange(vocab) // 7 % 5]).astype(np.float32)
    print("token logprobs ties", vocab, flush=True)
    compare(fdx, x, np.full(len(x), vocab - 1), 32)


@pytest.mark.parametrize("vocab", [50, 3001, 50257])
def test_tokens_ruled_out(fdx, vocab):
    r = np.random.default_rng(2)
    x = (4 * r.standard_normal((6, vocab))).astype(np.float32)
    x[0, 10:] = -np.inf                       # ten left, fewer than asked for
    x[1, :] = -np.inf
    x[1, 17] = 3                              # one left: certain
    x[2, :] = -np.inf                         # none left
    x[3, r.random(vocab) < 0.9] = -np.inf
    x[4, r.random(vocab) < 0.5] = np.finfo(np.float32).min   # the type's lowest value for a mask
    x[5, :] = np.finfo(np.float32).min
    print("token logprobs masked", vocab, flush=True)
    got = compare(fdx, x, np.array([3, 17, 5, 0, 0, 1]), 20)
    assert got["logprobs"][1] == 0 and got["entropy"][1] == 0 and got["top_logprobs"][1, 0] == 0
    assert got["logprobs"][2] == -np.inf and got["entropy"][2] == 0 and (got["top_logprobs"][2] == -np.inf).all()
    assert np.array_equal(got["top_ids"][2], np.arange(20))


@pytest.mark.parametrize("vocab", [50, 50257])
def test_nan_and_infinity(fdx, vocab):
    r = np.random.default_rng(3)
    x = r.standard_normal((4, vocab)).astype(np.float32)
    x[0, 7] = np.nan
    x[1, vocab - 1] = np.inf
    x[2, :] = np.nan
    x[2, 3:5] = 1
    print("token logprobs odd", vocab, flush=True)
    got = fdx.token_logprobs(x, np.arange(4), 6)
    lp, entropy = reference(x[3:])
    for name in ("logprobs", "entropy", "top_logprobs"):
        assert np.isnan(got[name][:3]).all() and not np.isnan(got[name][3]).any()
    assert abs(got["logprobs"][3] - lp[0, 3]) < 1e-5 and abs(got["entropy"][3] - entropy[0]) < 1e-4
    for row in range(4):
        assert np.array_equal(got["top_ids"][row], order(x[row], 6))


def test_certain_rows(fdx):
    """One logit far above the rest: log probability and entropy go to zero and never past it."""
    x = np.zeros((5, 5000), np.float32)
    for i, gap in enumerate((5, 20, 60, 200, 3e38)):
        x[i, 4000] = gap
    got = compare(fdx, x, np.full(5, 4000), 2)
    assert (got["logprobs"] <= 0).all() and (got["entropy"] >= 0).all()


def test_large_logits(fdx):
    r = np.random.default_rng(4)
    x = (r.standard_normal((3, 3000)) * np.array([[1e4], [1e30], [1e-30]])).astype(np.float32)
    compare(fdx, x, np.array([1, 2, 3]), 5)


@pytest.mark.parametrize("shift,pad", [(0, 0), (1, 3), (2, 0), (3, 5)])
@pytest.mark.parametrize("rows,vocab", [(3, 50257), (40, 999)])
def test_strides_and_alignment(fdx, shift, pad, rows, vocab):
    """Rows that start at any multiple of four bytes; the gaps between them count for nothing."""
    r = np.random.default_rng(5)
    x = np.full((rows, vocab + pad), 1e30, np.float32)
    x[:, :vocab] = r.standard_normal((rows, vocab))
    buf = fdx.DevBuf.from_host(np.concatenate([np.full(shift, 1e30, np.float32), x.ravel()]))
    top, ids = 4, r.integers(0, vocab, rows).astype(np.int32)
    di, dl, de, dt, dtl = fdx.DevBuf.from_host(ids, np.int32), fdx.DevBuf(4 * rows), fdx.DevBuf(4 * rows), fdx.DevBuf(4 * rows * top), fdx.DevBuf(4 * rows * top)
    scratch = fdx.DevBuf(fdx.lib.fdx_token_logprobs_scratch_bytes(ctypes.c_int64(rows), vocab, top))
    print("token logprobs strides", shift, pad, rows, vocab, flush=True)
    fdx.check(fdx.lib.fdx_token_logprobs_f32(ctypes.c_void_p(buf.ptr.value + 4 * shift), ctypes.c_int64(vocab + pad), ctypes.c_int64(rows), vocab,
                                             di.ptr, top, dl.ptr, de.ptr, dt.ptr, dtl.ptr, scratch.ptr, None))
    lp, entropy = reference(x[:, :vocab])
    assert np.abs(dl.to_host((rows,)) - lp[np.arange(rows), ids]).max() < 1e-5
    assert np.abs(de.to_host((rows,)) - entropy).max() < 1e-4
    assert np.array_equal(dt.to_host((rows, top), np.int32), np.stack([order(row, top) for row in x[:, :vocab]]))


def test_ids_outside_the_vocabulary(fdx):
    x = np.zeros((3, 10), np.float32)
    assert (fdx.token_logprobs(x, np.array([-1, -100, -2**31]))["logprobs"] == 0).all()
    for bad in (10, 2**31 - 1):
        with pytest.raises(fdx.FdxError, match="less than the number of logits"):
            fdx.token_logprobs(x, np.array([0, bad, 1]))


def test_runs_are_equal(fdx):
    x = np.random.default_rng(6).standard_normal((9, 50257)).astype(np.float32)
    first = fdx.token_logprobs(x, np.arange(9), 32)
    for _ in range(3):
        again = fdx.token_logprobs(x, np.arange(9), 32)
        assert all(np.array_equal(first[name], again[name]) for name in first)


@pytest.mark.parametrize("rows,vocab", [(5, 50257), (600, 1021)])   # a row in parts and in one; rows that start beyond 2^32 floats
def test_rows_beyond_32_bits(fdx, rows, vocab):
    r, top = np.random.default_rng(7), 5
    ld = (1 << 32) // (rows - 2) + 3
    x = r.standard_normal((rows, vocab)).astype(np.float32)
    buf = fdx.DevBuf(4 * (ld * (rows - 1) + vocab))
    print("token logprobs far rows", rows, vocab, ld, flush=True)
    for i in range(rows):
        fdx.check(fdx.lib.fdx_h2d(ctypes.c_void_p(buf.ptr.value + 4 * ld * i), x[i].ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(4 * vocab)))
    ids = r.integers(0, vocab, rows).astype(np.int32)
    di, dl, dt, dtl = fdx.DevBuf.from_host(ids, np.int32), fdx.DevBuf(4 * rows), fdx.DevBuf(4 * rows * top), fdx.DevBuf(4 * rows * top)
    scratch = fdx.DevBuf(fdx.lib.fdx_token_logprobs_scratch_bytes(ctypes.c_int64(rows), vocab, top))
    fdx.check(fdx.lib.fdx_token_logprobs_f32(buf.ptr, ctypes.c_int64(ld), ctypes.c_int64(rows), vocab, di.ptr, top, dl.ptr, None, dt.ptr, dtl.ptr,
                                             scratch.ptr, None))
    lp, _ = reference(x)
    got, best = dl.to_host((rows,)), dt.to_host((rows, top), np.int32)
    buf.free()
    want = lp[np.arange(rows), ids]
    assert (np.abs(got - want) <= 4e-6 + 2.0 ** -22 * np.abs(want)).all()
    assert np.array_equal(best, np.stack([order(row, top) for row in x]))
