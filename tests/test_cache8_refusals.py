"""What the entry points for caches in 8 bits, page tables and beams refuse, without a GPU: arguments are checked before anything is launched."""
import ctypes

import numpy as np
import pytest

from cache8 import E4M3, HostCache, decode, encode

P = ctypes.c_void_p(1 << 20)   # never followed: the calls below are refused
I64 = ctypes.c_int64
INVALID, UNSUPPORTED = 1, 4


class Ptr:
    ptr = P


class Null:
    ptr = None


def odd(by):
    return type("Odd", (), dict(ptr=ctypes.c_void_p((1 << 20) + by)))


def pages8(fdx, **change):
    args = dict(k=Ptr, v=Ptr, kind="i8", n_pages=10, page_size=16, kv_heads=2, dk=64, dv=64, table=Ptr, table_width=4, lens=Ptr, n_seqs=3,
                max_len=64, k_scale=Ptr, v_scale=Ptr, block=8)
    raw = {key: change.pop(key) for key in list(change) if key not in args}
    args.update(change)
    c = fdx.KvPages8(**args)
    for key, value in raw.items():
        setattr(c.pages, key, value)
    return c


def refused(fdx, status, code, text):
    assert status == code, (status, fdx.lib.fdx_last_error())
    assert text in fdx.lib.fdx_last_error().decode()


def append(fdx, cache, k=P, ldk=128, v=P, ldv=128, starts=P, tokens=5):
    return fdx.lib.fdx_kv8_append_f32(k, I64(ldk), v, I64(ldv), starts, tokens, cache, None)


def paged(fdx, cache, q=P, ldq=256, starts=P, tokens=5, max_new=2, heads=4, out=P, ldo=256, scratch=P):
    return fdx.lib.fdx_mha_paged8_f32(q, I64(ldq), starts, tokens, max_new, heads, cache, out, I64(ldo), scratch, None)


T = ctypes.c_void_p(1 << 30)   # apart from P


def fork8(fdx, cache, parents=P, new_table=T, new_lens=ctypes.c_void_p(1 << 29), scratch=P):
    return fdx.lib.fdx_kv8_fork(cache, parents, None, new_table, new_lens, None, scratch, None)


@pytest.mark.parametrize("change,text", [
    (dict(k=Null), "null"), (dict(v=Null), "null"), (dict(table=Null), "null"), (dict(lens=Null), "null"), (dict(k_scale=Null), "null"),
    (dict(v_scale=Null), "null"), (dict(type=0), "type 0"), (dict(type=1), "type 1"), (dict(type=4), "type 4"), (dict(type=-1), "type -1"),
    (dict(n_pages=0), "shape"), (dict(page_size=0), "shape"), (dict(kv_heads=-1), "shape"), (dict(dk=0), "shape"), (dict(dv=0), "shape"),
    (dict(n_seqs=0), "shape"), (dict(table_width=0), "shape"), (dict(max_len=0), "shape"), (dict(max_len=65), "reach"),
    (dict(n_pages=1 << 27), "2^31"), (dict(block=0), "divide"), (dict(block=-8), "divide"), (dict(block=5), "divide"), (dict(block=32), "divide"),
    (dict(k_scale=odd(2)), "aligned"), (dict(v_scale=odd(1)), "aligned")])
def test_caches(fdx, change, text):
    c = ctypes.byref(pages8(fdx, **change))
    for call in (append, paged, fork8):
        refused(fdx, call(fdx, c), INVALID, text)


def test_other_caches(fdx):
    """The calls for fp32 and bf16 pages refuse 8 bits."""
    c = pages8(fdx)
    for kind in (2, 3):
        c.pages.type = kind
        p = ctypes.byref(c.pages)
        refused(fdx, fdx.lib.fdx_kv_append_f32(P, I64(128), P, I64(128), P, 5, p, None), INVALID, "type %d" % kind)
        refused(fdx, fdx.lib.fdx_mha_paged_f32(P, I64(256), P, 5, 2, 4, p, P, I64(256), P, None), INVALID, "type %d" % kind)
        refused(fdx, fdx.lib.fdx_kv_fork(p, P, None, T, ctypes.c_void_p(1 << 29), None, P, None), INVALID, "type %d" % kind)
    for call in (append, paged, fork8):
        refused(fdx, call(fdx, None), INVALID, "null")


def test_append(fdx):
    for change, text in ((dict(k=None), "null"), (dict(v=None), "null"), (dict(starts=None), "null"), (dict(ldk=127), "overlap"), (dict(ldv=0), "overlap"),
                         (dict(tokens=0), "tokens"), (dict(tokens=-4), "tokens"), (dict(tokens=(1 << 24) + 1), "tokens")):
        refused(fdx, append(fdx, ctypes.byref(pages8(fdx)), **change), INVALID, text)
    for change in (dict(kv_heads=1 << 20, dk=1, dv=1, block=1), dict(n_seqs=1 << 23)):
        c = pages8(fdx, **change)
        refused(fdx, append(fdx, ctypes.byref(c), tokens=1 << 20, ldk=1 << 20, ldv=1 << 20), INVALID, "too many")
    c = pages8(fdx, n_pages=1, page_size=1 << 24, kv_heads=1, dk=65, dv=65, block=1 << 24)
    refused(fdx, append(fdx, ctypes.byref(c)), INVALID, "2^30 elements")


def test_paged(fdx):
    for change, text in ((dict(q=None), "null"), (dict(out=None), "null"), (dict(starts=None), "null"), (dict(ldq=255), "overlap"),
                         (dict(ldo=255), "overlap"), (dict(tokens=0), "shape"), (dict(max_new=0), "shape"), (dict(heads=0), "shape"),
                         (dict(heads=3, ldq=256), "share"), (dict(tokens=1 << 25, heads=4), "too many")):
        refused(fdx, paged(fdx, ctypes.byref(pages8(fdx)), **change), INVALID, text)
    for change in (dict(dk=129), dict(dv=192)):
        refused(fdx, paged(fdx, ctypes.byref(pages8(fdx, **change)), ldq=1024, ldo=1024), UNSUPPORTED, "depths up to 128")
    c = ctypes.byref(pages8(fdx, page_size=4096, max_len=16384))
    assert fdx.lib.fdx_mha_paged8_scratch_bytes(5, 2, 4, c) > 0
    for scratch in (None, ctypes.c_void_p((1 << 20) + 4)):
        refused(fdx, paged(fdx, c, scratch=scratch), INVALID, "scratch")
    assert fdx.lib.fdx_mha_paged8_scratch_bytes(5, 2, 4, None) == 0
    for args in ((0, 2, 4), (5, 0, 4), (5, 2, 0), (5, 2, 3)):
        assert fdx.lib.fdx_mha_paged8_scratch_bytes(*args, c) == 0


def test_fork(fdx):
    c = pages8(fdx)
    for change, text in ((dict(parents=None), "null"), (dict(new_table=None), "null"), (dict(new_lens=None), "null"), (dict(scratch=None), "scratch"),
                         (dict(scratch=ctypes.c_void_p((1 << 20) + 8)), "scratch"), (dict(new_table=P), "overlap"), (dict(new_lens=P), "overlap"),
                         (dict(new_table=ctypes.c_void_p((1 << 20) + 44)), "overlap"), (dict(new_table=ctypes.c_void_p((1 << 20) - 44)), "overlap"),
                         (dict(new_lens=ctypes.c_void_p((1 << 20) + 8)), "overlap"), (dict(new_lens=ctypes.c_void_p((1 << 30) + 16)), "overlap"), (dict(parents=T), "overlap")):
        refused(fdx, fork8(fdx, ctypes.byref(c), **change), INVALID, text)
    c = pages8(fdx, n_seqs=1 << 20, table_width=1 << 11)
    refused(fdx, fork8(fdx, ctypes.byref(c)), INVALID, "2^31")
    c = pages8(fdx, n_seqs=(1 << 23) + 1)
    refused(fdx, fork8(fdx, ctypes.byref(c)), INVALID, "2^23")
    assert fdx.lib.fdx_kv_fork_scratch_bytes(None) == 0 and fdx.lib.fdx_kv8_fork_scratch_bytes(None) == 0
    assert fdx.lib.fdx_kv8_fork_scratch_bytes(ctypes.byref(pages8(fdx, n_pages=0))) == 0


def test_beams(fdx):
    def call(x=P, ld=100, n=3, beams=4, vocab=100, scores=P, done=P, end_id=7, keep=8, parents=P, tokens=P, new_scores=P, new_done=P, scratch=P):
        return fdx.lib.fdx_beam_select_f32(x, I64(ld), n, beams, vocab, scores, done, end_id, keep, parents, tokens, new_scores, new_done, scratch, None)
    for change, text in ((dict(x=None), "null"), (dict(scores=None), "null"), (dict(parents=None), "null"), (dict(tokens=None), "null"),
                         (dict(new_scores=None), "null"), (dict(n=0), "beams"), (dict(n=-1), "beams"), (dict(beams=0), "beams"), (dict(beams=33), "beams"),
                         (dict(n=1 << 22), "beams"), (dict(vocab=0), "logits"), (dict(vocab=(1 << 24) + 1, ld=1 << 25), "logits"), (dict(ld=99), "overlap"),
                         (dict(keep=0), "continuations"), (dict(keep=33), "continuations"), (dict(beams=2, vocab=3, end_id=2, keep=7), "continuations"),
                         (dict(end_id=100), "end_id"), (dict(end_id=-1), "end_id"), (dict(end_id=-1, done=None), "end_id"), (dict(end_id=-1, new_done=None), "end_id"),
                         (dict(scratch=None), "scratch"), (dict(scratch=ctypes.c_void_p((1 << 20) + 4)), "scratch")):
        refused(fdx, call(**change), INVALID, text)
    at = [ctypes.c_void_p((i + 2) << 20) for i in range(7)]
    apart = dict(zip(("x", "scores", "done", "parents", "tokens", "new_scores", "new_done"), at))
    outs = ("parents", "tokens", "new_scores", "new_done")
    same = [dict(apart, **{a: apart[b]}) for a in outs for b in apart if a != b]   # keep is not beams
    same += [dict(apart, keep=4, **{a: apart[b]}) for a in outs for b in apart if a != b and (a, b) not in (("new_scores", "scores"), ("new_done", "done"))]
    near = [dict(apart, new_scores=ctypes.c_void_p(apart["scores"].value + by), keep=4) for by in (-44, -4, 4, 44)]
    near += [dict(apart, new_done=ctypes.c_void_p(apart["x"].value + 4 * (11 * 100 + 99))), dict(apart, tokens=ctypes.c_void_p(apart["x"].value - 92))]
    for change in same + near:
        refused(fdx, call(**change), INVALID, "overlap")
    for args in ((0, 4, 100, 8), (3, 0, 100, 8), (3, 4, 0, 8), (3, 4, 100, 0), (-1, 4, 100, 8)):
        assert fdx.lib.fdx_beam_select_scratch_bytes(*args) == 0


class HostBuf:
    """Memory that no call looks into."""

    def __init__(self, nbytes=0):
        self.ptr = P

    @classmethod
    def from_host(cls, arr, dtype=None):
        return cls()


def test_python_calls(fdx, monkeypatch):
    monkeypatch.setattr(fdx, "DevBuf", HostBuf)
    for kind, block in (("i8", 3), ("e4m3", 0), ("i8", 32), ("f32", 4), ("bf16", 16), ("i4", None)):
        with pytest.raises(fdx.FdxError):
            fdx.PagedCache(9, 16, 2, 8, 6, 3, 20, kind, block)
    c = fdx.PagedCache(9, 16, 2, 8, 6, 3, 20, "i8")
    assert c.block == 16 and c.pages().block == 16 and c.pages().pages.type == 2
    for parents in ([0, 1], [0, 1, 3], [0, 1, 2.5], [0, 1, 2 ** 32], [[0, 1, 2]], [0, 1, None]):
        with pytest.raises(fdx.FdxError, match="parents"):
            fdx.kv_fork(c, parents)
    x = np.zeros((2, 3, 10), np.float32)
    for scores, done in ((np.zeros((2, 4)), None), (np.zeros(6), None), (np.zeros((2, 3)), np.zeros((3, 2)))):
        with pytest.raises(fdx.FdxError, match="shape"):
            fdx.beam_select(x, scores, 3, done, 0)
    with pytest.raises(fdx.FdxError, match="end_id"):
        fdx.beam_select(x, np.zeros((2, 3)), 3, np.zeros((2, 3)))
    got = fdx.beam_select(np.zeros((0, 3, 10)), np.zeros((0, 3)), 4)
    assert sorted(got) == ["parents", "scores", "tokens"] and got["scores"].shape == (0, 4)


def test_release_of_shared_pages(fdx, monkeypatch):
    """A page is free when no sequence has it."""
    monkeypatch.setattr(fdx, "DevBuf", HostBuf)
    c = fdx.PagedCache(9, 4, 2, 8, 6, 3, 20, "e4m3", 2)
    c.table[0, :2], c.table[1, :2], c.table[2, :1] = [5, 1], [5, 7], [3]   # 0 and 1 have page 5 in common, as kv_fork leaves them
    c.lens[:] = [7, 6, 2]
    c.free = [8, 6, 4, 2, 0]
    c.release(1)
    assert c.free == [8, 6, 4, 2, 0, 7] and c.lens.tolist() == [7, 0, 2] and (c.table[1] == -1).all()
    c.release(0)
    assert c.free == [8, 6, 4, 2, 0, 7, 5, 1]


def test_fork_that_fails_leaves_the_cache(fdx, monkeypatch):
    monkeypatch.setattr(fdx, "DevBuf", HostBuf)
    c = fdx.PagedCache(9, 4, 2, 8, 6, 3, 20, "e4m3", 2)
    c.grow([5, 0, 4])
    table, lens, free = c.table.copy(), c.lens.copy(), list(c.free)

    def fail(*args):
        raise fdx.FdxError("failed on purpose")
    for name in ("check", "_raise_if_set"):
        with monkeypatch.context() as m:
            m.setattr(fdx, "check", lambda status: None)
            m.setattr(fdx.lib, "fdx_kv8_fork", lambda *args: 0)
            m.setattr(fdx, name, fail)
            with pytest.raises(fdx.FdxError, match="on purpose"):
                fdx.kv_fork(c, [0, 0, 2])
        assert np.array_equal(c.table, table) and np.array_equal(c.lens, lens) and c.free == free


def test_the_definition(fdx):
    """The host's codes: nearest, ties to even; every code is its own value's."""
    x = np.random.default_rng(0).uniform(-448, 448, 5000).astype(np.float32) * np.float32(2.0) ** np.random.default_rng(1).integers(-14, 1, 5000)
    x = x.astype(np.float32)
    near = decode(encode(x, "e4m3"), "e4m3")
    every = np.concatenate([E4M3, -E4M3]).astype(np.float64)
    assert (np.abs(near.astype(np.float64) - x) == np.abs(every[:, None] - x.astype(np.float64)).min(0)).all()
    assert E4M3[-1] == 448 and E4M3[1] == 2.0 ** -9
    assert decode(encode(np.float32([17, 19, 2.0 ** -10, 3 * 2.0 ** -10, -17, 1e9, 464]), "e4m3"), "e4m3").tolist() == [16, 20, 0, 2.0 ** -8, -16, 448, 448]
    assert encode(np.float32([0.5, 1.5, -2.5, 127.4, -300]), "i8").view(np.int8).tolist() == [0, 2, -2, 127, -127]
    h = HostCache(2, 4, 1, 2, 2, "i8", 2)
    h.append(lambda p: p, 0, np.float32([[[1, -0.5]], [[2, 0]], [[127, 1]]]), 0)
    h.append(lambda p: p, 3, np.float32([[[254, 3]]]), 0)
    assert h.scales[0].ravel()[:2].tolist() == [np.float32(2) / np.float32(127), 2.0] and decode(h.codes[0][2:4, 0], "i8").tolist() == [[64, 0], [127, 2]]


def test_paged_sizes_beyond_every_limit(fdx):
    """Numbers that the call refuses are refused whatever they are, and need no scratch memory."""
    most = 2 ** 31 - 1
    for n_seqs in ((1 << 21) + 1, (1 << 30) - 1, 1 << 30, most):
        for max_len in (1, 64):
            c = ctypes.byref(pages8(fdx, n_seqs=n_seqs, max_len=max_len))
            assert fdx.lib.fdx_mha_paged8_scratch_bytes(5, 2, 4, c) == 0
            refused(fdx, paged(fdx, c), INVALID, "too many")
    c = ctypes.byref(pages8(fdx, n_pages=1, page_size=1 << 24, table_width=most, max_len=most, n_seqs=most, block=1))
    assert fdx.lib.fdx_mha_paged8_scratch_bytes(5, 2, 4, c) == 0
    refused(fdx, paged(fdx, c), INVALID, "2^30")
    for tokens, max_new, heads in ((most, most, 2), (5, most, most - 1), (most, most, most - 1)):
        c = ctypes.byref(pages8(fdx))
        assert fdx.lib.fdx_mha_paged8_scratch_bytes(tokens, max_new, heads, c) == 0
        refused(fdx, paged(fdx, c, tokens=tokens, max_new=max_new, heads=heads), INVALID, "too many")
    c = ctypes.byref(pages8(fdx, kv_heads=1 << 23, dk=1, dv=1))
    assert fdx.lib.fdx_mha_paged8_scratch_bytes(5, 2, 1 << 23, c) == 0
    refused(fdx, paged(fdx, c, heads=1 << 23), INVALID, "too many")


def test_beams_of_numbers_beyond_32_bits(fdx, monkeypatch):
    """No number reaches the library as another one: those that 32 bits cannot hold are refused, every negative end_id is none."""
    monkeypatch.setattr(fdx, "DevBuf", HostBuf)
    x, scores = np.zeros((2, 3, 10), np.float32), np.zeros((2, 3))
    for change in (dict(keep=2 ** 32 + 3), dict(keep=-2 ** 32 + 3), dict(keep=2 ** 31), dict(end_id=2 ** 32 + 7), dict(end_id=2 ** 31), dict(end_id=2.5), dict(keep=1.5)):
        with pytest.raises(fdx.FdxError, match="32 bits|whole numbers"):
            fdx.beam_select(x, scores, **dict(dict(keep=3), **change))
    seen = []

    def call(*args):
        seen.append(args[7:9])
        return INVALID
    monkeypatch.setattr(fdx.lib, "fdx_beam_select_f32", call)
    for end_id, want in ((-1, -1), (-2 ** 32 + 7, -1), (np.int64(7), 7)):
        with pytest.raises(fdx.FdxError):
            fdx.beam_select(x, scores, np.int64(3), None, end_id)
        assert seen[-1] == (want, 3) and all(type(a) is int for a in seen[-1])


def test_release_of_any_table(fdx, monkeypatch):
    """Pages go back in their order unless another sequence has them, wherever in its row; numbers that are none of the cache are nobody's."""
    monkeypatch.setattr(fdx, "DevBuf", HostBuf)
    r = np.random.default_rng(0)
    for trial in range(200):
        n, width, n_pages = int(r.integers(1, 6)), int(r.integers(1, 9)), int(r.integers(1, 40))
        c = fdx.PagedCache(n_pages, 4, 1, 1, 1, n, 4 * width, "f32" if trial % 2 else "i8")
        c.table[:] = np.where(r.random((n, width)) < 0.4, -1, r.integers(0, n_pages + (7 if trial % 5 == 0 else 0), (n, width)))
        c.lens[:], c.free = 1, [99]
        seq = int(r.integers(0, n))
        others = set(np.delete(c.table, seq, 0).ravel().tolist())
        want = [99] + [int(p) for p in c.table[seq] if p >= 0 and int(p) not in others]
        rest = np.delete(c.table, seq, 0)
        c.release(seq)
        assert c.free == want and all(type(p) is int for p in c.free)
        assert (c.table[seq] == -1).all() and c.lens[seq] == 0 and np.array_equal(np.delete(c.table, seq, 0), rest)
        c.release(seq)
        assert c.free == want


def test_release_takes_a_look_at_the_table(fdx, monkeypatch):
    """Ending one of many long sequences costs a few passes over the table at most: measured against one search of it."""
    import time
    monkeypatch.setattr(fdx, "DevBuf", HostBuf)
    n, width = 256, 500
    c = fdx.PagedCache(n * width, 16, 1, 1, 1, n, 16 * width, "bf16")
    c.grow([16 * width] * n)

    def least(calls):
        times = []
        for call in calls:
            begin = time.perf_counter()
            call()
            times.append(time.perf_counter() - begin)
        return min(times)
    search = least([lambda: np.isin(c.table[0], c.table)] * 8)
    release = least([lambda s=s: c.release(s) for s in range(16)])
    print("release %.3f ms, a search %.3f ms" % (1e3 * release, 1e3 * search))
    assert release <= 3 * search and len(c.free) == 16 * width
