"""What the entry points for packed prompts, paged caches and token scores refuse, and the arithmetic their kernels find rows and
pages with, without a GPU: arguments are checked before anything is launched."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = ctypes.c_void_p(1 << 20)   # never followed: the calls below are refused
I64 = ctypes.c_int64
INVALID, UNSUPPORTED = 1, 4


class Ptr:
    ptr = P


def pages(fdx, **change):
    args = dict(k=Ptr, v=Ptr, kind="f32", n_pages=10, page_size=16, kv_heads=2, dk=64, dv=64, table=Ptr, table_width=4, lens=Ptr, n_seqs=3,
                max_len=64)
    raw = {key: change.pop(key) for key in list(change) if key not in args}
    args.update(change)
    c = fdx.KvPages(**args)
    for key, value in raw.items():
        setattr(c, key, value)
    return c


def refused(fdx, status, code, text):
    assert status == code, (status, fdx.lib.fdx_last_error())
    assert text in fdx.lib.fdx_last_error().decode()


class Null:
    ptr = None


@pytest.mark.parametrize("change,text", [
    (dict(k=Null), "null"), (dict(v=Null), "null"), (dict(table=Null), "null"), (dict(lens=Null), "null"), (dict(type=2), "type 2"),
    (dict(type=-1), "type -1"), (dict(n_pages=0), "shape"), (dict(page_size=0), "shape"), (dict(kv_heads=-1), "shape"), (dict(dk=0), "shape"),
    (dict(dv=0), "shape"), (dict(n_seqs=0), "shape"), (dict(table_width=0), "shape"), (dict(max_len=0), "shape"), (dict(max_len=65), "reach"),
    (dict(n_pages=1 << 27), "2^31"), (dict(k=type("Odd", (), dict(ptr=ctypes.c_void_p((1 << 20) + 2)))), "aligned")])
def test_caches(fdx, change, text):
    c = ctypes.byref(pages(fdx, **change))
    refused(fdx, fdx.lib.fdx_kv_append_f32(P, I64(128), P, I64(128), P, 5, c, None), INVALID, text)
    refused(fdx, fdx.lib.fdx_mha_paged_f32(P, I64(256), P, 5, 2, 4, c, P, I64(256), P, None), INVALID, text)


def test_append(fdx):
    c = ctypes.byref(pages(fdx))

    def call(k=P, ldk=128, v=P, ldv=128, starts=P, tokens=5, cache=c):
        return fdx.lib.fdx_kv_append_f32(k, I64(ldk), v, I64(ldv), starts, tokens, cache, None)
    for change, text in ((dict(k=None), "null"), (dict(v=None), "null"), (dict(starts=None), "null"), (dict(cache=None), "null"),
                         (dict(ldk=127), "overlap"), (dict(ldv=0), "overlap"), (dict(tokens=0), "tokens"), (dict(tokens=-4), "tokens"),
                         (dict(tokens=(1 << 25) + 1), "tokens")):
        refused(fdx, call(**change), INVALID, text)


def test_paged(fdx):
    def call(q=P, ldq=256, starts=P, tokens=5, max_new=2, heads=4, cache=None, out=P, ldo=256, scratch=P):
        return fdx.lib.fdx_mha_paged_f32(q, I64(ldq), starts, tokens, max_new, heads, ctypes.byref(cache or pages(fdx)), out, I64(ldo), scratch,
                                         None)
    for change, text in ((dict(q=None), "null"), (dict(out=None), "null"), (dict(starts=None), "null"), (dict(ldq=255), "overlap"),
                         (dict(ldo=255), "overlap"), (dict(tokens=0), "shape"), (dict(max_new=0), "shape"), (dict(heads=0), "shape"),
                         (dict(heads=3, ldq=256), "share"), (dict(tokens=1 << 25, heads=4), "too many")):
        refused(fdx, call(**change), INVALID, text)
    for change in (dict(dk=129), dict(dv=192)):
        refused(fdx, call(cache=pages(fdx, **change), ldq=1024, ldo=1024), UNSUPPORTED, "depths up to 128")


def test_paged_scratch(fdx):
    """Long caches of few sequences are summed in ranges, which takes memory of the caller's."""
    c = ctypes.byref(pages(fdx, page_size=4096, max_len=16384))
    assert fdx.lib.fdx_mha_paged_scratch_bytes(5, 2, 4, c) > 0
    for scratch in (None, ctypes.c_void_p((1 << 20) + 4)):
        refused(fdx, fdx.lib.fdx_mha_paged_f32(P, I64(256), P, 5, 2, 4, c, P, I64(256), scratch, None), INVALID, "scratch")


@pytest.mark.parametrize("max_len", [257, 4097, 32769, 131072, 1 << 30])
@pytest.mark.parametrize("heads,kv_heads", [(32, 8), (12, 12), (8, 1), (64, 1)])
def test_paged_scratch_is_bounded(fdx, max_len, heads, kv_heads):
    """Sums of key ranges: of 2^21 rows for tiles, and of some 2^18 for few rows (4096 workgroups and one more for each sequence and key head, of which
    there are fewer than that, 32 rows each), however many tokens and sequences a call has and however long they may get."""
    most = 0
    for dv in (1, 64, 128):
        for n_seqs in (1, 3, 64, 500, 4000, 1 << 18):
            c = ctypes.byref(pages(fdx, page_size=1 << 20, n_pages=1 << 10, table_width=1 << 10, kv_heads=kv_heads, dv=dv, n_seqs=n_seqs, max_len=max_len))
            for tokens in (1, 100, 1000, 2000, 4000, 8192, 16384, 1 << 16, (1 << 25) // heads):
                for max_new in (1, 5, tokens):
                    need = fdx.lib.fdx_mha_paged_scratch_bytes(tokens, max_new, heads, c)
                    assert need <= 4 * (dv + 2) * ((1 << 21) + (1 << 18) + (1 << 14)), (n_seqs, tokens, max_new, need)
                    most = max(most, need)
    assert max_len == 257 or most > 0


def test_numbers_of_ranges(fdx):
    """Up to 64 for few rows and 16 for tiles, where the length leaves a remainder too; sums of a row and range are m, l and `depth` values."""
    for max_len in [16385, 32768, 32769, 40000, 65535, 65537, (1 << 20) + 1] + list(range(33000, 36000, 7)):
        c = ctypes.byref(pages(fdx, page_size=1 << 20, n_pages=1 << 10, table_width=1 << 10, kv_heads=1, dv=62, n_seqs=1, max_len=max_len))
        assert 0 < fdx.lib.fdx_mha_paged_scratch_bytes(1, 1, 1, c) <= 64 * 4 * 64, max_len
        assert 0 < fdx.lib.fdx_mha_paged_scratch_bytes(1000, 1000, 1, c) - fdx.lib.fdx_mha_paged_scratch_bytes(32, 32, 1, c) <= 16 * 4 * 64 * 1000
    for tokens in range(4096, 9000):
        assert fdx.lib.fdx_mha_packed_scratch_bytes(tokens, tokens // 512, 1, 1, 62, 62) <= 16 * 4 * 64 * tokens, tokens


@pytest.mark.parametrize("tokens,heads,kv_heads", [(1000, 4, 4), (4000, 16, 16), (300, 16, 1)])
def test_packed_scratch(fdx, tokens, heads, kv_heads):
    """Key ranges of a few long prompts and prompts that are split once take memory of the caller's."""
    assert fdx.lib.fdx_mha_packed_scratch_bytes(tokens, 1, heads, kv_heads, 64, 64) > 0
    for scratch in (None, ctypes.c_void_p((1 << 20) + 4)):
        refused(fdx, fdx.lib.fdx_mha_packed_f32(P, I64(64 * heads), P, I64(64 * kv_heads), P, I64(64 * kv_heads), P, 1, tokens, heads, kv_heads, 64, 64, 0,
                                                P, I64(64 * heads), scratch, None), INVALID, "scratch")


def test_packed(fdx):
    def call(q=P, ldq=256, k=P, ldk=128, v=P, ldv=128, starts=P, n_seqs=3, tokens=5, heads=4, kv_heads=2, dk=64, dv=64, out=P, ldo=256):
        return fdx.lib.fdx_mha_packed_f32(q, I64(ldq), k, I64(ldk), v, I64(ldv), starts, n_seqs, tokens, heads, kv_heads, dk, dv, 1, out,
                                          I64(ldo), P, None)
    for change, text in ((dict(q=None), "null"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(starts=None), "null"),
                         (dict(out=None), "null"), (dict(n_seqs=0), "shape"), (dict(tokens=0), "shape"), (dict(heads=0), "shape"),
                         (dict(kv_heads=0), "shape"), (dict(dk=0), "shape"), (dict(dv=-1), "shape"), (dict(kv_heads=3, ldk=256, ldv=256), "share"),
                         (dict(kv_heads=8, ldk=1024, ldv=1024), "share"), (dict(ldq=255), "overlap"), (dict(ldk=1), "overlap"),
                         (dict(ldv=127), "overlap"), (dict(ldo=128), "overlap"), (dict(tokens=1 << 25), "too many"),
                         (dict(n_seqs=(1 << 22) + 1), "too many"), (dict(n_seqs=1 << 21, heads=8, kv_heads=4, ldq=512, ldk=256, ldv=256, ldo=512), "too many"),
                         (dict(tokens=(1 << 23) + 1), "too many")):
        refused(fdx, call(**change), INVALID, text)
    refused(fdx, call(dk=130, ldq=600, ldk=300), UNSUPPORTED, "depths up to 128, not 130 and 64")


def test_scores(fdx):
    def call(x=P, ld=100, rows=3, vocab=100, ids=P, top=5, logprobs=P, entropy=P, top_ids=P, top_logprobs=P):
        return fdx.lib.fdx_token_logprobs_f32(x, I64(ld), I64(rows), vocab, ids, top, logprobs, entropy, top_ids, top_logprobs, P, None)
    for change, text in ((dict(x=None), "null"), (dict(rows=0), "rows"), (dict(rows=(1 << 23) + 1), "rows"), (dict(vocab=0), "rows"),
                         (dict(vocab=(1 << 24) + 1, ld=1 << 25), "rows"), (dict(ld=99), "overlap"), (dict(ids=None), "together"),
                         (dict(logprobs=None), "together"), (dict(top=-1), "alternatives"), (dict(top=33), "alternatives"),
                         (dict(top=8, vocab=7), "alternatives"), (dict(top_ids=None), "with top"), (dict(top_logprobs=None), "with top"),
                         (dict(top=0), "with top"),
                         (dict(ids=None, logprobs=None, entropy=None, top=0, top_ids=None, top_logprobs=None), "nothing asked")):
        refused(fdx, call(**change), INVALID, text)


def test_scratch_sizes_of_refused_calls_are_zero(fdx):
    """A size for arguments that the call itself refuses: an answer, not a crash."""
    assert fdx.lib.fdx_mha_packed_scratch_bytes(0, 1, 1, 1, 64, 64) == 0
    for heads, kv_heads in ((1, 2), (3, 2), (5, 7)):
        for tokens in (5, 600, 5000):
            assert fdx.lib.fdx_mha_packed_scratch_bytes(tokens, 1, heads, kv_heads, 64, 64) == 0
            refused(fdx, fdx.lib.fdx_mha_packed_f32(P, I64(512), P, I64(512), P, I64(512), P, 1, tokens, heads, kv_heads, 64, 64, 1, P, I64(512), P, None),
                    INVALID, "share")
    assert fdx.lib.fdx_mha_packed_scratch_bytes(5, 1, 4, 0, 64, 64) == 0
    assert fdx.lib.fdx_mha_paged_scratch_bytes(5, 1, 4, None) == 0
    for change in (dict(kv_heads=0), dict(max_len=0), dict(n_seqs=-3), dict(dk=0), dict(dv=0)):
        assert fdx.lib.fdx_mha_paged_scratch_bytes(5, 1, 4, ctypes.byref(pages(fdx, **change))) == 0
    assert fdx.lib.fdx_mha_paged_scratch_bytes(0, 1, 4, ctypes.byref(pages(fdx))) == 0
    assert fdx.lib.fdx_mha_paged_scratch_bytes(5, 0, 4, ctypes.byref(pages(fdx))) == 0
    assert fdx.lib.fdx_token_logprobs_scratch_bytes(I64(0), 100, 5) == 0
    assert fdx.lib.fdx_token_logprobs_scratch_bytes(I64(5), -1, 5) == 0


def test_rows_and_pages_on_the_host(tmp_path):
    exe = str(tmp_path / "kv_pages_test.bin")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=undefined",
                           "-I" + os.path.join(ROOT, "frugally-deep_amd", "csrc"), os.path.join(ROOT, "tests", "cpp", "kv_pages_test.cpp"),
                           "-o", exe])
    out = subprocess.run([exe], capture_output=True, text=True, timeout=300, env=dict(os.environ, ASAN_OPTIONS="detect_leaks=0"))
    assert out.returncode == 0 and "kv_pages done" in out.stdout, (out.stdout, out.stderr[-3000:])


class HostBuf:
    """Memory that no call looks into."""

    def __init__(self, nbytes=0):
        self.ptr = P

    @classmethod
    def from_host(cls, arr, dtype=None):
        return cls()


def cache_on_host(fdx, monkeypatch, **change):
    args = dict(n_pages=9, page_size=4, kv_heads=2, dk=8, dv=6, n_seqs=3, max_len=20)
    args.update(change)
    monkeypatch.setattr(fdx, "DevBuf", HostBuf)
    return fdx.PagedCache(**args)


@pytest.mark.parametrize("how", ["memory", "call", "flag"])
def test_append_that_fails_leaves_the_cache(fdx, monkeypatch, how):
    """Lengths, page table and free pages (their order too) are those in front of the call, and the next call takes the same pages."""
    cache = cache_on_host(fdx, monkeypatch)
    cache.grow([5, 0, 4])
    table, lens, free = cache.table.copy(), cache.lens.copy(), list(cache.free)
    k, v = np.zeros((12, 16), np.float32), np.zeros((12, 12), np.float32)

    def fail(*args):
        raise fdx.FdxError("failed on purpose")
    with monkeypatch.context() as m:
        m.setattr(fdx, "check", fail if how == "call" else lambda status: None)
        m.setattr(fdx, "_raise_if_set", fail if how == "flag" else lambda flag, message: None)
        m.setattr(fdx.lib, "fdx_kv_append_f32", lambda *args: 0)
        if how == "memory":
            m.setattr(HostBuf, "from_host", classmethod(lambda cls, arr, dtype=None: fail()))
        with pytest.raises(fdx.FdxError, match="on purpose"):
            fdx.kv_append(cache, k, v, [2, 9, 1])
    assert np.array_equal(cache.table, table) and np.array_equal(cache.lens, lens) and cache.free == free
    with pytest.raises(fdx.FdxError, match="free pages"):
        fdx.kv_append(cache, np.zeros((34, 16), np.float32), np.zeros((34, 12), np.float32), [8, 17, 9])
    assert np.array_equal(cache.table, table) and np.array_equal(cache.lens, lens) and cache.free == free
    with monkeypatch.context() as m:
        m.setattr(fdx, "_raise_if_set", lambda flag, message: None)
        m.setattr(fdx.lib, "fdx_kv_append_f32", lambda *args: 0)
        fdx.kv_append(cache, k, v, [2, 9, 1])
    assert cache.lens.tolist() == [7, 9, 5] and sorted(cache.free + [int(x) for x in cache.table.ravel() if x >= 0]) == list(range(9))


def test_nothing_new(fdx, monkeypatch):
    """Batches without a row: nothing to write, no rows of attention; shapes are checked all the same."""
    cache = cache_on_host(fdx, monkeypatch)
    cache.grow([5, 0, 4])
    none = lambda width: np.zeros((0, width), np.float32)
    fdx.kv_append(cache, none(16), none(12), [0, 0, 0])
    assert cache.lens.tolist() == [5, 0, 4]
    assert fdx.mha_paged(cache, none(32), [0, 0, 0], 4).shape == (0, 24)
    for lengths in ([0, 0], []):
        assert fdx.mha_packed(none(32), none(16), none(12), lengths, 4, 2, 8, 6).shape == (0, 24)
    with pytest.raises(fdx.FdxError, match="q of shape"):
        fdx.mha_paged(cache, none(32), [0, 1, 0], 4)
    with pytest.raises(fdx.FdxError, match="q of shape"):
        fdx.mha_paged(cache, none(16), [0, 0, 0], 4)
    with pytest.raises(fdx.FdxError, match="v of shape"):
        fdx.mha_packed(none(32), none(16), none(16), [0], 4, 2, 8, 6)


@pytest.mark.parametrize("lengths", [[2.5, 2.5], [float("nan"), 5], [1e30, 5], [2**32, 5], [2**32 - 3, 8], [2**63 - 1, 2**63 - 1], [2**64 - 1, 6], [5, 1],
                                     [7, -2], ["5"], [None]])
def test_lengths_that_are_none(fdx, monkeypatch, lengths):
    """Numbers that 32 bits or whole numbers would make others of are refused before anything is cut or kept."""
    cache = cache_on_host(fdx, monkeypatch, n_seqs=2)
    q, k, v = np.zeros((5, 32), np.float32), np.zeros((5, 16), np.float32), np.zeros((5, 12), np.float32)
    with pytest.raises(fdx.FdxError, match="lengths"):
        fdx.mha_packed(q, k, v, lengths, 4, 2, 8, 6)
    with pytest.raises(fdx.FdxError):
        fdx.kv_append(cache, k, v, lengths)
    with pytest.raises(fdx.FdxError):
        fdx.mha_paged(cache, q, lengths, 4)
    assert cache.lens.tolist() == [0, 0]


@pytest.mark.parametrize("ids", [[0, 10], [0, 2**31], [2**32, 1], [2**32 + 3, 1], [0, 2**63], [2**64 - 1, 1], [0.5, 1], [1e30, 0], [float("nan"), 0], ["0", "1"]])
def test_ids_that_are_none(fdx, monkeypatch, ids):
    monkeypatch.setattr(fdx, "DevBuf", HostBuf)
    with pytest.raises(fdx.FdxError, match="less than the number of logits|whole numbers"):
        fdx.token_logprobs(np.zeros((2, 10), np.float32), ids)


def test_numbers_in_any_type(fdx):
    """Whole numbers of every type are taken as they are."""
    for dtype in (np.int8, np.uint8, np.int32, np.int64, np.uint64, np.float32, np.float64):
        assert fdx._whole("ids", np.array([0, 7, 100], dtype)).tolist() == [0, 7, 100]
    assert fdx._whole("ids", [-2**63, 2**62 + 1, True]).tolist() == [-2**63, 2**62 + 1, 1]
    assert fdx._whole("lengths", []).shape == (0,) and fdx._whole("lengths", 5).shape == ()
