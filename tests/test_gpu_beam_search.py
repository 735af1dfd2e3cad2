"""A beam search of a one-layer decoder over a cache in 8 bits, step by step on the device: page tables follow the beams, keys and values go into
their pages, attention reads them, its output meets the vocabulary, the best continuations are chosen; nothing but the chosen tokens comes to the host.
Beside it the same search in 64 bits over a cache on the host (cache8.py) without pages: every beam has its own list of positions, copied whole."""
import ctypes

import numpy as np
import pytest

from cache8 import HostCache

pytestmark = pytest.mark.gpu
I64 = ctypes.c_int64


class Beam:
    """One beam's cache on the host, a block's codes and scale for each `block` positions: what HostCache does, in pages of its own."""

    def __init__(self, kv, d, kind, block, most):
        self.host, self.length = HostCache(1, -(-most // block) * block, kv, d, d, kind, block), 0

    def copy(self):
        other = Beam.__new__(Beam)
        other.host = HostCache.__new__(HostCache)
        other.host.__dict__.update(self.host.__dict__, codes=[c.copy() for c in self.host.codes], scales=[s.copy() for s in self.host.scales])
        other.length = self.length
        return other

    def append(self, k, v):
        for which, x in enumerate((k, v)):
            self.host.append(lambda p: p, self.length, x, which)
        self.length += len(k)

    def attend(self, q, heads):
        kv = self.host.kv
        k, v = (self.host.values(np.arange(self.length), w).reshape(self.length, kv, -1) for w in (0, 1))
        out = []
        for h in range(heads):
            x = k[:, h * kv // heads] @ q[h] / np.sqrt(len(q[h]))
            e = np.exp(x - x.max())
            out.append(e / e.sum() @ v[:, h * kv // heads])
        return np.concatenate(out)


class Decoder:
    """Embeddings that are queries, keys and values at once, one attention layer, a head; prompts of three users."""
    beams, heads, kv, d, vocab, steps, prompt, end_id = 4, 4, 2, 64, 2003, 24, (13, 5, 21), 7

    def __init__(self, seed):
        r = np.random.default_rng(seed)
        self.emb = {name: r.standard_normal((self.vocab, width * self.d)).astype(np.float32) for name, width in (("q", self.heads), ("k", self.kv), ("v", self.kv))}
        self.head = (r.standard_normal((self.vocab, self.heads * self.d)) * 0.3).astype(np.float32)
        self.prompts = [r.integers(0, self.vocab, m) for m in self.prompt]
        self.n, self.most = len(self.prompt) * self.beams, max(self.prompt) + self.steps + 1

    def first(self):
        """(tokens, scores) of the first step: a prompt's last token, one live beam each"""
        return np.array([self.prompts[i // self.beams][-1] for i in range(self.n)]), np.where(np.arange(self.n) % self.beams == 0, 0.0, -np.inf)


def search(m, kind, block, apart):
    """(parents, tokens, scores, ended) of every step in 64 bits, or None if two candidates beside each other come nearer than `apart`"""
    host, out = [], []
    for p in m.prompts:
        b = Beam(m.kv, m.d, kind, block, m.most)
        b.append(m.emb["k"][p[:-1]].reshape(-1, m.kv, m.d), m.emb["v"][p[:-1]].reshape(-1, m.kv, m.d))
        host += [b.copy() for _ in range(m.beams)]
    (tokens, scores), done = m.first(), np.zeros(m.n, bool)
    for _ in range(m.steps):
        logits = np.empty((m.n, m.vocab))
        for i, b in enumerate(host):
            b.append(m.emb["k"][tokens[i]].reshape(1, m.kv, m.d), m.emb["v"][tokens[i]].reshape(1, m.kv, m.d))
            logits[i] = m.head.astype(np.float64) @ b.attend(m.emb["q"][tokens[i]].reshape(m.heads, m.d).astype(np.float64), m.heads)
        chosen = []
        for g in range(0, m.n, m.beams):
            every = []
            for b in range(g, g + m.beams):
                if scores[b] == -np.inf:
                    continue
                if done[b]:
                    every.append((scores[b], b, m.end_id))
                    continue
                lse = logits[b].max() + np.log(np.exp(logits[b] - logits[b].max()).sum())
                every += [(scores[b] + logits[b][t] - lse, b, int(t)) for t in np.argsort(-logits[b], kind="stable")[:m.beams + 1]]
            every.sort(key=lambda e: (-e[0], e[1]))
            if any(a[0] - b[0] < apart for a, b in zip(every[:m.beams], every[1:])):
                return None
            chosen += every[:m.beams]
        host = [host[b].copy() for _, b, _ in chosen]
        done = np.array([t == m.end_id or bool(done[b]) for _, b, t in chosen])
        scores, tokens = np.array([s for s, _, _ in chosen]), np.array([t for _, _, t in chosen])
        out.append(([b for _, b, _ in chosen], tokens.tolist(), scores, done.astype(int).tolist()))
    return out


@pytest.mark.parametrize("kind,page,block", [("i8", 16, 16), ("e4m3", 8, 4), ("i8", 5, 1)])
def test_beam_search(fdx, kind, page, block):
    # a step's log probabilities are off by the error of its logits, sums of 256 products of 0.3 and values of one: 2e-6; 24 steps: 5e-5
    apart = 5e-5
    for seed in range(30):   # the first decoder whose candidates are further apart than that
        m = Decoder(seed)
        want = search(m, kind, block, apart)
        if want:
            break
    assert want
    n, heads, kv, d, vocab, beams = m.n, m.heads, m.kv, m.d, m.vocab, m.beams
    print("beam search", kind, page, block, seed, flush=True)

    # a prompt is written once, its beams go on from their group's first
    c = fdx.PagedCache(n * (-(-m.most // page)) + 2 * n, page, kv, d, d, n, -(-m.most // page) * page, kind, block)
    np.random.default_rng(1).shuffle(c.free)
    ids = np.concatenate([p[:-1] for p in m.prompts])
    fdx.kv_append(c, m.emb["k"][ids], m.emb["v"][ids], [m.prompt[i // beams] - 1 if i % beams == 0 else 0 for i in range(n)])
    fdx.kv_fork(c, np.arange(n) // beams * beams)
    ints = lambda a: fdx.DevBuf.from_host(np.asarray(a, np.int32), np.int32)
    cache = [c.pages(), c.pages()]                    # two tables that take turns
    tables, lens = [ints(c.table), ints(c.table)], [ints(c.lens), ints(c.lens)]
    for z in (0, 1):
        cache[z].pages.table, cache[z].pages.lens = tables[z].ptr, lens[z].ptr
    grow, starts, flag, free = ints(np.ones(n)), ints(np.arange(n + 1)), ints([0]), ints([0])
    # one workspace for all calls: they follow each other on one stream
    scratch = fdx.DevBuf(max(fdx.lib.fdx_kv8_fork_scratch_bytes(ctypes.byref(cache[0])), fdx.lib.fdx_mha_paged8_scratch_bytes(n, 1, heads, ctypes.byref(cache[0])),
                             fdx.lib.fdx_beam_select_scratch_bytes(n // beams, beams, vocab, beams)))
    rows, out = {name: fdx.DevBuf(4 * n * e.shape[1]) for name, e in m.emb.items()}, fdx.DevBuf(4 * n * heads * d)
    first, start = m.first()
    tokens, parents, new_parents, done, new_done = ints(first), ints(np.arange(n)), ints(np.arange(n)), ints(np.zeros(n)), ints(np.zeros(n))
    scores, new_scores = fdx.DevBuf.from_host(start), fdx.DevBuf.from_host(start)
    at, lib, check = 0, fdx.lib, fdx.check
    for step, (want_parents, want_tokens, want_scores, want_done) in enumerate(want):
        check(lib.fdx_kv8_fork(ctypes.byref(cache[at]), parents.ptr, grow.ptr, tables[1 - at].ptr, lens[1 - at].ptr, free.ptr, scratch.ptr, flag.ptr))
        at = 1 - at
        now = tokens.to_host((n,), np.int32)
        for name, e in m.emb.items():
            check(lib.fdx_h2d(rows[name].ptr, np.ascontiguousarray(e[now]).ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(4 * n * e.shape[1])))
        check(lib.fdx_kv8_append_f32(rows["k"].ptr, I64(kv * d), rows["v"].ptr, I64(kv * d), starts.ptr, n, ctypes.byref(cache[at]), flag.ptr))
        check(lib.fdx_mha_paged8_f32(rows["q"].ptr, I64(heads * d), starts.ptr, n, 1, heads, ctypes.byref(cache[at]), out.ptr, I64(heads * d),
                                     scratch.ptr, flag.ptr))
        x = fdx.DevBuf.from_host(out.to_host((n, heads * d)) @ m.head.T)
        check(lib.fdx_beam_select_f32(x.ptr, I64(vocab), n // beams, beams, vocab, scores.ptr, done.ptr, m.end_id, beams, new_parents.ptr, tokens.ptr,
                                      new_scores.ptr, new_done.ptr, scratch.ptr, flag.ptr))
        parents, new_parents, scores, new_scores, done, new_done = new_parents, parents, new_scores, scores, new_done, done
        assert parents.to_host((n,), np.int32).tolist() == want_parents, step
        assert tokens.to_host((n,), np.int32).tolist() == want_tokens, step
        assert np.abs(scores.to_host((n,)) - want_scores).max() <= apart
        assert done.to_host((n,), np.int32).tolist() == want_done
        assert int(flag.to_host((1,), np.int32)[0]) == 0
    used = set(tables[at].to_host(c.table.shape, np.int32).ravel().tolist()) - {-1}
    assert int(free.to_host((1,), np.int32)[0]) == c.n_pages - len(used)
    assert lens[at].to_host((n,), np.int32).tolist() == [m.prompt[i // beams] - 1 + m.steps for i in range(n)]
