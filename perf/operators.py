"""The operators a program serves prompts and scores tokens with, as timed cases: attention over packed prompts, keys and values
written to the pages of a cache, attention of new tokens over such pages, and log probabilities of tokens.

A case names an operator and its sizes.  The operators:

  packed    attention inside each of several sequences whose rows lie one behind the other (fdx_mha_packed_f32); query heads share
            key / value heads
  append    the keys and values of new tokens into the pages of their sequences (fdx_kv_append_f32)
  paged     the new tokens of every sequence, one or a chunk of them, over all keys in its pages (fdx_mha_paged_f32)
  logprobs  per row of logits: the log probability of a given token, the entropy, the likeliest tokens (fdx_token_logprobs_f32)

Sequence lengths follow from a case's numbers alone: between `short` and `long`, spread over their logarithm, the first one `long`.
The pages of a sequence are scattered over the cache.
"""
import ctypes
import importlib
import math
import random

import torch

own = False

VOCAB = 50257   # the decoder's vocabulary


def listed():
    return [
        # one short prompt on the decoder's heads: all latency
        dict(name="packed_one_37", op="packed", seqs=1, short=37, long=37, heads=12, kv_heads=12, dk=64, dv=64, causal=True),
        # prompts of a batch of users, none as long as another, nothing padded
        dict(name="packed_24_ragged", op="packed", seqs=24, short=9, long=700, heads=12, kv_heads=12, dk=64, dv=64, causal=True),
        # sentences for the encoder, both directions
        dict(name="packed_48_encoder", op="packed", seqs=48, short=20, long=256, heads=8, kv_heads=8, dk=64, dv=64, causal=False),
        # two long documents, four query heads on a key head
        dict(name="packed_2_long", op="packed", seqs=2, short=4001, long=8192, heads=32, kv_heads=8, dk=128, dv=128, causal=True),
        # one step of a batch of generating users: a row each
        dict(name="append_64_step", op="append", seqs=64, short=100, long=4000, new_short=1, new_long=1, kv_heads=8, dk=128, dv=128,
             page=16, kind="bf16"),
        # prompts on their way into the cache
        dict(name="append_prompts", op="append", seqs=20, short=700, long=4000, new_short=300, new_long=4000, kv_heads=8, dk=128, dv=128,
             page=64, kind="f32"),
        # one user's next token on the decoder's heads
        dict(name="paged_1_token", op="paged", seqs=1, short=201, long=201, new_short=1, new_long=1, heads=12, kv_heads=12, dk=64, dv=64,
             page=16, kind="f32"),
        # a loaded server's step: a token each, contexts from short to long, cache in half the bytes
        dict(name="paged_64_tokens", op="paged", seqs=64, short=300, long=7900, new_short=1, new_long=1, heads=32, kv_heads=8, dk=128,
             dv=128, page=16, kind="bf16"),
        # prompts cut into chunks beside users with one token each
        dict(name="paged_12_chunks", op="paged", seqs=12, short=400, long=12000, new_short=1, new_long=1024, heads=32, kv_heads=8, dk=128,
             dv=128, page=32, kind="f32"),
        # the scores of one step's tokens, with a few alternatives
        dict(name="logprobs_16", op="logprobs", rows=16, vocab=VOCAB, top=5, masked=False),
        # a constrained decoder: most of the vocabulary ruled out
        dict(name="logprobs_5_masked", op="logprobs", rows=5, vocab=32001, top=20, masked=True),
        # the tokens of prompts scored at once
        dict(name="logprobs_2048", op="logprobs", rows=2048, vocab=VOCAB, top=20, masked=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_HEADS = [(12, 12, 64, 64), (8, 8, 64, 64), (32, 8, 128, 128), (16, 4, 64, 64), (8, 1, 128, 128), (10, 5, 80, 80), (6, 6, 32, 32),
          (28, 4, 128, 128), (4, 2, 96, 64)]


def draw(rng):
    most = {}
    for case in listed():
        w = work(case)
        most[case["op"]] = [max(a, b) for a, b in zip(most.get(case["op"], (0, 0)), (w["bytes"], w["flops"]))]
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] <= most[case["op"]][0] and w["flops"] <= most[case["op"]][1]:
            return case


def _draw(rng):
    op = rng.choice(["packed", "packed", "append", "paged", "paged", "paged", "logprobs"])
    if op == "logprobs":
        rows = _log_int(rng, 1, 2048)
        return dict(op=op, rows=rows, vocab=rng.choice([VOCAB, _log_int(rng, 1000, 131072 if rows <= 700 else VOCAB)]),
                    top=rng.choice([0, 1, 5, rng.randint(2, 32)]), masked=rng.random() < 0.25)
    heads, kv_heads, dk, dv = rng.choice(_HEADS)
    if op == "packed":
        long = _log_int(rng, 16, 6000)
        return dict(op=op, seqs=_log_int(rng, 1, max(1, min(64, 24000 // long))), short=rng.randint(1, long), long=long, heads=heads,
                    kv_heads=kv_heads, dk=dk, dv=dv, causal=rng.random() < 0.75)
    long = _log_int(rng, 64, 8000)
    seqs = _log_int(rng, 1, max(1, min(64, 160000 // long)))
    page, kind, short = rng.choice([16, 32, 64, 128, rng.randint(5, 200)]), rng.choice(["f32", "bf16"]), rng.randint(1, long)
    if op == "append":
        new_long = rng.choice([1, _log_int(rng, 2, long)])
        most = max(1, 30000 // new_long)
        return dict(op=op, seqs=min(seqs, most), short=short, long=long, new_short=rng.randint(1, new_long), new_long=new_long,
                    kv_heads=kv_heads, dk=dk, dv=dv, page=page, kind=kind)
    new_long = rng.choice([1, 1, rng.randint(2, 16), _log_int(rng, 16, 600)])
    most = max(1, int(2e7 / (long * new_long)))
    return dict(op=op, seqs=min(seqs, most), short=short, long=long, new_short=rng.randint(1, new_long), new_long=new_long, heads=heads,
                kv_heads=kv_heads, dk=dk, dv=dv, page=page, kind=kind)


# ---------------------------------------------------------------- sizes that follow from a case

def _spread(count, short, long):
    rng = random.Random("%d %d %d" % (count, short, long))
    return [long] + [_log_int(rng, short, long) for _ in range(count - 1)]


def _sizes(case):
    """(keys of every sequence, new tokens of every sequence); a sequence has at least as many keys as new tokens"""
    lens = _spread(case["seqs"], case["short"], case["long"])
    if case["op"] == "packed":
        return lens, lens
    new = _spread(case["seqs"], case["new_short"], case["new_long"])
    if case["op"] == "paged":
        new = new[1:] + new[:1]   # the longest chunk is not the one with the longest context
    return lens, [min(n, length) for n, length in zip(new, lens)]


def _starts(new):
    out = [0]
    for n in new:
        out.append(out[-1] + n)
    return out


# ---------------------------------------------------------------- inputs

class _Buf:
    """A torch tensor's memory in the form that the framework's calls take."""

    def __init__(self, t):
        self.tensor, self.ptr = t, ctypes.c_void_p(t.data_ptr())


def _out(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    st = dict(case)
    if case["op"] == "logprobs":
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        # a few tokens stand out in every row
        x = 2.5 * normal(rows, vocab)
        x.scatter_add_(1, torch.randint(0, vocab, (rows, 6), generator=gen, device="cuda"), 8 * torch.rand((rows, 6), generator=gen, device="cuda"))
        if case["masked"]:
            x[torch.rand((rows, vocab), generator=gen, device="cuda") > max(0.02, 200 / vocab)] = -math.inf
            x[:, 0] = 0.0   # the end of the text is always allowed
        ids = torch.where(torch.rand((rows,), generator=gen, device="cuda") < 0.5, x.argmax(1),
                          torch.randint(0, vocab, (rows,), generator=gen, device="cuda")).to(torch.int32)
        if case["masked"]:
            ids = torch.where(torch.isinf(x[torch.arange(rows, device="cuda"), ids.long()]), torch.zeros_like(ids), ids)
        st.update(x=x, ids=ids, logprobs=_out(rows), entropy=_out(rows))
        if top:
            st.update(top_ids=_out(rows, top, dtype=torch.int32), top_logprobs=_out(rows, top))
        if own:
            fdx = _fdx()
            st.update(scratch=_out(fdx.lib.fdx_token_logprobs_scratch_bytes(ctypes.c_int64(rows), vocab, top) // 4 + 4))
        torch.cuda.synchronize()   # the framework works on a stream of its own
        return st

    lens, new = _sizes(case)
    starts, kv, dk, dv = _starts(new), case["kv_heads"], case["dk"], case["dv"]
    tokens = starts[-1]
    st.update(lens_list=lens, starts_list=starts, tokens=tokens, starts=torch.tensor(starts, dtype=torch.int32, device="cuda"))
    if case["op"] != "paged":
        st.update(k=normal(tokens, kv * dk), v=normal(tokens, kv * dv))
    if case["op"] != "append":
        st.update(q=1.5 * normal(tokens, case["heads"] * dk), out=_out(tokens, case["heads"] * dv))
    if case["op"] != "packed":
        page = case["page"]
        counts = [-(-length // page) for length in lens]
        n_pages, width = sum(counts) + 3, max(counts)
        kind = torch.float32 if case["kind"] == "f32" else torch.bfloat16
        order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
        table, at = torch.full((case["seqs"], width), -1, dtype=torch.int32, device="cuda"), 0
        for s, count in enumerate(counts):
            table[s, :count] = order[at:at + count]
            at += count
        st.update(table=table, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                  k_pages=normal(n_pages, page, kv, dk).to(kind), v_pages=normal(n_pages, page, kv, dv).to(kind))
    if own:
        fdx = _fdx()
        if case["op"] == "packed":
            need = fdx.lib.fdx_mha_packed_scratch_bytes(tokens, case["seqs"], case["heads"], kv, dk, dv)
            st.update(scratch=_out(need // 4 + 4))
        else:
            st.update(cache=fdx.KvPages(_Buf(st["k_pages"]), _Buf(st["v_pages"]), case["kind"], n_pages, page, kv, dk, dv,
                                        _Buf(st["table"]), width, _Buf(st["lens"]), case["seqs"], max(lens)))
            if case["op"] == "paged":
                need = fdx.lib.fdx_mha_paged_scratch_bytes(tokens, max(new), case["heads"], ctypes.byref(st["cache"]))
                st.update(scratch=_out(need // 4 + 4), max_new=max(new))
    torch.cuda.synchronize()   # the framework works on a stream of its own
    return st


# ---------------------------------------------------------------- the framework's calls

def _fdx():
    return importlib.import_module("frugally-deep_amd")


def _p(t):
    return ctypes.c_void_p(t.data_ptr())


def _run_own(st):
    fdx, i64 = _fdx(), ctypes.c_int64
    if st["op"] == "logprobs":
        top, vocab = st["top"], st["vocab"]
        fdx.check(fdx.lib.fdx_token_logprobs_f32(
            _p(st["x"]), i64(vocab), i64(st["rows"]), vocab, _p(st["ids"]), top, _p(st["logprobs"]), _p(st["entropy"]),
            _p(st["top_ids"]) if top else None, _p(st["top_logprobs"]) if top else None, _p(st["scratch"]), None))
        return {key: st[key] for key in ("logprobs", "entropy", "top_ids", "top_logprobs") if key in st}
    kv, dk, dv, tokens = st["kv_heads"], st["dk"], st["dv"], st["tokens"]
    if st["op"] == "packed":
        heads = st["heads"]
        fdx.check(fdx.lib.fdx_mha_packed_f32(
            _p(st["q"]), i64(heads * dk), _p(st["k"]), i64(kv * dk), _p(st["v"]), i64(kv * dv), _p(st["starts"]), st["seqs"], tokens,
            heads, kv, dk, dv, int(st["causal"]), _p(st["out"]), i64(heads * dv), _p(st["scratch"]), None))
        return st["out"]
    if st["op"] == "append":
        fdx.check(fdx.lib.fdx_kv_append_f32(_p(st["k"]), i64(kv * dk), _p(st["v"]), i64(kv * dv), _p(st["starts"]), tokens,
                                            ctypes.byref(st["cache"]), None))
        return dict(k_pages=st["k_pages"], v_pages=st["v_pages"])
    heads = st["heads"]
    fdx.check(fdx.lib.fdx_mha_paged_f32(_p(st["q"]), i64(heads * dk), _p(st["starts"]), tokens, st["max_new"], heads,
                                        ctypes.byref(st["cache"]), _p(st["out"]), i64(heads * dv), _p(st["scratch"]), None))
    return st["out"]


# ---------------------------------------------------------------- the plain forms

def _slots(st, seq, first, last):
    """rows of the cache, its pages one behind the other, that hold positions first .. last - 1 of a sequence"""
    at = torch.arange(first, last, device="cuda")
    return st["table"][seq].long()[at // st["page"]] * st["page"] + at % st["page"]


def _plain_attention(q, k, v, hidden_from):
    """q [n][heads][dk], k [keys][kv][dk], v [keys][kv][dv]; query i sees the keys below hidden_from[i]"""
    n, heads, dk = q.shape
    keys, kv = k.shape[:2]
    group = heads // kv
    out = torch.empty((n, heads, v.shape[2]), device="cuda")
    hidden = torch.arange(keys, device="cuda")[None, :] >= hidden_from[:, None]
    scale = 1.0 / math.sqrt(dk)
    step = max(1, min(kv, 300_000_000 // max(1, n * group * keys)))   # heads at a time, by the memory of their scores
    for h in range(0, kv, step):
        m = min(step, kv - h)
        qs = q[:, h * group:(h + m) * group].reshape(n, m, group, dk).permute(1, 2, 0, 3).reshape(m, group * n, dk)
        s = torch.matmul(qs, k[:, h:h + m].permute(1, 2, 0).contiguous()) * scale
        s = s.view(m, group, n, keys).masked_fill_(hidden, -math.inf)
        s = torch.exp(s - s.amax(-1, keepdim=True))
        s = s / s.sum(-1, keepdim=True)
        o = torch.matmul(s.view(m, group * n, keys), v[:, h:h + m].permute(1, 0, 2).contiguous())
        out[:, h * group:(h + m) * group] = o.view(m, group, n, -1).permute(2, 0, 1, 3).reshape(n, m * group, -1)
    return out


def _run_plain(st):
    if st["op"] == "logprobs":
        x, rows = st["x"], torch.arange(st["rows"], device="cuda")
        shifted = x - x.amax(1, keepdim=True)
        e = torch.exp(shifted)
        total = e.sum(1, keepdim=True)
        log_total = torch.log(total)
        weighted = torch.where(e > 0, e * shifted, torch.zeros_like(e)).sum(1)
        out = dict(logprobs=shifted[rows, st["ids"].long()] - log_total[:, 0], entropy=log_total[:, 0] - weighted / total[:, 0])
        if st["top"]:
            best = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :st["top"]]
            out.update(top_ids=best.to(torch.int32), top_logprobs=torch.gather(shifted, 1, best) - log_total)
        return out
    starts, kv, dk, dv = st["starts_list"], st["kv_heads"], st["dk"], st["dv"]
    if st["op"] == "append":
        k_rows, v_rows = st["k_pages"].view(-1, kv, dk), st["v_pages"].view(-1, kv, dv)
        for s, length in enumerate(st["lens_list"]):
            a, b = starts[s], starts[s + 1]
            slots = _slots(st, s, length - (b - a), length)
            k_rows[slots] = st["k"][a:b].view(b - a, kv, dk).to(k_rows.dtype)
            v_rows[slots] = st["v"][a:b].view(b - a, kv, dv).to(v_rows.dtype)
        return dict(k_pages=st["k_pages"], v_pages=st["v_pages"])
    heads, out = st["heads"], torch.empty_like(st["out"])
    for s, length in enumerate(st["lens_list"]):
        a, b = starts[s], starts[s + 1]
        if st["op"] == "packed":
            k, v = st["k"][a:b].view(-1, kv, dk), st["v"][a:b].view(-1, kv, dv)
        else:
            slots = _slots(st, s, 0, length)
            k, v = st["k_pages"].view(-1, kv, dk)[slots].float(), st["v_pages"].view(-1, kv, dv)[slots].float()
        hidden_from = torch.arange(length - (b - a), length, device="cuda") + 1
        if not st.get("causal", True):
            hidden_from = torch.full_like(hidden_from, length)
        out[a:b] = _plain_attention(st["q"][a:b].view(-1, heads, dk), k, v, hidden_from).view(b - a, heads * dv)
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["op"] == "logprobs":
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        # per logit: difference, exponential, two sums, a product
        return {"bytes": 4 * rows * (vocab + 3 + 2 * top), "flops": 5 * rows * vocab}
    lens, new = _sizes(case)
    kv, dk, dv, tokens = case["kv_heads"], case["dk"], case["dv"], sum(new)
    held = 2 if case.get("kind") == "bf16" else 4
    if case["op"] == "append":
        return {"bytes": tokens * kv * (dk + dv) * (4 + held) + 4 * sum(-(-n // case["page"]) for n in new), "flops": 0}
    heads = case["heads"]
    # query i of n new ones sees length - n + i + 1 keys
    pairs = sum(n * (length - n) + n * (n + 1) // 2 if case.get("causal", True) else n * length for n, length in zip(new, lens))
    nbytes = 4 * tokens * heads * (dk + dv) + sum(lens) * kv * (dk + dv) * held
    if case["op"] == "paged":
        nbytes += 4 * sum(-(-length // case["page"]) for length in lens)
    return {"bytes": nbytes, "flops": 2 * heads * pairs * (dk + dv)}


# ---------------------------------------------------------------- from the definitions, in 64 bits

def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    f64 = torch.float64
    if case["op"] == "logprobs":
        rows, top = case["rows"], case["top"]
        logprobs, entropy, ids, alternatives = [], [], [], []
        for r in range(rows):
            x = st["x"][r].to(f64)
            lse = torch.logsumexp(x, 0)
            lp = x - lse
            p = lp.exp()
            logprobs.append(lp[st["ids"][r].long()])
            entropy.append(-(p[p > 0] * lp[p > 0]).sum())
            if top:   # the largest values; where two are equal, the lower index
                cut = torch.topk(x, top).values[-1]
                index = torch.nonzero(x >= cut)[:, 0].cpu().tolist()
                value = x[index].cpu().tolist()
                best = sorted(zip(value, index), key=lambda vi: (-vi[0], vi[1]))[:top]
                ids.append([i for _, i in best])
                alternatives.append(lp[[i for _, i in best]])
        out = dict(logprobs=torch.stack(logprobs), entropy=torch.stack(entropy))
        if top:
            out.update(top_ids=torch.tensor(ids, dtype=torch.int32, device="cuda"), top_logprobs=torch.stack(alternatives))
        return out
    lens, new = _sizes(case)
    kv, dk, dv, starts = case["kv_heads"], case["dk"], case["dv"], _starts(new)
    if case["op"] == "append":
        table, page = st["table"].cpu().tolist(), case["page"]
        where = [table[s][pos // page] * page + pos % page for s in range(case["seqs"]) for pos in range(lens[s] - new[s], lens[s])]
        where = torch.tensor(where, device="cuda")
        out = {}
        for name, d in (("k", dk), ("v", dv)):
            pages = st[name + "_pages"].to(f64)
            pages.view(-1, kv * d).index_copy_(0, where, st[name].to(f64))
            out[name + "_pages"] = pages
        return out
    heads = case["heads"]
    group, out = heads // kv, torch.zeros((starts[-1], heads, dv), dtype=f64, device="cuda")
    for s in range(case["seqs"]):
        a, n, length = starts[s], new[s], lens[s]
        if case["op"] == "packed":
            keys, values = st["k"][a:a + n].view(n, kv, dk), st["v"][a:a + n].view(n, kv, dv)
        else:
            page = case["page"]
            held = st["table"][s, :-(-length // page)].long()
            keys, values = st["k_pages"][held].reshape(-1, kv, dk)[:length], st["v_pages"][held].reshape(-1, kv, dv)[:length]
        for h in range(heads):
            kh, vh = keys[:, h // group].to(f64), values[:, h // group].to(f64)
            for i in range(0, n, 2048):
                m = min(2048, n - i)
                x = st["q"][a + i:a + i + m, h * dk:(h + 1) * dk].to(f64) @ kh.t() / math.sqrt(dk)
                if case.get("causal", True):
                    x = x.masked_fill(torch.ones_like(x, dtype=torch.bool).triu(length - n + i + 1), -math.inf)
                out[a + i:a + i + m, h] = torch.softmax(x, -1) @ vh
    return out.view(starts[-1], heads * dv)
