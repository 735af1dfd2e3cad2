"""The operators of a beam search over a key / value cache in 8 bits, as timed cases.

A case names an operator and its sizes.  The operators:

  append   the keys and values of new tokens into pages of 8-bit codes, a scale for each block of tokens and key head
           (fdx_kv8_append_f32)
  paged    the new tokens of every sequence, one or a chunk of them, over all keys in such pages (fdx_mha_paged8_f32)
  beam     of all continuations of a sequence's beams the best ones (fdx_beam_select_f32)
  fork     the page table after a selection: sequence i goes on as a copy of sequence parents[i], with room for more tokens
           (fdx_kv_fork, fdx_kv8_fork)

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
MOST_CODE = {"i8": 127.0, "e4m3": 448.0}
TINY = 2.0 ** -126
ELEMENT = {"f32": torch.float32, "bf16": torch.bfloat16, "i8": torch.int8, "e4m3": torch.float8_e4m3fn}
BYTES = {"f32": 4, "bf16": 2, "i8": 1, "e4m3": 1}


def listed():
    return [
        # one step of a batch of generating users: a token each, most of them into a block that is partly filled
        dict(name="append_64_step", op="append", seqs=64, short=100, long=4000, new_short=1, new_long=1, kv_heads=8, dk=128, dv=128,
             page=16, block=16, kind="e4m3"),
        # prompts on their way into the cache
        dict(name="append_prompts", op="append", seqs=20, short=700, long=4000, new_short=300, new_long=4000, kv_heads=8, dk=128, dv=128,
             page=64, block=32, kind="i8"),
        # one user's next token on the decoder's heads
        dict(name="paged_1_token", op="paged", seqs=1, short=201, long=201, new_short=1, new_long=1, heads=12, kv_heads=12, dk=64, dv=64,
             page=16, block=16, kind="i8"),
        # a loaded server's step: a token each, contexts from short to long
        dict(name="paged_64_tokens", op="paged", seqs=64, short=300, long=7900, new_short=1, new_long=1, heads=32, kv_heads=8, dk=128,
             dv=128, page=16, block=16, kind="e4m3"),
        # one user's next token behind a book
        dict(name="paged_1_long", op="paged", seqs=1, short=100_003, long=100_003, new_short=1, new_long=1, heads=32, kv_heads=8, dk=128,
             dv=128, page=64, block=16, kind="i8"),
        # prompts cut into chunks beside users with one token each
        dict(name="paged_12_chunks", op="paged", seqs=12, short=400, long=12000, new_short=1, new_long=1024, heads=32, kv_heads=8, dk=128,
             dv=128, page=32, block=32, kind="i8"),
        # one user's four beams
        dict(name="beam_1x4", op="beam", seqs=1, beams=4, vocab=VOCAB, keep=4, masked=False, ended=False),
        # translations, five beams each and twice as many candidates, a grammar that rules out most of the vocabulary, some beams at their end
        dict(name="beam_16x5_masked", op="beam", seqs=16, beams=5, vocab=32001, keep=10, masked=True, ended=True),
        # a loaded server's step
        dict(name="beam_64x8", op="beam", seqs=64, beams=8, vocab=VOCAB, keep=8, masked=False, ended=True),
        # one user's four beams over the decoder's fp32 cache
        dict(name="fork_1x4", op="fork", groups=1, beams=4, short=201, long=201, prompt=37, kv_heads=12, dk=64, dv=64, page=16, block=16,
             kind="f32"),
        # a loaded server's beams
        dict(name="fork_64x8", op="fork", groups=64, beams=8, short=300, long=2900, prompt=200, kv_heads=8, dk=128, dv=128, page=64, block=16,
             kind="e4m3"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_HEADS = [(12, 12, 64, 64), (8, 8, 64, 64), (32, 8, 128, 128), (16, 4, 64, 64), (8, 1, 128, 128), (10, 5, 80, 80), (6, 6, 32, 32),
          (28, 4, 128, 128), (4, 2, 96, 64), (9, 3, 61, 45)]


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
    op = rng.choice(["append", "paged", "paged", "paged", "beam", "beam", "fork"])
    if op == "beam":
        beams = rng.choice([1, 4, rng.randint(2, 16)])
        seqs = _log_int(rng, 1, 512 // beams)
        return dict(op=op, seqs=seqs, beams=beams, vocab=rng.choice([VOCAB, _log_int(rng, 1000, 131072 if seqs * beams <= 190 else VOCAB)]),
                    keep=rng.choice([beams, min(32, 2 * beams)]), masked=rng.random() < 0.25, ended=rng.random() < 0.5)
    heads, kv_heads, dk, dv = rng.choice(_HEADS)
    block, kind = rng.choice([1, 8, 16, 32, 64, rng.randint(2, 40)]), rng.choice(["i8", "e4m3"])
    page = block * rng.choice([1, 2, 4]) if block >= 8 else block * rng.randint(3, 20)
    if op == "fork":
        long = _log_int(rng, 32, 4000)
        groups, beams = _log_int(rng, 1, 64), rng.choice([2, 4, rng.randint(2, 16)])
        return dict(op=op, groups=groups, beams=beams, short=rng.randint(1, long), long=long, prompt=rng.randint(0, long), kv_heads=kv_heads,
                    dk=dk, dv=dv, page=page, block=block, kind=rng.choice(["f32", "bf16", "i8", "e4m3"]))
    long = _log_int(rng, 64, 8000)
    seqs, short = _log_int(rng, 1, max(1, min(64, 160000 // long))), rng.randint(1, long)
    if op == "append":
        new_long = rng.choice([1, _log_int(rng, 2, long)])
        most = max(1, 30000 // new_long)
        return dict(op=op, seqs=min(seqs, most), short=short, long=long, new_short=rng.randint(1, new_long), new_long=new_long,
                    kv_heads=kv_heads, dk=dk, dv=dv, page=page, block=block, kind=kind)
    new_long = rng.choice([1, 1, rng.randint(2, 16), _log_int(rng, 16, 600)])
    most = max(1, int(2e7 / (long * new_long)))
    return dict(op=op, seqs=min(seqs, most), short=short, long=long, new_short=rng.randint(1, new_long), new_long=new_long, heads=heads,
                kv_heads=kv_heads, dk=dk, dv=dv, page=page, block=block, kind=kind)


# ---------------------------------------------------------------- sizes that follow from a case

def _spread(count, short, long):
    rng = random.Random("%d %d %d" % (count, short, long))
    return [long] + [_log_int(rng, short, long) for _ in range(count - 1)]


def _sizes(case):
    """(keys of every sequence, new tokens of every sequence); a sequence has at least as many keys as new tokens"""
    if case["op"] == "fork":   # the beams of a group are equally long
        lens = [n for n in _spread(case["groups"], case["short"], case["long"]) for _ in range(case["beams"])]
        return lens, [1] * len(lens)
    lens = _spread(case["seqs"], case["short"], case["long"])
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


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    st = dict(case)
    if case["op"] == "beam":
        _prepare_beam(st, gen, normal)
    else:
        lens, new = _sizes(case)
        starts, kv, dk, dv, kind, page = _starts(new), case["kv_heads"], case["dk"], case["dv"], case["kind"], case["page"]
        st.update(lens_list=lens, new_list=new, starts_list=starts, tokens=starts[-1], n=len(lens), lens=_ints(lens), starts=_ints(starts))
        if case["op"] == "append":
            # tokens differ in size, so that a block's scale grows now and then
            size = torch.exp(0.4 * normal(starts[-1], 1))
            st.update(k=normal(starts[-1], kv * dk) * size, v=normal(starts[-1], kv * dv) * size)
        if case["op"] == "paged":
            st.update(q=1.5 * normal(starts[-1], case["heads"] * dk), out=_out(starts[-1], case["heads"] * dv))
        _prepare_table(st, gen)
        # a page more than the cache has: there the plain form puts what belongs nowhere
        for name, d in (("k", dk), ("v", dv)):
            codes = normal(st["n_pages"] + 1, page, kv, d)
            if kind in MOST_CODE:
                codes.mul_(MOST_CODE[kind] / 3.2).clamp_(-MOST_CODE[kind], MOST_CODE[kind])
                codes = codes.round_() if kind == "i8" else codes
                scale = torch.exp(0.25 * normal(st["n_pages"] + 1, page // case["block"], kv)) * (3.2 / MOST_CODE[kind])
                st[name + "_scale"] = scale
            st[name + "_pages"] = codes.to(ELEMENT[kind])
            del codes
        if case["op"] == "fork":
            # most beams go on from a few of their group's
            beams = case["beams"]
            of = (torch.rand((case["groups"], beams), generator=gen, device="cuda") ** 2 * beams).long().clamp(max=beams - 1)
            st.update(parents=(of + torch.arange(case["groups"], device="cuda")[:, None] * beams).reshape(-1).to(torch.int32),
                      grow=torch.ones(len(lens), dtype=torch.int32, device="cuda"), new_table=torch.zeros_like(st["table"]),
                      new_lens=torch.zeros_like(st["lens"]), free_pages=_out(1, dtype=torch.int32))
    if own:
        _prepare_handles(st)
    torch.cuda.synchronize()   # the framework works on a stream of its own
    return st


def _prepare_beam(st, gen, normal):
    seqs, beams, vocab = st["seqs"], st["beams"], st["vocab"]
    rows = seqs * beams
    # a few tokens stand out in every row
    x = 2.5 * normal(rows, vocab)
    x.scatter_add_(1, torch.randint(0, vocab, (rows, 6), generator=gen, device="cuda"), 8 * torch.rand((rows, 6), generator=gen, device="cuda"))
    if st["masked"]:
        x[torch.rand((rows, vocab), generator=gen, device="cuda") > max(0.02, 200 / vocab)] = -math.inf
        x[:, 0] = 0.0   # the end of the text is always allowed
    done = torch.zeros((rows,), dtype=torch.int32, device="cuda")
    if st["ended"]:
        done = (torch.rand((rows,), generator=gen, device="cuda") < 0.15).to(torch.int32)
    scores = torch.sort(-12 - 2 * torch.rand((seqs, beams), generator=gen, device="cuda"), dim=1, descending=True).values.contiguous()
    keep = st["keep"]
    st.update(x=x, scores=scores, done=done, parents=_out(seqs, keep, dtype=torch.int32), tokens=_out(seqs, keep, dtype=torch.int32),
              new_scores=_out(seqs, keep), new_done=_out(seqs, keep, dtype=torch.int32))


def _prepare_table(st, gen):
    """Pages of every sequence; the beams of a group share the full pages of their prompt, and a fork has pages to take."""
    page, lens, fork = st["page"], st["lens_list"], st["op"] == "fork"
    counts = torch.tensor([-(-length // page) for length in lens])
    width = max(-(-(length + (1 if fork else 0)) // page) for length in lens)
    at = torch.arange(width)[None, :]
    first_of = torch.arange(len(lens))
    shared = torch.zeros(len(lens), dtype=torch.long)
    if fork:
        first_of = first_of // st["beams"] * st["beams"]
        shared = torch.minimum(torch.tensor(lens), torch.tensor(st["prompt"])) // page
    own_page = (at < counts[:, None]) & ((at >= shared[:, None]) | (first_of == torch.arange(len(lens)))[:, None])
    number = torch.cumsum(own_page.reshape(-1), 0).view(len(lens), width) - 1
    number = torch.where(at < shared[:, None], number[first_of], number)
    total = int(own_page.sum()) + (2 * len(lens) if fork else 0) + 3
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    there = (at < counts[:, None]).cuda()
    table = torch.where(there, order[number.clamp(min=0).cuda()], torch.full_like(order[:1], -1))
    st.update(table=table.contiguous(), n_pages=total, width=width)


# ---------------------------------------------------------------- the framework's calls

def _fdx():
    return importlib.import_module("frugally-deep_amd")


def _p(t):
    return ctypes.c_void_p(t.data_ptr())


def _prepare_handles(st):
    fdx = _fdx()
    if st["op"] == "beam":
        st["scratch"] = _out(fdx.lib.fdx_beam_select_scratch_bytes(st["seqs"], st["beams"], st["vocab"], st["keep"]) // 4 + 4)
        return
    eight = st["kind"] in MOST_CODE
    args = [_Buf(st["k_pages"]), _Buf(st["v_pages"]), st["kind"], st["n_pages"], st["page"], st["kv_heads"], st["dk"], st["dv"],
            _Buf(st["table"]), st["width"], _Buf(st["lens"]), st["n"], max(st["lens_list"]) + (1 if st["op"] == "fork" else 0)]
    if eight:
        cache = fdx.KvPages8(*args, _Buf(st["k_scale"]), _Buf(st["v_scale"]), st["block"])
    else:
        cache = fdx.KvPages(*args)
    st["cache"] = cache
    if st["op"] == "paged":
        need = fdx.lib.fdx_mha_paged8_scratch_bytes(st["tokens"], max(st["new_list"]), st["heads"], ctypes.byref(cache))
        st["scratch"] = _out(need // 4 + 4)
    elif st["op"] == "fork":
        need = (fdx.lib.fdx_kv8_fork_scratch_bytes if eight else fdx.lib.fdx_kv_fork_scratch_bytes)(ctypes.byref(cache))
        st["scratch"] = _out(need // 4 + 4)


def _run_own(st):
    fdx, i64 = _fdx(), ctypes.c_int64
    if st["op"] == "beam":
        fdx.check(fdx.lib.fdx_beam_select_f32(
            _p(st["x"]), i64(st["vocab"]), st["seqs"], st["beams"], st["vocab"], _p(st["scores"]), _p(st["done"]), 0, st["keep"],
            _p(st["parents"]), _p(st["tokens"]), _p(st["new_scores"]), _p(st["new_done"]), _p(st["scratch"]), None))
        return {key: st[key] for key in ("parents", "tokens", "new_scores", "new_done")}
    kv, dk, dv, cache = st["kv_heads"], st["dk"], st["dv"], ctypes.byref(st["cache"])
    if st["op"] == "append":
        fdx.check(fdx.lib.fdx_kv8_append_f32(_p(st["k"]), i64(kv * dk), _p(st["v"]), i64(kv * dv), _p(st["starts"]), st["tokens"], cache, None))
        return _pages(st)
    if st["op"] == "fork":
        call = fdx.lib.fdx_kv8_fork if st["kind"] in MOST_CODE else fdx.lib.fdx_kv_fork
        fdx.check(call(cache, _p(st["parents"]), _p(st["grow"]), _p(st["new_table"]), _p(st["new_lens"]), _p(st["free_pages"]),
                       _p(st["scratch"]), None))
        return dict(_pages(st), table=st["new_table"], lens=st["new_lens"], free_pages=st["free_pages"])
    heads = st["heads"]
    fdx.check(fdx.lib.fdx_mha_paged8_f32(_p(st["q"]), i64(heads * dk), _p(st["starts"]), st["tokens"], max(st["new_list"]), heads, cache,
                                         _p(st["out"]), i64(heads * dv), _p(st["scratch"]), None))
    return st["out"]


def _pages(st):
    """The cache as it is then: its codes (those of i8 as whole numbers) and their scales"""
    return {key: st[key][:st["n_pages"]] for key in ("k_pages", "v_pages", "k_scale", "v_scale") if key in st}


# ---------------------------------------------------------------- the plain forms

def _rows(codes, at):
    """rows of the cache, its pages one behind the other, as fp32 values of their codes"""
    flat = codes.view(-1, *codes.shape[2:])
    if codes.dtype == torch.float8_e4m3fn:
        return flat.view(torch.uint8)[at].view(codes.dtype).float()
    return flat[at].float()


def _put(codes, at, values):
    """values (fp32, whole numbers for i8) rounded to the codes' type, at rows of the cache"""
    flat, values = codes.view(-1, *codes.shape[2:]), values.to(codes.dtype)
    if codes.dtype == torch.float8_e4m3fn:
        flat, values = flat.view(torch.uint8), values.view(torch.uint8)
    flat[at] = values


def _to_code(x, kind):
    most = MOST_CODE[kind]
    return x.round().clamp(-most, most) if kind == "i8" else x.clamp(-most, most)


def _tokens_of(st):
    """of every new token: its sequence, its number in it, its position"""
    t = torch.arange(st["tokens"], device="cuda")
    starts = st["starts"].long()
    seq = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    j = t - starts[seq]
    return seq, j, st["lens"].long()[seq] - (starts[seq + 1] - starts[seq]) + j


def _plain_append(st):
    page, block, kind, kv = st["page"], st["block"], st["kind"], st["kv_heads"]
    seq, _, pos = _tokens_of(st)
    starts = st["starts"].long()
    table = st["table"].long()
    slot = table[seq, pos // page] * page + pos % page
    blk = slot // block
    first = st["lens"].long() - (starts[1:] - starts[:-1])          # position of each sequence's first new token
    first_slot = table[torch.arange(st["n"], device="cuda"), first // page] * page + first % page
    first_blk, old = first_slot // block, first % block             # tokens in front of it in its block
    inside = torch.arange(block, device="cuda")[None, :]
    old_rows = (first_blk * block)[:, None] + inside
    trash = st["n_pages"] * page
    old_rows = torch.where(inside < old[:, None], old_rows, torch.full_like(old_rows, trash))
    for name, d in (("k", st["dk"]), ("v", st["dv"])):
        x = st[name].view(-1, kv, d)
        scale = st[name + "_scale"].view(-1, kv)
        was = scale[first_blk]
        kept = torch.zeros_like(scale).scatter_reduce_(0, first_blk[:, None].expand(-1, kv), torch.where(old[:, None] > 0, was, 0.0), "amax")
        most = torch.zeros_like(scale).scatter_reduce_(0, blk[:, None].expand(-1, kv), x.abs().amax(2), "amax")
        # divided by a tensor: by a plain number it would be a product with the rounded reciprocal
        grown = torch.maximum((most / torch.full_like(most[:1], MOST_CODE[kind])).clamp(min=TINY), kept)
        scale[blk] = grown[blk]
        ratio = (was / grown[first_blk])[:, None, :, None]
        codes = st[name + "_pages"]
        _put(codes, old_rows, _to_code(_rows(codes, old_rows) * ratio, kind))
        _put(codes, slot, _to_code(x * (1.0 / grown[blk])[:, :, None], kind))
    return _pages(st)


def _plain_paged(st):
    page, block, kv, dk, dv, heads = st["page"], st["block"], st["kv_heads"], st["dk"], st["dv"], st["heads"]
    group, lens, new, starts = heads // kv, st["lens_list"], st["new_list"], st["starts_list"]
    seq, number, _ = _tokens_of(st)
    out = torch.empty((st["tokens"], heads, dv), device="cuda")
    # padded to the longest; sequences at a time by the memory of their scores (all of them in a decode step)
    step = max(1, 300_000_000 // (heads * max(new) * max(lens)))
    for a in range(0, st["n"], step):
        b = min(st["n"], a + step)
        m, keys, rows = b - a, max(lens[a:b]), max(new[a:b])
        at = torch.arange(keys, device="cuda")
        slots = (st["table"][a:b].long()[:, at // page] * page + at % page).clamp(min=0)
        k, v = (_rows(st[n + "_pages"], slots) * st[n + "_scale"].view(-1, kv)[slots // block][..., None] for n in ("k", "v"))
        token = (st["starts"][a:b].long()[:, None] + torch.arange(rows, device="cuda")).clamp(max=st["tokens"] - 1)
        q = st["q"].view(-1, kv, group, dk)[token].permute(0, 2, 3, 1, 4).reshape(m * kv, group * rows, dk)
        s = torch.matmul(q, k.permute(0, 2, 3, 1).reshape(m * kv, dk, keys)).view(m, kv, group, rows, keys) * (1.0 / math.sqrt(dk))
        length, count = st["lens"][a:b].long(), (st["starts"][a + 1:b + 1] - st["starts"][a:b]).long()
        sees = (length - count)[:, None] + torch.arange(1, rows + 1, device="cuda")
        s.masked_fill_(at >= sees[:, None, None, :, None], -math.inf)
        s = torch.exp(s - s.amax(-1, keepdim=True))
        s = s / s.sum(-1, keepdim=True)
        o = torch.matmul(s.view(m * kv, group * rows, keys), v.permute(0, 2, 1, 3).reshape(m * kv, keys, dv))
        o = o.view(m, heads, rows, dv)
        out[starts[a]:starts[b]] = o[seq[starts[a]:starts[b]] - a, :, number[starts[a]:starts[b]]]
    return out.view(st["tokens"], heads * dv)


def _plain_beam(st):
    seqs, beams, keep = st["seqs"], st["beams"], st["keep"]
    x = st["x"]
    # a row's best by logit, equal ones by id: as whole numbers that are all different
    bits = (x + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long() * 2 ** 32 + (2 ** 32 - 1 - torch.arange(st["vocab"], device="cuda"))
    ids = 2 ** 32 - 1 - torch.bitwise_and(torch.topk(order, min(keep, st["vocab"]), dim=1).values, 2 ** 32 - 1)
    wide = x.double()   # totals decide, also where they are near each other
    most = wide.amax(1, keepdim=True)
    log_sum = most + torch.log(torch.exp(wide - most).sum(1, keepdim=True))
    before, done = st["scores"].view(-1, 1).double(), st["done"].view(-1, 1) != 0
    total = before + (torch.gather(wide, 1, ids) - log_sum)
    first = torch.arange(ids.shape[1], device="cuda") == 0
    total = torch.where(done, torch.where(first, before, -math.inf), total).view(seqs, -1)
    ids = torch.where(done, torch.zeros_like(ids), ids).view(seqs, -1)
    total, best = torch.sort(total, dim=1, descending=True, stable=True)
    total, best = total[:, :keep], best[:, :keep]
    there = total > -math.inf
    parents = best // min(keep, st["vocab"]) + torch.arange(seqs, device="cuda")[:, None] * beams
    tokens = torch.gather(ids, 1, best)
    ended = (tokens == 0) | (st["done"][parents] != 0)
    return dict(parents=torch.where(there, parents, -1).to(torch.int32), tokens=torch.where(there, tokens, -1).to(torch.int32),
                new_scores=total.float(), new_done=(there & ended).to(torch.int32))


def _plain_fork(st):
    page, block, n_pages, n = st["page"], st["block"], st["n_pages"], st["n"]
    parents, me = st["parents"].long(), torch.arange(n, device="cuda")
    length = torch.where(parents >= 0, st["lens"].long()[parents.clamp(min=0)], 0)
    want = torch.where(parents >= 0, length + st["grow"].long(), 0)
    rows = st["table"].long()[parents.clamp(min=0)]
    at = torch.arange(st["width"], device="cuda")[None, :]
    full, part = length // page, length % page
    table = torch.where(at < full[:, None], rows, -1)
    used = torch.zeros(n_pages + 1, dtype=torch.bool, device="cuda")
    used[torch.where(table >= 0, table, n_pages)] = True
    # the partly filled page: the first that has it keeps it, unless it is a full page of another
    last = torch.where(part > 0, torch.gather(rows, 1, full.clamp(max=st["width"] - 1)[:, None])[:, 0], n_pages)
    first = torch.full((n_pages + 1,), n, device="cuda").scatter_reduce_(0, last, me, "amin")
    keeps = (part > 0) & (first[last] == me) & ~used[last]
    used[torch.where(keeps, last, n_pages)] = True
    copies = (part > 0) & ~keeps
    begin = full + keeps                                   # entries from here on are new pages
    end = (want + page - 1) // page
    count = end - begin
    free = torch.sort(used[:n_pages].to(torch.int8), stable=True).indices
    offset = torch.cumsum(count, 0) - count
    taken = free[(offset[:, None] + at - begin[:, None]).clamp(0, n_pages - 1)]
    table = torch.where((at == full[:, None]) & keeps[:, None], last[:, None], table)
    table = torch.where((at >= begin[:, None]) & (at < end[:, None]), taken, table)
    target = torch.where(copies, torch.gather(table, 1, full.clamp(max=st["width"] - 1)[:, None])[:, 0], n_pages)
    # what belongs nowhere goes to the page behind the cache's last
    inside = torch.arange(page, device="cuda")
    held = copies[:, None] & (inside < part[:, None])
    source_rows, target_rows = (torch.where(held, p[:, None], n_pages) * page + inside for p in (last, target))
    for name in ("k_pages", "v_pages"):
        flat = st[name].view(-1, *st[name].shape[2:])
        flat = flat.view(torch.uint8) if flat.dtype == torch.float8_e4m3fn else flat
        flat[target_rows] = flat[source_rows]
    if st["kind"] in MOST_CODE:
        held = held[:, ::block]
        for name in ("k_scale", "v_scale"):
            flat = st[name].view(-1, st["kv_heads"])
            blocks = [torch.where(held, p[:, None], n_pages) * (page // block) + inside[:page // block] for p in (last, target)]
            flat[blocks[1]] = flat[blocks[0]]
    left = n_pages - used[:n_pages].sum() - count.sum()
    return dict(_pages(st), table=table.to(torch.int32), lens=want.to(torch.int32), free_pages=left.view(1).to(torch.int32))


_PLAIN = {"append": _plain_append, "paged": _plain_paged, "beam": _plain_beam, "fork": _plain_fork}


def run(state):
    return _run_own(state) if own else _PLAIN[state["op"]](state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["op"] == "beam":
        rows, vocab = case["seqs"] * case["beams"], case["vocab"]
        # per logit: difference, exponential, sum, maximum
        return {"bytes": 4 * rows * (vocab + 2) + 16 * case["seqs"] * case["keep"], "flops": 4 * rows * vocab}
    lens, new = _sizes(case)
    kv, dk, dv, page, held = case["kv_heads"], case["dk"], case["dv"], case["page"], BYTES[case["kind"]]
    row = kv * (dk + dv) * held
    if case["op"] == "fork":
        # all but about half of the sequences copy the rows of their last page
        pages = sum(-(-(n + 1) // page) for n in lens)
        return {"bytes": 8 * pages + 16 * len(lens) + sum(n % page for n in lens) * row, "flops": 0}
    tokens = sum(new)
    if case["op"] == "append":
        blocks = sum(-(-n // case["block"]) for n in new)
        return {"bytes": tokens * (kv * (dk + dv) * 4 + row) + 8 * kv * blocks, "flops": 4 * tokens * kv * (dk + dv)}
    heads = case["heads"]
    # query i of n new ones sees length - n + i + 1 keys
    pairs = sum(n * (length - n) + n * (n + 1) // 2 for n, length in zip(new, lens))
    nbytes = 4 * tokens * heads * (dk + dv) + sum(lens) * row + sum(-(-n // case["block"]) * 8 * kv + -(-n // page) * 4 for n in lens)
    return {"bytes": nbytes, "flops": 2 * heads * pairs * (dk + dv)}


# ---------------------------------------------------------------- from the definitions, in 64 bits

def exact(case, seed):
    global own
    if case["op"] == "fork":
        return None   # nothing is computed
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    f64 = torch.float64
    if case["op"] == "beam":
        return dict(parents=None, tokens=None, new_done=None, new_scores=_exact_beam(st))
    lens, new, starts = st["lens_list"], st["new_list"], st["starts_list"]
    kv, dk, dv, page, block = case["kv_heads"], case["dk"], case["dv"], case["page"], case["block"]
    if case["op"] == "append":
        out, most = dict(k_pages=None, v_pages=None), MOST_CODE[case["kind"]]
        pages = st["table"].cpu().tolist()
        for name, d in (("k", dk), ("v", dv)):
            size = st[name].to(f64).abs().view(-1, kv, d).amax(2).cpu()
            scale = st[name + "_scale"][:st["n_pages"]].to(f64).cpu()
            for s, (length, n) in enumerate(zip(lens, new)):
                pos = length - n
                while pos < length:   # a block at a time
                    end = min(length, pos - pos % block + block)
                    t = starts[s] + pos - (length - n)
                    a = (size[t:t + end - pos].amax(0) / most).clamp(min=TINY)
                    at = scale[pages[s][pos // page], pos % page // block]
                    at.copy_(torch.maximum(a, at) if pos % block else a)
                    pos = end
            out[name + "_scale"] = scale
        return out
    heads, group = case["heads"], case["heads"] // kv
    out = torch.zeros((starts[-1], heads, dv), dtype=f64, device="cuda")
    for s in range(case["seqs"]):
        a, n, length = starts[s], new[s], lens[s]
        held = st["table"][s, :-(-length // page)].long()
        both = []
        for name, d in (("k", dk), ("v", dv)):
            codes = st[name + "_pages"].view(torch.uint8)[held].view(st[name + "_pages"].dtype).to(f64)
            values = codes.view(len(held), page // block, block, kv, d) * st[name + "_scale"][held].to(f64)[:, :, None, :, None]
            both.append(values.reshape(-1, kv, d)[:length])
        for h in range(heads):
            kh, vh = both[0][:, h // group], both[1][:, h // group]
            for i in range(0, n, 2048):
                m = min(2048, n - i)
                x = st["q"][a + i:a + i + m, h * dk:(h + 1) * dk].to(f64) @ kh.t() / math.sqrt(dk)
                x = x.masked_fill(torch.ones_like(x, dtype=torch.bool).triu(length - n + i + 1), -math.inf)
                out[a + i:a + i + m, h] = torch.softmax(x, -1) @ vh
    return out.view(starts[-1], heads * dv)


def _exact_beam(st):
    out = []
    for s in range(st["seqs"]):
        every = []
        for b in range(st["beams"]):
            r = s * st["beams"] + b
            before = st["scores"][s, b].double()
            if st["done"][r]:
                every.append(before[None])
                continue
            x = st["x"][r].double()
            x = x[x > -math.inf]
            every.append(before + torch.topk(x, min(st["keep"], len(x))).values - torch.logsumexp(x, 0))
        every = torch.sort(torch.cat(every), descending=True).values[:st["keep"]]
        out.append(torch.cat([every, torch.full((st["keep"] - len(every),), -math.inf, dtype=torch.float64, device="cuda")]))
    return torch.stack(out)
