"""Cases of the operators for shared prefixes and eviction: what one pass of each computes, plain and through the package.

Operators (the pool is ``[num_pages, 2, Hkv, page_size, D]``, the page table ``(indptr, indices, last_page_len)``):

* ``prefix``  attention of each sequence's newest tokens where groups of sequences share their first pages;
* ``weights`` the softmax weights that each key of a paged cache gets, summed over the new queries and a kv head's
  query heads and added to what it got before;
* ``keep``    which tokens of each head stay: the first ones, the newest ones and the heaviest of the rest;
* ``evict``   the kept tokens moved to the front of their sequences, page table and sums with them.

Lengths are a function of the case alone (``work`` counts them); the seed draws the values, the order of the
sequences and the physical order of the pages.
"""
import itertools
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # -- prefix: groups of sequences share pre tokens, each has its own after them, the newest `new` are asked
        # four samples of one prompt decode a token each: the latency of the smallest step
        dict(name="prefix decode, four samples", op="prefix", dtype="fp16", Hq=32, Hkv=8, D=128, P=16, B=4, groups=1,
             pre_lo=2048, pre_hi=2048, own_lo=17, own_hi=128, new=1, causal=True),
        # 64 conversations behind one system prompt decode a token each
        dict(name="prefix decode, batch of 64", op="prefix", dtype="fp16", Hq=32, Hkv=8, D=128, P=16, B=64, groups=1,
             pre_lo=8192, pre_hi=8192, own_lo=64, own_hi=1024, new=1, causal=True),
        # eight prompts with eight samples each verify five drafted tokens
        dict(name="prefix verify, eight groups", op="prefix", dtype="bf16", Hq=32, Hkv=8, D=128, P=64, B=64, groups=8,
             pre_lo=1024, pre_hi=16384, own_lo=100, own_hi=2000, new=5, causal=True),
        # new prompts behind three long documents, the 64-wide heads and the page size that no tile is a multiple of
        dict(name="prefix of prompts", op="prefix", dtype="bf16", Hq=64, Hkv=16, D=64, P=20, B=13, groups=3,
             pre_lo=6000, pre_hi=12000, own_lo=211, own_hi=513, new=512, causal=True),
        # -- weights: of n newest tokens on each sequence's whole cache
        # one conversation decodes one token
        dict(name="weights of one token", op="weights", dtype="fp16", Hq=32, Hkv=8, D=128, P=16, B=1, lo=2048,
             hi=2048, new=1, chunks=1, causal=True),
        # one decoded token in each of 64 sequences (the paged decode's benchmark batch)
        dict(name="weights while decoding", op="weights", dtype="fp16", Hq=32, Hkv=8, D=128, P=16, B=64, lo=512,
             hi=32768, new=1, chunks=64, causal=True),
        # a step of continuous batching: prompts beside sequences that decode
        dict(name="weights, mixed batch", op="weights", dtype="bf16", Hq=64, Hkv=16, D=64, P=20, B=16, lo=94,
             hi=4096, new=1024, chunks=8, causal=True),
        # the last chunk of a long prompt: 8192 tokens on top of 24576 (the largest case)
        dict(name="weights of a long prompt", op="weights", dtype="fp16", Hq=32, Hkv=8, D=128, P=16, B=1, lo=32768,
             hi=32768, new=8192, chunks=1, causal=True),
        # -- keep: the lists
        # 64 sequences of 512 to 32768 tokens cut back to 1024
        dict(name="keep in a batch of 64", op="keep", Hkv=8, B=64, layers=1, lo=512, hi=32768, budget=1024, sinks=4,
             recent=256),
        # one long conversation cut back to a quarter
        dict(name="keep in one sequence", op="keep", Hkv=8, B=1, layers=1, lo=131072, hi=131072, budget=32768,
             sinks=4, recent=1000),
        # -- evict: the pool
        # half of the cache of 48 conversations, in groups of three behind a shared prompt, goes
        dict(name="evict in a batch of 48", op="evict", dtype="fp16", Hkv=8, D=128, P=16, layers=1, B=48, share=3,
             lo=700, hi=4096, budget=1500, sinks=64, recent=256),
        # one conversation through a small model's four layers
        dict(name="evict in one sequence", op="evict", dtype="bf16", Hkv=8, D=64, P=20, layers=4, B=1, share=1,
             lo=8191, hi=8191, budget=2047, sinks=4, recent=300),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("prefix", "prefix", "weights", "weights", "keep", "evict"))
    dtype = rng.choice(("fp16", "bf16"))
    D = rng.choice((64, 128, 128))
    Hkv = rng.choice((1, 2, 4, 8, 8, 16))
    G = rng.choice((1, 2, 3, 4, 4, 5, 8))
    P = rng.choice((1, 5, 8, 16, 16, 16, 20, 32, 64, 128))
    heads = dict(op=op, dtype=dtype, Hq=Hkv * G, Hkv=Hkv, D=D, P=P)
    if op == "prefix":
        pre, mine = _log(rng, 16, 16384), _log(rng, 1, 2048)
        new, B = min(_log(rng, 1, 512), mine), _log(rng, 2, 96)
        # a plain form that fits the card
        while B > 2 and (B * Hkv * G * new * (pre + mine) > 2e9 or B * (pre + mine) * Hkv * D > 1.1e9):
            B = max(2, B // 2)
        while new > 1 and B * Hkv * G * new * (pre + mine) > 2e9:
            new //= 2
        return dict(heads, B=B, groups=rng.choice((1, 1, max(1, B // 8), max(1, B // 3))),
                    pre_lo=max(1, pre // rng.choice((1, 2, 5))), pre_hi=pre, own_lo=max(1, mine // rng.choice((1, 3))),
                    own_hi=mine, new=new, causal=rng.random() < 0.8)
    if op == "weights":
        hi = _log(rng, 1, 32768)
        lo = max(1, int(hi * rng.uniform(0.05, 1.0)))
        new, B = min(_log(rng, 1, 8192), hi), _log(rng, 1, 64)
        # at most half of the largest case's products, and a plain form that fits the card
        while B > 1 and (B * Hkv * G * new * hi > 4e9 or B * hi * Hkv * D > 1.1e9):
            B = max(1, B // 2)
        if Hkv * G * new * hi > 4e9:
            new = max(1, int(4e9 / (Hkv * G * hi)))
        return dict(heads, B=B, lo=lo, hi=hi, new=new, chunks=rng.choice((B, B, max(1, B // 4))),
                    causal=rng.random() < 0.8)
    hi = _log(rng, 8, 65536 if op == "keep" else 8192)
    B = _log(rng, 1, 64)
    layers = rng.choice((1, 1, 2, 4))
    width = 1 if op == "keep" else D
    while B > 1 and layers * B * hi * Hkv * width > (2.5e7 if op == "keep" else 2.5e8):
        B = max(1, B // 2)
    budget = max(1, int(hi * rng.uniform(0.03, 0.9)))
    sinks = rng.choice((0, 1, 4, 64))
    recent = int(budget * rng.choice((0, 0.1, 0.3)))
    if sinks + recent > budget:
        sinks = 0
    case = dict(op=op, Hkv=Hkv, B=B, layers=layers, lo=max(1, hi // rng.choice((1, 3, 10))), hi=hi, budget=budget,
                sinks=sinks, recent=recent)
    return case if op == "keep" else dict(case, dtype=dtype, D=D, P=P, share=rng.choice((1, 1, 2, 4)))


def _spread(lo, hi, n):
    """n whole numbers evenly spread over lo..hi (both ends held)."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _lens(case):
    return _spread(case["lo"], case["hi"], case["B"])


def _news(case):
    """New tokens of each sequence: a full or a somewhat shorter chunk for `chunks` of them, one token for the rest."""
    step, most, cut = max(1, case["B"] // case["chunks"]), case["chunks"], case["new"] // 16
    return [min(n, case["new"] - (i // step % 4) * cut) if i % step == 0 and i // step < most else 1
            for i, n in enumerate(_lens(case))]


def _pages(n, P):
    return -(-n // P)


def _families(case):
    """Of a `prefix` case: the groups' bounds in the batch, their shared pages, each sequence's own and new tokens."""
    B, g = case["B"], case["groups"]
    bounds = [B * i // g for i in range(g + 1)]
    shared = [n // case["P"] for n in _spread(case["pre_lo"], case["pre_hi"], g)]
    mine = _spread(case["own_lo"], case["own_hi"], B)
    return bounds, shared, mine, [min(n, case["new"] - i % 4 * (case["new"] // 16)) for i, n in enumerate(mine)]


def _kept(case, n):
    return min(n, case["budget"])


def work(case):
    op, es, Hkv = case["op"], 2, case["Hkv"]
    if op == "prefix":
        D, P = case["D"], case["P"]
        bounds, shared, mine, news = _families(case)
        group = [i for i in range(case["groups"]) for _ in range(bounds[i], bounds[i + 1])]
        lens = [shared[g] * P + n for g, n in zip(group, mine)]
        pairs = sum(n * (L - n) + (n * (n + 1) // 2 if case["causal"] else n * n) for n, L in zip(news, lens))
        keys = sum(shared) * P + sum(mine)
        rows = sum(news) * case["Hq"]
        return {"bytes": 2 * keys * Hkv * D * es + rows * (2 * D * es + 4) + 4 * sum(_pages(n, P) for n in lens),
                "flops": 4 * case["Hq"] * D * pairs}
    lens = _lens(case)
    if op == "weights":
        news = _news(case)
        pairs = sum(n * (L - n) + (n * (n + 1) // 2 if case["causal"] else n * n) for n, L in zip(news, lens))
        rows = sum(news) * case["Hq"]
        return {"bytes": sum(lens) * Hkv * (case["D"] * es + 8) + rows * (case["D"] * es + 4) +
                4 * sum(_pages(n, case["P"]) for n in lens), "flops": 2 * case["Hq"] * case["D"] * pairs}
    heads = case["layers"] * Hkv
    kept = sum(_kept(case, n) for n in lens)
    if op == "keep":
        return {"bytes": 4 * heads * (sum(lens) + kept), "flops": 0}
    # the rows behind the first tokens move, and all sums and the places they leave
    moved = sum(max(0, case["budget"] - case["sinks"]) for n in lens if n > case["budget"])
    return {"bytes": heads * (2 * moved * 2 * case["D"] * es + 4 * (kept + sum(lens) + kept)) +
            2 * 4 * sum(_pages(_kept(case, n), case["P"]) for n in lens), "flops": 0}


# ---------------------------------------------------------------------------
# what a program has in hand before the call
# ---------------------------------------------------------------------------

def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _indptr(counts):
    return _ints([0, *itertools.accumulate(counts)])


def _normal(shape, case, gen):
    return torch.randn(shape, generator=gen, device=DEV, dtype=TYPES[case["dtype"]])


def _table(case, rows, gen, extra=0):
    """CSR page table of sequences given as (length, shared pages, group): pages in random places of a pool with
    `extra` more, a group's first pages the same ones."""
    P, count, first, entries, pages, last = case["P"], 0, {}, [], [], []
    for n, shared, g in rows:
        if g not in first:
            first[g] = list(range(count, count + shared))
            count += shared
        k = _pages(n, P)
        entries += first[g] + list(range(count, count + k - shared))
        count += k - shared
        pages.append(k)
        last.append(n - P * (k - 1) if k else 0)
    place = torch.randperm(count + extra, generator=gen, device=DEV).to(torch.int32)
    return _indptr(pages), place[torch.tensor(entries, dtype=torch.long, device=DEV)], _ints(last), count + extra


def _sums(shape, lens, gen):
    """Accumulated weights as a cache has them: a long tail, many equal ones among the smallest."""
    w = torch.randn(shape, generator=gen, device=DEV).mul_(2.0).exp_()
    w = torch.where(w < 0.1, 0.0, w)
    return torch.where(torch.arange(shape[-1], device=DEV) < lens[:, None, None], w, 0.0)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    rng = random.Random(seed)
    s, op = dict(case), case["op"]
    Hkv = case["Hkv"]
    if op == "prefix":
        bounds, shared, mine, news = _families(case)
        order = list(range(case["groups"]))
        rng.shuffle(order)
        rows, new, sizes = [], [], []
        for g in order:
            members = list(range(bounds[g], bounds[g + 1]))
            rng.shuffle(members)
            rows += [(shared[g] * case["P"] + mine[b], shared[g], g) for b in members]
            new += [news[b] for b in members]
            sizes.append(len(members))
        s["indptr"], s["indices"], s["last"], N = _table(case, rows, gen)
        s["new_indptr"] = _indptr(new)
        s["group_indptr"], s["shared_pages"] = _indptr(sizes), _ints([shared[g] for g in order])
        s["max_len"], s["max_new"] = max(n for n, _, _ in rows), max(new)
        s["q"] = _normal((sum(new), case["Hq"], case["D"]), case, gen)
        s["cache"] = _normal((N, 2, Hkv, case["P"], case["D"]), case, gen)
        return s
    # families of `share` sequences stay together
    lens, share = _lens(case), case.get("share", 1)
    order = [list(range(i, min(i + share, case["B"]))) for i in range(0, case["B"], share)]
    rng.shuffle(order)
    order = [i for family in order for i in family]
    lens = [lens[i] for i in order]
    s["max_len"], s["lens"] = max(lens), _ints(lens)
    if op == "weights":
        news = _news(case)
        news = [news[i] for i in order]
        s["indptr"], s["indices"], s["last"], N = _table(case, [(n, 0, i) for i, n in enumerate(lens)], gen)
        s["new_indptr"], s["max_new"] = _indptr(news), max(news)
        s["q"] = _normal((sum(news), case["Hq"], case["D"]), case, gen)
        s["cache"] = _normal((N, 2, Hkv, case["P"], case["D"]), case, gen)
        # the attention before gave each row's log-sum-exp
        b, i, x = _scores(s)
        s["lse"] = x.logsumexp(-1).permute(0, 2, 1, 3)[b, i].flatten(1, 2).contiguous()
        del x
        s["sums"] = _sums((case["B"], Hkv, max(lens)), s["lens"], gen)
        s["out"] = torch.zeros_like(s["sums"])
        return s
    shape = (case["layers"], case["B"], Hkv, max(lens))
    s["sums"] = _sums(shape, s["lens"], gen)
    if op == "keep":
        return s
    # a family shares half of its shortest member's pages
    P, least = case["P"], {}
    for i, n in zip(order, lens):
        least[i // share] = min(n, least.get(i // share, n))
    rows = [(n, least[i // share] // 2 // P if share > 1 else 0, i // share) for i, n in zip(order, lens)]
    most = _pages(min(case["budget"], max(lens)), P)
    s["indptr"], s["indices"], s["last"], N = _table(case, rows, gen, extra=case["B"] * most if share > 1 else 3)
    s["cache"] = _normal((case["layers"], N, 2, Hkv, P, case["D"]), case, gen)
    s["keep"], s["kept"] = _keep(dict(s, sums=torch.rand(shape, generator=gen, device=DEV)))
    if case["layers"] == 1:
        for name in ("sums", "cache", "keep"):
            s[name] = s[name][0]
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _scores(s):
    """Sequence and number in its chunk of each new token, and all scaled scores [B, Hkv, n, G, L] in fp32, -inf where
    a query does not see the key."""
    Hkv, D, P, B = s["Hkv"], s["D"], s["P"], s["B"]
    G, at = s["Hq"] // Hkv, s["new_indptr"].long()
    t = torch.arange(s["q"].shape[0], device=DEV)
    b = torch.searchsorted(at, t, right=True) - 1
    i = t - at[b]
    length = ((s["indptr"][1:] - s["indptr"][:-1]).long() - 1) * P + s["last"].long()
    n, L = s["max_new"], s["max_len"]
    k = _rows(s, 0)
    q = torch.zeros((B, n, Hkv, G, D), device=DEV)
    q[b, i] = s["q"].float().unflatten(1, (Hkv, G))
    pos = torch.full((B, n), -1, dtype=torch.long, device=DEV)
    pos[b, i] = length[b] - (at[b + 1] - at[b]) + i
    x = torch.matmul(q.permute(0, 2, 1, 3, 4).reshape(B, Hkv, n * G, D), k.transpose(2, 3))
    x = x.mul_(1 / math.sqrt(D)).view(B, Hkv, n, G, L)
    j = torch.arange(L, device=DEV)
    hidden = (j >= length[:, None])[:, None] | (pos < 0)[..., None]
    if s["causal"]:
        hidden = hidden | (j > pos[..., None])
    return b, i, x.masked_fill_(hidden[:, None, :, None], -math.inf)


def _rows(s, which):
    """Keys (0) or values (1) of each sequence side by side, padded to the longest with zeros, [B, Hkv, L, D] in fp32."""
    P, L = s["P"], s["max_len"]
    j = torch.arange(L, device=DEV)
    length = ((s["indptr"][1:] - s["indptr"][:-1]).long() - 1) * P + s["last"].long()
    entry = (s["indptr"][:-1].long()[:, None] + torch.arange(_pages(L, P), device=DEV)).clamp(max=s["indices"].numel() - 1)
    x = s["cache"][s["indices"].long()[entry], which].permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :L]
    return torch.where((j < length[:, None])[:, None, :, None], x, 0).float()


def _prefix(s):
    b, i, x = _scores(s)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0, top)
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    out = torch.matmul(x.flatten(2, 3), _rows(s, 1)).view(*x.shape[:-1], s["D"])
    out = torch.where(total > 0, out / total, 0).permute(0, 2, 1, 3, 4)[b, i].flatten(1, 2)
    lse = (total.log() + top)[..., 0].permute(0, 2, 1, 3)[b, i].flatten(1, 2)
    return out.to(s["q"].dtype), lse


def _weights(s):
    b, i, x = _scores(s)
    lse = torch.zeros((s["B"], s["max_new"], s["Hq"]), device=DEV)
    lse[b, i] = s["lse"]
    x = x.sub_(lse.unflatten(2, (s["Hkv"], -1)).permute(0, 2, 1, 3)[..., None]).exp_()
    there = torch.arange(s["max_len"], device=DEV) < s["lens"][:, None, None]
    return torch.where(there, s["sums"] + x.sum((2, 3)), s["out"])


def _keep(s):
    w, n = s["sums"], s["lens"][:, None, None]
    j = torch.arange(w.shape[-1], device=DEV)
    always = (j < s["sinks"]) | (j >= n - s["recent"])
    w = torch.where(j >= n, -2.0, torch.where(always, math.inf, w))  # (no sum is negative)
    best = w.sort(dim=-1, descending=True, stable=True).indices[..., :s["budget"]]
    kept = s["lens"].clamp(max=s["budget"])
    i = torch.arange(best.shape[-1], device=DEV)
    best = torch.where(i < kept[:, None, None], best, w.shape[-1]).sort(-1).values
    best = torch.where(i < kept[:, None, None], best, 0)
    best = torch.cat((best, best.new_zeros((*best.shape[:-1], s["budget"] - best.shape[-1]))), -1)
    return best.int(), kept.int()


def _evict(s):
    P, kept, Hkv = s["P"], s["kept"].long(), s["Hkv"]
    one = s["layers"] == 1
    pool, keep, sums = (t[None] if one else t for t in (s["cache"], s["keep"], s["sums"]))
    M, B, E = keep.shape[-1], kept.numel(), _pages(keep.shape[-1], P)
    start, named = s["indptr"][:-1].long()[:, None], s["indices"].long()
    pages = (kept + P - 1) // P
    e = torch.arange(E, device=DEV)
    mine = e < pages[:, None]
    page = named[(start + e).clamp(max=named.numel() - 1)]
    # a page that others have too is not written: it stays where nothing of it moves and nothing will be appended
    end = torch.minimum((e + 1) * P, kept[:, None]).clamp(min=1) - 1
    moves = (keep.long().gather(-1, end[None, :, None].expand(keep.shape[0], B, Hkv, E)) != end[:, None]).any(2).any(0)
    others = torch.bincount(named, minlength=pool.shape[1])
    fresh = mine & (others[page] > 1) & (moves | (end + 1 < (e + 1) * P))
    dead = torch.argsort((others > 0).to(torch.uint8), stable=True)
    rank = (fresh.flatten().cumsum(0) - 1).view(B, E)
    page = torch.where(fresh, dead[rank.clamp(min=0)], page)
    # every kept row from its old place to its new one
    i = torch.arange(M, device=DEV)
    b, i = torch.nonzero(i < kept[:, None], as_tuple=True)
    l, h = torch.arange(keep.shape[0], device=DEV)[:, None, None], torch.arange(Hkv, device=DEV)[:, None]
    k = keep.long()[l, b, h, i]
    from_page = named[start[:, 0][b] + k // P]
    pool[l, page[b, i // P], :, h, i % P] = pool[l, from_page, :, h, k % P]
    moved = torch.zeros_like(sums)
    moved[l, b, h, i] = sums[l, b, h, k]
    j = torch.arange(sums.shape[-1], device=DEV)
    sums.copy_(torch.where(j < s["lens"][:, None, None], moved, sums))
    indptr = torch.cat((pages.new_zeros(1), pages.cumsum(0))).int()
    count = min(B * E, named.numel())
    place = torch.where(mine, indptr[:-1, None].long() + e, count)
    indices = torch.full((count + 1,), -1, dtype=torch.int32, device=DEV)
    indices[place] = torch.where(mine, page, -1).int()
    last = torch.where(kept > 0, kept - (pages - 1) * P, 0).int()
    return indptr, indices[:count], last, s["cache"], s["sums"]


_PLAIN = {"prefix": _prefix, "weights": _weights, "keep": _keep, "evict": _evict}


def run(state):
    s = state
    if not own:
        r = _PLAIN[s["op"]](s)
        return (r[0][0], r[1]) if s["op"] == "keep" and s["layers"] == 1 else r
    if s["op"] == "prefix":
        from attention_kernel_triton_b200.paged_prefix_attention import flash_attention_shared_prefix_paged_with_lse
        return flash_attention_shared_prefix_paged_with_lse(s["q"], s["new_indptr"], s["cache"], s["indptr"],
                                                            s["indices"], s["last"], s["group_indptr"],
                                                            s["shared_pages"], causal=s["causal"])
    from attention_kernel_triton_b200 import paged_kv_eviction as eviction
    if s["op"] == "weights":
        return eviction.accumulate_attention_weights_paged(s["sums"], s["q"], s["new_indptr"], s["cache"], s["indptr"],
                                                           s["indices"], s["last"], s["lse"], causal=s["causal"],
                                                           out=s["out"])
    if s["op"] == "keep":
        sums = s["sums"][0] if s["layers"] == 1 else s["sums"]
        return eviction.select_kept_tokens(sums, s["lens"], s["budget"], sinks=s["sinks"], recent=s["recent"])
    indptr, indices, last = eviction.evict_paged_kv_cache(s["cache"], s["indptr"], s["indices"], s["last"], s["keep"],
                                                          s["kept"], weights=s["sums"])
    return indptr, indices, last, s["cache"], s["sums"]


# ---------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------

def exact(case, seed):
    """Outputs of run() from the definitions; lists and moved rows hold nothing computed."""
    if case["op"] in ("keep", "evict"):
        return None
    s = prepare(case, seed)
    P, D, B, Hkv = s["P"], s["D"], s["B"], s["Hkv"]
    at, rows, last = s["indptr"].tolist(), s["new_indptr"].tolist(), s["last"].tolist()
    G = s["Hq"] // Hkv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    sums = s["sums"].double() if "sums" in s else None
    for b in range(B):
        L, n = (at[b + 1] - at[b] - 1) * P + last[b], rows[b + 1] - rows[b]
        pages = s["indices"][at[b]:at[b + 1]].long()
        for h in range(Hkv):
            K = s["cache"][pages, 0, h].reshape(-1, D)[:L].double()
            V = s["cache"][pages, 1, h].reshape(-1, D)[:L].double()
            step = max(1, 400_000_000 // (G * L))
            for r in range(0, n, step):
                m = min(step, n - r)
                there = slice(rows[b] + r, rows[b] + r + m), slice(h * G, (h + 1) * G)
                w = torch.einsum("tgd,ld->tgl", s["q"][there].double(), K) / math.sqrt(D)
                if s["causal"]:
                    mine = L - n + r + torch.arange(m, device=DEV)
                    hidden = torch.arange(L, device=DEV)[None] > mine[:, None]
                    w[hidden[:, None].expand_as(w)] = -math.inf
                if sums is not None:
                    sums[b, h, :L] += torch.exp(w - s["lse"][there].double()[..., None]).sum((0, 1))
                    continue
                z = torch.logsumexp(w, -1)
                out[there] = torch.einsum("tgl,ld->tgd", torch.exp(w - z[..., None]), V)
                lse[there] = z
    if sums is None:
        return out, lse
    there = torch.arange(sums.shape[-1], device=DEV) < s["lens"][:, None, None]
    return torch.where(there, sums, s["out"].double())
