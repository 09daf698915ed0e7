"""Cases of the paged-serving operators: what one pass of each computes, in a plain form and through the package.

Operators (the pool is ``[num_pages, 2, Hkv, page_size, D]``, the page table ``(indptr, indices, last_page_len)``):

* ``chunk``   attention of each sequence's newest tokens over its paged cache;
* ``append``  rotary positions applied to new queries and keys, keys and values written into the pool;
* ``rotary``  rotary positions on plain tensors, forward and gradient;
* ``fork``    a new batch of sequences made from parents: pages shared, partial last pages copied;
* ``compact`` live pages moved to the lowest page numbers.

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
        # -- chunk: n newest tokens of each sequence against its whole cache
        # four drafted tokens of one conversation are verified: the latency of the smallest serving step
        dict(name="chunk verify, one sequence", op="chunk", dtype="fp16", Hq=32, Hkv=8, D=128, P=16, B=1, lo=2048,
             hi=2048, new=4, chunks=1, causal=True),
        # five drafted tokens in each of 64 sequences of 512..32768 tokens (the paged decode's benchmark batch)
        dict(name="chunk verify, batch of 64", op="chunk", dtype="fp16", Hq=32, Hkv=8, D=128, P=16, B=64, lo=512,
             hi=32768, new=5, chunks=64, causal=True),
        # one step of continuous batching: eight whole prompts or chunks of them beside eight sequences that decode
        # one token; the 64-wide heads of the prefill benchmark and a page size that no tile is a multiple of
        dict(name="chunk mixed with decoding", op="chunk", dtype="bf16", Hq=64, Hkv=16, D=64, P=20, B=16, lo=94,
             hi=4096, new=1024, chunks=8, causal=True),
        # the last chunk of a long prompt: 8192 tokens on top of 24576, compute bound (the largest case)
        dict(name="chunk of a long prompt", op="chunk", dtype="fp16", Hq=32, Hkv=8, D=128, P=16, B=1, lo=32768,
             hi=32768, new=8192, chunks=1, causal=True),
        # -- append: rotate q and k, write k and v
        # one decoding step of 64 sequences
        dict(name="append while decoding", op="append", dtype="fp16", Hq=32, Hkv=8, D=128, P=16, B=64, lo=512,
             hi=4096, new=1, chunks=64, R=128, interleaved=False),
        # prompt chunks of four sequences, interleaved pairs on half of the head
        dict(name="append of prompt chunks", op="append", dtype="bf16", Hq=32, Hkv=8, D=128, P=16, B=4, lo=2048,
             hi=8192, new=4096, chunks=4, R=64, interleaved=True),
        # -- rotary: forward and gradient
        # a training step's queries and keys: 8 sequences of 1024 tokens
        dict(name="rotary, training step", op="rotary", dtype="bf16", Hq=64, Hkv=16, D=128, T=8192, R=128,
             interleaved=False, top=1024),
        # a few tokens with an odd head width, a part of the head rotated in interleaved pairs
        dict(name="rotary, few tokens", op="rotary", dtype="fp16", Hq=12, Hkv=12, D=80, T=77, R=20,
             interleaved=True, top=4096),
        # -- fork: beams and samples
        # beam search: 16 hypotheses, each of the better eight continued twice
        dict(name="fork of beams", op="fork", dtype="fp16", Hkv=8, D=128, P=16, layers=1, B=16, lo=300, hi=1500,
             children=16, parents=8),
        # 32 prompts, eight samples each, through all of a small model's four layers
        dict(name="fork of samples", op="fork", dtype="bf16", Hkv=8, D=64, P=64, layers=4, B=32, lo=512, hi=4096,
             children=256, parents=32),
        # -- compact: half of the sequences are gone, the pool shrinks
        dict(name="compact of a half empty pool", op="compact", dtype="fp16", Hkv=8, D=128, P=16, layers=1, B=64,
             lo=512, hi=4096, gone=2),
        # a small pool with a few dead pages
        dict(name="compact of a small pool", op="compact", dtype="bf16", Hkv=2, D=64, P=8, layers=2, B=12, lo=17,
             hi=600, gone=6),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("chunk", "chunk", "chunk", "append", "rotary", "fork", "compact"))
    dtype = rng.choice(("fp16", "bf16"))
    D = rng.choice((64, 128, 128))
    Hkv = rng.choice((1, 2, 4, 8, 8, 16))
    G = rng.choice((1, 2, 3, 4, 4, 5, 8))
    P = rng.choice((1, 5, 8, 16, 16, 16, 20, 32, 64, 128))
    if op == "chunk":
        hi = _log(rng, 1, 32768)
        lo = max(1, int(hi * rng.uniform(0.05, 1.0)))
        new = min(_log(rng, 1, 8192), hi)
        B = _log(rng, 1, 64)
        # at most half of the largest case's products, and a plain form that fits the card
        while B > 1 and (B * Hkv * G * new * hi > 4e9 or B * hi * Hkv * D > 1.1e9):
            B = max(1, B // 2)
        if Hkv * G * new * hi > 4e9:
            new = max(1, int(4e9 / (Hkv * G * hi)))
        return dict(op=op, dtype=dtype, Hq=Hkv * G, Hkv=Hkv, D=D, P=P, B=B, lo=lo, hi=hi, new=new,
                    chunks=rng.choice((B, B, max(1, B // 4))), causal=rng.random() < 0.8)
    if op == "append":
        hi = _log(rng, 8, 16384)
        B = _log(rng, 1, 128)
        while B > 1 and B * hi * Hkv * D > 2e8:
            B = max(1, B // 2)
        new = min(_log(rng, 1, 4096), hi)
        while new > 1 and B * new * Hkv * (G + 2) * D > 1e8:
            new = max(1, new // 2)
        R = rng.choice((D, D, D // 2, D // 4, 24, 10))
        return dict(op=op, dtype=dtype, Hq=Hkv * G, Hkv=Hkv, D=D, P=P, B=B, lo=max(1, hi // rng.choice((1, 2, 7))),
                    hi=hi, new=new, chunks=rng.choice((B, max(1, B // 3))), R=R, interleaved=rng.random() < 0.5)
    if op == "rotary":
        D = rng.choice((64, 80, 96, 128, 128, 256))
        T = _log(rng, 1, 32768)
        while T > 1 and T * Hkv * (G + 1) * D > 1.3e8:
            T //= 2
        return dict(op=op, dtype=dtype, Hq=Hkv * G, Hkv=Hkv, D=D, T=T, R=rng.choice((D, D, D // 2, 20, 32)),
                    interleaved=rng.random() < 0.5, top=_log(rng, 16, 131072))
    layers = rng.choice((1, 1, 2, 4))
    hi = _log(rng, 8, 8192)
    B = _log(rng, 2, 128)
    while B > 2 and layers * B * hi * Hkv * D > 2.5e8:
        B = max(2, B // 2)
    pool = dict(op=op, dtype=dtype, Hkv=Hkv, D=D, P=P, layers=layers, B=B, lo=max(1, hi // rng.choice((1, 3, 10))),
                hi=hi)
    if op == "fork":
        return dict(pool, children=B * rng.choice((1, 1, 2, 4)), parents=rng.choice((B, max(1, B // 2), max(1, B // 5))))
    return dict(pool, gone=rng.choice((2, 3, 8)))


def _lens(case):
    """Tokens of each sequence, evenly spread over lo..hi (both ends held)."""
    B, lo, hi = case["B"], case["lo"], case["hi"]
    return [hi] if B == 1 else [lo + (hi - lo) * i // (B - 1) for i in range(B)]


def _news(case):
    """New tokens of each sequence: a full or a somewhat shorter chunk for `chunks` of them, one token for the rest."""
    step, most, cut = max(1, case["B"] // case["chunks"]), case["chunks"], case["new"] // 16
    return [min(n, case["new"] - (i // step % 4) * cut) if i % step == 0 and i // step < most else 1
            for i, n in enumerate(_lens(case))]


def _pages(n, P):
    return -(-n // P)


def _parents(case):
    """Parent of each child: the first `parents` sequences in turn, children of one parent apart."""
    return [i % case["parents"] for i in range(case["children"])]


def work(case):
    op, es = case["op"], 2
    if op == "rotary":
        n = case["T"] * (case["Hq"] + case["Hkv"])
        rows = case["T"] * (case["R"] * 4 + 4)
        return {"bytes": 2 * (2 * n * case["D"] * es + rows), "flops": 2 * 3 * n * case["R"]}
    D, Hkv, P = case["D"], case["Hkv"], case["P"]
    lens = _lens(case)
    pages = [_pages(n, P) for n in lens]
    table = 4 * (sum(pages) + 2 * len(lens) + 1)
    if op == "chunk":
        news = _news(case)
        pairs = sum(n * (L - n) + (n * (n + 1) // 2 if case["causal"] else n * n) for n, L in zip(news, lens))
        rows = sum(news) * case["Hq"]
        return {"bytes": 2 * sum(lens) * Hkv * D * es + rows * (2 * D * es + 4) + table,
                "flops": 4 * case["Hq"] * D * pairs}
    if op == "append":
        T = sum(_news(case))
        return {"bytes": 2 * T * (case["Hq"] + 2 * Hkv) * D * es + T * case["R"] * 4 + 4 * (3 * len(lens) + T),
                "flops": 3 * T * (case["Hq"] + Hkv) * case["R"]}
    page = case["layers"] * 2 * Hkv * P * D * es
    if op == "fork":
        par = _parents(case)
        copies = sum(1 for i, p in enumerate(par) if p in par[:i] and lens[p] % P)
        return {"bytes": 2 * copies * page + table + 4 * (sum(pages[p] for p in par) + 3 * len(par)), "flops": 0}
    # compact: pages stand in a random order, so about the share of dead pages of the live ones has to move
    live = sum(p for i, p in enumerate(pages) if i % case["gone"])
    moved = live * (1 - live / max(1, sum(pages)))
    return {"bytes": 2 * moved * page + 2 * 4 * live, "flops": 0}


# ---------------------------------------------------------------------------
# what a program has in hand before the call
# ---------------------------------------------------------------------------

def _table(lens, P, order, gen, extra=0):
    """CSR page table of the sequences in `order`, their pages in random places of a pool with `extra` more."""
    pages = [_pages(lens[i], P) for i in order]
    n = sum(pages)
    indices = torch.randperm(n + extra, generator=gen, device=DEV)[:n].to(torch.int32)
    last = [lens[i] - P * (p - 1) for i, p in zip(order, pages)]
    return _indptr(pages), indices, torch.tensor(last, dtype=torch.int32, device=DEV), n + extra


def _normal(shape, case, gen):
    return torch.randn(shape, generator=gen, device=DEV, dtype=TYPES[case["dtype"]])


def _cos_sin(top, R):
    """fp32 table of a rotary embedding, as a model keeps it: cosines of R/2 angles, then their sines."""
    half = torch.arange(R // 2, device=DEV, dtype=torch.float64)
    angle = torch.arange(top, device=DEV, dtype=torch.float64)[:, None] * (10000.0 ** (-2 * half / R))
    return torch.cat((angle.cos(), angle.sin()), 1).float()


def _indptr(counts):
    return torch.tensor([0, *itertools.accumulate(counts)], dtype=torch.int32, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    rng = random.Random(seed)
    s = dict(case)
    op = case["op"]
    if op == "rotary":
        T, Hq, Hkv, D = case["T"], case["Hq"], case["Hkv"], case["D"]
        s["cos_sin"] = _cos_sin(case["top"], case["R"])
        s["positions"] = (torch.arange(T, device=DEV, dtype=torch.int32) + rng.randrange(case["top"])) % case["top"]
        for n, H in (("q", Hq), ("k", Hkv), ("dq", Hq), ("dk", Hkv)):
            s[n] = _normal((T, H, D), case, gen)
        return s
    lens, order = _lens(case), list(range(case["B"]))
    rng.shuffle(order)
    P, D, Hkv = case["P"], case["D"], case["Hkv"]
    if op in ("chunk", "append"):
        news = _news(case)
        s["indptr"], s["indices"], s["last"], N = _table(lens, P, order, gen)
        s["new_indptr"] = _indptr([news[i] for i in order])
        s["max_len"], s["max_new"] = max(lens), max(news)
        T = sum(news)
        if op == "chunk":
            s["q"] = _normal((T, case["Hq"], D), case, gen)
            s["cache"] = _normal((N, 2, Hkv, P, D), case, gen)
        else:
            # one projection's output holds queries, keys and values side by side
            qkv = _normal((T, case["Hq"] + 2 * Hkv, D), case, gen)
            s["q"], s["k"], s["v"] = qkv.split((case["Hq"], Hkv, Hkv), 1)
            s["cache"] = torch.zeros((N, 2, Hkv, P, D), dtype=TYPES[case["dtype"]], device=DEV)
            s["cos_sin"] = _cos_sin(max(lens), case["R"])
        return s
    if op == "fork":
        par = _parents(case)
        # room for the copies, and a few pages more
        s["indptr"], s["indices"], s["last"], N = _table(lens, P, order, gen, extra=case["children"] + 3)
        at = {i: j for j, i in enumerate(order)}
        s["parents"] = torch.tensor([at[p] for p in par], dtype=torch.int32, device=DEV)
        s["entries"] = sum(_pages(lens[p], P) for p in par)
    else:
        indptr, indices, last, N = _table(lens, P, order, gen)
        # the sequences that stay keep their pages; the others' pages are dead
        stay = [j for j, i in enumerate(order) if i % case["gone"]]
        at = indptr.tolist()
        s["indptr"] = _indptr([at[j + 1] - at[j] for j in stay])
        s["indices"] = torch.cat([indices[at[j]:at[j + 1]] for j in stay])
    shape = (N, 2, Hkv, P, D) if case["layers"] == 1 else (case["layers"], N, 2, Hkv, P, D)
    s["cache"] = _normal(shape, case, gen)
    s["num_pages"] = N
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _new_tokens(s):
    """Sequence, number in its chunk and position of each new token."""
    at = s["new_indptr"].long()
    t = torch.arange(s["q"].shape[0], device=DEV)
    b = torch.searchsorted(at, t, right=True) - 1
    pages = (s["indptr"][1:] - s["indptr"][:-1]).long()
    length = (pages - 1) * s["P"] + s["last"].long()
    i = t - at[b]
    return b, i, length[b] - (at[b + 1] - at[b]) + i, length


def _chunk(s):
    Hkv, D, P, B = s["Hkv"], s["D"], s["P"], s["B"]
    G = s["Hq"] // Hkv
    b, i, pos, length = _new_tokens(s)
    n, L = s["max_new"], _pages(s["max_len"], P) * P
    # keys and values of each sequence side by side, padded to the longest
    page = s["indptr"][:-1].long()[:, None] + torch.arange(L // P, device=DEV)
    inside = page < s["indptr"][1:, None]
    page = torch.where(inside, s["indices"].long()[page.clamp(max=s["indices"].numel() - 1)], 0)
    j = torch.arange(L, device=DEV)
    seen = j < length[:, None]
    kv = s["cache"][page].permute(2, 0, 3, 1, 4, 5).reshape(2, B, Hkv, L, D)
    k, v = kv[0].float(), torch.where(seen[:, None, :, None], kv[1], 0).float()
    del kv
    q = torch.zeros((B, n, Hkv, G, D), device=DEV)
    q[b, i] = s["q"].float().unflatten(1, (Hkv, G))
    at = torch.full((B, n), -1, dtype=torch.long, device=DEV)
    at[b, i] = pos
    x = torch.matmul(q.permute(0, 2, 1, 3, 4).reshape(B, Hkv, n * G, D), k.transpose(2, 3))
    x = x.mul_(1 / math.sqrt(D)).view(B, Hkv, n, G, L)
    x = x.masked_fill_(~seen[:, None, None, None], -math.inf)
    if s["causal"]:
        x = x.masked_fill_((j > at[:, :, None])[:, None, :, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0, top)
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    out = torch.matmul(x.view(B, Hkv, n * G, L), v).view(B, Hkv, n, G, D)
    out = torch.where(total > 0, out / total, 0).permute(0, 2, 1, 3, 4)[b, i].flatten(1, 2)
    lse = (total.log() + top)[..., 0].permute(0, 2, 1, 3)[b, i].flatten(1, 2)
    return out.to(s["q"].dtype), lse


def _rotate(x, cos, sin, interleaved):
    """x [T, H, D] in fp32 with the pairs of its first R values turned; cos, sin [T, R/2]."""
    R = 2 * cos.shape[1]
    cos, sin = cos[:, None], sin[:, None]
    x = x.float()
    if interleaved:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., R:]), -1)


def _append(s):
    b, i, pos, _ = _new_tokens(s)
    half, kind = s["R"] // 2, s["q"].dtype
    row = s["cos_sin"][pos]
    cos, sin = row[:, :half], row[:, half:]
    page = s["indices"].long()[s["indptr"].long()[b] + pos // s["P"]]
    s["cache"][page, 0, :, pos % s["P"]] = _rotate(s["k"], cos, sin, s["interleaved"]).to(kind)
    s["cache"][page, 1, :, pos % s["P"]] = s["v"]
    return _rotate(s["q"], cos, sin, s["interleaved"]).to(kind), s["cache"]


def _rotary(s):
    half, kind = s["R"] // 2, s["q"].dtype
    row = s["cos_sin"][s["positions"].long()]
    cos, sin = row[:, :half], row[:, half:]
    turn = lambda x, sin: _rotate(x, cos, sin, s["interleaved"]).to(kind)  # noqa: E731
    return turn(s["q"], sin), turn(s["k"], sin), turn(s["dq"], -sin), turn(s["dk"], -sin)


def _dead_first(live):
    """Numbers of the pages that `live` does not mark, ascending, then of the others."""
    return torch.argsort(live.to(torch.uint8), stable=True)


def _fork(s):
    par, P = s["parents"].long(), s["P"]
    pages = (s["indptr"][1:] - s["indptr"][:-1]).long()[par]
    end = pages.cumsum(0)
    child = torch.repeat_interleave(torch.arange(par.numel(), device=DEV), pages, output_size=s["entries"])
    e = torch.arange(s["entries"], device=DEV) - (end - pages)[child]
    indices = s["indices"].long()[s["indptr"].long()[par][child] + e]
    last = s["last"][par]
    again = (par[:, None] == par[None]).tril(-1).any(1)
    copied = torch.nonzero(again & (last < P) & (pages > 0))[:, 0]
    live = torch.zeros(s["num_pages"], dtype=torch.bool, device=DEV)
    live[indices] = True
    to = _dead_first(live)[:copied.numel()]
    at = end[copied] - 1
    pool = s["cache"] if s["layers"] > 1 else s["cache"][None]
    pool[:, to] = pool[:, indices[at]]
    indices[at] = to
    indptr = torch.cat((end.new_zeros(1), end))
    return indptr.int(), indices.int(), last, s["cache"]


def _compact(s):
    live = torch.zeros(s["num_pages"], dtype=torch.bool, device=DEV)
    live[s["indices"].long()] = True
    used = live.sum()
    low = torch.arange(s["num_pages"], device=DEV) < used
    source, target = torch.nonzero(live & ~low)[:, 0], torch.nonzero(low & ~live)[:, 0]
    pool = s["cache"] if s["layers"] > 1 else s["cache"][None]
    pool[:, target] = pool[:, source]
    to = torch.arange(s["num_pages"], device=DEV)
    to[source] = target
    return to[s["indices"].long()].int(), used.int(), s["cache"]


_PLAIN = {"chunk": _chunk, "append": _append, "rotary": _rotary, "fork": _fork, "compact": _compact}


def run(state):
    s = state
    if not own:
        return _PLAIN[s["op"]](s)
    if s["op"] == "chunk":
        from attention_kernel_triton_b200.paged_chunk_attention import flash_attention_chunk_paged_with_lse
        return flash_attention_chunk_paged_with_lse(s["q"], s["new_indptr"], s["cache"], s["indptr"], s["indices"],
                                                    s["last"], causal=s["causal"])
    if s["op"] == "append":
        from attention_kernel_triton_b200.rotary_embedding import append_rotary_paged_kv_cache
        q = append_rotary_paged_kv_cache(s["cache"], s["q"], s["k"], s["v"], s["new_indptr"], s["indptr"],
                                         s["indices"], s["last"], s["cos_sin"], interleaved=s["interleaved"])
        return q, s["cache"]
    if s["op"] == "rotary":
        from attention_kernel_triton_b200.rotary_embedding import apply_rotary_qk
        table = (s["cos_sin"], s["positions"])
        q, k = apply_rotary_qk(s["q"], s["k"], *table, interleaved=s["interleaved"])
        dq, dk = apply_rotary_qk(s["dq"], s["dk"], *table, interleaved=s["interleaved"], inverse=True)
        return q, k, dq, dk
    if s["op"] == "fork":
        from attention_kernel_triton_b200.paged_kv_pages import fork_paged_kv_cache
        return (*fork_paged_kv_cache(s["cache"], s["indptr"], s["indices"], s["last"], s["parents"],
                                     max_entries=s["entries"]), s["cache"])
    from attention_kernel_triton_b200.paged_kv_pages import compact_paged_kv_cache
    indices, used = compact_paged_kv_cache(s["cache"], s["indices"])
    return indices, used, s["cache"]


# ---------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------

def exact(case, seed):
    """Outputs of run() from the definitions; pages that are copied and numbered hold nothing computed."""
    if case["op"] in ("fork", "compact"):
        return None
    s = prepare(case, seed)

    def turn(x, rows, sign=1.0):
        # the pairs as complex numbers, turned by cos + i sin
        R = rows.shape[1]
        by = torch.complex(rows[:, :R // 2].double(), sign * rows[:, R // 2:].double())[:, None]
        y = x.double().clone()
        head = y[..., :R]
        pair = head.unflatten(-1, (R // 2, 2)) if s["interleaved"] else head.unflatten(-1, (2, R // 2)).transpose(-1, -2)
        z = torch.complex(pair[..., 0].contiguous(), pair[..., 1].contiguous()) * by
        pair.copy_(torch.stack((z.real, z.imag), -1))
        return y

    if case["op"] == "rotary":
        rows = s["cos_sin"][s["positions"].long()]
        return turn(s["q"], rows), turn(s["k"], rows), turn(s["dq"], rows, -1.0), turn(s["dk"], rows, -1.0)

    P, D, B = s["P"], s["D"], s["B"]
    at, rows, last = s["indptr"].tolist(), s["new_indptr"].tolist(), s["last"].tolist()
    length = [(at[b + 1] - at[b] - 1) * P + last[b] for b in range(B)]
    news = [rows[b + 1] - rows[b] for b in range(B)]

    if case["op"] == "append":
        pos = torch.cat([torch.arange(L - n, L) for L, n in zip(length, news)])
        first = torch.repeat_interleave(torch.tensor(at[:-1]), torch.tensor(news))
        page = s["indices"].long()[(first + pos // P).to(DEV)]
        pos = pos.to(DEV)
        cache = s["cache"].double()
        cache[page, 0, :, pos % P] = turn(s["k"], s["cos_sin"][pos])
        cache[page, 1, :, pos % P] = s["v"].double()
        return turn(s["q"], s["cos_sin"][pos]), cache

    G = s["Hq"] // s["Hkv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    for b, (L, n) in enumerate(zip(length, news)):
        pages = s["indices"][at[b]:at[b + 1]].long()
        for h in range(s["Hkv"]):
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
                z = torch.logsumexp(w, -1)
                out[there] = torch.einsum("tgl,ld->tgd", torch.exp(w - z[..., None]), V)
                lse[there] = z
    return out, lse
