"""More operators of a server's caches, as cases that can be timed: each in a
plain form (elementary torch operations) and, with ``own``, through
popcorn_amd's descriptors.

* ``prefix``: attention of a batch whose requests share long prefixes. A group
  of requests that follow each other has its prefix in pages of its own, read
  once for all of them; each request's other keys are in the request's pages. Beside the result
  stands the logarithm of each row's sum of exponentials.
* ``weights``: what the new tokens' attention gives each cached key, summed
  over tokens and the query heads of its KV head, added to what the key had.
* ``evict``: every KV head of a request keeps ``budget`` keys: its first and
  last ones and those of the highest weight (ties: the lowest index) among the others, moved to the
  cache's front in their order; with the weights and the kept keys' indices.
* ``release``: the lengths after an eviction, and the pages that it left empty.

A cache is [pages, KV heads, page size, head dim]; row r of a page table names
the pages of request r's keys in order.
"""
import math
import random

import numpy as np
import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_ENV = []


def _env():
    """The encoder that a program makes once, on torch's default stream."""
    if not _ENV:
        import popcorn_amd as pa

        lib = pa.KernelLibrary()
        _ENV.extend((pa, lib, pa.KernelCommandEncoder(lib)))
    return _ENV[0], _ENV[2]


def _t(x):
    """The framework's view of a torch tensor."""
    pa, _ = _env()
    dtype = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16", torch.int32: "i32"}[x.dtype]
    return pa.Tensor(x.data_ptr(), tuple(x.shape), dtype, owner=[x])


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(values):
    return torch.tensor(list(values), dtype=torch.int32, device="cuda")


def _ceil(a, b):
    return -(-a // b)


def _arange(n):
    return torch.arange(n, device="cuda")


def _rows(g, shape, dtype, std=1.0):
    return torch.randn(shape, device="cuda", generator=g).mul_(std).to(TORCH[dtype])


def _lengths(c):
    """(keys in the request's pages, new tokens) of each request: a case's own numbers, the same for every seed."""
    rng = random.Random(c["lens"])
    out = []
    for r in range(c["requests"]):
        past = int(math.exp(rng.uniform(math.log(c["past_lo"] + 1), math.log(c["past_hi"] + 1)))) - 1
        past = min(max(past, c["past_lo"]), c["past_hi"])
        new = rng.randint(c["chunk_lo"], c["chunk_hi"]) if r < c["chunks"] else c["few"]
        out.append((past, new))
    rng.shuffle(out)
    return out


def _prefixes(c):
    """(prefix lengths, first request of each group and the end): the last `alone` requests have no prefix."""
    rng = random.Random(c["lens"] + 1)
    g, inside = c["groups"], c["requests"] - c["alone"]
    lens = [c["prefix_hi"]] + [rng.randint(c["prefix_lo"], c["prefix_hi"]) for _ in range(g - 1)]
    cuts = sorted(rng.sample(range(1, inside), g - 1)) if g > 1 else []
    return lens, [0] + cuts + [inside]


def _table(lens, page, ids, columns):
    """A table of `lens` keys each, with pages from the front of ids; -1 where a request has none."""
    held = torch.tensor([_ceil(n, page) for n in lens], device="cuda")
    table = torch.full((len(lens), columns), -1, dtype=torch.int32, device="cuda")
    table[_arange(columns) < held.unsqueeze(1)] = ids[:sum(_ceil(n, page) for n in lens)].int()
    return table


def _starts(lens):
    starts = [0]
    for _, n in lens:
        starts.append(starts[-1] + n)
    return starts


def _gathered(cache, table):
    """The keys that a table's rows name, in f32: [rows, Nkv, columns * page, Hd]; -1 reads page 0."""
    x = cache[table.long().clamp(min=0)].transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[4]).float()


def _new_tokens(starts, most):
    """Rows [R, most] of the requests' last `most` new tokens (row 0 where one has fewer), and which there are."""
    n = (starts[1:] - starts[:-1]).long().clamp(max=most)
    i = _arange(most)
    there = i < n.unsqueeze(1)
    return torch.where(there, starts[1:].long().unsqueeze(1) - n.unsqueeze(1) + i, 0), there


# ---- prefix ------------------------------------------------------------------------


def _prefix_inputs(c, seed):
    g, lens, page, t = _gen(seed), _lengths(c), c["page"], c["dtype"]
    prefixes, groups = _prefixes(c)
    own_lens = [p + n for p, n in lens]
    held = [sum(_ceil(n, page) for n in x) for x in (prefixes, own_lens)]
    pages, tokens = sum(held) + 3, sum(n for _, n in lens)
    order = torch.randperm(pages, device="cuda", generator=g)
    q = _rows(g, (tokens + c["pad"], c["nq"], c["hd"]), t, 1.5)
    k, v = (_rows(g, (pages, c["nkv"], page, c["hd"]), t) for _ in range(2))
    return {"q": q, "k": k, "v": v, "prefix": _table(prefixes, page, order, _ceil(max(prefixes), page)),
            "prefix_lens": _ints(prefixes), "groups": _ints(groups),
            "table": _table(own_lens, page, order[held[0]:], _ceil(max(own_lens), page) + c["spare_columns"]),
            "starts": _ints(_starts(lens)), "keys": _ints(own_lens), "tokens": tokens, "most": max(n for _, n in lens),
            "out": torch.full_like(q, 7.0),  # rows behind the last request's stay as they are
            "lse": torch.full(q.shape[:2], 7.0, device="cuda")}


def _prefix_prepare(c, seed):
    s = _prefix_inputs(c, seed)
    s["case"] = c
    if own:
        pa, s["enc"] = _env()
        mask = pa.AttentionMask.causal_sliding_window(c["window"]) if c["window"] else pa.AttentionMask.causal
        s["kernel"] = pa.Kernels.SharedPrefixAttention(
            *(_t(s[n]) for n in ("q", "k", "v", "prefix", "prefix_lens", "groups", "table", "starts", "keys", "out")),
            scale=c["hd"] ** -0.5, mask=mask, sinks=c["sinks"], max_query_len=s["most"], lse=_t(s["lse"]))
    return s


def _prefix_run(s):
    c, t = s["case"], s["tokens"]
    nkv, per, hd = c["nkv"], c["nq"] // c["nkv"], c["hd"]
    starts, keys = s["starts"].long(), s["keys"].long()
    request = torch.searchsorted(starts, _arange(t), right=True) - 1
    group = torch.searchsorted(s["groups"].long(), request, right=True) - 1
    prefixes = s["prefix_lens"].long()
    before = torch.where(group < prefixes.numel(), prefixes[group.clamp(max=prefixes.numel() - 1)], 0)
    place = keys[request] - starts[request + 1] + _arange(t)  # of the token among its request's own keys
    q = s["q"][:t].float().mul(hd ** -0.5).view(t, nkv, per, hd)

    # all prefixes in a row, and which of them a token sees
    k, v = (_gathered(x, s["prefix"]) for x in (s["k"], s["v"]))
    width = k.shape[2]
    k, v = (x.transpose(0, 1).reshape(nkv, -1, hd) for x in (k, v))
    a = torch.matmul(q.transpose(0, 1).reshape(nkv, t * per, hd), k.transpose(1, 2).contiguous()).view(nkv, t, per, -1)
    j = _arange(width).repeat(prefixes.numel())
    of = torch.arange(prefixes.numel(), device="cuda").repeat_interleave(width)
    sees = (of == group.unsqueeze(1)) & (j < prefixes[of])
    if c["window"]:
        sees &= ((before + place).unsqueeze(1) - j < c["window"]) | (j < c["sinks"])
    a.masked_fill_(~sees.unsqueeze(1), -math.inf)

    # each request's own keys, padded to the longest
    rows, there = _new_tokens(starts, s["most"])
    r, i = torch.nonzero(there, as_tuple=True)
    k_own, v_own = (_gathered(x, s["table"]) for x in (s["k"], s["v"]))
    b = torch.matmul(q[rows].permute(0, 2, 1, 3, 4).reshape(len(rows), nkv, -1, hd), k_own.transpose(2, 3).contiguous())
    b = b.view(len(rows), nkv, s["most"], per, -1)
    x, at = _arange(b.shape[-1]), place[rows].unsqueeze(-1)
    sees = x <= at
    if c["window"]:
        sees &= (at - x < c["window"]) | (before[rows].unsqueeze(-1) + x < c["sinks"])
    b.masked_fill_(~sees[:, None, :, None], -math.inf)

    top = a.amax(-1).permute(1, 0, 2)  # [T, Nkv, per]
    top = torch.maximum(top, b.amax(-1)[r, :, i])
    a = torch.exp_(a.sub_(top.permute(1, 0, 2).unsqueeze(-1)))
    b = torch.exp_(b.sub_(top[rows].transpose(1, 2).unsqueeze(-1)))
    total = a.sum(-1).permute(1, 0, 2) + b.sum(-1)[r, :, i]
    o = torch.matmul(a.view(nkv, t * per, -1), v).view(nkv, t, per, hd).transpose(0, 1)
    o = o + torch.matmul(b.view(len(rows), nkv, s["most"] * per, -1), v_own).view(len(rows), nkv, s["most"], per, hd)[r, :, i]
    s["out"][:t] = o.div_(total.unsqueeze(-1)).reshape(t, c["nq"], hd).to(s["out"].dtype)
    s["lse"][:t] = (top + torch.log(total)).reshape(t, c["nq"])
    return s["out"], s["lse"]


def _prefix_exact(c, seed):
    s, lens, page = _prefix_inputs(c, seed), _lengths(c), c["page"]
    prefixes, groups = _prefixes(c)
    out, lse = s["out"].double(), s["lse"].double()

    def of(cache, table, n):
        ids = table[:_ceil(n, page)].long()
        return cache[ids].double().permute(1, 0, 2, 3).reshape(c["nkv"], -1, c["hd"])[:, :n]

    at, shared = 0, {}
    for r, (past, n) in enumerate(lens):
        g = next((g for g in range(len(prefixes)) if groups[g] <= r < groups[g + 1]), None)
        first = prefixes[g] if g is not None else 0
        if g not in shared:
            shared = {g: [of(s[x], s["prefix"][g], first) if first else None for x in ("k", "v")]}
        k, v = (torch.cat([x, y], 1) if first else y for x, y in zip(shared[g], (of(s[x], s["table"][r], past + n) for x in ("k", "v"))))
        pos, key = first + past + torch.arange(n, device="cuda").unsqueeze(1), torch.arange(first + past + n, device="cuda")
        hide = key > pos
        if c["window"]:
            hide |= (pos - key >= c["window"]) & (key >= c["sinks"])
        for h in range(c["nkv"]):
            for e in range(h * c["nq"] // c["nkv"], (h + 1) * c["nq"] // c["nkv"]):
                a = (s["q"][at:at + n, e].double() @ k[h].t().contiguous()) / math.sqrt(c["hd"])
                a.masked_fill_(hide, -math.inf)
                lse[at:at + n, e] = torch.logsumexp(a, -1)
                out[at:at + n, e] = torch.softmax(a, -1) @ v[h]
        at += n
    return out, lse


def _prefix_work(c):
    """(bytes, flops): a key that some token sees is read once, whoever shares it."""
    lens, (prefixes, groups) = _lengths(c), _prefixes(c)
    w, s = c["window"] or 1 << 40, c["sinks"]
    pairs = keys = 0
    for r, (past, n) in enumerate(lens):
        g = next((g for g in range(len(prefixes)) if groups[g] <= r < groups[g + 1]), None)
        first = prefixes[g] if g is not None else 0
        for i in range(first + past, first + past + n):
            pairs += min(i + 1, w) + min(s, max(i + 1 - w, 0))
        lo = max(first + past - w + 1, 0)  # of the request's first new token
        keys += past + n - max(lo - first, 0) + min(max(s - first, 0), max(lo - first, 0)) if n else 0
    for g, first in enumerate(prefixes):
        seen = [max(first + past - w + 1, 0) for past, n in lens[groups[g]:groups[g + 1]] if n]
        lo = min(min(seen), first) if seen else first
        keys += first - lo + min(s, lo)
    tokens = sum(n for _, n in lens)
    return (SIZE[c["dtype"]] * c["hd"] * (2 * c["nq"] * tokens + 2 * c["nkv"] * keys) + 4 * c["nq"] * tokens, 4.0 * c["nq"] * c["hd"] * pairs)


# ---- weights -----------------------------------------------------------------------


def _weights_inputs(c, seed):
    g, lens, page, t = _gen(seed), _lengths(c), c["page"], c["dtype"]
    held = [p + n for p, n in lens]
    pages, tokens = sum(_ceil(n, page) for n in held) + 3, sum(n for _, n in lens)
    q = _rows(g, (tokens + c["pad"], c["nq"], c["hd"]), t, 1.5)
    k = _rows(g, (pages, c["nkv"], page, c["hd"]), t)
    columns = _ceil(max(held), page) + c["spare_columns"]
    s = {"q": q, "k": k, "table": _table(held, page, torch.randperm(pages, device="cuda", generator=g), columns),
         "starts": _ints(_starts(lens)), "keys": _ints(held), "most": max(n for _, n in lens)}
    s["rows"] = min(s["most"], c["last_rows"] or s["most"])
    # what the attention before this call gave of each row; rows that do not count have some too
    s["lse"] = torch.full(q.shape[:2], 8.0, device="cuda")
    rows, there = _new_tokens(s["starts"], s["rows"])
    a = _weights_scores(c, s, rows)
    s["lse"][rows[there]] = torch.logsumexp(a, -1).transpose(1, 2)[there].reshape(-1, c["nq"])
    # what earlier steps gave each key, where there are keys
    s["weights"] = torch.rand((len(lens), c["nkv"], columns * page), device="cuda", generator=g).pow_(4.0)
    s["weights"].masked_fill_(_arange(columns * page) >= (s["keys"] - s["starts"].diff()).view(-1, 1, 1), 0.0)
    return s


def _weights_scores(c, s, rows):
    """The scaled products of the rows [R, n] with their requests' keys, -inf where they do not see one: [R, Nkv, n, per, keys]."""
    nkv, per, hd = c["nkv"], c["nq"] // c["nkv"], c["hd"]
    k = _gathered(s["k"], s["table"])
    q = s["q"].float().mul(hd ** -0.5)[rows].view(*rows.shape, nkv, per, hd).permute(0, 2, 1, 3, 4).reshape(len(rows), nkv, -1, hd)
    a = torch.matmul(q, k.transpose(2, 3).contiguous()).view(len(rows), nkv, rows.shape[1], per, -1)
    place = (s["keys"].long() - s["starts"][1:].long()).unsqueeze(1) + rows
    return a.masked_fill_((_arange(a.shape[-1]) > place.unsqueeze(-1))[:, None, :, None], -math.inf)


def _weights_prepare(c, seed):
    s = _weights_inputs(c, seed)
    s["case"] = c
    if own:
        pa, s["enc"] = _env()
        s["kernel"] = pa.Kernels.PagedAttentionWeights(
            *(_t(s[n]) for n in ("q", "k", "table", "starts", "keys", "lse", "weights")), scale=c["hd"] ** -0.5,
            last_rows=c["last_rows"], max_query_len=s["most"])
    return s


def _weights_run(s):
    c = s["case"]
    rows, there = _new_tokens(s["starts"], s["rows"])
    lse = s["lse"][rows].view(*rows.shape, c["nkv"], -1, 1).transpose(1, 2)
    a = torch.exp_(_weights_scores(c, s, rows).sub_(lse))
    a.masked_fill_(~there[:, None, :, None, None], 0.0)
    s["weights"] += a.sum((2, 3))
    return s["weights"]


def _weights_exact(c, seed):
    s, lens, page = _weights_inputs(c, seed), _lengths(c), c["page"]
    out, at, per = s["weights"].double(), 0, c["nq"] // c["nkv"]
    for r, (past, n) in enumerate(lens):
        lo = max(0, n - (c["last_rows"] or n))
        k = s["k"][s["table"][r, :_ceil(past + n, page)].long()].double().transpose(0, 1).reshape(c["nkv"], -1, c["hd"])[:, :past + n]
        hide = torch.arange(past + n, device="cuda") > past + torch.arange(lo, n, device="cuda").unsqueeze(1)
        for e in range(c["nq"]):
            a = (s["q"][at + lo:at + n, e].double() @ k[e // per].t().contiguous()) / math.sqrt(c["hd"]) - s["lse"][at + lo:at + n, e:e + 1].double()
            out[r, e // per, :past + n] += torch.exp(a).masked_fill(hide, 0.0).sum(0)
        at += n
    return out


def _weights_work(c):
    """(bytes, flops)"""
    pairs = keys = rows = 0
    for past, n in _lengths(c):
        m = min(n, c["last_rows"] or n)
        pairs += m * (past + n - m) + m * (m + 1) // 2
        keys += past + n if m else 0
        rows += m
    return (SIZE[c["dtype"]] * c["hd"] * (c["nq"] * rows + c["nkv"] * keys) + 4 * c["nq"] * rows + 8 * c["nkv"] * keys, 2.0 * c["nq"] * c["hd"] * pairs)


# ---- evict -------------------------------------------------------------------------


def _budgets(c):
    """(keys, budget) of each request"""
    return [(p + n, min(c["budget"], p + n)) for p, n in _lengths(c)]


def _evict_inputs(c, seed):
    g, page, t = _gen(seed), c["page"], c["dtype"]
    held = [n for n, _ in _budgets(c)]
    pages, columns = sum(_ceil(n, page) for n in held) + 3, _ceil(max(held), page) + c["spare_columns"]
    k, v = (_rows(g, (pages, c["nkv"], page, c["hd"]), t) for _ in range(2))
    keys = _ints(held)
    # a few heavy keys and many light ones, on a coarse grid so that some are alike
    w = torch.randn((len(held), c["nkv"], columns * page), device="cuda", generator=g).mul_(2.0).exp_().to(torch.bfloat16).float()
    w.masked_fill_(_arange(columns * page) >= keys.view(-1, 1, 1), 0.0)
    return {"weights": w, "k": k, "v": v, "table": _table(held, page, torch.randperm(pages, device="cuda", generator=g), columns),
            "keys": keys, "budgets": _ints([c["budget"]] * len(held)), "most": min(c["budget"], max(held)),
            "kept": torch.full(w.shape, -1, dtype=torch.int32, device="cuda"), "kept_weights": torch.full_like(w, 7.0)}


def _evict_prepare(c, seed):
    s = _evict_inputs(c, seed)
    s["case"] = c
    if own:
        pa, s["enc"] = _env()
        s["kernel"] = pa.Kernels.PagedEviction(*(_t(s[n]) for n in ("weights", "k", "v", "table", "keys", "budgets", "kept", "kept_weights")),
                                               first=c["first"], last=c["last"])
    return s


def _evict_run(s):
    c, w = s["case"], s["weights"]
    r, nkv, room = w.shape
    x = _arange(room)
    keys = s["keys"].long().view(-1, 1, 1)
    n = torch.minimum(keys, s["budgets"].long().view(-1, 1, 1))
    first = n.clamp(max=c["first"])
    last = torch.minimum(n - first, torch.tensor(c["last"], device="cuda"))
    # ranks: the first and the last ones before all others, then by weight, ties by index; what is no key last
    rank = torch.where((x < first) | (x >= keys - last), math.inf, w.double()).masked_fill_(x >= keys, -math.inf)
    order = torch.sort(rank, dim=2, descending=True, stable=True)[1][..., :s["most"]]
    j = x[:s["most"]]
    there = (j < n).expand(r, nkv, -1)
    kept = torch.sort(torch.where(there, order, room), dim=2)[0].clamp(max=room - 1)
    s["kept"][..., :s["most"]] = torch.where(there, kept.int(), s["kept"][..., :s["most"]])
    s["kept_weights"].zero_()
    s["kept_weights"][..., :s["most"]] = torch.where(there, w.gather(2, kept), 0.0)

    page = c["page"]
    a, h, to = torch.nonzero(there & (kept != j), as_tuple=True)  # what moves
    at = kept[a, h, to]
    src, dst = ((s["table"][a, i // page].long() * nkv + h) * page + i % page for i in (at, to))
    for cache in (s["k"], s["v"]):
        flat = cache.view(-1, c["hd"])
        flat[dst] = flat[src]
    return s["kept"], s["kept_weights"], s["k"], s["v"]


def _evict_exact(c, seed):
    s, page = _evict_inputs(c, seed), c["page"]
    w, table = s["weights"].double().cpu().numpy(), s["table"].long()
    kept, kept_w = s["kept"].cpu().numpy(), np.zeros_like(w)
    k, v = s["k"].double(), s["v"].double()
    for r, (keys, n) in enumerate(_budgets(c)):
        first = min(c["first"], n)
        last = min(c["last"], n - first)
        middle = np.arange(first, keys - last)
        slot = torch.arange(keys, device="cuda")
        pages, rows = table[r, slot // page], slot % page
        for h in range(c["nkv"]):
            chosen = middle[np.lexsort((middle, -w[r, h, middle]))[:n - first - last]]
            mine = np.sort(np.concatenate([np.arange(first), chosen, np.arange(keys - last, keys)])).astype(np.int64)
            kept[r, h, :n] = mine
            kept_w[r, h, :n] = w[r, h, mine]
            at = torch.from_numpy(mine).cuda()
            for cache in (k, v):
                cache[pages[:n], h, rows[:n]] = cache[pages[at], h, rows[at]]
    return torch.from_numpy(kept).cuda(), torch.from_numpy(kept_w).cuda(), k, v


def _evict_work(c):
    """(bytes, flops): weights, kept ones, their indices and about the share of kept rows that move (behind the first key that goes)."""
    lens = _budgets(c)
    room = (_ceil(max(n for n, _ in lens), c["page"]) + c["spare_columns"]) * c["page"]
    moved = sum(max(0, b - c["first"]) for n, b in lens if b < n)
    return (c["nkv"] * (4 * sum(n for n, _ in lens) + 4 * len(lens) * room + 4 * sum(b for _, b in lens) + 4 * SIZE[c["dtype"]] * c["hd"] * moved), 0)


# ---- release -----------------------------------------------------------------------


def _release_inputs(c, seed):
    held = [n for n, _ in _budgets(c)]
    columns = _ceil(max(held), c["page"]) + c["spare_columns"]
    ids = torch.randperm(sum(_ceil(n, c["page"]) for n in held) + 16, device="cuda", generator=_gen(seed))
    r = len(held)
    return {"keys": _ints(held), "budgets": _ints([c["budget"]] * r), "table": _table(held, c["page"], ids, columns),
            "out": (_ints([0] * r), torch.full((r * columns,), -1, dtype=torch.int32, device="cuda"), _ints([0]))}


def _release_prepare(c, seed):
    s = _release_inputs(c, seed)
    s["page"] = c["page"]
    if own:
        pa, s["enc"] = _env()
        lens, freed, counts = (_t(x) for x in s["out"])
        s["kernel"] = pa.Kernels.ReleasePages(_t(s["keys"]), _t(s["budgets"]), _t(s["table"]), page_size=c["page"], new_lens=lens,
                                              freed=freed, counts=counts)
    return s


def _release_run(s):
    page, (lens, freed, counts) = s["page"], s["out"]
    keys, x = s["keys"].long(), _arange(s["table"].shape[1])
    n = torch.minimum(keys, s["budgets"].long())
    lens.copy_(n)
    empty = (x >= ((n + page - 1) // page).unsqueeze(1)) & (x < ((keys + page - 1) // page).unsqueeze(1))
    at = torch.cumsum(empty.view(-1).long(), 0)
    counts[0] = at[-1]
    # (what stays goes where nothing has gone yet, one place behind the list, as it was)
    whole = torch.cat((freed, freed[:1]))
    whole.scatter_(0, torch.where(empty.view(-1), at - 1, freed.numel()), s["table"].view(-1))
    freed.copy_(whole[:-1])
    return s["out"]


def _release_exact(c, seed):
    s = _release_inputs(c, seed)
    table, freed, at, lens = s["table"].cpu().numpy(), s["out"][1].cpu().numpy(), 0, []
    for r, (keys, n) in enumerate(_budgets(c)):
        gone = table[r, _ceil(n, c["page"]):_ceil(keys, c["page"])]
        freed[at:at + gone.size] = gone
        at += gone.size
        lens.append(n)
    return _ints(lens), torch.from_numpy(freed).cuda(), _ints([at])


def _release_work(c):
    lens = _budgets(c)
    pages = sum(_ceil(n, c["page"]) - _ceil(b, c["page"]) for n, b in lens)
    return 4 * (3 * len(lens) + 1 + 2 * pages), 0


# ---- the cases ---------------------------------------------------------------------


def _case(kind, name=None, **sizes):
    """Requests: `chunks` of them bring chunk_lo .. chunk_hi new tokens, the others `few`."""
    base = dict(requests=1, chunks=0, chunk_lo=0, chunk_hi=0, few=1, past_lo=0, past_hi=0, page=16, lens=1, spare_columns=0)
    more = {"prefix": dict(pad=0, groups=1, alone=0, prefix_lo=0, prefix_hi=0, window=0, sinks=0), "weights": dict(pad=0, last_rows=0),
            "evict": dict(first=0, last=0)}.get(kind, {})
    return dict(({"name": name} if name else {}), work=kind, **dict(base, **dict(more, **sizes)))


def listed():
    return [
        # two answers to one prompt, sampled side by side: latency
        _case("prefix", "prefix_two", requests=2, prefix_hi=1024, past_lo=1, past_hi=200, nq=8, nkv=4, hd=256, dtype="bf16"),
        # a server's batch behind one long system prompt, a token each
        _case("prefix", "prefix_batch", requests=64, prefix_hi=8192, past_lo=50, past_hi=1500, nq=32, nkv=8, hd=128, dtype="f16",
              spare_columns=3),
        # many readers of one document
        _case("prefix", "prefix_document", requests=256, prefix_hi=16384, past_lo=20, past_hi=800, nq=16, nkv=4, hd=128, dtype="bf16", page=64),
        # three system prompts, questions that arrive whole, some requests with neither; rows padded to a captured graph's
        _case("prefix", "prefix_groups", requests=40, groups=3, alone=4, prefix_lo=900, prefix_hi=6000, chunks=3, chunk_lo=60, chunk_hi=400,
              past_hi=1000, nq=8, nkv=2, hd=128, dtype="bf16", page=32, pad=37),
        # a layer with a window and sinks: the prefix's middle has left it for some requests and not for others
        _case("prefix", "prefix_window", requests=24, prefix_hi=6000, past_lo=10, past_hi=3500, nq=8, nkv=4, hd=256, dtype="f16", window=4096,
              sinks=4),
        # a batch's step of decode: every cached key gets its share
        _case("weights", "weights_decode", requests=48, past_lo=100, past_hi=12000, nq=32, nkv=8, hd=128, dtype="f16", spare_columns=3),
        # a whole prompt, every row of it
        _case("weights", "weights_prompt", chunks=1, chunk_lo=4096, chunk_hi=4096, nq=8, nkv=4, hd=256, dtype="bf16", page=32),
        # prompts of odd lengths, seen by their last rows alone, before they are cut to a budget
        _case("weights", "weights_observed", requests=6, chunks=6, chunk_lo=700, chunk_hi=6000, last_rows=32, nq=8, nkv=2, hd=128, dtype="bf16",
              pad=11),
        # one long prompt cut to a quarter
        _case("evict", "evict_prompt", past_lo=8191, past_hi=8191, budget=2048, first=4, last=256, nkv=4, hd=256, dtype="bf16", page=32),
        # a server short of memory: many requests, some within their budget
        _case("evict", "evict_batch", requests=48, past_lo=300, past_hi=8000, budget=1000, first=4, last=128, nkv=8, hd=128, dtype="f16",
              spare_columns=3),
        # the pages that it gets back
        _case("release", "release_batch", requests=64, past_lo=300, past_hi=8000, budget=1000, spare_columns=8),
        _case("release", "release_many", requests=1500, past_lo=1, past_hi=4000, budget=777, page=32),
    ]


HEADS = [(8, 4, 256), (8, 1, 256), (32, 8, 128), (16, 4, 128), (8, 2, 128), (4, 2, 64), (6, 2, 80), (8, 2, 512)]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["prefix", "prefix", "prefix", "weights", "weights", "evict", "evict", "release"])
    nq, nkv, hd = rng.choice(HEADS)
    page, spare, lens = rng.choice([16, 32, 48, 64, 128]), rng.choice([0, 5]), rng.randrange(1 << 30)
    dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
    if kind == "prefix":
        requests = _log(rng, 2, 256)
        groups, alone = rng.choice([1, 1, 1, 2, 4]), rng.choice([0, 0, 1])
        groups = min(groups, requests - alone)
        prefix = _log(rng, 16, 16384)
        past = max(1, min(_log(rng, 1, 4000), 400000 // requests))
        chunks = rng.choice([0, 0, min(requests, rng.randint(1, 3))])
        hi = _log(rng, 2, 500) if chunks else 0
        few = rng.choice([1, 1, 1, rng.randint(2, 6)])
        tokens = requests * few + chunks * hi
        most = (8e9 if dtype == "f32" else 4e10) / (4.0 * nq * hd)  # pairs
        while tokens * (groups * prefix + past) > most and prefix > 16:
            prefix = max(16, prefix // 2)
        window = rng.choice([0, 0, 0, _log(rng, 16, 4096)])
        return _case(kind, requests=requests, groups=groups, alone=alone, prefix_lo=max(1, prefix // 3), prefix_hi=prefix, chunks=chunks,
                     chunk_lo=min(2, hi), chunk_hi=hi, few=few, past_hi=past, page=page, lens=lens, pad=rng.choice([0, 5]),
                     spare_columns=spare, nq=nq, nkv=nkv, hd=hd, dtype=dtype, window=window,
                     sinks=rng.choice([0, 1, 4, 64]) if window else 0)
    if kind == "weights":
        phase = rng.choice(["decode", "decode", "few", "prompt", "observed"])
        requests, chunks, hi, few, last = _log(rng, 1, 48), 0, 0, 1, 0
        if phase == "few":
            few = rng.randint(2, 12)
        elif phase != "decode":
            requests = chunks = rng.randint(1, 4)
            hi = _log(rng, 16, 2000)
            last = rng.choice([1, 16, 32, 64]) if phase == "observed" else 0
        past = max(1, min(_log(rng, 1, 12000), 400000000 // (requests * nkv * hd * SIZE[dtype])))
        rows = max(few, min(hi, last or hi))
        most = (4e9 if dtype == "f32" else 4e10) / (2.0 * nq * hd)
        while requests * rows * (past + max(hi, few)) > most and past > 1:
            past //= 2
        return _case(kind, requests=requests, chunks=chunks, chunk_lo=min(16, hi), chunk_hi=hi, few=few, past_hi=past, page=page, lens=lens,
                     pad=rng.choice([0, 5]), spare_columns=spare, last_rows=last, nq=nq, nkv=nkv, hd=hd, dtype=dtype)
    if kind == "evict":
        requests = _log(rng, 1, 48)
        past = max(16, min(_log(rng, 16, 16384), 200000000 // (requests * nkv * hd * SIZE[dtype])))
        return _case(kind, requests=requests, past_lo=past // 20, past_hi=past, budget=_log(rng, 1, past), first=rng.choice([0, 1, 4]),
                     last=rng.choice([0, 1, 32, 200]), page=page, lens=lens, spare_columns=spare, nkv=nkv, hd=hd, dtype=dtype)
    return _case(kind, requests=_log(rng, 1, 2048), past_hi=_log(rng, 2, 8000), budget=_log(rng, 1, 4000), page=page, lens=lens,
                 spare_columns=spare)


def _of(case, what):
    return globals()["_%s_%s" % (case["work"], what)]


def prepare(case, seed):
    return _of(case, "prepare")(case, seed) | {"work": case["work"]}


def run(state):
    if own:
        state["enc"].encode(state["kernel"])
        return {"prefix": lambda s: (s["out"], s["lse"]), "weights": lambda s: s["weights"],
                "evict": lambda s: (s["kept"], s["kept_weights"], s["k"], s["v"]), "release": lambda s: s["out"]}[state["work"]](state)
    return _of(state, "run")(state)


def work(case):
    return dict(zip(("bytes", "flops"), _of(case, "work")(case)))


def exact(case, seed):
    return _of(case, "exact")(case, seed)
