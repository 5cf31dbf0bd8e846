"""The operators of serving a batch of requests over a paged cache, as cases
that can be timed: each in a plain form (elementary torch operations) and, with
``own``, through popcorn_amd's descriptors.

* ``tables``: page tables, slots and positions of a step's new tokens from the
  requests' lengths and a list of free pages.
* ``write``: the new tokens' K and V rows into the pages of the cache.
* ``attention``: the new tokens of each request against its pages: causal,
  causal in a sliding window with a few first tokens that stay visible, or all
  keys.
* ``sample``: one token a row from the logits, by temperature, top-k, top-p and
  min-p, with the uniform random number given.

A cache is [pages, KV heads, page size, head dim]; row ``slot % page_size`` of
page ``slot // page_size`` holds the key (value) of one token.

A draw works on whole numbers: a token's weight is
``rint(2^40 exp((logit - highest) / temperature))``. Tokens rank by logit, ties
by index. Kept are the first ``top_k`` of them; of those the ones before which
less than ``top_p`` of their weight lies (the first always); of those the ones
of at least ``min_p 2^40``. The token is the first kept index whose running
weight passes ``floor(uniform x weight kept)``; -1 where nothing has weight.
"""
import math
import random

import numpy as np
import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
ONE = 1 << 40  # the heaviest token's weight
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


def _lengths(c):
    """(keys in the cache, new tokens) of each request: a case's own numbers, the same for every seed."""
    rng = random.Random(c["lens"])
    out = []
    for r in range(c["requests"]):
        past = int(math.exp(rng.uniform(math.log(c["past_lo"] + 1), math.log(c["past_hi"] + 1)))) - 1
        past = min(max(past, c["past_lo"]), c["past_hi"])
        new = rng.randint(c["chunk_lo"], c["chunk_hi"]) if r < c["chunks"] else c["few"]
        out.append((past, new))
    rng.shuffle(out)
    return out


# ---- tables ------------------------------------------------------------------------


def _tables_inputs(c, seed):
    lens, page = _lengths(c), c["page"]
    kept = [_ceil(p, page) for p, _ in lens]
    need = sum(_ceil(p + n, page) - _ceil(p, page) for p, n in lens)
    columns = max(_ceil(p + n, page) for p, n in lens) + c["spare_columns"]
    ids = torch.randperm(sum(kept) + need + 16, device="cuda", generator=_gen(seed)).to(torch.int32)
    table = torch.full((len(lens), columns), -1, dtype=torch.int32, device="cuda")
    column = torch.arange(columns, device="cuda")
    held = column < torch.tensor(kept, device="cuda").unsqueeze(1)
    table[held] = ids[:sum(kept)]
    return {"past": _ints(p for p, _ in lens), "new": _ints(n for _, n in lens), "free": ids[sum(kept):].contiguous(),
            "table": table, "tokens": sum(n for _, n in lens) + c["pad"]}


def _tables_prepare(c, seed):
    s = _tables_inputs(c, seed)
    r, t = s["past"].numel(), s["tokens"]
    s["out"] = (s["table"], *(torch.empty(n, dtype=torch.int32, device="cuda") for n in (r + 1, r, t, t, 2)))
    s["page"] = c["page"]
    if own:
        pa, s["enc"] = _env()
        d = [_t(x) for x in s["out"]]
        s["kernel"] = pa.Kernels.PageTables(_t(s["past"]), _t(s["new"]), _t(s["free"]), d[0], page_size=c["page"],
                                            query_starts=d[1], key_lens=d[2], positions=d[3], slots=d[4], counts=d[5])
    return s


def _tables_run(s):
    page, free = s["page"], s["free"].long()
    table, starts, key_lens, positions, slots, counts = s["out"]
    past, new = s["past"].long(), s["new"].long()
    held = (past + page - 1) // page
    need = (past + new + page - 1) // page - held
    ends, taken = torch.cumsum(new, 0), torch.cumsum(need, 0)
    starts[0] = 0
    starts[1:] = ends
    key_lens.copy_(past + new)
    counts[0], counts[1] = ends[-1], taken[-1]
    column = torch.arange(table.shape[1], device="cuda")
    k = column - held.unsqueeze(1)
    fresh = (k >= 0) & (k < need.unsqueeze(1))
    at = (taken - need).unsqueeze(1) + k
    table.copy_(torch.where(fresh, free[at.clamp(0, free.numel() - 1)].int(), table))
    t = torch.arange(positions.numel(), device="cuda")
    r = torch.searchsorted(ends, t, right=True).clamp(max=new.numel() - 1)
    live = t < ends[-1]
    pos = torch.where(live, past[r] + t - (ends - new)[r], 0)
    positions.copy_(pos)
    slots.copy_(torch.where(live, table[r, pos // page].long() * page + pos % page, -1))
    return s["out"]


def _tables_exact(c, seed):
    s, page = _tables_inputs(c, seed), c["page"]
    table, free = s["table"].cpu().numpy().astype(np.int64), s["free"].cpu().numpy()
    starts, key_lens, positions, slots, used = [0], [], [], [], 0
    for r, (past, new) in enumerate(_lengths(c)):
        first, last = _ceil(past, page), _ceil(past + new, page)
        table[r, first:last] = free[used:used + last - first]
        used += last - first
        pos = np.arange(past, past + new)
        positions.append(pos)
        slots.append(table[r, pos // page] * page + pos % page)
        starts.append(starts[-1] + new)
        key_lens.append(past + new)
    positions.append(np.zeros(c["pad"], np.int64))
    slots.append(np.full(c["pad"], -1))
    out = (table, starts, key_lens, np.concatenate(positions), np.concatenate(slots), [starts[-1], used])
    return tuple(torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda") for x in out)


# ---- write -------------------------------------------------------------------------


def _rows(g, shape, dtype, std=1.0):
    return torch.randn(shape, device="cuda", generator=g).mul_(std).to(TORCH[dtype])


def _write_inputs(c, seed):
    g, n = _gen(seed), c["pages"] * c["page"]
    k, v = (_rows(g, (c["tokens"], c["nkv"], c["hd"]), c["src"]) for _ in range(2))
    # whole pages in any order, as a table hands them out; the first request begins inside its page
    order = torch.randperm(c["pages"], device="cuda", generator=g)
    slots = (order.unsqueeze(1) * c["page"] + torch.arange(c["page"], device="cuda")).reshape(-1)
    slots = slots[c["page"] // 2:][:c["tokens"]] if c["prompt"] else torch.randperm(n, device="cuda", generator=g)[:c["tokens"]]
    slots = torch.cat((slots[:c["tokens"] - c["pad"]], torch.full((c["pad"],), -1, device="cuda"))).to(torch.int32)
    kc, vc = (torch.zeros(c["pages"], c["nkv"], c["page"], c["hd"], device="cuda", dtype=TORCH[c["dtype"]]) for _ in range(2))
    return {"k": k, "v": v, "slots": slots, "k_cache": kc, "v_cache": vc, "live": c["tokens"] - c["pad"]}


def _write_prepare(c, seed):
    s = _write_inputs(c, seed)
    if own:
        pa, s["enc"] = _env()
        s["kernel"] = pa.Kernels.PagedKVCacheWrite(_t(s["k"]), _t(s["v"]), _t(s["slots"]), _t(s["k_cache"]), _t(s["v_cache"]))
    s["out"] = (s["k_cache"], s["v_cache"])
    return s


def _write_run(s):
    page, live = s["k_cache"].shape[2], s["live"]
    slot = s["slots"][:live].long()
    for x, cache in ((s["k"], s["k_cache"]), (s["v"], s["v_cache"])):
        cache[slot // page, :, slot % page] = x[:live].to(cache.dtype)
    return s["out"]


def _write_exact(c, seed):
    s = _write_inputs(c, seed)
    out = []
    live = s["slots"] >= 0
    for x in (s["k"], s["v"]):
        y = torch.zeros(c["pages"] * c["page"], c["nkv"], c["hd"], dtype=torch.float64, device="cuda")
        y.index_copy_(0, s["slots"][live].long(), x[live].double())
        out.append(y.view(c["pages"], c["page"], c["nkv"], c["hd"]).transpose(1, 2).contiguous())
    return tuple(out)


# ---- attention ---------------------------------------------------------------------


def _attention_inputs(c, seed):
    g, lens, page, t = _gen(seed), _lengths(c), c["page"], c["dtype"]
    held = [_ceil(p + n, page) for p, n in lens]
    total, columns = sum(held), max(max(held), 1) + c["spare_columns"]
    tokens = sum(n for _, n in lens)
    pages = total + 3
    order = torch.randperm(pages, device="cuda", generator=g)[:total]
    q = _rows(g, (tokens + c["pad"], c["nq"], c["hd"]), t)
    k, v = (_rows(g, (pages, c["nkv"], page, c["hd"]), t) for _ in range(2))
    # what no request holds was never written: pages off the tables, rows behind the last key
    row = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    table = torch.full((len(lens), columns), -1, dtype=torch.int32, device="cuda")
    at = 0
    for r, ((p, n), h) in enumerate(zip(lens, held)):
        ids = order[at:at + h]
        table[r, :h] = ids.int()
        row.view(-1)[(ids.unsqueeze(1) * page + torch.arange(page, device="cuda")).view(-1)[:p + n]] = True
        at += h
    for x in (k, v):
        x.masked_fill_(~row.view(pages, 1, page, 1), math.nan)
    starts = [0]
    for _, n in lens:
        starts.append(starts[-1] + n)
    out = torch.full_like(q, 7.0)  # rows behind the last request's stay as they are
    return {"q": q, "k": k, "v": v, "table": table, "starts": _ints(starts), "keys": _ints(p + n for p, n in lens),
            "out": out, "lens": lens}


def _attention_prepare(c, seed):
    s = _attention_inputs(c, seed)
    s["case"] = c
    if own:
        pa, s["enc"] = _env()
        mask = {"causal": pa.AttentionMask.causal, "all": pa.AttentionMask.bidirectional,
                "window": pa.AttentionMask.causal_sliding_window(c["window"])}[c["mask"]]
        s["kernel"] = pa.Kernels.PagedAttention(_t(s["q"]), _t(s["k"]), _t(s["v"]), _t(s["table"]), _t(s["starts"]), _t(s["keys"]),
                                                _t(s["out"]), scale=c["hd"] ** -0.5, mask=mask, sinks=c["sinks"],
                                                max_query_len=max(n for _, n in s["lens"]))
    return s


def _hidden(c, past, lo, hi, keys):
    """Which of the keys the new tokens [lo, hi) of a request do not see."""
    i = torch.arange(past + lo, past + hi, device="cuda").unsqueeze(1)
    j = torch.arange(keys, device="cuda").unsqueeze(0)
    if c["mask"] == "all":
        return None
    if c["mask"] == "causal":
        return j > i
    return (j > i) | ((i - j >= c["window"]) & (j >= c["sinks"]))


def _attention_run(s):
    c, at = s["case"], 0
    nq, nkv, hd = c["nq"], c["nkv"], c["hd"]
    per = nq // nkv
    for r, (past, n) in enumerate(s["lens"]):
        if n == 0:
            continue
        keys = past + n
        ids = s["table"][r, :_ceil(keys, c["page"])].long()
        k, v = (x[ids].transpose(1, 2).reshape(-1, nkv, hd)[:keys].permute(1, 0, 2).float().contiguous() for x in (s["k"], s["v"]))
        for lo in range(0, n, 512):
            hi = min(n, lo + 512)
            q = s["q"][at + lo:at + hi].float().view(hi - lo, nkv, per, hd).permute(1, 0, 2, 3).reshape(nkv, -1, hd)
            a = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(hd ** -0.5).view(nkv, hi - lo, per, keys)
            hide = _hidden(c, past, lo, hi, keys)
            if hide is not None:
                a.masked_fill_(hide.view(1, hi - lo, 1, keys), -math.inf)
            a = torch.exp_(a.sub_(a.amax(-1, keepdim=True)))
            a = a.div_(a.sum(-1, keepdim=True))
            o = torch.matmul(a.view(nkv, -1, keys), v).view(nkv, hi - lo, per, hd)
            s["out"][at + lo:at + hi] = o.permute(1, 0, 2, 3).reshape(hi - lo, nq, hd).to(s["out"].dtype)
        at += n
    return s["out"]


def _attention_exact(c, seed):
    s = _attention_inputs(c, seed)
    out, at = s["out"].double(), 0
    nq, nkv, hd, page = c["nq"], c["nkv"], c["hd"], c["page"]
    for r, (past, n) in enumerate(s["lens"]):
        keys = past + n
        pages = s["table"][r].tolist()
        k = torch.cat([s["k"][p] for p in pages[:_ceil(keys, page)]] or [s["k"][0, :, :0]], 1)[:, :keys].double()
        v = torch.cat([s["v"][p] for p in pages[:_ceil(keys, page)]] or [s["v"][0, :, :0]], 1)[:, :keys].double()
        for h in range(nq):
            kt = k[h // (nq // nkv)].t().contiguous()
            for lo in range(0, n, 1024):
                hi = min(n, lo + 1024)
                a = (s["q"][at + lo:at + hi, h].double() @ kt) / math.sqrt(hd)
                hide = _hidden(c, past, lo, hi, keys)
                if hide is not None:
                    a.masked_fill_(hide, -math.inf)
                out[at + lo:at + hi, h] = torch.softmax(a, -1) @ v[h // (nq // nkv)]
        at += n
    return out


def _seen(c, past, n):
    """(pairs that the mask lets through, keys that some new token sees) of one request and head."""
    pairs, w, s = 0, c["window"], c["sinks"]
    if c["mask"] == "all":
        return n * (past + n), (past + n if n else 0)
    if c["mask"] == "causal":
        return n * past + n * (n + 1) // 2, (past + n if n else 0)
    for i in range(past, past + n):
        pairs += min(i + 1, w) + min(s, max(i + 1 - w, 0))
    first = max(past - w + 1, 0)
    return pairs, (past + n - first + min(s, first) if n else 0)


# ---- sample ------------------------------------------------------------------------


def _sample_inputs(c, seed):
    g, rows, v = _gen(seed), c["rows"], c["vocab"]
    x = torch.randn((rows, v), device="cuda", generator=g).mul_(c["spread"])
    x += 4.0 * c["spread"] * (torch.rand((rows, v), device="cuda", generator=g) < 20.0 / v)  # a few likely tokens
    x.masked_fill_(torch.rand((1, v), device="cuda", generator=g) < 0.01, -math.inf)  # tokens that are never to be drawn
    x = x.to(TORCH[c["dtype"]])

    def each(value, spread):  # requests differ in what they ask for
        return (value * (1.0 + spread * (torch.rand(rows, device="cuda", generator=g) - 0.5))).float()

    s = {"logits": x, "uniforms": torch.rand(rows, device="cuda", generator=g)}
    s["temperature"] = each(c["temperature"], 0.4) if c["temperature"] else None
    s["top_k"] = each(c["top_k"], 0.4).int().clamp(min=1) if c["top_k"] else None
    s["top_p"] = each(c["top_p"], 0.1).clamp(max=1.0) if c["top_p"] else None
    s["min_p"] = each(c["min_p"], 0.4) if c["min_p"] else None
    return s


def _sample_prepare(c, seed):
    s = _sample_inputs(c, seed)
    s["out"] = torch.empty(c["rows"], dtype=torch.int32, device="cuda")
    if own:
        pa, s["enc"] = _env()
        options = {n: _t(s[n]) for n in ("temperature", "top_k", "top_p", "min_p") if s[n] is not None}
        s["kernel"] = pa.Kernels.Sample(_t(s["logits"]), _t(s["uniforms"]), _t(s["out"]), **options)
    return s


def _share(u, z):
    """floor(u z) and whether something is left over, for u in [0, 1) to 31 bits and whole z below 2^62."""
    m = (u.double() * 2.0 ** 31).long()
    low = (z & 0x7fffffff) * m
    return (z >> 31) * m + (low >> 31), (low & 0x7fffffff) != 0


def _sample_run(s):
    x = s["logits"].double()
    value, index = torch.sort(x, dim=1, descending=True, stable=True)
    top = value[:, :1]
    t = 1.0 if s["temperature"] is None else s["temperature"].double().unsqueeze(1)
    w = torch.round(torch.exp(torch.where(value == top, 0.0, (value - top) / t)) * ONE).long()
    if s["top_k"] is not None:
        w *= torch.arange(x.shape[1], device="cuda") < s["top_k"].unsqueeze(1)
    if s["top_p"] is not None:
        run = torch.cumsum(w, 1)
        limit, more = _share(s["top_p"].clamp(0, 1).unsqueeze(1), run[:, -1:])
        keep = (run - w < limit + more) | (s["top_p"].unsqueeze(1) >= 1)
        keep[:, 0] = True
        w *= keep
    if s["min_p"] is not None:
        w *= w.double() >= s["min_p"].double().unsqueeze(1) * ONE
    run = torch.cumsum(torch.zeros_like(w).scatter_(1, index, w), 1)
    target, _ = _share(s["uniforms"].unsqueeze(1), run[:, -1:])
    first = torch.searchsorted(run, target, right=True).squeeze(1)
    s["out"].copy_(torch.where(run[:, -1] > 0, first, -1))
    return s["out"]


def _sample_exact(c, seed):
    s = {n: v.cpu().double().numpy() if v is not None else None for n, v in _sample_inputs(c, seed).items()}
    out = []
    for r, x in enumerate(s["logits"]):
        with np.errstate(invalid="ignore"):
            d = np.where(x == x.max(), 0.0, (x - x.max()) / (1.0 if s["temperature"] is None else s["temperature"][r]))
        w = np.rint(np.exp(d) * ONE).astype(np.int64)
        order = np.lexsort((np.arange(x.size), -x))
        kept = order if s["top_k"] is None else order[:int(s["top_k"][r])]
        if s["top_p"] is not None and s["top_p"][r] < 1.0:
            before = np.cumsum(w[kept]) - w[kept]
            part, whole = (int(s["top_p"][r] * 2 ** 31)) * int(w[kept].sum()), 2 ** 31
            kept = kept[(before < -(-part // whole)) | (np.arange(kept.size) == 0)]
        if s["min_p"] is not None:
            kept = kept[w[kept] >= s["min_p"][r] * ONE]
        kept = np.sort(kept)
        run = np.cumsum(w[kept])
        target = int(s["uniforms"][r] * 2 ** 31) * int(run[-1]) >> 31
        out.append(int(kept[np.searchsorted(run, target, side="right")]))
    return torch.tensor(out, dtype=torch.int32, device="cuda")


# ---- the cases ---------------------------------------------------------------------


def _case(kind, name=None, **sizes):
    return dict(({"name": name} if name else {}), work=kind, **sizes)


def _batch(kind, name=None, **sizes):
    """Requests: `chunks` of them bring chunk_lo .. chunk_hi new tokens, the others `few`."""
    base = dict(requests=1, chunks=0, chunk_lo=0, chunk_hi=0, few=1, past_lo=0, past_hi=0, page=16, lens=1, pad=0, spare_columns=0)
    return _case(kind, name, **dict(base, **sizes))


def listed():
    causal = dict(mask="causal", window=0, sinks=0)
    return [
        # a step of decode for a server's 256 requests: one new token each, a page now and then
        _batch("tables", "tables_decode", requests=256, past_lo=30, past_hi=8000, spare_columns=8),
        # many short prompts admitted in one step, the token count padded to a captured graph's
        _batch("tables", "tables_prompts", requests=48, chunks=40, chunk_lo=1, chunk_hi=1500, past_hi=700, pad=77, page=32),
        # one token of each of 64 requests, f16
        _case("write", "write_decode", tokens=64, pad=3, nkv=8, hd=128, page=16, pages=2048, src="f16", dtype="f16", prompt=False),
        # a long prompt's rows, bf16, as the RoPE and the norm leave them
        _case("write", "write_prompt", tokens=8000, pad=0, nkv=4, hd=256, page=32, pages=300, src="bf16", dtype="bf16", prompt=True),
        # a single stream of chat at 4096 tokens: latency
        _batch("attention", "attention_decode_one", nq=8, nkv=4, hd=256, dtype="bf16", past_lo=4096, past_hi=4096,
               spare_columns=16, **causal),
        # a server's batch: 64 requests of very different lengths, one token each
        _batch("attention", "attention_decode_batch", requests=64, nq=32, nkv=8, hd=128, dtype="f16", past_lo=100, past_hi=16000,
               spare_columns=3, **causal),
        # prompts' chunks among requests that decode, in one call with padded rows
        _batch("attention", "attention_mixed", requests=24, chunks=4, chunk_lo=100, chunk_hi=700, nq=16, nkv=4, hd=128, dtype="bf16",
               past_lo=0, past_hi=6000, page=64, pad=37, **causal),
        # a long prompt's chunk behind what the cache holds already
        _batch("attention", "attention_chunk", chunks=1, chunk_lo=2048, chunk_hi=2048, nq=8, nkv=4, hd=256, dtype="f16",
               past_lo=8192, past_hi=8192, page=32, **causal),
        # a layer with a window and sinks: long conversations, one of them reading a document
        _batch("attention", "attention_window", requests=12, chunks=1, chunk_lo=777, chunk_hi=777, nq=8, nkv=4, hd=256, dtype="bf16",
               past_lo=2000, past_hi=32000, page=16, mask="window", window=4096, sinks=4),
        # one stream's next token
        _case("sample", "sample_one", rows=1, vocab=256000, dtype="f32", spread=2.5, temperature=0.8, top_k=50, top_p=0.95, min_p=0),
        # a server's batch, nucleus only: the kept set is as large as the distribution makes it
        _case("sample", "sample_nucleus", rows=64, vocab=256000, dtype="bf16", spread=1.5, temperature=1.0, top_k=0, top_p=0.9,
              min_p=0),
        # every option at once, an odd vocabulary, f16
        _case("sample", "sample_all", rows=33, vocab=50257, dtype="f16", spread=2.0, temperature=1.2, top_k=400, top_p=0.92,
              min_p=0.02),
    ]


HEADS = [(8, 4, 256), (8, 1, 256), (32, 8, 128), (16, 4, 128), (8, 2, 128), (4, 2, 64), (6, 2, 80), (8, 2, 512)]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["tables", "write", "attention", "attention", "attention", "sample", "sample"])
    lens = rng.randrange(1 << 30)
    if kind == "tables":
        requests = _log(rng, 1, 2048)
        hi = _log(rng, 1, max(1, min(4096, 40000 // requests)))
        return _batch(kind, requests=requests, chunks=rng.randint(0, requests), chunk_lo=0, chunk_hi=hi, few=rng.choice([0, 1, 1, 4]),
                      past_hi=_log(rng, 1, 16384), page=rng.choice([16, 32, 48, 64, 128, 256]), lens=lens, pad=rng.choice([0, 1, 61]),
                      spare_columns=rng.choice([0, 7]))
    if kind == "write":
        _, nkv, hd = rng.choice(HEADS)
        tokens, page = _log(rng, 1, 16384), rng.choice([16, 32, 48, 64, 128, 256])
        src, dtype = rng.choice([("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("f32", "bf16")])
        return _case(kind, tokens=tokens, pad=rng.choice([0, tokens // 9]), nkv=nkv, hd=hd, page=page,
                     pages=_ceil(tokens, page) + rng.randint(1, 40), src=src, dtype=dtype, prompt=rng.random() < 0.5)
    if kind == "attention":
        nq, nkv, hd = rng.choice(HEADS)
        dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
        phase = rng.choice(["decode", "few", "chunk", "mixed"])
        requests, chunks, lo, hi, few = _log(rng, 1, 64), 0, 0, 0, 1
        if phase == "few":
            few = rng.randint(2, 12)
        elif phase == "chunk":
            requests = chunks = rng.randint(1, 4)
            lo, hi = 17, _log(rng, 32, 2048)
            lo = min(lo, hi)
        elif phase == "mixed":
            requests, chunks, lo, hi = rng.randint(4, 40), rng.randint(1, 3), 1, _log(rng, 16, 700)
        past = _log(rng, 1, 32768)
        past = max(1, min(past, 400000000 // (requests * nkv * hd * SIZE[dtype])))  # bytes of K
        most = (4e9 if dtype == "f32" else 100e9) / (4.0 * nq * hd)  # pairs
        while (chunks * hi + (requests - chunks) * few) * (past + max(hi, few)) > most and past > 1:
            past //= 2
        mask = rng.choice(["causal", "causal", "causal", "window", "all"])
        window = _log(rng, 16, 4096) if mask == "window" else 0
        return _batch(kind, requests=requests, chunks=chunks, chunk_lo=lo, chunk_hi=hi, few=few, nq=nq, nkv=nkv, hd=hd, dtype=dtype,
                      past_lo=0, past_hi=past, page=rng.choice([16, 32, 48, 64, 128, 256]), lens=lens, pad=rng.choice([0, 5]),
                      spare_columns=rng.choice([0, 9]), mask=mask, window=window,
                      sinks=rng.choice([0, 1, 4, 64]) if mask == "window" else 0)
    rows, vocab = _log(rng, 1, 64), _log(rng, 1000, 256000)
    return _case(kind, rows=rows, vocab=vocab, dtype=rng.choice(["f32", "f16", "bf16"]), spread=rng.uniform(0.5, 4.0),
                 temperature=rng.choice([0, rng.uniform(0.3, 2.0)]), top_k=rng.choice([0, 0, _log(rng, 1, 2000)]),
                 top_p=rng.choice([0, rng.uniform(0.3, 0.99)]), min_p=rng.choice([0, 0, rng.uniform(0.001, 0.3)]))


def prepare(case, seed):
    return {"tables": _tables_prepare, "write": _write_prepare, "attention": _attention_prepare,
            "sample": _sample_prepare}[case["work"]](case, seed) | {"work": case["work"]}


def run(state):
    if own:
        state["enc"].encode(state["kernel"])
        return state["out"]
    return {"tables": _tables_run, "write": _write_run, "attention": _attention_run, "sample": _sample_run}[state["work"]](state)


def work(case):
    c = case
    if c["work"] == "tables":
        lens, page = _lengths(c), c["page"]
        pages = sum(_ceil(p + n, page) - _ceil(p, page) for p, n in lens)
        tokens = sum(n for _, n in lens) + c["pad"]
        return {"bytes": 4 * (4 * len(lens) + 3 + 2 * pages + 2 * tokens), "flops": 0}
    if c["work"] == "write":
        n = 2 * (c["tokens"] - c["pad"]) * c["nkv"] * c["hd"]
        return {"bytes": n * (SIZE[c["src"]] + SIZE[c["dtype"]]) + 4 * c["tokens"], "flops": 0}
    if c["work"] == "attention":
        e, lens = SIZE[c["dtype"]], _lengths(c)
        pairs, keys = (sum(x) for x in zip(*(_seen(c, p, n) for p, n in lens)))
        tokens = sum(n for _, n in lens)
        return {"bytes": e * c["hd"] * (2 * c["nq"] * tokens + 2 * c["nkv"] * keys), "flops": 4.0 * c["nq"] * c["hd"] * pairs}
    return {"bytes": c["rows"] * (c["vocab"] * SIZE[c["dtype"]] + 4), "flops": 0}


def exact(case, seed):
    if case["work"] == "attention" and work(case)["flops"] > 4e11:
        return None
    return {"tables": _tables_exact, "write": _write_exact, "attention": _attention_exact, "sample": _sample_exact}[case["work"]](case, seed)
