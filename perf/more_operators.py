"""The operators of a serving step: what they compute, in elementary torch operations, and the calls of the framework.

  plan    pages for new tokens from a stack of free ones, block tables, positions and cache slots, from request lengths
  write   rotary embedding of the new tokens' q and k, k and v stored in their pages
  decode  attention of one new token per request over the paged cache, with a window and a cap on the scores where wanted
  sample  a token per row of logits from a given random number: temperature, top-k, top-p, min-p

The heads are the sky-1 model's (16 of 128, 16 or 4 for keys and values) and generic ones around them, the vocabulary is its 32768
and larger ones.  Queries and keys are N(0, 1) with a few keys that a query leans towards, pages lie in the cache in random order,
logits are N(0, 2.5) with a few high ones.  Lengths depend on the case alone; the seed decides whose they are.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


def listed():
    return [
        # One request in its first pages: latency.
        _decode("decode_1", batch=1, heads=16, kv_heads=16, dim=128, page=16, longest=777),
        # A serving batch of the LM, contexts of up to its double training length.
        _decode("decode_64", batch=64, heads=16, kv_heads=16, dim=128, page=16, longest=4096),
        # Two long documents, grouped heads.
        _decode("decode_long", batch=2, heads=32, kv_heads=4, dim=128, page=64, longest=131072),
        # Short heads in odd groups, odd pages, a window and capped scores.
        _decode("decode_window", batch=37, heads=24, kv_heads=2, dim=64, page=7, longest=5000, window=1000, softcap=30.0),
        # One step of a small batch.
        _write("write_8", tokens=8, heads=16, kv_heads=16, dim=128, page=16),
        # A prompt batch as large as the training step.
        _write("write_16384", tokens=16384, heads=16, kv_heads=16, dim=128, page=16),
        # A ragged prompt batch with padding, grouped heads, odd pages.
        _write("write_odd", tokens=4003, heads=16, kv_heads=4, dim=128, page=33, padding=0.1),
        # The plan of one step: a new token per request.
        _plan("plan_64", requests=64, page=16, new=1, longest=4096),
        # Many requests, some with a prompt to read in, some idle; not all get their pages.
        _plan("plan_1999", requests=1999, page=16, new=64, longest=2048, short=True),
        # One request's next token.
        _sample("sample_1", rows=1, vocab=32768, kinds="kp"),
        # A serving batch in which every request has its own settings.
        _sample("sample_256", rows=256, vocab=32768, kinds="mixed"),
        # A long vocabulary in f32, nucleus sampling without a limit on the count.
        _sample("sample_wide", rows=48, vocab=150001, kinds="p", dtype="f32"),
    ]


def _named(name, c):
    return {"name": name, **c} if name else c


def _decode(name, batch, heads, kv_heads, dim, page, longest, window=0, softcap=0.0):
    return _named(name, {"op": "decode", "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
                         "longest": longest, "window": window, "softcap": softcap})


def _write(name, tokens, heads, kv_heads, dim, page, padding=0.0):
    return _named(name, {"op": "write", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
                         "padding": padding})


def _plan(name, requests, page, new, longest, short=False):
    """new: tokens that a request brings at most; short: the free pages do not suffice for all."""
    return _named(name, {"op": "plan", "requests": requests, "page": page, "new": new, "longest": longest, "short": short})


def _sample(name, rows, vocab, kinds, dtype="bf16"):
    """kinds: which of top-k, top-p, min-p and greedy rows there are; "mixed": all, row by row."""
    return _named(name, {"op": "sample", "rows": rows, "vocab": vocab, "kinds": kinds, "dtype": dtype})


def draw(rng: random.Random):
    def log_uniform(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("decode", "decode", "write", "plan", "sample", "sample"))
    page = rng.choice((16, 16, 32, 64, 128, log_uniform(1, 256)))
    dim = rng.choice((64, 128, 128))
    kv_heads = rng.choice((1, 2, 3, 4, 8, 16))
    heads = kv_heads * rng.choice((1, 1, 2, 3, 4, 7, 8, 12, 16))
    if op == "decode":
        batch = log_uniform(1, 256)
        most = (1 << 28) // (batch * kv_heads * dim)
        longest = log_uniform(1, max(2, min(131072, most)))
        return _decode(None, batch, heads, kv_heads, dim, page, longest,
                       window=rng.choice((0, 0, log_uniform(1, 8192))), softcap=rng.choice((0.0, 0.0, round(rng.uniform(5, 60), 1))))
    if op == "write":
        return _write(None, log_uniform(1, max(2, min(16384, (1 << 26) // ((heads + 2 * kv_heads) * dim)))), heads, kv_heads, dim,
                      page, padding=rng.choice((0.0, 0.0, 0.2)))
    if op == "plan":
        return _plan(None, log_uniform(1, 4096), page, rng.choice((1, 1, log_uniform(1, 64))), log_uniform(1, 4096),
                     short=rng.random() < 0.3)
    vocab = log_uniform(100, 200000)
    return _sample(None, log_uniform(1, max(2, min(512, (1 << 23) // vocab))), vocab, rng.choice(("kp", "p", "k", "m", "none", "mixed")),
                   dtype=rng.choice(("bf16", "f32")))


# ------------------------------------------------------------------------------------------ inputs
def _spread(case):
    """The lengths of a decode case: from the longest down to a twentieth of it, evenly."""
    b, top = case["batch"], case["longest"]
    return [max(1, round(top * (1 - 0.95 * i / b))) for i in range(b)]


def _pages(tokens, page):
    return -(-tokens // page)


def _decode_inputs(case, on):
    b, h, hkv, d, page = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    lens = torch.tensor(_spread(case), device="cuda")[torch.randperm(b, **on)]
    used = (lens + page - 1) // page
    width, total = _pages(case["longest"], page), sum(_pages(n, page) for n in _spread(case))
    pages = total + 5
    take = torch.randperm(pages, **on)[:total]
    before = used.cumsum(0) - used
    at = torch.arange(width, device="cuda")
    live = at[None, :] < used[:, None]
    block_table = torch.where(live, take[torch.where(live, before[:, None] + at[None, :], 0)], -1)
    k_cache = torch.randn(pages, page, hkv, d, dtype=BF16, **on)
    v_cache = torch.randn(pages, page, hkv, d, dtype=BF16, **on)
    # a key of each request that its queries lean towards
    q = torch.randn(b, h, d, **on)
    j = (torch.rand(b, **on) * lens).long()
    lean = k_cache[block_table[torch.arange(b, device="cuda"), j // page], j % page].float()
    q = q + 0.5 * lean.repeat_interleave(h // hkv, 1)
    return {"q": q.to(BF16), "k_cache": k_cache, "v_cache": v_cache, "block_table": block_table.to(I32), "seq_lens": lens.to(I32)}


def _rope_table(positions, dim):
    half = dim // 2
    inv_freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") * 2.0 / dim)
    ang = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv_freq[None, :]
    return torch.cat([ang.cos(), ang.sin()], dim=1).to(F32)


def _write_inputs(case, on):
    t, h, hkv, d, page = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    qkv = torch.randn(t, h + 2 * hkv, d, dtype=BF16, **on)
    pages = _pages(t, page) + 3
    runs = torch.randperm(pages, **on)  # tokens fill one page after another, in random order of the pages
    i = torch.arange(t, device="cuda")
    slots = runs[i // page] * page + i % page
    live = i < t - int(case["padding"] * t)
    table = _rope_table(4096, d)
    positions = (i + torch.randint(0, 4096, (1,), **on)) % 4096
    return {"q": qkv[:, :h], "k": qkv[:, h:h + hkv], "v": qkv[:, h + hkv:], "table": table,
            "positions": torch.where(live, positions, -1).to(I32), "slots": torch.where(live, slots, -1).to(I32),
            "k_cache": torch.zeros(pages, page, hkv, d, dtype=BF16, device="cuda"),
            "v_cache": torch.zeros(pages, page, hkv, d, dtype=BF16, device="cuda")}


def _plan_lengths(case):
    """(cached, added) per request: contexts of every length, every seventh request idle where prompts are read in."""
    n, top, new = case["requests"], case["longest"], case["new"]
    cached = [(i * 7919) % (top + 1) for i in range(n)]
    added = [1 if new == 1 else (0 if i % 7 == 3 else 1 + (i * 104729) % new) for i in range(n)]
    return cached, added


def _plan_counts(case):
    """(rows, width, pages in use, pages wanted) of a plan case."""
    cached, added = _plan_lengths(case)
    page = case["page"]
    in_use = sum(_pages(c, page) for c in cached)
    wanted = sum(_pages(c + a, page) - _pages(c, page) for c, a in zip(cached, added))
    return sum(added), _pages(case["longest"] + case["new"], page), in_use, wanted


def _plan_inputs(case, on):
    page = case["page"]
    rows, width, in_use, wanted = _plan_counts(case)
    cached, added = _plan_lengths(case)
    order = torch.randperm(len(cached), **on)
    cached, added = torch.tensor(cached, device="cuda")[order], torch.tensor(added, device="cuda")[order]
    free = wanted // 2 if case["short"] else wanted + 9
    pages = in_use + free
    shuffled = torch.randperm(pages, **on)
    used = (cached + page - 1) // page
    before = used.cumsum(0) - used
    at = torch.arange(width, device="cuda")
    live = at[None, :] < used[:, None]
    table = torch.where(live, shuffled[torch.where(live, before[:, None] + at[None, :], 0)], -1)
    stack = torch.full((pages,), -1, device="cuda")
    stack[:free] = shuffled[in_use:]
    return {"cached": cached.to(I32), "added": added.to(I32), "block_table": table.to(I32), "free_pages": stack.to(I32),
            "free_count": torch.tensor([free], dtype=I32, device="cuda"), "rows": rows + 7, "pages": pages}


def _sample_inputs(case, on):
    r, v, kinds = case["rows"], case["vocab"], case["kinds"]
    z = torch.randn(r, v, **on).mul_(2.5)
    best = torch.randint(0, v, (r, 40), **on)
    z.scatter_add_(1, best, torch.rand(r, 40, **on).mul_(8.0))
    z[torch.rand(r, v, **on) < 0.01] = -torch.inf  # tokens that a grammar does not allow here
    z[:, v // 2] = 1.0
    i = torch.arange(r, device="cuda")
    which = lambda name, at: (i % 6 == at) | (i % 6 == 5) if kinds == "mixed" else torch.full_like(i, name in kinds, dtype=torch.bool)
    k = torch.where(which("k", 0), torch.randint(1, min(v, 200) + 1, (r,), **on), 0)
    p = torch.where(which("p", 1), 0.5 + 0.49 * torch.rand(r, **on), 1.0)
    m = torch.where(which("m", 2), 0.02 + 0.1 * torch.rand(r, **on), 0.0)
    t = 0.6 + 0.7 * torch.rand(r, **on)
    if kinds == "mixed":
        t = torch.where(i % 6 == 3, 0.0, t)  # greedy
    return {"logits": z.to(BF16 if case["dtype"] == "bf16" else F32), "uniform": torch.rand(r, **on), "temperature": t,
            "top_k": k.to(I32), "top_p": p, "min_p": m}


def _inputs(case, seed):
    on = dict(generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")
    make = {"decode": _decode_inputs, "write": _write_inputs, "plan": _plan_inputs, "sample": _sample_inputs}[case["op"]]
    return {"case": case, **make(case, on)}


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        import cleanlm_b200 as cdl

        s["serve"] = cdl.serve
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(s):
    if own:
        return {"decode": _own_decode, "write": _own_write, "plan": _own_plan, "sample": _own_sample}[s["case"]["op"]](s)
    return {"decode": _plain_decode, "write": _plain_write, "plan": _plain_plan, "sample": _plain_sample}[s["case"]["op"]](s)


def _own_decode(s):
    serve, case = s["serve"], s["case"]
    o = serve.attention_decode(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["seq_lens"],
                               serve.AttentionDecodeOpts(window=case["window"], softcap=case["softcap"]), lse=True)
    return {"out": o.out, "lse": o.lse}


def _own_write(s):
    o = s["serve"].cache_write(s["k"], s["v"], s["slots"], s["k_cache"], s["v_cache"], q=s["q"], table=s["table"],
                               positions=s["positions"])
    return {"q": o.q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_plan(s):
    serve = s["serve"]
    o = serve.cache_plan(s["cached"], s["added"], s["block_table"], s["free_pages"], s["free_count"],
                         serve.CachePlanOpts(page_size=s["case"]["page"], pages=s["pages"], rows=s["rows"]))
    return {"seq_lens": o.seq_lens, "cu_seqlens": o.cu_seqlens, "positions": o.positions, "slots": o.slots,
            "free_left": o.free_left, "block_table": s["block_table"]}


def _own_sample(s):
    serve = s["serve"]
    o = serve.sample(s["logits"], s["uniform"], serve.SampleOpts(temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                                                 min_p=s["min_p"]))
    return {"token": o.token, "logprob": o.logprob}


def _plain_decode(s):
    case = s["case"]
    h, hkv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    b, lens = s["q"].shape[0], s["seq_lens"].long()
    at = torch.arange(s["block_table"].shape[1] * page, device="cuda")
    sees = at[None, :] < lens[:, None]
    if case["window"]:
        sees &= at[None, :] >= lens[:, None] - case["window"]
    pages = s["block_table"].long().clamp(min=0)
    k = s["k_cache"][pages].float().reshape(b, -1, hkv, d).permute(0, 2, 3, 1)
    v = s["v_cache"][pages].float().reshape(b, -1, hkv, d).permute(0, 2, 1, 3)
    q = s["q"].float().reshape(b, hkv, h // hkv, d)
    x = (q @ k) / math.sqrt(d)
    if case["softcap"]:
        x = case["softcap"] * torch.tanh(x / case["softcap"])
    x = torch.where(sees[:, None, None, :], x, -torch.inf)
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    total = e.sum(-1, keepdim=True)
    out = (e @ torch.where(sees[:, None, :, None], v, 0.0)) / total
    return {"out": out.reshape(b, h, d).to(BF16), "lse": (m + total.log()).reshape(b, h)}


def _rotated(x, table, positions):
    half = x.shape[2] // 2
    live = (positions >= 0)[:, None, None]
    cs = table[positions.long().clamp(min=0)][:, None, :]
    cos, sin = cs[..., :half], cs[..., half:]
    lo, hi = x[..., :half].float(), x[..., half:].float()
    turned = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)
    return torch.where(live, turned, x.float()).to(BF16)


def _plain_write(s):
    hkv, d = s["case"]["kv_heads"], s["case"]["dim"]
    slots = s["slots"].long()
    live = slots >= 0
    slots = torch.where(live, slots, slots[0])  # the padding stores the first token once more
    k = _rotated(s["k"], s["table"], s["positions"])
    s["k_cache"].view(-1, hkv, d)[slots] = torch.where(live[:, None, None], k, k[:1])
    s["v_cache"].view(-1, hkv, d)[slots] = torch.where(live[:, None, None], s["v"], s["v"][:1])
    return {"q": _rotated(s["q"], s["table"], s["positions"]), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_plan(s):
    page, rows, table = s["case"]["page"], s["rows"], s["block_table"]
    c, a, free = s["cached"].long(), s["added"].long(), s["free_count"].long()
    ends = a.cumsum(0)
    old, width = (c + page - 1) // page, table.shape[1]
    fits = (c + a <= width * page) & (ends <= rows)
    need = torch.where(fits, (c + a + page - 1) // page - old, 0)
    upto = need.cumsum(0)
    served = fits & ((need == 0) | (upto <= free))
    left = free - torch.where(served & (need > 0), upto, 0).amax()
    # the new entries of the block tables
    i = torch.arange(width, device="cuda")
    j = i[None, :] - old[:, None]
    fresh = served[:, None] & (j >= 0) & (j < need[:, None])
    took = free - 1 - ((upto - need)[:, None] + j)
    table.copy_(torch.where(fresh, s["free_pages"][torch.where(fresh, took, 0)], table))
    # the rows of the batch
    r = torch.arange(rows, device="cuda")
    of = torch.searchsorted(ends, r, right=True)
    live = of < len(c)
    of = torch.where(live, of, 0)
    position = c[of] + r - (ends - a)[of]
    page_at = table[of, torch.where(live & served[of], position // page, 0)].long()
    slot = torch.where(live & served[of] & (page_at >= 0) & (page_at < s["pages"]), page_at * page + position % page, -1)
    cu = torch.cat([torch.zeros_like(ends[:1]), ends.clamp(max=rows)])
    return {"seq_lens": (c + torch.where(served, a, 0)).to(I32), "cu_seqlens": cu.to(I32),
            "positions": torch.where(live, position, -1).to(I32), "slots": slot.to(I32), "free_left": left.to(I32),
            "block_table": table}


def _plain_sample(s):
    z = s["logits"].double()
    v = z.shape[1]
    greedy = ~(s["temperature"] > 0)
    t = torch.where(greedy, 1.0, s["temperature"]).double()[:, None]
    order_z, order = z.sort(dim=1, descending=True, stable=True)
    w = ((order_z - order_z[:, :1]) / t).exp()
    mass = w.cumsum(1)
    k = torch.where(s["top_k"] > 0, s["top_k"], v).long().clamp(max=v)[:, None]
    p = s["top_p"].double()[:, None]
    n_p = torch.where(p < 1, (mass < p * mass.gather(1, k - 1)).sum(1, keepdim=True) + 1, v)
    n_m = (w >= s["min_p"].double()[:, None]).sum(1, keepdim=True)
    n = torch.minimum(torch.minimum(k, n_p), n_m).clamp(min=1)
    n = torch.where(greedy[:, None], 1, n)
    keep = torch.arange(v, device="cuda")[None, :] < n
    weight = torch.zeros_like(z).scatter_(1, order, torch.where(keep, w, 0.0))
    upto = weight.cumsum(1)
    total = mass.gather(1, n - 1)
    token = (upto <= s["uniform"].double()[:, None] * upto[:, -1:]).sum(1, keepdim=True).clamp(max=v - 1)
    logprob = (z.gather(1, token) - order_z[:, :1]) / t - total.log()
    return {"token": token[:, 0].to(I32), "logprob": torch.where(greedy, 0.0, logprob[:, 0]).float()}


# ------------------------------------------------------------------------------------------ what it takes
def work(case):
    if case["op"] == "decode":
        b, h, hkv, d, page = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["page"]
        keys = sum(min(n, case["window"] or n) for n in _spread(case))
        return {"bytes": 4.0 * keys * hkv * d + 4.0 * b * h * d + 4.0 * b * h + 4.0 * b + 4.0 * (keys // page + b),
                "flops": 4.0 * keys * h * d}
    if case["op"] == "write":
        t, h, hkv, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        live = t - int(case["padding"] * t)
        return {"bytes": 4.0 * (t * h + live * 2 * hkv) * d + 4.0 * min(live, 4096) * d + 8.0 * t,
                "flops": 3.0 * live * (h + hkv) * d}
    if case["op"] == "plan":
        rows, _, _, wanted = _plan_counts(case)
        return {"bytes": 16.0 * case["requests"] + 8.0 * wanted + 8.0 * rows + 4.0 * _pages(rows, case["page"]),
                "flops": float(8 * case["requests"] + 4 * rows)}
    r, v = case["rows"], case["vocab"]
    return {"bytes": float(r * v * (2 if case["dtype"] == "bf16" else 4) + 28 * r), "flops": 4.0 * r * v}


# ------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    f64 = dict(dtype=torch.float64, device="cuda")
    if case["op"] == "decode":
        b, h, hkv, d, page = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["page"]
        out, lse = torch.zeros(b, h, d, **f64), torch.zeros(b, h, **f64)
        for i, n in enumerate(s["seq_lens"].tolist()):
            pages = s["block_table"][i, :_pages(n, page)].long()
            first = max(0, n - case["window"]) if case["window"] else 0
            k = s["k_cache"][pages].flatten(0, 1)[first:n].double().repeat_interleave(h // hkv, 1)
            v = s["v_cache"][pages].flatten(0, 1)[first:n].double().repeat_interleave(h // hkv, 1)
            x = (k * s["q"][i].double()[None]).sum(2) * d ** -0.5  # [keys, heads]
            if case["softcap"]:
                x = torch.tanh(x / case["softcap"]) * case["softcap"]
            lse[i] = torch.logsumexp(x, 0)
            out[i] = ((x - lse[i]).exp()[..., None] * v).sum(0)
        return {"out": out, "lse": lse}
    if case["op"] == "write":
        t, h, hkv, d, page = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["page"]
        turn = torch.complex(s["table"][:, :d // 2].double(), s["table"][:, d // 2:].double())
        position, slot = s["positions"].long(), s["slots"].long()
        turn = torch.where((position >= 0)[:, None], turn[position.clamp(min=0)], torch.ones((), dtype=turn.dtype, device="cuda"))
        got = {}
        for name in ("q", "k"):
            x = s[name].double()
            y = torch.complex(x[..., :d // 2], x[..., d // 2:]) * turn[:, None, :]
            got[name] = torch.cat([y.real, y.imag], 2)
        caches = [torch.zeros(s["k_cache"].shape, **f64) for _ in range(2)]
        written = (slot >= 0).nonzero()[:, 0]
        for cache, new in zip(caches, (got["k"], s["v"].double())):
            cache[slot[written] // page, slot[written] % page] = new[written]
        return {"q": got["q"], "k_cache": caches[0], "v_cache": caches[1]}
    if case["op"] == "plan":
        page, rows, pages = case["page"], s["rows"], s["pages"]
        cached, added = s["cached"].tolist(), s["added"].tolist()
        table, stack, free = s["block_table"].tolist(), s["free_pages"].tolist(), s["free_count"].item()
        lens, cu, positions, slots = [], [0], [], []
        wanted = 0  # pages asked for so far, those of requests that got none among them
        left = free
        for i, (c, a) in enumerate(zip(cached, added)):
            old, new = _pages(c, page), _pages(c + a, page)
            fits = new <= len(table[i]) and cu[-1] + a <= rows
            wanted += new - old if fits else 0
            served = fits and (new == old or wanted <= free)
            if served and new > old:
                table[i][old:new] = [stack[free - 1 - (wanted - (new - old)) - j] for j in range(new - old)]
                left = free - wanted
            for j in range(a):
                positions.append(c + j)
                slots.append(table[i][(c + j) // page] * page + (c + j) % page if served else -1)
            cu.append(cu[-1] + a)
            lens.append(c + a if served else c)
        behind = [-1] * (rows - len(slots))
        on = dict(dtype=torch.int32, device="cuda")
        return {"seq_lens": torch.tensor(lens, **on), "cu_seqlens": torch.tensor(cu, **on),
                "positions": torch.tensor(positions + behind, **on), "slots": torch.tensor(slots + behind, **on),
                "free_left": torch.tensor([left], **on), "block_table": torch.tensor(table, **on)}
    token, logprob = torch.zeros(case["rows"], dtype=I32, device="cuda"), torch.zeros(case["rows"], **f64)
    temperature, top_k = s["temperature"].tolist(), s["top_k"].tolist()
    top_p, min_p, uniform = s["top_p"].tolist(), s["min_p"].tolist(), s["uniform"].tolist()
    for i in range(case["rows"]):
        z = s["logits"][i].double()
        if not temperature[i] > 0:
            token[i] = torch.nonzero(z == z.max())[0, 0]
            continue
        order = torch.argsort(z, descending=True, stable=True)
        if top_k[i] > 0:
            order = order[:top_k[i]]
        chance = torch.softmax(z[order] / temperature[i], 0)  # in falling order
        n = len(order)
        if top_p[i] < 1:
            n = min(n, int(torch.searchsorted(chance.cumsum(0), top_p[i])) + 1)
        if min_p[i] > 0:
            n = min(n, int((chance >= min_p[i] * chance[0]).sum()))
        kept = order[:max(n, 1)].sort().values
        x = z[kept] / temperature[i]
        chance = torch.softmax(x, 0)
        at = min(int(torch.searchsorted(chance.cumsum(0), uniform[i], right=True)), len(kept) - 1)
        token[i], logprob[i] = kept[at], x[at] - torch.logsumexp(x, 0)
    return {"token": token, "logprob": logprob}
