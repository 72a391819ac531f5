"""Operators of a serving step (cdl.serve) against their definitions in 64 bits (oracle/serve_ref.py), and a run of them together."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import serve_ref

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32
gpu = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=I32, device="cuda")


def f64(t):
    return t.detach().double().cpu().numpy()


# --------------------------------------------------------------------------- the cache's plan
def plan_inputs(cached, added, page_size, width=None, spare=3, seed=0):
    """Tables with every request's pages in use, the other pages on the stack in random order."""
    gen = np.random.default_rng(seed)
    count = lambda n: -(-max(n, 0) // page_size)
    width = width if width is not None else max([count(max(c, 0) + max(a, 0)) for c, a in zip(cached, added)] + [1])
    used = [min(count(c), width) for c in cached]
    need = sum(count(max(c, 0) + max(a, 0)) - count(c) for c, a in zip(cached, added))
    pages = sum(used) + need + spare
    order = gen.permutation(pages).tolist()
    table, at = [], 0
    for n in used:
        table.append(order[at:at + n] + [-7] * (width - n))
        at += n
    return table, order[at:] + [-9, -9], pages, need


def check_plan(cdl, cached, added, page_size, rows, free, table, stack, pages):
    t = ints(table).reshape(len(cached), -1)
    got = cdl.serve.cache_plan(ints(cached), ints(added), t, ints(stack), ints([free]),
                               cdl.serve.CachePlanOpts(page_size=page_size, pages=pages, rows=rows))
    want = serve_ref.cache_plan(cached, added, table, stack, free, page_size, pages, rows)
    names = ("seq_lens", "cu_seqlens", "positions", "slots", "free_left", "block_table")
    have = (got.seq_lens, got.cu_seqlens, got.positions, got.slots, got.free_left, t)
    for name, g, w in zip(names, have, want):
        w = [w] if name == "free_left" else w
        assert g.tolist() == w, name
    return got


@gpu
@pytest.mark.parametrize("page_size", [1, 7, 16, 256])
@pytest.mark.parametrize("cached,added", [
    ([0], [1]), ([16], [1]), ([15, 0, 33, 64], [1, 40, 0, 17]), ([5, 0, 0, 9], [0, 0, 0, 0]), ([100], [1000]),
    ([-3, 4], [2, -1]), ([31] * 64, [1] * 64),
])
def test_plan_gives_pages_in_order(cdl, gpu_ok, cached, added, page_size):
    table, stack, pages, need = plan_inputs(cached, added, page_size)
    rows = sum(max(a, 0) for a in added)
    for extra in (0, 5):
        check_plan(cdl, cached, added, page_size, rows + extra, need + 3, table, stack, pages)


@gpu
@pytest.mark.parametrize("requests", [1023, 1024, 1025, 3000])
@pytest.mark.parametrize("share", [1.0, 0.4])
def test_plan_of_many_requests(cdl, gpu_ok, requests, share):
    """More requests than a pass of the kernel has, with idle ones, and a stack that does not suffice."""
    gen = np.random.default_rng(requests)
    cached = gen.integers(0, 200, requests).tolist()
    added = (gen.integers(0, 30, requests) * (gen.random(requests) < 0.7)).tolist()
    table, stack, pages, need = plan_inputs(cached, added, 16, seed=requests)
    check_plan(cdl, cached, added, 16, sum(added) + 9, int(share * need), table, stack, pages)


@gpu
def test_plan_refuses_what_does_not_fit(cdl, gpu_ok):
    """A table row that is too short, rows that the batch does not have, pages outside the cache, lengths near 2^31."""
    big = 2 ** 31 - 1
    table = [[4, 5, 1, -1], [2, -1, -1, -1], [3, -1, -1, -1], [0, 9, -1, -1]]
    stack = [7, 8, 10, 6]
    for cached, added, rows, free, pages in [
        ([12, 3, 4, 6], [5, 1, 2, 1], 20, 4, 11),       # the first would need a fifth page
        ([12, 3, 4, 6], [0, 1, 9, 2], 6, 4, 11),        # the third has no rows left, nor then the fourth
        ([8, 4, 4, 8], [3, 3, 3, 3], 12, 4, 8),         # pages 8, 9 and 10 are outside
        ([big, 3, big, 6], [big, 1, 1, 2], 20, 4, 11),  # sums beyond 32 bits
        ([4, 4, 4, 8], [4, 4, 4, 4], 16, 2, 11),        # two pages for four requests
        ([4, 4, 4, 7], [4, 9, 4, 1], 32, 2, 11),        # the second asks for more than is left, the last for none
        ([4, 4, 4, 8], [4, 4, 4, 4], 16, 0, 11),
        ([4, 4, 4, 8], [4, 4, 4, 4], 16, -5, 11),
        ([4, 4, 4, 8], [4, 4, 4, 4], 16, 99, 11),       # a count above the stack's size
        ([4, 4, 4, 8], [4, 4, 4, 4], 0, 4, 11),
    ]:
        check_plan(cdl, cached, added, 4, rows, free, table, stack, pages)


@gpu
def test_plan_without_requests_or_width(cdl, gpu_ok):
    opts = cdl.serve.CachePlanOpts(page_size=16, pages=4, rows=3)
    none = torch.empty(0, dtype=I32, device="cuda")
    p = cdl.serve.cache_plan(none, none, torch.empty(0, 8, dtype=I32, device="cuda"), ints([3, 1]), ints([2]), opts)
    assert p.cu_seqlens.tolist() == [0] and p.slots.tolist() == p.positions.tolist() == [-1] * 3 and p.free_left.tolist() == [2]
    p = cdl.serve.cache_plan(ints([0]), ints([2]), torch.empty(1, 0, dtype=I32, device="cuda"), ints([3, 1]), ints([2]), opts)
    assert p.seq_lens.tolist() == [0] and p.slots.tolist() == [-1] * 3 and p.positions.tolist() == [0, 1, -1]


# --------------------------------------------------------------------------- the way into the cache
def rope_table(cdl, positions, dim):
    return cdl.sky1.rope_table(positions, dim)


def check_write(cdl, tokens, heads, kv_heads, dim, page_size, layout="packed", k_out=True, seed=0, rotated=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(BF16)
    qkv = rnd(tokens, heads + 2 * kv_heads, dim)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    pages = -(-tokens // page_size) + 2
    if layout == "packed":
        caches = [rnd(pages, page_size, kv_heads, dim) for _ in range(2)]
    elif layout == "heads_first":
        caches = [rnd(pages, kv_heads, page_size, dim).transpose(1, 2) for _ in range(2)]
    else:  # one tensor for both
        both = rnd(pages, page_size, 2, kv_heads, dim)
        caches = [both[:, :, 0], both[:, :, 1]]
    before = [c.clone() for c in caches]
    table = rope_table(cdl, 50, dim)
    rng = np.random.default_rng(seed)
    positions = rng.integers(0, 50, tokens)
    slots = rng.permutation(pages * page_size)[:tokens]
    if tokens > 2:
        positions[1], slots[1] = -1, -1               # padding
        positions[2] = 50                             # behind the table: not rotated
        slots[0] = pages * page_size                  # behind the cache: not stored
    ko = torch.empty_like(k, memory_format=torch.contiguous_format) if k_out and rotated else None
    if rotated:
        got = cdl.serve.cache_write(k, v, ints(slots), *caches, q=q, table=table, positions=ints(positions), k_out=ko)
    else:
        got = cdl.serve.cache_write(k, v, ints(slots), *caches)
    cs = f64(table)
    qn, kn, vn = f64(q), f64(k), f64(v)
    want = [f64(c) for c in before]
    size = np.abs(np.concatenate([cs[:, :dim // 2], cs[:, :dim // 2]], 1)) + np.abs(np.concatenate([cs[:, dim // 2:], cs[:, dim // 2:]], 1))

    def near(name, have, x, ref):
        # one rounding to bf16, and three of f32 terms of |x cos| + |x sin|
        bound = 2.0 ** -8 * np.abs(ref) + 3 * 2.0 ** -24 * 2 * np.abs(x).max()
        assert (np.abs(have - ref) <= bound).all(), name

    for i in range(tokens):
        kr = serve_ref.rotate(kn[i], cs, positions[i]) if rotated else kn[i]
        if rotated:
            near("q", f64(got.q[i]), qn[i], serve_ref.rotate(qn[i], cs, positions[i]))
            if ko is not None:
                near("k_out", f64(ko[i]), kn[i], kr)
        if 0 <= slots[i] < pages * page_size:
            at = slots[i] // page_size, slots[i] % page_size
            have = f64(caches[0][at])
            near("k_cache", have, kn[i], kr)
            want[0][at], want[1][at] = have, vn[i]
    assert np.array_equal(f64(caches[0]), want[0]) and np.array_equal(f64(caches[1]), want[1])  # nothing else was touched
    assert size.shape == cs.shape


@gpu
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,page_size", [
    (1, 16, 16, 128, 16), (3, 1, 1, 16, 1), (37, 8, 2, 64, 7), (130, 24, 3, 48, 16), (65, 5, 5, 256, 33), (300, 16, 4, 128, 64),
])
@pytest.mark.parametrize("layout", ["packed", "heads_first", "together"])
def test_write(cdl, gpu_ok, tokens, heads, kv_heads, dim, page_size, layout):
    check_write(cdl, tokens, heads, kv_heads, dim, page_size, layout, seed=tokens)


@gpu
def test_write_without_rotation(cdl, gpu_ok):
    check_write(cdl, 21, 4, 2, 128, 5, rotated=False)
    check_write(cdl, 21, 4, 2, 128, 5, k_out=False)


@gpu
def test_write_in_place(cdl, gpu_ok):
    """q and k rotated where they lie in the fused tensor: the values of a call into new tensors, and the bits of rope."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    qkv = torch.randn(40, 12, 128, generator=gen, device="cuda").to(BF16)
    table = rope_table(cdl, 64, 128)
    positions, slots = ints(list(range(10, 50))), ints(list(range(40))[::-1])
    res = []
    for in_place in (False, True):
        x = qkv.clone()
        q, k, v = x[:, :8], x[:, 8:10], x[:, 10:]
        caches = [torch.zeros(3, 16, 2, 128, dtype=BF16, device="cuda") for _ in range(2)]
        ko = k if in_place else torch.empty(40, 2, 128, dtype=BF16, device="cuda")
        o = cdl.serve.cache_write(k, v, slots, *caches, q=q, table=table, positions=positions, q_out=q if in_place else None, k_out=ko)
        assert in_place == (o.q.data_ptr() == x.data_ptr()) and torch.equal(v, qkv[:, 10:])
        res.append((o.q.clone(), o.k.clone(), *caches))
    assert all(torch.equal(a, b) for a, b in zip(*res))
    L, x = cdl._lib, qkv.clone()
    padded = torch.cat([torch.zeros(10, 12, 128, dtype=BF16, device="cuda"), x])  # rope's position is the row
    tx, tt = L.tensor_arg(padded), L.tensor_arg(table)
    L.check(L.lib.cdl_b200_rope(L.ref(tx), L.ref(tt), 10, 64, 0, None))
    torch.cuda.synchronize()
    assert torch.equal(padded[10:, :8], res[0][0]) and torch.equal(padded[10:, 8:10], res[0][1])


# --------------------------------------------------------------------------- attention over the cache
def decode_inputs(lens, heads, kv_heads, dim, page_size, layout="packed", seed=0, width=None, lean=0.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    count = [-(-max(n, 0) // page_size) for n in lens]
    width = width if width is not None else max(count + [1])
    pages = sum(count) + 2
    order = np.random.default_rng(seed).permutation(pages)
    table, at = np.full((len(lens), width), -1), 0
    for b, n in enumerate(count):
        table[b, :n] = order[at:at + n]
        at += n
    shape = (pages, kv_heads, page_size, dim) if layout == "heads_first" else (pages, page_size, kv_heads, dim)
    if layout == "together":
        both = rnd(pages, page_size, 2, kv_heads, dim).to(BF16)
        k, v = both[:, :, 0], both[:, :, 1]
    else:
        k, v = rnd(*shape).to(BF16), rnd(*shape).to(BF16)
        if layout == "heads_first":
            k, v = k.transpose(1, 2), v.transpose(1, 2)
    q = rnd(len(lens), heads, dim)
    for b, n in enumerate(lens):  # a key that the queries lean towards
        if n > 0 and lean:
            j = (n * 2) // 3
            key = k[table[b, j // page_size], j % page_size].float()
            q[b] += lean * key.repeat_interleave(heads // kv_heads, 0)
    # what lies behind a request's last key may be anything
    for b, n in enumerate(lens):
        if n > 0 and n % page_size:
            k[table[b, count[b] - 1], n % page_size:] = float("nan")
            v[table[b, count[b] - 1], n % page_size:] = float("inf")
    return q.to(BF16), k, v, ints(table).reshape(len(lens), width), ints(lens)


def check_decode(cdl, q, k, v, table, lens, scale=None, softcap=0.0, window=0, **more):
    opts = cdl.serve.AttentionDecodeOpts(softmax_scale=scale, softcap=softcap, window=window)
    got = cdl.serve.attention_decode(q, k, v, table, lens, opts, lse=True, **more)
    others = []
    if 0 < table.shape[1] * k.shape[1] <= 2048 and not more:  # the form for longer ones too: entries that no request reaches
        wide = torch.full((len(lens), 2048 // k.shape[1] + 2), -1, dtype=I32, device="cuda")
        wide[:, :table.shape[1]] = table
        others.append(cdl.serve.attention_decode(q, k, v, wide, lens, opts, lse=True))
    out, lse, spread, reach = serve_ref.attention_decode(f64(q), f64(k), f64(v), table.cpu().numpy(), lens.cpu().numpy(), scale,
                                                         softcap, window)
    n, dim = int(lens.max().clamp(min=1)), q.shape[2]
    # a score's roundings: of the sum of dim products, of the scale and the cap; the exponential's
    off = (dim + 8) * 2.0 ** -24 * reach + 2.0 ** -20
    bound = 2.0 ** -8 * (np.abs(out) + spread) + 2 * off[..., None] * spread + n * 2.0 ** -24 * spread
    for x in [got] + others:
        _check_decoded(x, out, lse, bound, off, n)
    return got


def _check_decoded(got, out, lse, bound, off, n):
    have, have_lse = f64(got.out), f64(got.lse)
    assert np.array_equal(np.isnan(have_lse), np.isnan(lse)) and np.array_equal(np.isneginf(have_lse), np.isneginf(lse))
    dead = np.isnan(lse)
    assert np.isnan(have[dead]).all() and (have[np.isneginf(lse)] == 0).all()
    fine = np.isfinite(lse)
    worst = (np.abs(have - out) / np.maximum(bound, 1e-30))[fine]
    assert worst.size == 0 or worst.max() <= 1, worst.max()
    lse_bound = off + n * 2.0 ** -24 + 2.0 ** -22 * np.abs(np.where(fine, lse, 0))
    assert (np.abs(have_lse - lse)[fine] <= lse_bound[fine]).all()


@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (16, 16), (8, 1), (6, 2), (24, 2), (16, 1), (51, 3), (40, 1)])
def test_decode_head_layouts(cdl, gpu_ok, dim, heads, kv_heads):
    """One head, groups of 1 to 40 query heads per kv head, some of them not whole tiles of 8 columns."""
    check_decode(cdl, *decode_inputs([5, 130, 1, 64], heads, kv_heads, dim, 16, seed=heads))


@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page_size", [1, 3, 7, 16, 32, 100, 1024])
def test_decode_page_sizes(cdl, gpu_ok, dim, page_size):
    check_decode(cdl, *decode_inputs([1, 15, 16, 17, 31, 32, 33, 500], 4, 2, dim, page_size, seed=page_size))


@gpu
@pytest.mark.parametrize("layout", ["heads_first", "together"])
def test_decode_cache_layouts(cdl, gpu_ok, layout):
    check_decode(cdl, *decode_inputs([77, 300, 8], 8, 4, 128, 16, layout, seed=3))


@gpu
@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 4, 1), (64, 9, 1), (128, 32, 2)])
def test_decode_long_and_ragged(cdl, gpu_ok, dim, heads, kv_heads):
    """Lengths whose shares are cut by many warps, among ones that a warp has to itself, and empty requests."""
    check_decode(cdl, *decode_inputs([20000, 0, 3, 9001, 16, 0, 4097], heads, kv_heads, dim, 16, seed=dim + heads))


@gpu
@pytest.mark.parametrize("batch", [127, 128, 129, 700])
def test_decode_many_requests(cdl, gpu_ok, batch):
    lens = [(7 * i) % 40 for i in range(batch)]
    check_decode(cdl, *decode_inputs(lens, 2, 1, 64, 8, seed=batch))


@gpu
@pytest.mark.parametrize("window", [1, 2, 16, 33, 499, 100000])
@pytest.mark.parametrize("softcap", [0.0, 5.0, 50.0])
def test_decode_window_and_cap(cdl, gpu_ok, window, softcap):
    inputs = decode_inputs([1, 33, 500, 0, 1300], 6, 2, 128, 16, seed=window, lean=2.0)
    check_decode(cdl, *inputs, window=window, softcap=softcap)
    check_decode(cdl, *inputs, window=window, softcap=softcap, scale=0.5)


@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch,heads,kv_heads", [(1, 1, 1), (1, 20, 2), (7, 4, 4), (16, 12, 3), (20, 16, 4), (33, 4, 4), (99, 2, 2), (205, 2, 2)])
def test_decode_short_lines(cdl, gpu_ok, dim, batch, heads, kv_heads):
    """Requests of at most 2048 keys, whose lines have 1 to 8 CTAs each; some with fewer keys than those have warps, some with none."""
    lens = [(2047, 0, 1, 15, 17, 33, 129, 500, 0, 64)[b % 10] + b // 10 for b in range(batch)]
    check_decode(cdl, *decode_inputs(lens, heads, kv_heads, dim, 16, seed=batch))


@gpu
@pytest.mark.parametrize("window", [2047, 2048, 2049, 3001])
def test_decode_long_windows(cdl, gpu_ok, window):
    check_decode(cdl, *decode_inputs([5000, 100, 2600, 0, 2049, 2048], 6, 2, 128, 16, seed=window, lean=2.0), window=window, softcap=30.0)


@gpu
def test_decode_short_lines_captured(cdl, gpu_ok):
    """Graphs of calls of two widths on one stream, replayed beside one another on two, on new lengths."""
    made, streams = [], [torch.cuda.Stream() for _ in range(2)]
    inputs = [decode_inputs([900, 17, 2000, 300], 8, 2, 128, 16, seed=30 + i) for i in range(2)]
    inputs[1] = (*inputs[1][:3], torch.cat([inputs[1][3], inputs[1][3] * 0 - 1], 1), inputs[1][4])
    torch.cuda.synchronize()
    for x in inputs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            made.append((graph, cdl.serve.attention_decode(*x, lse=True)))
    for lens in ([900, 17, 2000, 300], [0, 2000, 1, 44]):
        for x in inputs:
            x[4].copy_(ints(lens))
        want = [cdl.serve.attention_decode(*x, lse=True) for x in inputs]
        torch.cuda.synchronize()
        for st, (graph, _) in zip(streams, made):
            with torch.cuda.stream(st):
                for _ in range(5):
                    graph.replay()
        torch.cuda.synchronize()
        for w, (_, got) in zip(want, made):
            # (bits: keys behind a request's first length are NaN, which the second one's reaches)
            assert torch.equal(got.out.view(torch.int16), w.out.view(torch.int16)) and torch.equal(got.lse.view(I32), w.lse.view(I32))


@gpu
def test_decode_large_and_small_caps(cdl, gpu_ok):
    inputs = decode_inputs([400], 4, 4, 64, 16, seed=9)
    for cap in (1e-3, 1.0, 1e4, 1e30):
        check_decode(cdl, *inputs, softcap=cap)


@gpu
def test_decode_pages_that_are_not_there(cdl, gpu_ok):
    """Entries outside the cache: their keys do not count, and nothing is read there; lengths beyond the table and below 0."""
    q, k, v, table, lens = decode_inputs([100, 64, 40, 50], 4, 2, 128, 16, seed=4)
    table[0, 1], table[0, 3] = -1, k.shape[0]
    table[1, :] = 2 ** 31 - 1
    table[2, 0] = -2 ** 31
    check_decode(cdl, q, k, v, table, lens)
    check_decode(cdl, q, k, v, table, ints([2 ** 31 - 1, 112, -5, 7]))
    check_decode(cdl, q, k, v, table[:, :0], lens)
    check_decode(cdl, q, k[:0], v[:0], table, lens)


@gpu
@pytest.mark.parametrize("what", ["nan", "inf", "all_minus_inf", "some_minus_inf", "value_nan"])
def test_decode_special_scores(cdl, gpu_ok, what):
    """A NaN or +inf among a head's scores, scores of -inf; a NaN value reaches what sees it."""
    q, k, v, table, lens = decode_inputs([40, 300, 20], 4, 4, 128, 16, seed=5)
    q = q.abs() + 1.0  # products with an infinite key are infinite, with its sign
    page = int(table[1, 3])
    if what == "all_minus_inf":
        k[table[1].long()] = float("-inf")
        k[table[1].long()][300 // 16] = float("-inf")
    elif what == "value_nan":
        v[page, 2, 1] = float("nan")
        got = cdl.serve.attention_decode(q, k, v, table, lens).out
        assert got[1, 1].isnan().all() and not got[1, 0].isnan().any() and not got[0].isnan().any()
        return
    else:
        k[page, 2, 1] = {"nan": float("nan"), "inf": float("inf"), "some_minus_inf": float("-inf")}[what]
    check_decode(cdl, q, k, v, table, lens)


@gpu
def test_decode_strides_and_out(cdl, gpu_ok):
    """q as the heads of a fused product, out into a view, a table with longer rows."""
    q, k, v, table, lens = decode_inputs([40, 300, 20], 8, 4, 128, 16, seed=6)
    fused = torch.randn(3, 16, 128, device="cuda").to(BF16)
    fused[:, :8] = q
    wide = torch.full((3, table.shape[1] + 5), -1, dtype=I32, device="cuda")
    wide[:, :table.shape[1]] = table
    where = torch.full((3, 11, 256), 7.0, dtype=BF16, device="cuda")
    base = check_decode(cdl, q, k, v, table, lens)
    got = check_decode(cdl, fused[:, :8], k, v, wide[:, :table.shape[1]], lens, out=where[:, 2:10, 128:])
    assert torch.equal(got.out, base.out) and torch.equal(got.lse, base.lse)
    rest = where.clone()
    rest[:, 2:10, 128:] = 7.0
    assert (rest == 7.0).all()


@gpu
def test_decode_bits_do_not_depend_on_timing_or_scratch(cdl, gpu_ok):
    """Several streams at once, each with its scratch; scratch of other contents; a captured call replayed on new data."""
    inputs = [decode_inputs([900, 17, 4000, 300], 8, 2, 128, 16, seed=20 + i) for i in range(3)]
    want = [cdl.serve.attention_decode(*x, lse=True) for x in inputs]
    streams = [torch.cuda.Stream() for _ in inputs]
    n = cdl.serve.attention_decode_scratch_bytes(inputs[0][0], inputs[0][1])
    scratch = [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for _ in inputs]
    torch.cuda.synchronize()
    got = [[] for _ in inputs]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(cdl.serve.attention_decode(*inputs[i], lse=True, scratch=scratch[i]))
    torch.cuda.synchronize()
    for i, w in enumerate(want):
        assert all(torch.equal(g.out, w.out) and torch.equal(g.lse, w.lse) for g in got[i])
    # lengths and tables are read on the device: the captured call follows them
    static = [t.clone() for t in inputs[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cdl.serve.attention_decode(*static, lse=True, scratch=scratch[0])
    for x, w in list(zip(inputs, want))[::-1]:
        for a, b in zip(static, x):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.out, w.out) and torch.equal(out.lse, w.lse)


@gpu
def test_decode_of_nothing(cdl, gpu_ok):
    q, k, v, table, lens = decode_inputs([3], 2, 1, 64, 16)
    assert cdl.serve.attention_decode(q[:0], k, v, table[:0], lens[:0]).out.shape == (0, 2, 64)


# --------------------------------------------------------------------------- sampling
def check_sample(cdl, z, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    rows = z.shape[0]
    params = [temperature, top_k, top_p, min_p]
    got = cdl.serve.sample(z, u, cdl.serve.SampleOpts(*params))
    per_row = [x.tolist() if isinstance(x, torch.Tensor) else [x] * rows for x in params]
    zs, us = f64(z), u.tolist()
    for r in range(rows):
        token, logprob = serve_ref.sample(zs[r], us[r], *(x[r] for x in per_row))
        assert got.token[r].item() == token, (r, [x[r] for x in per_row])
        lp = got.logprob[r].item()
        # rounded once to f32; the sum behind it is 2^-30 off at most
        assert (lp != lp and logprob != logprob) or abs(lp - logprob) <= 2.0 ** -24 * abs(logprob) + 2.0 ** -30
    return got


def logits_of(rows, vocab, dtype, seed=0, spread=2.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    z = torch.randn(rows, vocab, generator=gen, device="cuda") * spread
    return z.to(dtype), torch.rand(rows, generator=gen, device="cuda")


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 1000, 1025, 4099, 32768, 50001, 131073])
def test_sample_vocabularies(cdl, gpu_ok, vocab, dtype):
    z, u = logits_of(6, vocab, dtype, seed=vocab)
    check_sample(cdl, z, u)
    check_sample(cdl, z, u, temperature=0.7, top_k=5)
    check_sample(cdl, z, u, top_p=0.8)
    check_sample(cdl, z, u, temperature=1.5, min_p=0.1)
    check_sample(cdl, z, u, temperature=1.2, top_k=50, top_p=0.9, min_p=0.02)
    check_sample(cdl, z, u, temperature=0.0)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_sample_settings_of_each_row(cdl, gpu_ok, dtype):
    rows, vocab = 60, 3001
    z, u = logits_of(rows, vocab, dtype, seed=2)
    gen = torch.Generator(device="cuda").manual_seed(3)
    rnd = lambda: torch.rand(rows, generator=gen, device="cuda")
    temperature, top_p, min_p = 2 * rnd(), 1.2 * rnd(), 0.3 * rnd() - 0.1
    temperature[::7] = 0.0
    temperature[1] = -1.0
    top_k = (rnd() * 2000).to(I32)
    top_k[::5] = 0
    top_k[3], top_k[4] = -4, 100000
    check_sample(cdl, z, u, temperature, top_k, top_p, min_p)
    check_sample(cdl, z, u, temperature, 0, top_p, 0.0)
    check_sample(cdl, z, u, 1.0, top_k, 1.0, min_p)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab", [7, 5000, 40000])
def test_sample_ties(cdl, gpu_ok, vocab, dtype):
    """Equal logits: the lowest indices count first, by number and by mass; all equal, two values, few values."""
    u = torch.tensor([0.0, 0.1, 0.5, 0.75, 0.999, 1 - 2.0 ** -24], device="cuda")
    flat = torch.full((6, vocab), 3.0, dtype=dtype, device="cuda")
    two = flat.clone()
    two[:, ::3] = 4.0
    few = (torch.arange(vocab, device="cuda") * 7919 % 5).to(dtype).repeat(6, 1)
    zero = torch.zeros(6, vocab, dtype=dtype, device="cuda")
    zero[:, ::2] = -0.0
    for z in (flat, two, few, zero):
        check_sample(cdl, z, u)
        for k in (1, 2, vocab // 2, vocab - 1, vocab):
            check_sample(cdl, z, u, top_k=k)
        for p in (1e-6, 0.3, 0.7, 0.999):
            check_sample(cdl, z, u, top_p=p)
        check_sample(cdl, z, u, top_k=vocab // 3 + 1, top_p=0.6)
        check_sample(cdl, z, u, min_p=1.0)
        check_sample(cdl, z, u, top_p=0.0)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_sample_masked_and_bad_rows(cdl, gpu_ok, dtype):
    vocab = 2000
    z, u = logits_of(9, vocab, dtype, seed=5)
    low = torch.finfo(dtype).min
    z[0, 100:] = -torch.inf
    z[1] = -torch.inf
    z[1, 1234] = -3.0
    z[2] = -torch.inf
    z[3, 77] = torch.nan
    z[4, 77] = torch.inf
    z[5, 5:] = low
    z[6] = low
    z[7] = low
    z[7, 9] = torch.finfo(dtype).max
    z[8, 0] = -torch.nan
    for more in ({}, {"top_k": 40}, {"top_p": 0.9}, {"min_p": 0.05}, {"top_k": 1500, "top_p": 0.99}, {"temperature": 0.0}):
        got = check_sample(cdl, z, u, **more)
        assert got.token[2] == got.token[3] == got.token[4] == got.token[8] == -1 and got.token[1] == 1234


@gpu
def test_sample_extreme_settings(cdl, gpu_ok):
    z, u = logits_of(8, 700, F32, seed=6)
    for t in (1e-30, 1e-6, 1e-2, 50.0, 1e30):
        check_sample(cdl, z, u, temperature=t)
        check_sample(cdl, z, u, temperature=t, top_p=0.5)
        check_sample(cdl, z, u, temperature=t, min_p=0.5)
    nan = float("nan")
    base = check_sample(cdl, z, u)
    for opts in ({"top_p": nan}, {"min_p": nan}):
        assert torch.equal(cdl.serve.sample(z, u, cdl.serve.SampleOpts(**opts)).token, base.token)
    greedy = cdl.serve.sample(z, u, cdl.serve.SampleOpts(temperature=nan))
    assert torch.equal(greedy.token.long(), z.argmax(1))
    odd = torch.tensor([-1.0, nan, 1.0, 2.0, torch.inf, -torch.inf, 0.0, 0.5], device="cuda")
    got = cdl.serve.sample(z, odd).token.tolist()
    w = torch.softmax(z.double(), 1)
    for r in (0, 1, 5):
        assert got[r] == 0
    for r in (2, 3, 4):
        assert got[r] == 699
    assert w.shape == z.shape
    # min_p above 1 keeps the largest
    check_sample(cdl, z, u, min_p=3.0)


@gpu
@pytest.mark.parametrize("vocab", [700, 5003, 40000])
def test_sample_of_an_infinite_temperature(cdl, gpu_ok, vocab):
    """Every entry that is not masked has the same weight."""
    z, u = logits_of(6, vocab, F32, seed=7)
    z[:, ::3] = -torch.inf
    for opts in ({}, {"min_p": 1.0}, {"min_p": 0.5}, {"top_p": 0.4}, {"top_k": 37}, {"top_k": 1500, "top_p": 0.7}):
        check_sample(cdl, z, u, temperature=torch.inf, **opts)


@gpu
@pytest.mark.parametrize("rows,vocab", [(3, 66001), (40, 66001), (70, 66001), (80, 66001), (50, 140001), (90, 140001)])
def test_sample_rows_shared_by_several_ctas(cdl, gpu_ok, rows, vocab):
    z, u = logits_of(rows, vocab, BF16, seed=rows)
    check_sample(cdl, z, u)
    check_sample(cdl, z, u, top_p=0.9)
    check_sample(cdl, z, u, top_k=50)
    check_sample(cdl, z, u, top_k=5000, min_p=0.01)


@gpu
def test_sample_draws_next_to_a_border(cdl, gpu_ok):
    """Random numbers as near to the borders between two tokens as f32 has them, on flat and on falling rows."""
    vocab = 30000
    z = (torch.randn(1, vocab, generator=torch.Generator(device="cuda").manual_seed(8), device="cuda") * 0.5).repeat(64, 1)
    w = np.exp(f64(z[0]) - f64(z[0]).max())
    cdf = np.cumsum(w) / w.sum()
    at = np.linspace(100, vocab - 100, 32).astype(int)
    u = np.float32(cdf[at])
    u = torch.tensor(np.concatenate([u, np.nextafter(u, np.float32(0))]), device="cuda")
    check_sample(cdl, z, u)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_sample_strides_and_repeats(cdl, gpu_ok, dtype):
    """Rows inside a wider tensor, at every offset; the same bits again, on another stream, from a graph, in another batch."""
    z, u = logits_of(5, 4096 + 64, dtype, seed=9)
    for off in (0, 1, 3, 8):
        for n in (4096, 4097, 4103):
            check_sample(cdl, z[:, off:off + n], u, top_k=20, top_p=0.9)
            check_sample(cdl, z[:, off:off + n], u, top_p=0.95)
    opts = cdl.serve.SampleOpts(temperature=0.9, top_p=0.9)
    one = cdl.serve.sample(z, u, opts)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        two = cdl.serve.sample(z, u, opts)
    torch.cuda.synchronize()
    assert torch.equal(one.token, two.token) and torch.equal(one.logprob, two.logprob)
    alone = [cdl.serve.sample(z[r:r + 1], u[r:r + 1], opts).token.item() for r in range(5)]
    assert alone == one.token.tolist()
    graph = torch.cuda.CUDAGraph()
    zs = z.clone()
    with torch.cuda.graph(graph):
        res = cdl.serve.sample(zs, u, opts)
    zs.copy_(z.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(res.token, cdl.serve.sample(z.flip(0).contiguous(), u, opts).token)
    assert cdl.serve.sample(z, u, opts, logprob=False).logprob is None
    assert cdl.serve.sample(z[:0], u[:0], opts).token.shape == (0,)


# --------------------------------------------------------------------------- far offsets
@gpu
def test_cache_of_more_than_2_31_elements(cdl, gpu_ok):
    """Pages whose elements lie beyond 2^31 from the cache's start: written and attended to."""
    pages, page_size, heads = 140000, 16, 8
    k = torch.empty(pages, page_size, heads, 128, dtype=BF16, device="cuda")  # 2.3 10^9 elements
    assert k.numel() > 2 ** 31
    v = torch.empty_like(k)
    gen = torch.Generator(device="cuda").manual_seed(0)
    new = torch.randn(2, 40, heads, 128, generator=gen, device="cuda").to(BF16)
    at = [pages - 1, 3, pages - 2]
    slots = [at[j // page_size] * page_size + j % page_size for j in range(40)]
    cdl.serve.cache_write(new[0], new[1], ints(slots), k, v)
    q = torch.randn(1, heads, 128, generator=gen, device="cuda").to(BF16)
    got = cdl.serve.attention_decode(q, k, v, ints([at]).reshape(1, 3), ints([40]), lse=True)
    small_k, small_v = (torch.zeros(3, page_size, heads, 128, dtype=BF16, device="cuda") for _ in range(2))
    small_k.view(48, heads, 128)[:40], small_v.view(48, heads, 128)[:40] = new[0], new[1]
    want = check_decode(cdl, q, small_k, small_v, ints([[0, 1, 2]]), ints([40]))
    assert torch.equal(got.out, want.out) and torch.equal(got.lse, want.lse)


@gpu
def test_logits_of_more_than_2_31_elements(cdl, gpu_ok):
    vocab = 150001
    rows = 2 ** 31 // vocab + 2
    z = torch.zeros(rows, vocab, dtype=BF16, device="cuda")
    z[-1, 77], z[-1, 99] = 30.0, 30.0
    z[-2, 5] = 40.0
    u = torch.full((rows,), 0.75, device="cuda")
    got = cdl.serve.sample(z, u, cdl.serve.SampleOpts(top_k=2)).token
    assert got[-1] == 99 and got[-2] == 5 and got[0] == 1
    assert cdl.serve.sample(z, u, cdl.serve.SampleOpts(temperature=0.0)).token[-2:].tolist() == [5, 77]


# --------------------------------------------------------------------------- refusals (no GPU: operands are checked first)
def status(cdl, name, *args):
    L = cdl._lib
    given = [L.tensor_bytes(a) if isinstance(a, torch.Tensor) else a for a in args]
    return getattr(L.packed_lib, name)(*given, None), L.last_error()


def swap(args, i, x):
    return [x if j == i else a for j, a in enumerate(args)]


def bf(*shape):
    return torch.zeros(*shape, dtype=BF16)


def i32(*shape):
    return torch.zeros(*shape, dtype=I32)


def test_plan_refusals(cdl):
    # page_size, pages, cached, added, block_table, free_pages, free_count | seq_lens, cu_seqlens, positions, slots, free_left
    good = [16, 9, i32(4), i32(4), i32(4, 3), i32(9), i32(1), i32(4), i32(5), i32(7), i32(7), i32(1)]
    call = lambda args: status(cdl, "cdl_b200_cache_plan", *args)
    for i, bad, message in [
        (0, 0, "page_size"), (0, -3, "page_size"), (1, -1, "page_size"), (1, 2 ** 30, "2^31"), (2, i32(3), "must be"),
        (3, i32(5), "added"), (3, torch.zeros(4), "added"), (3, i32(8)[::2], "added"), (4, i32(3, 3), "block_table"),
        (4, i32(4, 6)[:, ::2], "block_table"), (4, i32(1, 3).expand(4, 3), "overlap"), (4, torch.zeros(4, 3), "block_table"),
        (5, i32(3, 3), "free_pages"), (6, i32(2), "free_count"), (7, i32(5), "seq_lens"), (8, i32(4), "cu_seqlens"),
        (9, i32(6), "positions"), (10, i32(2, 7), "vectors"), (11, i32(0), "free_left"), (2, None, "required"), (6, None, "free_count"),
    ]:
        st, text = call(swap(good, i, bad))
        assert st == -1 and message in text, (i, message, st, text)
    for i, j in ((7, 2), (7, 3), (11, 6), (9, 10), (8, 7), (4, 2), (10, 5)):  # an output that is an input, or another output
        shared = i32(64)
        size = lambda a: shared[:a.numel()].view(a.shape)
        st, text = call(swap(swap(good, i, size(good[i])), j, size(good[j])))
        assert st == -1 and "overlap" in text, (i, j, text)


def test_write_refusals(cdl):
    # q, k, v, cos_sin, positions, slots, q_out, k_out, k_cache, v_cache
    good = [bf(5, 4, 32), bf(5, 2, 32), bf(5, 2, 32), torch.zeros(8, 32), i32(5), i32(5), bf(5, 4, 32), None, bf(3, 4, 2, 32), bf(3, 4, 2, 32)]
    call = lambda args: status(cdl, "cdl_b200_cache_write", *args)
    flat = bf(5 * 8 * 32 + 8)
    for i, bad, message in [
        (0, None, "together"), (6, None, "together"), (3, None, "together"), (4, None, "together"), (1, None, "required"),
        (0, bf(4, 4, 32), "q must be"), (0, torch.zeros(5, 4, 32), "q must be"), (1, bf(5, 64), "k must be"), (2, bf(5, 3, 32), "v must be"),
        (1, flat[1:1 + 320].view(5, 2, 32), "16-byte"), (1, flat[:5 * 68].view(5, 68)[:, :64].view(5, 2, 32), "16-byte"),
        (2, bf(5, 32, 2).transpose(1, 2), "contiguous"), (3, torch.zeros(8, 64), "cos_sin"), (3, torch.zeros(8, 64)[:, ::2], "cos_sin"),
        (4, i32(4), "positions"), (5, i32(6), "slots"), (5, torch.zeros(5), "slots"), (6, bf(5, 4, 64), "q_out"),
        (6, bf(1, 4, 32).expand(5, 4, 32), "overlap"), (8, bf(3, 4, 3, 32), "caches"), (8, bf(3, 4, 2, 64), "caches"),
        (9, bf(4, 4, 2, 32), "caches"), (9, torch.zeros(3, 4, 2, 32), "caches"), (8, bf(1, 4, 2, 32).expand(3, 4, 2, 32), "overlap"),
        (9, good[8], "overlap"), (6, good[1].expand(2, 5, 2, 32)[0].reshape(5, 2, 32), "q_out"), (7, good[2], "overlap"), (6, good[0][:, :, :], None),
    ]:
        if message is None:
            continue
        st, text = call(swap(good, i, bad))
        assert st == -1 and message in text, (i, message, st, text)
    # q_out and k_out without a table, head_dim off 16 or too long, q_out one row behind q
    st, text = call(swap(swap(good, 3, None), 4, None))
    assert st == -1 and "table" in text
    for d in (24, 4096):
        st, text = call([None, bf(5, 2, d), bf(5, 2, d), None, None, i32(5), None, None, bf(3, 4, 2, d), bf(3, 4, 2, d)])
        assert st == -1 and "head_dim" in text
    rows = bf(6, 4, 32)
    st, text = call(swap(swap(good, 0, rows[:5]), 6, rows[1:]))
    assert st == -1 and "overlaps an input" in text


def test_views_of_one_fused_tensor_are_told_apart(cdl):
    """q_out = q inside qkv beside k and v, k_cache and v_cache inside one tensor: not refused as overlapping (no tokens: nothing
    runs); a head further on is."""
    qkv = bf(0, 8, 32)
    both = bf(3, 4, 2, 2, 32)
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    args = [q, k, v, torch.zeros(8, 32), i32(0), i32(0), q, k, both[:, :, 0], both[:, :, 1]]
    assert status(cdl, "cdl_b200_cache_write", *args)[0] == 0
    pages = bf(3, 2, 4, 2, 32)
    assert status(cdl, "cdl_b200_cache_write", *args[:8], pages[:, 0], pages[:, 1])[0] == 0
    st, text = status(cdl, "cdl_b200_cache_write", *args[:8], both[:, :, 0], both[:, :, 0])
    assert st == -1 and "overlap" in text
    qkv = bf(2, 8, 32)
    st, text = status(cdl, "cdl_b200_cache_write", qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], torch.zeros(8, 32), i32(2), i32(2), qkv[:, 1:5], None,
                      both[:, :, 0], both[:, :, 1])
    assert st == -1 and "overlaps an input" in text


def test_decode_refusals(cdl):
    L = cdl._lib
    desc = lambda scale=0.0, cap=0.0, window=0: L.attn_decode_bytes(scale, cap, window)
    buf = torch.zeros(1 << 20, dtype=torch.uint8)
    at = (buf.data_ptr() + 255) // 256 * 256
    # desc, q, k_cache, v_cache, block_table, seq_lens, out, lse, scratch, bytes
    good = [desc(), bf(3, 4, 64), bf(5, 16, 2, 64), bf(5, 16, 2, 64), i32(3, 2), i32(3), bf(3, 4, 64), torch.zeros(3, 4), at, 1 << 40]
    call = lambda args: status(cdl, "cdl_b200_attn_decode", *args)
    nan, inf = float("nan"), float("inf")
    for i, bad, message in [
        (0, None, "required"), (0, desc(cap=-1.0), "softcap"), (0, desc(cap=nan), "softcap"), (0, desc(cap=inf), "softcap"),
        (0, desc(scale=nan), "softmax_scale"), (0, desc(scale=inf), "softmax_scale"), (0, desc(window=-1), "window"),
        (1, torch.zeros(3, 4, 64), "q must be"), (1, bf(3, 256), "q must be"), (1, bf(3, 3, 64), "multiple"), (1, bf(3, 4, 128), "differ"),
        (2, bf(5, 16, 64), "caches"), (2, torch.zeros(5, 16, 2, 64), "caches"), (3, bf(4, 16, 2, 64), "v_cache"), (3, None, "required"),
        (4, i32(4, 2), "block_table"), (4, torch.zeros(3, 2), "block_table"), (4, i32(3, 4)[:, ::2], "block_table"),
        (5, i32(4), "seq_lens"), (5, torch.zeros(3), "seq_lens"), (6, bf(3, 4, 128), "out"), (6, bf(1, 4, 64).expand(3, 4, 64), "overlap"),
        (6, good[1], "overlaps an input"), (7, torch.zeros(4, 3), "lse"), (7, bf(3, 4), "lse"), (8, None, "scratch"), (8, at + 16, "scratch"),
        (9, 1000, "scratch"), (2, bf(5, 16, 2, 72)[:, :, :, :64].transpose(2, 3), "caches"), (1, bf(3, 4, 65)[:, :, 1:], "q must have"),
        (2, bf(5, 16, 2, 65)[:, :, :, :64], "k_cache must have"),
    ]:
        st, text = call(swap(good, i, bad))
        assert st in (-1, -2) and (message in text or message == "caches" and "differ" in text), (i, message, st, text)
    st, text = call(swap(swap(swap(swap(good, 1, bf(3, 4, 96)), 2, bf(5, 16, 2, 96)), 3, bf(5, 16, 2, 96)), 6, bf(3, 4, 96)))
    assert st == -2 and "64 or 128" in text
    n = ctypes.c_size_t(0)
    assert L.packed_lib.cdl_b200_attn_decode_scratch_bytes(L.tensor_bytes(bf(5000, 1, 64)), L.tensor_bytes(bf(5, 16, 1, 64)), ctypes.byref(n)) == -2
    assert L.packed_lib.cdl_b200_attn_decode_scratch_bytes(L.tensor_bytes(bf(3, 4, 64)), L.tensor_bytes(bf(5, 16, 2, 64)), None) == -1


def test_sample_refusals(cdl):
    L = cdl._lib
    # desc, logits, uniform, temperature, top_k, top_p, min_p, token, logprob
    f = torch.zeros
    good = [L.sample_bytes(1.0, 0, 1.0, 0.0), f(4, 50), f(4), f(4), i32(4), f(4), f(4), i32(4), f(4)]
    call = lambda args: status(cdl, "cdl_b200_sample", *args)
    for i, bad, message in [
        (0, None, "required"), (1, f(200), "logits"), (1, i32(4, 50), "logits"), (1, f(4, 100)[:, ::2], "contiguous"), (1, f(4, 0), "empty"),
        (2, f(3), "uniform"), (2, i32(4), "uniform"), (2, f(8)[::2], "uniform"), (3, i32(4), "temperature"), (4, f(4), "top_k"),
        (5, f(5), "top_p"), (6, f(4, 1), "min_p"), (7, f(4), "token"), (7, None, "required"), (8, i32(4), "logprob"), (8, good[2], "overlaps"),
    ]:
        st, text = call(swap(good, i, bad))
        assert st == -1 and message in text, (i, message, st, text)
    shared = i32(4)
    st, text = call(swap(swap(good, 4, shared), 7, shared))
    assert st == -1 and "overlaps an input" in text


def test_python_refusals(cdl):
    """What the Python layer refuses by itself: operands that are not in device memory, shapes that it reads."""
    S = cdl.serve
    with pytest.raises(cdl._lib.CdlError, match="device memory"):
        S.cache_plan(i32(4), i32(4), i32(4, 3), i32(9), i32(1), S.CachePlanOpts(16, 9, 7))
    with pytest.raises(cdl._lib.CdlError, match="device memory"):
        S.attention_decode(bf(3, 4, 64), bf(5, 16, 2, 64), bf(5, 16, 2, 64), i32(3, 2), i32(3))
    with pytest.raises(cdl._lib.CdlError, match="device memory"):
        S.cache_write(bf(5, 2, 32), bf(5, 2, 32), i32(5), bf(3, 4, 2, 32), bf(3, 4, 2, 32))
    with pytest.raises(cdl._lib.CdlError, match="rows, vocab"):
        S.sample(torch.zeros(50), torch.zeros(1))


@gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_decode_of_2_31_keys(cdl, gpu_ok, dim):
    """The longest request there is: one large page again and again, whose keys all score the same; its last tile ends behind
    2^31 - 1.  And the window at its end."""
    page_size = 1 << 20
    k = torch.ones(1, page_size, 1, dim, dtype=BF16, device="cuda")
    v = torch.full_like(k, 3.0)
    q = torch.ones(1, 1, dim, dtype=BF16, device="cuda")
    table = torch.zeros(1, 2048, dtype=I32, device="cuda")
    n = 2 ** 31 - 1
    got = cdl.serve.attention_decode(q, k, v, table, ints([n]), lse=True)
    # equal weights: the mean is exact; the logarithm of a sum of 2^31 ones in f32, in parts of at most 2^24 of them each
    assert (got.out == 3.0).all()
    want = dim ** 0.5 + np.log(float(n))
    assert abs(got.lse.item() - want) <= 2.0 ** -20 * want
    v[0, page_size - 40:] = 5.0
    got = cdl.serve.attention_decode(q, k, v, table, ints([n]), cdl.serve.AttentionDecodeOpts(window=39))
    assert (got.out == 5.0).all()
