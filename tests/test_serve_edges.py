"""Calls of the serving operators (cdl.serve) at the ends of what they take, against their definitions in 64 bits (oracle/serve_ref.py),
and what they refuse there."""
import numpy as np
import pytest
import torch

from oracle import serve_ref

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32
gpu = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=I32, device="cuda")


# --------------------------------------------------------------------------- lengths
@gpu
def test_plan_of_lengths_around_2_31(cdl, gpu_ok):
    """A table that names pages again and again has room for more keys than 32 bits count: a request that would pass 2^31 - 1 is not
    served, whether it needs a page for that or not, and the one behind it is."""
    page_size, width, pages, big = 1 << 20, 2049, 1500, 2 ** 31 - 1
    table, stack = [[5] * 2048 + [-1]] * 6, [1, 2, 3]
    cached, added = [big - 1, big - 1, big, big - 3, big, 3], [1, 2, 3, 3, 0, 1]
    t = ints(table)
    got = cdl.serve.cache_plan(ints(cached), ints(added), t, ints(stack), ints([3]), cdl.serve.CachePlanOpts(page_size, pages, 12))
    want = serve_ref.cache_plan(cached, added, table, stack, 3, page_size, pages, 12)
    assert want[0] == [big, big - 1, big, big, big, 4]
    have = (got.seq_lens, got.cu_seqlens, got.positions, got.slots, got.free_left, t)
    for name, g, w in zip(("seq_lens", "cu_seqlens", "positions", "slots", "free_left", "block_table"), have, want):
        assert g.tolist() == ([w] if name == "free_left" else w), name


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


def null(cdl, t):
    """A tensor's shape and strides without memory, as a C caller may give them."""
    return bytes(8) + cdl._lib.tensor_bytes(t)[8:]


def test_write_refuses_null_pointers(cdl):
    # q, k, v, cos_sin, positions, slots, q_out, k_out, k_cache, v_cache
    good = [bf(5, 4, 32), bf(5, 2, 32), bf(5, 2, 32), torch.zeros(8, 32), i32(5), i32(5), bf(5, 4, 32), bf(5, 2, 32), bf(3, 4, 2, 32),
            bf(3, 4, 2, 32)]
    for i, t in enumerate(good):
        st, text = status(cdl, "cdl_b200_cache_write", *swap(good, i, null(cdl, t)))
        assert st == -1 and ("null pointer" in text or "must" in text), (i, st, text)
    # nothing to store to, nothing to rotate: no memory is needed
    none = [t[:0] if i < 8 and i != 3 else t for i, t in enumerate(good)]
    for i in (3, 8, 9):
        assert status(cdl, "cdl_b200_cache_write", *swap(none, i, null(cdl, good[i])))[0] == 0


def decode_call(cdl):
    """desc, q, k_cache, v_cache, block_table, seq_lens, out, lse, scratch, bytes of a call that is in order."""
    buf = torch.zeros(1024, dtype=torch.uint8)
    at = (buf.data_ptr() + 255) // 256 * 256  # (its contents are never reached)
    return [cdl._lib.attn_decode_bytes(0.0, 0.0, 0), bf(3, 4, 64), bf(5, 16, 2, 64), bf(5, 16, 2, 64), i32(3, 2), i32(3), bf(3, 4, 64),
            torch.zeros(3, 4), at, 1 << 40]


def test_decode_refuses_null_pointers(cdl):
    good = decode_call(cdl)
    for i in range(1, 8):
        st, text = status(cdl, "cdl_b200_attn_decode", *swap(good, i, null(cdl, good[i])))
        assert st == -1 and "null pointer" in text, (i, st, text)


def sized(cdl, t, *shape):
    """A tensor's memory and strides with sizes that a C caller may give."""
    x = cdl._lib.CdlTensor.from_buffer_copy(cdl._lib.tensor_bytes(t))
    x.shape[:len(shape)] = shape
    return bytes(x)


def test_negative_sizes_are_refused(cdl):
    """(A negative number of heads came to a division by zero on the host.)"""
    L, good = cdl._lib, decode_call(cdl)
    heads = swap(swap(swap(good, 1, sized(cdl, good[1], 3, -2, 64)), 6, sized(cdl, good[6], 3, -2, 64)), 7, None)
    st, text = status(cdl, "cdl_b200_attn_decode", *heads)
    assert st == -1 and "multiple" in text
    n = L.ctypes.c_size_t(0)
    assert L.packed_lib.cdl_b200_attn_decode_scratch_bytes(heads[1], L.tensor_bytes(good[2]), L.ctypes.byref(n)) == -1
    plan = [16, 9, i32(4), i32(4), i32(4, 3), i32(9), i32(1), i32(4), i32(5), i32(7), i32(7), i32(1)]
    for i in range(2, 12):
        st, text = status(cdl, "cdl_b200_cache_plan", *swap(plan, i, sized(cdl, plan[i], -3)))
        assert st == -1 and "must be" in text, (i, st, text)
    write = [bf(5, 4, 32), bf(5, 2, 32), bf(5, 2, 32), torch.zeros(8, 32), i32(5), i32(5), bf(5, 4, 32), bf(5, 2, 32), bf(3, 4, 2, 32),
             bf(3, 4, 2, 32)]
    sample = [L.sample_bytes(1.0, 0, 1.0, 0.0), torch.zeros(4, 50), torch.zeros(4), torch.zeros(4), i32(4), torch.zeros(4), torch.zeros(4),
              i32(4), torch.zeros(4)]
    for name, args in (("cdl_b200_attn_decode", good), ("cdl_b200_cache_write", write), ("cdl_b200_sample", sample)):
        for i, t in enumerate(args):
            for d in range(t.dim() if isinstance(t, torch.Tensor) else 0):
                shape = list(t.shape)
                shape[d] = -shape[d]
                st, text = status(cdl, name, *swap(args, i, sized(cdl, t, *shape)))
                assert st in (-1, -2), (name, i, d, st, text)


def bad_scratch(device):
    block = torch.zeros(1 << 20, dtype=torch.uint8, device=device)
    return [block[:1].expand(1 << 20), block[::2], block.view(1024, 1024).t()]


def test_views_are_no_scratch(cdl, monkeypatch):
    """One byte expanded to a million is one byte of memory: what a kernel stored there went past its end."""
    from cleanlm_b200 import ops

    with pytest.raises(cdl._lib.CdlError, match="device memory"):
        ops._scratch_args(torch.zeros(16, dtype=torch.uint8))
    monkeypatch.setattr(ops, "_require_cuda", lambda *tensors: None)
    whole = torch.zeros(16, 4, dtype=torch.float32)
    assert ops._scratch_args(whole[4:]) == (whole[4:].data_ptr(), 192)
    for x in bad_scratch("cpu"):
        with pytest.raises(cdl._lib.CdlError, match="scratch must be contiguous"):
            ops._scratch_args(x)


@gpu
def test_calls_refuse_views_as_scratch(cdl, gpu_ok):
    ops, S = cdl.ops, cdl.serve
    rnd = lambda *s: torch.randn(*s, device="cuda").to(BF16)
    q, cache = rnd(2, 4, 64), rnd(5, 16, 2, 64)
    x, dy, scale = rnd(16, 256), rnd(16, 256), rnd(256)
    r_inv, dscale = torch.ones(16, device="cuda"), torch.zeros(256, device="cuda")
    a = [rnd(1, 128, 2, 128) for _ in range(5)] + [torch.zeros(1, 2, 128, device="cuda")]
    packed = [t[0] for t in a[:5]] + [torch.zeros(2, 128, device="cuda")]
    cu = ops.AttentionOpts(cu_seqlens_q=ints([0, 128]), cu_seqlens_k=ints([0, 128]))
    for scratch in bad_scratch("cuda") + [torch.zeros(1 << 20, dtype=torch.uint8)]:
        for call in (lambda: S.attention_decode(q, cache, cache, ints([[0, 1], [2, 3]]), ints([20, 9]), scratch=scratch),
                     lambda: ops.norm_bwd(x, dy, scale, r_inv, dscale, scratch=scratch),
                     lambda: ops.norm_bwd(x, dy, scale, r_inv, dscale, scratch=scratch, variant=1),
                     lambda: ops.attention_bwd(*a, scratch=scratch),
                     lambda: ops.attention_bwd(*packed, cu, scratch=scratch),
                     lambda: ops.linear_cross_entropy(x, rnd(256, 512), ints([3] * 16), scratch=scratch)):
            with pytest.raises(cdl._lib.CdlError, match="scratch must be contiguous|device memory|current device"):
                call()
    torch.cuda.synchronize()


def test_decode_refuses_scales_and_caps_that_f32_cannot_divide(cdl):
    """cap tanh(scale x / cap) with a quotient of infinity made NaN of a score of 0, and a cap whose product with log2 e is
    infinite of every score."""
    good = decode_call(cdl)
    desc = cdl._lib.attn_decode_bytes
    for scale, cap in ((0.0, 1e-45), (0.0, 1e-40), (0.0, 3e38), (0.0, 2e37), (1e-10, 1e30), (1e20, 1e-30), (3e38, 0.0), (1e38, 1.0)):
        st, text = status(cdl, "cdl_b200_attn_decode", *swap(good, 0, desc(scale, cap, 0)))
        assert st == -1 and "quotient" in text, (scale, cap, st, text)


@gpu
def test_decode_at_the_ends_of_scales_and_caps(cdl, gpu_ok):
    """The largest and smallest caps and scales that are taken: scores of 0 among others, nothing turns NaN; where the cap is far
    above the scores it is as if there were none, where it is far below all scores are alike."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(*s, generator=gen, device="cuda").to(BF16) for s in ((2, 4, 64), (9, 16, 4, 64), (9, 16, 4, 64)))
    q[:, 1] = 0
    table, lens = ints([[0, 1, 2, 3], [4, 5, 6, 7]]), ints([60, 33])

    def call(scale, cap):
        return cdl.serve.attention_decode(q, k, v, table, lens, cdl.serve.AttentionDecodeOpts(softmax_scale=scale, softcap=cap), lse=True)

    plain, flat = call(None, 0.0), call(1e-30, 0.0)
    for scale, cap, like in ((None, 1e37, plain), (None, 1e20, plain), (None, 1e-37, flat), (2.0 ** 126, 2.0 ** 126 / 2 ** 70, None),
                             (1e-37, 1.0, flat), (1e-20, 1e10, flat), (2.0 ** 126, 0.0, None)):
        got = call(scale, cap)
        assert not got.out[:, 1].isnan().any() and not got.lse[:, 1].isnan().any(), (scale, cap)
        if like is not None:
            # weights that differ by a few roundings of scores below 2^5: 2^-20, and bf16's rounding of p and of the result
            assert ((got.out.float() - like.out.float()).abs() <= 2.0 ** -6 * v.float().abs().max()).all(), (scale, cap)
            assert ((got.lse - like.lse).abs() <= 2.0 ** -18).all(), (scale, cap)


def write_status(cdl, k_cache, v_cache, tokens=0):
    """Of a call without tokens, which checks its operands and launches nothing."""
    heads, dim = k_cache.shape[2:]
    new = bf(tokens, heads, dim)
    return status(cdl, "cdl_b200_cache_write", None, new, new, None, None, i32(tokens), None, None, k_cache, v_cache)


def test_caches_that_share_a_tensor_are_told_apart(cdl):
    """Keys and values side by side in every order of pages, slots, heads and halves, also with one head, one page or one slot."""
    import itertools

    for sizes in ((3, 4, 2), (1, 4, 2), (3, 1, 2), (3, 4, 1), (1, 1, 1)):
        extent = dict(zip("psh", sizes), t=2)
        for order in itertools.permutations("psht"):
            whole = bf(*(extent[c] for c in order), 16).permute(*(order.index(c) for c in "tpsh"), 4)
            st, text = write_status(cdl, whole[0], whole[1])
            assert st == 0, (sizes, order, text)
            st, text = write_status(cdl, whole[0], whole[0])
            assert st == -1 and "overlap" in text, (sizes, order)


def test_no_views_that_share_elements_are_let_through(cdl):
    """Random views of one buffer: whatever is not refused has no element twice."""
    import random

    rng, buffer = random.Random(3), torch.zeros(1 << 14, dtype=BF16)
    taken = apart = 0
    for _ in range(20000):
        shape = [rng.choice([1, 2, 3]) for _ in range(3)] + [16]
        views, cells = [], []
        for _ in range(2):
            stride = [8 * rng.choice([0, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 96]) for _ in range(3)] + [1]
            start = 8 * rng.randrange(64)
            views.append(buffer.as_strided(shape, stride, start))
            cells.append([start + i * stride[0] + j * stride[1] + k * stride[2] + d for i in range(shape[0]) for j in range(shape[1])
                          for k in range(shape[2]) for d in range(16)])
        none_twice = len(set(cells[0] + cells[1])) == 2 * len(cells[0])
        apart += none_twice
        if write_status(cdl, *views)[0] == 0:
            taken += 1
            assert none_twice, [(v.shape, v.stride(), v.storage_offset()) for v in views]
    assert taken > 1000 and apart > taken


# --------------------------------------------------------------------------- sampling
def check_sample(cdl, z, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    got = cdl.serve.sample(z, u, cdl.serve.SampleOpts(temperature, top_k, top_p, min_p))
    zs, us = z.double().cpu().numpy(), u.tolist()
    for r in range(z.shape[0]):
        token, logprob = serve_ref.sample(zs[r], us[r], temperature, top_k, top_p, min_p)
        assert got.token[r].item() == token, r
        # rounded once to f32; the sum behind it is 2^-30 off at most
        assert abs(got.logprob[r].item() - logprob) <= 2.0 ** -24 * abs(logprob) + 2.0 ** -30
    return got


def allowed_only(rows, vocab, allowed, dtype, seed):
    """Logits of `allowed` tokens of a vocabulary, the others masked."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    z = torch.full((rows, vocab), -torch.inf, device="cuda")
    for r in range(rows):
        at = torch.randperm(vocab, generator=gen, device="cuda")[:allowed]
        z[r, at] = torch.randn(allowed, generator=gen, device="cuda") * 2.5
    return z.to(dtype), torch.rand(rows, generator=gen, device="cuda")


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,vocab", [(3, 5003), (5, 40000), (3, 66001)])
def test_sample_more_than_there_are(cdl, gpu_ok, rows, vocab, dtype):
    """top_k of as many entries as are not masked, one less, one more and far more: what it does not cut is as without it."""
    for allowed in (1, 600, 2048, 3000):
        z, u = allowed_only(rows, vocab, allowed, dtype, vocab + allowed)
        for more in ({}, {"top_p": 0.9}, {"top_p": 0.9, "min_p": 0.2}, {"min_p": 0.01}, {"top_p": 0.5, "temperature": 1e4}):
            base = cdl.serve.sample(z, u, cdl.serve.SampleOpts(**more))
            for k in (allowed - 1, allowed, allowed + 1, vocab - 1):
                got = check_sample(cdl, z, u, top_k=k, **more)
                if k >= allowed:
                    assert torch.equal(got.token, base.token) and torch.equal(got.logprob, base.logprob), (allowed, more, k)


@gpu
@pytest.mark.parametrize("allowed", [100, 20000])
def test_a_top_k_that_cuts_nothing_costs_no_search(cdl, gpu_ok, allowed):
    """A masked row with a larger top_k takes about as long as without it; one CTA searching alone took 30 times that."""
    z, u = allowed_only(4, 150001, allowed, F32, allowed)

    def us(**opts):
        opts = cdl.serve.SampleOpts(top_p=0.9, **opts)
        cdl.serve.sample(z, u, opts)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(5):
                cdl.serve.sample(z, u, opts)
        times = []
        for _ in range(10):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            graph.replay()
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b) * 200)
        return min(times)

    alone = us()
    assert us(top_k=max(allowed, 2000)) <= 4 * alone and us(top_k=150000) <= 4 * alone


# --------------------------------------------------------------------------- attention: how the work is shared
def decode_batch(batch, longest, heads, kv_heads, dim, page_size, seed):
    """Requests of 1 to `longest` keys in pages in random order; a table wider than 2048 keys."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda", dtype=F32)
    lens = 1 + torch.randperm(longest, generator=gen, device="cuda")[torch.arange(batch, device="cuda") % longest]
    count = (lens + page_size - 1) // page_size
    pages = int(count.sum())
    order, at = torch.randperm(pages, generator=gen, device="cuda"), 0
    table = torch.full((batch, max(longest, 2064) // page_size + 1), -1, dtype=I32, device="cuda")
    for b, n in enumerate(count.tolist()):
        table[b, :n] = order[at:at + n]
        at += n
    k, v = (torch.empty(pages, page_size, kv_heads, dim, dtype=BF16, device="cuda") for _ in range(2))
    for c in (k, v):
        for i in range(0, pages, 4096):
            c[i:i + 4096] = rnd(*c[i:i + 4096].shape).to(BF16)
    return (2 * rnd(batch, heads, dim)).to(BF16), k, v, table, lens.to(I32)


def check_batch(cdl, q, k, v, table, lens):
    """Against the definition in 64 bits, request by request on the GPU; the bounds are those of the roundings of a score's sum of
    dim products and its scale, of p and of the result to bf16, and of the sum over n keys."""
    made = [cdl.serve.attention_decode(q, k, v, table, lens, lse=True)]
    if int(lens.max()) <= 2048:  # the form for tables of so few keys too
        made.append(cdl.serve.attention_decode(q, k, v, table[:, :2048 // k.shape[1]], lens, lse=True))
    group, dim, page_size = q.shape[1] // k.shape[2], q.shape[2], k.shape[1]
    assert table.shape[1] * page_size > 2048
    out, spread = torch.empty(q.shape, dtype=torch.float64, device="cuda"), torch.empty(q.shape, dtype=torch.float64, device="cuda")
    lse, reach = (torch.empty(q.shape[:2], dtype=torch.float64, device="cuda") for _ in range(2))
    for b, n in enumerate(lens.tolist()):
        at = table[b, :-(-n // page_size)].long()
        kb, vb = (c[at].flatten(0, 1)[:n].double().transpose(0, 1) for c in (k, v))  # [kv_heads, n, dim]
        qb = q[b].double().view(-1, group, dim) * dim ** -0.5
        s = qb @ kb.transpose(1, 2)
        reach[b] = (qb.abs() @ kb.abs().transpose(1, 2)).amax(2).flatten()
        lse[b] = s.logsumexp(2).flatten()
        p = s.softmax(2)
        out[b], spread[b] = (p @ vb).view(-1, dim), (p @ vb.abs()).view(-1, dim)
    n = lens.double()[:, None]
    off = (dim + 8) * 2.0 ** -24 * reach + 2.0 ** -20
    bound = 2.0 ** -8 * (out.abs() + spread) + (2 * off + n * 2.0 ** -24)[..., None] * spread
    for got in made:
        assert ((got.out.double() - out).abs() <= bound).all()
        assert ((got.lse.double() - lse).abs() <= off + n * 2.0 ** -24 + 2.0 ** -22 * lse.abs()).all()


@gpu
@pytest.mark.parametrize("batch,longest,heads,kv_heads,dim,page_size", [
    (64, 4096, 16, 16, 128, 16),   # 131000 tiles, 444 CTAs at once: more than 192 each, so there is a second set of parts
    (64, 4096, 192, 16, 64, 16),   # 65000 tiles, 12 heads per kv head: 296 at once
    (24, 9001, 32, 8, 128, 7),     # lines that several CTAs share, in both sets
    (575, 700, 4, 2, 64, 16), (576, 700, 4, 2, 64, 16),    # as many requests as leave an SM room for three CTAs, and one more
    (1700, 300, 2, 2, 128, 16), (4096, 130, 2, 1, 64, 8),  # two CTAs an SM
    (4096, 500, 8, 2, 64, 16),     # in two sets of parts
    (2, 700, 2048, 1, 64, 16), (3, 400, 1000, 8, 128, 5),  # groups of 2048 and 125
])
def test_decode_batches(cdl, gpu_ok, batch, longest, heads, kv_heads, dim, page_size):
    check_batch(cdl, *decode_batch(batch, longest, heads, kv_heads, dim, page_size, seed=batch + dim))


def test_shares_cover_all_tiles_once(tmp_path):
    """The kernel's own arithmetic of who has which tile, compiled for the host: parts follow one another from 0 to the last tile, none
    is empty, and the CTA that a tile is looked up for is the one whose part it is in."""
    import shutil
    import subprocess
    from pathlib import Path

    source = (Path(__file__).resolve().parent.parent / "clean-lm_b200" / "csrc" / "attn_decode.cu").read_text()
    start = source.index("constexpr int SETS")
    shares = source[start:source.index("\n};\n", start) + 4]
    (tmp_path / "shares.cpp").write_text("""
#include <cstdio>
#include <initializer_list>
#define __host__
#define __device__
#define __forceinline__ inline
""" + shares + """
int main() {
  for (int set : {1, 2, 3, 148, 296, 444}) {
    const long long edge = 192LL * set;
    for (long long n : {1LL, 2LL, set - 1LL, (long long)set, set + 1LL, 7LL * set, edge - 1, edge, edge + 1, edge + 12345, 3 * edge + 7,
                        (1LL << 31) + 5, 1LL << 40}) {
      if (n < 1) continue;
      const Shares s(n, set);
      if (s.ctas < 1 || s.ctas > SETS * set || s.begin(0) != 0 || s.begin(s.ctas) != n) return printf("ends %d %lld\\n", set, n), 1;
      if ((s.ctas > set) != (n >= edge)) return printf("sets %d %lld\\n", set, n), 1;
      for (int c = 0; c < s.ctas; ++c) {
        const long long a = s.begin(c), b = s.begin(c + 1);
        if (b <= a) return printf("empty %d %lld %d\\n", set, n, c), 1;
        for (long long u : {a, a + 1, (a + b) / 2, b - 1})
          if (u < b && s.of(u) != c) return printf("of %d %lld %lld\\n", set, n, u), 1;
      }
    }
  }
  return 0;
}
""")
    compiler = shutil.which("g++")
    assert compiler, "a host compiler is part of the toolkit's requirements"
    subprocess.run([compiler, "-O2", "-std=c++17", "-o", str(tmp_path / "shares"), str(tmp_path / "shares.cpp")], check=True)
    run = subprocess.run([str(tmp_path / "shares")], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout


# --------------------------------------------------------------------------- sizes
@gpu
@pytest.mark.parametrize("tokens,heads,kv_heads,dim", [(1, 1, 1, 2048), (7, 3, 2, 1040), (5, 300, 1, 16), (9, 2, 70, 48), (40, 16, 4, 128), (3, 0, 2, 64)])
def test_write_element_by_element(cdl, gpu_ok, tokens, heads, kv_heads, dim):
    """Head sizes up to the largest and any number of heads; each element within its own roundings."""
    gen = torch.Generator(device="cuda").manual_seed(dim + tokens)
    qkv = torch.randn(tokens, heads + 2 * kv_heads, dim, generator=gen, device="cuda").to(BF16)
    q, k, v = qkv.split([heads, kv_heads, kv_heads], 1)
    caches = [torch.full((4, 11, kv_heads, dim), 7.0, dtype=BF16, device="cuda") for _ in range(2)]
    slots = torch.randperm(44, generator=gen, device="cuda")[:tokens]
    positions = torch.randint(0, 900, (tokens,), generator=gen, device="cuda")
    table = cdl.sky1.rope_table(900, dim)
    k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    got = cdl.serve.cache_write(k, v, slots.to(I32), *caches, q=q, table=table, positions=positions.to(I32), k_out=k_out)
    cos, sin = (x[:, None] for x in table[positions].double().split(dim // 2, 1))

    def near(have, x):
        lo, hi = x.double().split(dim // 2, 2)
        want = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], 2)
        size = torch.cat([(lo * cos).abs() + (hi * sin).abs(), (hi * cos).abs() + (lo * sin).abs()], 2)
        # half a step of bf16, and f32's of two products and their sum
        assert ((have.double() - want).abs() <= 2.0 ** -8 * want.abs() + 4 * 2.0 ** -24 * size).all()

    near(got.q, q)
    near(got.k, k)
    k_flat, v_flat = (c.flatten(0, 1) for c in caches)
    assert torch.equal(k_flat[slots], got.k) and torch.equal(v_flat[slots], v)
    rest = torch.ones(44, dtype=torch.bool, device="cuda")
    rest[slots] = False
    assert (k_flat[rest] == 7).all() and (v_flat[rest] == 7).all()


@gpu
def test_plan_of_160000_requests(cdl, gpu_ok):
    """More rounds of 1024 requests than there are CTAs, with a table that is a part of a wider one."""
    rng, requests, page_size, pages = np.random.default_rng(1), 160001, 4, 400000
    cached, added = rng.integers(0, 6, requests), rng.integers(0, 3, requests)
    used = -(-cached // page_size)
    order = rng.permutation(pages)
    table = np.full((requests, 2), -1)
    mine = np.arange(2)[None] < used[:, None]
    table[mine] = order[:mine.sum()]
    stack = order[mine.sum():][:60000]
    rows = int(added.sum()) - 5
    want = serve_ref.cache_plan(cached.tolist(), added.tolist(), table.tolist(), stack.tolist(), len(stack), page_size, pages, rows)
    wide = torch.full((requests, 5), 9, dtype=I32, device="cuda")
    wide[:, :2] = ints(table)
    got = cdl.serve.cache_plan(ints(cached), ints(added), wide[:, :2], ints(stack), ints([len(stack)]),
                               cdl.serve.CachePlanOpts(page_size, pages, rows))
    have = (got.seq_lens, got.cu_seqlens, got.positions, got.slots, got.free_left, wide[:, :2])
    for name, g, w in zip(("seq_lens", "cu_seqlens", "positions", "slots", "free_left", "block_table"), have, want):
        assert torch.equal(g.cpu(), torch.tensor([w] if name == "free_left" else w, dtype=I32)), name
    assert (wide[:, 2:] == 9).all()


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_sample_of_three_million(cdl, gpu_ok, dtype):
    gen = torch.Generator(device="cuda").manual_seed(4)
    z = (torch.randn(2, 3000017, generator=gen, device="cuda") * 3).to(dtype)
    u = torch.tensor([0.3, 0.9999], device="cuda")
    for opts in ({}, {"top_p": 0.8}, {"top_k": 50}, {"top_k": 3000}, {"min_p": 1e-3}, {"temperature": 0.0}):
        check_sample(cdl, z, u, **opts)


@gpu
def test_sample_of_odd_random_numbers(cdl, gpu_ok):
    """Numbers outside [0, 1) beside ones inside, each row against the definition."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    z = torch.randn(10, 700, generator=gen, device="cuda")
    u = torch.tensor([-1.0, float("nan"), 1.0, 2.0, torch.inf, -torch.inf, 0.0, 0.5, 1 - 2.0 ** -24, 2.0 ** -140], device="cuda")
    check_sample(cdl, z, u)
    check_sample(cdl, z, u, top_k=30, top_p=0.8)


# --------------------------------------------------------------------------- threads
@gpu
def test_steps_of_several_threads(cdl, gpu_ok):
    """A step's four calls from four threads at once, each on its stream with a batch of its own size: the bits of the same calls one
    thread after the other."""
    import threading

    S, sizes = cdl.serve, (1, 60, 700, 2500)

    def inputs(batch):
        gen = torch.Generator(device="cuda").manual_seed(batch)
        rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
        q, k, v, table, lens = decode_batch(batch, 250, 4, 2, 64, 16, seed=batch)
        pages = k.shape[0] + batch
        k, v = (torch.cat([c, torch.zeros(batch, 16, 2, 64, dtype=BF16, device="cuda")]) for c in (k, v))
        stack = torch.arange(k.shape[0] - batch, k.shape[0], device="cuda").to(I32)
        return (rnd(batch, 8, 64).to(BF16), k, v, table, lens, torch.ones(batch, dtype=I32, device="cuda"), stack, ints([batch]), pages,
                rnd(batch, 5000), torch.rand(batch, generator=gen, device="cuda"), cdl.sky1.rope_table(260, 64))

    def step(qkv, k, v, table, lens, one, stack, count, pages, z, u, rope):
        table, k, v = table.clone(), k.clone(), v.clone()
        p = S.cache_plan(lens, one, table, stack, count, S.CachePlanOpts(16, pages, len(lens)))
        w = S.cache_write(qkv[:, 4:6], qkv[:, 6:], p.slots, k, v, q=qkv[:, :4], table=rope, positions=p.positions)
        a = S.attention_decode(w.q, k, v, table, p.seq_lens, lse=True)
        short = S.attention_decode(w.q, k, v, table[:, :20], p.seq_lens)
        t = S.sample(z, u, S.SampleOpts(top_p=0.9))
        return p.slots, p.free_left, k, v, a.out, a.lse, short.out, t.token, t.logprob

    data = [inputs(n) for n in sizes]
    want = [step(*x) for x in data]
    torch.cuda.synchronize()
    got, errors, start = [None] * len(sizes), [], threading.Barrier(len(sizes))

    def worker(i):
        try:
            torch.cuda.set_device(0)
            stream = torch.cuda.Stream()
            start.wait()
            with torch.cuda.stream(stream):
                for _ in range(10):
                    got[i] = step(*data[i])
            stream.synchronize()
        except Exception as e:  # raised below
            errors.append(e)

    threads = [threading.Thread(target=worker, args=(i,)) for i in range(len(sizes))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for w, g in zip(want, got):
        assert all(torch.equal(a, b) for a, b in zip(w, g))


def uneven(z, kind):
    """Logits whose parts a row's CTAs and threads find unlike: a masked or low range of the vocabulary, logits in order, equal ones."""
    z, vocab = z.clone(), z.shape[1]
    if kind == "half":
        z[:, vocab // 2:] = -torch.inf
    elif kind == "front":
        z[:, :vocab // 3] = -torch.inf
    elif kind == "low":
        z[:, vocab // 4:vocab // 2] -= 20
    elif kind == "order":
        z = z.float().sort(1, descending=True)[0].to(z.dtype)
    elif kind == "alike":  # the k-th has thousands of equals, in a few parts
        z[:, :vocab // 4], z[:, vocab // 4:] = 4.0, -5.0
    return z


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,vocab", [(3, 9001), (2, 40001), (3, 150001), (50, 66001), (100, 33000)])
def test_sample_top_k_of_uneven_rows(cdl, gpu_ok, rows, vocab, dtype):
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    z, u = (torch.randn(rows, vocab, generator=gen, device="cuda") * 2.5).to(dtype), torch.rand(rows, generator=gen, device="cuda")
    pick = torch.tensor([0, rows - 1], device="cuda")
    for kind in ("half", "front", "low", "order", "alike"):
        x = uneven(z, kind)
        for opts in ({"top_k": 1}, {"top_k": 50}, {"top_k": 300, "top_p": 0.8}, {"top_k": 384, "min_p": 0.2}, {"top_k": 1100}, {"top_k": 1024, "top_p": 0.9}):
            whole = cdl.serve.sample(x, u, cdl.serve.SampleOpts(**opts))
            some = check_sample(cdl, x[pick], u[pick], **opts)
            assert torch.equal(whole.token[pick], some.token) and torch.equal(whole.logprob[pick], some.logprob), (kind, opts)


@gpu
def test_top_k_of_a_masked_vocabulary_costs_no_search(cdl, gpu_ok):
    """Half the vocabulary masked, or a top_k of which three or four CTAs' bounds leave too many entries: a few passes more, where one
    CTA searching alone took 10 to 60 times as long."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    z, u = torch.randn(4, 150001, generator=gen, device="cuda") * 2.5, torch.rand(4, generator=gen, device="cuda")

    def us(x, **opts):
        opts = cdl.serve.SampleOpts(**opts)
        cdl.serve.sample(x, u, opts)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(5):
                cdl.serve.sample(x, u, opts)
        times = []
        for _ in range(10):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            graph.replay()
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b) * 200)
        return min(times)

    base = us(z, top_k=50)
    assert us(uneven(z, "half"), top_k=50) <= 6 * base and us(uneven(z, "half"), top_k=50, top_p=0.9) <= 6 * base
    assert us(z, top_k=1300) <= 3 * us(z, top_k=1600)
