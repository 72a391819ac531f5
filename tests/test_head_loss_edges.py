"""Losses of the head where values are extreme: whole slices of a row masked, differences of logits that a temperature makes
large.  The restatements in 64 bits are those of test_head_loss.py; tolerances are derived where they stand."""
import pytest
import torch

from oracle import head_loss_ref as ref
from test_head_loss import (BF16, F32, HALF, _check_distillation, _check_linear, _close, _entries, _hit, _operands, _stat)

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab,pad", [(9000, 0), (9001, 2), (40000, 8), (150000, 0)])
@pytest.mark.parametrize("tau,level", [(1.0, -200.0), (0.1, -14.0), (2.5, -3000.0)])
def test_distillation_slices_without_a_logit(cdl, gpu_ok, dtype, vocab, pad, tau, level):
    """Slices of a row (each has its own maximum) in which every logit is -inf, beside others that lie far below 0."""
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    rows = 7
    logits = (torch.randn(rows, vocab + pad, generator=gen, device="cuda") * 3 * tau + level).to(dtype)[:, :vocab]
    half = vocab // 2
    logits[0, half:] = float("-inf")
    logits[1, :half] = float("-inf")
    logits[2, vocab // 4:] = float("-inf")
    logits[3, : vocab - 20] = float("-inf")
    logits[4, 20:] = float("-inf")
    live = [(0, half), (half, vocab), (0, vocab // 4), (vocab - 20, vocab), (0, 20), (0, vocab), (0, half)]
    ids = torch.stack([torch.randint(a, b, (9,), generator=gen, device="cuda") for a, b in live]).to(torch.int32)
    teacher = torch.randn(rows, 9, generator=gen, device="cuda") * 3 * tau
    logits[6, half:] = float("-inf")
    o = _check_distillation(cdl, logits, ids, teacher, tau)
    assert bool(torch.isfinite(o.loss).all()) and bool((o.d_logits[0, half:] == 0).all())
    # what makes a row NaN makes its masked slices NaN, too
    logits[6, 3] = float("nan")
    logits[5] = float("-inf")
    o = cdl.ops.distillation(logits, ids, teacher, cdl.ops.DistillationOpts(temperature=tau))
    assert bool(torch.isnan(o.d_logits[5:]).all()) and bool(torch.isnan(o.loss[5:]).all())
    assert bool(torch.isfinite(o.d_logits[:5]).all())


@gpu
@pytest.mark.parametrize("t,v,layout", [(40, 1000, "rows"), (100, 5000, "tied"), (300, 4099, "rows"), (513, 1000, "tied")])
@pytest.mark.parametrize("tau,far", [(1e-6, 1.0), (1e-4, 1.0), (0.5, 2.0 ** 19), (1.0, 2.0 ** 20), (1e6, 2.0 ** 27)])
def test_linear_losses_of_far_logits(cdl, gpu_ok, t, v, layout, tau, far):
    """bf16 operands whose logits are sums of two values, b + k u with u near 4 tau, that 24 bits hold: exact in any order of
    summation, so that all errors are the loss's own.  |z| log2(e) / tau reaches 2^25, where the last place is 4, and the
    softmax is set by differences of a few u.

    Differences are exact; times log2(e) / tau, a factor off by 2^-22, those that count (probabilities above 2^-40) are off by 40 2^-22 =
    2^-17 at most in the exponent, so a probability by 2^-17 of itself, and from its sum by what _stat has.  d z is rounded to f16 and
    bf16 (2 * 2^-8)."""
    gen = torch.Generator(device="cuda").manual_seed(t + v)
    u = 2.0 ** round(torch.log2(torch.tensor(4 * tau)).item())
    coarse = torch.tensor([0.0, 12.0, -12.0, 24.0, -24.0, 30.0, -30.0, 28.0]) * far
    d = 64
    w = torch.randint(-64, 65, (d, v), generator=gen, device="cuda") * u
    w[:8] = coarse.cuda()[:, None]
    x = torch.zeros(t, d, device="cuda")
    rows = torch.arange(t, device="cuda")
    x[rows, rows % 8] = 1.0
    x[rows, torch.randint(8, d, (t,), generator=gen, device="cuda")] = 1.0
    x, w = x.to(BF16), w.to(BF16)
    assert torch.equal((x.double() @ w.double()).float().double(), x.double() @ w.double())
    if layout == "tied":
        w = w.t().contiguous().t()
    k = 20
    ids = torch.randint(0, v, (t, k), generator=gen, device="cuda", dtype=torch.int32)
    teacher = torch.randn(t, k, generator=gen, device="cuda") * 2 * tau
    ids[3:5, 1] = ids[3:5, 0]
    ids[5] = -1
    best = (x.double() @ w.double()).argmax(1).to(torch.int32)
    ids[6::5, 2] = best[6::5]
    forms = [((ids, teacher), cdl.ops.linear_distillation, lambda z: ref.distillation(z, ids, teacher, tau))]
    if tau == 1.0:
        targets = torch.where(rows % 3 == 0, best, ids[:, 3])
        forms.append(((targets,), cdl.ops.linear_cross_entropy, lambda z: ref.cross_entropy(z, targets)))
    for entries, fn, loss_of in forms:
        loss, lse, g, dx, dw = ref.linear(x, w, loss_of)
        o = fn(x, w, *entries, cdl.ops.LinearLossOpts(temperature=tau))
        _close("lse", o.lse, lse, 3 * _stat(v) + 2.0 ** -21 * lse.abs())
        # log q at an entry is a difference of up to 2 * 64 u = 512 tau or so: 2^-21 of it
        _close("loss", o.loss, loss, tau * tau * (6 * _stat(v) + 2.0 ** -21 * 1200 + 0 * loss))
        hit = _hit(entries[0] if len(entries) > 1 else entries[0][:, None], v)
        keep = (g != 0).any(1)[:, None]
        p_err = 2 * (_stat(v) + 2.0 ** -17)
        g_err = torch.where(keep, 2 * HALF[BF16] * g.abs() + p_err * (g.abs() + tau * hit) + 2.0 ** -30 * tau, 0.0)
        sums = 2.0 ** -23 * 40
        _close("dx", o.dx, dx, (g_err + sums * g.abs()) @ w.double().abs().t() + HALF[BF16] * dx.abs() + 1e-30)
        _close("dw", o.dw, dw, x.double().abs().t() @ (g_err + sums * g.abs()) + (HALF[BF16] + 2.0 ** -22) * dw.abs() + 1e-30)


@gpu
@pytest.mark.parametrize("t", [3, 130])
@pytest.mark.parametrize("d", [4096, 4097, 1 << 18])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_logits_of_long_sums(cdl, gpu_ok, t, d, sign):
    """Positive terms, which lose the most in an accumulator that truncates: 2^-23 of the sum in each of 256 steps of 16 and 8 more, which
    is all that one takes, then one rounding to nearest per 4096 terms.  What is put back is less.  (One accumulator for 2^18 terms was
    1.4e-3 off.)"""
    gen = torch.Generator(device="cuda").manual_seed(d)
    x = torch.rand(t, d, generator=gen, device="cuda").to(BF16)
    w = (torch.rand(d, 1, generator=gen, device="cuda") * sign / d * 64).to(BF16)
    w = torch.cat([w, -w], 1)
    z = x.double() @ w.double()
    targets = torch.arange(t, device="cuda", dtype=torch.int32) % 2
    o = cdl.ops.linear_cross_entropy(x, w, targets, cdl.ops.LinearLossOpts(grad=False))
    off = (264 * 2.0 ** -23 + (d // 4096 + 2) * 2.0 ** -24) * z.abs().amax(1)
    loss, lse, _ = ref.cross_entropy(z, targets)
    _close("lse", o.lse, lse, off + 2.0 ** -20)
    _close("loss", o.loss, loss, 2 * off + 2.0 ** -20 * (1 + loss))


@gpu
@pytest.mark.parametrize("t,d,v,k", [(5, 4097, 300, 0), (130, 8200, 700, 3), (700, 8264, 3001, 0), (1300, 12352, 2000, 9), (100, 20000, 520, 0)])
def test_linear_losses_of_wide_hidden_states(cdl, gpu_ok, t, d, v, k):
    """Logits that several accumulators make up, tile after tile."""
    gen = torch.Generator(device="cuda").manual_seed(t + d)
    x, w = _operands(gen, t, d, v, BF16, "rows")
    entries = _entries(gen, t, v, k)
    opts = cdl.ops.LinearLossOpts(temperature=1.0 if k == 0 else 1.7)
    o = _check_linear(cdl, x, w, entries, opts)
    fn = cdl.ops.linear_cross_entropy if k == 0 else cdl.ops.linear_distillation
    again = fn(x, w, *entries, opts)
    assert torch.equal(o.loss, again.loss) and torch.equal(o.dx, again.dx) and torch.equal(o.dw, again.dw)


@gpu
@pytest.mark.parametrize("n", [1, 3, 7, 9, 100, 127, 129, 200, 1101])
@pytest.mark.parametrize("t", [20, 300])
def test_weight_gradient_leaves_what_lies_behind_its_rows(cdl, gpu_ok, n, t):
    """Rows on the 16-byte grid that end inside 16 bytes: the columns behind them belong to something else."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    vocab = 40000
    x, w = _operands(gen, t, n, vocab, BF16, "tied")
    buffer = torch.full((vocab, (n + 7) // 8 * 8 + 8), 7.0, dtype=BF16, device="cuda")
    view = buffer[:, :n]
    _check_linear(cdl, x, w, _entries(gen, t, vocab, 0), cdl.ops.LinearLossOpts(), dw=view.t())
    view.fill_(7.0)
    assert bool((buffer == 7.0).all())


def _strided(extents, strides, dtype, device="cpu"):
    """A view of these strides in a buffer of its own, filled with 7, and the buffer."""
    buffer = torch.full((sum((n - 1) * s for n, s in zip(extents, strides)) + 1,), 7.0, dtype=dtype, device=device)
    return buffer.as_strided(extents, strides), buffer


ONE_WIDE = [((1, 3000), (12000, 4)), ((1, 3000), (24000, 8)), ((1, 3000), (3, 3)), ((1, 100000), (800000, 8)), ((1, 3000), (1, 1)),
            ((900, 1), (4, 1000)), ((900, 1), (8, 7200)), ((900, 1), (1, 5)), ((900, 1), (3, 1)), ((1, 1), (5, 9))]


@pytest.mark.parametrize("extents,strides", ONE_WIDE)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_stride_of_an_extent_of_one_does_not_matter(cdl, extents, strides, dtype):
    """The same memory described in several ways is one plan: one size of the scratch."""
    sizes = set()
    for other in (1, 4, 8, 1000, 800000):
        view = tuple(other if n == 1 else s for n, s in zip(extents, strides))
        w, _ = _strided(extents, view, dtype)
        x = torch.zeros(20, extents[0], dtype=dtype)
        sizes.add((cdl.ops.linear_loss_scratch_bytes(x, w, dx=x, dw=w), cdl.ops.linear_loss_scratch_bytes(x, w.contiguous(), dx=x, dw=w)))
    assert len(sizes) == 1


@gpu
@pytest.mark.parametrize("extents,strides", ONE_WIDE)
@pytest.mark.parametrize("dtype,out", [(BF16, BF16), (BF16, F32), (F32, F32)])
@pytest.mark.parametrize("t", [5, 20, 300])
def test_one_hidden_or_one_token_id_in_any_strides(cdl, gpu_ok, extents, strides, dtype, out, t):
    """Heads of one hidden value or one token id; nothing is written beyond the scratch that is asked for, nor between the
    elements of dw."""
    gen = torch.Generator(device="cuda").manual_seed(t)
    d, v = extents
    x = torch.randn(t, d, generator=gen, device="cuda").to(dtype)
    w, _ = _strided(extents, strides, dtype, "cuda")
    w.copy_(torch.randn(d, v, generator=gen, device="cuda"))
    entries = _entries(gen, t, v, 0)
    for accumulate in (False, True):
        dw, buffer = _strided(extents, strides, out, "cuda")
        before = dw.clone() if accumulate else None
        n = cdl.ops.linear_loss_scratch_bytes(x, w, cdl.ops.LinearLossOpts(accumulate=accumulate), dx=x, dw=dw)
        scratch = torch.full((n + (1 << 20),), 90, dtype=torch.uint8, device="cuda")
        _check_linear(cdl, x, w, entries, cdl.ops.LinearLossOpts(accumulate=accumulate), dw=dw, before=before, scratch=scratch[:n])
        assert bool((scratch[n:] == 90).all())
        dw.fill_(7.0)
        assert bool((buffer == 7.0).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_dx_in_place_of_x_has_its_strides(cdl, dtype):
    """Another stride from the same address: rows of x that a later chunk of rows reads would be overwritten."""
    buffer, w = torch.zeros(20, 48, dtype=dtype), torch.zeros(16, 40, dtype=dtype)
    size = cdl.ops.linear_loss_scratch_bytes
    x = buffer[:, :16]
    dense = buffer.flatten()[:320].view(20, 16)
    assert size(x, w, dx=x) > 0 and size(dense, w, dx=dense) > 0 and size(x[:1], w, dx=dense[:1]) > 0
    assert size(x, w, dx=torch.zeros(20, 16, dtype=dtype)) > 0 and size(x.t()[:0, :16], w, dx=x[:0]) == 0
    for a, b in ((x, dense), (dense, x), (buffer.flatten()[:320].view(16, 20).t(), dense)):
        with pytest.raises(cdl._lib.CdlError, match="dx must be x itself or lie elsewhere"):
            size(a, w, dx=b)


def test_loss_alone_is_not_taken_apart_for_gradients_that_are_not_wanted(cdl):
    """Without gradients the scratch holds statistics, not exponentials: many more rows fit into the same bytes."""
    def size(t, d, v, dtype, entries, chunk):
        x, w = torch.zeros(1, 1, dtype=dtype).expand(t, d), torch.zeros(1, 1, dtype=dtype).expand(d, v)
        return cdl.ops.linear_loss_scratch_bytes(x, w, cdl.ops.LinearLossOpts(chunk_rows=chunk), entries=entries)

    for t, d, v, dtype, entries in ((65536, 256, 32768, BF16, 1), (200000, 64, 32768, BF16, 1), (65536, 256, 32768, BF16, 64),
                                    (2000, 128, 100000, F32, 1)):
        assert size(t, d, v, dtype, entries, 0) == size(t, d, v, dtype, entries, t)
    # still bounded, whatever else a row holds
    operands = lambda t, d, v: 2 * (t * ((d + 7) // 8 * 8) + d * (v + 7))  # noqa: E731  (laid out anew)
    for t, d, v, entries in ((1 << 20, 64, 128, 1024), (1 << 24, 8, 1000, 3), (1 << 22, 8, 150000, 256)):
        assert size(t, d, v, BF16, entries, 0) <= (1 << 30) * 1.01 + operands(t, d, v)


@gpu
@pytest.mark.parametrize("t,d,v,k,dtype", [(500000, 16, 32768, 0, BF16), (300000, 16, 32768, 5, BF16), (3000, 16, 100001, 0, F32)])
def test_loss_alone_of_many_tokens(cdl, gpu_ok, t, d, v, k, dtype):
    """More than one chunk of rows, and as many as the caller asks for: the same statistics."""
    gen = torch.Generator(device="cuda").manual_seed(t)
    x, w = _operands(gen, t, d, v, dtype, "rows")
    entries = _entries(gen, t, v, k)
    fn = cdl.ops.linear_cross_entropy if k == 0 else cdl.ops.linear_distillation
    o = fn(x, w, *entries, cdl.ops.LinearLossOpts(grad=False))
    p = fn(x, w, *entries, cdl.ops.LinearLossOpts(grad=False, chunk_rows=1024 if dtype == F32 else 1 << 16))
    assert torch.equal(o.loss, p.loss) and torch.equal(o.lse, p.lse)
    rows = torch.cat([torch.arange(64), torch.arange(t - 64, t)]).cuda()
    _check_linear(cdl, x[rows], w, [e[rows] for e in entries], cdl.ops.LinearLossOpts(grad=False))
    want = fn(x[rows], w, *[e[rows] for e in entries], cdl.ops.LinearLossOpts(grad=False))
    _close("loss", o.loss[rows], want.loss, 2.0 ** -18 * (1 + want.loss.abs()))


# ------------------------------------------------------------------------------------------ what f32 operands keep
def _leading(v, bits):
    """f32 values cut off behind their first 8, 16 or 24 bits: one, two or three bf16 pieces."""
    return (v.view(torch.int32) & -(1 << (24 - bits))).view(torch.float32)


@gpu
@pytest.mark.parametrize("t", [20, 200])
@pytest.mark.parametrize("of_x,of_w", [(8, 24), (24, 8), (16, 16), (16, 8), (8, 16)])
def test_each_product_of_pieces_counts(cdl, gpu_ok, t, of_x, of_w):
    """The logsumexp of one token id is its logit.  With x and w of one to three pieces, positive, and every lower piece large, each of
    the products (0, 2), (2, 0), (1, 1), (1, 0), (0, 1) is 2^-17 of the logit and more, and those that are left out, (1, 2), (2, 1), (2, 2), are
    none.  Six steps of an accumulator cut 2^-23 each, putting back and rounding adds as much as two more."""
    gen = torch.Generator(device="cuda").manual_seed(t)

    def values(*shape, bits):  # 1.x with the first bits of every piece set
        v = torch.randint(0, 1 << 23, shape, generator=gen, device="cuda", dtype=torch.int32) | 0x3f80c0c0
        return _leading(v.view(torch.float32), bits)

    x, w = values(t, 16, bits=of_x), values(16, 1, bits=of_w)
    o = cdl.ops.linear_cross_entropy(x, w, torch.zeros(t, dtype=torch.int32, device="cuda"))
    z = (x.double() @ w.double())[:, 0]
    lower = [(a.double() - _leading(a, 8)) for a in (x, w)]
    assert ((lower[0] @ w.double())[:, 0].min() > 0) == (of_x > 8) and ((x.double() @ lower[1])[:, 0].min() > 0) == (of_w > 8)
    _close("lse", o.lse, z, 8 * 2.0 ** -23 * z)


@gpu
@pytest.mark.parametrize("t,d,v,layout", [(300, 200, 1500, "rows"), (100, 333, 2001, "tied"), (40, 600, 900, "rows"), (700, 515, 8190, "tied")])
def test_f32_gradients_in_the_2_norm(cdl, gpu_ok, t, d, v, layout):
    """Logits below 4: their rounding, the exponential's and the sum's leave d z 2^-20 off, the products of pieces and their sums 2^-22, the
    result's rounding less.  2^-19 in all; without any one of the six products of pieces it would be 8e-6 (four times as much)."""
    gen = torch.Generator(device="cuda").manual_seed(t + d)
    x, w = _operands(gen, t, d, v, F32, layout)
    targets = _entries(gen, t, v, 0)[0]
    o = cdl.ops.linear_cross_entropy(x, w, targets)
    _, _, _, dx, dw = ref.linear(x, w, lambda z: ref.cross_entropy(z, targets.long()))
    assert (o.dx - dx).norm() <= 2.0 ** -19 * dx.norm() and (o.dw - dw).norm() <= 2.0 ** -19 * dw.norm()


@gpu
@pytest.mark.parametrize("t", [40, 159])
def test_f32_gradient_with_a_large_first_term_is_as_good_as_f32_products(cdl, gpu_ok, t):
    """dx is the target's column and what 43583 small terms add.  In the accumulator of the first 256 of K some 16 steps behind the target's
    cut half a unit each on average, 0.7 2^-23 of the value on average over a binade: 11.5 2^-24; 4.3 2^-24 is put back.  171 parts rounded
    to nearest, independently: 3 2^-24.  8 2^-24 in the 2-norm, where one accumulator for all of K loses 22 (and f32 products 10)."""
    gen = torch.Generator(device="cuda").manual_seed(12)
    x = torch.randn(t, 576, generator=gen, device="cuda")
    w = torch.randn(576, 43584, generator=gen, device="cuda") * 0.02
    targets = torch.zeros(t, dtype=torch.int32, device="cuda")
    o = cdl.ops.linear_cross_entropy(x, w, targets)
    _, _, _, dx, _ = ref.linear(x, w, lambda z: ref.cross_entropy(z, targets.long()))
    assert ((o.dx - dx).norm() / dx.norm()).item() <= 10 * 2.0 ** -24


@gpu
def test_language_model_without_stored_logits_keeps_no_buffer_for_them(cdl, gpu_ok):
    sky1 = cdl.sky1
    blk = sky1.Sky1Config(batch=1, seqlen=128, hidden=128, heads=1, kv_heads=1, head_dim=128, ffn=256)
    m = sky1.Sky1LM(sky1.Sky1LMConfig(block=blk, layers=1, vocab=512, keep_logits=False), seed=4)
    assert m.logits is None and m.loss_tok is None
    tokens = torch.arange(128, dtype=torch.int32, device="cuda") % 512
    m.loss.zero_()
    m.forward_backward(tokens, (tokens + 1) % 512, 1.0 / 128)
    assert abs(m.loss.item() - torch.log(torch.tensor(512.0)).item()) < 0.5  # (weights of N(0, 0.02^2): logits near 0)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab", [100, 5000, 40001, 900001])
@pytest.mark.parametrize("tau", [0.25, 1.0])
def test_teacher_wants_what_the_lowest_value_masks(cdl, gpu_ok, dtype, vocab, tau):
    """The loss of an entry whose logit is the type's lowest value is finite: temperature p 3.4e38.  Rounded: p and three operations,
    2^-20; gradients are as they would be with any other mask."""
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    low = torch.finfo(dtype).min
    logits = (torch.randn(5, vocab, generator=gen, device="cuda") * tau).to(dtype)
    logits[:, 10:40] = low
    ids = torch.tensor([[12, -1, -1], [12, 3, 50], [1, 2, 60], [13, 13, 5], [11, 12, 13]], dtype=torch.int32, device="cuda")
    teacher = torch.randn(5, 3, generator=gen, device="cuda") * tau
    o = cdl.ops.distillation(logits, ids, teacher, cdl.ops.DistillationOpts(temperature=tau))
    loss, lse, grad = ref.distillation(logits.double(), ids, teacher, tau)
    fits = loss < torch.finfo(F32).max
    assert bool(fits[1:4].all()) and bool(torch.isfinite(o.loss[fits]).all())
    _close("loss", o.loss[fits], loss[fits], 2.0 ** -20 * loss[fits] + 2.0 ** -16)
    _close("d_logits", o.d_logits, grad, (HALF[dtype] + 2.0 ** -10 + _stat(vocab)) * grad.abs() + 2.0 ** -17 * _hit(ids, vocab) + 1e-9)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("t", [6, 40, 200])
def test_target_that_the_lowest_value_masks(cdl, gpu_ok, dtype, t):
    """The same from hidden states that pick one row of w each (the logits are w's values): x is one-hot."""
    gen = torch.Generator(device="cuda").manual_seed(t)
    low = torch.finfo(BF16).min / 2
    x = torch.zeros(t, 64, device="cuda")
    x[torch.arange(t), torch.arange(t) % 64] = 1.0
    w = torch.randn(64, 3000, generator=gen, device="cuda").to(BF16)
    w[:, 10:40] = low
    targets = torch.where(torch.arange(t, device="cuda") % 3 == 0, 12, 50).to(torch.int32)
    o = cdl.ops.linear_cross_entropy(x.to(dtype), w.to(dtype), targets)
    loss, lse, g, dx, _ = ref.linear(x, w, lambda z: ref.cross_entropy(z, targets.long()))
    # w has 8 bits: one piece, a sum of one term
    _close("lse", o.lse, lse, _stat(3000) * (2 + lse.abs()) + 2.0 ** -20 * (1 + 0 * lse))
    _close("loss", o.loss, loss, 2.0 ** -20 * loss + 2.0 ** -17)


@gpu
@pytest.mark.parametrize("t,v,k,dtype", [(70000, 32776, 0, BF16), (70000, 32776, 7, BF16), (24000, 100003, 0, F32)])
def test_gradients_beyond_32_bit_offsets(cdl, gpu_ok, t, v, k, dtype):
    """More than 2^31 logits in one chunk of rows, against the same call in chunks of the library's choice: statistics have the same bits,
    gradients are sums of the same d z over other K slices and chunks (how many depends on the rows of a chunk).  bf16: a sum of V or t terms in
    steps of 16 that cut 2^-23 each, 4375 at most, twice: 2^-10 of a value, and dx rounded to half a step on either side.  f32: parts of
    256, rounded to nearest, 400 of them, and 16 steps within: 2 * 416 * 2^-24 < 2^-14."""
    gen = torch.Generator(device="cuda").manual_seed(v)
    assert t * v > 2 ** 31
    x, w = _operands(gen, t, 64, v, dtype, "rows")
    entries = _entries(gen, t, v, k)
    fn = cdl.ops.linear_cross_entropy if k == 0 else cdl.ops.linear_distillation
    o, p = (fn(x, w, *entries, cdl.ops.LinearLossOpts(chunk_rows=c), dw=torch.empty(64, v, device="cuda")) for c in (t, 0))
    assert torch.equal(o.loss, p.loss) and torch.equal(o.lse, p.lse)
    sums = 2.0 ** -10 if dtype == BF16 else 2.0 ** -14
    assert (o.dx.double() - p.dx.double()).norm() <= (2 * HALF[dtype] + sums) * p.dx.double().norm()
    assert (o.dw - p.dw).norm() <= sums * p.dw.norm()
    rows = slice(t - 100, t)
    _check_linear(cdl, x[rows], w, [e[rows] for e in entries], cdl.ops.LinearLossOpts())
    tail = fn(x[rows], w, *[e[rows] for e in entries])
    assert (o.dx[rows].double() - tail.dx.double()).norm() <= (2 * HALF[dtype] + sums) * tail.dx.double().norm()


@gpu
@pytest.mark.parametrize("dtype,t", [(F32, 12), (F32, 300), (BF16, 50), (BF16, 3)])
def test_captured_calls_of_every_form_replay_with_new_inputs(cdl, gpu_ok, dtype, t):
    gen = torch.Generator(device="cuda").manual_seed(t)
    x, w = _operands(gen, t, 96, 3001, dtype, "tied")
    targets = _entries(gen, t, 3001, 0)[0]
    dw = torch.zeros(3001, 96, device="cuda").t()
    opts = cdl.ops.LinearLossOpts(accumulate=True)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        cdl.ops.linear_cross_entropy(x, w, targets, opts, dw=dw)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        o = cdl.ops.linear_cross_entropy(x, w, targets, opts, dw=dw)
    for _ in range(2):
        x.normal_(generator=gen)
        targets.random_(0, 3001, generator=gen)
        want = torch.zeros(3001, 96, device="cuda").t()
        p = cdl.ops.linear_cross_entropy(x, w, targets, opts, dw=want)
        dw.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o.loss, p.loss) and torch.equal(o.dx, p.dx) and torch.equal(dw, want)
