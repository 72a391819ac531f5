"""Losses of the head (linear_cross_entropy, distillation, linear_distillation) against 64-bit restatements of their
definitions (oracle/head_loss_ref.py).

Tolerances.  A statistic: the exponentials are within 2^-22 of themselves and, from the rounding of t = z log2(e) / tau,
2^-24 |t| ln 2; a sum over V of them adds at most (V / 512 + 16) 2^-24: `_stat` below, times 1 + |lse| for the parts that grow
with the values.  A probability carries that relative error, and the gradient's rounding to bf16 half a step, 2^-8 of the value.
From hidden states a logit is a sum of D products in the tensor core, whose every step of 16 products may cut 2^-23 of
the largest partial sum: (D / 16 + 8) 2^-23 |x| |w|.  The gradients' bounds follow from those of d z, which is rounded to bf16 up to
twice (2 * 2^-8): |d z error| |w|^T and |x|^T |d z error|, f32 sums of as many terms, and the result's own rounding."""
import ctypes
import threading

import pytest
import torch

from oracle import head_loss_ref as ref

gpu = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}


def _stat(vocab):
    return (vocab / 512 + 32) * 2.0 ** -24 + 2.0 ** -21


def _close(name, got, want, tol):
    got, want = got.double(), want.double()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), f"{name}: NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), f"{name}: infinities differ"
    fine = ~(nan | inf)
    tol = torch.nan_to_num(tol, nan=0.0)  # (of a row that does not count but holds NaN)
    off = (got - want).abs()[fine] - tol.expand_as(want)[fine]
    assert off.numel() == 0 or off.max() <= 0, f"{name}: {int((off > 0).sum())} of {off.numel()} beyond the bound, worst by {off.max():.3g}"


def _logits(gen, rows, vocab, dtype, pad=0, scale=3.0):
    buf = (torch.randn(rows, vocab + pad, generator=gen, device="cuda") * scale).to(dtype)
    return buf, buf[:, :vocab]


def _teacher(gen, rows, vocab, k, dtype):
    ids = torch.randint(0, vocab, (rows, k), generator=gen, device="cuda", dtype=torch.int32)
    logits = (torch.randn(rows, k, generator=gen, device="cuda") * 3).to(dtype)
    if rows > 2 and k > 1:
        ids[0, 1] = ids[0, 0]  # the same id twice
        ids[1] = -1  # a row of padding
        ids[2, : k // 2] = vocab  # ids beyond the vocabulary
        logits[1] = float("nan")
        logits[2, : k // 2] = float("inf")
    return ids, logits


def _check_distillation(cdl, logits, ids, teacher, tau, d_loss=None, grad_scale=1.0, d_logits=None):
    z = logits.double()
    vocab = z.shape[1]
    scale = torch.full((z.shape[0],), grad_scale, dtype=torch.float64, device=z.device)
    if d_loss is not None:
        scale = scale * d_loss.double()
    loss, lse, grad = ref.distillation(z, ids, teacher, tau, scale)
    o = cdl.ops.distillation(logits, ids, teacher, cdl.ops.DistillationOpts(temperature=tau, grad_scale=grad_scale, d_loss=d_loss),
                             d_logits=d_logits)
    e = _stat(vocab) * (2 + lse.abs())
    _close("lse", o.lse, lse, e)
    top = torch.where(z.abs() < 1e30, z.abs(), 0.0).amax(1) / tau  # (masks have no part in a result)
    e_loss = tau * tau * (_stat(vocab) * (4 + lse.abs()) + 2.0 ** -20 * (1 + top + _peak(teacher, ids, vocab, tau)))
    _close("loss", o.loss, loss, e_loss)
    p_err = _stat(vocab) + 2.0 ** -22 * (1 + lse.abs() + top)[:, None]
    s = (tau * scale.abs())[:, None]
    # bf16: the exponentials stand in f16 in between, half a step of which is 2^-11 of the value, or 2^-40 of the row's
    # largest: (1 + 2^-11)(1 + 2^-8) - 1 = 2^-8 + 2^-11 + 2^-19.
    half = HALF[logits.dtype] + (2.0 ** -11 + 2.0 ** -19 if logits.dtype == BF16 else 0.0)
    tol = half * grad.abs() + 2.0 ** -40 * s + 2 * p_err * (grad.abs() + 2.0 ** -10 * s) + 2.0 ** -19 * s * _hit(ids, vocab)
    _close("d_logits", o.d_logits, grad, tol + 1e-38)
    return o


def _peak(teacher, ids, vocab, tau):
    counts = (ids >= 0) & (ids < vocab) & torch.isfinite(teacher)
    t = torch.where(counts, teacher.double().abs(), 0.0)
    return (t.amax(1) if t.shape[1] else torch.zeros(t.shape[0], dtype=torch.float64, device=t.device)) / tau


def _hit(ids, vocab):
    """1 at the entries: there the difference q - p keeps the absolute errors of both."""
    hit = torch.zeros(ids.shape[0], vocab, dtype=torch.float64, device=ids.device)
    ids = ids.long()
    counts = (ids >= 0) & (ids < vocab)
    return hit.scatter_add_(1, torch.where(counts, ids, 0), counts.double()).clamp_(max=1.0)


@gpu
@pytest.mark.parametrize("rows,vocab,k,tau,dtype,pad", [
    (1, 1, 1, 1.0, F32, 0), (3, 7, 3, 2.0, BF16, 1), (1, 1000, 1, 1.0, BF16, 0), (37, 4099, 5, 0.7, BF16, 3), (5, 4099, 64, 3.0, F32, 0),
    (64, 8192, 33, 2.0, BF16, 16), (9, 32768, 64, 2.0, BF16, 0), (6, 32768, 300, 4.0, F32, 8), (4, 50001, 1024, 1.0, BF16, 0),
    (3, 150000, 20, 1.5, BF16, 0), (3, 150001, 20, 1.5, F32, 2), (17, 129, 129, 1.0, F32, 0), (300, 2048, 16, 1.0, BF16, 0),
    (700, 1003, 3, 1.0, BF16, 0), (200, 36861, 9, 1.0, BF16, 0), (2, 900001, 8, 1.0, BF16, 0), (2, 450001, 8, 2.0, F32, 0),
    (2, 400000, 1024, 2.0, F32, 4), (160, 2, 2, 1.0, BF16, 0), (160, 9, 4, 1.0, F32, 1), (3, 6000, 4, 1.0, F32, 0), (40, 10000, 4, 1.0, BF16, 0),
    (40, 14000, 40, 1.0, BF16, 0), (200, 14001, 40, 1.0, BF16, 0), (30, 26000, 3, 1.0, BF16, 0), (10, 45000, 3, 1.0, F32, 0), (2, 70000, 3, 1.0, F32, 0)])
def test_distillation(cdl, gpu_ok, rows, vocab, k, tau, dtype, pad):
    gen = torch.Generator(device="cuda").manual_seed(rows * 7 + vocab)
    _, logits = _logits(gen, rows, vocab, dtype, pad)
    ids, teacher = _teacher(gen, rows, vocab, k, dtype)
    d_loss = torch.rand(rows, generator=gen, device="cuda") + 0.5
    out = _check_distillation(cdl, logits, ids, teacher, tau, d_loss, 0.25)
    again = cdl.ops.distillation(logits, ids, teacher, cdl.ops.DistillationOpts(temperature=tau, grad_scale=0.25, d_loss=d_loss))
    assert torch.equal(out.d_logits, again.d_logits) and torch.equal(out.loss, again.loss)
    only = cdl.ops.distillation(logits, ids, teacher, cdl.ops.DistillationOpts(temperature=tau, grad=False))
    assert only.d_logits is None and torch.equal(only.loss, out.loss) and torch.equal(only.lse, out.lse)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab", [500, 4104, 70000])
def test_distillation_in_place_leaves_what_lies_beside(cdl, gpu_ok, dtype, vocab):
    gen = torch.Generator(device="cuda").manual_seed(3)
    buf, logits = _logits(gen, 11, vocab, dtype, pad=24)
    ids, teacher = _teacher(gen, 11, vocab, 8, BF16)
    want = cdl.ops.distillation(logits.clone(), ids, teacher)
    beside = buf[:, vocab:].clone()
    got = cdl.ops.distillation(logits, ids, teacher, d_logits=logits)
    assert got.d_logits is logits and torch.equal(logits, want.d_logits) and torch.equal(got.loss, want.loss)
    assert torch.equal(buf[:, vocab:], beside)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab", [1000, 33000])
def test_distillation_masked_logits_and_entries(cdl, gpu_ok, dtype, vocab):
    """Masked vocabulary (-inf, the lowest value), a teacher's -inf, rows without entries, NaN where nothing counts."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    _, logits = _logits(gen, 8, vocab, dtype)
    ids, teacher = _teacher(gen, 8, vocab, 6, F32)
    ids[3:] = torch.arange(6, dtype=torch.int32, device="cuda")
    logits[3, 6:] = float("-inf")
    logits[4, ::2] = torch.finfo(dtype).min
    logits[4, :6] = 1.0
    teacher[5, 2:] = float("-inf")  # two entries left
    teacher[6] = float("-inf")  # none left
    logits[7, 5] = float("-inf")  # the student rules out what the teacher wants: an infinite loss
    d_loss = torch.ones(8, device="cuda")
    d_loss[1] = d_loss[6] = float("nan")
    logits[1, 0] = float("nan")
    o = _check_distillation(cdl, logits, ids, teacher, 1.5, d_loss)
    assert bool((o.d_logits[1] == 0).all()) and bool((o.d_logits[6] == 0).all()) and o.loss[1] == 0 and o.loss[6] == 0
    assert torch.isinf(o.loss[7]) and bool(torch.isfinite(o.d_logits[7]).all())
    # a NaN, +inf, or nothing but -inf among the logits: NaN in that row alone
    logits[0, 1], logits[2, 3] = float("inf"), float("nan")
    logits[3] = float("-inf")
    o = cdl.ops.distillation(logits, ids, teacher, cdl.ops.DistillationOpts(temperature=1.5))
    for row in (0, 2, 3):
        assert torch.isnan(o.loss[row]) and bool(torch.isnan(o.d_logits[row]).any())
    assert bool(torch.isfinite(o.d_logits[4:]).all()) and bool(torch.isfinite(o.loss[4:7]).all())


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab", [100, 5000, 40001, 900001])
def test_distillation_rows_masked_with_the_lowest_value(cdl, gpu_ok, dtype, vocab):
    """Masks of the type's lowest (or largest) value, which times log2(e) is no f32: a row of nothing else is a uniform one, and a
    teacher of nothing else, too."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    _, logits = _logits(gen, 6, vocab, dtype)
    logits[0] = low
    logits[1, 50:] = low
    logits[2] = high
    logits[3], logits[3, 7] = low, high
    ids = torch.arange(8, dtype=torch.int32, device="cuda").expand(6, 8).contiguous()
    teacher = (torch.randn(6, 8, generator=gen, device="cuda") * 2).to(dtype)
    teacher[4], teacher[5, 3:] = low, low
    teacher[3], teacher[3, 7] = low, high  # (the student agrees: no loss)
    o = cdl.ops.distillation(logits, ids, teacher, cdl.ops.DistillationOpts(temperature=0.8))
    loss, lse, grad = ref.distillation(logits.double(), ids, teacher, 0.8)
    assert bool((torch.isfinite(o.loss) | (o.loss.double() == loss)).all()) and not bool(torch.isnan(o.d_logits).any())
    # the statistics as above; logits that large are rounded to 2^-24 of themselves in lse, and their differences are 0 or beyond 2^100
    e = _stat(vocab) * (8 + torch.log(torch.tensor(float(vocab))))
    rows = [0, 1, 2, 4, 5]
    _close("loss", o.loss[rows], loss[rows], torch.full_like(loss[rows], float(e) + 2.0 ** -18))
    assert abs(o.loss[3].item()) <= 1e-5
    finite = torch.isfinite(lse.float())
    _close("lse", o.lse[finite], lse[finite], e.cuda() + 2.0 ** -22 * lse[finite].abs())
    half = HALF[dtype] + 2.0 ** -10
    _close("d_logits", o.d_logits, grad, (half + 2 * float(e)) * grad.abs() + 2.0 ** -17 * _hit(ids, vocab) + 1e-9)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab,k", [(300, 5), (1000, 200), (9000, 64), (33000, 100), (50001, 300)])
def test_distillation_row_by_row(cdl, gpu_ok, dtype, vocab, k):
    """A row's bits do not depend on how many rows there are (and so on how many CTAs share one)."""
    gen = torch.Generator(device="cuda").manual_seed(8)
    _, logits = _logits(gen, 600, vocab, dtype, pad=(-vocab) % 8)
    ids, teacher = _teacher(gen, 600, vocab, k, dtype)
    o = cdl.ops.distillation(logits, ids, teacher, cdl.ops.DistillationOpts(temperature=1.3))
    for rows in (slice(0, 1), slice(2, 5), slice(100, 140)):
        p = cdl.ops.distillation(logits[rows], ids[rows], teacher[rows], cdl.ops.DistillationOpts(temperature=1.3))
        assert torch.equal(p.loss, o.loss[rows]) and torch.equal(p.lse, o.lse[rows]) and torch.equal(p.d_logits, o.d_logits[rows])


@gpu
def test_distillation_no_entries_no_rows(cdl, gpu_ok):
    logits = torch.randn(3, 100, device="cuda")
    none = torch.empty(3, 0, dtype=torch.int32, device="cuda")
    o = cdl.ops.distillation(logits, none, torch.empty(3, 0, device="cuda"))
    assert bool((o.loss == 0).all()) and bool((o.d_logits == 0).all())
    _close("lse", o.lse, torch.logsumexp(logits.double(), 1), torch.full((), 1e-5, device="cuda"))
    o = cdl.ops.distillation(logits[:0], none[:0], torch.empty(0, 0, device="cuda"))
    assert o.loss.shape == (0,) and o.d_logits.shape == (0, 100)


@gpu
def test_distillation_rows_beyond_32_bit_offsets(cdl, gpu_ok):
    rows, vocab = 66000, 32768 + 8
    assert rows * vocab > 2 ** 31
    logits = torch.empty(rows, vocab, dtype=BF16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(5)
    tail = slice(rows - 3, rows)
    logits.normal_(generator=gen)
    ids, teacher = _teacher(gen, rows, vocab, 4, BF16)
    want = cdl.ops.distillation(logits[tail].clone(), ids[tail], teacher[tail])
    o = cdl.ops.distillation(logits, ids, teacher, d_logits=logits)
    assert torch.equal(o.loss[tail], want.loss) and torch.equal(logits[tail], want.d_logits)


# ------------------------------------------------------------------------------------------ from the hidden states
def _operands(gen, t, d, v, dtype, layout):
    x = torch.randn(t, d, generator=gen, device="cuda")
    w = torch.randn(d, v, generator=gen, device="cuda") * (0.5 / d ** 0.5)
    if layout == "tied":
        w = w.t().contiguous().to(dtype).t()
    elif layout == "strided":  # neither dimension contiguous; x a column slice off the 16-byte grid
        w = torch.stack([w, w], 2).to(dtype)[:, :, 0]
        x = torch.cat([x[:, :1], x], 1)[:, 1:]
    elif layout == "columns":
        x = x.t().contiguous().t()
    x = x.to(dtype) if layout != "strided" else torch.cat([x[:, :3], x], 1).to(dtype)[:, 3:]
    return x, w.to(dtype) if layout != "strided" else w


def _check_linear(cdl, x, w, entries, opts, dw=None, before=None, **kw):
    tau, t = opts.temperature, x.shape[0]
    (d, v), dtype = w.shape, x.dtype
    scale = torch.full((t,), opts.grad_scale, dtype=torch.float64, device="cuda")
    if opts.d_loss is not None:
        scale = scale * opts.d_loss.double()

    def loss_of(z):
        return ref.cross_entropy(z, entries[0], scale) if len(entries) == 1 else ref.distillation(z, *entries, tau, scale)

    x64, w64 = x.double(), w.double()
    loss, lse, g, dx, dw_ref = ref.linear(x, w, loss_of)
    fn = cdl.ops.linear_cross_entropy if len(entries) == 1 else cdl.ops.linear_distillation
    o = fn(x, w, *entries, opts, dw=dw, **kw)
    keep = (g != 0).any(1)
    ax = torch.where(torch.isfinite(x64), x64.abs(), 0.0)
    dz = (d / 16 + 8) * 2.0 ** -23 * (ax @ w64.abs()).amax(1)  # of a logit
    if dtype == F32:
        dz = dz * 0.25  # chains of f32 additions
    e = _stat(v) * (3 + lse.abs()) + dz / tau
    _close("lse", o.lse, lse, e)
    extra = 2.0 ** -20 * (1 + lse.abs() + (_peak(entries[1], entries[0], v, tau) if len(entries) > 1 else 0))
    _close("loss", o.loss, loss, tau * tau * (2 * e + extra))
    twice = 2 * HALF[dtype]
    ids = entries[0] if len(entries) > 1 else entries[0][:, None]
    s = torch.where(keep, (tau * scale).abs(), 0.0)[:, None]
    p_err = (_stat(v) + 2.0 ** -20 * (1 + lse.abs()) + 2 * dz / tau)[:, None]
    p_err = torch.where(keep[:, None], p_err, 0.0)
    g_err = twice * g.abs() + 2 * p_err * (g.abs() + s * _hit(ids, v)) + 2.0 ** -30 * s
    g_abs, ax = torch.where(keep[:, None], g.abs(), 0.0), torch.where(keep[:, None], ax, 0.0)
    sums = 2.0 ** -23 * 40
    if opts.grad and o.dx is not None:
        assert o.dx.dtype == dtype
        _close("dx", o.dx, dx, (g_err + sums * g_abs) @ w64.abs().t() + HALF[dtype] * dx.abs() + 1e-30)
    if opts.grad and o.dw is not None:
        if before is not None:
            dw_ref = dw_ref + before.double()
        _close("dw", o.dw, dw_ref, ax.t() @ (g_err + sums * g_abs) + (HALF[o.dw.dtype] + 2.0 ** -22) * dw_ref.abs() + 1e-30)
        if before is None and t > 0 and bool(keep.any()):
            # roundings of at most 2^-8 each: d z twice, the result once
            off = (o.dw.double() - dw_ref).norm() / dw_ref.norm()
            assert off <= (3 * 2.0 ** -8 if dtype == BF16 else 2e-5), off
    return o


def _entries(gen, t, v, k):
    if k == 0:
        targets = torch.randint(0, v, (t,), generator=gen, device="cuda", dtype=torch.int32)
        if t > 2:
            targets[0], targets[1] = -1, v
        return (targets,)
    return _teacher(gen, t, v, k, BF16)


SHAPES = [(1, 64, 1000, 0, BF16, "rows"), (1, 8, 1, 0, BF16, "rows"), (7, 65, 129, 0, BF16, "rows"), (300, 128, 1001, 0, BF16, "tied"),
          (130, 96, 520, 0, BF16, "strided"), (129, 256, 4096, 0, BF16, "rows"), (513, 128, 2304, 0, BF16, "rows"),
          (65, 515, 770, 0, F32, "rows"), (40, 64, 301, 0, F32, "tied"), (33, 48, 100, 0, F32, "strided"), (70, 64, 300, 0, BF16, "columns"),
          (1, 64, 1000, 5, BF16, "rows"), (257, 256, 4097, 64, BF16, "rows"), (300, 72, 1001, 7, BF16, "tied"), (12, 128, 640, 300, BF16, "rows"),
          (50, 65, 300, 16, F32, "rows"), (200, 64, 8200, 1, BF16, "tied"), (600, 64, 128, 128, BF16, "rows"), (5, 64, 2000, 1024, BF16, "rows"),
          (100, 512, 3000, 0, BF16, "rows"), (128, 320, 40000, 0, BF16, "rows"), (128, 320, 40001, 9, BF16, "tied"), (700, 256, 30000, 33, BF16, "rows"),
          (3, 24, 270001, 6, F32, "rows"), (2, 16, 600001, 3, BF16, "rows"), (130, 16, 140000, 20, BF16, "tied")]


@gpu
@pytest.mark.parametrize("t,d,v,k,dtype,layout", SHAPES)
def test_linear_losses(cdl, gpu_ok, t, d, v, k, dtype, layout):
    gen = torch.Generator(device="cuda").manual_seed(t + v)
    x, w = _operands(gen, t, d, v, dtype, layout)
    entries = _entries(gen, t, v, k)
    d_loss = torch.rand(t, generator=gen, device="cuda") + 0.5
    opts = cdl.ops.LinearLossOpts(temperature=1.0 if k == 0 else 1.7, grad_scale=0.5, d_loss=d_loss)
    o = _check_linear(cdl, x, w, entries, opts)
    fn = cdl.ops.linear_cross_entropy if k == 0 else cdl.ops.linear_distillation
    again = fn(x, w, *entries, opts)
    assert all(torch.equal(a, b) for a, b in ((o.loss, again.loss), (o.lse, again.lse), (o.dx, again.dx), (o.dw, again.dw)))
    opts.grad = False
    only = fn(x, w, *entries, opts)
    assert only.dx is None and only.dw is None and torch.equal(only.loss, o.loss) and torch.equal(only.lse, o.lse)


@gpu
@pytest.mark.parametrize("k", [0, 9])
@pytest.mark.parametrize("chunk", [1, 100, 256])
def test_linear_losses_in_chunks_of_rows(cdl, gpu_ok, k, chunk):
    """Rows a chunk at a time: the statistics do not change at all, the weight gradient is a sum over chunks in f32."""
    gen = torch.Generator(device="cuda").manual_seed(chunk)
    t = 5 if chunk == 1 else 601
    for layout in ("rows", "tied", "columns"):
        x, w = _operands(gen, t, 64, 777, BF16, layout)
        entries = _entries(gen, t, 777, k)
        opts = cdl.ops.LinearLossOpts(chunk_rows=chunk)
        o = _check_linear(cdl, x, w, entries, opts)
        fn = cdl.ops.linear_cross_entropy if k == 0 else cdl.ops.linear_distillation
        whole = fn(x, w, *entries)
        assert torch.allclose(whole.loss, o.loss, rtol=1e-5, atol=1e-5)


@gpu
@pytest.mark.parametrize("layout", ["rows", "tied", "columns"])
@pytest.mark.parametrize("t,d,v,chunk", [(601, 64, 777, 600), (601, 130, 260, 100), (5, 64, 300, 1), (1200, 72, 520, 0), (260, 40, 12000, 0), (90, 700, 9000, 0)])
def test_linear_losses_of_f32_operands(cdl, gpu_ok, layout, t, d, v, chunk):
    """K slices of the products, rows in chunks (one row left for the last), gradients added to what is there."""
    gen = torch.Generator(device="cuda").manual_seed(t + v)
    x, w = _operands(gen, t, d, v, F32, layout)
    for k in (0, 11):
        entries = _entries(gen, t, v, k)
        o = _check_linear(cdl, x, w, entries, cdl.ops.LinearLossOpts(chunk_rows=chunk))
        before = torch.randn(d, v, generator=gen, device="cuda")
        dw = before.clone()
        fn = cdl.ops.linear_cross_entropy if k == 0 else cdl.ops.linear_distillation
        added = fn(x, w, *entries, cdl.ops.LinearLossOpts(chunk_rows=chunk, accumulate=True), dw=dw)
        # (f32 sums of other terms in another order: 2^-22 of the parts)
        assert bool(((added.dw - before - o.dw).abs() <= 2.0 ** -20 * (before.abs() + o.dw.abs() + 1)).all())


@gpu
@pytest.mark.parametrize("t", [40, 159])
def test_f32_gradient_whose_largest_term_comes_first(cdl, gpu_ok, t):
    """d x is the target's column and what tens of thousands of small terms add to it. A tensor-core accumulator drops up to a bit of
    the last place (2^-24) in each of its steps of 16; one takes 256 of K, so 16 steps lie behind the target's. The six products of pieces
    leave out three below 2^-24 each; the sums of 171 parts are rounded to nearest, 2^-25 times their square root as they are independent: 7
    of 2^-24. In all 26 2^-24 of the 2-norm."""
    gen = torch.Generator(device="cuda").manual_seed(12)
    x = torch.randn(t, 576, generator=gen, device="cuda")
    w = torch.randn(576, 43584, generator=gen, device="cuda") * 0.02
    targets = torch.zeros(t, dtype=torch.int32, device="cuda")
    o = cdl.ops.linear_cross_entropy(x, w, targets)
    _, _, _, dx, _ = ref.linear(x, w, lambda z: ref.cross_entropy(z, targets.long()))
    assert ((o.dx - dx).norm() / dx.norm()).item() <= 26 * 2.0 ** -24


@gpu
@pytest.mark.parametrize("t", [1, 4, 5, 8, 9, 16, 17])
@pytest.mark.parametrize("d,v,layout", [(1100, 9003, "rows"), (1101, 9002, "tied"), (515, 130, "rows"), (3, 700, "tied"), (1030, 2049, "strided")])
def test_f32_losses_of_few_tokens(cdl, gpu_ok, t, d, v, layout):
    """Rows anywhere, K slices and none, gradients that are written and added to, d x in place of x."""
    gen = torch.Generator(device="cuda").manual_seed(t + v)
    x, w = _operands(gen, t, d, v, F32, layout)
    rows, cols = (v, d) if layout == "tied" else (d, v)
    buffer = torch.randn(rows, cols + 3, generator=gen, device="cuda") * 0.01
    kept = buffer.clone()
    dw = buffer[:, 2:2 + cols].t() if layout == "tied" else buffer[:, 2:2 + cols]
    before = dw.clone()
    entries = _entries(gen, t, v, 0)
    _check_linear(cdl, x, w, entries, cdl.ops.LinearLossOpts(accumulate=True), dw=dw, before=before)
    assert torch.equal(buffer[:, :2], kept[:, :2]) and torch.equal(buffer[:, -1], kept[:, -1])
    o = _check_linear(cdl, x, w, _entries(gen, t, v, min(v, 40)), cdl.ops.LinearLossOpts(temperature=1.4))
    y = x.clone(memory_format=torch.contiguous_format)
    p = cdl.ops.linear_cross_entropy(y, w, *entries)
    q = cdl.ops.linear_cross_entropy(y, w, *entries, dx=y)
    assert q.dx.data_ptr() == y.data_ptr() and torch.equal(p.dx, q.dx) and torch.equal(p.dw, q.dw) and o.dw is not None


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("chunk", [0, 128])
def test_weight_gradient_is_added_to(cdl, gpu_ok, dtype, tied, chunk):
    gen = torch.Generator(device="cuda").manual_seed(8)
    x, w = _operands(gen, 300, 96, 1000, BF16, "tied" if tied else "rows")
    entries = _entries(gen, 300, 1000, 0)
    before = torch.randn(1000, 96, generator=gen, device="cuda").to(dtype).t() if tied else \
        torch.randn(96, 1000, generator=gen, device="cuda").to(dtype)
    dw = before.clone() if not tied else before.t().clone().t()
    o = _check_linear(cdl, x, w, entries, cdl.ops.LinearLossOpts(accumulate=True, chunk_rows=chunk), dw=dw, before=before)
    assert o.dw is dw
    # written, not added to: what it held does not matter
    dw.fill_(float("nan"))
    _check_linear(cdl, x, w, entries, cdl.ops.LinearLossOpts(chunk_rows=chunk), dw=dw)


@gpu
def test_gradients_on_their_own_and_odd_outputs(cdl, gpu_ok):
    """dx without dw, dw without dx, dx in place of x, a gradient with rows beside it that stay as they were."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    x, w = _operands(gen, 200, 64, 501, BF16, "rows")
    entries = _entries(gen, 200, 501, 0)
    both = cdl.ops.linear_cross_entropy(x, w, *entries)
    a = cdl.ops.linear_cross_entropy(x, w, *entries, cdl.ops.LinearLossOpts(grad_w=False))
    b = cdl.ops.linear_cross_entropy(x, w, *entries, cdl.ops.LinearLossOpts(grad_x=False))
    assert a.dw is None and torch.equal(a.dx, both.dx) and b.dx is None and torch.equal(b.dw, both.dw)
    buf = torch.full((220, 70), 7.0, dtype=BF16, device="cuda")
    wide = torch.full((70, 640), 7.0, device="cuda")
    o = cdl.ops.linear_cross_entropy(x, w, *entries, cdl.ops.LinearLossOpts(chunk_rows=64), dx=buf[3:203, 5:69], dw=wide[2:66, 3:504])
    assert torch.equal(o.dx, both.dx)
    assert bool((buf[:3] == 7).all()) and bool((buf[203:] == 7).all()) and bool((buf[:, :5] == 7).all()) and bool((buf[:, 69:] == 7).all())
    assert bool((wide[:2] == 7).all()) and bool((wide[66:] == 7).all()) and bool((wide[:, :3] == 7).all()) and bool((wide[:, 504:] == 7).all())
    assert (o.dw - both.dw.float()).norm() / both.dw.float().norm() <= 2.0 ** -8
    for chunk in (0, 64):
        y = x.clone()
        o = cdl.ops.linear_cross_entropy(y, w, *entries, cdl.ops.LinearLossOpts(chunk_rows=chunk), dx=y)
        assert torch.equal(y, both.dx) and (o.dw.float() - both.dw.float()).norm() / both.dw.float().norm() <= 2.0 ** -7


@gpu
@pytest.mark.parametrize("t,d,v,tied", [(3, 1100, 9001, False), (90, 1101, 9000, True), (600, 390, 20003, False), (257, 1030, 9472, False),
                                        (1, 9473, 1025, False)])
@pytest.mark.parametrize("wider,off", [(0, 0), (5, 2), (8, 3)])
def test_weight_gradient_of_rows_off_the_grid(cdl, gpu_ok, t, d, v, tied, wider, off):
    """Outputs of many tiles whose rows begin anywhere; what lies between and around the rows stays as it was."""
    gen = torch.Generator(device="cuda").manual_seed(t)
    x, w = _operands(gen, t, d, v, BF16, "tied" if tied else "rows")
    rows, cols = (v, d) if tied else (d, v)
    buffer = torch.full((rows + 2, cols + wider), 7.0, dtype=BF16, device="cuda")
    view = buffer[1:-1, off:off + cols]
    dw = view.t() if tied else view
    _check_linear(cdl, x, w, _entries(gen, t, v, 0), cdl.ops.LinearLossOpts(), dw=dw)
    view.fill_(7.0)
    assert bool((buffer == 7.0).all())


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("k", [0, 4])
def test_rows_that_do_not_count_add_nothing(cdl, gpu_ok, dtype, k):
    gen = torch.Generator(device="cuda").manual_seed(10)
    x, w = _operands(gen, 150, 64, 300, dtype, "rows")
    entries = list(_entries(gen, 150, 300, k))
    off = torch.arange(0, 150, 3, device="cuda")
    entries[0][off] = -5
    clean = x.clone()
    clean[off] = 0.0
    want = (cdl.ops.linear_cross_entropy if k == 0 else cdl.ops.linear_distillation)(clean, w, *entries)
    # bf16: the same bits.  f32: tiles of the products that hold a value without bf16 pieces (infinities, NaN) are summed in
    # another order, in which a logit differs by 2 * 64 * 2^-24 |x| |w| at most (each is that close to a chain of 64 f32
    # FMAs), a loss by twice that, a softmax by twice that of itself, and the gradients by its products; then f32 rounding.
    dz = 2 * 64 * 2.0 ** -24 * float((clean.double().abs() @ w.double().abs()).max())
    soft = torch.softmax(clean.double() @ w.double(), 1)
    soft[off] = 0.0
    tol_dx, tol_dw = 2 * dz * soft @ w.double().abs().t(), 2 * dz * clean.double().abs().t() @ soft

    def same(name, a, b, tol):
        if dtype == BF16:
            assert torch.equal(a, b), name
        else:
            _close(name, a, b, tol + 150 * 2.0 ** -23 * (1 + b.double().abs()))

    for poison in (float("nan"), float("inf"), torch.finfo(dtype).max):
        dirty = x.clone()
        dirty[off] = poison
        d_loss = torch.ones(150, device="cuda")
        d_loss[off] = float("nan")
        fn = cdl.ops.linear_cross_entropy if k == 0 else cdl.ops.linear_distillation
        o = fn(dirty, w, *entries, cdl.ops.LinearLossOpts(d_loss=d_loss))
        same("dw", o.dw, want.dw, tol_dw)
        same("dx", o.dx, want.dx, tol_dx)
        same("loss", o.loss, want.loss, torch.full_like(want.loss, 2 * dz).double())
        assert bool((o.loss[off] == 0).all()) and bool((o.dx[off] == 0).all())
    entries[0].fill_(-1)  # no row counts
    o = fn(dirty, w, *entries)
    assert bool((o.loss == 0).all()) and bool((o.dx == 0).all()) and bool((o.dw == 0).all())


@gpu
def test_no_tokens(cdl, gpu_ok):
    empty = torch.empty(0, 0, dtype=BF16, device="cuda")
    assert cdl.ops.linear_cross_entropy(empty, empty, torch.empty(0, dtype=torch.int32, device="cuda")).loss.shape == (0,)
    x, w = torch.empty(0, 64, dtype=BF16, device="cuda"), torch.randn(64, 100, device="cuda").to(BF16)
    o = cdl.ops.linear_cross_entropy(x, w, torch.empty(0, dtype=torch.int32, device="cuda"))
    assert o.loss.shape == (0,) and o.dx.shape == (0, 64) and bool((o.dw == 0).all())
    dw = torch.ones(64, 100, device="cuda")
    cdl.ops.linear_cross_entropy(x, w, torch.empty(0, dtype=torch.int32, device="cuda"), cdl.ops.LinearLossOpts(accumulate=True), dw=dw)
    assert bool((dw == 1).all())


@gpu
@pytest.mark.parametrize("k", [0, 5])
def test_gradients_against_differences(cdl, gpu_ok, k):
    """(L(p + h v) - L(p - h v)) / 2h along random directions v.  L is a sum of 40 f32 losses, each off by at most 1e-5
    (the bounds above at these sizes): 40 * 2e-5 / 2h at worst, and h^2 / 6 times a third derivative below 6 |v z|^3 a row
    (the third cumulant of a softmax, |v z| < 3 here): h = 1e-2 leaves 0.04 + 0.02 at values of about 10."""
    gen = torch.Generator(device="cuda").manual_seed(12)
    t, d, v, tau, h = 40, 24, 50, 1.0 if k == 0 else 2.0, 1e-2
    x, w = torch.randn(t, d, generator=gen, device="cuda"), torch.randn(d, v, generator=gen, device="cuda") * 0.3
    entries = _entries(gen, t, v, k)
    d_loss = torch.rand(t, generator=gen, device="cuda")
    fn = cdl.ops.linear_cross_entropy if k == 0 else cdl.ops.linear_distillation
    opts = cdl.ops.LinearLossOpts(temperature=tau, d_loss=d_loss)
    o = fn(x, w, *entries, opts)
    total = lambda a, b: (fn(a, b, *entries, cdl.ops.LinearLossOpts(temperature=tau, grad=False)).loss.double() * d_loss.double()).sum()  # noqa: E731
    for _ in range(4):
        vx = torch.randn(t, d, generator=gen, device="cuda") / d ** 0.5
        vw = torch.randn(d, v, generator=gen, device="cuda") / d ** 0.5
        along = (o.dx.double() * vx).sum() + (o.dw.double() * vw).sum()
        slope = (total(x + h * vx, w + h * vw) - total(x - h * vx, w - h * vw)) / (2 * h)
        assert abs(along - slope) <= 0.06 * (1 + tau * tau), (along, slope)


@gpu
def test_broadcast_upstream_gradient(cdl, gpu_ok):
    gen = torch.Generator(device="cuda").manual_seed(13)
    x, w = _operands(gen, 20, 64, 130, BF16, "rows")
    entries = _entries(gen, 20, 130, 0)
    one = torch.tensor([0.25], device="cuda")
    a = cdl.ops.linear_cross_entropy(x, w, *entries, cdl.ops.LinearLossOpts(d_loss=one.expand(20)))
    b = cdl.ops.linear_cross_entropy(x, w, *entries, cdl.ops.LinearLossOpts(grad_scale=0.25))
    assert torch.equal(a.dx, b.dx) and torch.equal(a.dw, b.dw)
    every_other = torch.stack([one.expand(20), torch.full((20,), float("nan"), device="cuda")], 1)[:, 0]
    c = cdl.ops.linear_cross_entropy(x, w, *entries, cdl.ops.LinearLossOpts(d_loss=every_other))
    assert torch.equal(a.dx, c.dx)


@gpu
def test_captured_calls_replay(cdl, gpu_ok):
    """Two graphs captured on one stream, with new inputs before each replay, replayed beside one another on two streams."""
    gen = torch.Generator(device="cuda").manual_seed(14)
    graphs, states = [], []
    side = torch.cuda.Stream()
    for i in range(2):
        x, w = _operands(gen, 1100, 128, 20000 + 8 * i, BF16, "rows")
        s = {"x": x, "w": w, "targets": _entries(gen, 1100, w.shape[1], 0)[0]}
        s["ids"], s["teacher"] = _teacher(gen, 1100, w.shape[1], 6, BF16)
        s["logits"] = _logits(gen, 64, 5000, BF16)[1]

        def call(s=s):
            a = cdl.ops.linear_cross_entropy(s["x"], s["w"], s["targets"], cdl.ops.LinearLossOpts(chunk_rows=512))
            b = cdl.ops.linear_distillation(s["x"], s["w"], s["ids"], s["teacher"])
            c = cdl.ops.distillation(s["logits"], s["ids"][:64], s["teacher"][:64])
            return (a.loss, a.lse, a.dx, a.dw, b.loss, b.dx, b.dw, c.loss, c.d_logits)

        s["call"] = call
        with torch.cuda.stream(side):
            call()
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            s["out"] = call()
        graphs.append(g)
        states.append(s)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for s in states:
            s["x"].normal_(generator=gen)
            s["targets"].random_(0, 20000, generator=gen)
        torch.cuda.synchronize()
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for s in states:
            for got, want in zip(s["out"], s["call"]()):
                assert torch.equal(got, want)


@gpu
def test_calls_from_threads_on_their_own_streams(cdl, gpu_ok):
    gen = torch.Generator(device="cuda").manual_seed(15)
    inputs = []
    for i in range(3):
        x, w = _operands(gen, 700, 128, 9000, BF16, "rows" if i else "tied")
        inputs.append((x, w, _entries(gen, 700, 9000, 0)[0], *_entries(gen, 700, 9000, 8)))

    def compute(x, w, targets, ids, teacher):
        a = cdl.ops.linear_cross_entropy(x, w, targets, cdl.ops.LinearLossOpts(chunk_rows=256))
        b = cdl.ops.linear_distillation(x, w, ids, teacher)
        return a.loss, a.dx, a.dw, b.loss, b.dx, b.dw

    want = [compute(*i) for i in inputs]
    torch.cuda.synchronize()
    got, errors = [None] * 3, []

    def worker(i):
        try:
            torch.cuda.set_device(0)
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                for _ in range(10):
                    got[i] = compute(*inputs[i])
                st.synchronize()
        except Exception as e:  # reported below
            errors.append(repr(e))

    threads = [threading.Thread(target=worker, args=(i,)) for i in range(3)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


@gpu
def test_losses_together_on_one_head(cdl, gpu_ok):
    """A step that trains a tied head on targets and on a teacher at once: the norm's output through both losses, dw the sum of
    both in f32, and each of them against the same loss of stored logits."""
    gen = torch.Generator(device="cuda").manual_seed(16)
    t, d, v, tau = 300, 256, 2000, 2.0
    x = cdl.ops.norm_fwd(torch.randn(t, d, generator=gen, device="cuda").to(BF16)).y
    table = (torch.randn(v, d, generator=gen, device="cuda") * 0.1).to(BF16)
    w, targets = table.t(), _entries(gen, t, v, 0)[0]
    ids, teacher = _teacher(gen, t, v, 12, BF16)
    d_table = torch.zeros(v, d, device="cuda")
    hard = cdl.ops.linear_cross_entropy(x, w, targets, cdl.ops.LinearLossOpts(grad_scale=0.7, accumulate=True), dw=d_table.t())
    soft = cdl.ops.linear_distillation(x, w, ids, teacher, cdl.ops.LinearLossOpts(temperature=tau, grad_scale=0.3, accumulate=True),
                                       dw=d_table.t())
    one = torch.ones(t, dtype=torch.float64, device="cuda")
    _, _, _, dx0, dw0 = ref.linear(x, w, lambda z: ref.cross_entropy(z, targets, 0.7 * one))
    _, _, _, dx1, dw1 = ref.linear(x, w, lambda z: ref.distillation(z, ids, teacher, tau, 0.3 * one))
    # d z rounded twice (2^-8 each), the result once: at most 3 * 2^-8 of the 2-norm
    for got, want in ((hard.dx, dx0), (soft.dx, dx1), (d_table.t(), dw0 + dw1)):
        assert (got.double() - want).norm() <= 3 * 2.0 ** -8 * want.norm()
    # logits stored in bf16 (|z| < 8 here: 2^-6 off at most): the losses move by twice that over tau, times tau^2
    logits = cdl.ops.matmul(x, w)
    assert float(logits.float().abs().max()) < 8
    stored = cdl.ops.distillation(logits, ids, teacher, cdl.ops.DistillationOpts(temperature=tau, grad_scale=0.3))
    assert bool(((stored.loss - soft.loss).abs() <= 2 * tau * 2.0 ** -6 + 1e-4).all())
    assert (cdl.ops.matmul(stored.d_logits, table).double() - dx1).norm() <= 2.0 ** -4 * dx1.norm()


@gpu
def test_language_model_without_stored_logits(cdl, gpu_ok):
    """Sky1LM with keep_logits=False against the same model with them.  Stored logits are rounded to bf16: |z| < 4 here (N(0, 0.32^2)),
    so they are 2^-7 off at most, losses twice that, softmax and gradients 2 * 2^-7 of themselves; bf16 roundings of both backward
    passes add at most as much again."""
    sky1 = cdl.sky1
    blk = sky1.Sky1Config(batch=2, seqlen=256, hidden=256, heads=2, kv_heads=2, head_dim=128, ffn=512)
    models = [sky1.Sky1LM(sky1.Sky1LMConfig(block=blk, layers=2, vocab=2048, keep_logits=k), seed=4) for k in (True, False)]
    assert models[1].logits is None
    gen = torch.Generator().manual_seed(7)
    data = torch.randint(0, 2048, (2, 2, 257), generator=gen, dtype=torch.int32)
    tokens, targets = (data[:, :, i:256 + i].reshape(2, -1).cuda() for i in (0, 1))
    targets[0, ::7] = -1
    for m in models:
        m.loss.zero_()
        for i in range(2):
            m.forward_backward(tokens[i], targets[i], 1.0 / tokens.numel())
    a, b = models
    assert abs(a.loss.item() - b.loss.item()) <= 2.0 ** -6
    for name, _, _ in a.layout:
        p, q = a.view("grads", name).double(), b.view("grads", name).double()
        assert (p - q).norm() <= 4 * 2.0 ** -7 * p.norm(), name
    for m in models:
        m.optimizer_step()
    assert cdl._lib.device_status() == 0


# ------------------------------------------------------------------------------------------ refusals (no GPU)
def _t(L, shape, strides=None, dtype=0, ptr=4096):
    t = L.CdlTensor(ptr=ptr, dtype=dtype, rank=len(shape))
    packed = 1
    for i in reversed(range(len(shape))):
        t.shape[i] = shape[i]
        t.stride[i] = strides[i] if strides else packed
        packed *= shape[i]
    return t


def _linear_status(L, temperature=1.0, distil=False, scratch=(0, 0), **other):
    a = {"x": _t(L, (8, 16)), "w": _t(L, (16, 40)), "targets": _t(L, (8,), dtype=L.CDL_I32), "d_loss": None,
         "loss": _t(L, (8,), dtype=L.CDL_F32), "lse": None, "dx": _t(L, (8, 16)), "dw": _t(L, (16, 40)),
         "ids": _t(L, (8, 4), dtype=L.CDL_I32), "teacher": _t(L, (8, 4)), "chunk": 0}
    a.update(other)
    desc = L.CdlHeadLossDesc(temperature, 1.0, 0, a["chunk"])
    r = lambda t: None if t is None else ctypes.byref(t)  # noqa: E731
    rest = [r(a[n]) for n in ("d_loss", "loss", "lse", "dx", "dw")] + [scratch[0] or None, scratch[1], None]
    if distil:
        return L.lib.cdl_b200_linear_distillation(ctypes.byref(desc), r(a["x"]), r(a["w"]), r(a["ids"]), r(a["teacher"]), *rest)
    return L.lib.cdl_b200_linear_cross_entropy(ctypes.byref(desc), r(a["x"]), r(a["w"]), r(a["targets"]), *rest)


def test_linear_refusals(cdl):
    L = cdl._lib
    i32, f32 = L.CDL_I32, L.CDL_F32
    for other, said in [
            ({"x": None}, "x must be"), ({"x": _t(L, (8, 16), dtype=f32)}, "same type"), ({"x": _t(L, (8, 16, 1))}, "x must be"),
            ({"w": _t(L, (17, 40))}, "hidden sizes differ"), ({"w": _t(L, (16, 0)), "dw": _t(L, (16, 0))}, "vocab is zero"),
            ({"x": _t(L, (8, 0)), "w": _t(L, (0, 40)), "dx": None, "dw": None}, "hidden is zero"),
            ({"targets": None}, "targets are required"), ({"targets": _t(L, (7,), dtype=i32)}, "targets must be"),
            ({"targets": _t(L, (8,), dtype=f32)}, "targets must be"), ({"targets": _t(L, (8,), (2,), dtype=i32)}, "targets must be"),
            ({"loss": None}, "loss is required"), ({"loss": _t(L, (8,))}, "loss must be"), ({"lse": _t(L, (9,), dtype=f32)}, "lse must be"),
            ({"d_loss": _t(L, (8,))}, "d_loss must be"), ({"dx": _t(L, (8, 16), dtype=f32)}, "dx must have"),
            ({"dx": _t(L, (8, 16), (8, 1))}, "dx must have"), ({"dx": _t(L, (8, 16), (1, 8))}, "dx must have"),
            ({"dw": _t(L, (16, 40), dtype=i32)}, "dw must be"), ({"dw": _t(L, (40, 16))}, "dw must be"),
            ({"dw": _t(L, (16, 40), (0, 1))}, "dw overlap"), ({"dw": _t(L, (16, 40), (20, 1))}, "dw overlap"),
            ({"dw": _t(L, (16, 40), (1, 8))}, "dw overlap"), ({"temperature": 2.0}, "temperature must be 1"),
            ({"temperature": 0.0}, "temperature must be positive"), ({"temperature": float("nan")}, "temperature must be positive"),
            ({"chunk": -1}, "chunk_rows"), ({}, "scratch must hold"), ({"scratch": (4096, 256)}, "scratch must hold"),
            ({"scratch": (4096 + 8, 1 << 30)}, "scratch must hold")]:
        assert _linear_status(L, **other) < 0 and said in L.last_error(), (other, L.last_error())
    for other, said in [
            ({"ids": None}, "required"), ({"teacher": None}, "required"), ({"ids": _t(L, (8, 5), dtype=i32)}, "teacher_logits must be"),
            ({"ids": _t(L, (8, 4))}, "teacher_ids must be"), ({"ids": _t(L, (8, 4), (1, 8), dtype=i32)}, "contiguous rows"),
            ({"teacher": _t(L, (8, 4), dtype=i32)}, "teacher_logits must be"), ({"teacher": _t(L, (9, 4))}, "teacher_logits must be"),
            ({"ids": _t(L, (8, 1025), dtype=i32), "teacher": _t(L, (8, 1025))}, "at most 1024"), ({}, "scratch must hold")]:
        assert _linear_status(L, distil=True, **other) < 0 and said in L.last_error(), (other, L.last_error())
    for tau in (0.0, -1.0, 1e-7, 2e6, float("inf"), float("nan")):
        assert _linear_status(L, distil=True, temperature=tau) < 0 and "temperature must be positive" in L.last_error()
    n = ctypes.c_size_t(0)
    x = _t(L, (8, 16))
    desc = L.CdlHeadLossDesc(1.0, 1.0, 0, 0)
    assert L.lib.cdl_b200_linear_loss_scratch_bytes(ctypes.byref(desc), ctypes.byref(x), None, 1, None, None, ctypes.byref(n)) < 0
    assert L.lib.cdl_b200_linear_loss_scratch_bytes(None, ctypes.byref(x), ctypes.byref(x), 1, None, None, ctypes.byref(n)) < 0
    assert L.lib.cdl_b200_linear_loss_scratch_bytes(ctypes.byref(desc), ctypes.byref(x), ctypes.byref(x), -1, None, None, ctypes.byref(n)) < 0


def test_distillation_refusals(cdl):
    L = cdl._lib
    base = {"logits": _t(L, (8, 40)), "ids": _t(L, (8, 4), dtype=L.CDL_I32), "teacher": _t(L, (8, 4)), "d_loss": None,
            "loss": _t(L, (8,), dtype=L.CDL_F32), "lse": None, "d_logits": _t(L, (8, 40), ptr=1 << 20)}
    for other, said in [
            ({"logits": None}, "logits must be"), ({"logits": _t(L, (8, 40), dtype=L.CDL_I32)}, "logits must be"),
            ({"logits": _t(L, (8, 40), (1, 8))}, "contiguous rows"), ({"logits": _t(L, (8, 0)), "d_logits": None}, "vocab is zero"),
            ({"d_logits": _t(L, (8, 40), dtype=L.CDL_F32)}, "d_logits must"), ({"d_logits": _t(L, (8, 40), (20, 1))}, "overlap"),
            ({"d_logits": _t(L, (8, 40), (48, 1))}, "themselves"), ({"ids": _t(L, (7, 4), dtype=L.CDL_I32)}, "teacher_ids must"),
            ({"loss": None}, "loss is required"), ({"lse": _t(L, (8,))}, "lse must be"),
            ({"logits": _t(L, (8, (1 << 30) + 1)), "d_logits": None}, "too large")]:
        a = {**base, **other}
        desc = L.CdlHeadLossDesc(1.0, 1.0, 0, 0)
        st = L.lib.cdl_b200_distillation(ctypes.byref(desc), *(None if a[n] is None else ctypes.byref(a[n]) for n in (
            "logits", "ids", "teacher", "d_loss", "loss", "lse", "d_logits")), None)
        assert st < 0 and said in L.last_error(), (other, L.last_error())


def test_front_ends_refuse_host_tensors_and_missing_gradients(cdl):
    x, w, ids = torch.zeros(4, 8), torch.zeros(8, 16), torch.zeros(4, dtype=torch.int32)
    for call in (lambda: cdl.ops.linear_cross_entropy(x, w, ids), lambda: cdl.ops.linear_distillation(x, w, ids[:, None], x[:, :1]),
                 lambda: cdl.ops.distillation(x, ids[:, None], x[:, :1]), lambda: cdl.ops.linear_cross_entropy(x[0], w, ids),
                 lambda: cdl.ops.distillation(x[0], ids[:, None], x[:, :1])):
        with pytest.raises(cdl._lib.CdlError):
            call()
    assert cdl.ops.linear_loss_scratch_bytes(x, w) > 0
    wider = cdl.ops.linear_loss_scratch_bytes(torch.zeros(100000, 8), torch.zeros(8, 32768), cdl.ops.LinearLossOpts())
    thin = cdl.ops.linear_loss_scratch_bytes(torch.zeros(1, 1).expand(1 << 26, 8), torch.zeros(8, 3))
    assert thin < 1.2e9, "a small vocabulary is padded to 128"
    assert wider < 100000 * 32768, "the scratch does not grow with the tokens"


def test_oracle_matches_torch_and_differences():
    gen = torch.Generator().manual_seed(0)
    z = torch.randn(6, 11, generator=gen, dtype=torch.float64)
    targets = torch.tensor([1, -1, 10, 3, 11, 0])
    loss, lse, g = ref.cross_entropy(z, targets)
    valid = (targets >= 0) & (targets < 11)
    want = torch.nn.functional.cross_entropy(z[valid], targets[valid], reduction="none")
    assert torch.allclose(loss[valid], want) and bool((loss[~valid] == 0).all()) and torch.allclose(lse, torch.logsumexp(z, 1))
    ids = torch.randint(-1, 12, (6, 4), generator=gen)
    ids[2], ids[3] = -1, 5
    teacher = torch.randn(6, 4, generator=gen, dtype=torch.float64)
    scale = torch.rand(6, generator=gen, dtype=torch.float64)
    f = lambda y: (ref.distillation(y, ids, teacher, 1.7)[0] * scale).sum()  # noqa: E731
    grad = ref.distillation(z, ids, teacher, 1.7, scale)[2]
    h = 1e-5
    for i in range(6):
        for j in range(11):
            e = torch.zeros_like(z)
            e[i, j] = h
            assert abs((f(z + e) - f(z - e)) / (2 * h) - grad[i, j]) < 1e-8
    # a teacher that holds the whole vocabulary: the divergence of two softmaxes
    full = torch.arange(11).expand(6, 11)
    t = torch.randn(6, 11, generator=gen, dtype=torch.float64)
    loss = ref.distillation(z, full, t, 2.0)[0]
    kl = torch.nn.functional.kl_div(torch.log_softmax(z / 2, 1), torch.log_softmax(t / 2, 1), log_target=True, reduction="none").sum(1)
    assert torch.allclose(loss, 4 * kl)
