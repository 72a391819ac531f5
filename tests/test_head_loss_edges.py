"""Losses of the head where values are extreme: whole slices of a row masked.  The restatements in 64 bits are those of
test_head_loss.py; tolerances are derived where they stand."""
import pytest
import torch

from test_head_loss import BF16, F32, _check_distillation

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
