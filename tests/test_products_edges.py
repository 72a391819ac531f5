"""Products that add to D: what lies behind D's rows stays as it was."""
import pytest
import torch

from test_head_loss import BF16, F32, _close

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("n", [1, 3, 34, 127, 301, 1101])
@pytest.mark.parametrize("k,deterministic", [(128, False), (4096, False), (4096, True)])
@pytest.mark.parametrize("kind", ["bf16", "mxfp8"])
def test_additions_leave_what_lies_behind_the_rows(cdl, gpu_ok, n, k, deterministic, kind):
    """D += A B in f32 with rows on the 16-byte grid that end inside 16 bytes, beside a row of A that is infinite: NaN there, and
    nowhere behind a row."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    m = 2048
    a = torch.randn(m, k, generator=gen, device="cuda").to(BF16)
    b = torch.randn(n, k, generator=gen, device="cuda").to(BF16)
    buffer = torch.full((m, (n + 3) // 4 * 4 + 4), -0.0, device="cuda")
    before = torch.randn(m, n, generator=gen, device="cuda")
    d = buffer[:, :n]
    d.copy_(before)
    if kind == "mxfp8":
        qa, qb = (cdl.mx.quantize(y, rowwise=True)[0] for y in (a, b))
        qb = qb.transposed()
        want = before.double() + cdl.mx.matmul_mx(qa, qb, out_dtype=F32).double()
        cdl.mx.matmul_mx(qa, qb, out=d, c=d, beta=1.0, variant=cdl._lib.GEMM_CTA_PAIR)
        tol = 2.0 ** -22 * (want.abs() + before.abs())
    else:
        a[7, 0] = float("inf")
        a[9, 1] = float("nan")
        b[0, :2] = 0.0
        want = before.double() + a.double() @ b.double().t()
        opts = cdl.ops.MatmulOpts(out=F32, c=d, beta=1.0, variant=cdl._lib.GEMM_CTA_PAIR, deterministic=deterministic)
        cdl.ops.matmul(a, b.t(), opts, out=d)
        # 16 products a step, each of which may cut 2^-23 of the largest partial sum; the result's rounding
        tol = (k / 16 + 8) * 2.0 ** -23 * torch.nan_to_num(a.double().abs(), posinf=0.0) @ b.double().abs().t() + 2.0 ** -23 * want.abs()
    _close("d", d, want, torch.nan_to_num(tol, posinf=0.0))
    behind = buffer[:, n:]
    assert bool(((behind == 0) & torch.signbit(behind)).all())
