"""Sizes of the 8-bit decoding calls at the limits of a single launch."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from vidchapters_amd import lib as L  # noqa: E402

DEV, BF = "cuda", torch.bfloat16
U32, UBF = 2.0 ** -24, 2.0 ** -8


@pytest.mark.parametrize("M,N,out,res", [(65535 * 64, 3, BF, True), (65535 * 64 + 70, 3, BF, True), (2 * 65535 * 64 + 1, 1, torch.float32, False)])
def test_product_of_more_rows_than_a_grid_has(M, N, out, res):
    """Fewer than eight columns go to the few-row kernels, 64 rows a block."""
    K = 16
    g = torch.Generator(device=DEV).manual_seed(1)
    A = torch.randint(-127, 128, (M, K), generator=g, device=DEV, dtype=torch.int8)
    B = torch.randint(-127, 128, (N, K), generator=g, device=DEV, dtype=torch.int8)
    sa, sb = torch.rand(M, generator=g, device=DEV) + 0.5, torch.rand(N, generator=g, device=DEV) + 0.5
    r = torch.randn(M, 8, generator=g, device=DEV).to(BF) if res else None
    C = torch.full((M + 1, 8), 7.0, dtype=out, device=DEV)
    L.gemm_q8(A, B, sa, sb, C, M, N, K, ldc=8, residual=r, ldr=8)
    assert (C[M:] == 7).all() and (C[:, N:] == 7).all()
    for a in range(0, M, 1 << 21):
        b = min(M, a + (1 << 21))
        acc = torch.stack([(A[a:b].int() * B[n].int()).sum(1) for n in range(N)], 1).double() * sa[a:b].double()[:, None] * sb.double()
        want, mag = (acc + r[a:b, :N].double(), acc.abs() + r[a:b, :N].double().abs()) if res else (acc, acc.abs())
        # fp32: the sum's conversion, two scales and alpha, bias, residual: 7 roundings of the terms' magnitude
        assert ((C[a:b, :N].double() - want).abs() <= mag * 7 * U32 + want.abs() * (UBF if out == BF else 0)).all(), a
