"""The int8 product's persistent tile loop: blocks that take several tiles, with one, two, three and more stages of 128 codes to a tile (the counted waits differ),
whole and partial last stages, whole tiles followed by further ones, and every write-out."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from vidchapters_amd import lib as L  # noqa: E402

DEV, BF = "cuda", torch.bfloat16
U32, UBF = 2.0 ** -24, 2.0 ** -8


def operands(M, N, K, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.rand(*s, generator=g, device=DEV)              # noqa: E731
    A = torch.randint(-127, 128, (M, K), generator=g, device=DEV, dtype=torch.int8)
    B = torch.randint(-127, 128, (N, K), generator=g, device=DEV, dtype=torch.int8)
    return A, B, r(M) * 0.02 + 0.001, r(N) * 0.02 + 0.001, r(N) - 0.5, (r(M, (N + 7) // 8 * 8) - 0.5).to(BF)


FORMS = [(BF, L.ACT_NONE, False), (BF, L.ACT_RELU, True), (torch.float32, L.ACT_NONE, True), (BF, L.ACT_GELU, False)]


@pytest.mark.parametrize("kind", [2, 3, 4], ids=["64x64", "128x128", "256x256"])
@pytest.mark.parametrize("K", [64, 128, 144, 384, 400, 768, 1040])
@pytest.mark.parametrize("form", range(4), ids=["plain", "residual", "fp32", "gelu"])
def test_blocks_of_several_tiles(kind, K, form):
    M, N = (5100, 4104) if K % 256 else (4864, 4099)                    # 340 / 323 tiles of 256 x 256 for 256 blocks, more of the smaller ones
    out, act, with_res = FORMS[form]
    A, B, sa, sb, bias, res = operands(M, N, K, K + kind)
    ld = (N + 7) // 8 * 8
    runs = []
    L.set_option("gemm_q8", kind)
    try:
        for _ in range(3):
            C = torch.full((M + 1, ld), 7.0, dtype=out, device=DEV)
            L.gemm_q8(A, B, sa, sb, C, M, N, K, ldc=ld, bias=bias, act=act, residual=res if with_res else None, ldr=ld)
            runs.append(C)
    finally:
        L.set_option("gemm_q8", 0)
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])
    C = runs[0]
    assert (C[M:] == 7).all() and (C[:, N:] == 7).all()
    acc = A.double() @ B.double().t().contiguous() * sa.double()[:, None] * sb.double()
    v, mag = acc + bias.double(), acc.abs() + bias.double().abs()
    if act == L.ACT_RELU:
        v = v.clamp_min(0)
    if act == L.ACT_GELU:
        v = v * torch.special.ndtr(v)
    if with_res:
        v, mag = v + res[:, :N].double(), mag + res[:, :N].double().abs()
    # fp32: the sum's conversion, two scales and alpha, bias, residual: 7 roundings of the terms' magnitude (the derivative of v Phi(v) stays below 1.13); GELU to
    # 3.6 half steps of v
    tol = mag * (7 if act != L.ACT_GELU else 7 * 1.13 + 3.6) * U32 + v.abs() * (UBF if out == BF else 0)
    assert ((C[:M, :N].double() - v).abs() <= tol).all()
