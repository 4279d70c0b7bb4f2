"""What the 8-bit decoding kernels hold between their inputs and the one rounding of their output, at inputs where fewer bits would show."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from vidchapters_amd import lib as L  # noqa: E402

DEV, BF, D = "cuda", torch.bfloat16, torch.float64


@pytest.mark.parametrize("G", [1, 2, 4, 16, 19])
@pytest.mark.parametrize("n", [70, 1400])                      # one piece of keys, and two with a join
@pytest.mark.parametrize("low", [16, 18, 20])
def test_attention_weights_hold_24_bits(G, n, low):
    """Two visible keys of equal score whose values all but cancel: v_0 = (1 + 2^-9 + 2^-low) c, v_1 = -(1 + 2^-9) c, output 2^-low c / 2.

    In fp32, (1 + 2^-9 + 2^-low) c is off by at most 2^-24 of itself per rounding and the running sum once more, so the output by at most 2 (2^-24 + 2^-9-24) c:
    a part 2^(low - 22) of it and a little, at most 0.26 at low = 20; weights of 16 bits lose the term whole."""
    H = 2
    kq = torch.randint(-127, 128, (1, H, n, 64), dtype=torch.int8, device=DEV)
    ks, vs = torch.ones(1, H, n, device=DEV), torch.ones(1, H, n, device=DEV)
    c = torch.randint(64, 128, (H, 64), device=DEV)
    vq = torch.randint(-127, 128, (1, H, n, 64), dtype=torch.int8, device=DEV)
    mask = torch.zeros(1, n, dtype=torch.uint8, device=DEV)
    a, b = 5, 37                                              # of one chunk of 64 keys
    mask[0, a] = mask[0, b] = 1
    vq[0, :, a], vq[0, :, b] = c.to(torch.int8), (-c).to(torch.int8)
    vs[0, :, a], vs[0, :, b] = 1 + 2.0 ** -9 + 2.0 ** -low, 1 + 2.0 ** -9
    q, o = torch.zeros(G, H * 64, dtype=BF, device=DEV), torch.empty(G, H * 64, dtype=BF, device=DEV)
    L.decode_attn_q8(q, kq, ks, vq, vs, o, n, group=G, key_mask=mask, workspace=L.decode_attn_q8_workspace(G, H, n, DEV))
    want = (c.double() * 2.0 ** -low / 2).reshape(1, -1)
    assert ((o.double() - want).abs() <= want * (2.0 ** (low - 22) * (1 + 2.0 ** -8) + 2.0 ** -8)).all(), float(((o.double() - want).abs() / want).max())


@pytest.mark.parametrize("kind", [1, 2, 3], ids=["few_rows", "64x64", "128x128"])
def test_gelu_within_its_bound(kind):
    """GELU of exact fp32 numbers v (one code of 1 per row and the row's scale): v Phi(v), off by at most 3.2 half steps of v.

    With T = Phi(-|v|), e = T / (1 - T), L = ln(1 / e), in units of 2^-24 |v|: the polynomial T (1 - T) |dL| <= 0.44, exponent and its product 2 L T (1 - T), exp2 to one
    unit 2 T (1 - T), 1 + e rounded T (1 - T), the reciprocal to one unit e, its product T, the last rounding max(T, 1 - T).  The sum is largest at v = 0:
    0.44 + 0.75 + 1 + 0.5 + 0.5 = 3.19."""
    M, N, K = 1 << 16, 8, 16
    A, B = torch.zeros(M, K, dtype=torch.int8, device=DEV), torch.zeros(N, K, dtype=torch.int8, device=DEV)
    A[:, 0] = 1
    B[:, 0] = 1
    sb = torch.ones(N, device=DEV)
    sb[1], sb[2], sb[3] = -1, 0.25, -0.25
    v = torch.cat([torch.linspace(0.3, 1.2, M // 2), torch.linspace(1.2, 12.0, M // 4), torch.logspace(-6, -0.5, M // 4)]).to(torch.float32).to(DEV)
    C = torch.empty(M, N, device=DEV)
    L.set_option("gemm_q8", kind)
    try:
        L.gemm_q8(A, B, v, sb, C, M, N, K, act=L.ACT_GELU)
    finally:
        L.set_option("gemm_q8", 0)
    x = v.double()[:, None] * sb.double()
    want = x * torch.special.ndtr(x)
    err = (C.double() - want).abs() / (x.abs() * 2.0 ** -24)
    assert float(err.max()) <= 3.2, (float(err.max()), float(x.flatten()[err.argmax()]))
    # infinities and NaN
    v[:4] = torch.tensor([float("inf"), float("-inf"), float("nan"), 0.0])
    L.gemm_q8(A, B, v, sb, C, M, N, K, act=L.ACT_GELU)
    assert float(C[0, 0]) == float("inf") and torch.isnan(C[1, 0]) and torch.isnan(C[2]).all() and (C[3] == 0).all()
