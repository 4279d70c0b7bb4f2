"""Views as operands of the 8-bit decoding calls, without a stride given: read and written where their rows lie."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from vidchapters_amd import lib as L  # noqa: E402

DEV, BF = "cuda", torch.bfloat16


def wide(t, fill, left=16, right=32):
    """a tensor of the same rows within wider ones, and the buffer that holds it"""
    buf = torch.full((t.shape[0], left + t.shape[1] + right), fill, dtype=t.dtype, device=DEV)
    view = buf[:, left:left + t.shape[1]]
    view.copy_(t)
    return view, buf


def untouched(buf, fill, cols, left=16):
    return bool((buf[:, :left] == fill).all() and (buf[:, left + cols:] == fill).all())


def test_rows_of_views():
    rows, cols = 37, 264
    g = torch.Generator(device=DEV).manual_seed(1)
    x, d = torch.randn(rows, cols, generator=g, device=DEV).to(BF), torch.randn(rows, cols, generator=g, device=DEV).to(BF)
    w = torch.randn(cols, generator=g, device=DEV)
    new = lambda dt: torch.zeros(rows, cols, dtype=dt, device=DEV)      # noqa: E731
    q, s, h, y = new(torch.int8), torch.zeros(rows, device=DEV), new(BF), new(BF)
    L.rmsnorm_q8(x, w, q, s, rows, cols, 1e-6, delta=d, h=h)
    L.dequant_q8(q, s, y, rows, cols)
    (xv, _), (dv, _), (qv, qb), (hv, hb), (yv, yb) = wide(x, 5), wide(d, 6), wide(new(torch.int8), 7), wide(new(BF), 8), wide(new(BF), 9)
    s2 = torch.zeros(rows, device=DEV)
    L.rmsnorm_q8(xv, w, qv, s2, rows, cols, 1e-6, delta=dv, h=hv)
    L.dequant_q8(qv, s2, yv, rows, cols)
    for got, want in ((qv, q), (s2, s), (hv, h), (yv, y)):
        assert torch.equal(got, want)
    assert untouched(qb, 7, cols) and untouched(hb, 8, cols) and untouched(yb, 9, cols)
    xf = x.float()
    L.quant_rows_q8(xf, q, s, rows, cols)
    qv.zero_()
    L.quant_rows_q8(wide(xf, 1)[0], qv, s2, rows, cols)
    assert torch.equal(qv, q) and torch.equal(s2, s) and untouched(qb, 7, cols)


@pytest.mark.parametrize("M", [1, 5, 300])
def test_product_of_views(M):
    N, K = 136, 96
    g = torch.Generator(device=DEV).manual_seed(M)
    A = torch.randint(-127, 128, (M, K), generator=g, device=DEV, dtype=torch.int8)
    B = torch.randint(-127, 128, (N, K), generator=g, device=DEV, dtype=torch.int8)
    sa, sb = torch.rand(M, generator=g, device=DEV), torch.rand(N, generator=g, device=DEV)
    r = torch.randn(M, N, generator=g, device=DEV).to(BF)
    want = torch.zeros(M, N, dtype=BF, device=DEV)
    L.gemm_q8(A, B, sa, sb, want, M, N, K, residual=r)
    (Av, _), (Bv, _), (rv, _), (Cv, Cb) = wide(A, 3), wide(B, 4), wide(r, 5), wide(torch.zeros_like(want), 6)
    L.gemm_q8(Av, Bv, sa, sb, Cv, M, N, K, residual=rv)
    assert torch.equal(Cv, want) and untouched(Cb, 6, N)
    # leading dimensions of views, whole tensors of wider and of more rows, and rows laid end to end
    if M == 300:
        C3 = torch.zeros(3, 100, N + 24, dtype=BF, device=DEV)
        L.gemm_q8(Av.view(3, 100, K), B, sa, sb, C3[..., :N], M, N, K, residual=r.view(3, 100, N))
        assert torch.equal(C3[..., :N].reshape(M, N), want) and (C3[..., N:] == 0).all()
    Ct, At = torch.zeros(M + 2, N + 8, dtype=BF, device=DEV), torch.zeros(M + 2, K + 16, dtype=torch.int8, device=DEV)
    At[:M, :K] = A
    L.gemm_q8(At, B, sa, sb, Ct, M, N, K, residual=r)
    if M > 1:
        assert torch.equal(Ct[:M, :N], want) and (Ct[M:] == 0).all() and (Ct[:, N:] == 0).all()
    else:
        assert torch.equal(Ct[:M, :N], want)
    flat = torch.zeros(M * N + 5, dtype=BF, device=DEV)
    L.gemm_q8(A.flatten(), B, sa, sb, flat, M, N, K, residual=r)
    assert torch.equal(flat[:M * N].view(M, N), want) and (flat[M * N:] == 0).all()


def test_logits_of_views():
    rows, V = 6, 500
    g = torch.Generator(device=DEV).manual_seed(2)
    z, u = torch.randn(rows, V, generator=g, device=DEV), torch.rand(rows, generator=g, device=DEV)
    tok, got = torch.zeros(rows, dtype=torch.long, device=DEV), torch.zeros(rows, dtype=torch.long, device=DEV)
    L.sample_step(z, rows, V, u, tok)
    last = torch.randn(rows, 3, V, generator=g, device=DEV)
    last[:, -1] = z
    for v in (wide(z, 50.0)[0], last[:, -1], last[:, -1:], torch.cat([z, torch.full((rows, 12), 60.0, device=DEV)], 1)):
        L.sample_step(v, rows, V, u, got)
        assert torch.equal(got, tok)


def test_sequence_rows_have_their_own_length():
    """The token of every step also goes into its column, with and without the row length; a step behind the last column writes none."""
    rows, V, steps = 5, 400, 4
    g = torch.Generator(device=DEV).manual_seed(3)
    z, u = torch.randn(rows, V, generator=g, device=DEV), torch.rand(steps, rows, generator=g, device=DEV)
    pos, tok = torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros(rows, dtype=torch.long, device=DEV)
    for kw in ({}, dict(seq_ld=0), dict(seq_ld=steps)):
        seq, want = torch.full((rows + 1, steps), -1, dtype=torch.long, device=DEV), torch.full((rows + 1, steps), -1, dtype=torch.long, device=DEV)
        for t in range(steps):
            pos.fill_(t)
            L.sample_step(z, rows, V, u, tok, seq_out=seq, pos_dev=pos, **kw)
            if t + 1 < steps:
                want[:rows, t + 1] = tok
        assert torch.equal(seq, want)
