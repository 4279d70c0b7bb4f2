"""8-bit decoding kernels against plain statements in 64 bits: rows to int8 codes (with the residual addition and RMSNorm), the int8 product, the int8
key / value cache and the attention that reads it, sampling from given numbers, and a run of them together.

Tolerances count roundings (half a step: fp32 2^-24, bf16 2^-8 relative to the value) and are written beside each check."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from vidchapters_amd import lib as L  # noqa: E402

DEV, BF, D = "cuda", torch.bfloat16, torch.float64
U32, UBF = 2.0 ** -24, 2.0 ** -8
TINY = 127 * 2.0 ** -126


def rnd(*shape, seed=0, scale=1.0, dtype=BF):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def codes(rows, cols, seed):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-127, 128, (rows, cols), generator=g).to(torch.int8)
    return q.to(DEV), (torch.rand(rows, generator=g) * 0.02 + 0.001).to(DEV)


def nan_equal(a, b):
    return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0))


# --------------------------------------------------------------------------------------------- rows -> codes
def check_codes(q, scale, y, slack):
    """y: the row values in 64 bits, slack: relative error of the kernel's fp32 y.  The code of y lies within half a step, up to the 127 codes' slack."""
    want = y.abs().amax(1).clamp_min(TINY) / 127
    assert ((scale.double() - want).abs() <= want * (slack + 3 * U32)).all()
    err = (q.double() * scale.double()[:, None] - y).abs() / want[:, None]
    assert float(err.max()) <= 0.5 + 127 * (2 * slack + 6 * U32), float(err.max())
    assert int(q.abs().amax()) <= 127


@pytest.mark.parametrize("rows,cols", [(1, 8), (3, 64), (5, 72), (131, 128), (67, 136), (35, 256), (9, 264), (64, 768), (37, 1024), (9, 1032), (7, 2048), (6, 4096), (3, 8192), (1025, 520)])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_quant_rows(rows, cols, dtype):
    x = rnd(rows, cols, seed=rows, dtype=dtype) * torch.logspace(-3, 3, rows, device=DEV)[:, None].to(dtype)
    q, s = torch.empty(rows, cols, dtype=torch.int8, device=DEV), torch.empty(rows, device=DEV)
    L.quant_rows_q8(x, q, s, rows, cols)
    check_codes(q, s, x.double(), 0.0)
    y = torch.empty(rows, cols, dtype=BF, device=DEV)
    L.dequant_q8(q, s, y, rows, cols)
    want = q.double() * s.double()[:, None]
    assert ((y.double() - want).abs() <= want.abs() * (UBF + 2 * U32)).all()


@pytest.mark.parametrize("rows,cols,add,store", [(1, 8, True, True), (77, 48, True, True), (50, 128, False, False), (33, 248, True, True), (64, 768, True, True), (65, 768, True, False), (33, 1024, False, False), (5, 2040, True, True),
                                                 (4, 4096, True, True), (2, 8192, False, False), (4099, 768, True, True)])
def test_rmsnorm_q8(rows, cols, add, store):
    x, d = rnd(rows, cols, seed=1, scale=2.0), rnd(rows, cols, seed=2)
    w = (1 + 0.3 * rnd(cols, seed=3, dtype=torch.float32)).contiguous()
    q, s = torch.empty(rows, cols, dtype=torch.int8, device=DEV), torch.empty(rows, device=DEV)
    h = torch.empty(rows, cols, dtype=BF, device=DEV) if store else None
    L.rmsnorm_q8(x, w, q, s, rows, cols, 1e-6, delta=d if add else None, h=h)
    sm = (x.float() + d.float()).to(BF) if add else x
    if store:
        assert torch.equal(h, sm)
    v = sm.double()
    y = v / (v.square().mean(1, keepdim=True) + 1e-6).sqrt() * w.double()
    # fp32: cols / 64 + 6 additions of positive squares, their square root, the reciprocal root to one unit (2 U32), three products
    check_codes(q, s, y, (cols / 128 + 10) * U32)


def test_rows_strided_in_place_and_untouched():
    rows, cols = 21, 264
    wide = rnd(rows, 400, seed=4)
    x, d = wide[:, 8:8 + cols], rnd(rows, 304, seed=5)[:, 40:40 + cols]
    w = torch.ones(cols, device=DEV)
    qbuf, sbuf = torch.full((rows + 2, 272), 77, dtype=torch.int8, device=DEV), torch.full((rows + 2,), 7.0, device=DEV)
    ref_q, ref_s, ref_h = torch.empty(rows, cols, dtype=torch.int8, device=DEV), torch.empty(rows, device=DEV), torch.empty(rows, cols, dtype=BF, device=DEV)
    L.rmsnorm_q8(x.contiguous(), w, ref_q, ref_s, rows, cols, 1e-6, delta=d.contiguous(), h=ref_h)
    before = wide.clone()
    L.rmsnorm_q8(x, w, qbuf, sbuf, rows, cols, 1e-6, delta=d, h=x, ldx=400, ldd=304, ldh=400, ldq=272)      # the sum replaces x
    assert torch.equal(qbuf[:rows, :cols], ref_q) and torch.equal(sbuf[:rows], ref_s) and torch.equal(x, ref_h)
    assert (qbuf[:, cols:] == 77).all() and (qbuf[rows:] == 77).all() and (sbuf[rows:] == 7).all()
    assert torch.equal(wide[:, :8], before[:, :8]) and torch.equal(wide[:, 8 + cols:], before[:, 8 + cols:])


def test_rows_of_zeros_tiny_values_and_infinities():
    cols = 64
    x = torch.zeros(6, cols, device=DEV)
    x[1, 3] = 1e-38                          # below the floor of the scale
    x[2, 5], x[3, 9], x[4, 0] = math.inf, math.nan, -math.inf
    x[5] = 3e38
    q, s, y = torch.full((6, cols), 9, dtype=torch.int8, device=DEV), torch.empty(6, device=DEV), torch.empty(6, cols, dtype=BF, device=DEV)
    L.quant_rows_q8(x, q, s, 6, cols)
    L.dequant_q8(q, s, y, 6, cols)
    assert (q[:1] == 0).all() and (y[0] == 0).all() and float(s[0]) == float(s[1]) == 2.0 ** -126
    assert int(q[1, 3]) == 1 and int(q[1].abs().sum()) == 1
    assert torch.isnan(s[2:5]).all() and (q[2:5] == 0).all() and torch.isnan(y[2:5]).all()
    assert (q[5] == 127).all() and torch.isfinite(s[5])
    xb = x.to(BF)
    for row in (2, 3, 4):
        L.rmsnorm_q8(xb[row:row + 1], torch.ones(cols, device=DEV), q[:1], s[:1], 1, cols, 1e-6)
        assert torch.isnan(s[0]) and (q[0] == 0).all()


# --------------------------------------------------------------------------------------------- product
def product_ref(A, B, sa, sb, alpha, bias, act, res):
    """(value, magnitude of the terms the fp32 epilogue adds) in 64 bits"""
    acc = A.double() @ B.double().t().contiguous() * sa.double()[:, None] * sb.double()[None] * alpha
    v, mag = acc, acc.abs()
    if bias is not None:
        v, mag = v + bias.double(), mag + bias.double().abs()
    if act == L.ACT_RELU:
        v = v.clamp_min(0)
    if act == L.ACT_GELU:
        v = 0.5 * v * (1 + torch.erf(v * 0.5 ** 0.5))
    if res is not None:
        v, mag = v + res.double(), mag + res.double().abs()
    return v, mag


SHAPES = [(1, 8, 16), (1, 2304, 768), (3, 5, 32), (17, 100, 48), (64, 768, 768), (64, 612, 128), (65, 130, 80), (37, 32228, 64), (100, 1000, 4096), (128, 128, 64),
          (200, 257, 144), (257, 520, 336), (300, 640, 1024), (513, 769, 400), (1000, 264, 2048), (1027, 2304, 768), (2050, 1032, 1040)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("out", [BF, torch.float32])
def test_gemm_q8(M, N, K, out):
    A, sa = codes(M, K, M + N)
    B, sb = codes(N, K, K + 1)
    ld = (N + 7) // 8 * 8 + 8
    bias, res = rnd(N, seed=5, dtype=torch.float32), rnd(M, ld, seed=6)
    for act, b, r, alpha in ((L.ACT_NONE, None, None, 1.0), (L.ACT_RELU, bias, None, 0.25), (L.ACT_GELU, bias, res, 0.125), (L.ACT_NONE, None, res, 1.0)):
        C = torch.full((M + 1, ld), 7.0, dtype=out, device=DEV)
        L.gemm_q8(A, B, sa, sb, C, M, N, K, ldc=ld, alpha=alpha, bias=b, act=act, residual=r, ldr=ld)
        want, mag = product_ref(A, B, sa, sb, alpha, b, act, None if r is None else r[:, :N])
        got = C[:M, :N].double()
        # fp32: the sum's conversion, two scales and alpha, bias, residual: 7 roundings of the terms' magnitude; erf to 4 units where it is used
        tol = mag * (7 if act != L.ACT_GELU else 16) * U32 + want.abs() * (UBF if out == BF else 0)
        bad = (got - want).abs() > tol
        assert not bad.any(), (act, int(bad.sum()), float(((got - want).abs() / tol.clamp_min(1e-30)).max()))
        assert (C[:M, N:] == 7).all() and (C[M:] == 7).all()      # nothing outside the product is written


@pytest.mark.parametrize("kind", [1, 2, 3, 4], ids=["few_rows", "64x64", "128x128", "256x256"])
@pytest.mark.parametrize("M,N,K", [(1, 8, 16), (70, 300, 48), (130, 257, 112), (300, 520, 64), (257, 513, 1040), (128, 512, 4096), (513, 769, 784)])
def test_gemm_q8_every_kernel_gives_the_same_bits(M, N, K, kind):
    A, sa = codes(M, K, 3)
    B, sb = codes(N, K, 4)
    ld = (N + 7) // 8 * 8
    res = rnd(M, ld, seed=6)
    want, mag = product_ref(A, B, sa, sb, 1.0, None, L.ACT_NONE, res[:, :N])
    auto, C = torch.zeros(M + 1, ld, dtype=BF, device=DEV), torch.zeros(M + 1, ld, dtype=BF, device=DEV)
    L.gemm_q8(A, B, sa, sb, auto, M, N, K, ldc=ld, residual=res, ldr=ld)
    L.set_option("gemm_q8", kind)
    try:
        L.gemm_q8(A, B, sa, sb, C, M, N, K, ldc=ld, residual=res, ldr=ld)
    finally:
        L.set_option("gemm_q8", 0)
    assert torch.equal(C, auto) and (C[M:] == 0).all()
    assert ((C[:M, :N].double() - want).abs() <= mag * 7 * U32 + want.abs() * UBF).all()


@pytest.mark.parametrize("kind", [2, 3, 4], ids=["64x64", "128x128", "256x256"])
@pytest.mark.parametrize("out,act,res", [(BF, L.ACT_RELU, False), (BF, L.ACT_NONE, True), (BF, L.ACT_GELU, True), (torch.float32, L.ACT_NONE, False)])
@pytest.mark.parametrize("N", [4104, 4099, 4101, 4094])
def test_gemm_q8_more_tiles_than_blocks(kind, out, act, res, N):
    """A block that takes several tiles, with every form of the write-out and rows and columns left over; the residual ends with its last value."""
    M, K = 5100, 144
    A, sa = codes(M, K, 13)
    B, sb = codes(N, K, 14)
    ld = (N + 7) // 8 * 8
    bias, r = rnd(N, seed=5, dtype=torch.float32), rnd((M - 1) * ld + N, seed=6).as_strided((M, N), (ld, 1)) if res else None
    C = torch.full((M + 1, ld), 7.0, dtype=out, device=DEV)
    L.set_option("gemm_q8", kind)
    try:
        L.gemm_q8(A, B, sa, sb, C, M, N, K, bias=bias, act=act, residual=r, ldc=ld, ldr=ld)
    finally:
        L.set_option("gemm_q8", 0)
    want, mag = product_ref(A, B, sa, sb, 1.0, bias, act, r)
    tol = mag * (7 if act != L.ACT_GELU else 16) * U32 + want.abs() * (UBF if out == BF else 0)
    assert ((C[:M, :N].double() - want).abs() <= tol).all() and (C[M:] == 7).all() and (C[:, N:] == 7).all()


def test_gemm_q8_few_columns_of_many_rows():
    """Fewer than eight columns go to the few-row kernels, whatever is asked for."""
    for M, N, K in ((70000, 1, 64), (40000, 5, 48), (66000, 7, 32)):
        A, sa = codes(M, K, 3)
        B, sb = codes(N, K, 4)
        r = rnd((M - 1) * 8 + N, seed=6).as_strided((M, N), (8, 1))
        want, mag = product_ref(A, B, sa, sb, 1.0, None, L.ACT_NONE, r)
        for kind in (0, 2, 3, 4):
            C = torch.full((M, 8), 7.0, dtype=BF, device=DEV)
            L.set_option("gemm_q8", kind)
            try:
                L.gemm_q8(A, B, sa, sb, C, M, N, K, residual=r, ldc=8, ldr=8)
            finally:
                L.set_option("gemm_q8", 0)
            assert ((C[:, :N].double() - want).abs() <= mag * 7 * U32 + want.abs() * UBF).all() and (C[:, N:] == 7).all()


def test_gemm_q8_codes_are_summed_exactly():
    """The largest sums int8 codes can have: all -128, K at its limit; and sums that differ by one."""
    K = 131056
    A = torch.full((3, K), -128, dtype=torch.int8, device=DEV)
    B = torch.full((9, K), -128, dtype=torch.int8, device=DEV)
    B[1, 0] = -127
    B[2] = 127
    one = torch.ones(16, device=DEV)
    C = torch.empty(3, 16, device=DEV)
    L.gemm_q8(A, B, one, one, C, 3, 9, K, ldc=16)
    want = (A[:1].double() @ B.double().t()).float().repeat(3, 1)        # one rounding of the exact sum
    assert torch.equal(C[:, :9], want)


def test_gemm_q8_strides_in_place_residual_and_nan_scales():
    M, N, K = 130, 96, 160
    A, sa = codes(M, 512, 1)
    B, sb = codes(N, 256, 2)
    a, b = A[:, 32:32 + K], B[:, 16:16 + K]
    C = rnd(M, 104, seed=3)
    old = C.clone()
    sa[7] = math.nan
    sb[5] = math.inf
    L.gemm_q8(a, b, sa, sb, C, M, N, K, lda=512, ldb=256, ldc=104, residual=C, ldr=104)
    want, mag = product_ref(a, b, sa, sb, 1.0, None, L.ACT_NONE, old[:, :N])
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(C[:, :N]), fine)
    err = (C[:, :N].double() - want)[fine].abs()
    assert (err <= (mag * 7 * U32 + want.abs() * UBF)[fine]).all()
    assert torch.equal(C[:, N:], old[:, N:])


def test_gemm_q8_row_strides_behind_2_31_bytes():
    """Rows of one tile that start further apart than 2^31 bytes, at the largest stride."""
    M, N, K, ld = 256, 200, 272, 1 << 24
    A, sa = codes(M, K, 1)
    B, sb = codes(N, K, 2)
    far = torch.empty((M - 1) * ld + K, dtype=torch.int8, device=DEV)
    a = far.as_strided((M, K), (ld, 1))
    a.copy_(A)
    want, C = torch.empty(M, N, dtype=BF, device=DEV), torch.empty(M, N, dtype=BF, device=DEV)
    L.gemm_q8(A, B, sa, sb, want, M, N, K)
    for kind in (1, 2, 3, 4):
        C.zero_()
        L.set_option("gemm_q8", kind)
        try:
            L.gemm_q8(a, B, sa, sb, C, M, N, K, lda=ld)
        finally:
            L.set_option("gemm_q8", 0)
        assert torch.equal(C, want), kind
    b = far.as_strided((N, K), (ld, 1))
    b.copy_(B)
    L.gemm_q8(A, b, sa, sb, C, M, N, K, ldb=ld)
    assert torch.equal(C, want)


def test_gemm_q8_rows_do_not_depend_on_their_batch():
    """Sums are exact and the epilogue is per value: a row's result is the same bits in any call, whatever kernel the size chose."""
    M, N, K = 700, 776, 768
    A, sa = codes(M, K, 8)
    B, sb = codes(N, K, 9)
    bias = rnd(N, seed=1, dtype=torch.float32)
    full = torch.empty(M, N, dtype=BF, device=DEV)
    L.gemm_q8(A, B, sa, sb, full, M, N, K, bias=bias, act=L.ACT_GELU)
    for m in (1, 5, 64, 65, 200):
        part = torch.empty(m, N, dtype=BF, device=DEV)
        L.gemm_q8(A, B, sa, sb, part, m, N, K, bias=bias, act=L.ACT_GELU)
        assert torch.equal(part, full[:m])


# --------------------------------------------------------------------------------------------- cache
def new_cache(E, H, n, fill=0):
    c = [torch.full((E, H, n, 64), fill, dtype=torch.int8, device=DEV), torch.full((E, H, n), float(fill), device=DEV)]
    return c + [t.clone() for t in c]


@pytest.mark.parametrize("E,H,T,n", [(1, 1, 1, 1), (3, 5, 1, 9), (64, 12, 1, 32), (2, 12, 7, 40), (2, 3, 8, 8), (5, 12, 33, 50), (2, 16, 130, 200)])
def test_kv_append_and_read(E, H, T, n):
    kv = rnd(E, T + 2, 2 * H * 64 + 8, seed=E + T, scale=3.0)
    k, v = kv[:, :, :H * 64], kv[:, :, H * 64:2 * H * 64]
    g = torch.Generator().manual_seed(1)
    pos = torch.randint(0, n - T + 1, (E,), generator=g).to(torch.int32).to(DEV)
    cnt = torch.randint(0, T + 1, (E,), generator=g).to(torch.int32).to(DEV)
    for count in (None, cnt):
        kq, ks, vq, vs = new_cache(E, H, n, 5)
        L.kv_append_q8(k, v, kq, ks, vq, vs, T, pos=pos, count=count)
        ko, vo = torch.full((E, T, H * 64), 7.0, dtype=BF, device=DEV), torch.full((E, T, H * 64), 7.0, dtype=BF, device=DEV)
        L.kv_read_q8(kq, ks, vq, vs, ko, vo, T, pos=pos, count=count)
        for x, q, s, back in ((k, kq, ks, ko), (v, vq, vs, vo)):
            live = torch.zeros(E, n, dtype=torch.bool, device=DEV)
            for e in range(E):
                m, p = T if count is None else int(cnt[e]), int(pos[e])
                live[e, p:p + m] = True
                if m:
                    y = x[e, :m].double().reshape(m * H, 64)
                    check_codes(q[e, :, p:p + m].transpose(0, 1).reshape(m * H, 64), s[e, :, p:p + m].t().reshape(-1), y, 0.0)
                    w = (q[e, :, p:p + m].double() * s[e, :, p:p + m, None].double()).transpose(0, 1).reshape(m, H * 64)
                    assert ((back[e, :m].double() - w).abs() <= w.abs() * (UBF + 2 * U32)).all()
                assert (back[e, m:] == 7).all()
            dead = ~live[:, None].expand(E, H, n)
            assert (q[dead] == 5).all() and (s[dead] == 5).all()      # rows that take no part stay as they were


def test_kv_append_drops_tokens_outside_the_cache():
    E, H, T, n = 3, 2, 9, 12
    k, v = rnd(E, T, H * 64, seed=1), rnd(E, T, H * 64, seed=2)
    pos = torch.tensor([-3, 8, 40], dtype=torch.int32, device=DEV)
    guard = new_cache(E + 2, H, n, 3)
    inner = [t[1:1 + E] for t in guard]
    L.kv_append_q8(k, v, *inner, T, pos=pos)
    want = new_cache(E, H, n, 3)
    L.kv_append_q8(k[:1, 3:].contiguous(), v[:1, 3:].contiguous(), *[t[:1] for t in want], 6, pos0=0)
    L.kv_append_q8(k[1:2, :4].contiguous(), v[1:2, :4].contiguous(), *[t[1:2] for t in want], 4, pos0=8)
    for a, b, c in zip(inner, want, guard):
        assert torch.equal(a, b) and (c[0] == 3).all() and (c[-1] == 3).all()
    ctr = torch.tensor([4], dtype=torch.int32, device=DEV)
    L.kv_append_q8(k, v, *inner, 1, pos0=1, pos_dev=ctr)               # the counter is added to pos0
    L.kv_append_q8(k, v, *want, 1, pos0=5)
    for a, b in zip(inner, want):
        assert torch.equal(a, b)


# --------------------------------------------------------------------------------------------- attention
def attn_ref(q, kq, ks, vq, vs, scale, G, klen, mask, bias):
    E, H, n, _ = kq.shape
    k, v = kq.double() * ks.double()[..., None], vq.double() * vs.double()[..., None]
    out, tol = torch.zeros(E * G, H, 64, dtype=D, device=DEV), torch.zeros(E * G, H, 64, dtype=D, device=DEV)
    for e in range(E):
        m = n if klen is None else min(max(int(klen[e]), 0), n)
        if m == 0:
            continue
        see = torch.ones(m, dtype=torch.bool, device=DEV) if mask is None else mask[e, :m] != 0
        for h in range(H):
            b = torch.zeros(m, dtype=D, device=DEV) if bias is None else bias[h, :m].double()
            s = see & (b > -math.inf)
            if not s.any():
                mean = v[e, h, :m].mean(0)
                out[e * G:(e + 1) * G, h] = mean
                tol[e * G:(e + 1) * G, h] = mean.abs() * UBF + v[e, h, :m].abs().mean(0) * (m / 4 + 8) * U32
                continue
            kk, vv, bb = k[e, h, :m][s], v[e, h, :m][s], b[s]
            x = q[e * G:(e + 1) * G].double().view(G, H, 64)[:, h]
            z = x @ kk.t().contiguous() * scale + bb
            p = torch.softmax(z, 1)
            out[e * G:(e + 1) * G, h] = p @ vv
            # a score: 16 additions of a lane, 2 across lanes, two scales, bias, log2 e; the weights carry it and their own rounding, sums at most 128 more
            dz = ((x.abs() @ kk.abs().t().contiguous() * abs(scale)).amax(1, keepdim=True) + bb.abs().amax() + 1) * 24 * U32
            tol[e * G:(e + 1) * G, h] = (p @ vv).abs() * UBF + 2 * (dz + 160 * U32) * (p @ vv.abs())
    return out.view(E * G, H * 64), tol.view(E * G, H * 64)


def attend(q, cache, n, **kw):
    o = torch.full_like(q, 9.0)
    G, H = kw.get("group", 1), cache[0].shape[1]
    L.decode_attn_q8(q, *cache, o, n, workspace=L.decode_attn_q8_workspace(q.shape[0], H, n, DEV), **kw)
    return o


def make_cache(E, H, n, seed):
    kq, ks = codes(E * H * n, 64, seed)
    vq, vs = codes(E * H * n, 64, seed + 1)
    return [kq.view(E, H, n, 64), ks.view(E, H, n), vq.view(E, H, n, 64), vs.view(E, H, n)]


@pytest.mark.parametrize("E,G,H,n", [(1, 1, 1, 1), (2, 1, 3, 2), (3, 1, 12, 63), (2, 2, 4, 64), (2, 3, 2, 65), (64, 1, 12, 100), (2, 4, 12, 511), (2, 5, 2, 512),
                                     (3, 1, 2, 513), (2, 8, 3, 1100), (1, 4, 16, 5000), (4, 1, 2, 1537), (1, 12, 2, 700), (1, 17, 1, 1030), (2, 1, 2, 1280), (2, 16, 2, 1281),
                                     (1, 33, 2, 2561)])
@pytest.mark.parametrize("form", ["plain", "len", "mask_bias", "all"])
def test_decode_attn_q8(E, G, H, n, form):
    cache = make_cache(E, H, n, n + G)
    q = rnd(E * G, H * 64, seed=3, scale=2.0)
    g = torch.Generator().manual_seed(E * n)
    klen = torch.randint(1, n + 1, (E,), generator=g).to(torch.int32).to(DEV) if form in ("len", "all") else None
    mask = bias = None
    if form in ("mask_bias", "all"):
        mask = (torch.rand(E, n + 3, generator=g) < 0.7).to(torch.uint8).to(DEV)
        bias = torch.randn(H, n + 5, generator=g).to(DEV)
        bias[:, ::7] = -math.inf
        if n > 600:
            mask[0, :min(n - 20, 1300)] = 0      # whole pieces without a visible key
    o = attend(q, cache, n, group=G, klen=klen, key_mask=mask, bias_row=bias, scale=0.5)
    want, tol = attn_ref(q, *cache, 0.5, G, klen, mask, bias)
    assert ((o.double() - want).abs() <= tol).all(), float(((o.double() - want).abs() / tol).max())


def test_decode_attn_q8_rows_without_keys_and_hidden_garbage():
    """No keys: zeros.  No visible key: the mean.  Masked keys and keys behind the length hold NaN and infinities: no part of any result."""
    for n in (40, 700, 1500):
        E, G, H = 5, 2, 3
        cache = make_cache(E, H, n, n)
        q = rnd(E * G, H * 64, seed=1)
        klen = torch.tensor([0, n, n, 7, -4], dtype=torch.int32, device=DEV)
        mask = torch.ones(E, n, dtype=torch.uint8, device=DEV)
        mask[2] = 0
        mask[1, 5:n - 2] = 0
        clean = attend(q, cache, n, group=G, klen=klen, key_mask=mask)
        want, tol = attn_ref(q, *cache, 1.0, G, klen, mask, None)
        assert ((clean.double() - want).abs() <= tol).all()
        assert (clean[:G] == 0).all() and (clean[4 * G:] == 0).all()
        for t, bad in ((cache[1], math.nan), (cache[3], math.inf), (cache[3], math.nan)):
            t[1, :, 5:n - 2] = bad
            t[3, :, 7:] = bad
        assert torch.equal(attend(q, cache, n, group=G, klen=klen, key_mask=mask), clean)
        cache[3][1, :, 0] = math.nan         # a visible NaN is not hidden
        assert torch.isnan(attend(q, cache, n, group=G, klen=klen, key_mask=mask)[G:2 * G]).all()
        everywhere = torch.full((H, n), -math.inf, device=DEV)
        fresh = make_cache(E, H, n, n)
        o = attend(q, fresh, n, group=G, bias_row=everywhere)
        want, tol = attn_ref(q, *fresh, 1.0, G, None, None, everywhere)
        assert ((o.double() - want).abs() <= tol).all()


def test_operands_whose_storage_is_too_small_are_refused():
    cache = make_cache(2, 1, 1300, 1)
    q = rnd(2, 64, seed=1)
    o = torch.empty_like(q)
    with pytest.raises(ValueError, match="storage"):                  # 264 elements over 66 of storage
        L.decode_attn_q8(q, *cache, o, 1300, workspace=torch.empty(1, 66, device=DEV).expand(4, 66))
    with pytest.raises(ValueError, match="contiguous"):
        L.decode_attn_q8(q, *cache, o, 1200, klen=torch.tensor([5], dtype=torch.int32, device=DEV).expand(2))
    with pytest.raises(ValueError, match="storage"):
        L.kv_append_q8(q[:, None], q[:, None], *cache, 1, pos=torch.zeros(1, dtype=torch.int32, device=DEV))
    a, s = codes(4, 64, 1)
    with pytest.raises(ValueError, match="storage"):
        L.gemm_q8(a, a, s, s, torch.empty(4, 6, dtype=BF, device=DEV), 4, 4, 64, ldc=8)      # 3 * 8 + 4 = 28 over 24
    with pytest.raises(RuntimeError, match="dtype"):
        L.dequant_q8(a.view(torch.uint8), s, torch.empty(4, 64, dtype=BF, device=DEV), 4, 64)


def test_decode_attn_q8_large_and_lowest_scores():
    """Scores far apart and biases at the type's lowest value: weights of exactly zero and one."""
    E, H, n = 2, 2, 600
    cache = make_cache(E, H, n, 4)
    q = rnd(E, H * 64, seed=2, scale=60.0)
    bias = torch.full((H, n), torch.finfo(torch.float32).min, device=DEV)
    bias[:, 77] = 0
    bias[1, 590] = 3e38
    o = attend(q, cache, n, bias_row=bias)
    want = torch.stack([cache[2][e, h, j].double() * cache[3][e, h, j].double() for e in range(E) for h, j in ((0, 77), (1, 590))]).view(E, H * 64)
    assert ((o.double() - want).abs() <= want.abs() * (UBF + 4 * U32)).all()


def test_decode_attn_q8_counter_bias_and_batch_independence():
    """pos_dev: *pos_dev + 1 keys and the bias row of that position; a sequence alone gives the bits it gives in a batch."""
    E, H, n = 6, 4, 1400
    cache = make_cache(E, H, n, 6)
    q = rnd(E, H * 64, seed=5)
    diag = rnd(H, 2 * n - 1, seed=7, dtype=torch.float32)
    ctr = torch.zeros(1, dtype=torch.int32, device=DEV)
    for t in (0, 1, 511, 512, 1279, 1280, 1399):
        ctr.fill_(t)
        o = attend(q, cache, n, pos_dev=ctr, bias_row=diag, bias_maxlen=n)
        row = diag[:, n - 1 - t:2 * n - 1 - t].contiguous()
        want, tol = attn_ref(q, *cache, 1.0, 1, torch.full((E,), t + 1), None, row)
        assert ((o.double() - want).abs() <= tol).all()
        alone = attend(q[2:3], [c[2:3] for c in cache], n, pos_dev=ctr, bias_row=diag, bias_maxlen=n)
        assert torch.equal(alone, o[2:3])


def test_decode_attn_q8_counter_behind_the_range():
    """A counter that ran past the keys: all of them, and the last position's bias row at most; a negative one: no keys."""
    E, G, H, n, top = 3, 2, 2, 90, 100
    cache = make_cache(E, H, n, 6)
    diag = rnd(H, 2 * top - 1, seed=7, dtype=torch.float32)
    for G in (1, 2):
        q = rnd(E * G, H * 64, seed=5)
        for t in (95, 99, 100, 5000, 2**31 - 2, -1, -7):
            o = attend(q, cache, n, group=G, pos_dev=torch.tensor([t], dtype=torch.int32, device=DEV), bias_row=diag, bias_maxlen=top)
            if t < 0:
                assert (o == 0).all()
                continue
            row = diag[:, top - 1 - min(t, top - 1):][:, :n].contiguous()
            want, tol = attn_ref(q, *cache, 1.0, G, None, None, row)
            assert ((o.double() - want).abs() <= tol).all()


def test_decode_attn_q8_cache_views_behind_2_31_bytes():
    """A long cache whose later entries start behind 2^31 codes, as views of a larger one."""
    E, H, n = 3, 1, 12_000_000
    kq = torch.zeros(E, H, n, 64, dtype=torch.int8, device=DEV)
    ks = torch.ones(E, H, n, device=DEV)
    at = 11_999_000
    small = make_cache(1, 1, 900, 3)
    kq[2, 0, at:at + 900] = small[0][0, 0]
    ks[2, 0, at:at + 900] = small[1][0, 0]
    view = [kq[2:, :, at:at + 900], ks[2:, :, at:at + 900]]
    q = rnd(1, 64, seed=1)
    assert torch.equal(attend(q, view + view, 900), attend(q, [small[0], small[1], small[0], small[1]], 900))
    k = rnd(E, 2, 64, seed=9)
    pos = torch.full((E,), n - 2, dtype=torch.int32, device=DEV)
    L.kv_append_q8(k, k, kq, ks, kq, ks, 2, pos=pos)
    back = torch.empty(E, 2, 64, dtype=BF, device=DEV)
    L.kv_read_q8(kq, ks, kq, ks, back, back.clone(), 2, pos=pos)
    assert ((back.float() - k.float()).abs() <= k.float().abs().amax(2, keepdim=True) * (0.51 / 127 + UBF)).all()


# --------------------------------------------------------------------------------------------- sampling
def sample_ref(z, u, T, top_k, top_p, min_p):
    """(token, log-probability, distance of the draw to the nearest decision) of one row in 64 bits"""
    z = z.double()
    V = z.numel()
    top = z.max()
    w = torch.exp(torch.where(z == top, torch.zeros_like(z), (z - top) / T))
    order = torch.sort(z, descending=True, stable=True).indices
    ws = w[order].clone()
    if top_k:
        ws[top_k:] = 0
    run = ws.cumsum(0)
    pre = torch.cat([run.new_zeros(1), run[:-1]])
    keep = (ws > 0) & (pre < top_p * run[-1]) & (ws >= min_p)
    near = 1.0
    if top_p < 1:
        near = float(((pre[1:] - top_p * run[-1]).abs() / run[-1])[ws[1:] > 0].min()) if V > 1 else 1.0
    kept = torch.zeros_like(w)
    kept[order[keep]] = w[order[keep]]
    run = kept.cumsum(0)
    past = run > u * run[-1]
    tok = int(past.nonzero()[0]) if past.any() else int(kept.nonzero()[-1])
    near = min(near, float((run / run[-1] - u).abs().min()) if u > 0 else near)
    return tok, math.log(float(kept[tok] / run[-1])), near


def sample(z, u, **kw):
    rows, V = z.shape
    tok, lp = torch.full((rows,), -1, dtype=torch.long, device=DEV), torch.empty(rows, device=DEV)
    L.sample_step(z, rows, V, u, tok, logp=lp, **kw)
    return tok, lp


CASES = [dict(), dict(top_k=1), dict(top_k=50, top_p=0.95), dict(top_p=0.9), dict(min_p=0.05), dict(temperature=0.3, top_p=0.5, min_p=0.01), dict(temperature=3.0, top_k=700, top_p=0.7),
         dict(temperature=1e-3, top_k=5), dict(top_p=1e-9), dict(min_p=1.0)]


@pytest.mark.parametrize("V", [1, 2, 63, 300, 4096, 4097, 32228, 40001, 131072])
@pytest.mark.parametrize("kind", [torch.float32, BF])
def test_sample_step(V, kind):
    rows = 6
    z = rnd(rows, V, seed=V, scale=2.5, dtype=torch.float32).to(kind)
    z[1] = (z[1].float() * 4).round().to(kind) / 4                    # many equal logits
    if V > 8:
        z[2, 3:7] = -math.inf
        z[3] = 1.0                                                    # one plateau
        z[4] = -math.inf
    g = torch.Generator().manual_seed(V)
    u = torch.rand(rows, generator=g).to(DEV)
    u[5] = 0.0
    for kw in CASES:
        tok, lp = sample(z, u, **kw)
        for r in range(rows):
            want, wlp, near = sample_ref(z[r].cpu(), float(u[r]), kw.get("temperature", 1.0), kw.get("top_k", 0), kw.get("top_p", 1.0), kw.get("min_p", 0.0))
            # weights are rounded to 2^-47 each: decisions nearer than V 2^-47 to a border may fall on the other side
            if near > V * 2.0 ** -46:
                assert int(tok[r]) == want, (kw, r, near)
                assert abs(float(lp[r]) - wlp) <= 4 * U32 * max(1.0, abs(wlp)) + V * 2.0 ** -46


def test_sample_step_infinities_nan_and_extreme_numbers():
    V = 5000
    z = rnd(7, V, seed=1, dtype=torch.float32)
    z[0, [40, 4000]] = math.inf
    z[1, [77, 3000]] = math.nan
    z[2] = -math.inf
    z[3, 1:] = -math.inf
    z[4] = torch.where(torch.arange(V, device=DEV) % 2 == 0, 0.0, -0.0)      # equal, whatever their sign
    u = torch.tensor([0.6, 0.5, 0.5, 0.999, 0.5, 1.0, math.nan], device=DEV)
    tok, lp = sample(z, u)
    assert tok[:5].tolist() == [4000, 77, 2500, 0, 2500]
    assert abs(float(lp[0]) - math.log(0.5)) < 1e-6 and math.isnan(float(lp[1])) and abs(float(lp[2]) + math.log(V)) < 1e-5 and float(lp[3]) == 0.0
    assert int(tok[5]) == V - 1 and int(tok[6]) == 0                  # from 1 on the last kept token, NaN counts as 0
    tok, _ = sample(z, torch.tensor([0.6] * 7, device=DEV), top_k=3)
    assert int(tok[4]) == 1 and int(tok[2]) == 1                      # ties: the lowest indexes


def test_sample_step_loop_arguments():
    """The captured loop's form: a table of numbers, the step counter, finished rows, the minimum length, the sequence column."""
    rows, V, steps, eos = 5, 700, 4, 9
    z = torch.full((rows, V + 4), -20.0, device=DEV)
    z[:, eos] = 5.0
    z[:, 30] = 0.0
    table = torch.full((steps, rows + 3), 0.5, device=DEV)
    un = torch.tensor([1, 0, 1, 1, 1], dtype=torch.int32, device=DEV)
    seq = torch.full((rows, steps + 1), -1, dtype=torch.long, device=DEV)
    pos = torch.zeros(1, dtype=torch.int32, device=DEV)
    tok, lp = torch.empty(rows, dtype=torch.long, device=DEV), torch.empty(rows, device=DEV)
    kw = dict(ld=V + 4, logp=lp, unfinished=un, eos_id=eos, pad_id=3, seq_out=seq, seq_ld=steps + 1, pos_dev=pos, min_length=2)
    L.sample_step(z, rows, V, table, tok, **kw)
    assert tok.tolist() == [30, 3, 30, 30, 30] and un.tolist() == [1, 0, 1, 1, 1] and seq[:, 1].tolist() == tok.tolist() and float(lp[1]) == 0.0
    pos.fill_(1)
    L.sample_step(z, rows, V, table, tok, **kw)
    assert tok.tolist() == [9, 3, 9, 9, 9] and un.tolist() == [0] * 5
    pos.fill_(7)                                                      # behind the table and the sequence: the last numbers, no column
    before = seq.clone()
    L.sample_step(z, rows, V, table, tok, **kw)
    assert torch.equal(seq, before) and tok.tolist() == [3] * 5


def test_sample_step_frequencies():
    """10000 draws follow the distribution: each frequency within five standard deviations."""
    n, V = 10000, 12
    z = rnd(1, V, seed=3, dtype=torch.float32).expand(n, V).contiguous()
    g = torch.Generator().manual_seed(0)
    tok, _ = sample(z, torch.rand(n, generator=g).to(DEV), temperature=0.7)
    p = torch.softmax(z[0].double() / 0.7, 0)
    f = torch.bincount(tok, minlength=V).double() / n
    assert ((f - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all()


# --------------------------------------------------------------------------------------------- the operators together
class Block:
    """One decoder layer and a head over an int8 cache, as a serving loop strings the operators together; every intermediate stays readable."""

    def __init__(self, B, H, ffn, V, maxlen, steps):
        d = self.d = H * 64
        self.B, self.H, self.ffn, self.V, self.n = B, H, ffn, V, maxlen
        self.w = {}
        for i, (name, rows, cols) in enumerate((("qkv", 3 * d, d), ("out", d, d), ("up", ffn, d), ("down", d, ffn), ("head", V, d))):
            wq, ws = torch.empty(rows, cols, dtype=torch.int8, device=DEV), torch.empty(rows, device=DEV)
            L.quant_rows_q8(rnd(rows, cols, seed=20 + i, scale=cols ** -0.5, dtype=torch.float32), wq, ws, rows, cols)
            self.w[name] = (wq, ws)
        self.emb, self.g = rnd(V, d, seed=30), [1 + 0.1 * rnd(d, seed=31 + i, dtype=torch.float32) for i in range(3)]
        self.bias = rnd(H, 2 * maxlen - 1, seed=40, dtype=torch.float32)
        self.kv = new_cache(B, H, maxlen)
        new = lambda *s, t=BF: torch.zeros(*s, dtype=t, device=DEV)  # noqa: E731
        self.x, self.h1, self.h2, self.h3, self.qkv, self.o, self.up, self.logits = (new(B, d), new(B, d), new(B, d), new(B, d), new(B, 3 * d), new(B, d), new(B, ffn),
                                                                                   new(B, (V + 7) // 8 * 8, t=torch.float32))
        self.a, self.f = new(B, d), new(B, d)
        self.codes = [(new(B, c, t=torch.int8), new(B, t=torch.float32)) for c in (d, d, d, ffn, d)]
        self.tok, self.lp, self.un = new(B, t=torch.long), new(B, t=torch.float32), torch.ones(B, dtype=torch.int32, device=DEV)
        self.seq, self.pos = new(B, maxlen + 1, t=torch.long), new(1, t=torch.int32)
        self.u = torch.rand(steps, B, generator=torch.Generator().manual_seed(3)).to(DEV)
        self.ws = L.decode_attn_q8_workspace(B, H, maxlen, DEV)
        self.ctr = new(1, t=torch.int32)

    def product(self, i, name, out, N, K, **kw):
        L.gemm_q8(self.codes[i][0], self.w[name][0], self.codes[i][1], self.w[name][1], out, self.B, N, K, **kw)

    def prefill(self, T):
        kv = rnd(self.B, T, 2 * self.d, seed=50)
        L.kv_append_q8(kv[:, :, :self.d], kv[:, :, self.d:], *self.kv, T)
        self.pos.fill_(T)
        self.ctr.zero_()
        self.tok.copy_(torch.arange(self.B, device=DEV))

    def step(self):
        B, d, c = self.B, self.d, self.codes
        self.x.copy_(self.emb[self.tok])
        L.rmsnorm_q8(self.x, self.g[0], *c[0], B, d, 1e-6, h=None)
        self.product(0, "qkv", self.qkv, 3 * d, d)
        q, k, v = self.qkv[:, :d], self.qkv[:, None, d:2 * d], self.qkv[:, None, 2 * d:]
        L.kv_append_q8(k, v, *self.kv, 1, pos_dev=self.pos)
        L.decode_attn_q8(q, *self.kv, self.o, self.n, pos_dev=self.pos, bias_row=self.bias, bias_maxlen=self.n, workspace=self.ws)
        L.quant_rows_q8(self.o, *c[1], B, d)
        self.product(1, "out", self.a, d, d)
        L.rmsnorm_q8(self.x, self.g[1], *c[2], B, d, 1e-6, delta=self.a, h=self.h1)
        self.product(2, "up", self.up, self.ffn, d, act=L.ACT_RELU)
        L.quant_rows_q8(self.up, *c[3], B, self.ffn)
        self.product(3, "down", self.h2, d, self.ffn, residual=self.h1)
        L.rmsnorm_q8(self.h2, self.g[2], *c[4], B, d, 1e-6)
        self.product(4, "head", self.logits, self.V, d, ldc=self.logits.shape[1])
        L.sample_step(self.logits, B, self.V, self.u, self.tok, ld=self.logits.shape[1], temperature=0.8, top_k=40, top_p=0.95, logp=self.lp, unfinished=self.un,
                      seq_out=self.seq, seq_ld=self.n + 1, pos_dev=self.ctr)
        self.pos.add_(1)
        self.ctr.add_(1)

    def state(self):
        return [t.clone() for t in (*self.kv, self.o, self.h1, self.h2, self.logits, self.tok, self.lp, self.seq)]


def test_operators_together_match_their_formulas():
    """Every value of two steps from the values in front of it; the second step reads what the first wrote into the cache."""
    b = Block(3, 2, 200 // 8 * 16, 500, 1500, 2)
    b.prefill(1395)
    for _ in range(2):
        pos = int(b.pos)
        b.step()
        norm = lambda x, g: x.double() * torch.rsqrt((x.double() ** 2).mean(1, keepdim=True) + 1e-6) * g.double()  # noqa: E731
        d, slack = b.d, (b.d / 64 + 14) * U32
        check_codes(*b.codes[0], norm(b.x, b.g[0]), slack)
        for i, name, got, r in ((0, "qkv", b.qkv, None), (1, "out", b.a, None), (3, "down", b.h2, b.h1), (4, "head", b.logits[:, :b.V], None)):
            want, mag = product_ref(b.codes[i][0], b.w[name][0], b.codes[i][1], b.w[name][1], 1.0, None, L.ACT_NONE, r)
            assert ((got.double() - want).abs() <= mag * 7 * U32 + want.abs() * (UBF if name != "head" else 0)).all(), name
        k = b.qkv[:, d:2 * d].double().reshape(-1, 64)
        check_codes(b.kv[0][:, :, pos].reshape(-1, 64), b.kv[1][:, :, pos].reshape(-1), k, 0.0)
        row = b.bias[:, b.n - 1 - pos:2 * b.n - 1 - pos].contiguous()
        want, tol = attn_ref(b.qkv[:, :d], *b.kv, 1.0, 1, torch.full((b.B,), pos + 1), None, row)
        assert ((b.o.double() - want).abs() <= tol).all()
        check_codes(*b.codes[1], b.o.double(), 0.0)
        s = b.x.double() + b.a.double()
        assert ((b.h1.double() - s).abs() <= s.abs() * (UBF + U32)).all()
        check_codes(*b.codes[2], norm(b.h1, b.g[1]), slack)
        check_codes(*b.codes[4], norm(b.h2, b.g[2]), slack)
        for r in range(b.B):
            tok, lp, near = sample_ref(b.logits[r, :b.V].cpu(), float(b.u[int(b.ctr) - 1, r]), 0.8, 40, 0.95, 0.0)
            if near > b.V * 2.0 ** -46:
                assert int(b.tok[r]) == tok == int(b.seq[r, int(b.ctr)]) and abs(float(b.lp[r]) - lp) <= 4 * U32 * max(1.0, abs(lp)) + b.V * 2.0 ** -46


def test_operators_together_captured_and_replayed():
    """Two loops, each captured once and replayed in turn with eager work between the replays, give the bits of the eager loop."""
    steps = 6
    eager = Block(3, 2, 416, 500, 1500, steps)
    eager.prefill(1390)
    eager.step()                                                      # loads every kernel before the capture
    blocks = [Block(3, 2, 416, 500, 1500, steps) for _ in range(2)]
    graphs = []
    for b in blocks:
        b.prefill(1390)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            b.step()
        graphs.append(graph)
        b.prefill(1390)
    for i in range(steps):
        if i:
            eager.step()
        for graph, b in zip(graphs, blocks):
            graph.replay()
            torch.cuda.synchronize()
            scratch = torch.randn(1000, device=DEV).sum().item()      # eager work between the replays
            assert math.isfinite(scratch)
            for x, y in zip(b.state(), eager.state()):
                assert torch.equal(x, y), i


def test_operators_on_a_side_stream():
    """The launches go to the current stream: a loop on a stream of its own, behind that stream's work, gives the same bits."""
    a, b = Block(2, 2, 128, 300, 1400, 2), Block(2, 2, 128, 300, 1400, 2)
    a.prefill(1380)
    a.step()
    a.step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        big = torch.randn(2048, 2048, device=DEV)
        for _ in range(20):
            big = big @ big * 0.01                                    # the stream is busy when the loop is enqueued
        b.prefill(1380)
        b.step()
        b.step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for x, y in zip(b.state(), a.state()):
        assert torch.equal(x, y)
