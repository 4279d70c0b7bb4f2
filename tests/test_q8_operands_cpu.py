"""Operands of the 8-bit decoding calls that do not lie as the call would read them are refused: this is looked at before the device, so it runs without a GPU.
Where a layout is fine, the call gets as far as the refusal of tensors on the CPU."""
import pytest
import torch

from vidchapters_amd import lib as L

BF = torch.bfloat16
refused = lambda: pytest.raises(ValueError, match="expected")       # noqa: E731
passes = lambda: pytest.raises(RuntimeError, match="GPU")           # noqa: E731


def operands(M=6, N=16, K=32):
    i8 = lambda *s: torch.zeros(*s, dtype=torch.int8)               # noqa: E731
    return dict(A=i8(M, K), B=i8(N, K), sA=torch.ones(M), sB=torch.ones(N), C_out=torch.zeros(M, N, dtype=BF), M=M, N=N, K=K)


@pytest.mark.parametrize("name,n", [("sA", 6), ("sB", 16), ("bias", 16)])
def test_vectors_cut_from_a_wider_tensor(name, n):
    a = operands()
    a[name] = torch.ones(n, 4)[:, 1:2]                              # [n, 1], four apart
    with refused():
        L.gemm_q8(**a)
    a[name] = torch.ones(n, 1)                                      # [n, 1], one behind the other
    with passes():
        L.gemm_q8(**a)
    a[name] = torch.ones(3, n + 4)[1:2, :n]                         # a row of a wider tensor
    with passes():
        L.gemm_q8(**a)


@pytest.mark.parametrize("name,rows,cols", [("A", 6, 32), ("B", 16, 32), ("C_out", 6, 16), ("residual", 6, 16)])
def test_rows_at_no_single_distance(name, rows, cols):
    dt = torch.int8 if name in "AB" else BF
    a = operands()
    a[name] = torch.zeros(2, rows // 2 + 1, cols + 16, dtype=dt)[:, :rows // 2, :cols]     # two batches, a gap between them
    with refused():
        L.gemm_q8(**a)
    a[name] = torch.zeros(rows, 2, cols, dtype=dt)[:, :, :cols // 2]                       # a row in two pieces
    with refused():
        L.gemm_q8(**a)
    for fine in (torch.zeros(rows, cols + 16, dtype=dt)[:, :cols], torch.zeros(2, rows // 2, cols + 16, dtype=dt)[..., :cols], torch.zeros(rows * cols, dtype=dt),
                 torch.zeros(rows + 3, cols + 48, dtype=dt), torch.zeros(rows, 2, cols, dtype=dt)[:, 1]):
        a[name] = fine
        with passes():
            L.gemm_q8(**a)


def test_a_single_row_in_pieces():
    q, s = torch.zeros(1, 64, dtype=torch.int8), torch.ones(1)
    with refused():
        L.quant_rows_q8(torch.zeros(1, 4, 32, dtype=BF)[:, :, :16], q, s, 1, 64)
    with passes():
        L.quant_rows_q8(torch.zeros(3, 80, dtype=BF)[1, :64], q, s, 1, 64)


def test_vectors_of_the_other_calls():
    two = lambda n, dt=torch.float32: torch.zeros(n, 2, dtype=dt)[:, :1]          # noqa: E731
    i32, f32 = torch.int32, torch.float32
    x, q, s, w = torch.zeros(4, 64, dtype=BF), torch.zeros(4, 64, dtype=torch.int8), torch.ones(4), torch.ones(64)
    kq, ks, kv = torch.zeros(4, 2, 10, 64, dtype=torch.int8), torch.ones(4, 2, 10), torch.zeros(4, 1, 128, dtype=BF)
    qa, z, u, tok = torch.zeros(4, 128, dtype=BF), torch.zeros(4, 300), torch.zeros(4), torch.zeros(4, dtype=torch.long)
    calls = [(lambda scale=s: L.quant_rows_q8(x, q, scale, 4, 64), dict(scale=two(4))),
             (lambda scale=s: L.dequant_q8(q, scale, x, 4, 64), dict(scale=two(4))),
             (lambda w=w, scale=s: L.rmsnorm_q8(x, w, q, scale, 4, 64, 1e-6), dict(w=two(64), scale=two(4))),
             (lambda **k: L.kv_append_q8(kv, kv, kq, ks, kq, ks, 1, **k), dict(pos=two(4, i32), count=two(4, i32))),
             (lambda **k: L.kv_read_q8(kq, ks, kq, ks, kv, kv, 1, **k), dict(pos=two(4, i32), count=two(4, i32))),
             (lambda **k: L.decode_attn_q8(qa, kq, ks, kq, ks, qa, 10, **k), dict(klen=two(4, i32), workspace=two(4))),
             (lambda u=u, tok=tok, **k: L.sample_step(z, 4, 300, u, tok, **k), dict(tok=two(4, torch.long), logp=two(4), unfinished=two(4, i32)))]
    for call, strided in calls:
        with passes():
            call()
        for name, t in strided.items():
            with refused():
                call(**{name: t})
            with passes():
                call(**{name: t.contiguous()})


def test_sequences_without_a_row_length():
    z, u, tok, pos = torch.zeros(4, 300), torch.zeros(5, 4), torch.zeros(4, dtype=torch.long), torch.zeros(1, dtype=torch.int32)
    for bad in (torch.zeros(4 * 9, dtype=torch.long), torch.zeros(3, 9, dtype=torch.long), torch.zeros(4, 20, dtype=torch.long)[:, :9]):
        with refused():
            L.sample_step(z, 4, 300, u, tok, seq_out=bad, pos_dev=pos)
    for fine, ld in ((torch.zeros(4, 9, dtype=torch.long), None), (torch.zeros(4 * 9, dtype=torch.long), 9), (torch.zeros(4, 20, dtype=torch.long)[:, :9], 20)):
        with passes():
            L.sample_step(z, 4, 300, u, tok, seq_out=fine, seq_ld=ld, pos_dev=pos)
