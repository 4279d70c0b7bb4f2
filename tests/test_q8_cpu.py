"""Refusals of the 8-bit decoding entry points: every check happens on the host before a launch, so these run without a GPU (the pointers are never
followed)."""
import ctypes

import pytest
import torch

from vidchapters_amd import lib as L

P = 1 << 20              # a plausible, 16-byte aligned address


# the addresses below stand for nothing: a call that is not refused must not find a device to be launched on
pytestmark = pytest.mark.skipif(torch.cuda.device_count() > 0, reason="refusals are checked where nothing can be launched")


def refused(rc, word):
    assert rc < 0
    msg = L.lib().v2s_last_error().decode()
    assert word in msg, msg


def test_rows_refusals():
    l = L.lib()
    ok = dict(x=P, dt=0, ldx=64, q=P, ldq=64, s=P, rows=4, cols=64)
    for change, word in ((dict(x=None), "NULL"), (dict(s=None), "NULL"), (dict(dt=7), "bf16 or fp32"), (dict(cols=60), "multiple of 8"), (dict(cols=8200, ldx=8200, ldq=8200), "8192"),
                         (dict(rows=0), "rows=0"), (dict(rows=1 << 24), "2^24"), (dict(ldx=56), "shorter"), (dict(ldq=63), "shorter"), (dict(ldx=68), "multiples of 8"), (dict(x=P + 2), "aligned"),
                         (dict(q=P + 4), "aligned")):
        a = {**ok, **change}
        refused(l.v2s_quant_rows_q8(a["x"], a["dt"], a["ldx"], a["q"], a["ldq"], a["s"], a["rows"], a["cols"], None), word)
    ok = dict(x=P, ldx=64, d=P, ldd=64, w=P, h=P, ldh=64, q=P, ldq=64, s=P, rows=4, cols=64, eps=1e-6)
    for change, word in ((dict(w=None), "NULL"), (dict(d=None), "needs delta"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(cols=12), "multiple of 8"),
                         (dict(ldd=8), "shorter"), (dict(ldh=60), "shorter"), (dict(ldh=76), "multiples"), (dict(d=P + 8), "aligned"), (dict(w=P + 4), "aligned"), (dict(rows=-1), "rows")):
        a = {**ok, **change}
        refused(l.v2s_rmsnorm_q8(a["x"], a["ldx"], a["d"], a["ldd"], a["w"], a["h"], a["ldh"], a["q"], a["ldq"], a["s"], a["rows"], a["cols"], a["eps"], None), word)
    refused(l.v2s_dequant_q8(P, 64, P, P, 60, 4, 64, None), "shorter")
    refused(l.v2s_dequant_q8(P, 64, P, P + 8, 64, 4, 64, None), "aligned")
    refused(l.v2s_dequant_q8(P, 64, None, P, 64, 4, 64, None), "NULL")


def test_gemm_refusals():
    def call(**kw):
        a = L.GemmQ8Args(M=4, N=8, K=64, A=P, B=P, lda=64, ldb=64, sA=P, sB=P, C=P, ldc=8, c_dtype=0, alpha=1.0, ldr=8)
        for k, v in kw.items():
            setattr(a, k, v)
        return L.lib().v2s_gemm_q8(ctypes.byref(a), None)
    for kw, word in ((dict(A=None), "NULL"), (dict(sB=None), "NULL"), (dict(M=0), "M=0"), (dict(K=72, lda=80, ldb=80), "multiple of 16"), (dict(K=131072, lda=131072, ldb=131072), "131056"),
                     (dict(lda=48), "shorter"), (dict(ldc=4), "shorter"), (dict(residual=P, ldr=0), "shorter"), (dict(c_dtype=5), "bf16 or fp32"), (dict(act=9), "activation"),
                     (dict(lda=72), "multiples of 16"), (dict(ldc=12), "multiples of 8"), (dict(C=P + 8), "aligned"), (dict(residual=P + 2), "aligned"), (dict(bias=P + 1), "aligned")):
        refused(call(**kw), word)
    assert L.lib().v2s_gemm_q8(None, None) < 0


def cache(**kw):
    c = L.KvQ8(k=P, ks=P, v=P, vs=P, e_rows=80, h_rows=40, entries=3, heads=2, maxlen=40)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def test_cache_refusals():
    for fn in (L.lib().v2s_kv_append_q8, L.lib().v2s_kv_read_q8):
        def call(c=None, k=P, bs=256, rs=128, T=2):
            return fn(ctypes.byref(c if c is not None else cache()), k, P, bs, rs, T, 0, None, None, None, None)
        for kw, word in ((dict(c=cache(ks=None)), "NULL"), (dict(k=None), "NULL"), (dict(T=0), "positive"), (dict(c=cache(maxlen=0)), "positive"), (dict(c=cache(h_rows=39)), "row strides"),
                         (dict(k=P + 8), "aligned"), (dict(rs=130), "multiples of 8"), (dict(c=cache(k=P + 8)), "aligned"), (dict(c=cache(entries=1 << 20, heads=1024), T=64), "too large"), (dict(c=cache(entries=1 << 16, heads=1024), T=8), "too large")):
            refused(call(**kw), word)
        assert fn(None, P, P, 8, 8, 1, 0, None, None, None, None) < 0


def test_attention_refusals():
    def call(**kw):
        a = L.DecodeAttnQ8Args(B=3, Nk=40, group=1, q=P, q_bs=128, cache=cache(), o=P, o_bs=128, scale=1.0)
        for k, v in kw.items():
            setattr(a, k, v)
        return L.lib().v2s_decode_attn_q8(ctypes.byref(a), None)
    for kw, word in ((dict(q=None), "NULL"), (dict(cache=cache(v=None)), "NULL"), (dict(B=4), "query rows"), (dict(B=3, group=2), "query rows"), (dict(Nk=41), "maxlen"), (dict(Nk=0), "positive"),
                     (dict(klen=P, pos_dev=P), "exclude"), (dict(bias_row=P, bias_ld=39), "bias"), (dict(bias_row=P, bias_ld=78, pos_dev=P, bias_maxlen=40), "bias"),
                     (dict(bias_row=P, bias_ld=200, pos_dev=P, bias_maxlen=39), "bias"), (dict(key_mask=P, mask_ld=39), "mask_ld"), (dict(q_bs=120), "shorter"), (dict(q_bs=132), "multiple of 8"),
                     (dict(q=P + 8), "aligned"), (dict(B=1 << 24, cache=cache(entries=1 << 24)), "too many")):
        refused(call(**kw), word)
    long = dict(cache=cache(e_rows=4000, h_rows=2000, maxlen=2000), Nk=2000)
    need = L.lib().v2s_decode_attn_q8_workspace_floats(3, 2, 2000)
    assert need > 0 and L.lib().v2s_decode_attn_q8_workspace_floats(3, 2, 40) == 0
    refused(call(**long), "workspace")
    refused(call(**long, workspace=P, workspace_bytes=need * 4 - 1), "workspace")


def test_sample_refusals():
    ok = dict(z=P, dt=1, ld=100, rows=2, V=100, T=1.0, k=0, p=1.0, m=0.0, u=P, u_ld=0, us=0, tok=P, seq=None, pos=None)
    nan = float("nan")
    for change, word in ((dict(z=None), "NULL"), (dict(u=None), "NULL"), (dict(dt=3), "fp32 or bf16"), (dict(V=0), "V=0"), (dict(V=200), "ld >= V"), (dict(V=131073, ld=140000), "131072"),
                         (dict(T=0.0), "temperature"), (dict(T=nan), "temperature"), (dict(k=-1), "top_k"), (dict(p=0.0), "top_p"), (dict(p=1.5), "top_p"), (dict(p=nan), "top_p"),
                         (dict(m=-0.1), "min_p"), (dict(m=1.1), "min_p"), (dict(seq=P), "pos_dev"), (dict(pos=P), "u_steps"), (dict(pos=P, u_ld=1, us=4), "u_ld"), (dict(rows=0), "rows=0"), (dict(rows=1 << 22, ld=100), "2^22")):
        a = {**ok, **change}
        refused(L.lib().v2s_sample_step(a["z"], a["dt"], a["ld"], a["rows"], a["V"], a["T"], a["k"], a["p"], a["m"], a["u"], a["u_ld"], a["us"], a["tok"], None, None, -1, 0,
                                        a["seq"], 5, a["pos"], 0, None), word)


def test_struct_sizes_match_the_binding():
    for name, t in (("v2s_gemm_q8_args", L.GemmQ8Args), ("v2s_kv_q8", L.KvQ8), ("v2s_decode_attn_q8_args", L.DecodeAttnQ8Args)):
        assert L.lib().v2s_sizeof(name.encode()) == ctypes.sizeof(t)


def test_wrappers_refuse_what_is_no_tensor_and_numbers_that_do_not_fit():
    q, s = torch.empty(4, 64, dtype=torch.int8), torch.empty(4)
    with pytest.raises(TypeError, match="tensor"):
        L.dequant_q8(q.numpy(), s, q, 4, 64)
    with pytest.raises(TypeError, match="tensor"):
        L.gemm_q8(q, q, s, s, None, 4, 4, 64)
    with pytest.raises(ValueError, match="32 bits"):
        L.dequant_q8(q, s, q, 1 << 40, 64)
    with pytest.raises(ValueError, match="32 bits"):
        L.dequant_q8(q, s, q, 4, 64, ldq=1 << 62)
    with pytest.raises(TypeError):
        L.quant_rows_q8(s, q, s, 4.0, 64)
    with pytest.raises(TypeError, match="arguments"):
        L._bind().gemm_q8(q)
    kq, ks = torch.empty(2, 3, 10, 64, dtype=torch.int8), torch.empty(2, 3, 10)
    for bad in (torch.empty(2, 10, 192), torch.empty(2, 1, 191), torch.empty(1, 2, 192), torch.empty(2, 192)):
        with pytest.raises(ValueError, match="k and v are"):
            L.kv_append_q8(bad, torch.empty(2, 2, 192), kq, ks, kq, ks, 2)
    with pytest.raises(ValueError, match="q and o are"):
        L.decode_attn_q8(torch.empty(2, 190), kq, ks, kq, ks, torch.empty(2, 190), 10)


def test_wrappers_refuse_tensors_that_are_not_on_the_gpu_and_wrong_shapes():
    q, s = torch.empty(4, 64, dtype=torch.int8), torch.empty(4)
    with pytest.raises(RuntimeError, match="GPU"):
        L.quant_rows_q8(torch.empty(4, 64, dtype=torch.bfloat16), q, s, 4, 64)
    kq, ks = torch.empty(2, 3, 10, 64, dtype=torch.int8), torch.empty(2, 3, 10)
    with pytest.raises(ValueError, match="cache"):
        L.kv_read_q8(kq, ks[:, :, :9], kq, ks, None, None, 1)
    with pytest.raises(ValueError, match="share"):
        L.kv_read_q8(kq, ks, kq.transpose(0, 1).contiguous().transpose(0, 1), ks, None, None, 1)
    with pytest.raises(ValueError, match=r"u is \[rows\]"):
        L.sample_step(torch.empty(4, 100), 4, 100, torch.empty(3), torch.empty(4, dtype=torch.long))
