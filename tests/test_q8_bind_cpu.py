"""The native argument module and the library have to come from one header: attach() compares the version and the sizes of the structs it fills."""
import ctypes

import pytest
import torch

from vidchapters_amd import lib as L

VERSION, SIZEOF = ctypes.CFUNCTYPE(ctypes.c_int), ctypes.CFUNCTYPE(ctypes.c_int64, ctypes.c_char_p)
NAMES = ("quant_rows_q8", "rmsnorm_q8", "dequant_q8", "gemm_q8", "kv_append_q8", "kv_read_q8", "decode_attn_q8", "sample_step")


def attach(version, sizeof):
    """attach() with these two functions in the library's place; callbacks live as long as the call"""
    address = lambda f: ctypes.cast(f, ctypes.c_void_p).value      # noqa: E731
    v, s = VERSION(version), SIZEOF(sizeof)
    return L._bind().attach(torch.cuda.current_device, lambda dev: 0, address(v), address(s), *(address(getattr(L.lib(), "v2s_" + n)) for n in NAMES))


def size_of(name):
    return L.lib().v2s_sizeof(name)


@pytest.mark.parametrize("version", [0, L.ABI_VERSION - 1, L.ABI_VERSION + 1])
def test_another_version_is_refused(version):
    with pytest.raises(RuntimeError, match=f"V2S_ABI_VERSION {version}"):
        attach(lambda: version, size_of)


@pytest.mark.parametrize("name", [b"v2s_gemm_q8_args", b"v2s_kv_q8", b"v2s_decode_attn_q8_args"])
@pytest.mark.parametrize("off", [-8, 8])
def test_a_struct_of_another_size_is_refused(name, off):
    with pytest.raises(RuntimeError, match=name.decode()):
        attach(lambda: L.ABI_VERSION, lambda n: size_of(n) + (off if n == name else 0))


def test_a_refused_library_leaves_the_attached_one_in_place():
    with pytest.raises(RuntimeError):
        attach(lambda: 0, size_of)
    with pytest.raises(RuntimeError, match="GPU"):
        L.quant_rows_q8(torch.zeros(2, 64), torch.zeros(2, 64, dtype=torch.int8), torch.zeros(2), 2, 64)


def test_missing_addresses_are_refused():
    with pytest.raises(TypeError):
        L._bind().attach(None, None)
    with pytest.raises(ValueError, match="NULL"):
        L._bind().attach(None, None, *([0] * 10))
