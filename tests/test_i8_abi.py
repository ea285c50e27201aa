"""The 8-bit path's entry points without a device: NULL arguments, descriptors' layout, sample_params."""
import ctypes as C

import numpy as np

import hayai_amd
from hayai_amd import _abi


def test_null_arguments_rejected():
    lib = _abi.load()
    for name, desc, pairs in [("hh_quant_i8_dev", _abi.QuantI8Desc(), 5), ("hh_rms_norm_i8_dev", _abi.RmsNormI8Desc(), 7),
                              ("hh_gemm_i8_dev", _abi.GemmI8Desc(), 6), ("hh_sample_dev", _abi.SampleDesc(), 5)]:
        assert getattr(lib, name)(None, C.byref(desc), *[None, 0] * pairs) == 2
        assert b"engine is NULL" in lib.hh_last_error()
    out = C.c_void_p()
    assert lib.hh_buf_wrap(None, None, 16, C.byref(out)) == 2


def test_descriptors_match_the_header():
    # x86-64 layout of the header's structs
    assert C.sizeof(_abi.QuantI8Desc) == 48 and _abi.QuantI8Desc.q_stride.offset == 40
    assert C.sizeof(_abi.RmsNormI8Desc) == 56 and _abi.RmsNormI8Desc.eps.offset == 4
    assert C.sizeof(_abi.GemmI8Desc) == 64 and _abi.GemmI8Desc.y_stride.offset == 56
    assert C.sizeof(_abi.SampleParams) == 16 and C.sizeof(_abi.SampleDesc) == 32


def test_sample_params_table():
    p = hayai_amd.HipEngine.sample_params(0.5, [1, 2, 3], 0.9)
    assert p.shape == (3,) and p.itemsize == 16 and p["top_k"].tolist() == [1, 2, 3]
    assert np.all(p["temperature"] == np.float32(0.5)) and np.all(p["min_p"] == 0)
    assert hayai_amd.HipEngine.sample_params(rows=4).shape == (4,)
    assert hayai_amd.HipEngine.sample_params().tobytes() == np.array([(1.0, 0, 1.0, 0.0)], p.dtype).tobytes()


def test_engine_stream_rejects_null():
    lib = _abi.load()
    out = C.c_void_p(1)
    assert lib.hh_engine_stream(None, C.byref(out)) == 2 and b"engine is NULL" in lib.hh_last_error()
    assert out.value is None
    assert lib.hh_engine_stream(None, None) == 2
