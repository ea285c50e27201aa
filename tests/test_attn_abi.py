"""The attention entry points without a device: NULL arguments, descriptors' layout, frequency factors."""
import ctypes as C
import math

import numpy as np
import pytest

import hayai_amd
from hayai_amd import _abi


def test_null_arguments_rejected():
    lib = _abi.load()
    kv = _abi.KvDesc()
    assert lib.hh_rope_kv_dev(None, C.byref(_abi.RopeDesc()), C.byref(kv), *[None, 0] * 8) == 2
    assert b"engine is NULL" in lib.hh_last_error()
    assert lib.hh_kv_copy_dev(None, C.byref(kv), 1, 0, None, 0, None, 0, 0) == 2
    assert b"engine is NULL" in lib.hh_last_error()


def test_descriptors_match_the_header():
    # x86-64 layout of the header's structs
    assert C.sizeof(_abi.KvDesc) == 48 and _abi.KvDesc.page_stride.offset == 40
    assert C.sizeof(_abi.RopeDesc) == 80 and _abi.RopeDesc.base.offset == 32 and _abi.RopeDesc.q_stride.offset == 48


def test_rope_factors_linear():
    f, m = hayai_amd.rope_factors(hayai_amd.ROPE_LINEAR, 64, 10000.0, 4.0)
    assert f.shape == (32,) and np.all(f == 4.0) and m == 1.0


@pytest.mark.parametrize("rot,base,scale,trained", [(128, 500000.0, 8.0, 8192), (64, 10000.0, 2.5, 2048), (2, 10000.0, 4.0, 100)])
def test_rope_factors_by_wavelength(rot, base, scale, trained):
    f, m = hayai_amd.rope_factors(hayai_amd.ROPE_BY_WAVELENGTH, rot, base, scale, trained)
    assert m == 1.0
    for i in range(rot // 2):
        w = 2 * math.pi * base ** (2 * i / rot)
        if w < trained / 4:
            want = 1.0
        elif w > trained:
            want = scale
        else:
            s = (trained / w - 1) / 3
            want = 1 / ((1 - s) / scale + s)
        assert abs(f[i] - want) <= want * 2.0**-23


@pytest.mark.parametrize("rot,base,scale,trained", [(128, 1000000.0, 4.0, 32768), (64, 10000.0, 16.0, 4096), (8, 10000.0, 2.0, 16)])
def test_rope_factors_yarn(rot, base, scale, trained):
    f, m = hayai_amd.rope_factors(hayai_amd.ROPE_YARN, rot, base, scale, trained)
    assert abs(m - (0.1 * math.log(scale) + 1)) < 1e-6

    def pair(times):
        return rot * math.log(trained / (times * 2 * math.pi)) / (2 * math.log(base))
    lo, hi = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), rot - 1)
    for i in range(rot // 2):
        r = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
        # the turned frequency is a mixture of the model's own and the slowed one
        assert abs(1 / f[i] - ((1 - r) + r / scale)) < 1e-6
    assert f[0] <= f[-1] <= scale * (1 + 1e-6)


def test_rope_factors_refused():
    lib, out = _abi.load(), (C.c_float * 256)()
    for args in [(3, 64, 1e4, 2.0, 100.0), (0, 63, 1e4, 2.0, 100.0), (0, 0, 1e4, 2.0, 100.0), (0, 258, 1e4, 2.0, 100.0),
                 (0, 64, 1.0, 2.0, 100.0), (0, 64, math.inf, 2.0, 100.0), (0, 64, 1e4, 0.5, 100.0), (0, 64, 1e4, math.nan, 100.0),
                 (0, 64, 1e4, 2.0, 0.0), (0, 64, math.nan, 2.0, 1.0)]:
        assert lib.hh_rope_factors(*args, C.cast(out, C.c_void_p), None) == 2, args
    assert lib.hh_rope_factors(0, 64, 1e4, 2.0, 100.0, None, None) == 2
    assert lib.hh_rope_factors(0, 64, 1e4, 2.0, 100.0, C.cast(out, C.c_void_p), None) == 0


def test_attention_null_arguments_and_layout():
    lib, kv = _abi.load(), _abi.KvDesc()
    assert lib.hh_attn_prompt_dev(None, C.byref(_abi.AttnPromptDesc()), C.byref(kv), *[None, 0] * 6) == 2
    assert b"engine is NULL" in lib.hh_last_error()
    assert lib.hh_attn_decode_dev(None, C.byref(_abi.AttnDecodeDesc()), C.byref(kv), *[None, 0] * 6) == 2
    assert b"engine is NULL" in lib.hh_last_error()
    assert C.sizeof(_abi.AttnPromptDesc) == 56 and _abi.AttnPromptDesc.table_stride.offset == 32
    assert C.sizeof(_abi.AttnDecodeDesc) == 56 and _abi.AttnDecodeDesc.prefix.offset == 24
