"""What the Q8_0 cache and shared-prefix decode refuse or compute on the host
(no GPU), and the format's numpy form against the oracle's quantizer."""
import ctypes

import numpy as np
import pytest

import oracle
from ramvamp_amd import _lib as L
from rows_util import q8_blocks, q8_values


@pytest.fixture(scope="module")
def lib():
    return L.load()


def test_the_numpy_format_is_the_oracle_s_quantizer():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((40, 256)).astype(np.float32) * 10.0 ** rng.uniform(-6, 4, (40, 1)).astype(np.float32)
    x[0] = 0
    x[1, :32] = np.arange(32) * 0.5 - 7.75
    codes, scales = q8_blocks(x)
    o = np.frombuffer(oracle.quantize_row_q8_0(x.reshape(-1)).tobytes(), np.uint8).reshape(-1, 36)
    assert np.array_equal(o[:, 4:].view(np.int8), codes.reshape(-1, 32))
    assert np.array_equal(o[:, :4].copy().view(np.float32).ravel(), scales.astype(np.float32).ravel())


def test_values_saturate_and_carry_nan_by_the_block():
    x = np.zeros((4, 64), np.float32)
    x[0, 0], x[0, 1], x[0, 2] = 1e30, -1e30, 1000.0
    x[1, 3], x[1, 4] = np.inf, 1.0
    x[2, 5] = np.nan
    x[3, 0] = 65468.0
    v = q8_values(x)
    assert v[0, 0] == 65472.0 and v[0, 1] == -65472.0 and v[0, 2] == 1031.0 and not v[0, 32:].any()
    assert np.isnan(v[1:3, :32]).all() and not v[1:3, 32:].any()
    assert v[3, 0] == 65472.0


@pytest.mark.parametrize("dims,code", [((1, 2, 48, 8), 1), ((1, 2, 544, 8), 1), ((0, 2, 64, 8), 1),
                                       ((1, 2, 64, 2 ** 60), 1), ((1, 2, 64, 8), 0), ((2, 3, 32, 1), 0)])
def test_projected_bytes(lib, dims, code):
    n, err = ctypes.c_uint64(), L.RvError()
    assert lib.rv_kv_projected_bytes(*dims, L.RV_ELEM_Q8_0, ctypes.byref(n), ctypes.byref(err)) == code
    if code == 0:
        assert n.value == 2 * dims[0] * dims[1] * dims[2] * dims[3] // 32 * 34
        more, err = ctypes.c_uint64(), L.RvError()
        assert lib.rv_kv_projected_device_bytes(*dims, L.RV_ELEM_Q8_0, ctypes.byref(more), ctypes.byref(err)) == 0
        assert more.value > n.value


def test_a_cache_too_large_for_the_kernels_is_refused_before_any_device_call(lib):
    h, err = ctypes.c_void_p(), L.RvError()
    assert lib.rv_kv_new(1, 1, 32, 2 ** 31 - 255, L.RV_ELEM_Q8_0, 0, ctypes.byref(h), ctypes.byref(err)) == 33
    assert lib.rv_kv_new(2 ** 45, 2 ** 8, 32, 1, L.RV_ELEM_Q8_0, 0, ctypes.byref(h), ctypes.byref(err)) == 1
    assert not h.value


def test_null_arguments(lib):
    err = L.RvError()
    e = ctypes.byref(err)
    assert lib.rv_kv_truncate_layer(None, 0, 0, e) == 32
    assert lib.rv_kv_append_each(None, 0, 1, None, None, 1, 0, e) == 32
    assert lib.rv_kv_read_rows(None, 0, 0, 1, None, None, 0, e) == 32
    assert lib.rv_decode_attention_shared(None, 0, 0, None, 0, None, 1, 1, 1.0, None, 0, e) == 32
    assert err.what == b"prefix"
    assert lib.rv_decode_step_shared(None, 0, 0, None, 0, 1, None, None, None, 1, None, 1, None, 1, 1e-6, 1e6, 1.0,
                                     None, 0, e) == 32


def test_the_row_kernels_keep_their_operands_in_registers(tmp_path):
    """What the compiled kernels ask of the card, read from the built library."""
    import os
    import re
    import subprocess

    from test_device_code import READELF, code_objects

    if not os.path.exists(READELF):
        pytest.skip("no llvm-readelf")
    path, found = tmp_path / "object", 0
    for obj in code_objects():
        path.write_bytes(obj)
        notes = subprocess.run([READELF, "--notes", str(path)], capture_output=True, text=True, check=True).stdout
        for entry in notes.split("\n  - ")[1:]:
            name = re.findall(r"^\s*\.name:\s+(_Z\S+)", entry, re.M)
            if name and re.search(r"rows_(narrow|wide|merge)_kernel", name[-1]):
                v = {k: int(x) for k, x in re.findall(r"^\s*\.(\w+):\s+(\d+)$", entry, re.M)}
                assert v["vgpr_spill_count"] == 0 and v["private_segment_fixed_size"] == 0, name[-1]
                found += 1
    assert found >= 20
