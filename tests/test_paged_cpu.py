"""Rotary frequencies, the paged cache's refusals on the host, and the paged
kernels' integer arithmetic (tests/paged_deal.cpp), without a GPU."""
import ctypes
import math
import os
import re
import subprocess

import numpy as np
import pytest

import ramvamp_amd as rv
from ramvamp_amd import _lib as L
from ramvamp_amd import build as B

HERE = os.path.dirname(os.path.abspath(__file__))


def test_dealing_and_places_on_the_host(tmp_path):
    exe = str(tmp_path / "paged_deal")
    subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), "-x", "hip", "--offload-host-only", "-O1",
                    "-std=c++17", "-o", exe, os.path.join(HERE, "paged_deal.cpp")], check=True, capture_output=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0 and not out.stdout, out.stdout


def partial_saves(asm):
    """Labels of blocks that save vector registers before they restore the exec mask
    there: of the lanes that went another way the copy holds nothing, yet it is read
    back for all of them."""
    found = []
    for body in re.findall(r"^_Z\S+:\s.*?\.Lfunc_end", asm, re.M | re.S):
        loops = set(re.findall(r"s_cbranch_execnz (\.LBB\d+_\d+)", body))
        lines = [l.strip() for l in body.splitlines()]
        for i, l in enumerate(lines):
            if not re.match(r"\.LBB\d+_\d+:", l) or l.split(":")[0] in loops:
                continue
            saves = False
            for t in lines[i + 1:i + 40]:
                if t.startswith(("s_or_b64 exec", "s_or_saveexec", "s_andn2_saveexec")):
                    if saves:
                        found.append(l.split(":")[0])
                    break
                if re.match(r"s_cbranch|s_branch|\.LBB|s_and_saveexec|s_endpgm", t):
                    break
                saves |= t.startswith(("v_accvgpr", "scratch_", "buffer_"))
    return found


def test_no_register_is_saved_under_a_partial_mask(tmp_path):
    """The attention kernels keep whole tiles in registers, more than 256 with the
    widest heads, and every value has to be kept for every lane."""
    planted = ("_Zk: ; @k\n s_and_saveexec_b64 s[0:1], vcc\n s_cbranch_execz .LBB0_2\n; %bb.1:\n v_mov_b32_e32 v1, 0\n"
               ".LBB0_2:\n{} s_or_b64 exec, exec, s[0:1]\n s_endpgm\n.Lfunc_end0:\n")
    assert partial_saves(planted.format(" v_accvgpr_write_b32 a0, v0\n")) == [".LBB0_2"]
    assert not partial_saves(planted.format(""))
    out = str(tmp_path / "attn.s")
    subprocess.run([B.HIPCC, *B.FLAGS, "--offload-device-only", "-S", "-o", out,
                    os.path.join(os.path.dirname(HERE), "ramvamp_amd", "csrc", "rv_paged_attn.hip")], check=True,
                   capture_output=True)
    with open(out) as f:
        asm = f.read()
    assert asm.count("paged_attn_kernel") > 20 and not partial_saves(asm)


def frequencies(d, theta, scaling, factor, trained, fast=32.0, slow=1.0):
    """Pair by pair, as the definition is written."""
    f, gain = [], 1.0
    if scaling == "ntk":
        theta = theta * factor ** (d / (d - 2))
    if scaling == "yarn":
        at = [d * math.log(trained / (2 * math.pi * b)) / (2 * math.log(theta)) for b in (fast, slow)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), d - 1)
        gain = 0.1 * math.log(factor) + 1
    for i in range(d // 2):
        x = theta ** (-2 * i / d)
        if scaling == "linear":
            x /= factor
        if scaling == "yarn":
            r = min(max((i - lo) / max(hi - lo, 0.001), 0), 1)
            x = x * (1 - r) + x / factor * r
        f.append(x)
    return np.array(f), gain


@pytest.mark.parametrize("d,theta,scaling,factor,trained", [
    (128, 1e6, "none", 1, 0), (128, 1e7, None, 1, 0), (2, 1e4, "none", 1, 0), (512, 0.5, "none", 1, 0),
    (64, 1e4, "linear", 8, 0), (128, 1e6, "ntk", 4, 0), (4, 1e4, "ntk", 1, 0),
    (128, 1e6, "yarn", 4, 32768), (32, 1e4, "yarn", 40, 4096), (64, 1e4, "yarn", 1, 1), (6, 1e6, "yarn", 2, 10 ** 9),
])
def test_rope_frequencies(d, theta, scaling, factor, trained):
    f, gain = rv.Rope(512, theta, rotary_dim=d, scaling=scaling, factor=factor, trained_positions=trained).frequencies()
    want, want_gain = frequencies(d, theta, scaling, factor, trained)
    # pow, log and a handful of f64 operations, each off by at most an ulp of values
    # that are no larger than what comes out (times the exponent's size for pow).
    assert np.all(np.abs(f - want) <= 64 * 2.0 ** -52 * want) and abs(gain - want_gain) <= 4 * 2.0 ** -52


def test_yarn_leaves_fast_pairs_and_interpolates_slow_ones():
    f, _ = rv.Rope(128, 1e6, scaling="yarn", factor=4, trained_positions=32768).frequencies()
    plain, _ = rv.Rope(128, 1e6).frequencies()
    assert f[0] == plain[0] and abs(f[-1] * 4 / plain[-1] - 1) < 1e-12


def test_other_betas_move_the_ramp():
    f, _ = rv.Rope(64, 1e4, scaling="yarn", factor=8, trained_positions=4096, beta_fast=16, beta_slow=2).frequencies()
    want, _ = frequencies(64, 1e4, "yarn", 8, 4096, 16, 2)
    assert np.allclose(f, want, rtol=1e-13, atol=0)


@pytest.mark.parametrize("kw,variant", [
    (dict(head_dim=0, rotary_dim=2), "InvalidHeadDim"), (dict(rotary_dim=0), "InvalidHeadDim"),
    (dict(rotary_dim=3), "InvalidHeadDim"), (dict(rotary_dim=130), "InvalidHeadDim"),
    (dict(head_dim=514), "Unsupported"), (dict(theta=0.0), "Unsupported"), (dict(theta=-1.0), "Unsupported"),
    (dict(theta=math.inf), "Unsupported"), (dict(theta=math.nan), "Unsupported"),
    (dict(scaling="linear", factor=0.5), "Unsupported"), (dict(scaling="linear", factor=math.nan), "Unsupported"),
    (dict(scaling="ntk", factor=math.inf), "Unsupported"), (dict(scaling="ntk", factor=2, rotary_dim=2), "Unsupported"),
    (dict(scaling="yarn", factor=2), "Unsupported"),
    (dict(scaling="yarn", factor=2, trained_positions=8, theta=1.0), "Unsupported"),
    (dict(scaling="yarn", factor=2, trained_positions=8, beta_slow=0.0), "Unsupported"),
    (dict(scaling="yarn", factor=2, trained_positions=8, beta_fast=1.0), "Unsupported"),
    (dict(scaling="yarn", factor=2, trained_positions=8, beta_fast=math.inf), "Unsupported"),
])
def test_rope_refusals(kw, variant):
    with pytest.raises(rv.RamvampError) as e:
        rv.Rope(**{"head_dim": 128, "theta": 1e6, **kw})
    assert e.value.variant == variant


def test_rope_names_are_checked():
    for kw in (dict(layout="neox"), dict(scaling="dynamic")):
        with pytest.raises(ValueError):
            rv.Rope(128, 1e6, **kw)
    err = L.RvError()
    h = ctypes.c_void_p()
    assert L.load().rv_rope_new(128, 128, 2, 1e6, 0, 1.0, 0, 32.0, 1.0, ctypes.byref(h), ctypes.byref(err)) == 33
    assert L.load().rv_rope_new(128, 128, 0, 1e6, 4, 1.0, 0, 32.0, 1.0, ctypes.byref(h), ctypes.byref(err)) == 33
    assert L.load().rv_rope_new(128, 128, 0, 1e6, 0, 1.0, 0, 32.0, 1.0, None, ctypes.byref(err)) == 32


@pytest.mark.parametrize("x,xs,out,os,rows,width,flags,code", [
    (4096, 128, 8192, 128, 2, 100, 0, 16), (4096, 128, 8192, 128, 2, 0, 0, 16),
    (4096, 100, 1 << 20, 128, 2, 128, 0, 25), (4096, 128, 1 << 20, 127, 2, 128, 0, 25),
    (4096, 128, 1 << 20, 128, 2, 128, 1, 33), (None, 128, 1 << 20, 128, 2, 128, 0, 32),
    (4096, 128, None, 128, 2, 128, 0, 32),
    (4096, 128, 4100, 128, 2, 128, 0, 33),             # shifted by a value
    (4096, 256, 4096, 128, 2, 128, 0, 33),             # x's first row is out's
    (4096, 256, 4096 + 4 * 64, 256, 8, 128, 0, 33),    # half a row further
    (4096, 256, 4096 + 4 * 320, 256, 8, 128, 0, 33),   # the next row's second half
])
def test_rope_rows_refusals(x, xs, out, os, rows, width, flags, code):
    """Refused before anything is queued: the addresses are never read."""
    rope, err = rv.Rope(128, 1e6), L.RvError()
    rc = L.load().rv_rope_rows(rope._h, x, xs, rows, width, 64, out, os, None, flags, ctypes.byref(err))
    assert rc == code == err.code
    assert L.load().rv_rope_rows(None, x, xs, rows, width, 64, out, os, None, 0, ctypes.byref(err)) == 32


def test_rope_frequencies_refusals():
    rope, err = rv.Rope(128, 1e6), L.RvError()
    buf = (ctypes.c_double * 64)()
    assert L.load().rv_rope_frequencies(rope._h, buf, 63, None, ctypes.byref(err)) == 25
    assert L.load().rv_rope_frequencies(None, buf, 64, None, ctypes.byref(err)) == 32
    assert L.load().rv_rope_frequencies(rope._h, None, 64, None, ctypes.byref(err)) == 32


def test_projected_bytes():
    assert rv.PagedKvCache.projected_bytes(48, 4, 128, 1000, 64, "f16") == 48 * 4 * 128 * 64000 * 2 * 2
    assert rv.PagedKvCache.projected_bytes(1, 4, 128, 3, 8, "f32") == 4 * 128 * 24 * 4 * 2
    assert rv.PagedKvCache.projected_bytes(2, 1, 96, 5, 1024, "q8_0") == 2 * 3 * 5 * 1024 * 34 * 2


@pytest.mark.parametrize("args,variant", [
    ((0, 4, 128, 8, 64, "f16"), "InvalidDims"), ((1, 0, 128, 8, 64, "f16"), "InvalidDims"),
    ((1, 4, 0, 8, 64, "f16"), "InvalidDims"), ((1, 4, 128, 0, 64, "f16"), "InvalidDims"),
    ((1, 4, 128, 8, 4, "f16"), "InvalidDims"), ((1, 4, 128, 8, 48, "f16"), "InvalidDims"),
    ((1, 4, 128, 8, 2048, "f16"), "InvalidDims"), ((1, 4, 100, 8, 64, "q8_0"), "InvalidDims"),
    ((1, 4, 513, 8, 64, "f32"), "Unsupported"), ((1, 4, 128, 2 ** 31, 64, "f16"), "Unsupported"),
    ((1, 2 ** 31, 128, 8, 64, "f16"), "Unsupported"), ((1, 65536, 1, 8, 64, "f16"), "Unsupported"), ((2 ** 60, 4, 128, 8, 64, "f16"), "InvalidDims"),
    ((2 ** 30, 65535, 128, 2 ** 30, 1024, "f32"), "InvalidDims"),
])
def test_geometry_refusals(args, variant):
    for call in (rv.PagedKvCache.projected_bytes, rv.PagedKvCache):
        with pytest.raises(rv.RamvampError) as e:
            call(*args)
        assert e.value.variant == variant


def test_calls_without_a_cache():
    lib, err = L.load(), L.RvError()
    t = L.RvPageTable(None, 0, 0, 0)
    e, b = ctypes.byref(err), ctypes.byref(t)
    assert lib.rv_paged_append_rows(None, 0, None, None, 0, None, 0, 0, None, None, b, None, 0, 0.0, 0, e) == 32
    assert lib.rv_paged_read_rows(None, 0, 0, None, None, b, None, None, 0, e) == 32
    assert lib.rv_paged_attention(None, 0, None, 0, 0, 0, b, None, 1.0, None, 0, 0, e) == 32
    assert lib.rv_paged_decode_step(None, 0, None, None, 0, None, 0, None, 0, 0, 0, None, 0, None, 0, 0.0, b, None, 1.0,
                                    None, 0, 0, e) == 32
    assert lib.rv_paged_set_stream(None, None, e) == lib.rv_paged_synchronize(None, e) == 32
    assert lib.rv_paged_device_status(None, e) == lib.rv_paged_set_tuning(None, 1, 2, e) == 32
    lib.rv_paged_free(None)
    lib.rv_rope_free(None)


def test_status_names():
    names = [L.load().rv_status_name(c).decode() for c in (56, 57, 58)]
    assert names == ["RV_PAGED_PAGE_OUT_OF_RANGE", "RV_PAGED_SEQUENCE_OUT_OF_RANGE", "RV_PAGED_POSITION_OUT_OF_RANGE"]


def test_host_tensors_are_refused():
    torch = pytest.importorskip("torch")
    x, at = torch.zeros(2, 128), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(TypeError):
        rv.rope_rows(x, at, rv.Rope(128, 1e6))
    with pytest.raises(TypeError):
        rv.rope_rows(np.zeros((2, 128), np.float32), at, rv.Rope(128, 1e6), x)


def test_joins_on_the_host(tmp_path):
    """Partials in lines of their own."""
    exe = str(tmp_path / "paged_joins")
    subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), "-x", "hip", "--offload-host-only", "-O1",
                    "-std=c++17", "-o", exe, os.path.join(HERE, "paged_joins.cpp")], check=True, capture_output=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0 and not out.stdout, out.stdout


def test_a_cache_passes_from_stream_to_stream_on_the_host(tmp_path):
    """Calls wait for all earlier ones, whatever was captured in between."""
    exe = str(tmp_path / "stream_order")
    subprocess.run([os.environ.get("CXX", "g++"), "-O1", "-std=c++17", "-o", exe, os.path.join(HERE, "stream_order.cpp")],
                   check=True, capture_output=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0 and not out.stdout, out.stdout


@pytest.mark.parametrize("at,code", [
    (8192, 33), (8188, 33), (8192 + 4 * 127, 33), (8192 + 4 * 255, 33), (8192 + 4 * 128 * 7 + 4 * 127, 33),
    (8192 + 4 * 256 * 7 + 4 * 127, 33), (8192 + 4 * 249, 33), (8192 - 4 * 7, 33), (4096, 33), (4096 + 4 * 120, 33),
])
def test_rotated_rows_over_their_positions_are_refused(at, code):
    """8 rows of 128 of a wider buffer, and positions that they reach, or a place of x
    that they are; the addresses are never read."""
    rope, err = rv.Rope(128, 1e6), L.RvError()
    out = 4096 if at < 8000 else 8192
    call = lambda p, rows: L.load().rv_rope_rows(rope._h, out, 256, rows, 128, p, out, 256, None, 0, ctypes.byref(err))
    assert call(at, 8) == code == err.code
    assert b"positions" in err.what


@pytest.mark.parametrize("kw", [dict(theta=5e-324), dict(theta=1e-308), dict(theta=1e308, scaling="ntk", factor=1e10),
                                dict(theta=1e6, rotary_dim=4, scaling="ntk", factor=1e200)])
def test_rope_bases_whose_angles_are_not_finite_are_refused(kw):
    with pytest.raises(rv.RamvampError) as e:
        rv.Rope(**{"head_dim": 512, **kw})
    assert e.value.variant == "Unsupported"


def test_rope_bases_at_the_ends_of_the_range():
    for theta in (1e-290, 1e308):
        f, _ = rv.Rope(512, theta).frequencies()
        assert np.all(np.isfinite(f * 2.0 ** 31)) and f[0] == 1.0


def test_masks_are_spelled_as_the_check_of_saves_reads_them(tmp_path):
    """A divergent branch of this compiler ends in a label and the mask's restoring below
    it, in the words that partial_saves looks for: another spelling fails here."""
    src, out = tmp_path / "k.hip", str(tmp_path / "k.s")
    src.write_text("#include <hip/hip_runtime.h>\n"
                   "__global__ void k(float* x, int n) {\n"
                   "  float y = x[threadIdx.x];\n"
                   "  if ((int)threadIdx.x < n) { y += x[threadIdx.x + 64]; __syncthreads(); x[threadIdx.x + 128] = y; }\n"
                   "  x[threadIdx.x] = y;\n}\n")
    subprocess.run([B.HIPCC, *B.FLAGS, "--offload-device-only", "-S", "-o", out, str(src)], check=True, capture_output=True)
    with open(out) as f:
        body = re.search(r"^_Z\S+:\s.*?\.Lfunc_end", f.read(), re.M | re.S).group()
    assert re.search(r"s_and_saveexec_b64 [^\n]*\n(?:[^\n]*\n)*?\s*s_cbranch_execz (\.LBB\d+_\d+)\n(?:[^\n]*\n)*?"
                     r"\1:[^\n]*\n(?:\s*;[^\n]*\n)*\s*s_or_b64 exec, exec,", body), body
