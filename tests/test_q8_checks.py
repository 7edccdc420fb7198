"""Refusals of the 8-bit floating point operators, without a device: the argument checks are plain C
(inferenz_b200/csrc/host/op_check.c), compiled here on their own and called with pointers that nothing reads."""
import ctypes
import os
import shutil
import subprocess

import pytest

from inferenz_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, BAD, UNSUPPORTED = 0, 1, 8
P = 1 << 20  # an aligned address


@pytest.fixture(scope="module")
def checks(tmp_path_factory):
    gcc = shutil.which("gcc", path="/usr/bin") or shutil.which("gcc")
    if not gcc:
        pytest.skip("no C compiler")
    so = str(tmp_path_factory.mktemp("q8") / "op_check.so")
    subprocess.run([gcc, "-std=gnu11", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC",
                    os.path.join(ROOT, "inferenz_b200", "csrc", "host", "op_check.c"), "-o", so], check=True)
    return ctypes.CDLL(so)


def _call(checks, name, args):
    err = ctypes.create_string_buffer(200)
    return getattr(checks, "inzg__check_" + name)(ctypes.byref(args), err, ctypes.c_size_t(200)), err.value.decode()


def _norm(**kw):
    return _lib.RmsnormQ8Args(**{**dict(n=4, cols=256, type=_lib.T_BF16, x=P, w=P, eps=1e-6, q=P, s=P), **kw})


def _silu(**kw):
    return _lib.SiluMulQ8Args(**{**dict(n=4, cols=256, type=_lib.T_F32, x=P, q=P, s=P), **kw})


def _matmul(**kw):
    return _lib.MatmulQ8Args(**{**dict(m=4, n=256, k=256, a=P, a_scale=P, w=P, w_scale=P, out=P, out_type=_lib.T_BF16), **kw})


def _grouped(**kw):
    return _lib.GroupedMatmulArgs(**{**dict(type=_lib.T_E4M3, groups=8, n=256, k=256, a_rows=16, entries=16, out_rows_n=16,
                                            a=P, a_scale=P, w=P, w_scale=P, off=P, out=P, out_type=_lib.T_F32), **kw})


@pytest.mark.parametrize("kw,want", [
    ({}, OK), ({"n": 0, "x": None, "w": None}, OK), ({"q": None, "s": None, "y": P}, OK), ({"res": P, "sum": P}, OK),
    ({"ldx": 257, "ldq": 300}, OK), ({"cols": 32768}, OK), ({"cols": 32769}, UNSUPPORTED), ({"cols": 0}, BAD),
    ({"n": -1}, BAD), ({"type": _lib.T_E4M3}, UNSUPPORTED), ({"type": 7}, UNSUPPORTED), ({"x": None}, BAD),
    ({"w": None}, BAD), ({"q": None, "s": None}, BAD), ({"s": None}, BAD), ({"q": None}, BAD), ({"ldx": 255}, BAD),
    ({"res": P, "ldres": 1}, BAD), ({"sum": P, "ldsum": 10}, BAD), ({"y": P, "ldy": -4}, BAD), ({"ldq": 200}, BAD),
    ({"lds": 1}, BAD), ({"eps": -1.0}, BAD), ({"eps": float("nan")}, BAD), ({"x": P + 1}, BAD), ({"w": P + 2}, BAD),
    ({"s": P + 2}, BAD), ({"ldx": 1 << 62}, BAD), ({"sum": P, "x": P, "ldx": 300}, BAD),
    ({"sum": P, "x": P, "ldx": 300, "ldsum": 300}, OK), ({"res": P + 64, "sum": P + 64, "ldsum": 300}, BAD),
])
def test_rmsnorm_q8(checks, kw, want):
    st, msg = _call(checks, "rmsnorm_q8", _norm(**kw))
    assert st == want and (st == OK or msg.startswith("rmsnorm_q8: "))


@pytest.mark.parametrize("kw,want", [
    ({}, OK), ({"n": 0, "x": None}, OK), ({"y": P}, OK), ({"cols": 0}, BAD), ({"cols": 1 << 30}, BAD), ({"n": -2}, BAD),
    ({"type": _lib.T_Q4L}, UNSUPPORTED), ({"ldx": 511}, BAD), ({"ldx": 512}, OK), ({"y": P, "ldy": 255}, BAD),
    ({"q": None}, BAD), ({"q": None, "s": None}, BAD), ({"x": P + 2}, BAD), ({"ldq": 8}, BAD), ({"ldx": 1 << 61}, BAD),
])
def test_silu_mul_q8(checks, kw, want):
    st, msg = _call(checks, "silu_mul_q8", _silu(**kw))
    assert st == want and (st == OK or msg.startswith("silu_mul_q8: "))


@pytest.mark.parametrize("kw,want", [
    ({}, OK), ({"m": 0, "a": None}, OK), ({"k": 1, "lda": 16, "ldw": 16}, OK), ({"k": 100, "lda": 112, "ldw": 112}, OK),
    ({"k": 100}, BAD), ({"lda": 264}, BAD), ({"ldw": 250}, BAD), ({"lda": 240}, BAD), ({"n": 0}, BAD), ({"k": 0}, BAD),
    ({"m": -1}, BAD), ({"a": P + 8}, BAD), ({"w": P + 8}, BAD), ({"out": P + 1}, BAD), ({"a_scale": None}, BAD),
    ({"w_scale": None}, BAD), ({"lda_scale": 1}, BAD), ({"ldo": 255}, BAD), ({"out_type": _lib.T_E4M3}, UNSUPPORTED),
    ({"out": None}, BAD), ({"m": 2**31 - 1, "n": 2**31 - 300}, UNSUPPORTED), ({"lda": 1 << 41}, UNSUPPORTED),
    ({"n": 2**31 - 1}, BAD), ({"a_scale": P + 2}, BAD),
])
def test_matmul_q8(checks, kw, want):
    st, msg = _call(checks, "matmul_q8", _matmul(**kw))
    assert st == want and (st == OK or msg.startswith("matmul_q8: "))


BF = {"type": _lib.T_BF16, "a_scale": None, "w_scale": None}


@pytest.mark.parametrize("kw,want", [
    ({}, OK), (BF, OK), ({**BF, "type": _lib.T_F16}, OK), ({**BF, "k": 8}, OK), ({**BF, "k": 4}, BAD),
    ({"entries": 0, "a": None, "off": None}, OK), ({"type": _lib.T_F32}, UNSUPPORTED), ({"groups": 0}, BAD),
    ({"groups": 2048}, OK), ({"groups": 2049}, UNSUPPORTED), ({"type": _lib.T_BF16}, BAD), ({"a_scale": None}, BAD),
    ({"a_rows": 15}, BAD), ({"a_rows": 15, "in_rows": P}, OK), ({"a_rows": 0, "in_rows": P}, BAD), ({"out_rows_n": 15}, BAD),
    ({"out_rows_n": 15, "out_rows": P}, OK), ({"out_rows_n": 0, "out_rows": P}, BAD), ({"off": None}, BAD),
    ({"off": P + 2}, BAD), ({"in_rows": P + 1}, BAD), ({"out_scale": P + 1}, BAD), ({"entries": -1}, BAD),
    ({"groups": 2000, "n": 2_000_000}, UNSUPPORTED), ({"ldw": 255}, BAD), ({"a": P + 4}, BAD),
    ({"out_type": 9}, UNSUPPORTED), ({"k": 0}, BAD), ({"n": -5}, BAD),
    ({"entries": 2**31 - 1, "a_rows": 2**31 - 1, "out_rows_n": 2**31 - 1, "n": 10_000}, UNSUPPORTED),
])
def test_grouped_matmul(checks, kw, want):
    st, msg = _call(checks, "grouped_matmul", _grouped(**kw))
    assert st == want and (st == OK or msg.startswith("grouped_matmul: "))


@pytest.mark.parametrize("a,want", [
    ((4, 10, 512, P, P, P, P, P, P), OK), ((4, 10, 512, P, None, P, P, P, None), OK),
    ((0, 10, 512, None, None, P, None, None, None), OK), ((4, 10, 2048, P, P, P, P, P, P), OK),
    ((4, 10, 2049, P, P, P, P, P, P), UNSUPPORTED), ((4, 0, 512, P, P, P, P, P, P), BAD),
    ((-1, 10, 512, P, P, P, P, P, P), BAD), ((4, 10, 0, P, P, P, P, P, P), BAD), ((4, 10, 512, P, P, None, P, P, P), BAD),
    ((4, 10, 512, None, P, P, P, P, P), BAD), ((4, 10, 512, P, P, P, None, P, P), BAD),
    ((4, 10, 512, P, P, P, P, None, P), BAD), ((4, 10, 512, P, P, P, P, P, None), BAD),
    ((4, 10, 512, P + 2, P, P, P, P, P), BAD), ((1 << 30, 10, 512, P, P, P, P, P, P), UNSUPPORTED),
])
def test_expert_lists(checks, a, want):
    err = ctypes.create_string_buffer(200)
    st = checks.inzg__check_expert_lists(*a[:3], *(ctypes.c_void_p(p) for p in a[3:]), err, ctypes.c_size_t(200))
    assert st == want and (st == OK or err.value.decode().startswith("expert_lists: "))


def test_no_arguments_or_context(checks):
    for name in ("rmsnorm_q8", "silu_mul_q8", "matmul_q8", "grouped_matmul"):
        err = ctypes.create_string_buffer(200)
        assert getattr(checks, "inzg__check_" + name)(None, err, ctypes.c_size_t(200)) == BAD
        assert getattr(_lib.lib, "inzg_" + name)(None, None) == BAD
    assert _lib.lib.inzg_expert_lists(None, 1, 1, 1, *[None] * 7) == BAD


def test_struct_layouts_match_the_header(tmp_path):
    """sizeof and offsets of the argument structs as a C compiler sees the header"""
    gcc = shutil.which("gcc", path="/usr/bin") or shutil.which("gcc")
    if not gcc:
        pytest.skip("no C compiler")
    pairs = {"inzg_rmsnorm_q8_args": _lib.RmsnormQ8Args, "inzg_silu_mul_q8_args": _lib.SiluMulQ8Args,
             "inzg_matmul_q8_args": _lib.MatmulQ8Args, "inzg_grouped_matmul_args": _lib.GroupedMatmulArgs}
    body = "".join(f'printf("{c} %zu\\n", sizeof({c}));' + "".join(
        f'printf("{c}.{f} %zu\\n", offsetof({c}, {f}));' for f, _ in t._fields_) for c, t in pairs.items())
    src = tmp_path / "s.c"
    src.write_text(f'#include <stddef.h>\n#include <stdio.h>\n#include "inzg.h"\nint main(void) {{ {body} return 0; }}\n')
    exe = str(tmp_path / "s")
    subprocess.run([gcc, "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    got = dict(ln.split() for ln in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.splitlines())
    for c, t in pairs.items():
        assert int(got[c]) == ctypes.sizeof(t)
        for f, _ in t._fields_:
            assert int(got[f"{c}.{f}"]) == getattr(t, f).offset


M31 = 2**31 - 1


@pytest.mark.parametrize("rows,want", [(M31, UNSUPPORTED), (M31 - 30, UNSUPPORTED), (M31 - 255, UNSUPPORTED), (M31 - 256, OK)])
def test_rows_that_round_up_past_32_bits(checks, rows, want):
    """the products number tiles of up to 128 entries in 32 bits: rounding the rows up to whole tiles must not pass them (the call was
    accepted and computed nothing)"""
    st, msg = _call(checks, "matmul_q8", _matmul(m=rows, n=1, k=16))
    assert st == want and (st == OK or "too many rows" in msg)
    st, msg = _call(checks, "grouped_matmul", _grouped(entries=rows, a_rows=rows, out_rows_n=rows, groups=1, n=1, k=16))
    assert st == want and (st == OK or "too many entries" in msg)
    st, msg = _call(checks, "grouped_matmul", _grouped(entries=rows, in_rows=P, out_rows=P, groups=1, n=1, k=16))
    assert st == want and (st == OK or "too many entries" in msg)


def _tile(checks, t, groups, entries, n, sms=148):
    return checks.inzg__grouped_matmul_tile(t, groups, entries, n, sms)


def test_which_tiles_a_product_takes(checks):
    """few entries per group, or few items, take tiles of 32 entries; the tests of the wide tiles have sizes that take those"""
    import test_gpu_q8 as gpu
    for case in gpu.LONG_LISTS + gpu.RAGGED:
        assert _tile(checks, *case) == 128
    e4m3, bf16 = _lib.T_E4M3, _lib.T_BF16
    assert [_tile(checks, e4m3, 512, m, 640) for m in (1, 320, 64 * 512, 64 * 512 + 1)] == [32, 32, 32, 128]
    assert [_tile(checks, e4m3, 1, m, 10240) for m in (1, 96, 97, 4000)] == [32, 32, 128, 128]
    assert [_tile(checks, bf16, 64, m, 1280) for m in (1, 40 * 64, 40 * 64 + 1)] == [32, 32, 128]
    assert [_tile(checks, bf16, 1, m, 40960) for m in (32, 33)] == [32, 128] and _tile(checks, bf16, 1, 192, 1280) == 32
    assert _tile(checks, e4m3, 2048, 2**31 - 256, 128) == 128 and _tile(checks, e4m3, 1, 2**31 - 256, 1) == 128
