"""The 8-bit integer operators without a GPU: the header and the binding
agree, and bad arguments are refused before a device is touched."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest

import uocr_moe as M

INCLUDE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
HEADER = os.path.join(INCLUDE, "uocr_int8.h")
BASE = 1 << 20  # an aligned address that is never read


def test_header_and_binding_agree():
    names = re.findall(r"^int (uocr_[a-z_0-9]+)\s*\(", open(HEADER).read(), re.M)
    assert sorted(names) == sorted(M.INT8_EXPORTS)
    for name in names:
        assert hasattr(M.lib(), name), name


def test_struct_layouts_match_the_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    structs = {"uocr_linear_w8a8_args": M.LinearW8A8Args, "uocr_grouped_w8a8_args": M.GroupedW8A8Args}
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "uocr_int8.h"', "int main(void) {"]
    for cname, cls in structs.items():
        lines.append(f'  printf("%zu\\n", sizeof({cname}));')
        lines += [f'  printf("%zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    subprocess.run([cc, "-I", INCLUDE, str(src), "-o", str(tmp_path / "layout")], check=True)
    got = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()
    want = []
    for cls in structs.values():
        want += [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]
    assert [int(v) for v in got] == want


def _quantize(**kw):
    a = dict(x=BASE, dtype=0, rows=4, cols=64, ldx=64, q=BASE, ldq=64, scales=BASE)
    a.update(kw)
    return M.lib().uocr_quantize_tokens(a["x"], a["dtype"], a["rows"], a["cols"], a["ldx"], a["q"], a["ldq"],
                                        a["scales"], None)


@pytest.mark.parametrize("wrong", [dict(rows=-1), dict(cols=-1), dict(dtype=2), dict(x=None), dict(q=None),
                                   dict(scales=None), dict(ldx=63), dict(ldq=63), dict(ldq=72), dict(q=BASE + 8),
                                   dict(x=BASE + 2), dict(x=BASE + 1, dtype=1)])
def test_quantize_tokens_refuses(wrong):
    assert _quantize(**wrong) == 1
    assert M.lib().uocr_last_error().decode().startswith("quantize_tokens: ")


def test_quantize_tokens_of_no_rows():
    assert _quantize(rows=0, x=None, q=None, scales=None) == 0


def _linear(**kw):
    a = dict(x=BASE, x_scales=BASE, w=BASE, w_scales=BASE, bias=None, residual=None, y=BASE, m=4, n=32, k=64, ldx=64,
             ldw=64, ldr=0, ldy=32, y_dtype=0, reserved=0)
    a.update(kw)
    return M.lib().uocr_linear_w8a8(ctypes.byref(M.LinearW8A8Args(**a)), None)


@pytest.mark.parametrize("wrong,code", [
    (dict(m=-1), 1), (dict(n=-1), 1), (dict(k=0), 1), (dict(m=1 << 31), 1), (dict(k=131072, ldx=131072, ldw=131072), 2),
    (dict(y_dtype=2), 1), (dict(reserved=1), 1), (dict(x=None), 1), (dict(x_scales=None), 1), (dict(w=None), 1),
    (dict(w_scales=None), 1), (dict(y=None), 1), (dict(ldx=48), 1), (dict(ldw=48), 1), (dict(ldy=31), 1),
    (dict(ldx=72), 1), (dict(ldw=72), 1), (dict(x=BASE + 4), 1), (dict(w=BASE + 8), 1), (dict(y=BASE + 2), 1),
    (dict(residual=BASE, ldr=16), 1), (dict(residual=BASE, ldr=33), 1), (dict(residual=BASE + 64 + 2, ldr=32), 1)])
def test_linear_w8a8_refuses(wrong, code):
    assert _linear(**wrong) == code
    assert M.lib().uocr_last_error().decode().startswith("linear_w8a8: ")


def test_linear_w8a8_of_no_rows_or_columns():
    assert _linear(m=0, x=None, x_scales=None, y=None) == 0
    assert _linear(n=0, w=None, w_scales=None, y=None) == 0
    assert M.lib().uocr_linear_w8a8(None, None) == 1


def _grouped(**kw):
    a = dict(x=BASE, x_scales=BASE, row_index=None, offsets=BASE, w=BASE, w_scales=BASE, w_up=None, w_up_scales=None,
             y=BASE, rows=8, x_rows=8, groups=4, n=32, k=64, ldx=64, ldw=64, ldy=32, y_dtype=1, reserved=0,
             workspace=None, workspace_bytes=0)
    a.update(kw)
    return M.lib().uocr_grouped_linear_w8a8(ctypes.byref(M.GroupedW8A8Args(**a)), None)


@pytest.mark.parametrize("wrong,code", [
    (dict(rows=-1), 1), (dict(groups=-1), 1), (dict(groups=513), 2), (dict(n=1 << 30), 1), (dict(k=0), 1),
    (dict(k=1 << 18), 2), (dict(y_dtype=3), 1), (dict(reserved=1), 1), (dict(offsets=None), 1), (dict(x=None), 1),
    (dict(x_scales=None), 1), (dict(w=None), 1), (dict(w_scales=None), 1), (dict(y=None), 1), (dict(x_rows=7), 1),
    (dict(x_rows=0, row_index=BASE), 1), (dict(w_up=BASE), 1), (dict(w_up=BASE + 8, w_up_scales=BASE), 1),
    (dict(rows=4096, row_index=BASE), 1), (dict(rows=4096, row_index=BASE, workspace=BASE, workspace_bytes=64), 1),
    (dict(rows=4096, row_index=BASE, workspace=BASE + 8, workspace_bytes=1 << 30), 1),
    (dict(ldx=63), 1), (dict(ldw=65), 1), (dict(ldy=16), 1), (dict(x=BASE + 1), 1)])
def test_grouped_linear_w8a8_refuses(wrong, code):
    assert _grouped(**wrong) == code
    assert M.lib().uocr_last_error().decode().startswith("grouped_linear_w8a8: ")


def test_grouped_linear_w8a8_of_nothing():
    assert _grouped(rows=0, x=None, y=None) == 0
    assert _grouped(n=0, w=None, y=None) == 0
    assert _grouped(groups=0) == 0
    assert M.lib().uocr_grouped_linear_w8a8(None, None) == 1


def test_grouped_w8a8_workspace():
    need = ctypes.c_int64(-1)

    def ask(**kw):
        a = dict(rows=4096, k=100, row_index=BASE, groups=4)
        a.update(kw)
        return M.lib().uocr_grouped_w8a8_workspace(ctypes.byref(M.GroupedW8A8Args(**a)), ctypes.byref(need))
    assert ask() == 0 and need.value == 4096 * 112
    assert ask(row_index=None) == 0 and need.value == 0
    assert ask(k=0) == 1 and ask(rows=-1) == 1 and ask(k=1 << 20) == 1
    assert M.lib().uocr_grouped_w8a8_workspace(None, None) == 1


def test_binding_refuses_wrong_tensors():
    """The binding checks what the C call cannot see: types, shapes and where the tensors are."""
    import torch
    x, s = torch.zeros(2, 16, dtype=torch.int8), torch.ones(2)
    with pytest.raises(ValueError):  # not on the GPU
        M.linear_w8a8(x, s, x, s, torch.zeros(2, 2))
    with pytest.raises(ValueError):
        M.quantize_tokens(torch.zeros(2, 16, dtype=torch.float16), x, s)


def test_cpp_wrapper(tmp_path):
    """The header-only C++ layer's int8 functions: the library's refusals as std::invalid_argument."""
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    src = tmp_path / "int8.cpp"
    src.write_text(r"""
#include <cstdio>
#include "uocr_moe.hpp"
template <typename F> static int throws(F&& f) {
  try { f(); } catch (const std::invalid_argument&) { return 1; }
  return 0;
}
int main() {
  uocr_linear_w8a8_args l{};
  l.m = l.n = 1;
  uocr_grouped_w8a8_args g{};
  g.rows = 4096, g.n = 1, g.k = 100, g.groups = 4, g.row_index = reinterpret_cast<const int32_t*>(16);
  std::printf("%d %d %d %lld\n", throws([&] { uocr_b200::linear_w8a8(nullptr, l); }),
              throws([&] { uocr_b200::grouped_linear_w8a8(nullptr, g); }),
              throws([&] { uocr_b200::quantize_tokens(nullptr, nullptr, UOCR_DTYPE_I32, 1, 1, 1, nullptr, 16, nullptr); }),
              static_cast<long long>(uocr_b200::grouped_w8a8_workspace(g)));
}
""")
    exe = tmp_path / "int8"
    lib = os.path.dirname(M.LIB_PATH)
    subprocess.run([cxx, "-std=c++17", "-I", INCLUDE, str(src), "-o", str(exe), M.LIB_PATH, f"-Wl,-rpath,{lib}"], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()
    assert out == ["1", "1", "1", str(4096 * 112)]


def test_int8_activations_need_int8_weights():
    plan = M.MoeDesc(256, 8, 2, 128, 128, 1, 32, M.WEIGHT_BF16, 1, 0, 0, M.PLAN_INT8_ACTIVATIONS)
    h = ctypes.c_void_p()
    assert M.lib().uocr_moe_plan_create(ctypes.byref(plan), ctypes.byref(h)) == 1 and not h.value
    assert "int8 weights" in M.lib().uocr_last_error().decode()
    dec = M.DecoderDesc(512, 1, 4, 1, 128, 256, 64, 32, 8, 2, 128, 256, 1e4, 1e-6, M.WEIGHT_BF16, 1, 0,
                        M.DECODER_INT8_ACTIVATIONS)
    assert M.lib().uocr_decoder_create(ctypes.byref(dec), ctypes.byref(h)) == 1 and not h.value
    assert "int8 weights" in M.lib().uocr_last_error().decode()
