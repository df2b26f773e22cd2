"""The operators for sequences that share a page, without a GPU: the header and
the binding agree, the rotary tables have their formulas' values, and bad
arguments are refused before a device is touched."""
import ctypes
import math
import os
import re
import shutil
import subprocess

import pytest

import uocr_moe as M

INCLUDE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
HEADER = os.path.join(INCLUDE, "uocr_beam.h")
BASE = 1 << 20  # an aligned address that is never read
BIG = 1 << 40   # bytes of a workspace that is never read


def test_header_and_binding_agree():
    names = re.findall(r"^int (uocr_[a-z_0-9]+)\s*\(", open(HEADER).read(), re.M)
    assert sorted(names) == sorted(M.BEAM_EXPORTS)
    for name in names:
        assert hasattr(M.lib(), name), name


def test_struct_layouts_match_the_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    structs = {"uocr_rotate_heads_args": M.RotateHeadsArgs, "uocr_prefix_attention_args": M.PrefixAttentionArgs,
               "uocr_beam_select_args": M.BeamSelectArgs, "uocr_reorder_states_args": M.ReorderStatesArgs,
               "uocr_beam_search_args": M.BeamSearchArgs}
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "uocr_beam.h"', "int main(void) {"]
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


# ---- rotary tables

def test_rope_frequencies_plain_and_linear():
    table, magnitude = M.rope_frequencies(128, 1e4)
    want = [1e4 ** (-i / 64) for i in range(64)]
    assert magnitude == 1.0 and all(abs(a - b) <= 2.0 ** -24 * b for a, b in zip(table.tolist(), want))
    table, _ = M.rope_frequencies(32, 5e5, M.ROPE_LINEAR, 8.0)
    want = [5e5 ** (-i / 16) / 8 for i in range(16)]
    assert all(abs(a - b) <= 2.0 ** -23 * b for a, b in zip(table.tolist(), want))


def test_rope_frequencies_ntk_keeps_the_highest_and_divides_the_lowest():
    plain, _ = M.rope_frequencies(64, 1e4)
    table, magnitude = M.rope_frequencies(64, 1e4, M.ROPE_NTK, 4.0)
    ratio = (plain / table).tolist()
    assert magnitude == 1.0 and ratio[0] == 1.0 and abs(ratio[-1] - 4.0) < 1e-5
    assert all(a < b for a, b in zip(ratio, ratio[1:]))


def test_rope_frequencies_yarn():
    plain, _ = M.rope_frequencies(128, 1e4)
    table, magnitude = M.rope_frequencies(128, 1e4, M.ROPE_YARN, 16.0, 4096)
    assert abs(magnitude - (0.1 * math.log(16.0) + 1.0)) < 1e-6
    for f, g in zip(plain.tolist(), table.tolist()):
        turns = 4096 * f / (2 * math.pi)
        if turns >= 40:
            assert f == g
        elif turns <= 0.8:
            assert abs(f / g - 16.0) < 1e-4
        else:
            assert 1.0 - 1e-6 <= f / g <= 16.0 + 1e-4
    same, one = M.rope_frequencies(128, 1e4, M.ROPE_YARN, 1.0, 4096)
    assert one == 1.0 and all(abs(a - b) <= 2.0 ** -23 * a for a, b in zip(plain.tolist(), same.tolist()))


@pytest.mark.parametrize("wrong", [dict(rotary_dim=0), dict(rotary_dim=7), dict(theta=1.0), dict(theta=math.inf),
                                   dict(theta=math.nan), dict(scaling=4), dict(scaling=-1), dict(factor=0.5),
                                   dict(factor=math.nan), dict(scaling=M.ROPE_YARN),
                                   dict(scaling=M.ROPE_NTK, rotary_dim=2)])
def test_rope_frequencies_refuses(wrong):
    a = dict(rotary_dim=64, theta=1e4, scaling=0, factor=2.0, original=0)
    a.update(wrong)
    out = (ctypes.c_float * 64)()
    assert M.lib().uocr_rope_frequencies(a["rotary_dim"], a["theta"], a["scaling"], a["factor"], a["original"],
                                         ctypes.addressof(out), None) == 1
    assert M.lib().uocr_last_error().decode().startswith("rope_frequencies: ")


# ---- refusals

def _call(fn, cls, defaults, wrong):
    a = dict(defaults)
    a.update(wrong)
    return getattr(M.lib(), fn)(ctypes.byref(cls(**a)), None)


ROTATE = dict(q=BASE, k=BASE, v=BASE, q_norm=None, k_norm=None, inv_freq=BASE, positions=BASE, cache_rows=None,
              slots=None, q_out=BASE, k_cache=BASE, v_cache=BASE, rows=4, q_heads=4, kv_heads=2, head_dim=64,
              rotary_dim=64, ldq=256, ldk=128, ldv=128, ldqo=256, caches=4, capacity=16, cache_stride=2048,
              head_stride=1024, eps=1e-6, magnitude=1.0, dtype=0, interleaved=0)


@pytest.mark.parametrize("wrong,code", [
    (dict(rows=-1), 1), (dict(rows=1 << 31), 1), (dict(q_heads=-1), 1), (dict(kv_heads=-1), 1), (dict(head_dim=60), 2),
    (dict(head_dim=264), 2), (dict(head_dim=0), 2), (dict(rotary_dim=12), 2), (dict(rotary_dim=72), 2),
    (dict(rotary_dim=-8), 2), (dict(dtype=2), 1), (dict(interleaved=2), 1), (dict(q=None), 1), (dict(q_out=None), 1),
    (dict(k=None), 1), (dict(v=None), 1), (dict(k_cache=None), 1), (dict(v_cache=None), 1), (dict(positions=None), 1),
    (dict(inv_freq=None), 1), (dict(ldq=255), 1), (dict(ldqo=255), 1), (dict(ldk=127), 1), (dict(ldv=127), 1),
    (dict(q=BASE + 2), 1), (dict(q_out=BASE + 1), 1), (dict(k=BASE + 1), 1), (dict(caches=0), 1), (dict(capacity=0), 1),
    (dict(k_cache=BASE + 8), 1), (dict(cache_stride=2052), 1), (dict(head_stride=1028), 1), (dict(head_stride=-1024), 1),
    (dict(dtype=1, q_out=BASE, ldqo=264), 1), (dict(head_stride=512, cache_stride=512), 1)])
def test_rotate_heads_refuses(wrong, code):
    base = dict(ROTATE, q_out=BASE + 4096)
    assert _call("uocr_rotate_heads", M.RotateHeadsArgs, base, wrong) == code
    assert M.lib().uocr_last_error().decode().startswith("rotate_heads: ")


def test_rotate_heads_of_nothing():
    assert _call("uocr_rotate_heads", M.RotateHeadsArgs, ROTATE, dict(rows=0, q=None, k=None, positions=None)) == 0
    assert _call("uocr_rotate_heads", M.RotateHeadsArgs, ROTATE, dict(q_heads=0, kv_heads=0)) == 0


ATTENTION = dict(q=BASE, prefix_k=BASE, prefix_v=BASE, prefix_lens=BASE, k=BASE, v=BASE, lens=BASE, ancestry=None,
                 row_offsets=None, out=BASE, lse=None, rows=6, sequences=6, prefixes=2, caches=6, heads=4, kv_heads=2,
                 head_dim=128, prefix_capacity=100, capacity=20, ldq=512, ldo=512, ld_ancestry=0, prefix_stride=25600,
                 prefix_head_stride=12800, cache_stride=5120, head_stride=2560, scale=0.1, reserved=0, workspace=BASE,
                 workspace_bytes=BIG)


@pytest.mark.parametrize("wrong,code", [
    (dict(rows=-1), 1), (dict(rows=5), 1), (dict(sequences=-1), 1), (dict(prefixes=0), 1), (dict(prefixes=4), 1),
    (dict(heads=0), 1), (dict(heads=5), 1), (dict(kv_heads=0), 1), (dict(head_dim=96), 2), (dict(reserved=1), 1),
    (dict(prefix_capacity=-1), 1), (dict(capacity=1 << 31), 1), (dict(q=None), 1), (dict(out=None), 1),
    (dict(prefix_lens=None), 1), (dict(lens=None), 1), (dict(prefix_k=None), 1), (dict(prefix_v=None), 1),
    (dict(k=None), 1), (dict(v=None), 1), (dict(caches=5), 1), (dict(caches=0), 1), (dict(ldq=504), 1),
    (dict(ldq=516), 1), (dict(q=BASE + 8), 1), (dict(out=BASE + 8), 1), (dict(ldo=500), 1), (dict(prefix_k=BASE + 2), 1),
    (dict(prefix_stride=25601), 1), (dict(head_stride=2564), 1), (dict(scale=math.inf), 1), (dict(scale=math.nan), 1),
    (dict(ancestry=BASE, ld_ancestry=19), 1), (dict(workspace=None), 1), (dict(workspace=BASE + 8), 1),
    (dict(workspace_bytes=1000), 1)])
def test_prefix_attention_refuses(wrong, code):
    assert _call("uocr_prefix_attention", M.PrefixAttentionArgs, ATTENTION, wrong) == code
    assert M.lib().uocr_last_error().decode().startswith("prefix_attention: ")


def test_prefix_attention_workspace_grows_with_the_rows():
    def need(**kw):
        out = ctypes.c_int64(-1)
        a = dict(ATTENTION)
        a.update(kw)
        assert M.lib().uocr_prefix_attention_workspace(ctypes.byref(M.PrefixAttentionArgs(**a)), ctypes.byref(out)) == 0
        return out.value
    assert need(rows=0, sequences=0) == 0 and need() > 0
    assert need(rows=600, sequences=6, row_offsets=BASE) >= need()
    assert _call("uocr_prefix_attention", M.PrefixAttentionArgs, ATTENTION, dict(rows=0, sequences=0, q=None)) == 0


SELECT = dict(logits=BASE, scores=BASE, finished=None, tokens=BASE, parents=BASE, new_scores=BASE + 4096,
              new_finished=None, batch=2, beams=4, select=4, vocab=1000, ld_logits=1000, dtype=0, eos=-1,
              workspace=BASE, workspace_bytes=BIG)


@pytest.mark.parametrize("wrong,code", [
    (dict(batch=-1), 1), (dict(vocab=0), 1), (dict(beams=0), 1), (dict(beams=33), 1), (dict(select=0), 1),
    (dict(select=33), 1), (dict(vocab=(1 << 20) + 1, ld_logits=1 << 21), 2), (dict(batch=1 << 30), 2), (dict(dtype=2), 1),
    (dict(eos=-2), 1), (dict(eos=1000), 1), (dict(logits=None), 1), (dict(scores=None), 1), (dict(tokens=None), 1),
    (dict(parents=None), 1), (dict(new_scores=None), 1), (dict(ld_logits=999), 1), (dict(logits=BASE + 2), 1),
    (dict(new_scores=BASE), 1), (dict(finished=BASE, new_finished=BASE), 1), (dict(workspace=None), 1),
    (dict(workspace=BASE + 4), 1), (dict(workspace_bytes=8), 1)])
def test_beam_select_refuses(wrong, code):
    assert _call("uocr_beam_select", M.BeamSelectArgs, SELECT, wrong) == code
    assert M.lib().uocr_last_error().decode().startswith("beam_select: ")


def test_beam_select_of_nothing():
    assert _call("uocr_beam_select", M.BeamSelectArgs, SELECT, dict(batch=0, logits=None)) == 0


REORDER = dict(state=BASE, parents=BASE, counts=None, layers=2, groups=3, beams=4, segments=2, units=8, unit_bytes=16,
               layer_stride=4096, row_stride=256, segment_stride=128)


@pytest.mark.parametrize("wrong,code", [
    (dict(layers=-1), 1), (dict(groups=-1), 1), (dict(beams=0), 1), (dict(beams=33), 1), (dict(segments=-1), 1),
    (dict(units=-1), 1), (dict(unit_bytes=0), 1), (dict(state=None), 1), (dict(parents=None), 1),
    (dict(row_stride=127), 1), (dict(segment_stride=64), 1), (dict(layer_stride=100), 1),
    (dict(groups=1 << 29), 2), (dict(layers=1 << 30, groups=1 << 20), 2)])
def test_reorder_states_refuses(wrong, code):
    assert _call("uocr_reorder_states", M.ReorderStatesArgs, REORDER, wrong) == code
    assert M.lib().uocr_last_error().decode().startswith("reorder_states: ")


def test_reorder_states_of_nothing():
    for none in (dict(layers=0), dict(groups=0), dict(segments=0), dict(units=0)):
        assert _call("uocr_reorder_states", M.ReorderStatesArgs, REORDER, dict(none, state=None)) == 0


@pytest.mark.parametrize("name", ["rotate_heads", "prefix_attention", "prefix_attention_workspace", "beam_select",
                                  "beam_select_workspace", "reorder_states"])
def test_null_arguments_are_refused(name):
    assert getattr(M.lib(), "uocr_" + name)(None, None) == 1


def test_binding_refuses_tensors_off_the_gpu():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a current device to compare with")
    with pytest.raises(ValueError):
        M.reorder_states(torch.zeros(4, 4), torch.zeros(4, dtype=torch.int32), 4)


def test_beam_search_refuses_before_a_decoder_is_touched():
    out = ctypes.c_int64()
    assert M.lib().uocr_decoder_beam_workspace(None, 4, 8, ctypes.byref(out)) == 1
    assert M.lib().uocr_decoder_beam_search(None, None, None) == 1
    args = M.BeamSearchArgs(4, 8, -1, 0, BASE, BASE, None, BASE, BIG)
    assert M.lib().uocr_decoder_beam_search(None, ctypes.byref(args), None) == 1
    assert M.lib().uocr_last_error().decode().startswith("decoder_beam_search: ")


def test_cpp_wrapper(tmp_path):
    """The header-only C++ layer's functions: values through it, the library's refusals as std::invalid_argument."""
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    src = tmp_path / "beam.cpp"
    src.write_text(r"""
#include <cstdio>
#include "uocr_moe.hpp"
template <typename F> static int throws(F&& f) {
  try { f(); } catch (const std::invalid_argument&) { return 1; }
  return 0;
}
int main() {
  float table[32];
  const float magnitude = uocr_b200::rope_frequencies(64, 1e4, UOCR_ROPE_YARN, 4.0, 4096, table);
  uocr_rotate_heads_args r{};
  r.rows = 1, r.q_heads = 1, r.head_dim = 7;
  uocr_prefix_attention_args a{};
  a.rows = -1;
  uocr_beam_select_args s{};
  s.batch = 1, s.beams = 33;
  uocr_reorder_states_args o{};
  o.layers = 1, o.groups = 1, o.beams = 33;
  std::printf("%d %d %d %d %d %d %.6f\n", throws([&] { uocr_b200::rotate_heads(nullptr, r); }),
              throws([&] { uocr_b200::prefix_attention(nullptr, a); }),
              throws([&] { uocr_b200::prefix_attention_workspace(a); }),
              throws([&] { uocr_b200::beam_select(nullptr, s); }),
              throws([&] { uocr_b200::beam_select_workspace(s); }),
              throws([&] { uocr_b200::reorder_states(nullptr, o); }), magnitude);
}
""")
    exe = tmp_path / "beam"
    lib = os.path.dirname(M.LIB_PATH)
    subprocess.run([cxx, "-std=c++17", "-I", INCLUDE, str(src), "-o", str(exe), M.LIB_PATH, f"-Wl,-rpath,{lib}"], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()
    assert out[:6] == ["1"] * 6 and abs(float(out[6]) - (0.1 * math.log(4.0) + 1)) < 1e-6


@pytest.mark.parametrize("wrong", [
    dict(head_stride=0), dict(head_stride=512), dict(head_stride=1016), dict(cache_stride=0), dict(cache_stride=1024),
    dict(cache_stride=2040), dict(kv_heads=1, cache_stride=1016), dict(caches=1, cache_stride=0, head_stride=1016),
    dict(head_stride=4096, cache_stride=1016), dict(head_stride=4088, cache_stride=1024)])
def test_rotate_heads_refuses_caches_that_overlap(wrong):
    """Each stride alone, in both orders of caches and heads: the caches are written."""
    base = dict(ROTATE, q_out=BASE + 4096)
    assert _call("uocr_rotate_heads", M.RotateHeadsArgs, base, wrong) == 1
    assert "overlap" in M.lib().uocr_last_error().decode()


@pytest.mark.parametrize("right", [dict(), dict(caches=1, cache_stride=0), dict(kv_heads=1, head_stride=0),
                                   dict(head_stride=4096, cache_stride=1024), dict(head_stride=1 << 40, cache_stride=1 << 30)])
def test_rotate_heads_takes_caches_that_lie_apart(right):
    """The first check behind the overlap's is the device's, which this machine may not have."""
    base = dict(ROTATE, q_out=BASE + 4096)
    import torch
    if torch.cuda.is_available():
        pytest.skip("the addresses are none of a device's")
    _call("uocr_rotate_heads", M.RotateHeadsArgs, base, right)
    assert "overlap" not in M.lib().uocr_last_error().decode()


@pytest.mark.parametrize("wrong", [
    dict(row_stride=128), dict(row_stride=255), dict(segment_stride=256), dict(layer_stride=3071), dict(layer_stride=128),
    dict(segment_stride=256, row_stride=256), dict(layers=1, groups=1, beams=2, segments=3, row_stride=300),
    dict(segments=1, layer_stride=1024), dict(layer_stride=256, row_stride=511)])
def test_reorder_states_refuses_rows_that_overlap(wrong):
    assert _call("uocr_reorder_states", M.ReorderStatesArgs, REORDER, wrong) == 1
    assert "overlap" in M.lib().uocr_last_error().decode()


@pytest.mark.parametrize("right", [
    dict(), dict(layer_stride=3072), dict(layer_stride=256, row_stride=512), dict(segment_stride=1536, row_stride=128),
    dict(layers=1, layer_stride=0), dict(segments=1, segment_stride=0, row_stride=128), dict(beams=1, groups=1, row_stride=0)])
def test_reorder_states_takes_any_order_of_layers_rows_and_segments(right):
    import torch
    if torch.cuda.is_available():
        pytest.skip("the addresses are none of a device's")
    _call("uocr_reorder_states", M.ReorderStatesArgs, REORDER, right)
    error = M.lib().uocr_last_error().decode()
    assert "overlap" not in error and "segment" not in error


def test_prefix_attention_workspace_depends_on_sizes_alone():
    """A query before scale, pitches and strides are set says what the call will need."""
    def need(**kw):
        out = ctypes.c_int64(-1)
        a = dict(ATTENTION)
        a.update(kw)
        assert M.lib().uocr_prefix_attention_workspace(ctypes.byref(M.PrefixAttentionArgs(**a)), ctypes.byref(out)) == 0
        return out.value
    unset = dict(scale=0.0, ldq=0, ldo=0, ld_ancestry=0, prefix_stride=0, prefix_head_stride=0, cache_stride=0, head_stride=0)
    for rows, sequences, prefixes, heads, kv in ((6, 6, 2, 4, 2), (40, 40, 1, 16, 4), (200, 4, 1, 8, 2), (700, 140, 70, 4, 4),
                                                 (6000, 24, 1, 16, 4), (128, 128, 16, 16, 4)):
        for keys, own in ((100, 20), (4096, 300), (33000, 2000), (70, 0), (0, 20)):
            sizes = dict(rows=rows, sequences=sequences, prefixes=prefixes, caches=sequences, heads=heads, kv_heads=kv,
                         prefix_capacity=keys, capacity=own, row_offsets=None if rows == sequences else BASE)
            assert need(**sizes) == need(**sizes, **unset), sizes
            assert need(**sizes) == need(**sizes, **dict(unset, scale=0.125))
            assert need(**sizes) == need(**sizes, **dict(unset, prefix_stride=keys * 1024, prefix_head_stride=keys * 128))
