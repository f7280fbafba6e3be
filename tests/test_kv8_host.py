"""8-bit KV states and drafted trees without a GPU: byte order and plans,
descriptors, sizes, masks, and every refusal. The refusals run against an
arena object with no device behind it: a refused call has to end before it
asks for one."""
from __future__ import annotations

import ctypes
import pathlib
import shutil
import subprocess

import numpy as np
import pytest

from kv8_cases import refusals
from kv8_util import held
from synapse_amd import capi

ROOT = pathlib.Path(__file__).resolve().parent.parent


def test_byte_order_and_plans():
    exe = ROOT / "tests" / "cpp" / "_bin" / "test_attend_rows_plan"
    assert exe.exists(), "build it with `python -m synapse_amd.build`"
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]


def test_descriptor_layouts_match_the_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no host C compiler")
    structs = {"syn_kv8_desc": capi.Kv8Desc, "syn_kv8_attn_desc": capi.Kv8AttnDesc}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{ROOT / "include" / "synapse_hip.h"}"',
             "int main(void) {"]
    for cname, ct in structs.items():
        lines.append(f'printf("{cname} @sizeof %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in ct._fields_]
    (tmp_path / "layout.c").write_text("\n".join([*lines, "return 0;", "}"]))
    subprocess.run([cc, "-std=c11", "-o", str(tmp_path / "layout"), str(tmp_path / "layout.c")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    got = dict(line.rsplit(" ", 1) for line in out.splitlines())
    for cname, ct in structs.items():
        assert int(got[f"{cname} @sizeof"]) == ctypes.sizeof(ct)
        for f, _ in ct._fields_:
            assert int(got[f"{cname} {f}"]) == getattr(ct, f).offset, (cname, f)


def test_state_bytes():
    # 64-position tiles of 64 x (hd rounded up to 32) bytes twice and 128 steps, per head.
    tile = 2 * 64 * 128 + 2 * 64 * 4
    assert capi.kv8_state_bytes(4096, 8, 128) == 8 * 64 * tile
    assert capi.kv8_state_bytes(4097, 8, 128) == 8 * 65 * tile
    assert capi.kv8_state_bytes(1, 1, 2) == 64 * 32 * 2 + 512
    assert capi.kv8_state_bytes(8192, 8, 128) < 0.52 * capi.kv_state_bytes(8192, 8, 128)
    for shape in [(0, 8, 128), (16, 0, 128), (16, 8, 0), (16, 8, 258), (16, 8, 7), (0x7fffffff, 8, 128)]:
        assert capi.kv8_state_bytes(*shape) == 0


def test_scratch_bytes():
    lib = capi.lib()
    for fn in (lib.syn_hip_kv8_attention_scratch_bytes, lib.syn_hip_attend_tree_scratch_bytes):
        assert fn(30, 8, 128, 4096, 1) == 0
        assert fn(32, 0, 128, 4096, 1) == 0
        assert fn(32, 8, 128, 64, 1) == 0  # one split
        assert fn(32, 8, 128, 4096, 1) > 0
        assert fn(32, 8, 128, 8192, 64) >= fn(32, 8, 128, 8192, 8) >= fn(32, 8, 128, 4096, 8)


def test_tree_mask():
    m = capi.tree_mask([-1, 0, 0, 1, -1, 3])
    assert m.shape == (6, 1) and m[:, 0].tolist() == [1, 3, 5, 11, 16, 43]
    wide = capi.tree_mask(list(range(-1, 39)))
    assert wide.shape == (40, 2) and wide[39].tolist() == [0xffffffff, 0xff]
    for bad in ([0], [-1, 1], [-2]):
        with pytest.raises(ValueError):
            capi.tree_mask(bad)


def test_the_oracle_rounds_quotients_exactly():
    """held() against whole-number arithmetic: q is nearest to x / d."""
    from fractions import Fraction

    g = np.random.default_rng(3)
    x = (g.standard_normal((40, 8)) * 10.0 ** g.integers(-30, 30, (40, 1))).astype(np.float32)
    q, d = held(x)
    for i in range(40):
        for j in range(8):
            r = Fraction(float(x[i, j])) / Fraction(float(d[i]))
            assert abs(r - int(q[i, j])) <= Fraction(1, 2), (i, j)


class _Arena(ctypes.Structure):  # the library's arena object: base, bytes, stream, device
    _fields_ = [("base", ctypes.c_void_p), ("bytes", ctypes.c_size_t), ("stream", ctypes.c_void_p),
                ("device", ctypes.c_int)]


@pytest.mark.parametrize("name,code,call", refusals(), ids=lambda x: x if isinstance(x, str) else "")
def test_refusals(name, code, call):
    arena = _Arena(base=256, bytes=32 << 20, stream=None, device=0)
    assert call(ctypes.addressof(arena)) == code, (name, capi.lib().syn_hip_last_error())
    assert capi.lib().syn_hip_last_error()


def test_no_rows_is_no_work():
    arena = _Arena(base=256, bytes=32 << 20, stream=None, device=0)
    c = capi.Kv8Desc(offset=0, max_ctx=100, n_kv_heads=2, head_dim=64)
    c16 = capi.KvDesc(k_offset=0, v_offset=1 << 20, max_ctx=100, n_kv_heads=2, head_dim=64, ctx_stride=128)
    L, a = capi.lib(), ctypes.addressof(arena)
    assert L.syn_hip_kv8_append(a, ctypes.byref(c), 0, 0, 0, 100, 0) == 0
    assert L.syn_hip_kv8_read(a, ctypes.byref(c), 0, 0, 0, 100, 0) == 0
    rows = (ctypes.c_uint32 * 3)(0, 1, 2)
    for fn, d in ((L.syn_hip_kv8_keep, c), (L.syn_hip_kv_keep, c16)):
        assert fn(a, ctypes.byref(d), 5, 9, None, 0) == 0
        assert fn(a, ctypes.byref(d), 5, 9, rows, 3) == 0  # in place already
