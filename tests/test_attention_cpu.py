"""The attention operators' host side, without a GPU: struct layouts, refusals without a handle, the rotation table."""

import ctypes
import math
import os
import subprocess

import pytest

from voxwerk_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"vw_kv_cache": _lib.VwKvCache, "vw_kv_batch": _lib.VwKvBatch, "vw_kv_prefix": _lib.VwKvPrefix,
           "vw_rope_rows": _lib.VwRopeRows, "vw_attn_rows": _lib.VwAttnRows}


def test_structs_match_the_header(tmp_path):
    lines = []
    for name, cls in STRUCTS.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"vwsampler.h\"\nint main(void) {\n"
                   + "\n".join(lines) + "\nreturn 0;\n}\n")
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, check=True).stdout
    want = {a: int(b) for a, b in (ln.split() for ln in out.splitlines())}
    for name, cls in STRUCTS.items():
        assert ctypes.sizeof(cls) == want[name]
        for f, _ in cls._fields_:
            assert getattr(cls, f).offset == want[f"{name}.{f}"], (name, f)


def test_no_handle_is_an_invalid_argument():
    lib = _lib.lib
    assert lib.vw_rope_append(None, None, None, None, None) == _lib.VW_ERR_INVALID_ARG
    assert lib.vw_prompt_attention(None, None, None, None, None) == _lib.VW_ERR_INVALID_ARG
    assert lib.vw_decode_attention(None, None, None, None, None, None) == _lib.VW_ERR_INVALID_ARG


def test_rope_angles():
    from voxwerk_b200 import RopeTable
    a, amplitude = RopeTable.angles(50, 8, base=100.0)
    assert amplitude == 1.0
    assert tuple(a.shape) == (50, 4)
    for p, i in ((0, 0), (7, 0), (49, 3), (13, 2)):
        assert math.isclose(float(a[p, i]), p * 100.0 ** (-2 * i / 8), rel_tol=1e-14)
    half, _ = RopeTable.angles(50, 8, base=100.0, linear=2.0)
    assert bool((half * 2 == a).all())


def test_yarn_angles_keep_fast_and_divide_slow_frequencies():
    from voxwerk_b200 import RopeTable
    plain, _ = RopeTable.angles(2, 128, base=1e6)
    scaled, amplitude = RopeTable.angles(2, 128, base=1e6, yarn=4.0, trained_positions=4096)
    assert math.isclose(amplitude, 0.1 * math.log(4.0) + 1.0)
    ratio = (plain[1] / scaled[1]).tolist()
    turns = (4096 * plain[1] / (2 * math.pi)).tolist()
    assert all(math.isclose(r, 1.0) for r, t in zip(ratio, turns) if t >= 32)
    assert all(math.isclose(r, 4.0) for r, t in zip(ratio, turns) if t <= 1)
    assert all(1.0 <= r <= 4.0 for r in ratio) and ratio == sorted(ratio)
    with pytest.raises(ValueError):
        RopeTable.angles(2, 128, yarn=4.0)
    with pytest.raises(ValueError):
        RopeTable.angles(2, 7)
