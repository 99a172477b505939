"""gplk_moe_cfg as Python passes it is the struct of include/gplk.h."""
from __future__ import annotations

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parent.parent


def test_packed_bytes_are_the_ctypes_structure(gplk):
    """The layer's wrapper packs the bytes of a MoeCfg instead of building one."""
    values = [(i + 1) * 0x01010101 for i in range(len(gplk.MoeCfg._fields_))]
    assert gplk._moe_cfg(*values) == bytes(gplk.MoeCfg(*values))


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_structure_is_the_header_s(gplk, tmp_path):
    names = [n for n, _ in gplk.MoeCfg._fields_]
    src = tmp_path / "cfg.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "gplk.h"\nint main(void) {\n'
                   '    printf("%zu\\n", sizeof(gplk_moe_cfg));\n'
                   + "".join(f'    printf("%zu %zu\\n", offsetof(gplk_moe_cfg, {n}), sizeof(((gplk_moe_cfg *)0)->{n}));\n'
                             for n in names) + "    return 0;\n}\n")
    subprocess.run(["gcc", "-I/usr/local/cuda/include", f"-I{REPO / 'include'}", "-o", str(tmp_path / "cfg"), str(src)],
                   check=True)
    size, *fields = subprocess.run([str(tmp_path / "cfg")], check=True, capture_output=True, text=True).stdout.splitlines()
    assert int(size) == ctypes.sizeof(gplk.MoeCfg)
    for name, line in zip(names, fields, strict=True):
        field = getattr(gplk.MoeCfg, name)
        assert [int(v) for v in line.split()] == [field.offset, field.size], name


def test_workspace_sizes_beyond_32_bits(gplk):
    """ctypes cuts what a C int cannot hold: such sizes are refused, not cut."""
    assert gplk.gemv_nvfp4_workspace_bytes(16, (1 << 32) + 8192, 8192) == 0
    assert gplk.moe_nvfp4_workspace_bytes(2, 8, 2, (1 << 32) + 256, 128) == 0
