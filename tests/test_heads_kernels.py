"""The kernels between projections and cache, and those that move pages, as the compiler made them (gfx950, no GPU): no
register spills, no packed fp32 arithmetic, wait states around the row swaps written as asm; and the level table of the
append against the format's midpoints."""
import os
import re

import numpy as np
import pytest

import cabi
from test_kernel_resources import CSRC, asm_mfma_hazards, compile_device, kernel_bodies


@pytest.mark.slow
@pytest.mark.parametrize("src", ["sjk_heads.hip", "sjk_pages.hip"])
def test_no_scratch_no_packed_fp32_no_hazards(src):
    remarks, asm = compile_device(src)
    names = re.findall(r"Function Name: (\S+)", remarks)
    scratch = [int(x) for x in re.findall(r"ScratchSize \[bytes/lane\]: (\d+)", remarks)]
    assert len(names) == len(scratch) > 0
    assert not [n for n, s in zip(names, scratch) if s], "register spills"
    assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", asm)
    bad = {n: asm_mfma_hazards(lines) for n, lines in kernel_bodies(asm).items()}
    assert not {n: b for n, b in bad.items() if b}


def test_level_table_against_the_midpoints():
    """the cell a value falls in and one comparison give the level of a search over all midpoints: for every midpoint, the
    floats next to it, the cells' own borders and values over the whole range"""
    text = open(os.path.join(CSRC, "sjk_heads.hip")).read()
    cells = int(re.search(r"LV_CELLS = (\d+);", text).group(1))
    scale = np.float32(re.search(r"LV_SCALE = ([\d.]+)f;", text).group(1))
    offset = np.float32(re.search(r"v \* LV_SCALE \+ ([\d.]+)f", text).group(1))
    tables = open(os.path.join(cabi.ROOT, "include", "sjk_tables.h")).read().replace("\\\n", " ")
    bits = re.search(r"define\s+SJK_TQ6_MIDPOINT_BITS_INIT\s*\{(.*?)\}", tables, re.S).group(1)
    mids = np.array([int(x, 0) for x in re.findall(r"0x[0-9A-Fa-f]+", bits)], np.uint32).view(np.float32)
    assert len(mids) == 63 and np.all(np.diff(mids) > 0)

    def cell(v):
        with np.errstate(over="ignore"):
            t = (v * scale).astype(np.float32) + offset
        return np.clip(t, 0, cells - 1).astype(np.int32)

    assert np.all(np.diff(cell(mids)) > 0)                   # one midpoint a cell
    base = np.array([np.sum(cell(mids) <= c) - 1 for c in range(cells)])
    mid = np.full(cells, -np.inf, np.float32)
    mid[cell(mids)] = mids
    v = [mids, np.linspace(-1, 1, 400001).astype(np.float32), np.float32([-np.inf, np.inf, -3e38, 3e38, 0.0, -0.0, 1e-45, -1e-45])]
    edges = ((np.arange(cells + 1) - offset) / scale).astype(np.float32)
    for x in (mids, edges):
        for d in (np.float32(-np.inf), np.float32(np.inf)):
            y = x
            for _ in range(4):
                y = np.nextafter(y, d)
                v.append(y)
    v = np.concatenate(v + [edges])
    got = base[cell(v)] + (~(v < mid[cell(v)])).astype(int)
    want = np.array([np.sum(~(x < mids)) for x in v])
    assert np.array_equal(got, want)
