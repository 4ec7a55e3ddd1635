"""The 4-bit tile kernels in the generated gfx950 code and their LDS layout: no GPU.

Their LDS DMA comes from inline assembly, as the bf16 GEMM's does, and their waits count on the epilogue's stores:
a stage's wait leaves that many younger operations outstanding, so each must be there.  The layout model evaluates
the slot expressions and checks that every chunk is where a fragment read looks for it, and that each pass of a
ds_read_b128 touches distinct banks.
"""

import re
from pathlib import Path

import pytest
from test_asm_hazards import HIPCC, ROOT, _assembly, _kernels, dma_hazards, early_uses

SRC = ROOT / "parallel_amd" / "csrc" / "mx4_tile.hip"
needs_hipcc = pytest.mark.skipif(not Path(HIPCC).exists(), reason="hipcc not available")


@needs_hipcc
def test_dma_has_its_wait_states_and_no_register_is_touched_early():
    lines = _assembly(SRC)
    assert sum(1 for l in lines if l.strip().startswith("buffer_load") and l.strip().endswith(" lds")) > 0
    assert not dma_hazards(lines)
    for name, start, end in _kernels(lines):
        assert not early_uses(lines[start:end]), name


@needs_hipcc
def test_every_epilogue_issues_the_stores_that_the_waits_count():
    text = "\n".join(_assembly(SRC))
    seen = 0
    for m in re.finditer(r"^(_Z\w*mx4_tile_kernelILi(\d+)ELi(\d+)ELi(\d+)E\w*):.*?^\.Lfunc_end", text, re.M | re.S):
        rows, epi = int(m.group(2)), int(m.group(4))
        per = {0: 2, 1: 1, 2: 2, 3: 4}[epi]  # bf16, act bf16, act mx4 (codes and scales), f32: per 16-row tile of a wave
        stores = len(re.findall(r"^\s*buffer_store_(?:dwordx4|dword|byte)\b", m.group(0), re.M))
        spills = len(re.findall(r"^\s*scratch_store", m.group(0), re.M))
        assert stores == per * rows // 32, (m.group(1), stores, spills)
        seen += 1
    assert seen == 12  # three tile heights, four outputs


def guarded(lines, wanted):
    """Lines that match ``wanted`` between a branch on an empty exec mask and its forward target: a wave whose lanes
    all take the other side would not issue them."""
    labels = {m.group(1): n for n, l in enumerate(lines) if (m := re.match(r"^(\.LBB\w+):", l))}
    found = []
    for n, line in enumerate(lines):
        m = re.match(r"\s*s_cbranch_execz (\.LBB\w+)", line)
        if m and labels.get(m.group(1), -1) > n:
            found += [l.strip() for l in lines[n:labels[m.group(1)]] if re.match(wanted, l)]
    return found


def test_scanner_flags_a_guarded_store():
    lines = ["  s_cbranch_execz .LBB1_2", "  buffer_store_dword v1, v2, s[0:3], 0 offen", ".LBB1_2:",
             "  buffer_store_dword v1, v2, s[0:3], 0 offen"]
    assert len(guarded(lines, r"\s*buffer_store")) == 1


@needs_hipcc
def test_no_counted_operation_depends_on_the_lanes():
    lines = _assembly(SRC)
    for name, start, end in _kernels(lines):
        assert not guarded(lines[start:end], r"\s*(buffer_store|buffer_load\w* .* lds$)"), name


def chunk_at(slot, key):
    x = slot ^ key
    return (x & 3) << 1 | x >> 2


@pytest.mark.parametrize("operand", ["a", "b"])
def test_fragment_reads_find_their_chunks_on_distinct_banks(operand):
    key = (lambda r: (r >> 1) & 7) if operand == "a" else (lambda r: ((r >> 1) & 1) | ((r >> 4) & 3) << 1)
    # rows of the lanes of one fragment: 16 neighbours, or rows 16 a + 4 j + b of 64
    fragments = [list(range(16))] if operand == "a" else [[16 * (i >> 2) + 4 * j + (i & 3) for i in range(16)]
                                                         for j in range(4)]
    holds = {(r, chunk_at(slot, key(r))): r * 128 + 16 * slot for r in range(64) for slot in range(8)}
    for rows in fragments:
        for s in range(2):
            at = {}
            for lane in range(64):
                i, q = lane & 15, lane >> 4
                at[lane] = rows[i] * 128 + (((4 * s + q) ^ (i >> 1)) << 4)
                assert at[lane] == holds[rows[i], 2 * q + s]  # 32-block 2 q + s of the row's eight
            first = list(range(0, 4)) + list(range(12, 16)) + list(range(20, 28))
            for half in (0, 32):
                for lanes in (first, [l for l in range(32) if l not in first]):
                    banks = {(at[half + l] // 4 + d) % 64 for l in lanes for d in range(4)}
                    assert len(banks) == 64
