"""The rotary and 8-bit cache kernels on the CPU, through the emulation in tests/emu/ and under the address sanitizer:
small sizes against their definitions, and device data (offsets, places, lengths) that no host check can see."""
from __future__ import annotations

import sys
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent
sys.path.insert(0, str(HERE / "emu"))

pytestmark = pytest.mark.emu
CASES = str(HERE / "emu" / "cache8_cases.py")


def _run(case, *args):
    import session
    rc, out = session.run(CASES, case, *map(str, args))
    assert rc == 0, f"{case}{args}: exit {rc}\n{out[-4000:]}"


@pytest.mark.parametrize("d,rotated,heads,interleaved", [(128, 128, 5, False), (256, 64, 4, False), (64, 64, 2, True)])
def test_rotary(d, rotated, heads, interleaved):
    _run("rotary", d, rotated, heads, interleaved)


@pytest.mark.parametrize("seqs,lengths,rows,hq,hkv,d,fmt,capacity", [
    (3, "130/1/0", "1/1/1", 4, 2, 128, "e4m3", 192),           # whole tiles, an empty sequence
    (2, "1100/70", "3/0", 4, 2, 256, "int8", 1280),            # shares of keys, 16 rows
    (2, "1200/333", "9/5", 6, 2, 256, "e4m3", 1280),           # 32 rows
    (2, "300/75", "70/75", 4, 2, 128, "int8", 320),            # tiles of 128 rows
    (1, "1100", "45", 3, 1, 256, "e4m3", 1280),                # and shares of them
])
def test_attend(seqs, lengths, rows, hq, hkv, d, fmt, capacity):
    _run("attend", seqs, lengths, rows, hq, hkv, d, fmt, capacity)


@pytest.mark.parametrize("d,fmt", [(256, "e4m3")])
def test_offsets_that_do_not_ascend(d, fmt):
    _run("offsets_that_do_not_ascend", d, fmt)


@pytest.mark.parametrize("d,fmt", [(128, "int8")])
def test_places_and_lengths_out_of_range(d, fmt):
    _run("places_and_lengths_out_of_range", d, fmt)


@pytest.mark.parametrize("blocks,keep,sink,recent", [(70, 20, 2, 3), (5, 1, 0, 1)])
def test_evict(blocks, keep, sink, recent):
    _run("evict", blocks, keep, sink, recent)
