"""Where the block-scaled attention keeps the parts of its outputs: no words in the scratch, whatever they
are, lead the join outside it (compiled for the host from the header that the kernels use)."""

import ctypes
import itertools
import pathlib
import shutil
import subprocess

import pytest

CSRC = pathlib.Path(__file__).resolve().parent.parent / "llmquant_b200" / "csrc"


@pytest.fixture(scope="module")
def parts(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    folder = tmp_path_factory.mktemp("parts")
    source = folder / "parts.cpp"
    source.write_text('#include "block_parts.cuh"\n'
                      'extern "C" long long slot(int rt, int runs, int heads, int run, int bh, int tile) '
                      '{ return lq::part_slot(rt, runs, heads, run, bh, tile); }\n'
                      'extern "C" int between(int first, int last, int runs) { return lq::parts_between(first, last, runs); }\n')
    out = folder / "parts.so"
    subprocess.run(["g++", "-x", "c++", "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{CSRC}", str(source), "-o", str(out)],
                   check=True, capture_output=True)
    lib = ctypes.CDLL(str(out))
    lib.slot.restype = ctypes.c_longlong
    return lib


WORDS = (-2 ** 31, -2 ** 31 + 1, -148, -1, 0, 1, 2, 7, 295, 296, 297, 3551, 3552, 2 ** 30, 2 ** 31 - 1)


@pytest.mark.parametrize("tiles,runs,heads,tile", [(1, 3552, 8, 8), (3, 394, 16, 16), (32, 8, 8, 128), (1, 296, 524288, 128)])
def test_the_join_stays_in_the_scratch(parts, tiles, runs, heads, tile):
    slots = tiles * (runs + heads) * tile
    taken = 0
    for first, last in itertools.product(WORDS, WORDS):
        n = parts.between(first, last, runs)
        assert (n > 0) == (0 <= first <= last < runs) and n in (0, last - first + 1)
        if n == 0:
            continue
        taken += 1
        for rt, bh in itertools.product((0, tiles - 1), (0, heads // 2, heads - 1)):
            begin = parts.slot(rt, runs, heads, first, bh, tile)
            assert 0 <= begin and begin + n * tile <= slots
    assert taken > 0


def test_parts_of_one_tile_do_not_overlap(parts):
    """Runs follow the line: run and (sequence, head) never go back, and one of them moves on with every part."""
    runs, heads, tile = 5, 7, 16
    line = [(0, 0), (0, 1), (1, 1), (2, 1), (2, 2), (2, 3), (3, 4), (4, 4), (4, 5), (4, 6)]
    slots = [parts.slot(rt, runs, heads, run, bh, tile) for rt in (0, 1) for run, bh in line]
    assert all(b - a >= tile for a, b in zip(slots, slots[1:]))


def test_rows_that_the_token_arithmetic_cannot_tell_are_refused():
    """row -> token is a 32-bit multiplication, exact for row * group < 2^32 up to the end of the last tile (128
    rows), whatever kernel takes the call."""
    from llmquant_b200 import native

    lib = native.library()
    for group, fits in ((65472, True), (65473, False), (65490, False), (65504, False)):
        assert ((group + 128) * group < 2 ** 32) == fits  # (one token: as many rows as heads)
        c = native.BlockKV(4096, 4096, 64, 64, 4096, 4096, 64, 8, 4, 1, 1, 128, 64, native.LQ_BF16)
        assert (lib.lq_block_attn_scratch_bytes(ctypes.byref(c), group, 1) > 0) == fits
