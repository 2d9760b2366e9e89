"""Workspace of the delta rule in chunks (csrc/linear_segments.cuh) on the host: every batch of a handle finds room in it, and none of it is
for what no batch can have."""
from __future__ import annotations

import ctypes
import random
import subprocess

import pytest

from conftest import PACKAGE_DIR

PAIR, HEAD, BORDER = 32768, 34176, 24 * 65536          # bytes of a tile and key head, of a tile and value head, of a head's borders
SOURCE = """
#include "linear_segments.cuh"
extern "C" size_t workspace(int k, int v, int tokens, int sequences) { return aima::chunk_workspace(k, v, tokens, sequences, 28, 32768, 34176); }
extern "C" size_t layout(int k, int v, int tokens, int sequences, int most, int rows, int places, int* segments) {
  const aima::ChunkLayout l = aima::chunk_layout(k, v, tokens, sequences, most, rows, places, 32768, 34176);
  *segments = l.cut.segments;
  if (l.pairs_at % 256 != 0 || l.heads_at % 256 != 0 || l.heads_at < l.pairs_at || l.bytes < l.heads_at) return ~size_t{0};
  return l.bytes;
}
extern "C" int begin(int segments, int eighths, int chunks, int which) { return aima::Segments(segments, eighths, chunks).begin(which); }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    folder = tmp_path_factory.mktemp("segments")
    (folder / "segments.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", str(PACKAGE_DIR / "csrc"), "-o", str(folder / "libsegments.so"), str(folder / "segments.cpp")],
                   check=True)
    lib = ctypes.CDLL(str(folder / "libsegments.so"))
    lib.workspace.restype = lib.layout.restype = ctypes.c_size_t
    return lib


@pytest.mark.parametrize("places", [148, 160, 132, 74, 16])
def test_every_batch_finds_room(lib, places):
    rng = random.Random(places)
    cut = 0
    for _ in range(3000):
        k = rng.choice([1, 1, 2, 3, 16, 37, 74, 128])
        v = k * rng.randint(1, max(1, min(4, 256 // k)))
        max_tokens = int(2 ** rng.uniform(5, 14))
        max_sequences = int(2 ** rng.uniform(0, 10))
        room = lib.workspace(k, v, max_tokens, max_sequences)
        segments = ctypes.c_int()
        for _ in range(8):
            sequences = rng.choice([1, min(2, max_sequences), rng.randint(1, max_sequences)])
            tokens = rng.choice([max_tokens, rng.randint(1, max_tokens)])
            offsets = rng.random() < 0.6
            most = rng.choice([tokens, rng.randint(1, tokens)]) if offsets else tokens // sequences
            if not offsets:
                tokens = most * sequences
            if most <= 28:                                        # token by token
                continue
            rows = 28 if sequences > 1 and offsets else 0         # as the entry chooses
            assert lib.layout(k, v, tokens, sequences, most, rows, places, ctypes.byref(segments)) <= room, (k, v, max_tokens, max_sequences, tokens, sequences, most)
            cut += segments.value > 1
    assert cut > 100 or places < 148


def tiles(tokens, sequences):
    return max(tokens // 64 + min(sequences, tokens // 29), tokens // 64 + 1)


@pytest.mark.parametrize("k,v,tokens,sequences,borders", [
    (1, 1, 64, 1, 0), (16, 32, 64, 1, 0), (16, 32, 64, 256, 0), (16, 32, 256, 4, 0),        # too short to be cut
    (25, 75, 8192, 4, 0), (128, 256, 8192, 1, 0),                                           # too many heads
    (16, 32, 8192, 256, 64), (16, 32, 8192, 1, 32), (74, 74, 8192, 8, 74), (1, 1, 8192, 256, 74), (1, 1, 8192, 3, 3)])
def test_borders_are_for_what_can_be_cut(lib, k, v, tokens, sequences, borders):
    assert lib.workspace(k, v, tokens, sequences) == borders * BORDER + tiles(tokens, sequences) * (k * PAIR + v * HEAD)


def test_segments_cover_all_chunks(lib):
    for segments in range(1, 9):
        for eighths in (8, 4, 3, 2):
            for chunks in list(range(1, 70)) + [128, 157, 1000]:
                at = [lib.begin(segments, eighths, chunks, i) for i in range(segments + 1)]
                assert at[0] == 0 and at[1] >= 1 and all(a <= b for a, b in zip(at, at[1:])) and at[-1] >= chunks
