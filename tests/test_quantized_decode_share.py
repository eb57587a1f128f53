"""How the tiles of an item fall to the warps of a cluster, from the header that the kernel takes it from. A warp that came out with more tiles than its item
has left would take two pieces, and only one has a place."""

import ctypes
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "flash-sparse-attention_b200", "csrc")


@pytest.fixture(scope="module")
def share(tmp_path_factory):
    d = tmp_path_factory.mktemp("share")
    (d / "share.cpp").write_text(f'#include "{os.path.abspath(os.path.join(CSRC, "fsa_quant_share.h"))}"\n'
                                 'extern "C" int share(int tiles, int warps, int w, int* first) { return fsa::quant_cluster_share(tiles, warps, w, first); }\n')
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-std=c++17", "-o", str(d / "share.so"), str(d / "share.cpp")], check=True)
    fn = ctypes.CDLL(str(d / "share.so")).share

    def call(tiles, warps, w):
        first = ctypes.c_int(-1)
        return fn(tiles, warps, w, ctypes.byref(first)), first.value

    return call


@pytest.mark.parametrize("warps", [8, 10, 12, 20, 48, 80, 96])
def test_pieces_of_one_number_of_tiles(share, warps):
    for tiles in [*range(1, 3 * warps + 2), 1000, 4 * warps, 2**26 + 5]:
        pieces = [share(tiles, warps, w) for w in range(warps)]
        counts = [n for n, _ in pieces]
        there = [p for p in pieces if p[0]]
        assert sum(counts) == tiles and counts == sorted(counts, key=lambda n: n == 0)  # those without any behind the others
        assert max(counts) - min(n for n, _ in there) <= 1
        at = 0
        for n, first in there:
            assert first == at and first + n <= tiles  # one after the other, none behind the item's end
            at += n


def test_a_cluster_reads_a_length_once():
    """The source: between a length and the piece that follows from it nothing reads it again."""
    with open(os.path.join(CSRC, "fsa_quant_dec.cuh")) as f:
        text = f.read()
    start = text.index("  if (p.cluster) {\n    // an item's tiles go round")
    branch = text[start:text.index("  } else {", start)]
    assert branch.count("walk.sequence(p)") == 1 and "keys_of" not in branch
    assert text.count("if (!p.cluster) walk.sequence(p);") == 1 and text.count("walk.sequence(p)") == 2
