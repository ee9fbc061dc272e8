"""The rule by which an epilogue warp of the 16-bit GEMM reuses its staging
buffer (model_b200/csrc/staging_turn.cuh), run on the host against a model of
the copy engine: bulk stores complete in order, as late as the waits allow,
and no block may be written where one of them still reads."""

import ctypes as C
import itertools
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HARNESS = """
#include "staging_turn.cuh"
extern "C" {
void* turn_new() { return new ml::StagingTurn; }
void turn_free(void* t) { delete static_cast<ml::StagingTurn*>(t); }
int turn_next(void* t, int wide, int bulk, int* stand) {
  const ml::StagingTurn::Place p = static_cast<ml::StagingTurn*>(t)->next(wide != 0, bulk != 0);
  *stand = p.stand;
  return p.offset;
}
}
"""
WIDE, HALF = 4096, 2048
KINDS = [(wide, bulk) for wide in (0, 1) for bulk in (0, 1)]


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    d = tmp_path_factory.mktemp("staging")
    src, so = d / "harness.cpp", d / "harness.so"
    src.write_text(HARNESS)
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-O1", "-shared", "-fPIC", str(src), "-o", str(so), "-I",
                    os.path.join(ROOT, "model_b200", "csrc")], check=True)
    lib = C.CDLL(str(so))
    lib.turn_new.restype = C.c_void_p
    lib.turn_free.argtypes = [C.c_void_p]
    lib.turn_next.argtypes = [C.c_void_p, C.c_int, C.c_int, C.POINTER(C.c_int)]

    def places(blocks):
        t, stand = lib.turn_new(), C.c_int()
        out = [(lib.turn_next(t, w, b, stand), stand.value) for w, b in blocks]
        lib.turn_free(t)
        return out
    return places


def conflicts(blocks, places):
    """Blocks written over what a bulk store may still read."""
    running, bad = [], []
    for i, ((wide, bulk), (at, stand)) in enumerate(zip(blocks, places)):
        running = running[len(running) - min(stand, len(running)):]
        end = at + (WIDE if wide else HALF)
        assert 0 <= at and end <= WIDE
        if any(a < end and at < b for a, b in running):
            bad.append(i)
        if bulk:
            running.append((at, end))
    return bad


@pytest.mark.parametrize("n", range(1, 8))
def test_no_block_over_a_running_store(rule, n):
    for blocks in itertools.product(KINDS, repeat=n):
        assert not conflicts(blocks, rule(blocks)), blocks


def test_blocks_of_16_bits_overlap_their_stores(rule):
    assert [s for _, s in rule([(0, 1)] * 6)] == [0, 1, 1, 1, 1, 1]
    assert [a for a, _ in rule([(0, 1)] * 4)] == [0, HALF, 0, HALF]


def test_the_model_finds_a_wait_that_is_too_short():
    # a float32 store followed by 16-bit blocks that let the latest store stand
    blocks = [(1, 1), (0, 1), (0, 1)]
    assert conflicts(blocks, [(0, 0), (HALF, 1), (0, 1)]) == [1]
    # a half that the warp copies out itself, between two stores of the other
    blocks = [(0, 1), (0, 0), (0, 1)]
    assert conflicts(blocks, [(0, 0), (HALF, 1), (0, 1)]) == [2]


def test_every_block_given_to_the_engine_has_to_reach_it(rule):
    # 16-bit blocks staged as if for bulk stores that are then not issued (rows
    # past the last token): the second one is written over the store before them
    blocks = [(0, 1)] * 4
    assert conflicts([(0, 1), (0, 1), (0, 0), (0, 0)], rule(blocks)) == [3]
    assert not conflicts([(0, 1), (0, 1)], rule([(0, 1), (0, 1)]))
