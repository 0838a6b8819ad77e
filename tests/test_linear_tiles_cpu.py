"""How the products of the linear layer are cut at the sizes that the GPU tests
rely on for their coverage (host arithmetic)."""

import ctypes

import pytest
import test_gpu_7b_linear_tiles as gates
import test_gpu_7d_linear_walks as walks

from peco_b200 import _native
from peco_b200.linear import ACTIVATIONS

SMS = 148


@pytest.fixture(scope="module")
def plan():
    from peco_b200 import build
    build.build()
    lib = _native.load()

    def cut(m, n, k_blocks, product=0, activation=0):
        values = (ctypes.c_int * 8)()
        assert lib.peco_linear_tiles(m, n, k_blocks, product, activation, values) == 0
        return dict(zip(("ctas", "columns", "accumulators", "splits", "stages", "tile_rows", "tile_columns", "band"), values))
    return cut


def _blocks(k):
    return -(-k // 64)


def _as_meant(p, cut):
    assert (p["ctas"], p["columns"], p["accumulators"], p["tile_rows"] % p["band"]) == cut and p["splits"] == 1
    return p["tile_rows"] * p["tile_columns"] / (SMS // p["ctas"])


def test_walks_of_the_forward(plan):
    several = set()
    for (b, rows, k, k2, n), act, *_, cut in walks.FORWARD:
        p = plan(b * rows, n, _blocks(k) + (_blocks(k2) if k2 else 0), 0, ACTIVATIONS[act])
        if _as_meant(p, cut) > 2:  # a third tile meets the first one's buffers again
            several.add((p["ctas"], p["accumulators"]))
    assert several == {(1, 1), (2, 1), (2, 2)}


def test_walks_of_the_gradients(plan):
    several = set()
    for (rows, k, n), cut in walks.BACKWARD:
        for product in (1, 2):  # rows and outputs change places
            p = plan(rows, k, _blocks(n), product)
            if _as_meant(p, cut) > 2:
                several.add((product, p["accumulators"]))
    assert several == {(1, 1), (1, 2), (2, 1), (2, 2)}


def test_walks_past_the_last_rows(plan):
    shapes = [m for m in gates.test_gate_without_bias_past_the_last_rows.pytestmark if m.args[0] == "rows,k,n"][0].args[1]
    for rows, k, n in shapes:
        p = plan(rows, n, _blocks(k))
        assert (p["ctas"], p["accumulators"], p["splits"]) == (2, 1, 1) and p["band"] == p["tile_rows"]
        assert 0 < rows % 256 <= 128 and p["tile_rows"] * p["tile_columns"] > 2 * SMS // 2


def test_sums_shared_out(plan):
    cuts = {(k, rows): plan(rows, n, _blocks(k)) for rows in (1, 31, 33, 97, 127, 130, 161, 255)
            for k, n in ((4096, 700), (2048, 5000))}
    shared = {key for key, p in cuts.items() if p["splits"] > 1}
    # every row count over one of the sums, single CTAs and pairs
    assert {rows for _, rows in shared} == {rows for _, rows in cuts} and {cuts[key]["ctas"] for key in shared} == {1, 2}


def test_sizes_out_of_range(plan):
    lib, values = _native.load(), (ctypes.c_int * 8)()
    for bad in ((0, 8, 1, 0, 0), (8, 0, 1, 0, 0), (8, 8, 0, 0, 0), (8, 8, 1, 3, 0), (8, 8, 1, 0, 4)):
        assert lib.peco_linear_tiles(*bad, values) == 1
