"""The launch that goes through a long rollout's parts (parts_kernel) hands states from wavefront to wavefront through LDS, two buffers in turn: a wavefront
may write a buffer again only behind a barrier that all reach once they have read it, whatever parts have cuts."""
import importlib

import pytest

build = importlib.import_module("mojo-rl_amd.build")

LOOP = """
_Z12parts_kernelv:
.LBB0_1:
\tglobal_store_dwordx4 v[0:1], v[2:5], off
\ts_cbranch_scc1 .LBB0_3
\tds_write_b128 v6, v[2:5]
\ts_barrier
\tds_read_b128 v[8:11], v7
.LBB0_3:
\ts_cbranch_scc0 .LBB0_1
\ts_endpgm
"""


def test_a_way_around_the_barrier_is_found():
    assert build.stores_around_barriers(LOOP.splitlines(), "parts_kernel") == {"_Z12parts_kernelv": ["global_store_dwordx4 v[0:1], v[2:5], off"]}
    assert build.stores_around_barriers(LOOP.splitlines(), "another") == {}


@pytest.mark.parametrize("old,new", [("\ts_cbranch_scc1 .LBB0_3\n", ""), (".LBB0_3:\n", ".LBB0_3:\n\ts_barrier\n"), ("\ts_cbranch_scc0 .LBB0_1\n", "")])
def test_a_barrier_on_every_way_is_enough(old, new):
    assert build.stores_around_barriers(LOOP.replace(old, new).splitlines(), "parts_kernel") == {"_Z12parts_kernelv": []}


def test_every_step_through_the_parts_has_a_barrier():
    found = build.stores_around_barriers(build.assembly("mrl_delta.hip"), "parts_kernel")
    shared = {k: v for k, v in found.items() if "parts_kernelILi16E" not in k}   # (keys up to 16: a single wavefront)
    assert len(found) == 8 and len(shared) == 6
    assert not any(shared.values()), shared
