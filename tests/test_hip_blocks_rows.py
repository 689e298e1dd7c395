"""The joint over more rows than its workgroups take at once, at every number of lanes a row takes: the second turn of the tables of sums, the rows read ahead, column sums over
several rows a workgroup (bounds: test_hip_blocks.check_join)."""
import pytest
import torch

from test_hip_blocks import DTYPES, check_join, ids

pytestmark = pytest.mark.gpu

# (256 compute units; a workgroup takes 256 / lanes rows at a time, two workgroups a unit backward and four forward, from 512 lanes on one and two)
ROWS = [(9000, 250), (9000, 256), (5000, 512), (2300, 1000), (2300, 1024), (1300, 1333), (1300, 2048), (700, 2051), (600, 4096), (600, 3002)]


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
@pytest.mark.parametrize("rows, width", ROWS)
def test_join_rows_over_several_turns(dt, rows, width):
    check_join(rows, width, dt, "layernorm", "layernorm", "full", "columns", seed=rows + width)
    check_join(rows, width, dt, "rmsnorm", "layernorm", "row", "number", params=dt, gate_act="silu", seed=rows + width + 1)


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
@pytest.mark.parametrize("rows, width", [(9000, 256), (1300, 2051), (600, 4096)])
@pytest.mark.parametrize("post, pre, gate, use", [(None, "rmsnorm", "none", (True, True)), ("layernorm", None, "full", (True, True)), ("none", "layernorm", "row", (False, True)),
                                                  ("rmsnorm", "none", "full", (True, False))])
def test_join_rows_over_several_turns_in_other_forms(dt, rows, width, post, pre, gate, use):
    check_join(rows, width, dt, post, pre, gate, "columns", seed=rows + width, use=use)
