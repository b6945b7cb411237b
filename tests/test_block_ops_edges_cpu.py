"""Refusals and first calls of the transformer-block operators that need no
GPU.  The pointers are made up and never read."""
import pytest

import ppdl
from test_block_ops_cpu import P, rotary


@pytest.mark.parametrize("heads,sizes", [
    (dict(out_head=7), {}), (dict(out_head=-7), {}), (dict(out_token=0), {}), (dict(out_token=4), {}),
    (dict(out_batch=5), dict(batch=2)), (dict(out_token=8), {}), (dict(out_token=-8), {}),
    (dict(out_batch=16), dict(batch=3)),
    # in place, with the strides of something else
    (dict(out_token=24), {}), (dict(out_head=40), {}), (dict(out_batch=80), dict(batch=2)),
])
def test_rotary_results_in_the_same_place(heads, sizes):
    """Results that share memory with one another or are written where other
    heads are still read."""
    assert rotary(heads, **sizes) == ppdl.PPDL_ERR_SHAPE
    assert ppdl.last_error().startswith("rotary: results that overlap")


def test_rotary_queries_and_keys_in_the_same_place():
    q = ppdl.RotaryHeads(P, 2 * P, 2, 64, 16, 8, 64, 16, 8)
    k = ppdl.RotaryHeads(3 * P, 2 * P, 1, 64, 16, 8, 64, 16, 8)
    assert rotary(q=ppdl.C.byref(q), k=ppdl.C.byref(k)) == ppdl.PPDL_ERR_SHAPE
    assert ppdl.last_error().endswith("the same place")
