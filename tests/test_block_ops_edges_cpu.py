"""Refusals and first calls of the transformer-block operators that need no
GPU.  The pointers are made up and never read."""
import os
import subprocess
import sys

import pytest
import torch

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


def test_rotary_sizes_of_more_than_31_bits():
    """Sizes that would be cut to 32 bits on their way into the library (a
    section of 2^32 + 1 pairs to one of one)."""
    one, freq = torch.zeros(1), torch.ones(1).double()
    for shape in ((1, 1, 1, 2 ** 32 + 2), (2 ** 32 + 1, 1, 1, 2), (1, 2 ** 31, 1, 2)):
        pos = torch.zeros(1, 1, 1, dtype=torch.int64).expand(1, *shape[:2])
        with pytest.raises(ValueError, match="31 bits"):
            ppdl.rotary(one.expand(shape), None, pos, freq, (1,))
    with pytest.raises(ValueError, match="31 bits"):
        ppdl._heads(one.expand(1, 1, 2 ** 32 + 1, 2), True, "q", (1, 1), 2, torch.float32)
    with pytest.raises(ValueError, match="31 bits"):
        ppdl._sections((2 ** 32 + 1,))
    assert list(ppdl._sections((3, 0, 5))) == [3, 0, 5]


FIRST = """
import sys, threading
sys.path.insert(0, sys.argv[1])
import torch, ppdl
x, q, s = torch.zeros(4, 16), torch.zeros(4, 16, dtype=torch.int8), torch.ones(4)
filled, go = threading.Event(), threading.Event()
class Slow(dict):
    def update(self, *a, **kw):
        super().update(*a, **kw)
        if threading.current_thread() is first:
            filled.set()
            assert go.wait(60)
setattr(ppdl, sys.argv[2], Slow())
def call(errors):
    for f in (lambda: ppdl.layernorm(x), lambda: ppdl.linear_i8(x, q, s), lambda: ppdl.quantize_rows(x)):
        try:
            f()
        except Exception as e:
            errors.append(type(e).__name__)
ours, theirs = [], []
first = threading.Thread(target=call, args=(theirs,))
first.start()
assert filled.wait(60)
call(ours)
go.set()
first.join()
assert ours == theirs == ["ValueError"] * 3, (ours, theirs)
"""


@pytest.mark.parametrize("name", ["_types", "_tt"])
def test_first_calls_of_two_threads(name):
    """A thread whose first call comes while another's is between filling one
    of the module's tables and the other: it is told that its tensors are on
    no GPU, not that a table lacks an entry."""
    subprocess.run([sys.executable, "-c", FIRST, os.path.dirname(ppdl.__file__), name], check=True, timeout=300)
