"""Which rows of a step of drafted tokens belong to whom, and what is left out: places of a batch that are not in use, sequences that do
not fit, through every op that reads a det_tree_ref, against the plain functions of tree_oracle.py in float64."""
import ctypes as C

import numpy as np
import pytest

import tree_oracle as to
from float_ops import code
from test_tree_ops_gpu import Attn, gpu, ints, load, random_masks, rope_tables, size_error, slots, store  # noqa: F401  (gpu: a fixture)

pytestmark = pytest.mark.gpu

SIZE_ERROR = 2
KEPT = 7.0                                                     # what buffers hold before a call


# ------------------------------------------------------------------------------------------------------------------ places not in use
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("unused", [0, 8, 3], ids=["NULL", "misaligned", "odd"])
def test_places_of_a_batch_that_are_not_in_use(unused, dtype, gpu, libs):  # noqa: F811
    """A captured step has as many places as its batch; those without rows hold no cache and any length, and that is no error."""
    rng = np.random.default_rng(3)
    nodes, lens = [0, 5, 0, 2, 0], [0, 130, 0, 0, 0]
    for masked in (0, 1):
        a = Attn(gpu, libs, dtype, 4, 2, 64, 64, lens, nodes, masks=random_masks(nodes, rng) if masked else None)
        for stale in (0, 2 ** 31 - 1, -4):
            op = a.op()
            op.seq.table = slots(gpu, libs, [c if n else unused or None for c, n in zip(a.caches, nodes)])
            op.seq.len = ints(gpu, [x if n else stale for x, n in zip(lens, nodes)])
            for flags in (0, 16, 32):
                op.out = store(gpu, np.full((a.s.rows, a.ldo), KEPT), dtype)[0]
                gpu.d.det_debug_set_float(flags)
                assert gpu.d.det_f_tree_attn(C.byref(op), None) == 0
                gpu.d.det_debug_set_float(0)
                assert size_error(gpu) == 0
                a.check(load(gpu, op.out, (a.s.rows, a.ldo), dtype))
