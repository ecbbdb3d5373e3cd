"""Which rows of a step of drafted tokens belong to whom, and what is left out: places of a batch that are not in use, sequences that do
not fit, through every op that reads a det_tree_ref, against the plain functions of tree_oracle.py in float64."""
import ctypes as C

import numpy as np
import pytest

import tree_oracle as to
from float_ops import code
from test_tree_ops_gpu import Attn, gpu, ints, load, random_masks, size_error, slots, store  # noqa: F401  (gpu: a fixture)

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


# ------------------------------------------------------------------------------------------------------------------ lengths near 2^31
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 31 - 2, -2 ** 31, -1])
def test_a_length_whose_rows_have_no_place_writes_nothing(length, dtype, gpu, libs):  # noqa: F811
    """len + node passes 2^31, or is negative: no row of the sequence has a place in its cache, whose neighbours in memory stay as they were."""
    H, G, d, cap, nodes = 2, 1, 16, 12, [4, 2]
    ld, rows = 2 * G * d, 6
    rng = np.random.default_rng(1)
    y = np.float32(rng.standard_normal((rows, (H + 2 * G) * d)))
    for order in (0, 1):
        lens = [length, 3] if order == 0 else [3, length]
        n = nodes[::1 if order == 0 else -1]
        first = [0, n[0], rows]
        caches = [store(gpu, np.full((cap, ld), KEPT), dtype)[0] for _ in lens]
        q = store(gpu, np.full((rows, H * d), KEPT), dtype)[0]
        ref = libs.TreeRef(table=slots(gpu, libs, caches), first=ints(gpu, first), len=ints(gpu, lens), seqs=2, rows=rows, max_nodes=4, max_len=cap)
        op = libs.FQkOp(heads=H, kv_heads=G, dim=d, vdim=d, rot_dims=0, half=0, eps=0.0, cap=cap, dtype=code(libs, dtype), y=gpu.f32(y), ldy=y.shape[1],
                        q_off=0, k_off=H * d, v_off=(H + G) * d, q=q, seq=ref)
        assert gpu.d.det_f_qk_rope(C.byref(op), None) == 0
        assert size_error(gpu) == SIZE_ERROR
        stored, good = store(gpu, y, dtype)[1], 1 - order
        r = slice(first[good], first[good + 1])
        want_q, want = np.full((rows, H * d), KEPT), [np.full((cap, ld), KEPT) for _ in lens]
        want_q[r], want[good][3:3 + n[good]] = stored[r, :H * d], stored[r, H * d:]
        assert np.array_equal(load(gpu, q, (rows, H * d), dtype), want_q)
        for p, c in zip(caches, want):
            assert np.array_equal(load(gpu, p, (cap, ld), dtype), c)
