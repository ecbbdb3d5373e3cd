"""Which rows of a step of drafted tokens belong to whom, and what is left out: places of a batch that are not in use, sequences that do
not fit, through every op that reads a det_tree_ref, against the plain functions of tree_oracle.py in float64."""
import ctypes as C
import decimal
import math

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


# ------------------------------------------------------------------------------------------------------------------ what does not fit
BAD = {  # first, lens, rows of the buffers, places of the table that hold no cache, sequences that are left out (caches of 12 rows, trees of 4)
    "full cache": ([0, 3, 5, 9], [10, 2, 1], 9, {}, {0}),
    "full cache, last": ([0, 2, 5, 9], [10, 2, 9], 9, {}, {2}),
    "large tree": ([0, 2, 7, 11], [1, 2, 3], 11, {}, {1}),
    "negative length": ([0, 2, 4, 8], [1, -1, 8], 8, {}, {1}),
    "largest length": ([0, 2, 4, 8], [2 ** 31 - 1, 10, 0], 8, {}, {0}),
    "rows behind the buffers": ([0, 2, 4, 8], [0, 1, 2], 6, {}, {2}),
    "no row in the buffers": ([0, 2, 6, 9], [0, 1, 2], 6, {}, {2}),
    "first row negative": ([-1, 2, 4, 8], [0, 1, 2], 9, {}, {0}),
    "no cache": ([0, 2, 4, 8], [0, 1, 2], 8, {1: None}, {1}),
    "misaligned cache": ([0, 2, 4, 8], [0, 1, 2], 8, {0: 8}, {0}),
    "all": ([0, 5, 5, 7], [0, 0, 11], 7, {}, {0, 2}),
}


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 24, 11], ids=["64", "24", "11 (no vectors)"])
@pytest.mark.parametrize("kind", BAD)
def test_a_sequence_that_does_not_fit_is_left_out_whole(kind, dim, dtype, gpu, libs):  # noqa: F811
    """Every row of q and every row of the cache of such a sequence stay as they were, rows among them that would have fitted alone; the
    attention of the same step leaves out the same sequences.  Without norm and rotation the rows are the activations, rounded once."""
    first, lens, rows, missing, bad = BAD[kind]
    H, G, cap, max_nodes, seqs = 4, 2, 12, 4, len(lens)
    kd = (dim + 7) // 8 * 8
    ld = 2 * G * kd
    rng = np.random.default_rng(dim)
    y = np.float32(rng.standard_normal((rows, (H + 2 * G) * dim)))
    caches = [store(gpu, np.full((cap, ld), KEPT), dtype)[0] for _ in lens]
    q = store(gpu, np.full((rows, H * kd), KEPT), dtype)[0]
    table = slots(gpu, libs, [missing.get(b, c) for b, c in enumerate(caches)])
    ref = libs.TreeRef(table=table, first=ints(gpu, first), len=ints(gpu, lens), seqs=seqs, rows=rows, max_nodes=max_nodes, max_len=cap)
    op = libs.FQkOp(heads=H, kv_heads=G, dim=dim, vdim=dim, rot_dims=0, half=0, eps=0.0, cap=cap, dtype=code(libs, dtype), y=gpu.f32(y), ldy=y.shape[1],
                    q_off=0, k_off=H * dim, v_off=(H + G) * dim, q=q, seq=ref)
    assert gpu.d.det_f_qk_rope(C.byref(op), None) == 0
    assert size_error(gpu) == SIZE_ERROR
    stored = store(gpu, y, dtype)[1].reshape(rows, H + 2 * G, dim)
    want_q, want = np.full((rows, H, kd), KEPT), [np.full((cap, 2 * G, kd), KEPT) for _ in lens]
    for b in set(range(seqs)) - bad:
        r = slice(first[b], first[b + 1])
        n = first[b + 1] - first[b]
        want_q[r] = 0.0
        want_q[r, :, :dim] = stored[r, :H]
        want[b][lens[b]:lens[b] + n] = 0.0
        want[b][lens[b]:lens[b] + n, :, :dim] = stored[r, H:]
    assert np.array_equal(load(gpu, q, (rows, H, kd), dtype), want_q)
    for p, c in zip(caches, want):
        assert np.array_equal(load(gpu, p, (cap, 2 * G, kd), dtype), c)
    mask = to.bits(np.ones((rows, 32), bool), 1)
    for masked in (0, 1):
        for flags in (0, 16, 32):
            out = store(gpu, np.full((rows, H * dim), -3.0), dtype)[0]
            ta = libs.FTreeOp(heads=H, kv_heads=G, dim=dim, vdim=dim, scale=0.3, cap=cap, dtype=code(libs, dtype), q=q, mask=gpu.put(mask) if masked else None,
                              mask_ld=masked, out=out, ldo=H * dim, scratch=gpu.space(gpu.d.det_f_tree_scratch_bytes(H, G, dim, max_nodes)), seq=ref)
            gpu.d.det_debug_set_float(flags)
            assert gpu.d.det_f_tree_attn(C.byref(ta), None) == 0
            gpu.d.det_debug_set_float(0)
            assert size_error(gpu) == SIZE_ERROR
            left = (load(gpu, out, (rows, H * dim), dtype) == -3.0).all(1)      # (a row may well be the 7 of the cached rows)
            own = np.zeros(rows, bool)
            for b in set(range(seqs)) - bad:
                own[first[b]:first[b + 1]] = True
            assert np.array_equal(left, ~own)


# ------------------------------------------------------------------------------------------------------------------ kept rows
class Kept:
    """det_f_tree_keep over `layers` caches of every sequence, with the table's entries as given (entry e belongs to sequence e % seqs)."""

    def __init__(self, gpu, libs, lens, lists, layers, cap, missing, most=6):  # noqa: F811
        self.gpu, self.lens, self.lists, self.cap, self.width = gpu, lens, lists, cap, 8
        seqs = len(lens)
        rng = np.random.default_rng(seqs)
        self.before = rng.standard_normal((layers * seqs, cap, self.width)).astype(np.float32)
        self.caches = [gpu.put(c) for c in self.before]
        keep = np.zeros((seqs, most), np.int32)
        for b, k in enumerate(lists):
            keep[b, :len(k)] = k
        self.out = ints(gpu, [-1] * seqs)
        op = libs.FKeepOp(caches=layers * seqs, seqs=seqs, cap=cap, row_bytes=self.width * 4, table=slots(gpu, libs, [missing.get(e, c) for e, c in enumerate(self.caches)]),
                          len=ints(gpu, lens), keep=gpu.put(keep), keep_ld=most, count=ints(gpu, [len(k) for k in lists]), max_count=most, len_out=self.out)
        assert gpu.d.det_f_tree_keep(C.byref(op), None) == 0

    def check(self, bad):
        """The sequences `bad` as they were in every layer, the others moved up."""
        seqs = len(self.lens)
        for e, p in enumerate(self.caches):
            want, b = self.before[e].copy(), e % seqs
            if b not in bad:
                for i, k in enumerate(self.lists[b]):
                    want[self.lens[b] + i] = self.before[e][self.lens[b] + k]
            assert np.array_equal(self.gpu.get(p, (self.cap, self.width)), want), e
        assert np.array_equal(self.gpu.get(self.out, seqs, np.int32), [-1 if b in bad else n + len(k) for b, (n, k) in enumerate(zip(self.lens, self.lists))])


@pytest.mark.parametrize("slot", [None, 8, 4096 + 4], ids=["NULL", "8", "4100"])
@pytest.mark.parametrize("layers,entry", [(1, 0), (3, 0), (3, 3), (3, 4), (3, 6), (3, 8), (400, 599), (400, 1199)])
def test_a_sequence_is_kept_in_all_layers_or_in_none(layers, entry, slot, gpu, libs):  # noqa: F811
    """One layer of a sequence holds no usable cache: none of its layers moves and its length stays, the other sequences move."""
    k = Kept(gpu, libs, [4, 5, 3], [[0, 2, 3], [1, 4], [0, 1, 5]], layers, 12, {entry: slot})
    assert size_error(gpu) == SIZE_ERROR
    k.check({entry % 3})


def test_sequences_that_keep_nothing_need_no_cache(gpu, libs):  # noqa: F811
    """Places of a batch that are not in use: count 0, no cache in any layer, or none in one; the new length is the old one."""
    k = Kept(gpu, libs, [0, 5, 3, 0], [[], [1, 4], [], []], 2, 12, {0: None, 4: None, 2: 8, 3: 4, 7: None})
    assert size_error(gpu) == 0
    k.check(set())


# ------------------------------------------------------------------------------------------------------------------ failed launches
def test_a_launch_that_fails_is_reported_and_ends_nothing(gpu, libs, capfd):  # noqa: F811
    """A stream whose capture was invalidated takes no kernel (an error of the host alone): every op returns 1 and names the CUDA error,
    nothing is written, and the same calls work afterwards."""
    rt = C.CDLL("libcudart.so.12")
    a = Attn(gpu, libs, "bf16", 4, 2, 64, 64, [130], [5])
    b = Attn(gpu, libs, "f32", 4, 2, 64, 64, [130], [5])
    y = gpu.f32(np.ones((5, 8 * 64), np.float32))
    q, tab = gpu.space(5 * 4 * 64 * 4), gpu.space(2 * 4 * 4 * 8)
    k = Kept(gpu, libs, [4, 5], [[0, 2, 3], [1, 4]], 2, 12, {})
    gpu.d.det_memset(q, 0, 5 * 4 * 64 * 4, None)
    gpu.d.det_memset(tab, 0, 2 * 4 * 4 * 8, None)
    ops = [(gpu.d.det_f_tree_attn, a.op()), (gpu.d.det_f_tree_attn, b.op()),
           (gpu.d.det_f_rope_table, libs.FRopeOp(dims=8, scaling=0, base=1e4, factor=1.0, mscale=1.0, n=8, cos=tab, sin=tab + 4 * 4 * 8)),
           (gpu.d.det_f_qk_rope, libs.FQkOp(heads=4, kv_heads=2, dim=64, vdim=64, rot_dims=0, half=0, eps=0.0, cap=a.cap, dtype=libs.DET_BF16, y=y, ldy=512,
                                            q_off=0, k_off=256, v_off=384, q=q, seq=a.s.ref(a.caches))),
           (gpu.d.det_f_tree_keep, libs.FKeepOp(caches=1, seqs=1, cap=a.cap, row_bytes=a.ld * 2, table=a.s.ref(a.caches).table, len=a.s.len_p,
                                                keep=ints(gpu, [1]), keep_ld=1, count=ints(gpu, [1]), max_count=1))]
    gpu.d.det_sync()
    before = load(gpu, a.caches[0], (a.cap, a.ld), "bf16")
    stream, graph = C.c_void_p(), C.c_void_p()
    assert rt.cudaStreamCreateWithFlags(C.byref(stream), 1) == 0
    assert rt.cudaStreamBeginCapture(stream, 2) == 0             # relaxed: other streams are not restricted
    assert rt.cudaStreamSynchronize(stream) != 0                 # not allowed in a capture, which it ends
    capfd.readouterr()
    for entry, op in ops:
        assert entry(C.byref(op), stream) == 1
        err = capfd.readouterr().err
        assert "the launch failed" in err and "refused" not in err
    rt.cudaStreamEndCapture(stream, C.byref(graph))
    assert not graph
    rt.cudaGetLastError()
    assert rt.cudaStreamDestroy(stream) == 0
    gpu.d.det_sync()
    assert (gpu.get(q, 5 * 4 * 64) == 0).all() and (gpu.get(tab, 2 * 4 * 8) == 0).all()
    assert np.array_equal(load(gpu, a.caches[0], (a.cap, a.ld), "bf16"), before, equal_nan=True)
    for x in (a, b):
        assert (load(gpu, x.out, (x.s.rows, x.ldo), x.dtype) == KEPT).all()
        x.check_each()
    k.check(set())
    assert size_error(gpu) == 0


# ------------------------------------------------------------------------------------------------------------------ far positions
def exact_frequencies(dims, base, scaling, factor, orig, low, high):
    """As decimals of 60 digits; everything that comes in is a binary64 number, taken as it is."""
    D = decimal.Decimal
    base, factor, orig, low, high = (D(x) for x in (base, factor, orig, low, high))
    log_base = base.ln()
    if scaling == "base":
        log_base += factor.ln() * dims / (dims - 2)
    f = [(-2 * i * log_base / dims).exp() for i in range(dims // 2)]
    if scaling == "linear":
        f = [x / factor for x in f]
    if scaling == "ramp":
        w = [min(max((orig * x / (2 * decimal_pi()) - low) / (high - low), D(0)), D(1)) for x in f]
        f = [x * (y + (1 - y) / factor) for x, y in zip(f, w)]
    return f


def decimal_pi():
    """16 atan(1/5) - 4 atan(1/239)."""
    def atan(n):
        x = decimal.Decimal(1) / n
        s, term, k = x, x, 1
        while abs(term) > decimal.Decimal(10) ** -65:
            term = -term / (n * n)
            k += 2
            s += term / k
        return s
    return 16 * atan(5) - 4 * atan(239)


@pytest.mark.parametrize("dims,base", [(8, 10007.0), (128, 1000003.0), (26, 500.5), (256, 3.0e7), (64, 0.37)])
@pytest.mark.parametrize("scaling,factor,low,high", [("plain", 1.0, 1.0, 2.0), ("linear", 7.3, 1.0, 2.0), ("base", 4.1, 1.0, 2.0), ("base", 0.3, 1.0, 2.0),
                                                     ("ramp", 32.7, 1.0, 32.0), ("ramp", 4.2, 0.0, 3.0), ("ramp", 11.0, 40.0, 41.0)])
def test_tables_of_far_positions(scaling, factor, low, high, dims, base, gpu, libs):  # noqa: F811
    """Every column at the first positions, at 2^20 and at the last ones of 31 bits, against frequencies and angles of 60 digits: within the
    bound that the header states, the angle's loss growing with the exponent of the frequency."""
    orig, m, n = 4096.0, np.float32(1.1), 5
    cols = dims // 2
    with decimal.localcontext() as ctx:
        ctx.prec = 60
        f = exact_frequencies(dims, base, scaling, factor, orig, low, high)
        turn = 2 * decimal_pi()
        for pos0 in (0, 2 ** 20, 2 ** 31 - 1 - n):
            cs, sn = gpu.space(4 * n * cols), gpu.space(4 * n * cols)
            op = libs.FRopeOp(dims=dims, scaling=["plain", "linear", "base", "ramp"].index(scaling), base=base, factor=factor, orig_ctx=orig, low=low, high=high,
                              mscale=m, pos0=pos0, n=n, cos=cs, sin=sn)
            assert gpu.d.det_f_rope_table(C.byref(op), None) == 0
            a = np.array([[float(p * x) for x in f] for p in range(pos0, pos0 + n)])
            rest = np.array([[float(p * x % turn) for x in f] for p in range(pos0, pos0 + n)])      # known to 2^-53 * 2 pi
            g = 2 * np.arange(cols) / dims * (abs(math.log2(base)) + (abs(math.log2(factor)) * dims / (dims - 2) if scaling == "base" else 0))
            loss = (5 * g + 9) * 2.0 ** -53 * (2 + factor * abs(low) / (high - low) if scaling == "ramp" else 1)
            tol = float(m) * (4 * to.U32 + a * loss) + 2.0 ** -50
            for p, want in ((cs, np.cos(rest)), (sn, np.sin(rest))):
                err = np.abs(gpu.get(p, n * cols).astype(float).reshape(n, cols) - float(m) * want)
                assert (err <= tol).all(), (err / tol).max()
