"""The ops of a step of drafted tokens through the C ABI against the plain functions of tree_oracle.py in float64: types, layouts, head
sizes, lengths from nothing to thousands of keys, masks that leave rows empty, rows that belong to nobody, lists that do not fit."""
import ctypes as C
import threading

import numpy as np
import pytest

import hybrid_oracle as ho
import tree_oracle as to
from float_ops import Gpu, code, round8

pytestmark = pytest.mark.gpu

U32 = to.U32
SIZE_ERROR = 2


@pytest.fixture
def gpu(libs):
    g = Gpu(libs)
    yield g
    g.free()


def ints(gpu, a):
    return gpu.put(np.asarray(a, np.int32))


def slots(gpu, libs, caches):
    return gpu.put(np.frombuffer(b"".join(bytes(libs.SeqSlot(cache=c)) for c in caches), np.uint8))


def store(gpu, a, dtype):
    """Values in the activation type: the pointer, and the values as stored."""
    if dtype == "f32":
        a = np.asarray(a, np.float32)
        return gpu.put(a), a.astype(float)
    b = ho.bf16_bits(np.asarray(a, np.float32))
    return gpu.put(b), ho.bf16_values(b).astype(float)


def load(gpu, p, shape, dtype):
    return gpu.get_act(p, shape, dtype)


def size_error(gpu):
    """The error word, cleared."""
    e = gpu.d.det_last_error()
    gpu.d.det_clear_error()
    return e


# ------------------------------------------------------------------------------------------------------------------ tables
@pytest.mark.parametrize("dims,n,pos0", [(2, 1, 0), (8, 5, 0), (64, 300, 7), (128, 1000, 1000000), (26, 77, 0), (6, 40, 2 ** 31 - 50), (256, 33, 3)])
@pytest.mark.parametrize("scaling", ["plain", "linear", "base", "ramp"])
def test_rotation_tables(dims, n, pos0, scaling, gpu, libs):
    """A sine or cosine in fp32 is off by one unit in the last place (2^-24 below 1), the two products behind it and the result by half
    of one each; what the angle loses in binary64 (a few 2^-53 of 2^31 radians at most, 2^-20) adds to it for far positions."""
    if scaling == "base" and dims == 2:
        return
    base, factor, orig, low, high, m = 10007.0, 4.0, 4096.0, 1.0, 32.0, 1.1
    cols = dims // 2
    guard = 4
    cs, sn = gpu.put(np.full(n * cols + guard, 9.0, np.float32)), gpu.put(np.full(n * cols + guard, 9.0, np.float32))
    op = libs.FRopeOp(dims=dims, scaling=["plain", "linear", "base", "ramp"].index(scaling), base=base, factor=factor, orig_ctx=orig, low=low,
                      high=high, mscale=m, pos0=pos0, n=n, cos=cs, sin=sn)
    assert gpu.d.det_f_rope_table(C.byref(op), None) == 0
    f = to.frequencies(dims, base, scaling, factor, orig, low, high)
    a = (pos0 + np.arange(n, dtype=np.float64))[:, None] * f
    tol = np.float32(m) * (4 * U32 + 8 * 2.0 ** -53 * np.abs(a))
    for p, want in ((cs, np.cos(a)), (sn, np.sin(a))):
        got = gpu.get(p, n * cols + guard).astype(float)
        assert (np.abs(got[:n * cols].reshape(n, cols) - np.float32(m) * want) <= tol).all()
        assert (got[n * cols:] == 9.0).all()


def test_rotation_table_of_all_positions(gpu, libs):
    """As many positions as 31 bits hold: the counters do not pass the end.  The bound is that of test_rotation_tables."""
    n, guard = 2 ** 31 - 1, 4
    cs, sn = gpu.space(4 * (n + guard)), gpu.space(4 * (n + guard))
    for p in (cs, sn):
        gpu.d.det_memcpy(p + 4 * n, np.full(guard, 9.0, np.float32).ctypes.data, 4 * guard, None)
        gpu.d.det_sync()
    op = libs.FRopeOp(dims=2, scaling=0, base=10007.0, factor=1.0, mscale=1.0, n=n, cos=cs, sin=sn)
    assert gpu.d.det_f_rope_table(C.byref(op), None) == 0
    for at in (0, 2 ** 30 - 3, n - 8):
        a = at + np.arange(8, dtype=np.float64)
        for p, want in ((cs, np.cos(a)), (sn, np.sin(a))):
            assert (np.abs(gpu.get(p + 4 * at, 8).astype(float) - want) <= 4 * U32 + 8 * 2.0 ** -53 * a).all()
    for p in (cs, sn):
        assert (gpu.get(p + 4 * n, guard) == 9.0).all()


# ------------------------------------------------------------------------------------------------------------------ norm and rotation
class Step:
    """The rows of several sequences: `nodes` rows each behind `lens` cached ones, `extra` rows of the buffers that are nobody's."""

    def __init__(self, gpu, libs, lens, nodes, extra=0, max_nodes=None, max_len=None):
        self.lens, self.nodes, self.extra = list(lens), list(nodes), extra
        self.first = np.concatenate([[0], np.cumsum(self.nodes)]).astype(int)
        self.owned = int(self.first[-1])
        self.rows = self.owned + extra
        self.gpu, self.libs = gpu, libs
        self.max_nodes, self.max_len = max_nodes or max(max(self.nodes), 1), max(self.lens) if max_len is None else max_len
        self.first_p, self.len_p = ints(gpu, self.first), ints(gpu, self.lens)

    def ref(self, caches):
        return self.libs.TreeRef(table=slots(self.gpu, self.libs, caches), first=self.first_p, len=self.len_p, seqs=len(self.lens), rows=self.rows,
                                 max_nodes=self.max_nodes, max_len=self.max_len)

    def each(self):
        """(row, sequence, node)"""
        for b, n in enumerate(self.nodes):
            for i in range(n):
                yield self.first[b] + i, b, i


def rope_tables(gpu, dims, n, base):
    a = np.arange(n)[:, None] * to.frequencies(dims, base)[None] if dims else np.zeros((n, 0))
    c, s = np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)
    return gpu.f32(np.append(c, 0)), gpu.f32(np.append(s, 0)), c.astype(float), s.astype(float)


QK = [  # heads, kv heads, dim, vdim, rotated, half, norm, rotated values, odd columns
    (6, 2, 64, 64, 64, 0, 1, 0, 0), (8, 1, 128, 128, 128, 1, 1, 0, 0), (5, 5, 40, 24, 24, 1, 1, 1, 0), (3, 1, 11, 30, 0, 0, 1, 1, 1),
    (4, 4, 72, 136, 8, 0, 0, 1, 0), (2, 1, 256, 200, 64, 1, 1, 0, 1), (2, 2, 24, 256, 24, 0, 1, 1, 0), (1, 1, 2, 1, 2, 1, 1, 0, 1),
    (40, 8, 128, 128, 64, 1, 1, 0, 0), (4, 2, 33, 7, 30, 1, 0, 0, 1)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", QK, ids=str)
def test_norm_rotation_and_cache_rows(shape, dtype, gpu, libs):
    """Per element: the normalised value is off by (d / 2 + 6) u at most (a sum of squares in fp32 under a root, a quotient, two
    products), the rotation adds 3 u of both terms; the result is rounded once to the activation type."""
    H, G, d, v, rot, half, normed, vrot, odd = shape
    rng = np.random.default_rng(H * d + v)
    for lens, nodes, extra, with_pos in [([7], [1], 0, 0), ([0, 3, 50, 9], [4, 0, 9, 1], 3, 1), ([2] * 40, [1, 2, 0, 3] * 10, 1, 0)]:
        s = Step(gpu, libs, lens, nodes, extra)
        kd, vd = round8(d), round8(v)
        ld, cap, eps, table = G * (kd + vd), max(lens) + max(nodes) + 2, 1e-5, 90
        qo = 3 if odd else 0
        ko, vo = qo + H * d + (1 if odd else 0), qo + H * d + G * d + (1 if odd else 0)
        ldy = vo + G * v + (2 if odd else -(vo + G * v) % 4)
        y = np.float32(rng.standard_normal((s.rows, ldy)) * 2)
        qn, kn = np.float32(rng.uniform(0.5, 1.5, (2, d)))
        kt, vt = rope_tables(gpu, rot, table, 300.0), rope_tables(gpu, v - v % 2, table, 500.0)
        pos = rng.integers(0, table, s.rows) if with_pos else np.array([lens[b] + i for _, b, i in s.each()] + [0] * extra)
        sentinel = 7.0
        caches = [store(gpu, np.full((cap, ld), sentinel), dtype)[0] for _ in lens]
        q, _ = store(gpu, np.full((s.rows, H * kd), sentinel), dtype)
        op = libs.FQkOp(heads=H, kv_heads=G, dim=d, vdim=v, rot_dims=rot, half=half, eps=eps, q_norm=gpu.f32(qn) if normed else None,
                        k_norm=gpu.f32(kn) if normed else None, cap=cap, dtype=code(libs, dtype), y=gpu.f32(y), ldy=ldy, q_off=qo, k_off=ko, v_off=vo,
                        rope_len=table, rope_cos=kt[0], rope_sin=kt[1], vrope_cos=vt[0] if vrot else None, vrope_sin=vt[1] if vrot else None,
                        pos=ints(gpu, pos) if with_pos else None, q=q, seq=s.ref(caches))
        assert gpu.d.det_f_qk_rope(C.byref(op), None) == 0
        got_q = load(gpu, q, (s.rows, H, kd), dtype)
        got_c = [load(gpu, c, (cap, ld), dtype) for c in caches]
        unit = to.UNIT[dtype]

        def check(got, x, w, p, tables, n, halves):
            z = to.norm(x, w, eps)
            a = to.rotate(z, tables[2][p], tables[3][p], halves) if n else z
            big = np.abs(z)
            big[:n] = np.repeat(np.maximum(big[0:n:2], big[1:n:2]), 2) if not halves else np.tile(np.maximum(big[:n // 2], big[n // 2:n]), 2)
            tol = unit * np.abs(a) + (len(x) / 2 + 6 + 8) * 2 * U32 * big + 1e-37
            assert (np.abs(got[:len(x)] - a) <= tol).all(), np.abs(got[:len(x)] - a).max()
            assert (got[len(x):] == 0).all()

        for r, b, i in s.each():
            row, slot = y[r].astype(float), lens[b] + i
            for h in range(H):
                check(got_q[r, h], row[qo + h * d:qo + (h + 1) * d], qn.astype(float) if normed else None, pos[r], kt, rot, half)
            for g in range(G):
                c = got_c[b][slot]
                check(c[g * kd:(g + 1) * kd], row[ko + g * d:ko + (g + 1) * d], kn.astype(float) if normed else None, pos[r], kt, rot, half)
                check(c[G * kd + g * vd:G * kd + (g + 1) * vd], row[vo + g * v:vo + (g + 1) * v], None, pos[r], vt, v if vrot else 0, 0)
        assert (got_q[s.owned:] == sentinel).all()
        for b, c in enumerate(got_c):
            own = np.zeros(cap, bool)
            own[lens[b]:lens[b] + nodes[b]] = True
            assert (c[~own] == sentinel).all()
        assert size_error(gpu) == 0


def test_rows_that_do_not_fit_are_left_out(gpu, libs):
    """A cache that is full, a position outside the tables, a tree larger than the bound: reported, and the other sequences are right."""
    H, G, d = 2, 1, 16
    rng = np.random.default_rng(0)
    ld, cap = G * 2 * d, 12
    for lens, nodes, pos, max_nodes, bad in [([10, 2], [3, 2], None, 4, {2}), ([3, 2], [2, 2], [1, 60, 1, 2], 4, {1}), ([3, 2], [2, 2], [-1, 5, 1, 2], 4, {0}),
                                             ([-1, 2], [2, 2], None, 4, {0, 1}), ([1, 2], [5, 2], None, 4, {4})]:
        s = Step(gpu, libs, lens, nodes, max_nodes=max_nodes, max_len=12)
        y = np.float32(rng.standard_normal((s.rows, (H + 2 * G) * d)))
        kt = rope_tables(gpu, d, 50, 100.0)
        caches = [store(gpu, np.full((cap, ld), 7.0), "f32")[0] for _ in lens]
        q, _ = store(gpu, np.full((s.rows, H * d), 7.0), "f32")
        op = libs.FQkOp(heads=H, kv_heads=G, dim=d, vdim=d, rot_dims=d, half=0, eps=0.0, cap=cap, dtype=libs.DET_F32, y=gpu.f32(y), ldy=y.shape[1],
                        q_off=0, k_off=H * d, v_off=(H + G) * d, rope_len=50, rope_cos=kt[0], rope_sin=kt[1], pos=ints(gpu, pos) if pos else None, q=q,
                        seq=s.ref(caches))
        assert gpu.d.det_f_qk_rope(C.byref(op), None) == 0
        assert size_error(gpu) == SIZE_ERROR
        got = gpu.get(q, (s.rows, H * d))
        kept = gpu.get(caches[1], (cap, ld))
        for r, b, i in s.each():
            assert (got[r] == 7.0).all() == (r in bad)
            if b == 1:
                assert np.array_equal(kept[lens[1] + i, G * d:], y[r, (H + G) * d:])


# ------------------------------------------------------------------------------------------------------------------ attention
class Attn:
    """A step's attention over random caches; everything behind what may be read is NaN."""

    def __init__(self, gpu, libs, dtype, heads, kv, d, v, lens, nodes, *, masks=None, extra=0, gate=False, vrot=False, cap=None, seed=0, sharp=1.0,
                 max_nodes=None, max_len=None, ldo=None):
        self.gpu, self.libs, self.dtype, self.H, self.G, self.d, self.v = gpu, libs, dtype, heads, kv, d, v
        self.s = Step(gpu, libs, lens, nodes, extra, max_nodes, max_len)
        rng = np.random.default_rng(seed)
        self.kd, self.vd = round8(d), round8(v)
        self.ld, self.cap = kv * (self.kd + self.vd), cap or max(a + n for a, n in zip(lens, nodes)) + 3
        self.scale = sharp / np.sqrt(d)
        self.caches, self.values = [], []
        for b, (a, n) in enumerate(zip(lens, nodes)):
            c = rng.standard_normal((self.cap, self.ld))
            c[:, :kv * self.kd].reshape(self.cap, kv, self.kd)[..., d:] = 0
            c[:, kv * self.kd:].reshape(self.cap, kv, self.vd)[..., v:] = 0
            c[a + n:] = np.nan
            if masks is not None:      # a node that nobody attends holds nothing
                c[a:a + n][~masks[b].any(0)] = np.nan
            p, val = store(gpu, c, dtype)
            self.caches.append(p)
            self.values.append(val)
        q = rng.standard_normal((self.s.rows, heads, self.kd))
        q[..., d:] = 0
        self.qp, self.q = store(gpu, q, dtype)
        self.masks = masks
        words = (self.s.max_nodes + 31) // 32 + 1
        self.mask_ld = words
        self.mask_p = None
        if masks is not None:
            def wide(m):                                       # bits behind the tree are not looked at
                return to.bits(np.concatenate([m, np.ones((len(m), words * 32 - m.shape[1]), bool)], 1), words)
            w = np.concatenate([wide(m) for m in masks] + [np.full((extra, words), 0xffffffff, np.uint32)])
            self.mask_p = gpu.put(w)
        self.gate = np.float32(rng.standard_normal((self.s.rows, heads + 1))) if gate else None
        self.vt = rope_tables(gpu, v, 64, 50.0) if vrot else None
        self.pos = rng.integers(0, 64, self.s.rows)
        self.ldo = ldo or heads * v
        self.out, _ = store(gpu, np.full((self.s.rows, self.ldo), 7.0), dtype)
        self.scratch = gpu.space(gpu.d.det_f_tree_scratch_bytes(heads, kv, v, self.s.max_nodes))

    def op(self):
        return self.libs.FTreeOp(heads=self.H, kv_heads=self.G, dim=self.d, vdim=self.v, scale=self.scale, cap=self.cap, dtype=code(self.libs, self.dtype),
                                 q=self.qp, mask=self.mask_p, mask_ld=self.mask_ld if self.mask_p else 0,
                                 gate=self.gpu.f32(self.gate) if self.gate is not None else None, ldg=self.H + 1, pos=ints(self.gpu, self.pos), rope_len=64,
                                 vrope_cos=self.vt[0] if self.vt else None, vrope_sin=self.vt[1] if self.vt else None, out=self.out, ldo=self.ldo,
                                 scratch=self.scratch, seq=self.s.ref(self.caches))

    def call(self, flags=0):
        self.out, _ = store(self.gpu, np.full((self.s.rows, self.ldo), 7.0), self.dtype)
        op = self.op()
        self.gpu.d.det_debug_set_float(flags)
        try:
            assert self.gpu.d.det_f_tree_attn(C.byref(op), None) == 0
        finally:
            self.gpu.d.det_debug_set_float(0)
        return load(self.gpu, self.out, (self.s.rows, self.ldo), self.dtype)

    def call_each(self):
        """The outputs of every kernel of the type (bfloat16: the one for many rows, the one for few)."""
        return [self.call(f) for f in ((0,) if self.dtype == "f32" else (16, 32))]

    def check_each(self):
        for got in self.call_each():
            self.check(got)

    def seen(self, b):
        a, n = self.s.lens[b], self.s.nodes[b]
        m = self.masks[b] if self.masks is not None else np.tril(np.ones((n, n), bool))
        return np.concatenate([np.ones((n, a), bool), m], 1)

    def check(self, got, rows=None):
        """Every owned row (or every row of the sequences `rows`) within the bound, the others as they were."""
        H, G, d, v, kd, vd = self.H, self.G, self.d, self.v, self.kd, self.vd
        for b, (a, n) in enumerate(zip(self.s.lens, self.s.nodes)):
            if n == 0:
                continue
            r = slice(self.s.first[b], self.s.first[b] + n)
            if rows is not None and b not in rows:
                assert (got[r] == 7.0).all()
                continue
            c, seen = self.values[b], self.seen(b)
            for h in range(H):
                g = h * G // H
                out, weight, size = to.attend(self.q[r, h, :d], c[:a + n, g * kd:g * kd + d], c[:a + n, G * kd + g * vd:G * kd + g * vd + v], seen, self.scale)
                tol = to.attention_bound(out, weight, size, d, a + n, self.dtype)
                if self.vt:
                    tol = np.repeat(tol[:, 0::2] + tol[:, 1::2], 2, 1) * (1 + 8 * U32)
                    out = np.stack([to.rotate(out[i], self.vt[2][self.pos[r][i]], -self.vt[3][self.pos[r][i]], False) for i in range(n)])
                if self.gate is not None:
                    w = 1 / (1 + np.exp(-self.gate[r, h].astype(float)))[:, None]
                    out, tol = out * w, tol * w + 8 * U32 * np.abs(out * w)
                if self.dtype == "bf16":
                    tol = tol + to.U16 * np.abs(out)
                err = np.abs(got[r, h * v:(h + 1) * v] - out)
                assert (err <= tol).all(), (b, h, (err / tol).max(), err.max())
        assert (got[self.s.owned:] == 7.0).all()
        assert (got[:, H * v:] == 7.0).all()


def random_masks(nodes, rng, empty=0.0):
    """Trees, with some rows that attend nothing of their own tree (padding)."""
    out = []
    for n in nodes:
        m = to.tree_mask([int(rng.integers(-1, i)) if i else -1 for i in range(n)])
        m[rng.random(n) < empty] = False
        out.append(m)
    return out


HEADS = [(6, 2, 40, 24), (1, 1, 16, 8), (5, 5, 20, 12), (3, 1, 11, 30), (20, 1, 64, 64), (8, 2, 128, 128), (4, 4, 72, 136), (2, 1, 256, 200), (2, 2, 24, 256),
         (4, 2, 192, 128), (7, 1, 112, 112), (2, 1, 1, 1)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_attention_of_trees(heads, dtype, gpu, libs):
    rng = np.random.default_rng(sum(heads))
    for lens, nodes, extra in [([0], [1], 0), ([1], [1], 0), ([130], [7], 0), ([0, 63, 64, 65, 200, 5], [3, 1, 16, 0, 33, 2], 2), ([700], [64], 1)]:
        a = Attn(gpu, libs, dtype, *heads, lens, nodes, masks=random_masks(nodes, rng), extra=extra, seed=len(nodes))
        a.check_each()
    assert size_error(gpu) == 0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads", [(6, 2, 40, 24), (8, 2, 128, 128), (2, 1, 256, 200), (20, 1, 64, 64)], ids=str)
def test_attention_of_runs(heads, dtype, gpu, libs):
    """No mask: prompts and single tokens, at the edges of the tiles."""
    for lens, nodes in [([0], [1]), ([127], [1]), ([128], [1]), ([0], [200]), ([61, 0, 300], [70, 129, 1]), ([5], [333])]:
        a = Attn(gpu, libs, dtype, *heads, lens, nodes, seed=lens[0], ldo=heads[0] * heads[3] + 5)
        a.check_each()
    assert size_error(gpu) == 0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_that_attend_nothing(dtype, gpu, libs):
    """Padding rows behind no cache get zeros; behind a cache they attend the cache alone; NaN where nobody looks has no influence."""
    rng = np.random.default_rng(4)
    for lens in ([0, 0, 90], [0, 0, 0]):
        nodes = [9, 40, 20]
        masks = random_masks(nodes, rng, empty=0.4)
        masks[0][:] = False
        a = Attn(gpu, libs, dtype, 4, 2, 64, 64, lens, nodes, masks=masks)
        for got in a.call_each():
            a.check(got)
            assert (got[:9] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf], ids=str)
def test_values_that_are_not_finite_stay_with_the_rows_that_attend_them(bad, dtype, gpu, libs):
    """A node's value row is not finite: its own row and its descendants' get it, its siblings' and ancestors' do not."""
    n, a0 = 37, 90
    parents = [-1] + [(i - 1) // 2 for i in range(1, n)]
    m = to.tree_mask(parents)
    a = Attn(gpu, libs, dtype, 4, 2, 64, 64, [a0], [n], masks=[m])
    c = a.values[0].copy()
    node, col = 6, 5
    c[a0 + node, 2 * 64 + col] = bad                           # one element of key/value head 0
    c[a0 + 9, :64] = np.nan                                    # the key of another node, in the same head
    a.caches[0], a.values[0] = store(gpu, c, dtype)
    hit, lost = m[:, node], m[:, 9]
    for got in a.call_each():
        for h in range(4):
            x = got[:, h * 64:(h + 1) * 64]
            if h >= 2:
                assert np.isfinite(x).all()
                continue
            assert np.isnan(x[lost]).all()
            assert np.isfinite(np.delete(x[~lost], col, 1)).all()
            assert np.isfinite(x[~lost & ~hit]).all()
            one = x[hit & ~lost, col]
            assert (np.isnan(one) if np.isnan(bad) else one == bad).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("masked", [0, 1])
def test_values_of_the_cache_that_are_not_finite_reach_every_row(masked, dtype, gpu, libs):
    """A cached value beside the tree (in the same tile, and far ahead of it) is attended by every row; in a run a token's value reaches
    the tokens from it on."""
    rng = np.random.default_rng(12)
    for at, bad in [(149, np.inf), (3, -np.inf), (148, np.nan)]:
        a = Attn(gpu, libs, dtype, 2, 1, 64, 64, [150], [40], masks=random_masks([40], rng) if masked else None)
        c = a.values[0].copy()
        c[at, 64 + 9] = bad
        c[150 + 30, 64 + 20] = bad                             # node 30
        a.caches[0], a.values[0] = store(gpu, c, dtype)
        hit = a.seen(0)[:, 150 + 30]
        for got in a.call_each():
            for x in np.moveaxis(got.reshape(40, 2, 64), 1, 0):
                assert (np.isnan(x[:, 9]) if np.isnan(bad) else x[:, 9] == bad).all()
                assert (np.isnan(x[hit, 20]) if np.isnan(bad) else x[hit, 20] == bad).all()
                assert np.isfinite(np.delete(x, [9, 20], 1)).all() and np.isfinite(x[~hit, 20]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gates_and_rotated_values(dtype, gpu, libs):
    rng = np.random.default_rng(2)
    for gate, vrot in [(1, 0), (0, 1), (1, 1)]:
        for heads, lens, nodes in [((6, 2, 40, 24), [5, 300], [4, 13]), ((8, 2, 128, 128), [2000, 64], [20, 1]), ((2, 1, 64, 256), [100], [90])]:
            a = Attn(gpu, libs, dtype, *heads, lens, nodes, masks=random_masks(nodes, rng), gate=gate, vrot=vrot)
            a.check_each()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_long_unequal_contexts_are_shared_out(dtype, gpu, libs):
    """Contexts that many CTAs share next to contexts that one finishes; weights that peak on single keys far away."""
    rng = np.random.default_rng(8)
    lens = [9000, 3, 0, 517, 4100, 64, 2049]
    nodes = [5, 1, 2, 17, 64, 30, 1]
    a = Attn(gpu, libs, dtype, 10, 2, 128, 128, lens, nodes, masks=random_masks(nodes, rng), sharp=4.0)
    a.check_each()
    b = Attn(gpu, libs, dtype, 4, 1, 64, 64, [20000], [1], sharp=3.0)
    b.check_each()
    b.check_each()                                          # the scratch as the first call left it


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads", [(8, 2, 64, 64), (4, 1, 128, 128), (2, 1, 200, 256), (5, 5, 40, 24)], ids=str)
def test_pieces_stay_in_the_scratch(heads, dtype, gpu, libs):
    """Every CTA leaves pieces; what lies behind det_f_tree_scratch_bytes stays as it was."""
    rng = np.random.default_rng(sum(heads))
    for lens, nodes in [([7000], [16]), ([2500, 900, 3100], [64, 70, 12]), ([3000], [300])]:
        masks = random_masks(nodes, rng) if nodes[0] < 100 else None
        a = Attn(gpu, libs, dtype, *heads, lens, nodes, masks=masks)
        n, guard = gpu.d.det_f_tree_scratch_bytes(heads[0], heads[1], heads[3], max(nodes)), 4096
        a.scratch = gpu.space(n + guard)
        gpu.d.det_memset(a.scratch + n, 0x5a, guard, None)
        a.check_each()
        assert (gpu.get(a.scratch + n, guard, np.uint8) == 0x5a).all()


@pytest.mark.parametrize("heads", [(4, 4, 64, 64), (6, 3, 40, 24), (1, 1, 16, 8), (5, 1, 96, 96), (2, 1, 128, 256), (3, 1, 24, 200)], ids=str)
def test_few_rows_of_long_and_short_contexts_in_32_bits(heads, gpu, libs):
    """Up to 16 rows of a key/value head: the kernel that spreads the keys over its warps (larger values, or many tiles) and the other one,
    with masks, values that are not finite, and NaN that nobody attends."""
    rng = np.random.default_rng(heads[0] * heads[3])
    for lens, nodes in [([40], [1]), ([33, 0, 700], [3, 2, 1]), ([30000, 29000], [2, 1])]:
        a = Attn(gpu, libs, "f32", *heads, lens, nodes, masks=random_masks(nodes, rng), sharp=2.0)
        a.check_each()
    for max_len in (0, 10 ** 6):                               # either choice for the same rows
        a = Attn(gpu, libs, "f32", *heads, [300], [3], masks=[np.eye(3, dtype=bool)])
        a.s.max_len = max_len
        a.check_each()
        H, G, d, v = heads
        c = a.values[0].copy()
        at = 302 - 1, G * round8(d) + v - 1                    # the last value of node 1, which node 1 alone attends
        c[at] = np.inf
        a.caches[0], a.values[0] = store(gpu, c, "f32")
        got = a.call().reshape(3, H, v)
        hit = np.arange(H) * G // H == 0 if G > 1 else np.ones(H, bool)
        assert (got[1, hit, v - 1] == np.inf).all() and np.isfinite(got[[0, 2]]).all() and np.isfinite(got[1, :, :v - 1]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_small_sequences(dtype, gpu, libs):
    rng = np.random.default_rng(5)
    nodes = [int(n) for n in rng.integers(0, 4, 300)]
    lens = [int(n) for n in rng.integers(0, 150, 300)]
    a = Attn(gpu, libs, dtype, 4, 2, 32, 32, lens, nodes, masks=random_masks(nodes, rng), extra=4)
    a.check_each()


def test_results_repeat_and_do_not_depend_on_the_bounds(gpu, libs):
    rng = np.random.default_rng(6)
    nodes, lens = [6, 3, 1], [3000, 17, 800]
    masks = random_masks(nodes, rng)
    a = Attn(gpu, libs, "bf16", 8, 2, 128, 128, lens, nodes, masks=masks)
    for flags in (0, 16, 32):
        assert np.array_equal(a.call(flags), a.call(flags))
    for bound in (0, 100000):
        a.s.max_len = bound
        a.check(a.call())
        a.check_each()


def test_sequences_that_do_not_fit_are_left_out(gpu, libs):
    rng = np.random.default_rng(7)
    for dtype in ("f32", "bf16"):
        for lens, nodes, cap, max_nodes, bad in [([50, 20], [8, 4], 52, 8, 0), ([10, 20], [8, 4], 60, 6, 0), ([-5, 20], [8, 4], 60, 8, 0)]:
            good = [max(x, 0) for x in lens]
            a = Attn(gpu, libs, dtype, 4, 2, 64, 64, good, nodes, masks=random_masks(nodes, rng), cap=70)
            a.s.max_nodes = max_nodes
            op = a.op()
            op.cap, op.seq.len = cap, ints(gpu, lens)
            # the caches keep 70 rows: a smaller cap only narrows what may be read
            for flags in (16, 32):
                gpu.d.det_debug_set_float(flags)
                assert gpu.d.det_f_tree_attn(C.byref(op), None) == 0
                gpu.d.det_debug_set_float(0)
                assert size_error(gpu) == SIZE_ERROR
                a.check(load(gpu, a.out, (a.s.rows, a.ldo), dtype), rows={1 - bad})


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_largest_bounds(dtype, gpu, libs):
    """A caller that bounds nothing (cap and max_len the largest int): results as ever, and a length that no tile count fits is left out
    without a look at its cache."""
    rng = np.random.default_rng(17)
    nodes, top = [8, 4], 2 ** 31 - 1
    a = Attn(gpu, libs, dtype, 4, 2, 64, 64, [50, 20], nodes, masks=random_masks(nodes, rng))
    op = a.op()
    op.cap, op.seq.max_len = top, top
    for lens, rows in [([50, 20], None), ([top - 100, 20], {1}), ([top - 8, 20], {1})]:
        op.seq.len = ints(gpu, lens)
        for flags in (0, 16, 32):
            op.out = a.out = store(gpu, np.full((a.s.rows, a.ldo), 7.0), dtype)[0]
            gpu.d.det_debug_set_float(flags)
            assert gpu.d.det_f_tree_attn(C.byref(op), None) == 0
            gpu.d.det_debug_set_float(0)
            assert size_error(gpu) == (0 if rows is None else SIZE_ERROR)
            a.check(load(gpu, a.out, (a.s.rows, a.ldo), dtype), rows=rows)


def test_a_run_equals_the_attention_op_of_the_models(gpu, libs):
    """The same projections through det_f_attn and through det_f_qk_rope + det_f_tree_attn, over the same kind of cache."""
    H, G, d, v, n = 6, 2, 64, 64, 150
    rng = np.random.default_rng(9)
    y = np.float32(rng.standard_normal((n, H * d + G * (d + v))))
    kt, vt = rope_tables(gpu, d, 200, 100.0), rope_tables(gpu, v, 200, 70.0)
    cap = 160
    out, cache = [], []
    for dtype in ("f32", "bf16"):
        c1, c2 = (gpu.space(4 * cap * gpu.d.det_f_attn_ld(G, d, v)) for _ in range(2))
        q, o = gpu.space(4 * n * H * d), gpu.space(4 * n * H * v)
        yp = gpu.f32(y)
        tables = dict(rope_cos=kt[0], rope_sin=kt[1], vrope_cos=vt[0], vrope_sin=vt[1])
        op = libs.FAttnOp(heads=H, kv_heads=G, dim=d, vdim=v, rot_dims=d, scale=0.2, cap=cap, M=n, dtype=code(libs, dtype), y=yp, ldy=y.shape[1], q_off=0,
                          k_off=H * d, v_off=(H + G) * d, gate_off=-1, q=q, out=o, ldo=H * v, max_pos=n - 1,
                          scratch=gpu.space(gpu.d.det_f_attn_scratch_bytes(v)), seq=libs.SeqRef(one=libs.SeqSlot(cache=c1)), **tables)
        gpu.d.det_f_attn_prep(C.byref(op), None)
        gpu.d.det_f_attn(C.byref(op), None)
        want, rows = load(gpu, o, (n, H * v), dtype), load(gpu, c1, (cap, G * (d + v)), dtype)
        s = Step(gpu, libs, [0], [n])
        qk = libs.FQkOp(heads=H, kv_heads=G, dim=d, vdim=v, rot_dims=d, half=0, eps=0.0, cap=cap, dtype=code(libs, dtype), y=yp, ldy=y.shape[1], q_off=0,
                        k_off=H * d, v_off=(H + G) * d, rope_len=200, q=q, seq=s.ref([c2]), **tables)
        assert gpu.d.det_f_qk_rope(C.byref(qk), None) == 0
        ta = libs.FTreeOp(heads=H, kv_heads=G, dim=d, vdim=v, scale=0.2, cap=cap, dtype=code(libs, dtype), q=q, out=o, ldo=H * v, pos=ints(gpu, range(n)),
                          rope_len=200, vrope_cos=vt[0], vrope_sin=vt[1], scratch=gpu.space(gpu.d.det_f_tree_scratch_bytes(H, G, v, n)), seq=s.ref([c2]))
        assert gpu.d.det_f_tree_attn(C.byref(ta), None) == 0
        got = load(gpu, o, (n, H * v), dtype)
        assert np.array_equal(load(gpu, c2, (cap, G * (d + v)), dtype), rows)
        # both within the bound of the definition: twice the bound apart (weights sum to 1, values below 5)
        tol = {"f32": 2e-4, "bf16": 4 * to.U16 * 5}[dtype]
        assert np.abs(got - want).max() <= tol


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nodes", [1, 3, 20, 70])
def test_scores_that_rise_and_fall_along_the_keys(nodes, dtype, gpu, libs):
    """The running maximum moves far from tile to tile, by little, or not at all: the reference of the weights follows it."""
    n = 900
    for low, high in [(-40.0, 60.0), (60.0, -40.0), (0.0, 4.0), (-300.0, 300.0), (5.0, 5.0)]:
        a = Attn(gpu, libs, dtype, 4, 1, 64, 64, [n], [nodes], masks=[to.tree_mask(list(range(-1, nodes - 1)))], seed=nodes)
        c = a.values[0].copy()
        ramp = np.linspace(low, high, n + nodes)
        c[:n + nodes, :64] *= 0.1
        c[:n + nodes, 0] = ramp                                # the first element carries the trend (q's is 8: scale * 8 = 1)
        a.caches[0], a.values[0] = store(gpu, c, dtype)
        q = a.q.copy()
        q[..., 0] = 8.0
        a.qp, a.q = store(gpu, q, dtype)
        a.check_each()
    assert size_error(gpu) == 0


def test_rows_behind_the_fourth_gigabyte(gpu, libs):
    """Byte offsets inside one cache pass 32 bits: rows are written, moved and attended there by every kernel."""
    H, G, d = 8, 8, 128
    for dtype, esize in (("bf16", 2), ("f32", 4)):
        ld = gpu.d.det_f_attn_ld(G, d, d)
        at = (1 << 32) // (ld * esize) + 1000
        cap = at + 300
        cache = gpu.d.det_malloc(cap * ld * esize)
        assert cache
        rng = np.random.default_rng(5)
        for nodes in (2, 40, 200):
            s = Step(gpu, libs, [at], [nodes])
            ref = s.ref([cache])
            y = np.float32(rng.standard_normal((nodes, (H + 2 * G) * d)))
            y[:, H * d:(H + G) * d] = 0.0                      # keys of zero: a row's weights are even over everything it sees
            y[:, :H * d] *= 0.1
            q, out = gpu.space(4 * nodes * H * d), gpu.space(4 * nodes * H * d)
            qk = libs.FQkOp(heads=H, kv_heads=G, dim=d, vdim=d, rot_dims=0, half=0, eps=0.0, cap=cap, dtype=code(libs, dtype), y=gpu.f32(y), ldy=y.shape[1],
                            q_off=0, k_off=H * d, v_off=(H + G) * d, q=q, seq=ref)
            assert gpu.d.det_f_qk_rope(C.byref(qk), None) == 0
            m = to.tree_mask([-1] * nodes)                     # every node by itself
            ta = libs.FTreeOp(heads=H, kv_heads=G, dim=d, vdim=d, scale=1.0, cap=cap, dtype=code(libs, dtype), q=q, mask=gpu.put(to.bits(m, 7)), mask_ld=7,
                              out=out, ldo=H * d, scratch=gpu.space(gpu.d.det_f_tree_scratch_bytes(H, G, d, nodes)), seq=ref)
            assert gpu.d.det_f_tree_attn(C.byref(ta), None) == 0
            got = load(gpu, out, (nodes, H * d), dtype)
            v = y[:, (H + G) * d:].astype(float)
            if dtype == "bf16":
                v = ho.bf16_values(ho.bf16_bits(np.float32(v))).astype(float)
            # all other keys and values are zero: the weight is 1 / (at + 1), known to 2 u_act and the sum of `at` terms in fp32
            want = v / (at + 1)
            tol = np.abs(want) * (4 * to.UNIT[dtype] + (at / 16 + 100) * U32) + 1e-12
            assert (np.abs(got - want) <= tol).all(), np.abs(got / np.where(want == 0, 1, want) - 1).max()
            kept = [1, nodes - 1] if nodes > 2 else [1]
            op = libs.FKeepOp(caches=1, seqs=1, cap=cap, row_bytes=ld * esize, table=ref.table, len=s.len_p, keep=ints(gpu, kept), keep_ld=2,
                              count=ints(gpu, [len(kept)]), max_count=2)
            assert gpu.d.det_f_tree_keep(C.byref(op), None) == 0
            rows = np.zeros((len(kept), ld), np.uint16 if esize == 2 else np.float32)
            gpu.d.det_memcpy(rows.ctypes.data, cache + at * ld * esize, rows.nbytes, None)
            gpu.d.det_sync()
            rows = ho.bf16_values(rows).astype(float) if esize == 2 else rows.astype(float)
            assert np.array_equal(rows[:, G * d:], v[kept])
            gpu.d.det_memset(cache + at * ld * esize, 0, 250 * ld * esize, None)
        gpu.d.det_free(cache)
    assert size_error(gpu) == 0


def test_calls_on_two_streams_and_replays_of_two_graphs(gpu, libs):
    """Calls with scratch of their own overlap on two streams; two captured calls that share scratch are replayed in turn, with other
    lengths."""
    rt = C.CDLL("libcudart.so.12")
    streams = [C.c_void_p() for _ in range(2)]
    for s in streams:
        assert rt.cudaStreamCreateWithFlags(C.byref(s), 1) == 0
    rng = np.random.default_rng(11)
    cases = [Attn(gpu, libs, "bf16", 16, 2, 128, 128, [6000, 40], [30, 5], masks=random_masks([30, 5], rng), seed=i) for i in range(2)]
    ops = [a.op() for a in cases]
    gpu.d.det_sync()
    for _ in range(20):
        for op, s in zip(ops, streams):
            assert gpu.d.det_f_tree_attn(C.byref(op), s) == 0
    gpu.d.det_sync()
    for a in cases:
        a.check(load(gpu, a.out, (a.s.rows, a.ldo), "bf16"))
    for s in streams:
        assert rt.cudaStreamDestroy(s) == 0
    graphs = []
    for op in ops:
        op.scratch = ops[0].scratch
        gpu.d.det_graph_begin()
        assert gpu.d.det_f_tree_attn(C.byref(op), None) == 0
        graphs.append(gpu.d.det_graph_end())
        assert graphs[-1]
    for lens in ([6000, 40], [77, 3000], [0, 129], [6000, 40]):
        for a in cases:
            fits = [min(x, a.cap - n) for x, n in zip(lens, a.s.nodes)]
            b = np.array(fits, np.int32)
            gpu.d.det_memcpy(a.s.len_p, b.ctypes.data, 8, None)
            gpu.d.det_sync()
            a.s.lens = fits
            for i, (n, first) in enumerate(zip(a.s.nodes, fits)):   # every row of the cache holds something
                c = np.nan_to_num(a.values[i], nan=0.5)
                a.values[i] = c
                bits = ho.bf16_bits(np.float32(c))
                gpu.d.det_memcpy(a.caches[i], bits.ctypes.data, bits.nbytes, None)
                gpu.d.det_sync()
        for g in (graphs[0], graphs[1], graphs[1], graphs[0]):
            gpu.d.det_graph_launch(g)
        gpu.d.det_sync()
        for a in cases:
            a.check(load(gpu, a.out, (a.s.rows, a.ldo), "bf16"))
    for g in graphs:
        gpu.d.det_graph_free(g)


def test_calls_from_two_threads(gpu, libs):
    """Two host threads queue calls of the same kernels with other sizes (other shared memory) at once: none is refused, all are right."""
    rng = np.random.default_rng(31)
    rt = C.CDLL("libcudart.so.12")
    for dtype in ("f32", "bf16"):
        cases = [Attn(gpu, libs, dtype, *heads, [70, 300], [9, 3], masks=random_masks([9, 3], rng)) for heads in [(4, 2, 16, 128), (4, 2, 128, 128)]]
        streams, ops = [C.c_void_p() for _ in cases], [a.op() for a in cases]
        for s in streams:
            assert rt.cudaStreamCreateWithFlags(C.byref(s), 1) == 0
        for flags in (16, 32):
            gpu.d.det_debug_set_float(flags)
            gpu.d.det_sync()
            codes = [[], []]
            threads = [threading.Thread(target=lambda i=i: codes[i].extend(gpu.d.det_f_tree_attn(C.byref(ops[i]), streams[i]) for _ in range(300))) for i in (0, 1)]
            for t in threads:
                t.start()
            for t in threads:
                t.join()
            gpu.d.det_debug_set_float(0)
            assert rt.cudaDeviceSynchronize() == 0
            assert codes == [[0] * 300] * 2
            for a in cases:
                a.check(load(gpu, a.out, (a.s.rows, a.ldo), dtype))
        for s in streams:
            assert rt.cudaStreamDestroy(s) == 0


# ------------------------------------------------------------------------------------------------------------------ kept rows
@pytest.mark.parametrize("row_bytes", [16, 48, 4096, 4112])
def test_kept_rows_move_up(row_bytes, gpu, libs):
    rng = np.random.default_rng(row_bytes)
    layers, cap = 3, 70
    lens = [0, 5, 30, 61, 8]
    lists = [[0], [], [0, 1, 2, 5, 6, 9, 12, 20, 21, 33], [8], list(range(40))]
    width = row_bytes // 4
    caches = rng.standard_normal((layers * len(lens), cap, width)).astype(np.float32)
    ptr = [gpu.put(c) for c in caches]
    keep = np.full((len(lens), 45), -9, np.int32)
    for b, k in enumerate(lists):
        keep[b, :len(k)] = k
    out = ints(gpu, [-1] * len(lens))
    op = libs.FKeepOp(caches=len(ptr), seqs=len(lens), cap=cap, row_bytes=row_bytes, table=slots(gpu, libs, ptr), len=ints(gpu, lens), keep=gpu.put(keep),
                      keep_ld=45, count=ints(gpu, [len(k) for k in lists]), max_count=40, len_out=out)
    assert gpu.d.det_f_tree_keep(C.byref(op), None) == 0
    for e, p in enumerate(ptr):
        b = e % len(lens)
        want = caches[e].copy()
        for i, k in enumerate(lists[b]):
            want[lens[b] + i] = caches[e][lens[b] + k]
        assert np.array_equal(gpu.get(p, (cap, width)), want)
    assert np.array_equal(gpu.get(out, len(lens), np.int32), [a + len(k) for a, k in zip(lens, lists)])
    assert size_error(gpu) == 0


def test_lists_that_do_not_fit_move_nothing(gpu, libs):
    cap, width = 20, 8
    rng = np.random.default_rng(1)
    good = [0, 2, 3]
    for length, bad in [(5, [0, 2, 2]), (5, [3, 1]), (5, [-1, 2]), (5, [0, 15]), (-3, [0, 1]), (19, [0, 1]), (21, []), (5, [0, 1, 2, 3, 4])]:
        caches = rng.standard_normal((2, cap, width)).astype(np.float32)
        ptr = [gpu.put(c) for c in caches]
        keep = np.full((2, 6), 0, np.int32)
        keep[0, :len(bad)], keep[1, :3] = bad, good
        out = ints(gpu, [-1, -1])
        op = libs.FKeepOp(caches=2, seqs=2, cap=cap, row_bytes=width * 4, table=slots(gpu, libs, ptr), len=ints(gpu, [length, 4]), keep=gpu.put(keep), keep_ld=6,
                          count=ints(gpu, [len(bad), 3]), max_count=4, len_out=out)
        assert gpu.d.det_f_tree_keep(C.byref(op), None) == 0
        assert size_error(gpu) == SIZE_ERROR
        assert np.array_equal(gpu.get(ptr[0], (cap, width)), caches[0])
        want = caches[1].copy()
        want[[4, 5, 6]] = caches[1][[4, 6, 7]]
        assert np.array_equal(gpu.get(ptr[1], (cap, width)), want)
        assert np.array_equal(gpu.get(out, 2, np.int32), [-1, 7])


# ------------------------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_drafting_equals_decoding_token_by_token(dtype, half, gpu, libs):
    """Prompts of two sequences, a tree behind each, the accepted paths kept, then one more token: the accepted nodes' rows and the last
    token's equal the same tokens as plain runs.  The steps of the tree are captured once and replayed with other lengths."""
    H, G, d, v, rot, cap = 6, 2, 64, 48, 32, 220
    width = H * d + G * (d + v)
    rng = np.random.default_rng(3)
    kd, vd = round8(d), round8(v)
    ld = G * (kd + vd)
    esize = 4 if dtype == "f32" else 2
    ntab = 256
    cs, sn = gpu.space(4 * ntab * rot // 2), gpu.space(4 * ntab * rot // 2)
    rope = libs.FRopeOp(dims=rot, scaling=libs.DET_ROPE_RAMP, base=1000.0, factor=2.0, orig_ctx=64.0, low=1.0, high=8.0, mscale=1.0, n=ntab, cos=cs, sin=sn)
    assert gpu.d.det_f_rope_table(C.byref(rope), None) == 0
    qn, kn = gpu.f32(rng.uniform(0.5, 1.5, d)), gpu.f32(rng.uniform(0.5, 1.5, d))
    parents = [[-1, 0, 0, 1, 1, 2, 3, 6, -1, 8], [-1, -1, 1, 2, 2, 3]]
    paths = [[0, 1, 3, 6, 7], [1, 2, 3, 5]]
    masks = [to.tree_mask(p) for p in parents]
    prompts, nodes = [100, 31], [10, 6]
    max_nodes = 16

    def runner(caches):
        """Buffers of a step that can be captured: `call` queues it, `fill` gives it rows."""
        rows = 2 * max_nodes
        y, q, out = gpu.space(4 * rows * width), gpu.space(4 * rows * H * kd), gpu.space(4 * rows * H * v)
        first, lens, pos, mask = gpu.space(12), gpu.space(8), gpu.space(4 * rows), gpu.space(4 * rows)
        ref = libs.TreeRef(table=slots(gpu, libs, caches), first=first, len=lens, seqs=2, rows=rows, max_nodes=max_nodes, max_len=cap)
        qk = libs.FQkOp(heads=H, kv_heads=G, dim=d, vdim=v, rot_dims=rot, half=half, eps=1e-6, q_norm=qn, k_norm=kn, cap=cap, dtype=code(libs, dtype), y=y,
                        ldy=width, q_off=0, k_off=H * d, v_off=(H + G) * d, rope_len=ntab, rope_cos=cs, rope_sin=sn, pos=pos, q=q, seq=ref)
        ta = libs.FTreeOp(heads=H, kv_heads=G, dim=d, vdim=v, scale=0.3, cap=cap, dtype=code(libs, dtype), q=q, mask=mask, mask_ld=1, out=out, ldo=H * v,
                          scratch=gpu.space(gpu.d.det_f_tree_scratch_bytes(H, G, v, max_nodes)), seq=ref)
        keep = [qk, ta]

        def call():
            assert gpu.d.det_f_qk_rope(C.byref(keep[0]), None) == 0
            assert gpu.d.det_f_tree_attn(C.byref(keep[1]), None) == 0

        def put(p, a):
            a = np.ascontiguousarray(a)
            gpu.d.det_memcpy(p, a.ctypes.data, a.nbytes, None)
            gpu.d.det_sync()

        def fill(rows_y, at, seen, positions):
            put(first, np.array([0, len(rows_y[0]), len(rows_y[0]) + len(rows_y[1])], np.int32))
            put(lens, np.array(at, np.int32))
            put(pos, np.array(positions, np.int32))
            put(mask, np.concatenate([to.bits(m, 1) for m in seen if len(m)]))
            put(y, np.concatenate(rows_y).astype(np.float32))

        def read():
            n = rows * H * v
            a = load(gpu, out, (n,), dtype)
            return a.reshape(rows, H * v)
        return call, fill, read, lens, ref

    def depth(p):
        out = []
        for x in p:
            out.append(0 if x < 0 else out[x] + 1)
        return out

    text = [rng.standard_normal((n, width)) for n in prompts]
    draft = [rng.standard_normal((n, width)) for n in nodes]
    final = [rng.standard_normal((1, width)) for _ in nodes]
    chain = lambda n: np.tril(np.ones((n, n), bool))  # noqa: E731

    # the tree
    caches = [gpu.space(cap * ld * esize) for _ in range(2)]
    call, fill, read, lens_p, ref = runner(caches)
    gpu.d.det_sync()
    gpu.d.det_graph_begin()
    call()
    graph = gpu.d.det_graph_end()
    assert graph

    def feed(run, which, at0):
        """Sequence rows through the step in portions of max_nodes."""
        at = list(at0)
        done = [0, 0]
        while any(done[b] < len(which[b]) for b in range(2)):
            part = [which[b][done[b]:done[b] + max_nodes] for b in range(2)]
            pos = np.concatenate([at[b] + np.arange(len(part[b])) for b in range(2)])
            run(part, at, [chain(len(p)) for p in part], pos)
            for b in range(2):
                done[b] += len(part[b])
                at[b] += len(part[b])
        return at

    def replay(part, at, seen, pos):
        fill(part, at, seen, pos)
        gpu.d.det_graph_launch(graph)
        gpu.d.det_sync()

    at = feed(replay, text, [0, 0])
    assert at == prompts
    pos = np.concatenate([at[b] + np.array(depth(parents[b])) for b in range(2)])
    replay(draft, at, masks, pos)
    tree = read()
    count, kept = ints(gpu, [len(p) for p in paths]), np.zeros((2, 8), np.int32)
    for b, p in enumerate(paths):
        kept[b, :len(p)] = p
    new_len = gpu.space(8)
    op = libs.FKeepOp(caches=2, seqs=2, cap=cap, row_bytes=ld * esize, table=ref.table, len=lens_p, keep=gpu.put(kept), keep_ld=8, count=count, max_count=8,
                      len_out=new_len)
    assert gpu.d.det_f_tree_keep(C.byref(op), None) == 0
    at = list(gpu.get(new_len, 2, np.int32))
    assert at == [prompts[b] + len(paths[b]) for b in range(2)]
    replay(final, at, [chain(1)] * 2, at)
    last = read()

    # the same tokens one after the other
    plain = [gpu.space(cap * ld * esize) for _ in range(2)]
    call2, fill2, read2, _, _ = runner(plain)
    rows = [[], []]

    def direct(part, at, seen, pos):
        fill2(part, at, seen, pos)
        call2()
        got = read2()
        rows[0].extend(got[:len(part[0])])
        rows[1].extend(got[len(part[0]):len(part[0]) + len(part[1])])

    feed(direct, [np.concatenate([text[b], draft[b][paths[b]], final[b]]) for b in range(2)], [0, 0])
    for b in range(2):
        first = 0 if b == 0 else nodes[0]
        # both sides within the op's bound of the same values: weights sum to 1, values below 5
        tol = {"f32": 2e-4, "bf16": 4 * to.U16 * 5}[dtype]
        for i, node in enumerate(paths[b]):
            assert np.abs(tree[first + node] - rows[b][prompts[b] + i]).max() <= tol
        assert np.abs(last[b] - rows[b][-1]).max() <= tol
        assert np.array_equal(load(gpu, caches[b], (cap, ld), dtype)[:at[b] + 1], load(gpu, plain[b], (cap, ld), dtype)[:at[b] + 1])
    gpu.d.det_graph_free(graph)
    assert size_error(gpu) == 0
