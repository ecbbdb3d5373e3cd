"""Cases of the operators that a step of drafted tokens needs over a key/value cache, each in a plain form (elementary torch
operations) and as the call of this library's entry point:

  table   det_f_rope_table   cosines and sines of the position rotation, with the scalings for long contexts
  prep    det_f_qk_rope      norm of every query and key head, rotation, and the rows' entries in the caches, in one pass
  attn    det_f_tree_attn    attention of the rows (a token, a prompt, a tree of drafted tokens) of several sequences over their caches
  keep    det_f_tree_keep    the accepted rows of every tree move to the end of the cache proper, in all layers

`own` chooses: False, the plain form; True, the library.  Sizes: 40 query and 8 key/value heads of 128 with contexts of 512 to 8192
in batches of 32 are the serving shapes of bench.py; the others are generic.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
SCALINGS = {"none": 0, "linear": 1, "base": 2, "ramp": 3}


def round8(n):
    return (n + 7) // 8 * 8


# ---------------------------------------------------------------------------------------------------------------- cases
def _attn(name, heads, kv, dim, vdim, dtype, seqs, lo, hi, nodes, tree, **more):
    return dict(name=name, op="attn", heads=heads, kv=kv, dim=dim, vdim=vdim, dtype=dtype, seqs=seqs, lo=lo, hi=hi, nodes=nodes,
                tree=tree, gate=more.get("gate", False), vrot=more.get("vrot", False), padded=more.get("padded", False))


def _prep(name, heads, kv, dim, vdim, rot, half, norm, dtype, seqs, lo, hi, nodes, **more):
    return dict(name=name, op="prep", heads=heads, kv=kv, dim=dim, vdim=vdim, rot=rot, half=half, norm=norm, dtype=dtype, seqs=seqs,
                lo=lo, hi=hi, nodes=nodes, vrot=more.get("vrot", False))


def _table(name, dims, n, pos0, base, scaling, factor, orig, mscale):
    return dict(name=name, op="table", dims=dims, n=n, pos0=pos0, base=base, scaling=scaling, factor=factor, orig=orig, low=1.0,
                high=32.0, mscale=mscale)


def _keep(name, kv, dim, vdim, seqs, layers, lo, hi, nodes, most):
    return dict(name=name, op="keep", kv=kv, dim=dim, vdim=vdim, seqs=seqs, layers=layers, lo=lo, hi=hi, nodes=nodes, most=most)


def listed():
    return [
        # one token of one sequence: what a decoded token costs when nothing was drafted; latency counts
        _attn("attn token 2k", 40, 8, 128, 128, "bf16", 1, 2048, 2048, 1, False),
        # a wide tree over one long conversation
        _attn("attn tree 61 at 32k", 40, 8, 128, 128, "bf16", 1, 32749, 32749, 61, True),
        # a serving step: 32 conversations of unequal length, trees padded to one size so that the step can be captured
        _attn("attn 32 trees of 16", 40, 8, 128, 128, "bf16", 32, 512, 8192, 16, True, padded=True),
        # a prompt behind an earlier conversation
        _attn("attn prompt 2048 at 6k", 40, 8, 128, 128, "bf16", 1, 6144, 6144, 2048, False),
        # 32-bit activations, odd head sizes, an output gate and rotated values
        _attn("attn f32 odd heads", 6, 2, 40, 24, "f32", 5, 100, 3001, 13, True, gate=True, vrot=True),
        # one token's rows
        _prep("prep token", 40, 8, 128, 128, 128, False, True, "bf16", 1, 2048, 2048, 1),
        # a serving step's rows in 32 bits, part of the head rotated, halves
        _prep("prep 32 trees of 16 f32", 40, 8, 128, 128, 64, True, True, "f32", 32, 512, 1024, 16),
        # a long prompt's rows
        _prep("prep prompt 8192", 40, 8, 128, 128, 128, True, True, "bf16", 1, 37, 37, 8192),
        # tables of a short and of a stretched long context
        _table("table 4096", 64, 4096, 0, 10000.0, "none", 1.0, 4096.0, 1.0),
        _table("table 262144 ramp", 128, 262144, 0, 1000000.0, "ramp", 8.0, 32768.0, 1.2),
        # the accepted path of one tree in 8 layers, and of 32 trees
        _keep("keep 1 path", 8, 128, 128, 1, 8, 300, 300, 61, 9),
        _keep("keep 32 paths", 8, 128, 128, 32, 8, 64, 256, 16, 7),
    ]


def _unnamed(case):
    return {k: v for k, v in case.items() if k != "name"}


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "prep", "prep", "table", "keep"])
    kv = rng.choice([1, 2, 3, 4, 5, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 5, 7, 8])
    dim = rng.choice([40, 64, 72, 80, 96, 112, 128, 128, 128, 192, 256])
    vdim = dim if rng.random() < 0.7 else rng.choice([24, 64, 96, 128])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    seqs = _log(rng, 1, 32)
    hi = _log(rng, 1, 32768)
    lo = rng.choice([hi, hi // 2, hi // 7, 0])
    if op == "attn":
        tree = rng.random() < 0.7
        nodes = _log(rng, 1, 64) if tree else _log(rng, 1, 2048)
        if dtype == "f32":
            nodes = min(nodes, 96)
        while seqs > 1 and (seqs * (hi + nodes) * heads * nodes > 2048 * 8192 * 40 or seqs * (hi + nodes) * kv * (dim + vdim) > 1.0e9):
            seqs = (seqs + 1) // 2
        while heads * nodes * (hi + nodes) * (4 if dtype == "f32" else 1) > 2048 * 8192 * 40:
            hi //= 2
            lo //= 2
        return _unnamed(_attn("", heads, kv, dim, vdim, dtype, seqs, lo, hi, nodes, tree, gate=rng.random() < 0.3, vrot=rng.random() < 0.3,
                     padded=tree and rng.random() < 0.5))
    if op == "prep":
        rows = _log(rng, 1, 8192)
        seqs = min(seqs, rows)
        hi = min(hi, 2048)
        return _unnamed(_prep("", heads, kv, dim, vdim, rng.choice([dim, dim // 2 // 2 * 2, dim // 4 // 2 * 2, 0]), rng.random() < 0.5,
                     rng.random() < 0.7, dtype, seqs, min(lo, hi), hi, max(1, rows // seqs), vrot=rng.random() < 0.3))
    if op == "table":
        dims = 2 * rng.randrange(4, 65)
        return _unnamed(_table("", dims, _log(rng, 1, 262144), rng.choice([0, 0, _log(rng, 1, 100000)]), rng.choice([500.0, 10000.0, 1000000.0]),
                      rng.choice(sorted(SCALINGS)), rng.choice([2.0, 4.0, 8.0, 32.0]), rng.choice([2048.0, 8192.0, 32768.0]),
                      rng.choice([1.0, 1.2])))
    nodes = _log(rng, 2, 64)
    return _unnamed(_keep("", kv, dim, vdim, seqs, rng.randrange(1, 9), min(lo, 128), min(hi, 256), nodes, _log(rng, 1, nodes)))


def _spread(case):
    """Cached rows ahead of the step and rows of the step, per sequence: the same for every seed."""
    n = case["seqs"]
    part = [(0.381966 + 0.618034 * i) % 1.0 for i in range(n)]
    lens = [case["hi"] if i == 0 else int(case["lo"] + (case["hi"] - case["lo"]) * part[i]) for i in range(n)]
    most = case["nodes"]
    nodes = [most if i == 0 or case.get("padded") else 1 + int(part[i] * most) % most for i in range(n)]
    return lens, nodes


def _real(case):
    """Rows of each tree that hold a token; those behind are padding whose mask is empty."""
    _, nodes = _spread(case)
    return [max(1, n - (3 * i) % n) if case.get("padded") else n for i, n in enumerate(nodes)]


# ---------------------------------------------------------------------------------------------------------------- inputs
def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def _ints(a):
    return torch.tensor(np.ascontiguousarray(a), dtype=torch.int32, device=DEV)


def _angles(dims, n, base=10000.0):
    f = base ** (-torch.arange(0, dims, 2, device=DEV, dtype=torch.float64) / max(dims, 1))
    a = torch.arange(n, device=DEV, dtype=torch.float64)[:, None] * f
    return torch.cos(a).float().contiguous(), torch.sin(a).float().contiguous()


def _slots(caches):
    """The table of per-sequence slots (recurrent state, previous row, cache) that the library's ops read."""
    t = torch.zeros(caches.shape[0], 3, dtype=torch.int64)
    t[:, 2] = caches.data_ptr() + torch.arange(caches.shape[0]) * (caches.stride(0) * caches.element_size())
    return t.to(DEV)


def _trees(case, rng):
    """Parents of every row's node (-1: the root, the last cached token) and the rows' masks over their own tree, as words of bits."""
    _, nodes = _spread(case)
    words = (case["nodes"] + 31) // 32
    masks, depth = [], []
    for n, real in zip(nodes, _real(case)):
        m = np.zeros((n, words * 32), bool)
        d = np.zeros(n, np.int64)
        for i in range(real):
            p = int(rng.integers(-1, i)) if i else -1
            if p >= 0:
                m[i], d[i] = m[p], d[p] + 1
            m[i, i] = True
        masks.append(m)
        depth.append(d)
    m = np.concatenate(masks)
    bits = np.packbits(m.reshape(len(m), words, 32), axis=2, bitorder="little").view(np.uint32)[:, :, 0]
    return bits.view(np.int32), np.concatenate(depth)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    rng = np.random.default_rng(seed)
    s = {"case": dict(case)}
    op = case["op"]
    if op == "table":
        # a stream of tables: the base differs a little from state to state, as from model to model
        s["base"] = case["base"] * (1.0 + 0.01 * float(rng.random()))
        s["cos"] = torch.zeros(case["n"], case["dims"] // 2, device=DEV)
        s["sin"] = torch.zeros_like(s["cos"])
        return s
    lens, nodes = _spread(case)
    first = np.concatenate([[0], np.cumsum(nodes)])
    rows, seqs = int(first[-1]), case["seqs"]
    s["first"], s["len"], s["rows"] = _ints(first), _ints(lens), rows
    act = torch.float32 if case.get("dtype") == "f32" else torch.bfloat16
    kd, vd, G = round8(case["dim"]), round8(case["vdim"]), case["kv"]
    ld = G * (kd + vd)
    cap = max(a + b for a, b in zip(lens, nodes)) + 5
    if op == "keep":
        caches = _normal(g, seqs * case["layers"], cap, ld, dtype=torch.bfloat16)
        keep, count = np.zeros((seqs, case["nodes"]), np.int64), np.zeros(seqs, np.int64)
        for b, n in enumerate(nodes):
            count[b] = min(n, int(rng.integers(1, case["most"] + 1)))
            keep[b, :count[b]] = np.sort(rng.choice(n, count[b], replace=False))
        s |= {"cache": caches, "table": _slots(caches), "keep": _ints(keep), "count": _ints(count), "len_out": torch.zeros_like(s["len"])}
        return s
    s["pos"] = _ints(np.concatenate([a + np.arange(n) for a, n in zip(lens, nodes)]))
    H, d, v = case["heads"], case["dim"], case["vdim"]
    if op == "prep":
        caches = torch.zeros(seqs, cap, ld, device=DEV, dtype=act)
        s |= {"y": _normal(g, rows, H * d + G * (d + v)) * 1.7, "q": torch.zeros(rows, H * kd, device=DEV, dtype=act)}
        if case["norm"]:
            s |= {"qn": 0.5 + torch.rand(d, generator=g, device=DEV), "kn": 0.5 + torch.rand(d, generator=g, device=DEV)}
        s["kt"] = _angles(case["rot"], cap)
    else:
        # keys of unequal length, as a norm weight and a model leave them: some positions draw far more weight than others
        caches = _normal(g, seqs, cap, ld, dtype=act)
        caches[:, :, :G * kd] *= (0.3 + 1.2 * torch.rand(seqs, cap, 1, generator=g, device=DEV)).to(act)
        if kd != d:
            caches[:, :, :G * kd].view(seqs, cap, G, kd)[..., d:] = 0
        if vd != v:
            caches[:, :, G * kd:].view(seqs, cap, G, vd)[..., v:] = 0
        q = _normal(g, rows, H * kd, dtype=act)
        q.view(rows, H, kd)[..., d:] = 0
        s |= {"q": q, "out": torch.zeros(rows, H * v, device=DEV, dtype=act), "scale": 1.0 / math.sqrt(d)}
        if case["tree"]:
            bits, depth = _trees(case, rng)
            s["mask"] = torch.from_numpy(bits.copy()).to(DEV)
            s["pos"] = _ints(np.repeat(np.array(lens), nodes) + depth)
        if case["gate"]:
            s["gate"] = _normal(g, rows, H)
    s |= {"cache": caches, "table": _slots(caches)}
    if case["vrot"]:
        s["vt"] = _angles(v, cap)
    return s


# ---------------------------------------------------------------------------------------------------------------- plain forms
def _places(s):
    """Sequence and place in its tree of every row."""
    r = torch.arange(s["rows"], device=DEV)
    b = (r[:, None] >= s["first"][None, 1:]).sum(1)
    return b, r - s["first"][b]


def _plain_table(s):
    c = s["case"]
    i = torch.arange(0, c["dims"], 2, device=DEV, dtype=torch.float64)
    base = s["base"]
    if c["scaling"] == "base":
        base = base * c["factor"] ** (c["dims"] / (c["dims"] - 2))
    f = base ** (-i / c["dims"])
    if c["scaling"] == "linear":
        f = f / c["factor"]
    if c["scaling"] == "ramp":
        turns = c["orig"] * f / (2 * math.pi)
        w = ((turns - c["low"]) / (c["high"] - c["low"])).clamp(0, 1)
        f = f * (w + (1 - w) / c["factor"])
    a = (c["pos0"] + torch.arange(c["n"], device=DEV, dtype=torch.float64))[:, None] * f
    return (torch.cos(a) * c["mscale"]).float(), (torch.sin(a) * c["mscale"]).float()


def _turn(x, cos, sin, half):
    """The leading 2 * cos.shape[-1] elements of the last axis, rotated."""
    n = cos.shape[-1]
    if n == 0:
        return x
    a, b = (x[..., :n], x[..., n:2 * n]) if half else (x[..., 0:2 * n:2], x[..., 1:2 * n:2])
    u, w = a * cos - b * sin, b * cos + a * sin
    return torch.cat([u, w, x[..., 2 * n:]] if half else [torch.stack([u, w], -1).flatten(-2), x[..., 2 * n:]], -1)


def _pad(x, to):
    return torch.nn.functional.pad(x, (0, to - x.shape[-1]))


def _plain_prep(s):
    c, y = s["case"], s["y"]
    H, G, d, v, M = c["heads"], c["kv"], c["dim"], c["vdim"], s["rows"]
    kd, vd = round8(d), round8(v)
    q, k, x = y[:, :H * d].view(M, H, d), y[:, H * d:(H + G) * d].view(M, G, d), y[:, (H + G) * d:].view(M, G, v)
    if c["norm"]:
        q = q / torch.sqrt((q * q).mean(-1, keepdim=True) + 1e-6) * s["qn"]
        k = k / torch.sqrt((k * k).mean(-1, keepdim=True) + 1e-6) * s["kn"]
    pos = s["pos"].long()
    cos, sin = (t[pos][:, None] for t in s["kt"])
    q, k = _turn(q, cos, sin, c["half"]), _turn(k, cos, sin, c["half"])
    if c["vrot"]:
        cos, sin = (t[pos][:, None] for t in s["vt"])
        x = _turn(x, cos, sin, False)
    s["q"].copy_(_pad(q, kd).reshape(M, H * kd))
    b, i = _places(s)
    s["cache"][b, s["len"][b] + i] = torch.cat([_pad(k, kd).reshape(M, G * kd), _pad(x, vd).reshape(M, G * vd)], 1).to(s["cache"].dtype)
    return s["q"], s["cache"]


def _plain_attn(s):
    c = s["case"]
    H, G, d, v, B, n = c["heads"], c["kv"], c["dim"], c["vdim"], c["seqs"], c["nodes"]
    kd, vd, per = round8(d), round8(v), H // G
    lens, nodes = _spread(c)
    K = max(a + m for a, m in zip(lens, nodes))
    b, i = _places(s)
    q = torch.zeros(B, n, G, per, d, device=DEV)
    q[b, i] = s["q"].view(-1, G, per, kd)[..., :d].float()
    keys = s["cache"][:, :K, :G * kd].view(B, K, G, kd)[..., :d].float().permute(0, 2, 3, 1)
    values = s["cache"][:, :K, G * kd:].view(B, K, G, vd)[..., :v].float().permute(0, 2, 1, 3)
    scores = torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(B, G, per * n, d), keys).view(B, G, per, n, K) * s["scale"]
    t = torch.arange(K, device=DEV)[None] - s["len"][:, None]                    # place in the tree, negative ahead of it
    if c["tree"]:
        bits = torch.zeros(B, n, s["mask"].shape[1] * 32, dtype=torch.bool, device=DEV)
        bits[b, i] = (((s["mask"][:, :, None] >> torch.arange(32, device=DEV)) & 1) != 0).flatten(1)
        seen = torch.gather(bits, 2, t.clamp(0, n - 1)[:, None].expand(B, n, K)) & (t < n)[:, None]
    else:
        seen = t[:, None] <= torch.arange(n, device=DEV)[None, :, None]
    seen = (seen | (t < 0)[:, None])[:, None, None]
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, G, per * n, K), values).view(B, G, per, n, v) / torch.where(total == 0, 1.0, total)
    o = o.permute(0, 3, 1, 2, 4)[b, i].reshape(-1, H, v)
    if c["vrot"]:
        cos, sin = (x[s["pos"].long()][:, None] for x in s["vt"])
        o = _turn(o, cos, -sin, False)
    if c["gate"]:
        o = o / (1.0 + torch.exp(-s["gate"]))[..., None]
    s["out"].copy_(o.reshape(-1, H * v))
    return s["out"]


def _plain_keep(s):
    c, B = s["case"], s["case"]["seqs"]
    n = s["keep"].shape[1]
    i = torch.arange(n, device=DEV)[None]
    src = torch.where(i < s["count"][:, None], s["keep"], i) + s["len"][:, None]   # a row that is not kept is copied onto itself
    dst = i + s["len"][:, None]
    cap = s["cache"].shape[1]
    src, dst = src.clamp(max=cap - 1).repeat(c["layers"], 1), dst.clamp(max=cap - 1).repeat(c["layers"], 1)
    e = torch.arange(B * c["layers"], device=DEV)[:, None]
    rows = s["cache"][e, src]
    real = (i < s["count"][:, None]).repeat(c["layers"], 1)[..., None]
    s["cache"][e, dst] = torch.where(real, rows, s["cache"][e, dst])
    torch.add(s["len"], s["count"], out=s["len_out"])
    return s["cache"], s["len_out"]


# ---------------------------------------------------------------------------------------------------------------- the library
def _descriptor(s):
    """The call's descriptor: sizes and pointers, which a program keeps with its buffers."""
    import ctypes as C
    from det_b200 import capi
    lib, c = capi.cuda(), s["case"]
    if lib.det_init() != 0:
        raise RuntimeError("no usable GPU")
    ptr = lambda k: s[k].data_ptr() if k in s else None  # noqa: E731
    if c["op"] == "table":
        op = capi.FRopeOp(dims=c["dims"], scaling=SCALINGS[c["scaling"]], base=s["base"], factor=c["factor"], orig_ctx=c["orig"],
                          low=c["low"], high=c["high"], mscale=c["mscale"], pos0=c["pos0"], n=c["n"], cos=ptr("cos"), sin=ptr("sin"))
        return lib.det_f_rope_table, op, C.byref(op), (s["cos"], s["sin"])
    lens, nodes = _spread(c)
    if c["op"] == "keep":
        cache = s["cache"]
        op = capi.FKeepOp(caches=cache.shape[0], seqs=c["seqs"], cap=cache.shape[1], row_bytes=cache.shape[2] * 2, table=ptr("table"),
                          len=ptr("len"), keep=ptr("keep"), keep_ld=s["keep"].shape[1], count=ptr("count"), max_count=min(c["most"], c["nodes"]),
                          len_out=ptr("len_out"))
        return lib.det_f_tree_keep, op, C.byref(op), (cache, s["len_out"])
    ref = capi.TreeRef(table=ptr("table"), first=ptr("first"), len=ptr("len"), seqs=c["seqs"], rows=s["rows"], max_nodes=max(nodes), max_len=max(lens))
    dtype = capi.DET_F32 if c["dtype"] == "f32" else capi.DET_BF16
    vt = s["vt"] if c["vrot"] else None
    turned = dict(vrope_cos=vt[0].data_ptr(), vrope_sin=vt[1].data_ptr()) if vt else {}
    cap = s["cache"].shape[1]
    if c["op"] == "prep":
        H, G, d = c["heads"], c["kv"], c["dim"]
        op = capi.FQkOp(heads=H, kv_heads=G, dim=d, vdim=c["vdim"], rot_dims=c["rot"], half=int(c["half"]), eps=1e-6, q_norm=ptr("qn"), k_norm=ptr("kn"),
                        cap=cap, dtype=dtype, y=ptr("y"), ldy=s["y"].shape[1], q_off=0, k_off=H * d, v_off=(H + G) * d, rope_len=cap,
                        rope_cos=s["kt"][0].data_ptr(), rope_sin=s["kt"][1].data_ptr(), pos=ptr("pos"), q=ptr("q"), seq=ref, **turned)
        return lib.det_f_qk_rope, op, C.byref(op), (s["q"], s["cache"])
    s["scratch"] = torch.empty(lib.det_f_tree_scratch_bytes(c["heads"], c["kv"], c["vdim"], max(nodes)), dtype=torch.uint8, device=DEV)
    op = capi.FTreeOp(heads=c["heads"], kv_heads=c["kv"], dim=c["dim"], vdim=c["vdim"], scale=s["scale"], cap=cap, dtype=dtype, q=ptr("q"),
                      mask=ptr("mask"), mask_ld=s["mask"].shape[1] if c["tree"] else 0, gate=ptr("gate"), ldg=c["heads"], pos=ptr("pos"),
                      rope_len=cap, out=ptr("out"), ldo=s["out"].shape[1], scratch=ptr("scratch"), seq=ref, **turned)
    return lib.det_f_tree_attn, op, C.byref(op), s["out"]


PLAIN = {"table": _plain_table, "prep": _plain_prep, "attn": _plain_attn, "keep": _plain_keep}


def run(state):
    if own:
        if "call" not in state:
            state["call"] = _descriptor(state)
        entry, _, ref, out = state["call"]
        if entry(ref, None) != 0:
            raise RuntimeError("the call was refused")
        return out
    return PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------------------------- what a pass needs
def work(case):
    if case["op"] == "table":
        return {"bytes": case["n"] * case["dims"] * 4, "flops": 0}
    lens, nodes = _spread(case)
    kd, vd, G = round8(case["dim"]), round8(case["vdim"]), case["kv"]
    ld = G * (kd + vd)
    if case["op"] == "keep":
        return {"bytes": 2 * 2 * ld * case["layers"] * sum(min(n, (case["most"] + 1) // 2) for n in nodes), "flops": 0}
    size = 4 if case["dtype"] == "f32" else 2
    H, d, v, rows = case["heads"], case["dim"], case["vdim"], sum(nodes)
    if case["op"] == "prep":
        return {"bytes": rows * (4 * (H * d + G * (d + v)) + 4 * case["rot"] + size * (H * kd + ld)), "flops": rows * (H + G) * d * 8}
    keys = sum(a + n for a, n in zip(lens, nodes))
    pairs = sum(n * a + (r * (r + 1) // 2) for a, n, r in zip(lens, nodes, nodes if not case["tree"] else [0] * len(nodes)))
    if case["tree"]:
        pairs += sum(n * max(1, int(math.log2(n + 1))) for n in nodes)           # the expected depth of a node
    return {"bytes": size * (keys * ld + rows * H * (kd + v)), "flops": 2 * pairs * H * (d + v)}


# ---------------------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "table":
        j = np.arange(case["dims"] // 2, dtype=np.float64)
        d, base, factor = float(case["dims"]), s["base"], case["factor"]
        if case["scaling"] == "base":
            base *= math.pow(factor, d / (d - 2.0))
        freq = np.exp2(-2.0 * j / d * math.log2(base))
        if case["scaling"] == "linear":
            freq = freq / factor
        elif case["scaling"] == "ramp":
            full = case["orig"] * freq / math.tau                               # turns within the context of the training
            keep = np.clip((full - case["low"]) / (case["high"] - case["low"]), 0.0, 1.0)
            freq = keep * freq + (1.0 - keep) * (freq / factor)
        at = torch.from_numpy(freq).to(DEV)[None] * torch.arange(case["pos0"], case["pos0"] + case["n"], device=DEV, dtype=torch.float64)[:, None]
        z = torch.polar(torch.full_like(at, case["mscale"]), at)
        return z.real.contiguous(), z.imag.contiguous()
    if case["op"] == "keep":
        before, cache = s["cache"].double(), s["cache"].double()
        kept, counts, lens = s["keep"].tolist(), s["count"].tolist(), s["len"].tolist()
        for e in range(cache.shape[0]):
            b = e % case["seqs"]
            for i in range(counts[b]):
                cache[e, lens[b] + i] = before[e, lens[b] + kept[b][i]]
        return cache, None
    lens, nodes = _spread(case)
    H, G, d, v = case["heads"], case["kv"], case["dim"], case["vdim"]
    kd, vd, per = round8(d), round8(v), H // G
    turn_of = lambda t, p: torch.complex(t[0][p].double(), t[1][p].double())  # noqa: E731

    def pairs(x, z):                                                            # neighbours (2i, 2i + 1) as complex numbers
        m = z.shape[-1]
        if m:
            x = torch.cat([torch.view_as_real(torch.view_as_complex(x[..., :2 * m].reshape(*x.shape[:-1], m, 2).contiguous()) * z).flatten(-2),
                           x[..., 2 * m:]], -1)
        return x

    if case["op"] == "prep":
        y, at = s["y"].double(), s["pos"].long()

        def head(x, w):
            if case["norm"]:
                x = x * w.double() * torch.rsqrt(x.square().sum(-1, keepdim=True) / d + 1e-6)
            m, z = case["rot"] // 2, turn_of(s["kt"], at)[:, None]
            if not case["half"]:
                return pairs(x, z)
            order = torch.arange(2 * m, device=DEV).view(2, m).t().reshape(-1)   # halves to neighbours
            t = pairs(x[..., :2 * m][..., order], z)
            return torch.cat([t[..., 0::2], t[..., 1::2], x[..., 2 * m:]], -1)

        q = head(y[:, :H * d].reshape(-1, H, d), s.get("qn"))
        k = head(y[:, H * d:(H + G) * d].reshape(-1, G, d), s.get("kn"))
        x = y[:, (H + G) * d:].reshape(-1, G, v)
        if case["vrot"]:
            x = pairs(x, turn_of(s["vt"], at)[:, None])
        cache, r = s["cache"].double(), 0
        rows = torch.cat([_pad(k, kd).flatten(1), _pad(x, vd).flatten(1)], 1)
        for b, (a, n) in enumerate(zip(lens, nodes)):
            cache[b, a:a + n] = rows[r:r + n]
            r += n
        return _pad(q, kd).flatten(1), cache
    out = torch.zeros(s["rows"], H, v, device=DEV, dtype=torch.float64)
    r0 = 0
    for b, (a, n) in enumerate(zip(lens, nodes)):
        see = torch.ones(n, a + n, dtype=torch.bool, device=DEV)
        if case["tree"]:
            words = s["mask"][r0:r0 + n].cpu().numpy().view(np.uint32)
            see[:, a:] = torch.from_numpy(np.unpackbits(words.view(np.uint8), axis=1, bitorder="little")[:, :n] != 0).to(DEV)
        else:
            see[:, a:] = torch.ones(n, n, dtype=torch.bool, device=DEV).tril()
        cache = s["cache"][b, :a + n]
        for h in range(H):
            g = h // per
            k = cache[:, g * kd:g * kd + d].double()
            x = cache[:, G * kd + g * vd:G * kd + g * vd + v].double()
            w = (s["q"][r0:r0 + n, h * kd:h * kd + d].double() @ k.t() * s["scale"]).masked_fill(~see, -math.inf)
            some = see.any(1, keepdim=True)
            w = torch.softmax(torch.where(some, w, 0.0), 1) * some
            out[r0:r0 + n, h] = w @ x
        r0 += n
    if case["vrot"]:
        out = pairs(out, turn_of(s["vt"], s["pos"].long()).conj()[:, None])
    if case["gate"]:
        out = out * torch.sigmoid(s["gate"].double())[..., None]
    return out.flatten(1)
