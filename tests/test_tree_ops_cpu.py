"""What the ops of a step of drafted tokens refuse, before anything is launched: no GPU is needed, and the pointers are never read."""
import ctypes as C

import pytest

P = 1 << 20     # a 16-byte aligned address that nothing reads


def ref(libs, **kw):
    return libs.TreeRef(**{**dict(table=P, first=P, len=P, seqs=2, rows=5, max_nodes=4, max_len=10), **kw})


def rope(libs, **kw):
    return libs.FRopeOp(**{**dict(dims=64, scaling=0, base=1e4, factor=2.0, orig_ctx=4096.0, low=1.0, high=32.0, mscale=1.0, pos0=0, n=8,
                                  cos=P, sin=P), **kw})


def qk(libs, seq=None, **kw):
    return libs.FQkOp(**{**dict(heads=4, kv_heads=2, dim=64, vdim=64, rot_dims=64, half=0, eps=1e-6, q_norm=P, k_norm=P, cap=32,
                                dtype=libs.DET_BF16, y=P, ldy=512, q_off=0, k_off=256, v_off=384, rope_len=32, rope_cos=P, rope_sin=P, q=P,
                                seq=seq or ref(libs)), **kw})


def attn(libs, seq=None, **kw):
    return libs.FTreeOp(**{**dict(heads=4, kv_heads=2, dim=64, vdim=64, scale=0.1, cap=32, dtype=libs.DET_BF16, q=P, mask=P, mask_ld=1, out=P,
                                  ldo=256, scratch=P, seq=seq or ref(libs)), **kw})


def keep(libs, **kw):
    return libs.FKeepOp(**{**dict(caches=4, seqs=2, cap=32, row_bytes=512, table=P, len=P, keep=P, keep_ld=4, count=P, max_count=4), **kw})


NAN = float("nan")
BAD_ROPE = [dict(dims=0), dict(dims=7), dict(dims=-2), dict(n=-1), dict(pos0=-1), dict(pos0=2 ** 31 - 4), dict(base=0.0), dict(base=-2.0), dict(base=NAN),
            dict(mscale=NAN), dict(scaling=4), dict(scaling=-1), dict(scaling=1, factor=0.0), dict(scaling=2, dims=2),
            dict(scaling=3, high=1.0), dict(scaling=3, orig_ctx=0.0), dict(scaling=3, low=NAN), dict(cos=None), dict(sin=None)]
BAD_QK = [dict(heads=0), dict(kv_heads=-1), dict(dim=0), dict(dim=257), dict(vdim=300), dict(cap=0), dict(dtype=2), dict(rot_dims=3),
          dict(rot_dims=66), dict(rot_dims=-2), dict(half=2), dict(vrope_cos=P), dict(vrope_sin=P), dict(vdim=63, vrope_cos=P, vrope_sin=P),
          dict(ldy=-1), dict(k_off=-4), dict(eps=-1.0), dict(eps=NAN), dict(y=None), dict(q=None), dict(q=P + 8), dict(rope_cos=None),
          dict(rope_len=0)]
BAD_ATTN = [dict(heads=0), dict(heads=5), dict(kv_heads=0), dict(dim=0), dict(dim=264), dict(vdim=0), dict(cap=0), dict(dtype=-1),
            dict(scale=0.0), dict(scale=-1.0), dict(scale=NAN), dict(scale=float("inf")), dict(mask_ld=0), dict(ldo=255), dict(gate=P, ldg=3),
            dict(vrope_cos=P), dict(vrope_cos=P, vrope_sin=P), dict(vrope_cos=P, vrope_sin=P, pos=P, rope_len=0), dict(q=None), dict(out=None),
            dict(scratch=None), dict(q=P + 4), dict(scratch=P + 8), dict(scratch=P + 64)]
BAD_KEEP = [dict(caches=-1), dict(seqs=-1), dict(cap=0), dict(max_count=-1), dict(max_count=5), dict(max_count=2000, keep_ld=2000), dict(row_bytes=0),
            dict(row_bytes=24), dict(caches=3), dict(table=None), dict(len=None), dict(keep=None), dict(count=None), dict(len_out=P)]
BAD_REF = [dict(seqs=-1), dict(rows=-1), dict(max_len=-1), dict(max_nodes=-1), dict(seqs=70000), dict(table=None), dict(first=None), dict(len=None)]


def refused(entry, op, capfd):
    assert entry(C.byref(op), None) == 1
    assert "refused" in capfd.readouterr().err


@pytest.mark.parametrize("kw", BAD_ROPE, ids=str)
def test_table_refusals(kw, libs, capfd):
    refused(libs.cuda().det_f_rope_table, rope(libs, **kw), capfd)


@pytest.mark.parametrize("kw", BAD_QK, ids=str)
def test_norm_and_rotation_refusals(kw, libs, capfd):
    refused(libs.cuda().det_f_qk_rope, qk(libs, **kw), capfd)


@pytest.mark.parametrize("kw", BAD_ATTN, ids=str)
def test_attention_refusals(kw, libs, capfd):
    refused(libs.cuda().det_f_tree_attn, attn(libs, **kw), capfd)


@pytest.mark.parametrize("kw", BAD_KEEP, ids=str)
def test_keep_refusals(kw, libs, capfd):
    refused(libs.cuda().det_f_tree_keep, keep(libs, **kw), capfd)


@pytest.mark.parametrize("kw", BAD_REF, ids=str)
def test_rows_refusals(kw, libs, capfd):
    d = libs.cuda()
    refused(d.det_f_qk_rope, qk(libs, seq=ref(libs, **kw)), capfd)
    refused(d.det_f_tree_attn, attn(libs, seq=ref(libs, **kw)), capfd)


def test_a_masked_tree_is_bounded_and_a_run_is_not(libs, capfd):
    refused(libs.cuda().det_f_tree_attn, attn(libs, seq=ref(libs, max_nodes=libs.DET_MAX_TREE + 1), mask_ld=40), capfd)
    refused(libs.cuda().det_f_tree_attn, attn(libs, seq=ref(libs, max_nodes=1 << 24)), capfd)


def test_null_descriptors(libs, capfd):
    d = libs.cuda()
    for entry in (d.det_f_rope_table, d.det_f_qk_rope, d.det_f_tree_attn, d.det_f_tree_keep):
        assert entry(None, None) == 1


def test_nothing_to_do_is_no_refusal(libs):
    d = libs.cuda()
    assert d.det_f_rope_table(C.byref(rope(libs, n=0)), None) == 0
    for kw in (dict(seqs=0), dict(rows=0)):
        assert d.det_f_qk_rope(C.byref(qk(libs, seq=ref(libs, **kw))), None) == 0
        assert d.det_f_tree_attn(C.byref(attn(libs, seq=ref(libs, **kw))), None) == 0
    assert d.det_f_tree_attn(C.byref(attn(libs, seq=ref(libs, max_nodes=0))), None) == 0
    assert d.det_f_tree_keep(C.byref(keep(libs, caches=0)), None) == 0
    assert d.det_f_tree_keep(C.byref(keep(libs, seqs=0)), None) == 0


def test_scratch_size_is_known_without_a_device(libs):
    d = libs.cuda()
    one, tree = d.det_f_tree_scratch_bytes(40, 8, 128, 1), d.det_f_tree_scratch_bytes(40, 8, 128, 64)
    assert 0 < one <= tree <= 256 << 20
    assert d.det_f_tree_scratch_bytes(40, 8, 128, 1 << 20) <= 256 << 20
    assert d.det_f_tree_scratch_bytes(0, 0, 0, 0) > 0


def test_ctypes_mirror_has_the_layout_the_c_compiler_gives_the_header(libs, tmp_path):
    import os
    import shutil
    import subprocess
    from pathlib import Path
    root = Path(__file__).resolve().parent.parent
    inc = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda")) / "include"
    if shutil.which("gcc") is None or not (inc / "cuda_runtime.h").exists():
        pytest.skip("needs gcc and the CUDA headers")
    pairs = {"det_tree_ref": libs.TreeRef, "det_frope_op": libs.FRopeOp, "det_fqk_op": libs.FQkOp, "det_ftree_op": libs.FTreeOp, "det_fkeep_op": libs.FKeepOp}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "det_b200.h"', "int main(void) {"]
    for name, mirror in pairs.items():
        lines.append(f'  printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in mirror._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-I", str(root / "include"), "-I", str(inc), str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    for name, mirror in pairs.items():
        assert int(got[name]) == C.sizeof(mirror), name
        for f, _ in mirror._fields_:
            assert int(got[f"{name}.{f}"]) == getattr(mirror, f).offset, f"{name}.{f}"
