"""What the ops of a step of drafted tokens take or refuse before anything is launched: no GPU is needed, and the pointers are never read."""
import ctypes as C

from test_tree_ops_cpu import attn, qk, ref


def test_a_bound_of_no_rows_is_nothing_to_do_for_every_op(libs):
    """max_nodes = 0 with rows in the buffers: norms with rotation and attention agree."""
    d = libs.cuda()
    for rows in (1, 5):
        seq = ref(libs, max_nodes=0, rows=rows)
        assert d.det_f_qk_rope(C.byref(qk(libs, seq=seq)), None) == 0
        assert d.det_f_tree_attn(C.byref(attn(libs, seq=seq)), None) == 0


def test_a_scale_that_passes_32_bits_in_the_exponent_s_base_is_refused(libs, capfd):
    """Scores are taken as exponents of 2: scale * log2 e is what has to be finite, or rows of equal scores would get NaN."""
    d = libs.cuda()
    for scale in (2.4e38, 3.4e38):
        assert d.det_f_tree_attn(C.byref(attn(libs, scale=scale)), None) == 1
        assert "bad scale" in capfd.readouterr().err
