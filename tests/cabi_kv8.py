"""ctypes mirrors of vfa_kv8_params and vfa_qk_norm_rotary_params (include/vfa.h), for the refusal tests."""
import ctypes as C

import cabi

_i, _l, _p, _z = C.c_int, C.c_int64, C.c_void_p, C.c_size_t


class VfaKv8Params(C.Structure):
    _fields_ = [("a", cabi.VfaParams), ("k_scale", _p), ("v_scale", _p),
                ("k_scale_batch_stride", _l), ("k_scale_row_stride", _l), ("k_scale_head_stride", _l),
                ("v_scale_batch_stride", _l), ("v_scale_row_stride", _l), ("v_scale_head_stride", _l),
                ("scale_block", _i), ("num_pages", _i), ("cu_seqlens_new", _p), ("k_out", _p), ("v_out", _p),
                ("ko_batch_stride", _l), ("ko_row_stride", _l), ("ko_head_stride", _l),
                ("vo_batch_stride", _l), ("vo_row_stride", _l), ("vo_head_stride", _l),
                ("cu_seqlens_out", _p), ("rows_out", _l), ("seqlen_out", _i), ("workspace", _p), ("workspace_bytes", _z)]


class VfaQkNormRotaryParams(C.Structure):
    _fields_ = [("dtype", _i), ("weight_fp32", _i), ("table_fp32", _i), ("b", _i), ("s", _i), ("h", _i), ("h_k", _i), ("d", _i),
                ("q", _p), ("k", _p)] + [(n, _l) for n in ("q_batch_stride", "q_row_stride", "q_head_stride", "k_batch_stride", "k_row_stride", "k_head_stride")] + [
                ("q_weight", _p), ("k_weight", _p), ("rotary_cos", _p), ("rotary_sin", _p), ("table_rows", _i), ("rotary_dim", _i),
                ("is_rotary_interleaved", _i), ("positions", _p), ("positions_batch_stride", _l), ("eps", C.c_float), ("q_out", _p), ("k_out", _p)] + [
                (n, _l) for n in ("qo_batch_stride", "qo_row_stride", "qo_head_stride", "ko_batch_stride", "ko_row_stride", "ko_head_stride")] + [
                ("dq_out", _p), ("dk_out", _p)] + [
                (n, _l) for n in ("dqo_batch_stride", "dqo_row_stride", "dqo_head_stride", "dko_batch_stride", "dko_row_stride", "dko_head_stride")] + [
                ("dq_weight", _p), ("dk_weight", _p), ("workspace", _p), ("stream", _p)]


def lib():
    l = cabi.lib()
    for n in ("vfa_kv8_workspace", "vfa_qk_norm_rotary_bwd_workspace", "vfa_kv8_params_sizeof", "vfa_qk_norm_rotary_params_sizeof"):
        getattr(l, n).restype = _z
    l.vfa_last_error.restype = C.c_char_p
    return l


def kv8(**over):
    """A valid argument block (pointers that are never followed: the tests refuse, or only plan); over: field -> value,
    'a.' fields of the embedded vfa_params by their own names."""
    P = VfaKv8Params()
    a = P.a
    a.dtype, a.b, a.h, a.h_k, a.d, a.seqlen_q, a.seqlen_k = 1, 2, 8, 2, 128, 1, 1024
    a.q = a.k = a.v = a.out = a.softmax_lse = 4096
    a.softmax_scale = 0.1
    a.k_batch_stride = a.v_batch_stride = 1024 * 256
    a.k_row_stride = a.v_row_stride = 256
    a.k_head_stride = a.v_head_stride = 128
    a.window_size_left = a.window_size_right = -1
    P.k_scale = P.v_scale = 4096
    P.scale_block, P.num_pages = 64, 2
    for n, v in over.items():
        setattr(P if hasattr(type(P), n) and n != "a" else a, n, v)
    return P


def qk(**over):
    P = VfaQkNormRotaryParams()
    P.dtype, P.b, P.s, P.h, P.h_k, P.d = 1, 1, 4, 8, 2, 128
    for n in ("q", "k", "q_weight", "k_weight", "rotary_cos", "rotary_sin", "q_out", "k_out", "dq_out", "dk_out"):
        setattr(P, n, 4096)
    P.table_rows, P.rotary_dim, P.eps = 16, 64, 1e-6
    for n, v in over.items():
        setattr(P, n, v)
    return P
