"""The C entry points of the quantised block refuse what they cannot run before any device
work: pointers off their element's alignment, factors that are not finite.  No GPU needed."""

import ctypes

import pytest

from fusionpass_b200 import _lib

HOST = (ctypes.c_char * 4096)()  # never read: every call here is refused
BASE = (ctypes.addressof(HOST) + 255) // 256 * 256


def p(off=0):
    return ctypes.c_void_p(BASE + off)


@pytest.mark.parametrize("dtype, size", [(_lib.FPK_F16, 2), (_lib.FPK_BF16, 2), (_lib.FPK_F32, 4)])
@pytest.mark.parametrize("which", ["addend", "w", "sum", "y", "scale"])
def test_rms_norm_refuses_pointers_off_their_elements(dtype, size, which):
    d = _lib.RmsDesc(size=ctypes.sizeof(_lib.RmsDesc), version=_lib.FPK_ABI_VERSION, dtype=dtype, rows=2, cols=8,
                     q_stride=16, eps=1e-6)
    at = {k: p(size // 2 if which == k else 0) for k in ("addend", "w", "sum", "y")}
    quant = which == "scale"
    a, bc = (ctypes.c_void_p * 2)(p(), at["addend"]), (ctypes.c_int32 * 2)(0, 0)
    rc = _lib.load().fpk_rms_norm_fwd(ctypes.byref(d), a, bc, 2, at["w"], at["sum"], None if quant else at["y"],
                                      p() if quant else None, p(2) if quant else None, None)
    assert rc == _lib.FPK_ERR_ALIGN


@pytest.mark.parametrize("which", ["x_scale", "w_scale", "bias", "y"])
def test_linear_refuses_pointers_off_their_elements(which):
    d = _lib.LinearDesc(size=ctypes.sizeof(_lib.LinearDesc), version=_lib.FPK_ABI_VERSION, out_dtype=_lib.FPK_F32,
                        m=2, n=8, k=16, x_stride=16, w_stride=16, y_stride=8)
    at = {k: p(2 if which == k else 0) for k in ("x_scale", "w_scale", "bias", "y")}
    rc = _lib.load().fpk_linear_int_fwd(ctypes.byref(d), p(), at["x_scale"], p(), at["w_scale"], at["bias"], at["y"],
                                        None, 0, None)
    assert rc == _lib.FPK_ERR_ALIGN


def _score(**kw):
    return _lib.ScoreDesc(**{**dict(size=ctypes.sizeof(_lib.ScoreDesc), version=_lib.FPK_ABI_VERSION,
                                    dtype=_lib.FPK_F16, head_dim=64, batch=1, heads=2, kv_heads=2, q_len=4, k_len=4,
                                    scale=1.0), **kw})


@pytest.mark.parametrize("which", ["slopes", "prefix_lens", "doc_ids", "kv_lens"])
def test_score_attention_refuses_pointers_off_their_elements(which):
    d = _score(**{which: BASE + 2})
    assert _lib.load().fpk_score_attention_workspace(ctypes.byref(d)) == _lib.FPK_ERR_ALIGN


@pytest.mark.parametrize("scale, cap", [(3e38, 0.0), (-3e38, 0.0), (1.0, 1e-39), (1e10, 1e-29)])
def test_score_attention_refuses_factors_beyond_f32(scale, cap):
    lib = _lib.load()
    for dtype in (_lib.FPK_F16, _lib.FPK_F32):
        d = _score(dtype=dtype, scale=scale, softcap=cap)
        assert lib.fpk_score_attention_workspace(ctypes.byref(d)) == _lib.FPK_ERR_UNSUPPORTED
