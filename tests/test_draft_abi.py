"""The C entry points of the 8-bit cache, tree attention and verify_draft refuse what they cannot
run before any device work.  No GPU needed."""

import ctypes

import pytest

from fusionpass_b200 import _lib

HOST = (ctypes.c_char * 4096)()  # never read: every call here is refused, or has nothing to do
BASE = (ctypes.addressof(HOST) + 255) // 256 * 256
X3 = ctypes.c_int64 * 3


def p(off=0):
    return ctypes.c_void_p(BASE + off)


def made(cls, base, kw):
    return cls(**{**dict(size=ctypes.sizeof(cls), version=_lib.FPK_ABI_VERSION), **base, **kw})


def cache(**kw):
    st = X3(2048, 256, 16)
    return made(_lib.CacheDesc, dict(dtype=_lib.FPK_F16, head_dim=16, batch=1, heads=2, rows=4, room=16, k_strides=st,
                                     v_strides=st, k_cache_strides=st, v_cache_strides=st, k_scale_strides=X3(32, 16, 1),
                                     v_scale_strides=X3(32, 16, 1), past_lens=BASE), kw)


def tree(**kw):
    st = X3(2048, 256, 16)
    return made(_lib.TreeDesc, dict(dtype=_lib.FPK_F16, head_dim=16, batch=1, heads=2, kv_heads=2, nodes=4, room=16,
                                    scale=1.0, parents_stride=4, q_strides=st, k_strides=st, v_strides=st, o_strides=st,
                                    parents=BASE, past_lens=BASE), kw)


def verify(**kw):
    return made(_lib.VerifyDesc, dict(batch=1, nodes=2, vocab=8, tokens=BASE, parents=BASE, target=BASE, uniform=BASE,
                                      path=BASE, counts=BASE, next=BASE), kw)


INVALID, UNSUPPORTED, ALIGN = _lib.FPK_ERR_INVALID, _lib.FPK_ERR_UNSUPPORTED, _lib.FPK_ERR_ALIGN


@pytest.mark.parametrize("kw, rc", [
    (dict(size=4), INVALID), (dict(version=9), INVALID), (dict(dtype=7), INVALID), (dict(batch=-1), INVALID),
    (dict(head_dim=24), UNSUPPORTED), (dict(room=(1 << 30) + 1), UNSUPPORTED), (dict(past_lens=None), INVALID),
    (dict(past_lens=BASE + 2), ALIGN), (dict(lens=BASE + 1), ALIGN), (dict(k_strides=X3(2048, 256, 12)), ALIGN),
    (dict(v_cache_strides=X3(2048, 256, 8)), ALIGN), (dict(rows=0), 0), (dict(batch=0), 0)])
def test_cache_write(kw, rc):
    f = _lib.load().fpk_cache_write
    assert f(ctypes.byref(cache(**kw)), p(), p(), p(), p(), p(), p(), None) == rc


@pytest.mark.parametrize("i", range(6))
def test_cache_write_pointers(i):
    f = _lib.load().fpk_cache_write
    at = [p() for _ in range(6)]
    at[i] = None
    assert f(ctypes.byref(cache()), *at, None) == INVALID
    at[i] = p(2)
    assert f(ctypes.byref(cache()), *at, None) == ALIGN


def test_cache_read_takes_all_rows():
    f = _lib.load().fpk_cache_read
    assert f(ctypes.byref(cache()), p(), p(), p(), p(), p(), p(), None) == INVALID
    assert f(None, p(), p(), p(), p(), p(), p(), None) == INVALID


@pytest.mark.parametrize("kw, entry, rc", [
    (dict(size=1), {}, INVALID), (dict(n_caches=65), {}, UNSUPPORTED), (dict(n_path=257), {}, UNSUPPORTED),
    (dict(n_path=-1), {}, INVALID), (dict(path=None), {}, INVALID), (dict(counts=BASE + 2), {}, ALIGN),
    ({}, dict(row_bytes=0), INVALID), ({}, dict(heads=-1), INVALID), ({}, dict(data=None), INVALID),
    ({}, dict(room=(1 << 30) + 1), UNSUPPORTED), (dict(batch=0), {}, 0), (dict(n_path=0), {}, 0), ({}, dict(heads=0), 0),
    ({}, dict(room=0, data=None), 0)])
def test_cache_keep(kw, entry, rc):
    d = made(_lib.KeepDesc, dict(batch=1, n_caches=1, n_path=2, path_stride=2, path=BASE, counts=BASE, past_lens=BASE), kw)
    c = _lib.KeepCache(**{**dict(data=BASE, strides=X3(512, 256, 16), room=16, heads=2, row_bytes=16), **entry})
    assert _lib.load().fpk_cache_keep(ctypes.byref(d), ctypes.byref(c), None) == rc


@pytest.mark.parametrize("kw, rc", [
    (dict(size=4), INVALID), (dict(dtype=5), INVALID), (dict(flags=2), INVALID), (dict(nodes=-1), INVALID),
    (dict(kv_heads=0), INVALID), (dict(heads=3), INVALID), (dict(scale=float("nan")), INVALID),
    (dict(scale=3e38), UNSUPPORTED), (dict(head_dim=8), UNSUPPORTED), (dict(nodes=257), UNSUPPORTED),
    (dict(batch=65536), UNSUPPORTED), (dict(room=(1 << 30) + 1), UNSUPPORTED), (dict(parents=BASE + 2), ALIGN),
    (dict(tree_lens=BASE + 1), ALIGN), (dict(past_lens=None), INVALID), (dict(q_strides=X3(2048, 256, 12)), ALIGN),
    (dict(o_strides=X3(2048, 0, 16)), ALIGN), (dict(flags=1), INVALID), (dict(batch=0), 0), (dict(nodes=0), 0)])
def test_tree_attention(kw, rc):
    f = _lib.load().fpk_tree_attention_fwd
    assert f(ctypes.byref(tree(**kw)), p(), p(), p(), p(), None, 0, None) == rc


@pytest.mark.parametrize("kw, rc", [
    (dict(size=4), INVALID), (dict(nodes=0), INVALID), (dict(vocab=0), INVALID), (dict(nodes=257), UNSUPPORTED),
    (dict(vocab=(1 << 22) + 1), UNSUPPORTED), (dict(target=None), INVALID), (dict(path=None), INVALID),
    (dict(draft=BASE + 2), ALIGN), (dict(uniform=BASE + 1), ALIGN), (dict(batch=0), 0)])
def test_verify_draft(kw, rc):
    assert _lib.load().fpk_verify_draft(ctypes.byref(verify(**kw)), None) == rc


def test_descriptors_match_the_header():
    """Sizes of the C structures by their fields: 64-bit members are aligned to 8 bytes."""
    assert ctypes.sizeof(_lib.CacheDesc) == 16 + 4 * 8 + 6 * 24 + 16
    assert ctypes.sizeof(_lib.KeepCache) == 48 and ctypes.sizeof(_lib.KeepDesc) == 56
    assert ctypes.sizeof(_lib.TreeDesc) == 16 + 5 * 8 + 8 + 8 + 6 * 24 + 40
    assert ctypes.sizeof(_lib.VerifyDesc) == 8 + 8 + 8 + 32 + 24 + 72
