"""GPU: score attention at the ends of its arguments' ranges."""

import ctypes

import pytest
import torch

from fusionpass_b200 import _lib, fpkern
from tests._score_ref import close, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [_lib.FPK_F16, _lib.FPK_F32])
@pytest.mark.parametrize("q_len", [1, 100])
@pytest.mark.parametrize("prefix", [2 ** 31, 2 ** 62, 2 ** 63 - 1])
def test_a_prefix_beyond_all_keys_is_shared_as_all_keys_are(dtype, q_len, prefix):
    """The keys to share among CTAs are counted without overflow: the same workspace, the same parts."""
    d = _lib.ScoreDesc(size=ctypes.sizeof(_lib.ScoreDesc), version=_lib.FPK_ABI_VERSION, dtype=dtype, head_dim=64, batch=1,
                       heads=2, kv_heads=2, q_len=q_len, k_len=8192, scale=1.0, window=50, prefix=8192)
    lib = _lib.load()
    torch.cuda.current_device()
    want = lib.fpk_score_attention_workspace(ctypes.byref(d))
    assert want > 0
    d.prefix = prefix
    assert lib.fpk_score_attention_workspace(ctypes.byref(d)) == want


@pytest.mark.parametrize("dt", [torch.float16, torch.float32])
@pytest.mark.parametrize("Sq", [1, 100])
def test_windows_and_prefixes_of_any_size(dt, Sq):
    g = torch.Generator(device="cuda").manual_seed(Sq)
    q, k, v = (torch.randn(1, 2, n, 64, generator=g, device="cuda").to(dt) for n in (Sq, 1000, 1000))
    for kw in ({"prefix": 2 ** 63 - 1, "window": 50}, {"prefix": 2 ** 63 - 1}, {"window": 2 ** 63 - 1},
               {"window": 2 ** 63 - 1, "prefix": 3}, {"window": 2 ** 31, "prefix": 2 ** 32 + 5}):
        for causal in (False, True):
            small = {n: min(x, 4000) for n, x in kw.items()}
            ref, bound = reference(q, k, v, 0.125, causal=causal, **small)
            close(fpkern.score_attention(q, k, v, 0.125, causal=causal, **kw), ref, bound)
    assert fpkern.poll_status() == 0
