"""Host checks of the paged-cache entry points at their edges (no GPU): refused before any launch."""
import pytest
import torch

from bytes_b200 import _native as N
from test_paged_cpu import F, I, SZ, VP, at, cache, fake


def append_summary(code=None, scale=None, tokens=3, kc=None, k_scale=1.0, v_scale=1.0):
    c = cache()
    kc = kc or c["k"]
    if tokens == 0:
        c["table"], c["lens"] = fake((0, 4), N.BD_I32), fake((0,), N.BD_I32)
    k = fake((tokens, 2, 64), N.BD_BF16)
    f = N.lib().bd_paged_append_summary
    f.restype = I
    return f(at(k), at(k), None, None, None, I(0), None, at(c["table"]), at(c["lens"]), F(k_scale), F(v_scale), at(kc),
             at(fake((6, 2, 16, 64), kc.dtype)), None, at(code), at(scale), None)


@pytest.mark.parametrize("tokens", [3, 0])
def test_append_with_a_bad_summary_is_refused_as_a_whole(tokens):
    """The summary's own refusal comes before the append's launch, which without a GPU would answer 8 (BD_ERR_CUDA)."""
    if torch.cuda.is_available() and tokens:
        pytest.skip("made-up pointers: only where nothing can be launched")
    code, scale = fake((6, 2, 2, 64), N.BD_I8), fake((6, 2), N.BD_F32)
    assert append_summary(code, scale, tokens) == (8 if tokens else 0)
    assert append_summary(fake((5, 2, 2, 64), N.BD_I8), scale, tokens) == 3
    assert append_summary(fake((6, 2, 2, 64), N.BD_F32), scale, tokens) == 2
    assert append_summary(fake((6, 2, 2, 64), N.BD_I8, strides=(256, 128, 1, 2)), scale, tokens) == 4
    assert append_summary(code, fake((6, 3), N.BD_F32), tokens) == 3
    assert append_summary(code, None, tokens) == 1
    assert append_summary(None, scale, tokens) == 1


@pytest.mark.parametrize("x", [0.0, -1.0, float("inf"), float("nan"), 1e-39])
def test_scales_that_cannot_be_divided_by_are_refused(x):
    """(Calls of nothing, which launch nothing if they are let through.)"""
    code, scale = fake((6, 2, 2, 64), N.BD_I8), fake((6, 2), N.BD_F32)
    kc, q = fake((6, 2, 16, 64), N.BD_F8E4M3), fake((0, 8, 64), N.BD_BF16)
    table, lens = fake((0, 4), N.BD_I32), fake((0,), N.BD_I32)
    attn, summ = N.lib().bd_paged_decode_attn, N.lib().bd_paged_block_summary
    attn.restype = summ.restype = I
    for a, b in ((x, 1.0), (1.0, x), (1.0, 1.0)):
        rc = 0 if a == b else 9
        assert append_summary(code, scale, 0, kc, k_scale=a, v_scale=b) == rc
        assert attn(at(q), at(kc), at(kc), at(table), at(lens), None, F(0.1), F(a), F(b), at(q), None, VP(0), SZ(0),
                    None) == rc
    assert summ(at(kc), at(table), at(lens), None, I(0), F(x), at(code), at(scale), None) == 9


def test_chained_call_refuses_the_summary_of_another_cache():
    """(A call of no sequences, which launches nothing if it is let through.)"""
    f = N.lib().bd_paged_sparse_decode_attn
    f.restype = I
    q, kc = fake((0, 8, 64), N.BD_BF16), fake((6, 2, 16, 64), N.BD_BF16)
    table, lens, sel = fake((0, 4), N.BD_I32), fake((0,), N.BD_I32), fake((0, 2, 3), N.BD_I32)
    for blocks, rc in ((6, 0), (5, 3), (7, 3)):
        code, scale = fake((blocks, 2, 2, 64), N.BD_I8), fake((blocks, 2), N.BD_F32)
        assert f(at(q), at(kc), at(kc), at(code), at(scale), at(table), at(lens), I(0), I(1), F(0.1), F(1.0), F(1.0),
                 at(sel), at(q), None, VP(0x10000), SZ(1 << 20), None) == rc
