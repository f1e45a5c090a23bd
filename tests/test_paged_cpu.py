"""Host checks of the paged-cache entry points (no GPU): malformed requests are refused before any launch."""
import ctypes

import pytest
import torch

from bytes_b200 import _native as N

VP, F, I, SZ = ctypes.c_void_p, ctypes.c_float, ctypes.c_int, ctypes.c_size_t


def fake(shape, dtype, ptr=0x10000, strides=None):
    """Descriptor with a device pointer that is never read."""
    d = N.BdTensor()
    d.data, d.dtype, d.ndim = ptr, dtype, len(shape)
    s = 1
    for i in range(len(shape) - 1, -1, -1):
        d.shape[i], d.stride[i] = shape[i], s if strides is None else strides[i]
        s *= shape[i]
    return d


def at(d):
    return VP(ctypes.addressof(d)) if d is not None else None


def cache(**kw):
    base = dict(k=fake((6, 2, 16, 64), N.BD_BF16), v=fake((6, 2, 16, 64), N.BD_BF16), table=fake((3, 4), N.BD_I32),
                lens=fake((3,), N.BD_I32))
    base.update(kw)
    return base


def attn(q=None, out=None, lse=None, selected=None, k_scale=1.0, v_scale=1.0, ws=0, ws_bytes=0, **kw):
    c = cache(**kw)
    q = q if q is not None else fake((3, 8, 64), N.BD_BF16)
    out = out if out is not None else fake((3, 8, 64), N.BD_BF16)
    f = N.lib().bd_paged_decode_attn
    f.restype = I
    return f(at(q), at(c["k"]), at(c["v"]), at(c["table"]), at(c["lens"]), at(selected), F(0.1), F(k_scale), F(v_scale),
             at(out), at(lse), VP(ws), SZ(ws_bytes), None)


def test_decode_attn_refusals():
    assert attn(q=fake((3, 7, 64), N.BD_BF16), out=fake((3, 7, 64), N.BD_BF16)) == 3   # heads
    assert attn(q=fake((2, 8, 64), N.BD_BF16), out=fake((2, 8, 64), N.BD_BF16)) == 3   # sequences
    assert attn(q=fake((3, 8, 64), N.BD_I8)) == 2
    assert attn(v=fake((6, 2, 16, 64), N.BD_F16)) == 2
    assert attn(v=fake((5, 2, 16, 64), N.BD_BF16)) == 3
    assert attn(k=fake((6, 2, 16, 64), N.BD_I32), v=fake((6, 2, 16, 64), N.BD_I32)) == 2
    assert attn(table=fake((3, 4), N.BD_I64)) == 2
    assert attn(lens=fake((4,), N.BD_I32)) == 3
    assert attn(out=fake((3, 8, 32), N.BD_BF16)) == 3
    assert attn(out=fake((3, 8, 64), N.BD_U8)) == 2
    assert attn(lse=fake((3, 7), N.BD_F32)) == 3
    assert attn(selected=fake((3, 8, 2), N.BD_I32)) == 3
    assert attn(selected=fake((3, 2, 2), N.BD_I64)) == 2
    assert attn(k_scale=0.5) == 9
    assert attn(k=fake((6, 2, 16, 64), N.BD_F8E4M3), v=fake((6, 2, 16, 64), N.BD_F8E4M3), k_scale=-1.0) == 9
    big = fake((6, 2, 16, 300), N.BD_BF16)
    assert attn(q=fake((3, 8, 300), N.BD_BF16), out=fake((3, 8, 300), N.BD_BF16), k=big, v=big) == 7
    assert attn(k=None) == 1 and attn(v=None) == 1
    wide = dict(table=fake((3, 4096), N.BD_I32))
    assert attn(**wide) == 6 and b"workspace" in N.lib().bd_last_error()                # no workspace


def append(k=None, v=None, q=None, q_out=None, cos=None, sin=None, cu=None, k_scale=1.0, v_scale=1.0, kc=None, vc=None):
    c = cache()
    k = k if k is not None else fake((3, 2, 64), N.BD_BF16)
    v = v if v is not None else fake((3, 2, 64), N.BD_BF16)
    f = N.lib().bd_paged_append
    f.restype = I
    return f(at(k), at(v), at(q), at(cos), at(sin), I(0), at(cu), at(c["table"]), at(c["lens"]), F(k_scale), F(v_scale),
             at(kc or c["k"]), at(vc or c["v"]), at(q_out), None)


def test_append_refusals():
    assert append(k=fake((4, 2, 64), N.BD_BF16), v=fake((4, 2, 64), N.BD_BF16)) == 3     # one token a sequence
    assert append(v=fake((3, 2, 64), N.BD_F16)) == 2
    assert append(k=fake((3, 3, 64), N.BD_BF16), v=fake((3, 3, 64), N.BD_BF16)) == 3
    assert append(q=fake((3, 8, 64), N.BD_BF16)) == 1                                    # q without q_out
    assert append(q=fake((3, 8, 64), N.BD_BF16), q_out=fake((3, 7, 64), N.BD_BF16)) == 3
    assert append(cos=fake((99, 32), N.BD_F32)) == 1
    assert append(cos=fake((99, 33), N.BD_F32), sin=fake((99, 33), N.BD_F32)) == 3
    assert append(cos=fake((99, 32), N.BD_BF16), sin=fake((99, 32), N.BD_BF16)) == 2
    assert append(cu=fake((3,), N.BD_I32)) == 3
    assert append(v_scale=2.0) == 9


def test_select_and_summary_refusals():
    lib = N.lib()
    sel, summ = lib.bd_paged_select, lib.bd_paged_block_summary
    sel.restype = summ.restype = I
    c = cache()
    q, code, scale = fake((3, 8, 64), N.BD_BF16), fake((6, 2, 2, 64), N.BD_I8), fake((6, 2), N.BD_F32)

    def select(q=q, code=code, scale=scale, block=16, sink=0, recent=1, budget=3, ws=0):
        return sel(at(q), at(code), at(scale), at(c["table"]), at(c["lens"]), I(block), I(sink), I(recent),
                   at(fake((3, 2, budget), N.BD_I32)), VP(0), SZ(ws), None)

    assert select(code=fake((6, 2, 2, 64), N.BD_U8)) == 2
    assert select(code=fake((6, 2, 2, 32), N.BD_I8)) == 3
    assert select(scale=fake((6, 3), N.BD_F32)) == 3
    assert select(q=fake((3, 7, 64), N.BD_BF16)) == 3
    assert select(block=0) == 9
    assert select(sink=2, recent=2) == 9
    assert select(q=fake((3, 2 * 129, 64), N.BD_BF16)) == 7
    assert select() == 6

    def summary(code=code, scale=scale, cu=None, new=0, k_scale=1.0):
        return summ(at(c["k"]), at(c["table"]), at(c["lens"]), at(cu), I(new), F(k_scale), at(code), at(scale), None)

    assert summary(code=fake((6, 2, 64, 2), N.BD_I8)) == 3
    assert summary(code=fake((6, 2, 2, 64), N.BD_I8, strides=(256, 128, 1, 2))) == 4
    assert summary(k_scale=0.5) == 9
    assert summary(new=-1) == 9
    assert summary(cu=fake((4,), N.BD_I32)) == 9


def test_workspaces():
    """Of one row a CTA nothing is needed by the tiles; a larger table needs more; a bad request nothing."""
    f = N.lib().bd_paged_decode_attn_workspace
    f.restype = SZ
    q, c = fake((3, 8, 64), N.BD_BF16), cache()
    small = f(at(q), at(c["k"]), at(c["v"]), at(c["table"]), at(c["lens"]), None)
    wide = f(at(q), at(c["k"]), at(c["v"]), at(fake((3, 70000), N.BD_I32)), at(c["lens"]), None)
    assert 0 < small < wide
    assert f(at(fake((3, 7, 64), N.BD_BF16)), at(c["k"]), at(c["v"]), at(c["table"]), at(c["lens"]), None) == 0


def test_python_layer_refuses_cpu_tensors():
    from bytes_b200 import paged
    kc = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q, k = torch.zeros(1, 8, 64, dtype=torch.bfloat16), torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    code, scale = paged.new_block_summary(kc)
    with pytest.raises(ValueError):
        paged.paged_decode_attn(q, kc, kc, table, lens, 1.0)
    with pytest.raises(ValueError):
        paged.paged_append(k, k, kc, kc, table, lens)
    with pytest.raises(ValueError):
        paged.paged_block_summary(kc, table, lens, code, scale)
    with pytest.raises(ValueError):
        paged.paged_sparse_decode_attn(q, kc, kc, code, scale, table, lens, 1, 1.0)


def test_restatement_on_one_page():
    """The plain restatement itself, on a case small enough to write out."""
    from oracle import paged as plain
    k = torch.tensor([[[[1.0, 0.0], [0.0, 2.0]]]])
    v = torch.tensor([[[[3.0, 0.0], [0.0, 5.0]]]])
    table, lens = torch.zeros(1, 1, dtype=torch.int32), torch.tensor([2], dtype=torch.int32)
    out, lse, _, _ = plain.decode_attn(torch.tensor([[[1.0, 1.0]]]), k, v, table, lens, 1.0)
    e1, e2 = torch.tensor(1.0).double().exp(), torch.tensor(2.0).double().exp()
    assert torch.allclose(out[0, 0], torch.stack([3 * e1, 5 * e2]) / (e1 + e2)) and torch.allclose(lse[0, 0], (e1 + e2).log())
    code, s = plain.summary_of(torch.tensor([[1.0, -2.0], [0.5, 4.0]]))
    assert code.tolist() == [[16, -64], [32, 127]] and s == torch.tensor(4.0) / torch.tensor(127.0)
    y, _ = plain.rotate(torch.tensor([[1.0, 2.0, 3.0, 4.0]]).double(), torch.tensor([0.0, 1.0]).double(),
                        torch.tensor([1.0, 0.0]).double(), False)
    assert y.tolist() == [[-3.0, 2.0, 1.0, 4.0]]
