"""The paged-cache operators at their edges: what reaches which kernel, lengths that change between calls, values that are
not numbers, streams and host threads. Inputs and bounds are those of test_gpu_paged.py."""
import math

import pytest
import torch

from bytes_b200 import paged
from oracle import paged as plain
from test_gpu_paged import (BF16, F16, F32, FP8, attention_inputs, bits, check_attention, expected_summary, gen, table_for,
                            to_cache)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------- lengths of an earlier step
@pytest.mark.parametrize("lens", [[700, 90], [4000, 0, 9, 2500], [30] * 200])
def test_lengths_changed_right_before_a_captured_call(cuda, lens):
    """The kernels that read the lengths ahead of their wait see what the kernel before the call wrote, whatever an
    earlier replay left in the SMs."""
    q, kc, vc, table, clen, ks, vs = attention_inputs(lens, 8, 2, 128, 16, BF16, BF16, 21)
    gq, gk, gv, gt, gl = (t.to(cuda) for t in (q, kc, vc, table, clen))
    code, scale = paged.new_block_summary(gk)
    paged.paged_block_summary(gk, gt, gl, code, scale)
    steps = [torch.randint(0, n + 1, (8,), generator=gen(n + 1)) for n in lens]
    now = torch.zeros_like(gl)

    def call():
        gl.copy_(now)
        return paged.paged_sparse_decode_attn(gq, gk, gv, code, scale, gt, gl, 5, 128 ** -0.5), \
            paged.paged_decode_attn(gq, gk, gv, gt, gl, 128 ** -0.5)

    now.copy_(gl)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for i in range(8):
        now.copy_(torch.stack([s[i] for s in steps]).int())
        for _ in range(2):
            graph.replay()
        torch.cuda.synchronize()
        kept = [x.clone() for x in got]
        torch.cuda.synchronize()
        for a, b in zip(kept, call()):
            assert torch.equal(bits(a), bits(b))
        for b in (now == 0).nonzero()[:, 0].tolist():
            assert (kept[0][b] == 0).all() and (kept[1][b] == 0).all()


# ------------------------------------------------------------------------------------ refusals
@pytest.mark.parametrize("tokens", [2, 0])
def test_a_refused_append_has_written_nothing(cuda, tokens):
    nb, Hk, D, block = 6, 2, 64, 16
    kc = torch.zeros(nb, Hk, block, D, dtype=BF16, device=cuda)
    vc = torch.zeros_like(kc)
    table = torch.arange(6, dtype=torch.int32, device=cuda).view(2, 3)[:tokens]
    lens = torch.ones(tokens, dtype=torch.int32, device=cuda)
    k = torch.ones(tokens, Hk, D, dtype=BF16, device=cuda)
    code, scale = paged.new_block_summary(kc)
    for c, s in ((code[:1], scale), (code.float(), scale), (code, scale[:, :1]), (code, scale.double().half()),
                 (code.transpose(2, 3).contiguous().transpose(2, 3), scale), (code.cpu(), scale)):
        with pytest.raises(ValueError):
            paged.paged_append(k, k, kc, vc, table, lens, summary=c, summary_scale=s)
    torch.cuda.synchronize()
    assert not kc.any() and not vc.any() and not code.any()
    paged.paged_append(k, k, kc, vc, table, lens, summary=code, summary_scale=scale)
    assert bool(kc.any()) == bool(code.any()) == (tokens > 0)
