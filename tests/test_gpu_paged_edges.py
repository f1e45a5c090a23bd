"""The paged-cache operators at their edges: what reaches which kernel, lengths that change between calls, values that are
not numbers, streams and host threads. Inputs and bounds are those of test_gpu_paged.py."""
import ctypes
import math
import re
import threading

import pytest
import torch

from bytes_b200 import _native as N
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


def test_tables_and_lengths_of_other_types(cuda):
    """64-bit entries that 32 bits do not hold name no page and are long lengths, whatever their lower halves say;
    shorter integers are taken as they are; what is no integer is refused."""
    q, kc, vc, table, lens, ks, vs = attention_inputs([100, 333], 8, 2, 128, 16, BF16, BF16, 51)
    table[1, 2] = -1
    table[0, 1] = -1
    gq, gk, gv, gt, gl = (t.to(cuda) for t in (q, kc, vc, table, lens))
    want = paged.paged_decode_attn(gq, gk, gv, gt, gl, 0.1)
    wide = gt.long()
    wide[1, 2] = (1 << 32) + 3
    wide[0, 1] = -(1 << 32) + 4
    assert torch.equal(paged.paged_decode_attn(gq, gk, gv, wide, gl.long(), 0.1), want)
    assert torch.equal(paged.paged_decode_attn(gq, gk, gv, gt.short(), gl.short(), 0.1), want)
    full = paged.paged_decode_attn(gq, gk, gv, gt, torch.full_like(gl, 2 ** 31 - 1), 0.1)
    assert torch.equal(paged.paged_decode_attn(gq, gk, gv, gt, torch.full_like(gl, 2 ** 31 - 1).long() + (1 << 33), 0.1), full)
    sel = torch.tensor([[[0, 2, (1 << 32) + 1], [0, 1 << 40, 3]]] * 2, device=cuda)
    plain_sel = sel.clamp(max=1 << 20).int()
    assert torch.equal(paged.paged_decode_attn(gq, gk, gv, gt, gl, 0.1, selected=sel),
                       paged.paged_decode_attn(gq, gk, gv, gt, gl, 0.1, selected=plain_sel))
    k = torch.ones(2, 2, 128, dtype=BF16, device=cuda)
    kept = gk.clone()
    paged.paged_append(k, k, gk, gv, wide, torch.tensor([17, 33], device=cuda))  # into those two entries
    assert torch.equal(gk, kept)
    for bad in (gt.float(), gt.bool()):
        with pytest.raises(ValueError):
            paged.paged_decode_attn(gq, gk, gv, bad, gl, 0.1)
    with pytest.raises(ValueError):
        paged.paged_append(k, k, gk, gv, gt, gl.float())
    with pytest.raises(ValueError):
        paged.paged_append(k, k, gk, gv, gt, gl, cu_seqlens=torch.tensor([0.0, 1.0, 2.0], device=cuda))
    with pytest.raises(ValueError):
        paged.paged_decode_attn(gq, gk, gv, gt, gl, 0.1, selected=plain_sel.float())
    assert torch.equal(gk, kept)


# ---------------------------------------------------------------------------- not quite numbers
FORMS = {  # lengths; q heads, kv heads, D, block, q, cache
    "a cluster a row": ([1, 40, 700, 2000], 8, 2, 128, 16, BF16, BF16),
    "a cluster a row, f16": ([1, 40, 700, 2000], 20, 2, 64, 8, F16, F16),
    "a cluster a row, 8-bit": ([1, 40, 700, 2000], 8, 2, 128, 16, BF16, FP8),
    "shared out, joined by rows": ([1, 40, 700, 9000] + [300] * 36, 8, 2, 128, 16, BF16, BF16),
    "shared out, joined by cuts": ([1, 40, 700, 9000] + [100] * 530, 8, 2, 64, 16, F16, FP8),
    "any type": ([1, 40, 700, 2000], 8, 2, 128, 16, F32, BF16),
    "any head dim": ([1, 40, 700, 9000], 6, 3, 40, 5, F16, F16),
}


def check_rows(q, kc, vc, table, lens, ks, vs, cuda):
    """As check_attention, where a row of the plain form may be NaN."""
    scaling = q.shape[-1] ** -0.5
    want, want_lse, weight, reach = plain.decode_attn(q, kc, vc, table, lens, scaling, ks, vs)
    got, lse = paged.paged_decode_attn(q.to(cuda), kc.to(cuda), vc.to(cuda), table.to(cuda), lens.to(cuda), scaling,
                                       k_scale=ks, v_scale=vs, return_lse=True)
    got, lse = got.double().cpu(), lse.double().cpu()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(lse.isnan(), want_lse.isnan())
    # (a value that is NaN leaves its row's other channels as they are, but not the bound of the whole)
    good = ~want.isnan()
    score = ((q.shape[-1] + 4) * 2.0 ** -23 * reach)[..., None].expand_as(want)
    p = 0.0 if kc.dtype == F32 or q.dtype == F32 else torch.finfo(BF16 if kc.dtype == BF16 else F16).eps / 2
    unit = torch.finfo(q.dtype).eps / 2
    tol = (p + 2 * score + 2.0 ** -16) * weight + unit * want.abs() * 1.01 + 2.0 ** -25
    assert ((got - want).abs() <= tol)[good].all()


@pytest.mark.parametrize("where", ["first", "last", "all"])
@pytest.mark.parametrize("form", list(FORMS))
def test_live_nan_reaches_its_rows_and_no_others(cuda, form, where):
    """A key that is NaN makes the rows of its KV head NaN wherever it lies, a value only its channel of them."""
    lens, Hq, Hk, D, block, qdt, cdt = FORMS[form]
    q, kc, vc, table, clen, ks, vs = attention_inputs(lens, Hq, Hk, D, block, qdt, cdt, 31)
    nan = torch.tensor(float("nan")).to(cdt)

    def at(b):
        t = {"first": [0], "last": [lens[b] - 1], "all": range(lens[b])}[where]
        return [(int(table[b, i // block]), i % block) for i in t]

    for b, h in ((0, 0), (1, 1), (3, 1)):
        for page, row in at(b):
            kc[page, h, row, D // 2] = nan
    for page, row in at(2):
        vc[page, 0, row, 3] = nan
    check_rows(q, kc, vc, table, clen, ks, vs, cuda)


@pytest.mark.parametrize("form", [f for f in FORMS if FORMS[f][-1] != FP8])
def test_scores_of_infinity(cuda, form):
    """-inf throughout: a row of zeros. -inf in some tokens: they have no weight. +inf: NaN, as inf - inf is."""
    lens, Hq, Hk, D, block, qdt, cdt = FORMS[form]
    q, kc, vc, table, clen, ks, vs = attention_inputs(lens, Hq, Hk, D, block, qdt, cdt, 32)
    q[..., 1] = q[..., 1].abs() + 0.5  # the sign of an infinite score is its key's
    for b, every, to in ((0, 1, -math.inf), (1, 1, -math.inf), (2, 3, -math.inf), (3, 1000, math.inf)):
        for i in range(0, lens[b], every):
            kc[int(table[b, i // block]), :, i % block, 1] = to
    keep = [0, 1]
    got, lse = paged.paged_decode_attn(q.to(cuda), kc.to(cuda), vc.to(cuda), table.to(cuda), clen.to(cuda), D ** -0.5,
                                       return_lse=True)
    assert (got[keep] == 0).all() and (lse[keep] == -math.inf).all()
    want, want_lse, weight, _ = plain.decode_attn(q, kc, vc, table, clen, D ** -0.5)
    assert want[3].isnan().all() and got[3].isnan().all() and lse[3].isnan().all()
    # sequence 2 as if every third token were not there
    assert not want[2].isnan().any()
    reach = (q[2].double().abs().amax(-1) * 16).max() * D ** 0.5  # |k| < 16, some sum of |q k| at most
    p = 0.0 if F32 in (qdt, cdt) else torch.finfo(BF16 if cdt == BF16 else F16).eps / 2
    tol = (p + 2 * (D + 4) * 2.0 ** -23 * reach + 2.0 ** -16) * weight[2] + torch.finfo(qdt).eps / 2 * want[2].abs() * 1.01 \
        + 2.0 ** -25
    assert ((got[2].double().cpu() - want[2]).abs() <= tol).all()


@pytest.mark.parametrize("heads", [4, 12])
@pytest.mark.parametrize("lens", [[40, 700], [9000, 3]])
def test_infinite_query_beside_large_ones(cuda, heads, lens):
    """Over an 8-bit cache a KV head's bf16 queries share a power of two: one that is infinite makes its own row NaN and
    leaves the others, which f16 could not hold unscaled, what they are."""
    q, kc, vc, table, clen, _, vs = attention_inputs(lens, 2 * heads, 2, 128, 16, BF16, FP8, 33)
    q = (q.float() * 1e5).bfloat16()
    q[0, 1, 5] = math.inf
    q[1, 0, 7] = float("nan")
    check_rows(q, kc, vc, table, clen, 1e-6, vs, cuda)


ODD_KEYS = [(4, 128, 16, BF16), (12, 64, 32, F16), (1, 256, 64, FP8), (3, 40, 5, F32), (8, 128, 8, FP8), (2, 96, 16, BF16)]


def odd_keys(Hk, D, block, cdt, g, lens):
    """Keys of which some are NaN (in a channel's every row, in one, in all of a page) or infinite."""
    table, nb = table_for(lens, block, g)
    kc = to_cache(torch.randn(nb, Hk, block, D, generator=g) * 3, cdt, 1.0)
    nan, inf = float("nan"), float("nan" if cdt == FP8 else "inf")
    for i, (rows, ch, to) in enumerate([(slice(None), 3, nan), (0, slice(None), nan), (slice(1, 3), 7, nan),
                                        (slice(None), slice(None), nan), (1, 5, inf), (0, 6, -inf), (slice(None), 2, inf)]):
        kc[int(table[1, i]), :, rows, ch] = to
    kc[int(table[0, 0]), :, 0, 1] = nan  # its only token
    page = int(table[1, 7])  # every other channel half way between two codes, and no more than the smallest numbers
    kc[page, :, :, 0] = 127.0
    kc[page, :, :, 1::2] = 20.5 if cdt != FP8 else 20.0
    kc[page, :, :, 2] = nan
    kc[int(table[1, 8])] = torch.finfo(cdt).tiny * 2
    kc[int(table[1, 8]), :, :, 5] = nan
    return kc, table, nb


@pytest.mark.parametrize("Hk,D,block,cdt", ODD_KEYS)
def test_summary_of_keys_that_are_not_numbers(cuda, Hk, D, block, cdt):
    lens = [1, block * 9 - 2]
    kc, table, nb = odd_keys(Hk, D, block, cdt, gen(D + block), lens)
    ks = 0.3 if cdt == FP8 else 1.0
    gk = kc.to(cuda)
    code, scale = paged.new_block_summary(gk)
    want_code, want_scale = code.cpu().clone(), scale.cpu().clone()
    paged.paged_block_summary(gk, table.to(cuda), torch.tensor(lens, device=cuda), code, scale, k_scale=ks)
    expected_summary(kc, table, lens, block, torch.tensor(ks, dtype=F32), want_code, want_scale)
    assert torch.isfinite(scale).all()
    assert torch.equal(scale.cpu(), want_scale) and torch.equal(code.cpu(), want_code)


@pytest.mark.parametrize("Hk,D,block,cdt", ODD_KEYS)
def test_choice_for_queries_and_keys_that_are_not_numbers(cuda, Hk, D, block, cdt):
    g = gen(D + block + 1)
    lens = [1, block * 40 - 2]
    kc, table, nb = odd_keys(Hk, D, block, cdt, g, lens)
    qdt = {BF16: BF16, F16: F16, FP8: BF16, F32: F32}[cdt]
    q = torch.randn(2, 3 * Hk, D, generator=g).to(qdt)
    q[1, 0, 4] = float("nan")
    q[1, 1] = float("nan")
    if Hk > 1:
        q[1, 3, 9], q[1, 4, 0] = math.inf, -math.inf
    q[0, 0, 0] = math.inf
    gk = kc.to(cuda)
    code, scale = paged.new_block_summary(gk)
    clen = torch.tensor(lens, dtype=torch.int32)
    paged.paged_block_summary(gk, table.to(cuda), clen.to(cuda), code, scale)
    for budget in (3, 11):
        got = paged.paged_select_blocks(q.to(cuda), code, scale, table.to(cuda), clen.to(cuda), budget, block)
        assert torch.equal(got.cpu(), plain.select(q, code.cpu(), scale.cpu(), table, clen, budget, block, 0, 1))


@pytest.mark.parametrize("heads,D,cdt", [(4, 128, BF16), (12, 128, BF16), (8, 64, BF16), (3, 256, BF16), (16, 256, F16),
                                         (4, 128, F16), (10, 64, F16)])
@pytest.mark.parametrize("lens", [[700, 1, 40], [9000, 300] + [150] * 60])
def test_weights_over_16_bit_caches_keep_more_than_16_bits(cuda, heads, D, cdt, lens):
    """test_gpu_paged.py's bound with the weights' rounding at 2^-16 (bf16: 2^-8 twice over) and 2^-22 (f16) in place of
    2^-8 and 2^-11: where a row's values cancel, the output's own rounding does not hide it."""
    q, kc, vc, table, clen, ks, vs = attention_inputs(lens, 2 * heads, 2, D, 16, cdt, cdt, 91)
    want, _, weight, reach = plain.decode_attn(q, kc, vc, table, clen, D ** -0.5)
    got = paged.paged_decode_attn(*(t.to(cuda) for t in (q, kc, vc, table, clen)), D ** -0.5).double().cpu()
    score = (D + 4) * 2.0 ** -23 * reach[..., None]
    p = 2.0 ** -16 if cdt == BF16 else 2.0 ** -22
    tol = (p + 2 * score + 2.0 ** -16) * weight + torch.finfo(cdt).eps / 2 * want.abs() * 1.01 + 2.0 ** -25
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()


# ----------------------------------------------------------------------- streams, host threads
def select_through_c(q, code, scale, table, lens, block, out, ws, stream):
    """A call of the C entry point itself: ctypes lets other host threads run meanwhile, the Python layer's glue does not."""
    f = N.lib().bd_paged_select
    f.restype = ctypes.c_int
    d = [N.ref(N.desc(t)) for t in (q, code, scale, table, lens, out)]
    I = ctypes.c_int  # noqa: E741
    args = (*d[:5], I(block), I(0), I(1), d[5], ctypes.c_void_p(ws.data_ptr()), ctypes.c_size_t(ws.numel()),
            ctypes.c_void_p(stream.cuda_stream))
    return lambda: f(*args)


def test_choice_from_two_host_threads_with_unlike_heads(cuda):
    """Head counts that need different amounts of shared memory of the same kernel, launched by two threads at once."""
    block, D, calls = 16, 256, 5000
    work = []
    for heads in (128, 97):
        g = gen(heads)
        table, nb = table_for([block * 90], block, g)
        code = torch.randint(-127, 128, (nb, 1, 2, D), generator=g).to(torch.int8).to(cuda)
        scale = torch.rand(nb, 1, generator=g).to(cuda)
        q = torch.randn(1, heads, D, generator=g).bfloat16().to(cuda)
        lens = torch.tensor([block * 90], dtype=torch.int32, device=cuda)
        want = paged.paged_select_blocks(q, code, scale, table.to(cuda), lens, 7, block)
        work.append((q, code, scale, table.to(cuda), lens, block, torch.empty_like(want),
                     torch.empty(1 << 16, dtype=torch.uint8, device=cuda), torch.cuda.Stream(), want))
    torch.cuda.synchronize()
    bad, start = [], threading.Barrier(2)

    def run(w):
        call = select_through_c(*w[:9])
        start.wait()
        for _ in range(calls):
            rc = call()
            if rc:
                bad.append((rc, N.lib().bd_last_error()))
                return

    threads = [threading.Thread(target=run, args=(w,)) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not bad
    for w in work:
        assert torch.equal(w[6], w[9])


def test_calls_on_two_streams_at_once(cuda):
    """The same chains of calls on two streams, whose kernels come early and overlap: each as it is alone."""
    def inputs(seed):
        x = attention_inputs([3000, 0, 40, 777], 28, 4, 128, 16, BF16, FP8 if seed % 2 else BF16, seed)
        q, kc, vc, table, lens = (t.to(cuda) for t in x[:5])
        return q, kc, vc, table, lens, x[5], x[6], *paged.new_block_summary(kc), \
            torch.randn(4, 4, 128, generator=gen(seed)).bfloat16().to(cuda)

    def chain(q, kc, vc, table, lens, ks, vs, code, scale, k):
        n, out = lens.clone(), []
        paged.paged_block_summary(kc, table, n, code, scale, k_scale=ks)
        for _ in range(6):
            n += 1
            paged.paged_append(k, k, kc, vc, table, n, k_scale=ks, v_scale=vs, summary=code, summary_scale=scale)
            out.append(paged.paged_sparse_decode_attn(q, kc, vc, code, scale, table, n, 9, 0.1, k_scale=ks, v_scale=vs))
            out.append(paged.paged_decode_attn(q, kc, vc, table, n, 0.1, k_scale=ks, v_scale=vs))
        return out

    alone = [chain(*inputs(seed)) for seed in (41, 42)]
    torch.cuda.synchronize()
    ready = [inputs(seed) for seed in (41, 42)]
    streams = [torch.cuda.Stream() for _ in ready]
    torch.cuda.synchronize()
    got = []
    for s, x in zip(streams, ready):
        with torch.cuda.stream(s):
            got.append(chain(*x))
    torch.cuda.synchronize()
    for a, b in zip(alone, got):
        for x, y in zip(a, b):
            assert torch.equal(bits(x), bits(y))


def test_counts_past_32_bits_and_summaries_of_other_shapes(cuda):
    """Refused with their own message, not cut to their lower halves; nothing as large as asked for is made first."""
    kc = torch.zeros(6, 2, 16, 64, dtype=BF16, device=cuda)
    code, scale = paged.new_block_summary(kc)
    table, lens = torch.zeros(1, 3, dtype=torch.int32, device=cuda), torch.ones(1, dtype=torch.int32, device=cuda)
    q = torch.zeros(1, 8, 64, dtype=BF16, device=cuda)
    big = 1 << 32

    def select(match, code=code, budget=2, block=16, **kw):
        with pytest.raises(ValueError, match=match):
            paged.paged_select_blocks(q, code, scale, table, lens, budget, block, **kw)
        if block == 16:
            with pytest.raises(ValueError, match=match):
                paged.paged_sparse_decode_attn(q, kc, kc, code, scale, table, lens, budget, 1.0, **kw)

    select("block_size", block=big + 16)
    select("sink_blocks", sink_blocks=big)
    select("recent_blocks", recent_blocks=big + 1)
    select("chosen pages", budget=1 << 50)
    select("summary", code=code[0])


# ------------------------------------------------------------------- which kernels a call launches
def launched(call):
    """[(kernel's name and template arguments, CTAs of a cluster)] of a captured call."""
    drv = pytest.importorskip("cuda.bindings.driver")

    def ok(r):
        assert int(r[0]) == 0, r
        return r[1] if len(r) == 2 else r[1:]

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    handle, out = drv.CUgraph(graph.raw_cuda_graph()), []
    n = ok(drv.cuGraphGetNodes(handle, 0))[1]
    for node in ok(drv.cuGraphGetNodes(handle, n))[0][:n]:
        if ok(drv.cuGraphNodeGetType(node)) != drv.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL:
            continue
        p = ok(drv.cuGraphKernelNodeGetParams(node))
        name = (ok(drv.cuFuncGetName(p.func)) if int(p.func) else ok(drv.cuKernelGetName(p.kern))).decode()
        found = re.search(r"\d(paged_[a-z_]+kernel)(I(?:L[ib]\d+E|\d*[a-zA-Z_]\w*?)*E)?", name)
        cluster = ok(drv.cuGraphKernelNodeGetAttribute(
            node, drv.CUlaunchAttributeID.CU_LAUNCH_ATTRIBUTE_CLUSTER_DIMENSION)).clusterDim.x
        out.append((found.group(1), [int(x) for x in re.findall(r"Li(\d+)E", found.group(2) or "")], cluster))
    return out


def widened(table, columns):
    wide = torch.full((table.shape[0], columns), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    return wide


# lengths, KV heads, columns of the table (0: as the lengths need); what follows from them: CTAs of a row's cluster, or
# the join and how many heads a CTA of it takes
PATHS = {
    "a CTA a row": ([150, 0, 33] * 8, 2, 0, 1),
    "two CTAs a row": ([700, 0, 333, 1, 90, 1024] * 3, 2, 0, 2),
    "four CTAs a row": ([900, 0, 1000, 17] * 3, 2, 0, 4),
    "eight CTAs a row": ([3000, 0, 1777, 16], 2, 0, 8),
    "sixteen CTAs a row": ([5000, 15], 2, 0, 16),
    "joined by rows, a head a CTA": ([4000, 0, 9, 2500], 2, 60000, "one"),
    "joined by rows, several heads a CTA": ([30, 0, 9, 50, 71, 18, 2000] * 45, 2, 0, "rows"),
    "joined by cuts": ([70, 0, 9, 50, 71, 18, 1000] * 155, 2, 0, "cuts"),
}


@pytest.mark.parametrize("heads,D,qdt,cdt", [(4, 128, BF16, BF16), (7, 128, BF16, FP8), (8, 64, F16, F16),
                                             (16, 64, BF16, FP8), (8, 256, F16, FP8), (11, 128, F16, F16),
                                             (2, 256, BF16, BF16), (9, 64, BF16, BF16), (16, 256, BF16, BF16),
                                             (12, 256, BF16, FP8), (10, 256, F16, F16), (13, 128, BF16, FP8)])
@pytest.mark.parametrize("path", list(PATHS))
def test_each_path_of_the_attention(cuda, path, heads, D, qdt, cdt):
    """Each way of sharing the work out, seen to be the one that runs."""
    if torch.cuda.get_device_properties(cuda).multi_processor_count != 148:
        pytest.skip("the sizes are for 148 SMs")
    lens, Hk, columns, want = PATHS[path]
    q, kc, vc, table, clen, ks, vs = attention_inputs(lens, heads * Hk, Hk, D, 16 if heads % 2 else 8, qdt, cdt, heads)
    if columns:
        table = widened(table, columns)
    on = [t.to(cuda) for t in (q, kc, vc, table, clen)]
    got = launched(lambda: paged.paged_decode_attn(*on, 0.1, k_scale=ks, v_scale=vs))
    assert got[0][0] == "paged_attn_tile_kernel"
    if isinstance(want, int):
        assert len(got) == 1 and max(1, got[0][2]) == want, got
    else:
        name, args, _ = got[1]
        many = 4 if D == 256 else 8
        if want == "cuts" or path == "joined by rows, several heads a CTA" and name.endswith("cuts_kernel") and heads > many:
            assert name == "paged_tile_join_cuts_kernel", got  # (two groups of heads are twice as many CTAs)
        else:
            assert name == "paged_tile_join_kernel" and args[-1] == (1 if want == "one" else many), got
    check_attention(q, kc, vc, table, clen, ks, vs, cuda)


@pytest.mark.parametrize("qdt,cdt,D,block", [(F32, BF16, 128, 16), (BF16, F16, 128, 16), (F16, F16, 96, 16), (BF16, BF16, 64, 12)])
def test_what_the_tiles_cannot_take_goes_to_the_general_form(cuda, qdt, cdt, D, block):
    q, kc, vc, table, clen, ks, vs = attention_inputs([50, 0, 700], 6, 2, D, block, qdt, cdt, 61)
    on = [t.to(cuda) for t in (q, kc, vc, table, clen)]
    assert [x[0] for x in launched(lambda: paged.paged_decode_attn(*on, 0.1))] == ["paged_attn_generic_kernel", "paged_join_kernel"]
    check_attention(q, kc, vc, table, clen, ks, vs, cuda)


# -------------------------------------------------------------------------- tables, pages, types
@pytest.mark.parametrize("D,cdt", [(128, BF16), (64, FP8), (40, F32)])
def test_choice_and_summaries_at_a_wide_table(cuda, D, cdt):
    """A table far wider than the lengths, as a loop that replays a graph has it: summaries, choice and chained attention
    as at a table of their own width."""
    lens = [700, 20, 0, 1, 5000]
    q, kc, vc, table, clen, ks, vs = attention_inputs(lens, 8, 2, D, 16, F32 if cdt == F32 else BF16, cdt, 71)
    gq, gk, gv, gl = (t.to(cuda) for t in (q, kc, vc, clen))
    both = []
    for t in (table, widened(table, 9000), widened(table, 70000)):
        gt = t.to(cuda)
        code, scale = paged.new_block_summary(gk)
        paged.paged_block_summary(gk, gt, gl, code, scale, k_scale=ks)
        out, sel = paged.paged_sparse_decode_attn(gq, gk, gv, code, scale, gt, gl, 6, 0.1, sink_blocks=1, recent_blocks=2,
                                                  k_scale=ks, v_scale=vs, return_selected=True)
        both.append((code, scale, sel, out))
    want = plain.select(q, both[0][0].cpu(), both[0][1].cpu(), table, clen, 6, 16, 1, 2)
    for code, scale, sel, out in both:
        assert torch.equal(code, both[0][0]) and torch.equal(scale, both[0][1])
        assert torch.equal(sel.cpu(), want)
        # (how the rows are shared out, and with that the order of the sums, follows from the chosen pages alone)
        assert torch.equal(bits(out), bits(both[0][3]))


def touched(lens, new, block, columns, packed):
    """Pages of each sequence that an append of new[b] tokens lies in."""
    out = []
    for n, m in zip(lens, new):
        last = (n - 1) // block if n > 0 else -1
        if last >= columns:
            last = columns - 1 if packed else -1
        out.append(range(max(n - m, 0) // block, last + 1) if m else range(0))
    return out


@pytest.mark.parametrize("Hk,D,block,cdt", [(4, 128, 16, FP8), (3, 64, 32, F16), (2, 256, 8, BF16), (2, 40, 5, F32),
                                            (1, 64, 16, FP8), (2, 96, 12, F16)])
@pytest.mark.parametrize("packed", [True, False])
def test_append_keeps_summaries_of_every_type(cuda, packed, Hk, D, block, cdt):
    """The touched pages' summaries are the rebuild's, all others stay; some tokens have no place."""
    new = [1, 3 * block + 2, 0, block, 7, 2] if packed else [1] * 6
    past = [block - 1, 3, 30, 2 * block, 4 * block - 2, block]
    lens = [a + b for a, b in zip(new, past)]
    if not packed:
        lens[2] = 0  # idle
    g = gen(D + block)
    table, nb = table_for(lens, block, g, extra_columns=0)
    table = table[:, :4]              # sequences that reach past it
    table[3, 2] = -1                  # a page that is none
    qdt = {FP8: BF16, F16: F16, BF16: BF16, F32: F32}[cdt]
    ks, vs = (0.25, 0.5) if cdt == FP8 else (1.0, 1.0)
    kc, vc = (to_cache(torch.randn(nb, Hk, block, D, generator=g), cdt, 1.0).to(cuda) for _ in "kv")
    k, v = (torch.randn(sum(new), Hk, D, generator=g).to(qdt).to(cuda) for _ in "kv")
    code, scale = paged.new_block_summary(kc)
    code.fill_(77)
    scale.fill_(-1.0)
    cu = torch.tensor([0] + new).cumsum(0).int().to(cuda) if packed else None
    gt, gl = table.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda)
    paged.paged_append(k, v, kc, vc, gt, gl, cu_seqlens=cu, k_scale=ks, v_scale=vs, summary=code, summary_scale=scale)
    every = paged.new_block_summary(kc)
    paged.paged_block_summary(kc, gt, gl, *every, k_scale=ks)
    pages = [int(table[b, j]) for b, r in enumerate(touched(lens, new, block, 4, packed)) for j in r]
    pages = sorted(p for p in pages if 0 <= p < nb)
    assert pages
    others = [p for p in range(nb) if p not in pages]
    assert torch.equal(code[pages], every[0][pages]) and torch.equal(scale[pages], every[1][pages])
    assert (code[others] == 77).all() and (scale[others] == -1).all()
    # and the rebuild's are the plain form's
    want = torch.zeros(nb, Hk, 2, D, dtype=torch.int8), torch.zeros(nb, Hk)
    expected_summary(kc.cpu(), table, [min(n, 4 * block) for n in lens], block, torch.tensor(ks, dtype=F32), *want)
    assert torch.equal(every[0].cpu(), want[0]) and torch.equal(every[1].cpu(), want[1])


def test_choice_and_summaries_past_32_bit_offsets(cuda):
    """Summaries of more than 2^32 bytes over a cache of more than 2^31: pages at the far end."""
    nb, Hk, block, D = 140000, 64, 1, 256
    kc = torch.zeros(nb, Hk, block, D, dtype=FP8, device=cuda)
    far = [nb - 1, 3, nb - 7, nb // 2 + 1, nb - 2]
    g = gen(81)
    for p in far:
        kc[p] = to_cache(torch.randn(Hk, block, D, generator=g), FP8, 1.0).to(cuda)
    code, scale = paged.new_block_summary(kc)
    table, lens = torch.tensor([far], dtype=torch.int32), torch.tensor([5], dtype=torch.int32)
    paged.paged_block_summary(kc, table.to(cuda), lens.to(cuda), code, scale)
    small = torch.zeros(5, Hk, 2, D, dtype=torch.int8), torch.zeros(5, Hk)
    local = torch.arange(5, dtype=torch.int32)[None]
    expected_summary(kc[far].cpu(), local, [5], block, torch.tensor(1.0), *small)
    assert torch.equal(code[far].cpu(), small[0]) and torch.equal(scale[far].cpu(), small[1])
    q = torch.randn(1, 2 * Hk, D, generator=g).bfloat16()
    for budget in (2, 4):
        got = paged.paged_select_blocks(q.to(cuda), code, scale, table.to(cuda), lens.to(cuda), budget, block, recent_blocks=0)
        assert torch.equal(got.cpu(), plain.select(q, *small, local, lens, budget, block, 0, 0))
    # summaries with rows that no vector load can take
    odd = code.view(nb, Hk, -1).new_zeros(16, Hk, 2 * D + 1)
    assert odd[..., 1:].unflatten(2, (2, D)).stride(1) % 16  # (the general form; its offsets are the same products)
    at = odd[..., 1:].unflatten(2, (2, D))
    at[:5] = small[0].to(cuda)
    s = torch.zeros(16, Hk, device=cuda)
    s[:5] = small[1].to(cuda)
    got = paged.paged_select_blocks(q.to(cuda), at, s, local.to(cuda), lens.to(cuda), 3, block, recent_blocks=0)
    assert torch.equal(got.cpu(), plain.select(q, *small, local, lens, 3, block, 0, 0))
