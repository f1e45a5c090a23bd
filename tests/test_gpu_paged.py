"""The paged-cache operators against the plain restatement in oracle/paged.py.

Tolerances follow from the arithmetic, element by element:
* append: the two products and their sum are rounded in fp32 (3 * 2^-24 of the products'
  magnitudes), then once to the stored type (half its unit, plus half its smallest subnormal).
* attention: a score is off by at most (D + 4) * 2^-23 of its sum of |q k| (fp32 sums, some of them
  truncating), which moves every weight by that factor, twice over with the denominator's; a weight
  is rounded to the cache's type where the tensor cores take it (2^-8 bf16, 2^-11 f16; fp8 caches
  are read as f16) or not at all; 2^-16 covers the fp32 sums over tokens; then the output's rounding.
* summaries and choices: equal.
"""
import math

import pytest
import torch

from bytes_b200 import paged
from oracle import paged as plain

pytestmark = pytest.mark.gpu

BF16, F16, F32, FP8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
# the largest relative rounding of a type (half its eps), and half its smallest subnormal
UNIT = {t: torch.finfo(t).eps / 2 for t in (BF16, F16, F32, FP8)}
TINY = {BF16: 0.0, F16: 2.0 ** -25, F32: 0.0, FP8: 2.0 ** -10}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def table_for(lens, block, g, spare=3, extra_columns=2):
    """Pages in random order; columns past a sequence's pages name no page."""
    counts = [-(-max(n, 0) // block) for n in lens]
    wide = max(1, max(counts) + extra_columns)
    order = torch.randperm(sum(counts) + spare, generator=g).tolist()
    table = torch.full((len(lens), wide), -1, dtype=torch.int32)
    for b, c in enumerate(counts):
        for j in range(c):
            table[b, j] = order.pop()
    return table, sum(counts) + spare


def to_cache(x, dtype, scale):
    return (x.float() / scale).clamp(-448, 448).to(dtype) if dtype == FP8 else x.to(dtype)


def bits(x):
    return x.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[x.element_size()])


def angles(positions, r, base=10000.0):
    a = torch.arange(positions).double()[:, None] * base ** (-torch.arange(0, r, 2).double() / r)
    return a.cos().float(), a.sin().float()


# ------------------------------------------------------------------------------------- append
APPEND = [
    # new tokens, tokens before, q heads, kv heads, D, block, rotated channels, interleaved, input, cache
    ([1], [0], 28, 4, 128, 16, 128, False, BF16, BF16),
    ([1, 1, 1, 1], [15, 16, 17, 700], 32, 8, 128, 16, 128, False, BF16, FP8),
    ([1, 37, 5, 64], [0, 0, 30, 3], 16, 2, 128, 16, 64, False, BF16, BF16),
    ([3, 1, 50], [7, 0, 1], 12, 12, 64, 32, 64, True, F16, F16),
    ([2, 40], [5, 61], 8, 1, 256, 8, 256, True, BF16, FP8),
    ([2, 9], [5, 0], 4, 2, 96, 12, 48, False, F32, F32),
    ([6, 4], [1, 20], 6, 3, 40, 5, 10, True, F32, BF16),
    ([17], [100], 8, 8, 64, 64, 0, False, BF16, BF16),
]


@pytest.mark.parametrize("case", APPEND)
@pytest.mark.parametrize("split", [False, True])
def test_append(cuda, case, split):
    new, past, Hq, Hk, D, block, r, inter, dt, cdt = case
    g = gen(sum(new) + D)
    lens = [a + b for a, b in zip(new, past)]
    table, nb = table_for(lens, block, g)
    T = sum(new)
    ks, vs = (0.25, 0.5) if cdt == FP8 else (1.0, 1.0)
    if split:  # views of one projection's rows, pages kept token-major
        qkv = torch.randn(T, (Hq + 2 * Hk) * D, generator=g).to(dt)
        q, k, v = (x.unflatten(1, (-1, D)) for x in qkv.split([Hq * D, Hk * D, Hk * D], 1))
        kc, vc = (to_cache(torch.randn(nb, block, Hk, D, generator=g), cdt, 1.0).transpose(1, 2) for _ in "kv")
    else:
        q, k, v = (torch.randn(T, h, D, generator=g).to(dt) for h in (Hq, Hk, Hk))
        kc, vc = (to_cache(torch.randn(nb, Hk, block, D, generator=g), cdt, 1.0) for _ in "kv")
    cos, sin = angles(max(lens), r) if r else (None, None)
    cu = None if max(new) == 1 else torch.tensor([0] + new).cumsum(0).int()
    clen = torch.tensor(lens, dtype=torch.int32)
    dev = lambda t: None if t is None else t.to(cuda)  # noqa: E731
    gk, gv = kc.to(cuda), vc.to(cuda)
    if split:
        dqkv = qkv.to(cuda)
        dq, dk, dv = (x.unflatten(1, (-1, D)) for x in dqkv.split([Hq * D, Hk * D, Hk * D], 1))
        assert gk.stride(1) != block * D or Hk == 1
    else:
        dq, dk, dv = q.to(cuda), k.to(cuda), v.to(cuda)
    got = paged.paged_append(dk, dv, gk, gv, table.to(cuda), clen.to(cuda), q=dq, cos=dev(cos), sin=dev(sin),
                             interleaved=inter, cu_seqlens=dev(cu), k_scale=ks, v_scale=vs)
    got, gk, gv = got.cpu(), gk.cpu(), gv.cpu()
    untouched = torch.ones(nb, block, dtype=torch.bool)
    seen = 0
    for t, page, row, ek, ev, eq, mk, mq in plain.append(k, v, q, cos, sin, inter, cu, table, clen, nb, block):
        untouched[page, row] = False
        seen += 1
        for x, want, mag, typ, sc in ((gk[page, :, row], ek, mk, cdt, ks), (gv[page, :, row], ev, 0 * ev, cdt, vs),
                                      (got[t], eq, mq, dt, 1.0)):
            want, mag = want / sc, mag / sc
            tol = UNIT[typ] * want.abs() * 1.01 + TINY[typ] + 3 * 2.0 ** -24 * (mag + want.abs())
            if typ == FP8:
                want = want.clamp(-448, 448)
            assert ((x.double() - want).abs() <= tol).all()
    assert seen == T
    for a, b in ((gk, kc), (gv, vc)):
        same = (bits(a.contiguous()) == bits(b.contiguous())).all(-1).all(1)
        assert same[untouched].all()


def test_append_tokens_without_a_place(cuda):
    """Padding past cu_seqlens, an idle sequence, a full block table, a page entry outside the cache,
    a position past the rows of cos: nothing is written and the query rows are zeros."""
    g = gen(5)
    Hq, Hk, D, block, nb = 4, 2, 64, 16, 4
    table = torch.tensor([[0, 1], [2, 99], [-1, 3], [3, 1]], dtype=torch.int32)
    cos, sin = (x.to(cuda) for x in angles(40, D))
    q, k, v = (torch.randn(9, h, D, generator=g).bfloat16().to(cuda) for h in (Hq, Hk, Hk))

    def run(new, lens, rows=40):
        kc, vc = (torch.full((nb, Hk, block, D), 7.0, dtype=BF16, device=cuda) for _ in "kv")
        cu = torch.tensor([0] + new).cumsum(0).int().to(cuda)
        got = paged.paged_append(k, v, kc, vc, table.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda), q=q,
                                 cos=cos[:rows], sin=sin[:rows], cu_seqlens=cu)
        wrote = (kc != 7).any(-1).any(1), (vc != 7).any(-1).any(1)
        assert torch.equal(*wrote)
        return (got != 0).any(-1).any(-1).tolist(), sorted(map(tuple, wrote[0].nonzero().tolist()))

    # sequence 0: one token at 3; 1: two at 15, 16 (page 99 is none); 2: two at 15 (page -1), 16; 3: idle
    live, wrote = run([1, 2, 2, 0], [4, 17, 17, 0])
    assert live == [True, True, False, False, True, False, False, False, False]
    assert wrote == [(0, 3), (2, 15), (3, 0)]
    # more new tokens than the sequence holds; past the block table; past the rows of cos (rows 0..4)
    live, wrote = run([3, 2, 0, 2], [2, 34, 0, 6], rows=5)
    assert live == [False, True, True, False, False, True, False, False, False]
    assert wrote == [(0, 0), (0, 1), (3, 4)]


# ---------------------------------------------------------------------------------- summaries
def expected_summary(kc, table, lens, block, ks, code, scale, first=None):
    nb, Hk = kc.shape[:2]
    for b, n in enumerate(lens):
        for j in range((first[b] if first else 0) // block, -(-n // block)):
            p = int(table[b, j])
            if not 0 <= p < nb:
                continue
            for h in range(Hk):
                code[p, h], scale[p, h] = plain.summary_of(kc[p, h, :min(block, n - j * block)].float() * ks)


@pytest.mark.parametrize("Hk,D,block,cdt", [(4, 128, 16, BF16), (12, 64, 32, F16), (1, 256, 64, FP8), (3, 40, 5, F32),
                                            (8, 128, 8, FP8), (2, 128, 128, BF16)])
def test_block_summary(cuda, Hk, D, block, cdt):
    g = gen(Hk * D)
    lens = [0, 1, block, block + 1, 5 * block - 1]
    table, nb = table_for(lens, block, g)
    table[4, 1] = nb + 5  # names no page
    ks = 0.3 if cdt == FP8 else 1.0
    kc = to_cache(torch.randn(nb, Hk, block, D, generator=g) * 3, cdt, 1.0)
    kc[int(table[2, 0])] = 0  # a page of zeros
    # stale values past a sequence's end must not count
    kc[int(table[3, 1]), :, 1:] = float("nan")
    gk = kc.to(cuda)
    code, scale = paged.new_block_summary(gk)
    want_code, want_scale = code.cpu().clone(), scale.cpu().clone()
    paged.paged_block_summary(gk, table.to(cuda), torch.tensor(lens, device=cuda), code, scale, k_scale=ks)
    expected_summary(kc, table, lens, block, torch.tensor(ks, dtype=F32), want_code, want_scale)
    assert torch.equal(scale.cpu(), want_scale)
    assert torch.equal(code.cpu(), want_code)


@pytest.mark.parametrize("new,past,block", [([1, 1, 1], [15, 16, 200], 16), ([20, 1, 70], [9, 0, 33], 16),
                                            ([5, 64], [0, 62], 64), ([7, 3], [2, 30], 8)])
def test_append_keeps_summaries(cuda, new, past, block):
    g = gen(sum(new))
    Hq, Hk, D = 8, 4, 128
    lens = [a + b for a, b in zip(new, past)]
    table, nb = table_for(lens, block, g)
    kc, vc = (torch.randn(nb, Hk, block, D, generator=g).bfloat16().to(cuda) for _ in "kv")
    k, v = (torch.randn(sum(new), Hk, D, generator=g).bfloat16().to(cuda) for _ in "kv")
    code, scale = paged.new_block_summary(kc)
    cos, sin = (x.to(cuda) for x in angles(max(lens), D))
    cu = None if max(new) == 1 else torch.tensor([0] + new).cumsum(0).int().to(cuda)
    got = paged.paged_append(k, v, kc, vc, table.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda), cos=cos,
                             sin=sin, cu_seqlens=cu, summary=code, summary_scale=scale)
    assert got is None
    want_code, want_scale = torch.zeros(nb, Hk, 2, D, dtype=torch.int8), torch.zeros(nb, Hk)
    expected_summary(kc.cpu(), table, lens, block, torch.tensor(1.0), want_code, want_scale, first=past)
    assert torch.equal(scale.cpu(), want_scale) and torch.equal(code.cpu(), want_code)


# ----------------------------------------------------------------------------------- attention
def attention_inputs(lens, Hq, Hk, D, block, qdt, cdt, seed, token_major=False):
    g = gen(seed)
    table, nb = table_for(lens, block, g)
    ks, vs = (0.11, 0.37) if cdt == FP8 else (1.0, 1.0)
    shape = (nb, block, Hk, D) if token_major else (nb, Hk, block, D)
    kc, vc = (to_cache(torch.randn(shape, generator=g) * m, cdt, s) for m, s in ((2.0, ks), (1.0, vs)))
    if token_major:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    q = (torch.randn(len(lens), Hq, D, generator=g) * 1.5).to(qdt)
    return q, kc, vc, table, torch.tensor(lens, dtype=torch.int32), ks, vs


def check_attention(q, kc, vc, table, lens, ks, vs, cuda, selected=None, q4=False):
    D = q.shape[-1]
    scaling = D ** -0.5
    want, want_lse, weight, reach = plain.decode_attn(q, kc, vc, table, lens, scaling, ks, vs, selected)
    gq = q.to(cuda).unsqueeze(2) if q4 else q.to(cuda)
    got, lse = paged.paged_decode_attn(gq, kc.to(cuda), vc.to(cuda), table.to(cuda), lens.to(cuda), scaling, k_scale=ks,
                                       v_scale=vs, selected=None if selected is None else selected.to(cuda),
                                       return_lse=True)
    assert got.shape == gq.shape and got.dtype == q.dtype
    got, lse = got.reshape(q.shape).double().cpu(), lse.double().cpu()
    score = (D + 4) * 2.0 ** -23 * reach
    p = 0.0 if kc.dtype == F32 or q.dtype == F32 else UNIT[BF16 if kc.dtype == BF16 else F16]
    tol = (p + 2 * score[..., None] + 2.0 ** -16) * weight + UNIT[q.dtype] * want.abs() * 1.01 + TINY[q.dtype]
    assert torch.isfinite(got).all()
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol.clamp(min=1e-30)).max()
    empty = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert (got[empty] == 0).all()
    off = (lse - want_lse)[~empty].abs()
    assert (off <= score[~empty] + 2.0 ** -16 + 2.0 ** -23 * want_lse[~empty].abs()).all()


LENS = [0, 1, 15, 16, 17, 64, 333, 1000]
ATTN = [
    # q heads, kv heads, D, block, q, cache
    (28, 4, 128, 16, BF16, BF16), (32, 8, 128, 16, BF16, FP8), (12, 12, 64, 32, F16, F16), (8, 1, 256, 16, BF16, BF16),
    (32, 2, 128, 64, BF16, BF16), (48, 1, 64, 16, F16, FP8), (40, 8, 64, 8, BF16, FP8), (6, 2, 256, 32, F16, FP8),
    (20, 1, 256, 8, F16, F16), (16, 16, 128, 128, BF16, BF16), (8, 2, 128, 16, F32, BF16), (8, 2, 128, 16, F16, BF16),
    (8, 2, 128, 16, F32, F32), (9, 3, 40, 5, BF16, BF16), (4, 4, 96, 48, BF16, FP8), (2, 1, 1, 1, F32, F32),
    (24, 24, 256, 256, BF16, FP8), (40, 2, 128, 8, F16, F16),
]


@pytest.mark.parametrize("Hq,Hk,D,block,qdt,cdt", ATTN)
def test_decode_attn(cuda, Hq, Hk, D, block, qdt, cdt):
    x = attention_inputs(LENS, Hq, Hk, D, block, qdt, cdt, Hq + D)
    check_attention(*x, cuda)


# How the work is shared out depends on how many rows there are and how long they and the block table are:
# a CTA a row, cut rows joined row by row (a head a CTA, eight heads a CTA), many rows joined by
# what cuts them, running sums of one sequence a lane, of one and of several a group.
SHARED_OUT = {
    "a CTA a row": lambda g: ([700, 0, 333, 1, 90, 1024] * 3, 2),
    "two CTAs a row": lambda g: ([1200, 0, 333, 1, 90, 2024, 16, 17] * 3, 2),
    "eight CTAs a row": lambda g: ([3000, 0, 1777, 16], 2),
    "sixteen CTAs a row": lambda g: ([5000, 15], 2),
    "few rows, one CTA a head": lambda g: ([4000, 0, 9, 2500], 2),
    "few long rows": lambda g: ([30000, 0, 9, 2500], 2),
    "eight heads a CTA": lambda g: (torch.randint(0, 1500, (40,), generator=g).tolist() + [3001], 2),
    "many rows, long and short": lambda g: (torch.randint(0, 90, (310,), generator=g).tolist() + [2777, 0, 1500], 2),
    "many rows alike": lambda g: ([100] * 160, 4),
    "several sequences a group": lambda g: (torch.randint(0, 20, (1500,), generator=g).tolist() + [600], 1),
    "by cuts, long and short": lambda g: (torch.randint(0, 90, (600,), generator=g).tolist() + [2777, 0, 1500], 4),
    "by cuts, alike": lambda g: ([100] * 530, 4),
    "by cuts, several sequences a group": lambda g: ([900] + torch.randint(0, 20, (2200,), generator=g).tolist(), 1),
    "nothing": lambda g: ([0] * 50, 2),
    "one among many empty": lambda g: ([0] * 1200 + [555] + [0] * 30, 1),
}


@pytest.mark.parametrize("heads,D,qdt,cdt", [(4, 128, BF16, BF16), (7, 128, BF16, FP8), (1, 64, F16, F16),
                                             (16, 64, BF16, FP8), (8, 256, F16, FP8), (11, 128, F16, F16),
                                             (2, 256, BF16, BF16), (9, 64, BF16, BF16), (16, 256, BF16, BF16),
                                             (12, 256, BF16, FP8), (10, 256, F16, F16), (13, 128, BF16, FP8)])
@pytest.mark.parametrize("how", list(SHARED_OUT))
def test_decode_attn_shared_out(cuda, how, heads, D, qdt, cdt):
    lens, Hk = SHARED_OUT[how](gen(len(how)))
    block = 16 if heads % 2 else 8
    x = attention_inputs(lens, heads * Hk, Hk, D, block, qdt, cdt, heads + D)
    check_attention(*x, cuda)


@pytest.mark.parametrize("cdt", [BF16, FP8])
def test_decode_attn_wide_table(cuda, cdt):
    """A block table far wider than the lengths: what is planned from it must not show in the result."""
    q, kc, vc, table, lens, ks, vs = attention_inputs([300, 20, 0, 1], 8, 2, 128, 16, BF16, cdt, 8)
    wide = torch.full((4, 70000), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    check_attention(q, kc, vc, wide, lens, ks, vs, cuda)


@pytest.mark.parametrize("cdt", [BF16, F16, FP8])
def test_decode_attn_token_major_pages_and_4d_query(cuda, cdt):
    qdt = F16 if cdt == F16 else BF16
    x = attention_inputs([130, 1, 0, 999], 28, 4, 128, 16, qdt, cdt, 3, token_major=True)
    check_attention(*x, cuda, q4=True)


@pytest.mark.parametrize("cdt,lens", [(BF16, [20011]), (FP8, [9000, 3, 0, 40001]), (F16, [1] * 300 + [5000])])
def test_decode_attn_long_and_many(cuda, cdt, lens):
    qdt = F16 if cdt == F16 else BF16
    x = attention_inputs(lens, 16, 4, 128, 16, qdt, cdt, 11)
    check_attention(*x, cuda)


@pytest.mark.parametrize("cdt", [BF16, F16, FP8, F32])
@pytest.mark.parametrize("block", [8, 16, 64])
def test_stale_values_do_not_count(cuda, cdt, block):
    """NaN and infinities in pages' unused rows, in pages of nobody, and table entries of no page."""
    qdt = {BF16: BF16, F16: F16, FP8: BF16, F32: F32}[cdt]
    q, kc, vc, table, lens, ks, vs = attention_inputs([3, 100, 31, 77], 8, 2, 64, block, qdt, cdt, 7)
    bad = torch.ones(kc.shape[0], block, dtype=torch.bool)
    for b, n in enumerate(lens.tolist()):
        for t in range(n):
            bad[int(table[b, t // block]), t % block] = False
    mask = bad[:, None, :, None].expand_as(kc)
    kc = kc.float().masked_fill(mask, float("nan")).to(cdt)
    vc = vc.float().masked_fill(mask, float("nan" if cdt == FP8 else "inf")).to(cdt)
    table[1, 1] = -7           # a page that is missing inside a sequence
    table[3, 0] = 1 << 30      # and one far outside the cache
    check_attention(q, kc, vc, table, lens, ks, vs, cuda)


def test_decode_attn_large_scores_and_lowest_values(cuda):
    """Scores of hundreds (weights under- and overflow without a running maximum), keys at the type's
    lowest value: their weights are zero, and a row of nothing else is an average."""
    q, kc, vc, table, lens, ks, vs = attention_inputs([200, 64, 16], 8, 2, 128, 16, BF16, BF16, 9)
    q = (q.float() * 12).bfloat16()
    check_attention(q, kc, vc, table, lens, ks, vs, cuda)
    q = torch.ones_like(q)
    low = torch.finfo(BF16).min
    kc[int(table[0, 2])] = low / 256  # one page far below the others
    kc[int(table[2, 0])] = low / 256  # the whole of sequence 2: equal scores
    got = paged.paged_decode_attn(q.to(cuda), kc.to(cuda), vc.to(cuda), table.to(cuda), lens.to(cuda), 128 ** -0.5).cpu()
    want = plain.decode_attn(q, kc, vc, table, lens, 128 ** -0.5)[0]
    assert torch.isfinite(got).all() and ((got.double() - want).abs() <= 2.0 ** -6).all()


def test_lengths_beyond_the_table(cuda):
    q, kc, vc, table, lens, ks, vs = attention_inputs([48, 20], 8, 2, 128, 16, BF16, BF16, 2)
    table = table[:, :2]
    check_attention(q, kc, vc, table, torch.tensor([2 ** 31 - 1, -5], dtype=torch.int32), ks, vs, cuda)


def test_decode_attn_past_32_bit_offsets(cuda):
    """A cache of more than 2^32 bytes (and 2^31 elements): pages at its far end."""
    nb, Hk, block, D = 140000, 1, 128, 128
    kc = torch.zeros(nb, Hk, block, D, dtype=BF16, device=cuda)
    vc = torch.zeros_like(kc)
    g = gen(1)
    far = [nb - 1, nb - 7, nb // 2 + 1]
    for p in far:
        kc[p], vc[p] = (torch.randn(Hk, block, D, generator=g).bfloat16().to(cuda) for _ in "kv")
    table = torch.tensor([far], dtype=torch.int32)
    q = torch.randn(1, 8, D, generator=g).bfloat16()
    got = paged.paged_decode_attn(q.to(cuda), kc, vc, table.to(cuda), torch.tensor([300], device=cuda), D ** -0.5).cpu()
    small = torch.tensor([[0, 1, 2]], dtype=torch.int32)
    want = plain.decode_attn(q, kc[far].cpu(), vc[far].cpu(), small, torch.tensor([300]), D ** -0.5)
    tol = (UNIT[BF16] + 2.0 ** -14) * want[2] + UNIT[BF16] * want[0].abs() * 1.01
    assert ((got.double() - want[0]).abs() <= tol).all()
    # the append reaches there as well
    k, v = (torch.randn(1, Hk, D, generator=g).bfloat16().to(cuda) for _ in "kv")
    paged.paged_append(k, v, kc, vc, table.to(cuda), torch.tensor([301], device=cuda))
    assert torch.equal(kc[far[2], 0, 300 % block], k[0, 0]) and torch.equal(vc[far[2], 0, 300 % block], v[0, 0])


# -------------------------------------------------------------------------------------- choice
SELECT = [
    # q heads, kv heads, D, block, budget, sink, recent, cache
    (28, 4, 128, 16, 8, 0, 1, BF16), (32, 8, 128, 16, 20, 1, 4, BF16), (12, 12, 64, 32, 5, 1, 1, F16),
    (8, 1, 256, 16, 200, 2, 2, FP8), (16, 2, 64, 8, 3, 0, 0, FP8), (6, 3, 40, 5, 7, 3, 4, F32),
    (40, 2, 128, 16, 33, 1, 2, BF16),
]


@pytest.mark.parametrize("Hq,Hk,D,block,budget,sink,recent,cdt", SELECT)
def test_select_and_sparse(cuda, Hq, Hk, D, block, budget, sink, recent, cdt):
    qdt = {BF16: BF16, F16: F16, FP8: BF16, F32: F32}[cdt]
    lens = [0, 1, block * 3 + 1, block * 40, block * 61 + 2]
    q, kc, vc, table, clen, ks, vs = attention_inputs(lens, Hq, Hk, D, block, qdt, cdt, Hq + budget)
    # equal pages: the lower one is to be taken; a query of zeros: every score is zero
    for j in (5, 9, 21):
        kc[int(table[3, j])] = kc[int(table[3, 2])]
    q[4, :Hq // Hk] = 0
    gk = kc.to(cuda)
    code, scale = paged.new_block_summary(gk)
    paged.paged_block_summary(gk, table.to(cuda), clen.to(cuda), code, scale, k_scale=ks)
    out, got = paged.paged_sparse_decode_attn(q.to(cuda), gk, vc.to(cuda), code, scale, table.to(cuda), clen.to(cuda),
                                              budget, D ** -0.5, sink_blocks=sink, recent_blocks=recent, k_scale=ks,
                                              v_scale=vs, return_selected=True)
    want = plain.select(q, code.cpu(), scale.cpu(), table, clen, budget, block, sink, recent)
    assert torch.equal(got.cpu(), want)
    check_attention(q, kc, vc, table, clen, ks, vs, cuda, selected=want)
    direct = paged.paged_decode_attn(q.to(cuda), gk, vc.to(cuda), table.to(cuda), clen.to(cuda), D ** -0.5, k_scale=ks,
                                     v_scale=vs, selected=got)
    assert torch.equal(bits(out), bits(direct))


@pytest.mark.parametrize("lens,budget,spread", [
    ([70000, 16, 33000], 64, 3), ([5000] * 40, 17, 3), ([131072], 1, 3),
    ([150000], 3000, 1),        # past the pages that registers hold, the threshold among equal scores
    ([140000, 131072], 200, 10 ** 6), ([33000, 8192 * 16 + 1, 600 * 16], 513, 10 ** 6), ([2048 * 16 + 5], 2048, 2)])
def test_select_long(cuda, lens, budget, spread):
    """Many pages and few sequences, many sequences, a budget of one; summaries drawn directly, with
    many equal scores or (a large spread of the scales) hardly any."""
    g = gen(budget)
    Hq, Hk, D, block = 8, 2, 64, 16
    table, nb = table_for(lens, block, g)
    code = torch.randint(-4, 5, (nb, Hk, 2, D), generator=g).to(torch.int8)
    scale = torch.randint(1, spread + 1, (nb, Hk), generator=g).float()
    q = torch.randint(-2, 3, (len(lens), Hq, D), generator=g).bfloat16()
    clen = torch.tensor(lens, dtype=torch.int32)
    got = paged.paged_select_blocks(q.to(cuda), code.to(cuda), scale.to(cuda), table.to(cuda), clen.to(cuda), budget,
                                    block, recent_blocks=1).cpu()
    c127 = torch.tensor(127.0)
    for b in range(0, len(lens), 7):
        n = -(-lens[b] // block)
        at = table[b, :n].long()
        for h in range(Hk):
            x = q[b, 4 * h:4 * h + 4].float()
            top = x.abs().amax(1, keepdim=True)
            w = (x * (c127 / top)).round()
            whole = w.clamp(max=0) @ code[at, h, 0].float().T + w.clamp(min=0) @ code[at, h, 1].float().T
            score = (whole * (top / c127)).amax(0) * scale[at, h]
            score[n - 1:] = math.inf
            want = score.sort(stable=True, dim=0, descending=True)[1][:budget].sort()[0].int()
            assert torch.equal(got[b, h, :want.numel()], want) and (got[b, h, want.numel():] == -1).all()


def test_select_equal_scores_and_missing_pages(cuda):
    """All scores equal (the lowest pages), all zero, negative ones, and entries of no page, which come last."""
    Hq, Hk, D, block, n = 4, 1, 64, 16, 3000
    table = torch.arange(n, dtype=torch.int32)[None].clone()
    lens = torch.tensor([n * block], dtype=torch.int32)
    q = torch.ones(1, Hq, D).bfloat16()
    for value, scale in ((3, 1.0), (0, 0.0), (-5, 2.0)):
        code = torch.full((n, Hk, 2, D), value, dtype=torch.int8)
        s = torch.full((n, Hk), scale)
        got = paged.paged_select_blocks(q.to(cuda), code.to(cuda), s.to(cuda), table.to(cuda), lens.to(cuda), 100, block,
                                        sink_blocks=2, recent_blocks=3).cpu()
        assert torch.equal(got[0, 0], torch.tensor(list(range(97)) + [n - 3, n - 2, n - 1], dtype=torch.int32))
    table[0, 10:2990] = -1
    got = paged.paged_select_blocks(q.to(cuda), code.to(cuda), s.to(cuda), table.to(cuda), lens.to(cuda), 30, block,
                                    recent_blocks=1).cpu()
    assert torch.equal(got[0, 0], torch.tensor(list(range(20)) + list(range(2990, 3000)), dtype=torch.int32))


def test_selected_lists_of_the_caller(cuda):
    """Any order, repeats (counted once per occurrence), entries of no page."""
    q, kc, vc, table, lens, ks, vs = attention_inputs([100, 333, 5, 0], 16, 2, 128, 16, BF16, BF16, 4)
    sel = torch.tensor([[[6, 0, -1, 3, 3], [2, 50, -9, 1 << 30, 4]], [[20, 19, 18, 0, 7], [-1, -1, -1, -1, -1]],
                        [[0, 1, 2, 3, 4], [1, -1, 0, -1, 5]], [[0, 1, 2, 3, 4], [0, 0, 0, 0, 0]]], dtype=torch.int32)
    check_attention(q, kc, vc, table, lens, ks, vs, cuda, selected=sel)
    check_attention(q, kc, vc, table, lens, ks, vs, cuda, selected=sel[..., :0])


# ------------------------------------------------------------------------------ streams, graphs
def test_other_stream_and_graph_replay(cuda):
    """On a side stream, and captured once then replayed as the lengths grow (they are read on the device)."""
    q, kc, vc, table, lens, ks, vs = attention_inputs([40, 200], 28, 4, 128, 16, BF16, BF16, 6)
    gq, gk, gv, gt, gl = (t.to(cuda) for t in (q, kc, vc, table, lens))
    code, scale = paged.new_block_summary(gk)
    k, v = (torch.randn(2, 4, 128, device=cuda).bfloat16() for _ in "kv")
    cos, sin = (x.to(cuda) for x in angles(300, 128))

    def step():
        r = paged.paged_append(k, v, gk, gv, gt, gl, q=gq, cos=cos, sin=sin, summary=code, summary_scale=scale)
        return r, paged.paged_decode_attn(r, gk, gv, gt, gl, 128 ** -0.5), \
            paged.paged_sparse_decode_attn(r, gk, gv, code, scale, gt, gl, 3, 128 ** -0.5, return_selected=True)

    paged.paged_block_summary(gk, gt, gl, code, scale)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r, dense, (sparse, chosen) = step()
    for _ in range(3):
        gl += 1
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in (r, dense, sparse, chosen, gk, gv, code)]
        for a, b in zip(kept, [*step()[:2], *step()[2], gk, gv, code]):
            assert torch.equal(a, b)


def test_empty_batches(cuda):
    kc = torch.zeros(4, 2, 16, 64, dtype=BF16, device=cuda)
    table, lens = torch.zeros(0, 3, dtype=torch.int32, device=cuda), torch.zeros(0, dtype=torch.int32, device=cuda)
    q = torch.zeros(0, 8, 64, dtype=BF16, device=cuda)
    k = torch.zeros(0, 2, 64, dtype=BF16, device=cuda)
    code, scale = paged.new_block_summary(kc)
    assert paged.paged_append(k, k, kc, kc.clone(), table, lens, q=q, summary=code, summary_scale=scale).shape == q.shape
    paged.paged_block_summary(kc, table, lens, code, scale)
    out, sel = paged.paged_sparse_decode_attn(q, kc, kc, code, scale, table, lens, 2, 1.0, return_selected=True)
    assert out.shape == q.shape and sel.shape == (0, 2, 2)
    # a table without columns, a cache without pages: rows of nothing
    table, lens = torch.zeros(2, 0, dtype=torch.int32, device=cuda), torch.tensor([3, 0], dtype=torch.int32, device=cuda)
    q = torch.ones(2, 8, 64, dtype=BF16, device=cuda)
    assert (paged.paged_decode_attn(q, kc, kc, table, lens, 1.0) == 0).all()
    assert (paged.paged_decode_attn(q, kc[:0], kc[:0], torch.zeros_like(table).new_zeros(2, 1), lens, 1.0) == 0).all()
    out, sel = paged.paged_sparse_decode_attn(q, kc, kc, code, scale, table, lens, 2, 1.0, return_selected=True)
    assert (out == 0).all() and (sel == -1).all()


# ------------------------------------------------------------------------------------ refusals
def test_refusals(cuda):
    nb, Hq, Hk, D, block = 6, 8, 2, 64, 16
    kc = torch.zeros(nb, Hk, block, D, dtype=BF16, device=cuda)
    vc, f8 = kc.clone(), kc.to(FP8)
    table, lens = torch.zeros(2, 3, dtype=torch.int32, device=cuda), torch.ones(2, dtype=torch.int32, device=cuda)
    k, q = torch.zeros(2, Hk, D, dtype=BF16, device=cuda), torch.zeros(2, Hq, D, dtype=BF16, device=cuda)
    cos, sin = (x.to(cuda) for x in angles(64, D))
    code, scale = paged.new_block_summary(kc)
    bad = pytest.raises(ValueError)

    def append(k=k, v=k, kc=kc, vc=vc, table=table, lens=lens, **kw):
        with bad:
            paged.paged_append(k, v, kc, vc, table, lens, **kw)

    append(k=k.cpu())
    append(k=k[:1], v=k[:1])                                    # one token each without cu_seqlens
    append(v=k.half())
    append(k=k.to(FP8), v=k.to(FP8))
    append(k=k[..., :32], v=k[..., :32])
    append(k=k[:, :1], v=k[:, :1])
    append(kc=kc[0])
    append(vc=vc.half())
    append(vc=vc[:3])
    append(table=table[:1])
    append(q=q.half())
    append(q=q[:1])
    append(cos=cos)
    append(cos=cos, sin=sin[:5])
    append(cos=cos.half(), sin=sin.half())
    append(cos=torch.cat([cos, cos], 1), sin=torch.cat([sin, sin], 1))
    append(cu_seqlens=torch.zeros(2, dtype=torch.int32, device=cuda))
    append(k_scale=2.0)
    append(kc=f8, vc=f8.clone(), k_scale=0.0)
    append(kc=f8, vc=f8.clone(), v_scale=float("nan"))
    append(summary=code)
    append(summary=code[:1], summary_scale=scale)
    append(summary=code.float(), summary_scale=scale)

    def attn(q=q, kc=kc, vc=vc, table=table, lens=lens, **kw):
        with bad:
            paged.paged_decode_attn(q, kc, vc, table, lens, 1.0, **kw)

    attn(q=q.cpu())
    attn(q=q[:, :7])
    attn(q=q[..., :32])
    attn(q=q[:1])
    attn(q=q[0])
    attn(q=q.to(FP8))
    attn(q=q[:, :, None].expand(2, Hq, 2, D))
    attn(kc=kc[..., :32])
    attn(vc=f8)
    attn(kc=kc.to(torch.int8), vc=vc.to(torch.int8))
    attn(kc=torch.zeros(nb, Hk, block, 264, dtype=BF16, device=cuda), vc=torch.zeros(nb, Hk, block, 264, dtype=BF16, device=cuda),
         q=torch.zeros(2, Hq, 264, dtype=BF16, device=cuda))
    attn(lens=lens[:1])
    attn(table=table[0])
    attn(v_scale=0.5)
    attn(selected=torch.zeros(2, Hq, 3, dtype=torch.int32, device=cuda))

    def sparse(q=q, code=code, scale=scale, budget=2, **kw):
        with bad:
            paged.paged_sparse_decode_attn(q, kc, vc, code, scale, table, lens, budget, 1.0, **kw)

    sparse(budget=0)
    sparse(sink_blocks=2, recent_blocks=1)
    sparse(sink_blocks=-1)
    sparse(code=code[..., :32])
    sparse(code=code.to(torch.uint8))
    sparse(code=code.transpose(2, 3).contiguous().transpose(2, 3))
    sparse(scale=scale[:, :1])
    sparse(q=q[:, :3])
    with bad:
        paged.paged_block_summary(kc, table, lens, code, scale, k_scale=2.0)
    with bad:
        paged.paged_block_summary(kc, table, lens, code, scale[:2])
