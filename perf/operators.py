"""The paged key-value cache's operators as a serving loop calls them, for measurement.

Four operators over one cache of pages ([num_blocks, kv_heads, block, head_dim], with a block table
and the sequences' lengths): the append of new tokens with the position rotation on the way, the
8-bit summary of each page's keys, the attention of one new token over all pages, and the attention
over the pages that the summaries' scores select.

``run`` computes them in elementary torch operations in 32 bits, or through ``bytes_b200.paged``
where ``own`` is true.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "fp8": torch.float8_e4m3fn, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "fp8": 1, "f32": 4}
_FP8_MAX = 448.0


# ------------------------------------------------------------------------------------- the cases
def listed():
    """Head layouts, lengths and page sizes of the repository's own configurations (28 query heads over
    4 KV heads at 8K, 32K and 131072 tokens; 32 over 8 at 32K with 64 pages of 16), and generic ones."""
    gqa = dict(q_heads=28, kv_heads=4, head_dim=128, block=16)
    gqa8 = dict(q_heads=32, kv_heads=8, head_dim=128, block=16)
    return [
        # one user's decode step: a single new token, where only latency counts
        dict(name="append_step_one", op="append", batch=1, new_lo=1, new_hi=1, past_lo=4096, past_hi=4096,
             rotary=128, interleaved=False, cache="bf16", summary=False, **gqa),
        # a full batch's decode step into an 8-bit cache, sequences of all ages
        dict(name="append_step_batch_fp8", op="append", batch=128, new_lo=1, new_hi=1, past_lo=5, past_hi=1500,
             rotary=128, interleaved=False, cache="fp8", summary=False, **gqa8),
        # a batch of prompts of very different lengths, summaries kept for the sparse attention
        dict(name="append_prompts_summary", op="append", batch=11, new_lo=37, new_hi=6001, past_lo=0, past_hi=0,
             rotary=128, interleaved=False, cache="bf16", summary=True, **gqa8),
        # summaries of a few short sequences, rebuilt after their pages came from elsewhere
        dict(name="summary_short", op="summary", batch=3, len_lo=50, len_hi=700, cache="bf16", **gqa),
        # summaries of a whole batch at 32K
        dict(name="summary_32k", op="summary", batch=8, len_lo=30001, len_hi=32768, cache="bf16", **gqa),
        # one short conversation: latency
        dict(name="attn_one_short", op="attn", batch=1, len_lo=777, len_hi=777, cache="bf16", **gqa),
        # small multi-head model in f16, pages of 32, from a first token to a few thousand
        dict(name="attn_mha_f16", op="attn", batch=24, len_lo=1, len_hi=3001, cache="f16", q_heads=12, kv_heads=12,
             head_dim=64, block=32),
        # a serving batch: sequences from a page to 8K, no two alike
        dict(name="attn_ragged", op="attn", batch=64, len_lo=33, len_hi=8192, cache="bf16", **gqa8),
        # 32K contexts in an 8-bit cache with larger pages
        dict(name="attn_32k_fp8", op="attn", batch=8, len_lo=32768, len_hi=32768, cache="fp8", q_heads=28, kv_heads=4,
             head_dim=128, block=64),
        # the longest: eight sequences of 131072 tokens
        dict(name="attn_128k", op="attn", batch=8, len_lo=131072, len_hi=131072, cache="bf16", **gqa),
        # 16 sequences at 32K, 64 pages of 16 for each KV head
        dict(name="sparse_32k", op="sparse", batch=16, len_lo=32768, len_hi=32768, cache="bf16", budget=64, sink=1,
             recent=4, **gqa8),
        # one long document in an 8-bit cache: few rows, many pages
        dict(name="sparse_one_128k_fp8", op="sparse", batch=1, len_lo=131072, len_hi=131072, cache="fp8", budget=128,
             sink=1, recent=8, **gqa),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: any operator, type, head layout, page size and lengths of the listed ranges."""
    heads = rng.choice([(28, 4), (32, 8), (12, 12), (16, 2), (8, 1), (40, 8), (24, 24), (32, 2)])
    case = dict(op=rng.choice(["append", "append", "summary", "attn", "attn", "attn", "sparse", "sparse"]),
                q_heads=heads[0], kv_heads=heads[1], head_dim=rng.choice([64, 128, 128, 128, 256]),
                block=rng.choice([16, 16, 32, 64]), cache=rng.choice(["bf16", "bf16", "f16", "fp8"]))
    # at most as many values of one cache, or of new tokens, as the largest listed cases have
    most = 8 * 131072 * 4 * 128 // (case["kv_heads"] * case["head_dim"])
    most_new = 15000 * 48 * 128 // ((heads[0] + 2 * heads[1]) * case["head_dim"])
    if case["op"] == "append":
        step = rng.random() < 0.5
        case["batch"] = _log_int(rng, 1, 256 if step else 32)
        hi = 1 if step else _log_int(rng, 2, max(2, min(6000, most_new // case["batch"])))
        past = rng.choice([0, 1]) * _log_int(rng, 1, 2000)
        case.update(new_lo=1 if step else _log_int(rng, 1, hi), new_hi=hi, past_lo=min(past, _log_int(rng, 1, 2000)),
                    past_hi=past, interleaved=rng.random() < 0.3, summary=rng.random() < 0.5,
                    rotary=rng.choice([case["head_dim"], case["head_dim"], case["head_dim"] // 2]))
        return case
    sparse = case["op"] == "sparse"
    case["batch"] = _log_int(rng, 1, 16 if sparse else 128)
    hi = _log_int(rng, 500 if sparse else 1, max(600, min(131072, most // case["batch"] // (1 if case["op"] == "attn" else 4))))
    case.update(len_lo=max(1, hi if rng.random() < 0.3 else _log_int(rng, 1, hi)), len_hi=hi)
    if sparse:
        case.update(budget=_log_int(rng, 8, 256), sink=rng.choice([0, 1, 2]), recent=rng.choice([1, 2, 4]))
    return case


def _ladder(n, lo, hi):
    """n lengths from lo to hi, evenly spread over their logarithm (lo may be 0: then evenly)."""
    if n == 1:
        return [hi]
    if lo < 1:
        return [round(lo + (hi - lo) * i / (n - 1)) for i in range(n)]
    return [round(lo * (hi / lo) ** (i / (n - 1))) for i in range(n)]


def _lengths(c):
    """(new tokens, length after them) of each sequence."""
    n = c["batch"]
    if c["op"] == "append":
        new = _ladder(n, c["new_lo"], c["new_hi"])
        return new, [a + b for a, b in zip(new, _ladder(n, c["past_lo"], c["past_hi"]))]
    return [0] * n, _ladder(n, c["len_lo"], c["len_hi"])


def _act(c):
    return "f16" if c["cache"] == "f16" else "bf16"


def work(c):
    new, full = _lengths(c)
    D, Hq, Hk, bs, cb = c["head_dim"], c["q_heads"], c["kv_heads"], c["block"], _SIZE[c["cache"]]
    B, T = len(full), sum(new)
    blocks = [-(-n // bs) for n in full]
    per_summary = Hk * (2 * D + 4)
    if c["op"] == "append":
        ab = _SIZE[_act(c)]
        bytes_ = T * D * ab * (2 * Hq + 2 * Hk) + T * 2 * Hk * D * cb
        bytes_ += (max(full) - min(f - n for f, n in zip(full, new))) * c["rotary"] * 4
        flops = 3 * T * (Hq + Hk) * c["rotary"]
        touched = [-(-f // bs) - (f - n) // bs for f, n in zip(full, new)]
        bytes_ += 4 * (2 * B + sum(touched))
        if c["summary"]:
            bytes_ += sum((f - n) % bs for f, n in zip(full, new)) * Hk * D * cb + sum(touched) * per_summary
            flops += 2 * T * Hk * D
    elif c["op"] == "summary":
        bytes_ = sum(full) * Hk * D * cb + sum(blocks) * (per_summary + 4) + 4 * B
        flops = 2 * sum(full) * Hk * D
    else:
        seen = sum(full)
        bytes_ = 2 * B * Hq * D * _SIZE[_act(c)] + 4 * B + 4 * sum(blocks)
        flops = 0
        if c["op"] == "sparse":
            picked = [min(n, c["budget"]) for n in blocks]
            # the last page is always among the chosen, and may be partly filled
            seen = sum(p * bs - (n * bs - f) for p, n, f in zip(picked, blocks, full))
            bytes_ += sum(blocks) * per_summary + 4 * B * Hk * c["budget"]
            flops += 4 * sum(blocks) * Hq * D
        bytes_ += 2 * seen * Hk * D * cb
        flops += 4 * seen * Hq * D
    return {"bytes": bytes_, "flops": flops}


# ------------------------------------------------------------------------------------ the inputs
def _values(shape, g, outliers):
    """N(0,1); keys have 4 of 128 channels eight times as large, as real keys do."""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)
    if outliers:
        at = torch.randperm(shape[-1], generator=g, device="cuda")[:max(1, shape[-1] // 32)]
        x[..., at] *= 8
    return x


def _store(x, dtype, inv):
    """x as the cache's type holds it (8-bit: over its scale, within the type's range)."""
    if dtype == torch.float8_e4m3fn:
        x = (x.float() * inv).clamp(-_FP8_MAX, _FP8_MAX)
    return x.to(dtype)


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    new, full = _lengths(c)
    order = torch.randperm(len(full), generator=g, device="cuda").tolist()
    new, full = [new[i] for i in order], [full[i] for i in order]
    B, Hq, Hk, D, bs = len(full), c["q_heads"], c["kv_heads"], c["head_dim"], c["block"]
    act, cache = _TYPES[_act(c)], _TYPES[c["cache"]]
    fp8 = c["cache"] == "fp8"
    s = {"op": c["op"], "k_scale": 0.125 if fp8 else 1.0, "v_scale": 0.0156 if fp8 else 1.0, "new": new,
         "most_new": max(new), "scaling": D ** -0.5}
    lens = torch.tensor(full, device="cuda", dtype=torch.int32)
    counts = (lens + bs - 1) // bs
    wide, total = -(-max(full) // bs), int(counts.sum())
    pool = total + 3
    table = torch.zeros(B, wide, device="cuda", dtype=torch.int32)
    used = torch.arange(wide, device="cuda")[None] < counts[:, None]
    table[used] = torch.randperm(pool, generator=g, device="cuda")[:total].int()
    s.update(lens=lens, table=table)
    k = _values((pool, Hk, bs, D), g, True)
    s["k_cache"] = _store(k, cache, 1 / s["k_scale"])
    del k
    if c["op"] != "summary":
        s["v_cache"] = _store(_values((pool, Hk, bs, D), g, False), cache, 1 / s["v_scale"])
    if c["op"] == "append":
        T = sum(new)
        # the projection's output, one row a token: queries, keys and values side by side
        qkv = _values((T, (Hq + 2 * Hk) * D), g, False).to(act)
        s["q"] = qkv[:, :Hq * D].unflatten(1, (Hq, D))
        s["k"] = qkv[:, Hq * D:(Hq + Hk) * D].unflatten(1, (Hk, D))
        s["v"] = qkv[:, (Hq + Hk) * D:].unflatten(1, (Hk, D))
        r = c["rotary"]
        angle = torch.arange(max(full), device="cuda").double()[:, None] * 10000.0 ** (
            -torch.arange(0, r, 2, device="cuda").double() / r)
        s.update(cos=angle.cos().float(), sin=angle.sin().float(), interleaved=c["interleaved"], cu=None)
        if max(new) > 1 or c["new_hi"] > 1:
            s["cu"] = torch.tensor([0] + new, device="cuda").cumsum(0).int()
    else:
        s["q"] = _values((B, Hq, 1, D), g, False).to(act)
    if c["op"] == "summary" or c.get("summary"):
        s["summary"] = torch.zeros(pool, Hk, 2, D, device="cuda", dtype=torch.int8)
        s["summary_scale"] = torch.zeros(pool, Hk, device="cuda")
    elif c["op"] == "sparse":
        x = s["k_cache"].float() * s["k_scale"]
        ends = torch.full((pool,), bs, device="cuda")
        ends[table[torch.arange(B, device="cuda"), (counts - 1).long()].long()] = (lens - (counts - 1) * bs).long()
        dead = (torch.arange(bs, device="cuda")[None] >= ends[:, None])[:, None, :, None]
        lo, hi = x.masked_fill(dead, math.inf).amin(2), x.masked_fill(dead, -math.inf).amax(2)
        s["summary"], s["summary_scale"] = _codes(lo, hi)
        s.update(budget=c["budget"], sink=c["sink"], recent=c["recent"])
    return s


# ------------------------------------------------------------------------------- the plain forms
def _codes(lo, hi):
    """8-bit codes [.., 2, D] and scale [..] of channelwise minima and maxima [.., D]."""
    both = torch.stack([lo, hi], -2)
    top = both.abs().amax((-1, -2))
    scale = top / torch.full_like(top, 127.0)
    code = torch.where(top[..., None, None] > 0, both / scale[..., None, None], torch.zeros_like(both))
    return code.round().clamp(-127, 127).to(torch.int8), scale


def _rotate(x, cos, sin, interleaved):
    """x [T, H, D] in 32 bits, its first 2 * cos.shape[-1] channels rotated by pairs."""
    half = cos.shape[-1]
    cos, sin = cos[:, None], sin[:, None]
    y = x.float().clone()
    if interleaved:
        a, b = x[..., 0:2 * half:2].float(), x[..., 1:2 * half:2].float()
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :half].float(), x[..., half:2 * half].float()
        y[..., :half], y[..., half:2 * half] = a * cos - b * sin, b * cos + a * sin
    return y


def _summarise(s, start, most):
    """The summaries of the pages from token `start` on, `most` pages at most for a sequence."""
    bs, lens, table = s["k_cache"].shape[2], s["lens"].long(), s["table"].long()
    page = torch.minimum(start[:, None] // bs + torch.arange(most, device=lens.device), (lens[:, None] - 1) // bs)
    at = table.gather(1, page)
    x = s["k_cache"][at].float() * s["k_scale"]  # [B, most, Hk, bs, D]
    dead = page[..., None] * bs + torch.arange(bs, device=lens.device) >= lens[:, None, None]
    dead = dead[:, :, None, :, None]
    code, scale = _codes(x.masked_fill(dead, math.inf).amin(3), x.masked_fill(dead, -math.inf).amax(3))
    s["summary"][at] = code
    s["summary_scale"][at] = scale


def _attend(s, table, live):
    """Attention of q over the pages of table [B, Hk, n], of which the tokens live [B, Hk, n * bs] count."""
    q, Hk = s["q"][:, :, 0].float(), s["k_cache"].shape[1]
    B, Hq, D = q.shape
    head = torch.arange(Hk, device=q.device)[None, :, None]
    k = s["k_cache"][table, head].flatten(2, 3).float()  # [B, Hk, n * bs, D]
    score = q.view(B, Hk, Hq // Hk, D) @ k.transpose(2, 3) * (s["scaling"] * s["k_scale"])
    del k
    score = score.masked_fill(~live[:, :, None], -math.inf)
    p = (score - score.amax(-1, keepdim=True)).exp()
    v = s["v_cache"][table, head].flatten(2, 3).float()
    out = p @ v / p.sum(-1, keepdim=True) * s["v_scale"]
    return out.reshape(B, Hq, 1, D).to(s["q"].dtype)


def _plain_append(s):
    bs, T = s["k_cache"].shape[2], s["q"].shape[0]
    lens, t = s["lens"].long(), torch.arange(T, device=s["q"].device)
    if s["cu"] is None:
        seq, at = t, lens - 1
    else:
        cu = s["cu"].long()
        seq = torch.searchsorted(cu, t, right=True) - 1
        at = lens[seq] - cu[seq + 1] + t
    cos, sin = s["cos"][at], s["sin"][at]
    page, row = s["table"][seq, at // bs].long(), at % bs
    k = _rotate(s["k"], cos, sin, s["interleaved"])
    s["k_cache"][page, :, row] = _store(k, s["k_cache"].dtype, 1 / s["k_scale"])
    s["v_cache"][page, :, row] = _store(s["v"].float(), s["v_cache"].dtype, 1 / s["v_scale"])
    q = _rotate(s["q"], cos, sin, s["interleaved"]).to(s["q"].dtype)
    if "summary" in s:
        n = torch.ones_like(lens) if s["cu"] is None else s["cu"].long().diff()
        _summarise(s, lens - n, (s["most_new"] - 1) // bs + 2)
    return q


def _plain_sparse(s):
    q, (B, wide) = s["q"][:, :, 0].float(), s["table"].shape
    bs, Hk, D = s["k_cache"].shape[2], s["k_cache"].shape[1], q.shape[-1]
    top = q.abs().amax(-1, keepdim=True)
    full = torch.full_like(top, 127.0)
    q8 = torch.where(top > 0, (q * (full / top)).round(), torch.zeros_like(q)).view(B, Hk, -1, D)
    q_scale = (top / full).view(B, Hk, -1, 1)
    at = s["table"].long()
    both = s["summary"][at].float().permute(0, 2, 3, 4, 1)  # [B, Hk, 2, D, wide]
    whole = q8.clamp(max=0) @ both[:, :, 0] + q8.clamp(min=0) @ both[:, :, 1]
    score = (whole * q_scale).amax(2) * s["summary_scale"][at].transpose(1, 2)  # [B, Hk, wide]
    block, used = torch.arange(wide, device=q.device), (s["lens"].long() + bs - 1)[:, None] // bs
    forced = (block < s["sink"]) | (block >= used - s["recent"])
    score = torch.where(forced[:, None], torch.full_like(score, math.inf), score)
    score = torch.where((block < used)[:, None], score, torch.full_like(score, -math.inf))
    n = min(s["budget"], wide)
    got = score.sort(stable=True, dim=-1, descending=True)[1][..., :n].sort(-1)[0]  # [B, Hk, n]
    # sequences with fewer pages than the budget: those pages, then none
    got = torch.where(got < used[..., None], got, torch.full_like(got, -1))
    pos = got.clamp(min=0)[..., None] * bs + torch.arange(bs, device=q.device)
    live = (got >= 0)[..., None] & (pos < s["lens"].long()[:, None, None, None])
    table = at[:, None].expand(B, Hk, wide).gather(2, got.clamp(min=0))
    out = _attend(s, table, live.flatten(2))
    chosen = torch.full((B, Hk, s["budget"]), -1, device=q.device, dtype=torch.int32)
    chosen[..., :n] = got.int()
    return out, chosen


def _values_of(s):
    """The summaries as the values that they stand for."""
    return s["summary"] * s["summary_scale"][..., None, None]


def run(s):
    if own:
        from bytes_b200 import paged
    if s["op"] == "append":
        if own:
            q = paged.paged_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["lens"], q=s["q"],
                                   cos=s["cos"], sin=s["sin"], interleaved=s["interleaved"], cu_seqlens=s["cu"],
                                   k_scale=s["k_scale"], v_scale=s["v_scale"], summary=s.get("summary"),
                                   summary_scale=s.get("summary_scale"))
        else:
            q = _plain_append(s)
        got = {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
        if "summary" in s:
            got["summary"] = _values_of(s)
        return got
    if s["op"] == "summary":
        if own:
            paged.paged_block_summary(s["k_cache"], s["table"], s["lens"], s["summary"], s["summary_scale"],
                                      k_scale=s["k_scale"])
        else:
            _summarise(s, torch.zeros_like(s["lens"]).long(), s["table"].shape[1])
        return {"summary": _values_of(s)}
    if s["op"] == "attn":
        if own:
            return paged.paged_decode_attn(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["scaling"],
                                           k_scale=s["k_scale"], v_scale=s["v_scale"])
        B, Hk, bs = s["lens"].numel(), s["k_cache"].shape[1], s["k_cache"].shape[2]
        live = torch.arange(s["table"].shape[1] * bs, device=s["q"].device) < s["lens"][:, None, None]
        return _attend(s, s["table"].long()[:, None].expand(B, Hk, -1), live.expand(B, Hk, -1))
    if own:
        return paged.paged_sparse_decode_attn(s["q"], s["k_cache"], s["v_cache"], s["summary"], s["summary_scale"],
                                              s["table"], s["lens"], s["budget"], s["scaling"], sink_blocks=s["sink"],
                                              recent_blocks=s["recent"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                                              return_selected=True)
    return _plain_sparse(s)


# --------------------------------------------------------------------------------- in 64 bits
def _exact_attention(s, pages):
    """Sequence by sequence and head by head; pages(b, h) gives the sequence's page numbers."""
    q, kc, vc = s["q"], s["k_cache"], s["v_cache"]
    B, Hq, _, D = q.shape
    Hk, bs = kc.shape[1], kc.shape[2]
    G, out = Hq // Hk, torch.zeros(B, Hq, 1, D, dtype=torch.float64, device=q.device)
    lens = s["lens"].tolist()
    for b in range(B):
        for h in range(Hk):
            logical = pages(b, h)
            at = s["table"][b].long()[logical]
            n = logical.numel() * bs
            if int(logical[-1]) == (lens[b] - 1) // bs:
                n -= (int(logical[-1]) + 1) * bs - lens[b]
            k = kc[at, h].reshape(-1, D)[:n].double() * s["k_scale"]
            v = vc[at, h].reshape(-1, D)[:n].double() * s["v_scale"]
            w = torch.softmax(torch.einsum("gd,td->gt", q[b, h * G:(h + 1) * G, 0].double(), k) * s["scaling"], 1)
            out[b, h * G:(h + 1) * G, 0] = torch.einsum("gt,td->gd", w, v)
    return out


def _exact_choice(s, b, h, lens):
    """The chosen pages. Rounding to 8 bits, and the two products with a scale, are by the definition in
    32 bits; the sum over channels is a whole number."""
    Hk, bs = s["k_cache"].shape[1], s["k_cache"].shape[2]
    G, n = s["q"].shape[1] // Hk, -(-lens[b] // bs)
    at = s["table"][b, :n].long()
    lo, hi = s["summary"][at, h, 0].long(), s["summary"][at, h, 1].long()
    best = None
    for x in s["q"][b, h * G:(h + 1) * G, 0].float():
        top = x.abs().max()
        if top > 0:
            whole = torch.round(x * (top.new_tensor(127.0) / top)).long()
            value = torch.maximum(whole * lo, whole * hi).sum(1).float() * (top / top.new_tensor(127.0))
        else:
            value = torch.zeros(n, device=x.device)
        best = value if best is None else torch.maximum(best, value)
    score = (best * s["summary_scale"][at, h]).tolist()
    forced = set(range(min(n, s["sink"]))) | set(range(max(0, n - s["recent"]), n))
    ranked = sorted(range(n), key=lambda j: (j not in forced, -score[j] if j not in forced else 0, j))
    return torch.tensor(sorted(ranked[:s["budget"]]), device=s["q"].device)


def exact(c, seed):
    s = prepare(c, seed)
    lens, bs = s["lens"].tolist(), c["block"]
    every = torch.arange(s["table"].shape[1], device="cuda")
    if c["op"] == "attn":
        return _exact_attention(s, lambda b, h: every[:-(-lens[b] // bs)])
    if c["op"] == "sparse":
        return _exact_attention(s, lambda b, h: _exact_choice(s, b, h, lens)), None
    first = [0] * len(lens)
    got = {}
    stored = s["k_cache"].double()
    if c["op"] == "append":
        first = [n - m for n, m in zip(lens, s["new"])]
        r, T = c["rotary"], s["q"].shape[0]
        seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), torch.tensor(s["new"], device="cuda"))
        at = torch.cat([torch.arange(a, n, device="cuda") for a, n in zip(first, lens)])
        turn = torch.complex(s["cos"].double(), s["sin"].double())[at][:, None]

        def rotated(x):
            x = x.double()
            pairs = x[..., :r].unflatten(-1, (r // 2, 2) if c["interleaved"] else (2, r // 2))
            if not c["interleaved"]:
                pairs = pairs.transpose(-1, -2)
            pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            if not c["interleaved"]:
                pairs = pairs.transpose(-1, -2)
            return torch.cat([pairs.flatten(-2), x[..., r:]], -1)

        def held(x, scale):
            return (x / scale).clamp(-_FP8_MAX, _FP8_MAX) if c["cache"] == "fp8" else x

        slot = s["table"][seq, at // bs].long() * bs + at % bs
        values = s["v_cache"].double()
        for pages, x in ((stored, held(rotated(s["k"]), s["k_scale"])), (values, held(s["v"].double(), s["v_scale"]))):
            flat = pages.transpose(1, 2).reshape(-1, pages.shape[1], pages.shape[3])
            flat[slot] = x
            pages.copy_(flat.unflatten(0, (-1, bs)).transpose(1, 2))
        got.update(q=rotated(s["q"]), k_cache=stored, v_cache=values)
        if not c["summary"]:
            return got
    seen = torch.zeros(s["summary"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        j = every[first[b] // bs:-(-n // bs)]
        at = s["table"][b].long()[j]
        for part, whole in ((at[:-1], True), (at[-1:], False)):
            x = stored[part] * s["k_scale"]
            if not whole:
                x = x[:, :, :n - int(j[-1]) * bs]
            if part.numel():
                seen[part] = torch.stack([x.amin(2), x.amax(2)], 2)
    got["summary"] = seen
    return got
