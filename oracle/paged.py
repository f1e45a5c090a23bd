"""Plain restatement of the paged-cache operators, sequence by sequence, in 64 bits (the 8-bit
summaries and scores, which are defined in fp32, in fp32). No counterpart in the reference."""
import torch

FP8_MAX = 448.0


def places(context_lens, n_tokens, cu_seqlens=None):
    """(sequence, position) of every packed token; None for tokens past the last sequence."""
    lens = context_lens.tolist()
    cu = list(range(len(lens) + 1)) if cu_seqlens is None else cu_seqlens.tolist()
    out = [None] * n_tokens
    for b, n in enumerate(lens):
        for i, t in enumerate(range(cu[b], cu[b + 1])):
            out[t] = (b, n - (cu[b + 1] - cu[b]) + i)
    return out


def page_of(block_table, num_blocks, block, place):
    """Physical page and row of a (sequence, position), or None."""
    if place is None:
        return None
    b, pos = place
    if pos < 0 or pos >= block_table.shape[1] * block:
        return None
    p = int(block_table[b, pos // block])
    return (p, pos % block) if 0 <= p < num_blocks else None


def rotate(x, cos, sin, interleaved):
    """x [H, D] float64 rotated with one row of cos, sin [r/2]; and the sum of the magnitudes of the
    two products of each channel (for error bounds)."""
    half = cos.shape[-1]
    y, mag = x.clone(), torch.zeros_like(x)
    if interleaved:
        a, b = x[:, 0:2 * half:2], x[:, 1:2 * half:2]
        y[:, 0:2 * half:2], y[:, 1:2 * half:2] = a * cos - b * sin, b * cos + a * sin
        mag[:, 0:2 * half:2], mag[:, 1:2 * half:2] = (a * cos).abs() + (b * sin).abs(), (b * cos).abs() + (a * sin).abs()
    else:
        a, b = x[:, :half], x[:, half:2 * half]
        y[:, :half], y[:, half:2 * half] = a * cos - b * sin, b * cos + a * sin
        mag[:, :half], mag[:, half:2 * half] = (a * cos).abs() + (b * sin).abs(), (b * cos).abs() + (a * sin).abs()
    return y, mag


def append(k, v, q, cos, sin, interleaved, cu_seqlens, block_table, context_lens, num_blocks, block):
    """[(token, page, row, k row, v row, q row, magnitudes of k, of q)] of the tokens that have a place."""
    out = []
    for t, place in enumerate(places(context_lens, k.shape[0], cu_seqlens)):
        at = page_of(block_table, num_blocks, block, place)
        if at is None or (cos is not None and place[1] >= cos.shape[0]):
            continue
        rows = [x[t].double() if x is not None else None for x in (k, v, q)]
        mags = [torch.zeros_like(r) if r is not None else None for r in rows]
        if cos is not None:
            c, s = cos[place[1]].double(), sin[place[1]].double()
            for i in (0, 2):
                if rows[i] is not None:
                    rows[i], mags[i] = rotate(rows[i], c, s, interleaved)
        out.append((t, at[0], at[1], rows[0], rows[1], rows[2], mags[0], mags[2]))
    return out


def summary_of(keys):
    """keys f32 [n, D] of one page and head (scaled) -> (codes int8 [2, D], scale f32)."""
    nan = keys.isnan()
    both = torch.stack([keys.masked_fill(nan, float("inf")).amin(0), keys.masked_fill(nan, float("-inf")).amax(0)])
    both = both.masked_fill(nan.all(0), 0.0)
    top = both.abs().max().clamp(max=torch.finfo(torch.float32).max)
    s = top / torch.tensor(127.0)
    code = (both / s).round().clamp(-127, 127) if top > 0 else torch.zeros_like(both)
    return code.to(torch.int8), s


def length(context_lens, block_table, b, block):
    return max(0, min(int(context_lens[b]), block_table.shape[1] * block))


def select(q, summary, summary_scale, block_table, context_lens, budget, block, sink, recent):
    """q [B, Hq, D] -> int32 [B, Hk, budget]."""
    B, Hq, D = q.shape
    Hk, nb = summary.shape[1], summary.shape[0]
    G = Hq // Hk
    out = torch.full((B, Hk, budget), -1, dtype=torch.int32)
    c127 = torch.tensor(127.0)
    for b in range(B):
        n = -(-length(context_lens, block_table, b, block) // block)
        for h in range(Hk):
            scores = []
            for j in range(n):
                p = int(block_table[b, j])
                if not 0 <= p < nb:
                    scores.append(float("-inf"))
                    continue
                best = None
                for x in q[b, h * G:(h + 1) * G].float():
                    x = x.masked_fill(x.isnan(), 0.0)
                    top = x.abs().max().clamp(max=torch.finfo(torch.float32).max)
                    w = (x * (c127 / top)).round().clamp(-127, 127) if top > 0 else torch.zeros(D)
                    w = w.to(torch.int64)
                    lo, hi = summary[p, h, 0].to(torch.int64), summary[p, h, 1].to(torch.int64)
                    s = torch.maximum(w * lo, w * hi).sum().float() * (top / c127)
                    best = s if best is None else torch.maximum(best, s)
                scores.append(float(best * summary_scale[p, h]))
            forced = [j < sink or j >= n - recent for j in range(n)]
            rank = sorted(range(n), key=lambda j: (not forced[j], 0.0 if forced[j] else -scores[j], j))
            got = sorted(rank[:budget])
            out[b, h, :len(got)] = torch.tensor(got, dtype=torch.int32)
    return out


def decode_attn(q, k_cache, v_cache, block_table, context_lens, scaling, k_scale=1.0, v_scale=1.0, selected=None):
    """(out, lse, weight, reach) in float64: out [B, Hq, D]; lse [B, Hq]; weight [B, Hq, D] the sum of
    p |v| (the scale of errors in p); reach [B, Hq] the largest scaling * sum |q k| (the scale of errors
    in a score)."""
    B, Hq, D = q.shape
    nb, Hk, block, _ = k_cache.shape
    G = Hq // Hk
    out, weight = torch.zeros(B, Hq, D, dtype=torch.float64), torch.zeros(B, Hq, D, dtype=torch.float64)
    lse, reach = torch.full((B, Hq), float("-inf"), dtype=torch.float64), torch.zeros(B, Hq, dtype=torch.float64)
    for b in range(B):
        n = length(context_lens, block_table, b, block)
        for h in range(Hk):
            pages = range(-(-n // block)) if selected is None else selected[b, h].tolist()
            ks, vs = [], []
            for j in pages:
                live = min(block, n - j * block) if 0 <= j < block_table.shape[1] else 0
                p = int(block_table[b, j]) if live > 0 else -1
                if live > 0 and 0 <= p < nb:
                    ks.append(k_cache[p, h, :live].double())
                    vs.append(v_cache[p, h, :live].double())
            if not ks:
                continue
            k, v = torch.cat(ks) * k_scale, torch.cat(vs) * v_scale
            x = q[b, h * G:(h + 1) * G].double()
            s = x @ k.T * scaling
            top = s.amax(1, keepdim=True)
            e = (s - top).exp()
            l = e.sum(1, keepdim=True)
            rows = slice(h * G, (h + 1) * G)
            out[b, rows], weight[b, rows] = e @ v / l, e @ v.abs() / l
            lse[b, rows] = (top + l.log())[:, 0]
            reach[b, rows] = (x.abs() @ k.abs().T).amax(1) * abs(scaling)
    return out, lse, weight, reach
