"""Definitions in 64 bits of what single requests ask of a batch (adapters, changes of logits,
log-probabilities), with bounds on how far 32-bit sums and one rounding of the output may be from them."""
import math

import torch

D = torch.float64
STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}   # one rounding, relative to the value
F = 2.0 ** -24


def adapters(x, a, b, scale, ranks, widths, row_adapter, base):
    """(out in 64 bits, the most that a right kernel may be off by). One rounding of the output; a sum of n products in
    32 bits is off by at most n 2^-24 of the sum of their sizes; 16-bit rows keep 16 bits of h (two numbers of 8 bits
    each), and their products are exact in 32 bits."""
    out, room = base.to(D).clone(), F * base.to(D).abs()
    r, k = b.shape[2], x.shape[1]
    for t, g in enumerate(row_adapter.tolist()):
        if not 0 <= g < a.shape[0]:
            room[t] = 0   # (the row itself)
            continue
        rank, s, at = min(max(int(ranks[g]), 0), r), abs(float(scale[g])), 0
        if rank == 0:
            continue
        for i, w in enumerate(widths):
            A, B = a[g, i * r:i * r + rank].to(D), b[g, at:at + w, :rank].to(D)
            h, sizes = A @ x[t].to(D), A.abs() @ x[t].to(D).abs()
            out[t, at:at + w] += scale[g].to(D) * (B @ h)
            off_h = (k + 16) * F * sizes + (2.0 ** -16 * h.abs() if x.dtype == torch.bfloat16 else 0)
            room[t, at:at + w] += s * (B.abs() @ (off_h + (2 * rank + 8) * F * (h.abs() + off_h)))
            at += w
    live = torch.tensor([0 <= g < a.shape[0] for g in row_adapter.tolist()])[:, None].to(out.device)
    return out, torch.where(live, room * (1 + 2.0 ** -7) + STEP[x.dtype] * out.abs(), torch.zeros_like(room))


def adjusted(logits, repetition=None, presence=None, frequency=None, histories=None, biases=None, masks=None, mask_rows=None):
    """(rows in 64 bits, the most that a right kernel may be off by). histories: per row a list of (token, count,
    generated); biases: per row a list of (token, value); masks: lists of truth values. Six roundings of sums no larger than
    the sum of their parts."""
    v, size = logits.to(D).cpu().clone(), logits.to(D).cpu().abs().clone()
    rows, vocab = v.shape
    for r in range(rows):
        counts = {}
        for token, c, g in (histories or [[]] * rows)[r]:
            old = counts.get(token, (0, 0))
            counts[token] = (old[0] + c, old[1] + g)
        for token, (c, g) in counts.items():
            if not 0 <= token < vocab or (c, g) == (0, 0):
                continue
            x = float(v[r, token])
            p = float(repetition[r]) if repetition is not None else 1.0
            if p != 1.0 and x != 0 and not math.isinf(x) and c:
                try:
                    power = p ** c
                except OverflowError:
                    power = math.inf
                x = (x / power if power else math.inf) if x > 0 else x * power
                if abs(x) > torch.finfo(torch.float32).max:   # (no 32-bit number: infinite)
                    x = math.copysign(math.inf, x)
            size[r, token] = max(abs(x), 2.0 ** -126)
            if g:
                f = float(frequency[r]) if frequency is not None else 0.0
                q = float(presence[r]) if presence is not None else 0.0
                x = x - f * g - q
                size[r, token] += abs(f * g) + abs(q)
            v[r, token] = x
        for token, b in dict((biases or [[]] * rows)[r]).items():
            if 0 <= token < vocab:
                v[r, token] += b
                size[r, token] += abs(b) if math.isfinite(b) else 0
        if masks is not None and 0 <= int(mask_rows[r]) < len(masks):
            v[r, ~torch.tensor(masks[int(mask_rows[r])], dtype=torch.bool)] = -math.inf
    return v, 6 * F * size


def logprobs(logits, tokens, top):
    """(log-probabilities of the tokens, tokens before them, the best tokens, theirs) in 64 bits, and the two
    bounds: roundings of the difference to the maximum, of the logarithm and of the result; the sum of exponentials
    is off by a step of each argument (weighted by its share), two of the exponential and 64 of its additions."""
    x = logits.to(D).cpu()
    rows, vocab = x.shape
    m = x.max(dim=1, keepdim=True).values
    shares = torch.softmax(x, dim=1)
    d = torch.where(shares > 0, (x - m).abs(), torch.zeros_like(x))
    log_sum = torch.log(torch.exp(x - m).sum(dim=1, keepdim=True))
    logp = x - m - log_sum
    of_sum = 2 * F * (shares * d).sum(dim=1, keepdim=True) + (8 + 64) * F + 2 * F * log_sum.abs()
    room = of_sum + F * (torch.nan_to_num(x - m, neginf=0).abs() + torch.nan_to_num(logp, neginf=0).abs())
    t = tokens.long().cpu()[:, None]
    at = torch.arange(vocab)
    mine = x.gather(1, t)
    before = ((x > mine) | ((x == mine) & (at < t))).sum(dim=1)
    best = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
    return (logp.gather(1, t)[:, 0], before, best, logp.gather(1, best)), (room.gather(1, t)[:, 0], room.gather(1, best))


def pack(allowed):
    """Truth values of tokens as 32-bit words, bit t % 32 of word t // 32."""
    words = [0] * (-(-len(allowed) // 32))
    for t, a in enumerate(allowed):
        if a:
            words[t // 32] |= 1 << (t % 32)
    return [w - (1 << 32) if w >> 31 else w for w in words]


def lists(rows):
    """Lists of tuples, one a row, as offsets and flat columns."""
    offsets = [0]
    for r in rows:
        offsets.append(offsets[-1] + len(r))
    flat = [e for r in rows for e in r]
    return offsets, [list(c) for c in zip(*flat)]


def close(got, want, room):
    """Within the bound; where the definition is not finite, the same."""
    got, want, room = got.to(D).cpu(), want.to(D).cpu(), room.to(D).cpu()
    fine = torch.isfinite(want)
    same = torch.where(fine, torch.zeros_like(want, dtype=torch.bool), (got == want) | (got.isnan() & want.isnan()))
    off = torch.where(fine, (got - want).abs(), torch.zeros_like(want))
    off = torch.where(torch.isnan(off), torch.full_like(off, math.inf), off)
    bad = torch.where(fine, off > room, ~same)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} are off, first at {bad.nonzero()[0].tolist()}: "
                           f"{got[bad][0]:.9g} for {want[bad][0]:.9g}, room {room[bad][0]:.3g}")
