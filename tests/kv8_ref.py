"""Plain 64-bit references of the operators over an 8-bit cache and of the test
of drafted tokens, on the CPU."""

import math

import numpy as np
import torch

BLOCK = 16
E4M3 = torch.float8_e4m3fn

# The e4m3 magnitudes in order (code 127 is NaN).
VALUES = torch.arange(127, dtype=torch.uint8).view(E4M3).double()


def nearest_code(x):
    """Codes (uint8) of the nearest e4m3 values of x (f64), ties to the even code."""
    between = (VALUES[1:] + VALUES[:-1]) / 2
    at = torch.bucketize(x.abs(), between)  # between[at - 1] < |x| <= between[at]
    tie = (at < 126) & (x.abs() == between[at.clamp(max=125)])
    at = torch.where(tie, at + at % 2, at)
    code = at.to(torch.uint8) | torch.where(torch.signbit(x), 128, 0).to(torch.uint8)
    return torch.where(torch.isfinite(x), code, torch.tensor(127, dtype=torch.uint8))


def scale_for(top):
    """The smallest power of two, 2^-64 at least, whose 448-fold reaches top."""
    e = -64
    while top > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def decode(codes):
    return codes.view(E4M3).double()


def append(codes, scales, slots, x):
    """Cells `slots` (-1: skipped) of one pool become x [tokens, kv_heads, D]
    (f64). codes uint8 [pages, kv_heads, page_tokens, D], scales f32; in place."""
    pages, kvh, pt, D = codes.shape
    blocks = {}
    for t, s in enumerate(slots):
        if 0 <= s < pages * pt:
            blocks.setdefault(s // BLOCK, []).append((s % BLOCK, t))
    for block, cells in blocks.items():
        page, part = block // (pt // BLOCK), block % (pt // BLOCK)
        first = min(c for c, _ in cells)
        for h in range(kvh):
            new = torch.stack([x[t, h] for _, t in cells])
            finite = new[torch.isfinite(new)].abs()
            need = scale_for(float(finite.max()) if finite.numel() else 0.0)
            old = float(scales[page, h, part])
            scale = max(old, need) if first > 0 else need
            if first > 0 and scale != old:
                held = decode(codes[page, h, part * BLOCK:part * BLOCK + first])
                codes[page, h, part * BLOCK:part * BLOCK + first] = nearest_code(held * (old / scale))
            for (c, _), row in zip(cells, new):
                codes[page, h, part * BLOCK + c] = nearest_code(row / scale)
            scales[page, h, part] = scale


def cached(codes, scales, table, length):
    """Values [length, kv_heads, D] (f64) of one sequence's positions, and which lie on a page of the pool."""
    pages, kvh, pt, D = codes.shape
    out, good = torch.zeros(length, kvh, D, dtype=torch.float64), torch.zeros(length, dtype=torch.bool)
    for i in range(-(-length // pt)):
        page, n = int(table[i]) if i < len(table) else -1, min(pt, length - i * pt)
        if 0 <= page < pages:
            v = decode(codes[page]) * scales[page].double().repeat_interleave(BLOCK, 1)[..., None]
            out[i * pt:i * pt + n] = v.transpose(0, 1)[:n]
            good[i * pt:i * pt + n] = True
    return out, good


def attend(q, k, v, v_codes, v_scales, seen):
    """(o, tolerance) of one head's rows: q [n, D], k, v, v_codes [L, D],
    v_scales [L] f64, seen bool [n, L].

    The tolerance counts the kernel's roundings. Scores: q enters as e4m3 parts
    of a power of two's multiples, off by at most 2^-19 of the row's largest
    element in each dimension, and f32 sums lose at most D steps of 2^-23 of sum
    |q k| (an accumulator may truncate), so a softmax weight is off by delta =
    (2^-19 max|q| sum|k| + D 2^-23 sum|q k|) / sqrt(D) + 2^-20 (scaling,
    exponential, rescaling) on either side of the quotient. Weights enter the
    second product times V's scale as two e4m3 parts: off by 2^-8 of themselves
    (a part is off by 2^-4 of what it rounds), or by half the codes' smallest
    step, 2^-10, where the row's largest lies at 2^5 or above (a row's reference is
    set so that the largest of it lies in (2^5, 2^6], and moves before one passes
    2^8.75): 2^-15 of that, times the code of V. The sum over L keys L 2^-23; the output 2^-8 of the value."""
    D = q.shape[1]
    s = (q @ k.T / math.sqrt(D)).masked_fill(~seen, -math.inf)
    p = torch.softmax(s, 1)
    p = torch.where(seen.any(1, keepdim=True), p, torch.zeros_like(p))
    o, mag = p @ v, p @ v.abs()
    sums = torch.where(seen, (q.abs() @ k.abs().T) * D * 2.0 ** -23
                       + q.abs().amax(1, keepdim=True) * k.abs().sum(1) * 2.0 ** -19, torch.zeros_like(p)).amax(1, keepdim=True)
    delta = sums / math.sqrt(D) + 2.0 ** -20
    step = (p * v_scales).amax(1, keepdim=True) * 2.0 ** -15 * (seen.double() @ v_codes.abs())
    return o, (mag * (2.0 ** -8 + 2 * delta + k.shape[0] * 2.0 ** -23) + step) * 1.01 + o.abs() * 2.0 ** -8


def verify(p, q, tokens, row_starts, accept_u, sample_u, out):
    """Lists (accepted, tokens) of cheetah_cuda_op_verify_drafts; `out` is what the rows held.
    p, q (or None) f32 arrays."""
    accepted, out, vocab = [], list(out), p.shape[1]
    clean = lambda a: np.where(a > 0, a, 0.0).astype(np.float64)  # noqa: E731  (NaN, too)
    for b, (r0, r1) in enumerate(zip(row_starts, row_starts[1:])):
        if r1 <= r0:
            accepted.append(-1)
            continue
        r = r0
        while r + 1 < r1:
            x = tokens[r + 1]
            if not 0 <= x < vocab:
                break
            if not float(accept_u[r]) * (1.0 if q is None else float(clean(q[r])[x])) < float(clean(p[r])[x]):
                break
            r += 1
        w = clean(p[r])
        if r + 1 < r1:
            left = w.copy()
            if q is not None:
                left = np.maximum(w - clean(q[r]), 0.0)
            elif 0 <= tokens[r + 1] < vocab:
                left[tokens[r + 1]] = 0.0
            if left.sum() > 0:
                w = left
        total = math.fsum(w.tolist()) if np.isfinite(w).all() else math.inf
        if not 0 < total < math.inf:
            token = -1
        else:
            past = np.nonzero((np.cumsum(w) > float(sample_u[b]) * total) & (w > 0))[0]
            token = int(past[0]) if len(past) else int(np.nonzero(w)[0][-1])
        accepted.append(r - r0)
        for i in range(r0, r1):
            out[i] = tokens[i + 1] if i < r else token if i == r else -1
    return accepted, out
