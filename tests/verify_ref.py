"""Plain 64-bit references of the operators that verify drafted tokens, one
sequence, row and head at a time, on the CPU."""

import math

import numpy as np
import torch


def page_slots(cached, new, free, free_count, table, num_pages, page_tokens, max_tokens):
    """Python restatement of cheetah_cuda_op_page_slots (lists and a numpy table)."""
    table = np.array(table, dtype=np.int64)
    capacity = table.shape[1] * page_tokens
    free_count = min(max(free_count, 0), len(free))
    starts, lens, pos, ids, slots = [0], [], [], [], []
    asked, pages, taken, refused = 0, 0, 0, 0
    for b, (c, n) in enumerate(zip(cached, new)):
        ok = c >= 0 and n >= 0 and c + n <= capacity
        n = n if ok else 0
        asked += n
        ok = ok and asked <= max_tokens
        have = -(-c // page_tokens)
        need = -(-(c + n) // page_tokens) - have if ok else 0
        pages += need
        got = ok and (need == 0 or pages <= free_count)
        if got:
            table[b, have:have + need] = free[pages - need:pages]
            taken += need
        else:
            refused += 1
        starts.append(min(asked, max_tokens))
        lens.append(c + n if got else 0)
        for i in range(starts[-1] - starts[-2]):
            ids.append(b)
            pos.append(c + i if got else -1)
            page = table[b, (c + i) // page_tokens] if got else -1
            slots.append(page * page_tokens + (c + i) % page_tokens if 0 <= page < num_pages else -1)
    pad = [-1] * (max_tokens - starts[-1])
    return dict(table=table, row_starts=starts, seq_lens=lens, positions=pos + pad, seq_ids=ids + pad, slots=slots + pad,
                counts=[min(asked, 2 ** 31 - 1), taken, refused])


def norm_rope_head(x, weight, eps, cos, sin):
    """(result, sum of the magnitudes its last addition joins) of one head, f64."""
    y = x.double()
    if weight is not None:
        y = y * (weight.double() / torch.sqrt((y * y).mean() + eps))
    half = cos.numel()
    z, mag = y.clone(), y.abs().clone()
    a, b = y[:half], y[half:2 * half]
    c, s = cos.double(), sin.double()
    z[:half], z[half:2 * half] = a * c - b * s, b * c + a * s
    mag[:half], mag[half:2 * half] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return z, mag


def tree_row(q, k, v, seen):
    """(o, tolerance) of one row and head: q [D], k/v [L, D] f64, seen bool [L].

    The tolerance counts the kernel's roundings: products of bf16 values are
    exact in f32 and their sums lose at most D steps of 2^-23 of sum |q k| (an
    accumulator may truncate), so a softmax weight is off by delta = D 2^-23
    max_j sum|q k_j|/sqrt(D) + 2^-20 (scaling, exponential, rescaling); its
    rounding to bf16 adds 2^-8; the f32 sum over L keys L 2^-23; the output's
    rounding 2^-8 of the value."""
    D = q.numel()
    if not bool(seen.any()):
        return torch.zeros(D, dtype=torch.float64), torch.zeros(D, dtype=torch.float64)
    k, v = k[seen], v[seen]
    p = torch.softmax(k @ q / math.sqrt(D), 0)
    o, mag = p @ v, p @ v.abs()
    delta = D * 2.0 ** -23 * float((k.abs() @ q.abs()).max()) / math.sqrt(D) + 2.0 ** -20
    tol = mag * (2.0 ** -8 + 2 * delta + k.shape[0] * 2.0 ** -23) * 1.01 + o.abs() * 2.0 ** -8
    return o, tol


def logprobs_row(x, token, top):
    """Row of logits in f64: dict of the outputs and `tol` (logprob-like,
    entropy). Each exponential is off by a few steps of 2^-24 plus the rounding
    of its argument; a sum adds at most vocab/128 + 64 roundings (partial sums
    per thread, then a tree)."""
    x = x.double()
    bad = bool(torch.isnan(x).any()) or bool((x == math.inf).any()) or not bool((x > -math.inf).any())
    if bad:
        return dict(bad=True)
    m = x.max()
    gap = torch.where(x > -math.inf, m - x, torch.zeros_like(x))
    e = torch.exp(x - m)
    s = e.sum()
    log_s = torch.log(s)
    u = 2.0 ** -24
    steps = x.numel() / 128 + 64
    rel = float((e * (8 + gap)).sum() / s) * u + steps * u  # of S
    h = log_s + (gap * e).sum() / s
    order = torch.sort(x, descending=True, stable=True)
    known = 0 <= token < x.numel()
    out = dict(bad=False, known=known, entropy=float(h), top_ids=order.indices[:top].tolist(),
               top_logprobs=((order.values[:top] - m) - log_s), rel=rel, log_s=float(log_s), m=float(m))
    out["tol_entropy"] = 2 * rel * (1.0 + float(h)) + float((e * gap * (8 + gap)).sum() / s) * u + 4 * u * float(h)
    if known:
        out["logprob"] = float((x[token] - m) - log_s)
        out["rank"] = 1 + int((x > x[token]).sum())
    return out


def tol_logprob(ref, value):
    """Tolerance of a log probability `value` of the row `ref` describes."""
    u = 2.0 ** -24
    return ref["rel"] + 4 * u * (abs(value) + abs(ref["log_s"]) + 1e-6)


def random_tree(rng, n):
    """Parent of each node (-1: the context)."""
    return [int(rng.integers(-1, i)) if i else -1 for i in range(n)]


def tree_bits(parents):
    """(bool [n, n] ancestors-or-self, depth [n])."""
    n = len(parents)
    seen, depth = np.zeros((n, n), bool), np.zeros(n, np.int64)
    for i, p in enumerate(parents):
        if p >= 0:
            seen[i], depth[i] = seen[p], depth[p] + 1
        seen[i, i] = True
    return seen, depth


def pack_bits(rows, words):
    """bool [rows, n] -> int64 [rows, words]."""
    padded = np.zeros((rows.shape[0], words * 64), bool)
    padded[:, :rows.shape[1]] = rows[:, :words * 64]
    return np.packbits(padded, axis=1, bitorder="little").view(np.int64)
