"""Performance cases of the operators over a key/value cache held in 8 bits, and
of the test that keeps or drops drafted tokens.

The cache is paged like the 16-bit one: codes are e4m3, and the 16 cells of a
block share one scale per KV head, a power of two (K and V apart). A serving
step over it runs them in this order: `qk_norm_rope_kv8` normalises and rotates
q and k and appends K/V in 8 bits, `attention_kv8` attends from each sequence's
new rows over its cache (causal, with an optional sliding window beside which
the first `sinks` positions stay visible), and `verify_drafts` tests the drafted
tokens against the target's probabilities and samples the one that follows the
last kept. `kv8_read` takes cells back out of the cache, as a program does that
moves a prefix to a 16-bit pool.

`run` computes a case in plain torch, or through the library when `own` is
set. Lengths of a ragged batch come from the case (so that `work` knows them);
values, page ids and tokens come from the seed.
"""

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
E4M3 = torch.float8_e4m3fn
BLOCK = 16    # cells that share a scale
TOP = 448.0   # the largest e4m3 value
LEAST = -64   # log2 of the smallest scale


# ---- cases ------------------------------------------------------------------

def listed():
    return [
        # One decoded token of one sequence (the 0.5B head geometry, f32 projections as the GEMV path leaves them).
        dict(name="append-token-1", op="append", batch=1, new_lo=1, new_hi=1, cached_lo=701, cached_hi=701, q_heads=14,
             kv_heads=2, head_dim=64, rotary_dim=64, dtype="f32", norm=True, page_tokens=64, lengths=1),
        # The drafted tokens of a serving batch (the 7B head geometry): most blocks hold earlier tokens.
        dict(name="append-verify-256", op="append", batch=256, new_lo=1, new_hi=7, cached_lo=0, cached_hi=8192, q_heads=28,
             kv_heads=4, head_dim=128, rotary_dim=128, dtype="bf16", norm=True, page_tokens=64, lengths=2),
        # Prompt chunks of a long prefill.
        dict(name="append-prompt-4", op="append", batch=4, new_lo=8000, new_hi=8192, cached_lo=0, cached_hi=100, q_heads=28,
             kv_heads=4, head_dim=128, rotary_dim=128, dtype="bf16", norm=True, page_tokens=64, lengths=3),
        # A short prefix taken out of the cache for a sequence that continues in 16 bits.
        dict(name="read-prefix-701", op="read", tokens=701, kv_heads=2, head_dim=64, dtype="bf16", page_tokens=64),
        # A full context taken out.
        dict(name="read-prefix-32768", op="read", tokens=32768, kv_heads=4, head_dim=128, dtype="bf16", page_tokens=64),
        # One user, one token, a short conversation: latency.
        dict(name="attend-one-short", op="attend", batch=1, ctx_lo=700, ctx_hi=700, rows_lo=1, rows_hi=1, q_heads=14,
             kv_heads=2, head_dim=64, page_tokens=64, window=0, sinks=0, lengths=4),
        # One user, three drafted tokens at the end of a full 32k context.
        dict(name="attend-one-long", op="attend", batch=1, ctx_lo=32700, ctx_hi=32700, rows_lo=4, rows_hi=4, q_heads=14,
             kv_heads=2, head_dim=64, page_tokens=64, window=0, sinks=0, lengths=5),
        # A decode step of a serving batch with ragged contexts.
        dict(name="attend-serve-64", op="attend", batch=64, ctx_lo=1000, ctx_hi=16000, rows_lo=1, rows_hi=1, q_heads=28,
             kv_heads=4, head_dim=128, page_tokens=64, window=0, sinks=0, lengths=6),
        # Small drafts over long conversations, of which a window and the first tokens stay visible.
        dict(name="attend-window-32", op="attend", batch=32, ctx_lo=2000, ctx_hi=16000, rows_lo=1, rows_hi=9, q_heads=28,
             kv_heads=4, head_dim=128, page_tokens=64, window=4096, sinks=4, lengths=7),
        # A prompt chunk of two sequences, one of them behind a long prefix: most arithmetic.
        dict(name="attend-prompt-2", op="attend", batch=2, ctx_lo=0, ctx_hi=6000, rows_lo=2000, rows_hi=2048, q_heads=28,
             kv_heads=4, head_dim=128, page_tokens=64, window=0, sinks=0, lengths=8),
        # One user's four drafted tokens.
        dict(name="verify-one", op="verify", batch=1, drafts_lo=4, drafts_hi=4, vocab=151936, given=True, lengths=9),
        # The drafts of a serving batch, odd counts.
        dict(name="verify-serve-96", op="verify", batch=96, drafts_lo=0, drafts_hi=8, vocab=152064, given=True, lengths=10),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(14, 2, 64), (28, 4, 128), (32, 8, 64), (4, 4, 64), (8, 4, 128), (12, 2, 128), (8, 2, 64)]


def draw(rng):
    op = rng.choice(["append", "read", "attend", "attend", "verify"])
    while True:
        q_heads, kv_heads, head_dim = rng.choice(HEADS)
        if op == "append":
            new_hi, cached_hi = _log_int(rng, 1, 8192), _log_int(rng, 1, 16384)
            case = dict(op=op, batch=_log_int(rng, 1, 512), new_lo=_log_int(rng, 1, new_hi), new_hi=new_hi,
                        cached_lo=rng.choice([0, cached_hi]), cached_hi=cached_hi, q_heads=q_heads, kv_heads=kv_heads,
                        head_dim=head_dim, rotary_dim=rng.choice([head_dim, head_dim, head_dim // 2]),
                        dtype=rng.choice(["bf16", "f32"]), norm=rng.random() < 0.6, page_tokens=rng.choice([16, 64, 128]),
                        lengths=rng.randrange(1 << 20))
        elif op == "read":
            case = dict(op=op, tokens=_log_int(rng, 1, 32768), kv_heads=kv_heads, head_dim=head_dim,
                        dtype=rng.choice(["bf16", "f32"]), page_tokens=rng.choice([16, 48, 64, 128]))
        elif op == "attend":
            ctx_hi, rows_hi = _log_int(rng, 1, 32000), _log_int(rng, 1, rng.choice([8, 64, 2048]))
            case = dict(op=op, batch=_log_int(rng, 1, 96), ctx_lo=rng.choice([0, ctx_hi // 2, ctx_hi]), ctx_hi=ctx_hi,
                        rows_lo=rng.choice([1, rows_hi]), rows_hi=rows_hi, q_heads=q_heads, kv_heads=kv_heads,
                        head_dim=head_dim, page_tokens=rng.choice([16, 48, 64, 64, 128]),
                        window=rng.choice([0, 0, 48, _log_int(rng, 16, 4096)]), sinks=rng.choice([0, 1, 4, 130]),
                        lengths=rng.randrange(1 << 20))
        else:
            case = dict(op=op, batch=_log_int(rng, 1, 256), drafts_lo=rng.choice([0, 1, 3]), drafts_hi=rng.choice([3, 5, 8, 16]),
                        vocab=rng.choice([1000, 32001, 128256, 151936, 152064, _log_int(rng, 1, 200000)]),
                        given=rng.random() < 0.7, lengths=rng.randrange(1 << 20))
        top = max((c for c in listed() if c["op"] == op), key=_cost)
        if _cost(case) <= _cost(top) and work(case)["bytes"] <= work(top)["bytes"]:
            return case


def _lengths(case):
    """(cached positions, new rows) of each sequence of a ragged batch."""
    rng = random.Random(case["lengths"])
    lo, hi = {"append": (case.get("cached_lo"), case.get("cached_hi")), "attend": (case.get("ctx_lo"), case.get("ctx_hi")),
              "verify": (0, 0)}[case["op"]]
    nlo, nhi = {"append": (case.get("new_lo"), case.get("new_hi")), "attend": (case.get("rows_lo"), case.get("rows_hi")),
                "verify": (1 + case.get("drafts_lo", 0), 1 + case.get("drafts_hi", 0))}[case["op"]]
    return [rng.randint(lo, hi) for _ in range(case["batch"])], [rng.randint(nlo, nhi) for _ in range(case["batch"])]


def _cost(case):
    """What the plain form pads a case to (a bound on its time and memory)."""
    if case["op"] == "append":
        return case["batch"] * case["new_hi"] * (case["q_heads"] + 2 * case["kv_heads"]) * case["head_dim"]
    if case["op"] == "read":
        return case["tokens"] * case["kv_heads"] * case["head_dim"]
    if case["op"] == "attend":
        return case["batch"] * (case["ctx_hi"] + case["rows_hi"]) * (case["q_heads"] * case["rows_hi"] + 300 * case["kv_heads"]) * case["head_dim"]
    return case["batch"] * (case["drafts_hi"] + 1) * case["vocab"]


def _seen(ctx, n, window, sinks):
    """(distinct keys read, pairs of a row and a key that it sees) of one sequence."""
    i = np.arange(n, dtype=np.int64) + ctx  # positions
    low = np.maximum(i - window + 1, 0) if window else np.zeros_like(i)
    pairs = int((i - low + 1 + np.minimum(low, sinks)).sum())
    keys = int(ctx + n - low[0] + min(low[0], sinks)) if n else 0
    return keys, pairs


def work(case):
    """Bytes and operations one pass cannot do without."""
    if case["op"] == "append":
        t, d = sum(_lengths(case)[1]), case["head_dim"]
        e = 2 if case["dtype"] == "bf16" else 4
        heads = case["q_heads"] + 2 * case["kv_heads"]
        return {"bytes": t * (heads * d * e + case["q_heads"] * d * e + 2 * case["kv_heads"] * d + 8 + case["rotary_dim"] * 4),
                "flops": t * heads * d * 6}
    if case["op"] == "read":
        cells = 2 * case["tokens"] * case["kv_heads"] * case["head_dim"]
        return {"bytes": cells * (1 + (2 if case["dtype"] == "bf16" else 4)) + 4 * case["tokens"], "flops": cells}
    if case["op"] == "attend":
        d = case["head_dim"]
        seen = [_seen(c, n, case["window"], case["sinks"]) for c, n in zip(*_lengths(case))]
        rows = sum(_lengths(case)[1])
        return {"bytes": sum(k for k, _ in seen) * case["kv_heads"] * (2 * d + 8 / BLOCK) + 2 * rows * case["q_heads"] * d * 2,
                "flops": 4 * d * case["q_heads"] * sum(p for _, p in seen)}
    # The row that the next token is taken from; where a draft is dropped also the draft model's (not counted).
    return {"bytes": case["batch"] * case["vocab"] * 4 + 24 * sum(_lengths(case)[1]), "flops": 2 * case["batch"] * case["vocab"]}


# ---- inputs -----------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    return {"append": _prepare_append, "read": _prepare_read, "attend": _prepare_attend, "verify": _prepare_verify}[case["op"]](case, seed)


def _int32(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


def _pool(gen, pages, kv_heads, page_tokens, head_dim, spread):
    """Codes and scales of a filled pool: normal values whose size varies from block to block."""
    codes = torch.empty(pages, kv_heads, page_tokens, head_dim, dtype=E4M3, device="cuda")
    scales = torch.empty(pages, kv_heads, page_tokens // BLOCK, device="cuda")
    step = max(1, (1 << 27) // (kv_heads * page_tokens * head_dim))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        x = torch.randn(n, kv_heads, page_tokens // BLOCK, BLOCK * head_dim, device="cuda", generator=gen)
        x *= torch.exp(spread * torch.randn(n, kv_heads, page_tokens // BLOCK, 1, device="cuda", generator=gen))
        s = _scale_of(x.abs().amax(-1))
        scales[p:p + n] = s
        codes[p:p + n] = (x / s[..., None]).to(E4M3).reshape(n, kv_heads, page_tokens, head_dim)
    return codes, scales


def _scale_of(top):
    """The smallest power of two whose 448-fold reaches `top`."""
    m, e = torch.frexp(top)
    e = torch.where(top > 0, e - 9 + (m > 0.875).to(e.dtype), LEAST).clamp(min=LEAST)
    return torch.ldexp(torch.ones_like(top), e)


def _rope(positions, rotary_dim, theta=1e6):
    freq = theta ** (-torch.arange(0, rotary_dim, 2, device="cuda", dtype=torch.float64) / rotary_dim)
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * freq
    return angle.cos().float().contiguous(), angle.sin().float().contiguous()


def _prepare_append(case, seed):
    g = _gen(seed)
    cached, new = (np.array(x, dtype=np.int64) for x in _lengths(case))
    qh, kh, d, pt = case["q_heads"], case["kv_heads"], case["head_dim"], case["page_tokens"]
    # The pool holds the pages that the new tokens lie on; the pages before them are not touched.
    first, last = cached // pt, (cached + new - 1) // pt
    base = np.concatenate([[0], np.cumsum(last - first + 1)])
    num_pages = int(base[-1]) + 3
    seq = np.repeat(np.arange(len(new)), new)
    pos = np.arange(int(new.sum())) - np.repeat(np.cumsum(new) - new, new) + cached[seq]
    order = torch.randperm(num_pages, device="cuda", generator=g)
    page = order[torch.from_numpy(base[seq] + pos // pt - first[seq]).cuda()]
    slots = page * pt + torch.from_numpy(pos % pt).cuda()
    positions = int((cached + new).max())
    qkv = (torch.randn(len(seq), qh + 2 * kh, d, device="cuda", generator=g) * 2.0).to(DTYPES[case["dtype"]])
    k_codes, k_scales = _pool(g, num_pages, kh, pt, d, 0.5)
    v_codes, v_scales = _pool(g, num_pages, kh, pt, d, 0.5)
    cos, sin = _rope(positions, case["rotary_dim"])
    weight = lambda: 1.0 + 0.2 * torch.randn(d, device="cuda", generator=g) if case["norm"] else None  # noqa: E731
    return dict(op="append", qkv=qkv, q_heads=qh, kv_heads=kh, positions=_int32(pos), slots=slots.to(torch.int32), cos=cos, sin=sin,
                k_codes=k_codes, v_codes=v_codes, k_scales=k_scales, v_scales=v_scales, q_norm=weight(), k_norm=weight(), eps=1e-6)


def _prepare_read(case, seed):
    g = _gen(seed)
    t, pt = case["tokens"], case["page_tokens"]
    num_pages = -(-t // pt) + 2
    k_codes, k_scales = _pool(g, num_pages, case["kv_heads"], pt, case["head_dim"], 0.5)
    v_codes, v_scales = _pool(g, num_pages, case["kv_heads"], pt, case["head_dim"], 0.5)
    pages = torch.randperm(num_pages, device="cuda", generator=g)
    at = torch.arange(t, device="cuda")
    return dict(op="read", k_codes=k_codes, v_codes=v_codes, k_scales=k_scales, v_scales=v_scales,
                slots=(pages[at // pt] * pt + at % pt).to(torch.int32), dtype=DTYPES[case["dtype"]])


def _prepare_attend(case, seed):
    g = _gen(seed)
    ctx, rows = _lengths(case)
    pt, qh, kh, d = case["page_tokens"], case["q_heads"], case["kv_heads"], case["head_dim"]
    pages_of = [-(-(c + n) // pt) for c, n in zip(ctx, rows)]
    num_pages = sum(pages_of) + 3
    k_codes, k_scales = _pool(g, num_pages, kh, pt, d, 0.25)
    v_codes, v_scales = _pool(g, num_pages, kh, pt, d, 0.5)
    # Shuffled distinct pages of each sequence, -1 behind them.
    order = torch.randperm(num_pages, device="cuda", generator=g).to(torch.int32)
    counts = torch.tensor(pages_of, device="cuda")
    col = torch.arange(max(pages_of), device="cuda")
    at = ((torch.cumsum(counts, 0) - counts)[:, None] + col).clamp(max=num_pages - 1)
    table = torch.where(col < counts[:, None], order[at], torch.full_like(order[at], -1)).contiguous()
    q = (torch.randn(sum(rows), qh, d, device="cuda", generator=g) * 1.5).to(torch.bfloat16)
    return dict(op="attend", q=q, k_codes=k_codes, v_codes=v_codes, k_scales=k_scales, v_scales=v_scales, table=table,
                seq_lens=_int32([c + n for c, n in zip(ctx, rows)]), row_starts=_int32(np.concatenate([[0], np.cumsum(rows)])),
                window=case["window"], sinks=case["sinks"], longest=max(c + n for c, n in zip(ctx, rows)), most=max(rows))


def _prepare_verify(case, seed):
    g = _gen(seed)
    rows, vocab = _lengths(case)[1], case["vocab"]
    total = sum(rows)
    starts = np.concatenate([[0], np.cumsum(rows)])
    # A few likely tokens above the rest; the draft model says nearly the same.
    x = 2.0 * torch.randn(total, vocab, device="cuda", generator=g)
    hot = torch.randint(0, vocab, (total, 12), device="cuda", generator=g)
    x.scatter_add_(1, hot, 12.0 * torch.rand(total, 12, device="cuda", generator=g))
    p = torch.softmax(x, -1)
    q = torch.softmax(x.add_(torch.randn(total, vocab, device="cuda", generator=g), alpha=0.4), -1)
    # Row r's distribution gives the token of row r + 1.
    drawn = torch.searchsorted(torch.cumsum(q, -1), torch.rand(total, 1, device="cuda", generator=g)).clamp(max=vocab - 1)[:, 0]
    tokens = torch.cat([drawn.new_zeros(1), drawn[:-1]]).to(torch.int32)
    return dict(op="verify", p=p, q=q if case["given"] else None, tokens=tokens, row_starts=_int32(starts),
                accept_u=torch.rand(total, device="cuda", generator=g), sample_u=torch.rand(len(rows), device="cuda", generator=g))


# ---- one pass ---------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    return {"append": _plain_append, "read": _plain_read, "attend": _plain_attend, "verify": _plain_verify}[state["op"]](state)


def _run_own(s):
    from cheetah_b200 import runtime as R
    if s["op"] == "append":
        q = R.qk_norm_rope_kv8(s["qkv"], s["q_heads"], s["kv_heads"], s["positions"], s["slots"], s["cos"], s["sin"],
                               s["k_codes"], s["v_codes"], s["k_scales"], s["v_scales"], q_norm=s["q_norm"],
                               k_norm=s["k_norm"], eps=s["eps"])
        return dict(q=q, k_codes=s["k_codes"], v_codes=s["v_codes"], k_scales=s["k_scales"], v_scales=s["v_scales"])
    if s["op"] == "read":
        k, v = R.kv8_read(s["k_codes"], s["v_codes"], s["k_scales"], s["v_scales"], s["slots"], dtype=s["dtype"])
        return dict(k=k, v=v)
    if s["op"] == "attend":
        return R.attention_kv8(s["q"], s["k_codes"], s["v_codes"], s["k_scales"], s["v_scales"], s["table"], s["seq_lens"],
                               s["row_starts"], sliding_window=s["window"], sinks=s["sinks"])
    r = R.verify_drafts(s["p"], s["q"], s["tokens"], s["row_starts"], s["accept_u"], s["sample_u"])
    return dict(accepted=r.accepted, tokens=r.tokens)


def _normed(x, weight, eps):
    return x if weight is None else x * (torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight.to(x.dtype))


def _rotated(x, cos, sin):
    half = cos.shape[-1]
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _plain_append(s):
    qh, kh = s["q_heads"], s["kv_heads"]
    at = s["positions"].long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    q = _rotated(_normed(s["qkv"][:, :qh].float(), s["q_norm"], s["eps"]), cos, sin)
    # A code is decided in 64 bits: values lie next to the border of two codes.
    k = _rotated(_normed(s["qkv"][:, qh:qh + kh].double(), s["k_norm"], s["eps"]), cos.double(), sin.double())
    _plain_write(k, s["k_codes"], s["k_scales"], s["slots"].long())
    _plain_write(s["qkv"][:, qh + kh:].double(), s["v_codes"], s["v_scales"], s["slots"].long())
    return dict(q=q.to(s["qkv"].dtype), k_codes=s["k_codes"], v_codes=s["v_codes"], k_scales=s["k_scales"], v_scales=s["v_scales"])


def _to_e4m3(x):
    """Nearest e4m3 value of 64-bit ones, ties to even: the steps are 2^-9 up to 2^-6 and an eighth of the power of two below."""
    _, e = torch.frexp(x)
    e = (e - 4).clamp(min=-9)
    return torch.ldexp(torch.round(torch.ldexp(x, -e)), e).to(E4M3)


def _plain_write(x, codes, scales, slots):
    """Cells `slots` of a pool become x [tokens, kv_heads, head_dim]."""
    pages, kh, pt, d = codes.shape
    blocks = pages * (pt // BLOCK)
    block, cell = slots // BLOCK, slots % BLOCK
    first = torch.full((blocks,), BLOCK, device="cuda").scatter_reduce(0, block, cell, "amin")
    top = torch.zeros(blocks, kh, dtype=torch.float64, device="cuda")
    top = top.scatter_reduce(0, block[:, None].expand(-1, kh), x.abs().amax(-1), "amax")
    old = scales.transpose(1, 2).reshape(blocks, kh).clone()
    new = _scale_of(top).float()
    new = torch.where((first > 0)[:, None], torch.maximum(old, new), new)
    new = torch.where((first < BLOCK)[:, None], new, old)
    # Cells ahead of the first new one keep their values, in the new scale.
    held = codes.view(pages, kh, pt // BLOCK, BLOCK, d)
    ratio = (old / new).double().view(pages, pt // BLOCK, kh).transpose(1, 2)[..., None, None]
    keep = (torch.arange(BLOCK, device="cuda") < torch.where(first < BLOCK, first, 0)[:, None]).view(pages, 1, pt // BLOCK, BLOCK, 1)
    moved = torch.where(keep, _to_e4m3(held.double() * ratio).view(torch.uint8), held.view(torch.uint8)).view(pages, kh, pt, d)
    moved[slots // pt, :, slots % pt] = _to_e4m3(x / new.double()[block][:, :, None]).view(torch.uint8)
    codes.view(torch.uint8).copy_(moved)
    scales.copy_(new.view(pages, pt // BLOCK, kh).transpose(1, 2))


def _plain_read(s):
    pt = s["k_codes"].shape[2]
    page, cell = s["slots"].long() // pt, s["slots"].long() % pt

    def take(codes, scales):
        x = codes.view(torch.uint8)[page, :, cell].view(E4M3).float()
        return (x * scales[page, :, cell // BLOCK][:, :, None]).to(s["dtype"])

    return dict(k=take(s["k_codes"], s["k_scales"]), v=take(s["v_codes"], s["v_scales"]))


def _plain_attend(s):
    total, qh, d = s["q"].shape
    kh, pt = s["k_codes"].shape[1:3]
    batch, longest, most = s["table"].shape[0], s["longest"], s["most"]
    starts = s["row_starts"].long()
    rows = starts[1:] - starts[:-1]
    ctx = s["seq_lens"].long() - rows
    key = torch.arange(longest, device="cuda")
    page = s["table"].long()[:, key // pt].clamp(min=0)

    def cached(codes, scales):  # [batch, kv_heads, longest, d]
        x = codes.view(torch.uint8)[page, :, key % pt].view(E4M3).float()
        return (x * scales[page, :, (key % pt) // BLOCK][..., None]).transpose(1, 2)

    k = cached(s["k_codes"], s["k_scales"])
    i = torch.arange(most, device="cuda")
    row = (starts[:-1, None] + i).clamp(max=total - 1)
    q = s["q"][row].float().reshape(batch, most, kh, qh // kh, d).permute(0, 2, 3, 1, 4).reshape(batch, kh, -1, d)
    pos = ctx[:, None, None] + i[None, :, None]
    seen = (key <= pos) & (key < s["seq_lens"][:, None, None])
    if s["window"]:
        seen = seen & ((key + s["window"] > pos) | (key < s["sinks"]))
    seen = seen[:, None, None]
    score = (q @ k.transpose(2, 3)).reshape(batch, kh, qh // kh, most, longest) / math.sqrt(d)
    del k
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total_e = e.sum(-1, keepdim=True)
    p = e.div_(torch.where(total_e > 0, total_e, 1.0)).reshape(batch, kh, -1, longest)
    v = cached(s["v_codes"], s["v_scales"])
    v = torch.where((key[None, :] < s["seq_lens"][:, None])[:, None, :, None], v, 0.0)
    o = (p @ v).reshape(batch, kh, qh // kh, most, d).permute(0, 3, 1, 2, 4).reshape(batch, most, qh, d)
    t = torch.arange(total, device="cuda")
    b = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    return o[b, t - starts[b]].to(torch.bfloat16)


def _plain_verify(s):
    p, q, starts = s["p"], s["q"], s["row_starts"].long()
    total, vocab = p.shape
    r = torch.arange(total, device="cuda")
    b = torch.searchsorted(starts[1:].contiguous(), r, right=True)
    last = starts[1:] - 1
    # Row r tests the token of row r + 1; products of two 32-bit numbers are exact in 64.
    draft = s["tokens"].long()[(r + 1).clamp(max=total - 1)][:, None]
    p_x = p.gather(1, draft)[:, 0].double()
    q_x = torch.ones_like(p_x) if q is None else q.gather(1, draft)[:, 0].double()
    passed = (s["accept_u"].double() * q_x < p_x) & (r < last[b])
    end = torch.where(passed, total, r)
    stop = torch.full_like(last, total).scatter_reduce(0, b, end, "amin")
    accepted = stop - starts[:-1]
    # What is left of the target's distribution where a draft was dropped.
    w = p[stop].double()
    dropped = (stop < last)[:, None]
    if q is None:
        left = w.scatter(1, draft[stop], 0.0)
    else:
        left = (w - q[stop].double()).clamp(min=0.0)
    left = torch.where(dropped, left, w)
    left = torch.where(left.sum(-1, keepdim=True) > 0, left, w)
    run_sum = torch.cumsum(left, -1)
    at = s["sample_u"].double()[:, None] * run_sum[:, -1:]
    following = torch.searchsorted(run_sum, at, right=True).clamp(max=vocab - 1)[:, 0]
    kept = torch.where(r < stop[b], s["tokens"].long()[(r + 1).clamp(max=total - 1)], torch.where(r == stop[b], following[b], -1))
    return dict(accepted=accepted.to(torch.int32), tokens=kept.to(torch.int32))


# ---- the definitions in 64 bits ----------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "read": _exact_read, "attend": _exact_attend, "verify": _exact_verify}[case["op"]](s)


def _exact_append(s):
    qh, kh = s["q_heads"], s["kv_heads"]
    x = s["qkv"].double()
    c, sn = s["cos"].double()[s["positions"].long()], s["sin"].double()[s["positions"].long()]
    half = c.shape[1]

    def head(h, weight):
        y = x[:, h]
        if weight is not None:
            y = y / (y.pow(2).mean(-1, keepdim=True) + s["eps"]).sqrt() * weight.double()
        z = y.clone()
        z[:, :half] = y[:, :half] * c - y[:, half:2 * half] * sn
        z[:, half:2 * half] = y[:, half:2 * half] * c + y[:, :half] * sn
        return z

    out = dict(q=torch.stack([head(h, s["q_norm"]) for h in range(qh)], 1))
    slots = s["slots"].cpu().numpy().astype(np.int64)
    pt = s["k_codes"].shape[2]
    blocks, of_row = np.unique(slots // BLOCK, return_inverse=True)
    first = np.full(len(blocks), BLOCK)
    np.minimum.at(first, of_row, slots % BLOCK)
    # The e4m3 values in order, and what lies between two of them: a tie goes to the even one.
    values = torch.arange(127, dtype=torch.uint8, device="cuda").view(E4M3).double()
    between = (values[1:] + values[:-1]) / 2

    def nearest(y):
        at = torch.bucketize(y.abs(), between)
        tie = (y.abs() == between[at.clamp(max=125)]) & (at < 126)
        return values[torch.where(tie, at + at % 2, at)] * torch.sign(y)

    for name, heads, weight in (("k", range(qh, qh + kh), s["k_norm"]), ("v", range(qh + kh, qh + 2 * kh), None)):
        codes, scales = s[name + "_codes"].double(), s[name + "_scales"].double()
        lead = torch.from_numpy(first).cuda()
        page, part = (torch.from_numpy(a).cuda() for a in np.divmod(blocks, pt // BLOCK))
        row_block = torch.from_numpy(of_row).cuda()
        row_page, row_cell = (torch.from_numpy(a).cuda() for a in np.divmod(slots, pt))
        for h, head_at in enumerate(heads):
            y = head(head_at, weight) if name == "k" else x[:, head_at]
            top = torch.zeros(len(blocks), dtype=torch.float64, device="cuda").index_reduce_(0, row_block, y.abs().amax(-1), "amax")
            need = torch.exp2(torch.ceil(torch.log2(top.clamp(min=1e-300) / TOP)).clamp(min=LEAST))
            need = torch.where(top > TOP * need, 2 * need, torch.where((top <= TOP * need / 2) & (need > 2.0 ** LEAST), need / 2, need))
            old = scales[page, h, part]
            scale = torch.where(lead > 0, torch.maximum(old, need), need)
            cell = part[:, None] * BLOCK + torch.arange(BLOCK, device="cuda")
            held = codes[page[:, None], h, cell]
            moved = nearest(held * (old / scale)[:, None, None])
            codes[page[:, None], h, cell] = torch.where((torch.arange(BLOCK, device="cuda") < lead[:, None])[..., None], moved, held)
            codes[row_page, h, row_cell] = nearest(y / scale[row_block][:, None])
            scales[page, h, part] = scale
        out[name + "_codes"], out[name + "_scales"] = codes, scales
    return dict(q=out["q"], k_codes=out["k_codes"], v_codes=out["v_codes"], k_scales=out["k_scales"], v_scales=out["v_scales"])


def _exact_read(s):
    pt = s["k_codes"].shape[2]
    out = {}
    for name in ("k", "v"):
        per_cell = s[name + "_scales"].double().repeat_interleave(BLOCK, 2)
        cells = (s[name + "_codes"].double() * per_cell[..., None]).transpose(1, 2).flatten(0, 1)
        assert cells.shape[0] % pt == 0
        out[name] = cells[s["slots"].long()]
    return out


def _exact_attend(s):
    total, qh, d = s["q"].shape
    kh, pt = s["k_codes"].shape[1:3]
    starts, lens = s["row_starts"].tolist(), s["seq_lens"].tolist()
    out = torch.zeros(total, qh, d, dtype=torch.float64, device="cuda")
    for b, length in enumerate(lens):
        r0, r1 = starts[b], starts[b + 1]
        pages = s["table"][b, :-(-length // pt)].long()
        k, v = ((s[n + "_codes"].view(torch.uint8)[pages].view(E4M3).double()
                 * s[n + "_scales"][pages].double().repeat_interleave(BLOCK, 2)[..., None]).transpose(1, 2).reshape(-1, kh, d)[:length]
                for n in ("k", "v"))
        behind = torch.arange(length - (r1 - r0), length, device="cuda")[:, None] - torch.arange(length, device="cuda")
        hidden = behind < 0
        if s["window"]:
            hidden |= (behind >= s["window"]) & (torch.arange(length, device="cuda") >= s["sinks"])
        for h in range(qh):
            a = (s["q"][r0:r1, h].double() @ k[:, h * kh // qh].T / math.sqrt(d)).masked_fill(hidden, -math.inf)
            out[r0:r1, h] = torch.softmax(a, -1) @ v[:, h * kh // qh]
    return out


def _exact_verify(s):
    starts, tokens = s["row_starts"].tolist(), s["tokens"].tolist()
    accept_u, sample_u = s["accept_u"].double().tolist(), s["sample_u"].double().tolist()
    accepted, out = [], []
    for b, (r0, r1) in enumerate(zip(starts, starts[1:])):
        r, dropped = r0, False
        while r + 1 < r1:
            x = tokens[r + 1]
            if not accept_u[r] * (1.0 if s["q"] is None else float(s["q"][r, x])) < float(s["p"][r, x]):
                dropped = True
                break
            r += 1
        w = s["p"][r].double()
        if dropped:
            if s["q"] is None:
                left = w.clone()
                left[tokens[r + 1]] = 0.0
            else:
                left = torch.maximum(w - s["q"][r].double(), torch.zeros_like(w))
            w = left if float(left.sum()) > 0 else w
        upto = torch.cumsum(w, 0)
        past = upto > sample_u[b] * upto[-1]
        accepted.append(r - r0)
        out += tokens[r0 + 1:r + 1] + [int(past.int().argmax())] + [-1] * (r1 - r - 1)
    return dict(accepted=_int32(accepted), tokens=_int32(out))
