"""Performance cases of the operators that verify drafted tokens.

One verification step of a serving batch runs them in this order: `page_slots`
gives every new token its cell of the paged KV pool, `qk_norm_rope` normalises
and rotates q and k and appends K/V at those cells, `tree_attention` attends
from the drafted nodes over the cache and their own ancestors, and
`token_logprobs` scores the drafted tokens from the logits.

`run` computes a case in plain torch, or through the library when `own` is
set. Lengths of a ragged batch come from the case (so that `work` knows them);
values, page ids, trees and tokens come from the seed.
"""

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---- cases ------------------------------------------------------------------

def listed():
    return [
        # A decode/verify step of a serving batch: 64 sequences, up to 16 drafted tokens each.
        dict(name="slots-verify-64", op="slots", batch=64, new_lo=1, new_hi=16, cached_lo=0, cached_hi=8192,
             page_tokens=64, lengths=1),
        # Admission of a burst of prompts: 256 sequences, most of them new, about a million tokens.
        dict(name="slots-admit-256", op="slots", batch=256, new_lo=128, new_hi=8192, cached_lo=0, cached_hi=1024,
             page_tokens=64, lengths=2),
        # One decoded token of one sequence (the 0.5B head geometry, f32 projections as the GEMV path leaves them).
        dict(name="qk-token-1", op="qk", tokens=1, q_heads=14, kv_heads=2, head_dim=64, rotary_dim=64, dtype="f32",
             kv_dtype="bf16", norm=True, page_tokens=64),
        # The drafted tokens of 64 sequences (the 7B head geometry), odd count.
        dict(name="qk-verify-1021", op="qk", tokens=1021, q_heads=28, kv_heads=4, head_dim=128, rotary_dim=128,
             dtype="bf16", kv_dtype="bf16", norm=True, page_tokens=64),
        # Prompt chunks of a long prefill.
        dict(name="qk-prompt-32768", op="qk", tokens=32768, q_heads=28, kv_heads=4, head_dim=128, rotary_dim=128,
             dtype="bf16", kv_dtype="bf16", norm=True, page_tokens=64),
        # One user, a small tree, a short conversation: latency.
        dict(name="tree-one-short", op="tree", batch=1, ctx_lo=700, ctx_hi=700, nodes_lo=8, nodes_hi=8, q_heads=14,
             kv_heads=2, head_dim=64, page_tokens=64, window=0, lengths=3),
        # One user, a wide tree at the end of a full 32k context.
        dict(name="tree-one-long", op="tree", batch=1, ctx_lo=32700, ctx_hi=32700, nodes_lo=64, nodes_hi=64,
             q_heads=14, kv_heads=2, head_dim=64, page_tokens=64, window=0, lengths=4),
        # A serving batch with ragged contexts and small drafts.
        dict(name="tree-serve-32", op="tree", batch=32, ctx_lo=128, ctx_hi=8192, nodes_lo=1, nodes_hi=16, q_heads=28,
             kv_heads=4, head_dim=128, page_tokens=64, window=0, lengths=5),
        # A large batch of wide trees: most arithmetic.
        dict(name="tree-wide-64", op="tree", batch=64, ctx_lo=3000, ctx_hi=8000, nodes_lo=40, nodes_hi=64, q_heads=28,
             kv_heads=4, head_dim=128, page_tokens=64, window=0, lengths=6),
        # The log probability of one sampled token with the five alternatives an API answer lists.
        dict(name="logprobs-token-1", op="logprobs", rows=1, vocab=151936, dtype="f32", top=5),
        # Drafted tokens of a batch, rounded logits, the most alternatives.
        dict(name="logprobs-verify-500", op="logprobs", rows=500, vocab=152064, dtype="bf16", top=20),
        # Scoring a prompt chunk.
        dict(name="logprobs-score-2048", op="logprobs", rows=2048, vocab=151936, dtype="f32", top=1),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["slots", "qk", "tree", "tree", "logprobs"])
    while True:
        if op == "slots":
            new_hi = _log_int(rng, 1, 8192)
            case = dict(op=op, batch=_log_int(rng, 1, 2048), new_lo=_log_int(rng, 1, new_hi), new_hi=new_hi, cached_lo=0,
                        cached_hi=_log_int(rng, 1, 16384), page_tokens=rng.choice([16, 32, 64, 128]),
                        lengths=rng.randrange(1 << 20))
        elif op == "qk":
            q_heads, kv_heads, head_dim = rng.choice([(14, 2, 64), (28, 4, 128), (32, 8, 64), (4, 4, 64), (8, 4, 128),
                                                      (12, 2, 128), (8, 2, 64)])
            case = dict(op=op, tokens=_log_int(rng, 1, 32768), q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim,
                        rotary_dim=rng.choice([head_dim, head_dim, head_dim // 2]), dtype=rng.choice(["bf16", "f32"]),
                        kv_dtype=rng.choice(["bf16", "bf16", "f32"]), norm=rng.random() < 0.6,
                        page_tokens=rng.choice([16, 64, 128]))
        elif op == "tree":
            q_heads, kv_heads, head_dim = rng.choice([(14, 2, 64), (28, 4, 128), (32, 8, 64), (4, 4, 64), (8, 4, 128),
                                                      (12, 2, 128), (8, 2, 64)])
            ctx_hi, nodes_hi = _log_int(rng, 1, 32000), _log_int(rng, 1, 130)
            case = dict(op=op, batch=_log_int(rng, 1, 96), ctx_lo=rng.choice([0, ctx_hi // 2, ctx_hi]), ctx_hi=ctx_hi,
                        nodes_lo=rng.choice([1, nodes_hi]), nodes_hi=nodes_hi, q_heads=q_heads, kv_heads=kv_heads,
                        head_dim=head_dim, page_tokens=rng.choice([16, 64, 64, 128]),
                        window=rng.choice([0, 0, 0, 48, _log_int(rng, 16, 4096)]), lengths=rng.randrange(1 << 20))
        else:
            case = dict(op=op, rows=_log_int(rng, 1, 2048), vocab=rng.choice([1000, 1024, 32001, 128256, 151936, 152064,
                                                                              _log_int(rng, 1, 200000)]),
                        dtype=rng.choice(["bf16", "f32"]), top=rng.choice([0, 1, 5, 20, 32]))
        top = max((c for c in listed() if c["op"] == op), key=_cost)
        if _cost(case) <= _cost(top) and work(case)["bytes"] <= work(top)["bytes"]:
            return case


def _lengths(case):
    """(cached positions, new tokens) of each sequence of a ragged batch."""
    rng = random.Random(case["lengths"])
    if case["op"] == "slots":
        lo, hi, nlo, nhi = case["cached_lo"], case["cached_hi"], case["new_lo"], case["new_hi"]
    else:
        lo, hi, nlo, nhi = case["ctx_lo"], case["ctx_hi"], case["nodes_lo"], case["nodes_hi"]
    return ([rng.randint(lo, hi) for _ in range(case["batch"])], [rng.randint(nlo, nhi) for _ in range(case["batch"])])


def _cost(case):
    """What the plain form pads a case to (a bound on its time and memory)."""
    if case["op"] == "slots":
        return case["batch"] * (case["new_hi"] + 64 + case["cached_hi"] // case["page_tokens"])
    if case["op"] == "qk":
        return case["tokens"] * (case["q_heads"] + 2 * case["kv_heads"]) * case["head_dim"] * (2 if case["dtype"] == "f32" else 1)
    if case["op"] == "tree":
        return case["batch"] * (case["ctx_hi"] + case["nodes_hi"]) * case["q_heads"] * case["nodes_hi"] * case["head_dim"]
    return case["rows"] * case["vocab"] * (4 if case["dtype"] == "f32" else 2)


def work(case):
    """Bytes and operations one pass cannot do without."""
    if case["op"] == "slots":
        cached, new = _lengths(case)
        pt = case["page_tokens"]
        pages = sum(-(-(c + n) // pt) - -(-c // pt) for c, n in zip(cached, new))
        return {"bytes": 12 * sum(new) + 8 * pages + 20 * case["batch"] + 16, "flops": 0}
    if case["op"] == "qk":
        t, d = case["tokens"], case["head_dim"]
        e, k = (2 if case["dtype"] == "bf16" else 4), (2 if case["kv_dtype"] == "bf16" else 4)
        heads = case["q_heads"] + 2 * case["kv_heads"]
        return {"bytes": t * (heads * d * e + case["q_heads"] * d * e + 2 * case["kv_heads"] * d * k + 8
                              + case["rotary_dim"] * 4),
                "flops": t * heads * d * 6}
    if case["op"] == "tree":
        ctx, nodes = _lengths(case)
        window, d = case["window"], case["head_dim"]
        kept = [min(c, window) if window else c for c in ctx]
        keys = sum(c + n for c, n in zip(kept, nodes))
        rows = sum(nodes)
        # Half of a tree's node pairs at most are ancestor and descendant; counted as half.
        pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(kept, nodes))
        return {"bytes": keys * case["kv_heads"] * d * 4 + 2 * rows * case["q_heads"] * d * 2,
                "flops": 4 * d * case["q_heads"] * pairs}
    e = 2 if case["dtype"] == "bf16" else 4
    return {"bytes": case["rows"] * (case["vocab"] * e + 16 + 8 * case["top"]), "flops": 5 * case["rows"] * case["vocab"]}


# ---- inputs -----------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    return {"slots": _prepare_slots, "qk": _prepare_qk, "tree": _prepare_tree, "logprobs": _prepare_logprobs}[case["op"]](case, seed)


def _int32(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


def _page_table(gen, pages_of, width, num_pages):
    """Shuffled distinct pages of each sequence, -1 behind them; and the pages left."""
    order = torch.randperm(num_pages, device="cuda", generator=gen).to(torch.int32)
    counts = torch.tensor(pages_of, device="cuda")
    starts = torch.cumsum(counts, 0) - counts
    col = torch.arange(width, device="cuda")
    at = (starts[:, None] + col[None, :]).clamp(max=num_pages - 1)
    table = torch.where(col[None, :] < counts[:, None], order[at], torch.full_like(order[at], -1))
    return table.contiguous(), order[sum(pages_of):].contiguous()


def _prepare_slots(case, seed):
    cached, new = _lengths(case)
    pt = case["page_tokens"]
    have = [-(-c // pt) for c in cached]
    need = sum(-(-(c + n) // pt) for c, n in zip(cached, new)) - sum(have)
    width = -(-(case["cached_hi"] + case["new_hi"]) // pt)
    num_pages = sum(have) + need + 5
    table, free = _page_table(_gen(seed), have, width, num_pages)
    return dict(op="slots", cached=_int32(cached), new=_int32(new), free=free, free_count=_int32([free.numel()]),
                table=table, num_pages=num_pages, page_tokens=pt, max_tokens=sum(new))


def _rope(positions, rotary_dim, theta=1e6):
    freq = theta ** (-torch.arange(0, rotary_dim, 2, device="cuda", dtype=torch.float64) / rotary_dim)
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * freq
    return angle.cos().float().contiguous(), angle.sin().float().contiguous()


def _prepare_qk(case, seed):
    g = _gen(seed)
    t, qh, kh, d, pt = case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"], case["page_tokens"]
    qkv = (torch.randn(t, qh + 2 * kh, d, device="cuda", generator=g) * 2.0).to(DTYPES[case["dtype"]])
    num_pages = -(-t // pt) + 2
    pools = [torch.randn(num_pages, kh, pt, d, device="cuda", generator=g).to(DTYPES[case["kv_dtype"]]) for _ in range(2)]
    # Cells in page order of a shuffled page list, as a sequence's tokens take them.
    pages = torch.randperm(num_pages, device="cuda", generator=g)
    at = torch.arange(t, device="cuda")
    cos, sin = _rope(4096, case["rotary_dim"])
    weight = lambda: 1.0 + 0.2 * torch.randn(d, device="cuda", generator=g) if case["norm"] else None  # noqa: E731
    return dict(op="qk", qkv=qkv, q_heads=qh, kv_heads=kh, positions=(torch.randint(0, 4096, (t,), device="cuda", generator=g)).to(torch.int32),
                slots=(pages[at // pt] * pt + at % pt).to(torch.int32), cos=cos, sin=sin, k_pool=pools[0], v_pool=pools[1],
                q_norm=weight(), k_norm=weight(), eps=1e-6)


def _prepare_tree(case, seed):
    g = _gen(seed)
    rng = np.random.default_rng(seed)
    ctx, nodes = _lengths(case)
    pt, qh, kh, d, n_max = case["page_tokens"], case["q_heads"], case["kv_heads"], case["head_dim"], max(nodes)
    pages_of = [-(-(c + n) // pt) for c, n in zip(ctx, nodes)]
    num_pages = sum(pages_of) + 3
    table, _ = _page_table(g, pages_of, max(pages_of), num_pages)
    pools = [torch.randn(num_pages, kh, pt, d, device="cuda", generator=g, dtype=torch.bfloat16) for _ in range(2)]
    # Random trees: node i hangs below an earlier node or the context; its mask
    # row holds its ancestors and itself, 64 to a word.
    words = -(-n_max // 64)
    seen = np.zeros((len(nodes), n_max, n_max), dtype=bool)
    depth = np.zeros((len(nodes), n_max), dtype=np.int64)
    at = np.arange(len(nodes))
    for i in range(n_max):
        parent = rng.integers(-1, max(i, 1), len(nodes)) if i else np.full(len(nodes), -1)
        seen[:, i] = np.where(parent[:, None] >= 0, seen[at, parent], False)
        depth[:, i] = np.where(parent >= 0, depth[at, parent] + 1, 0)
        seen[:, i, i] = True
    live = np.arange(n_max)[None, :] < np.array(nodes)[:, None]
    rows = np.zeros((sum(nodes), words * 64), dtype=bool)
    rows[:, :n_max] = seen[live]
    mask = np.packbits(rows, axis=1, bitorder="little").view(np.int64)
    positions = (depth + np.array(ctx)[:, None])[live]
    q = (torch.randn(sum(nodes), qh, d, device="cuda", generator=g) * 1.5).to(torch.bfloat16)
    return dict(op="tree", q=q, k_pool=pools[0], v_pool=pools[1], table=table, seq_lens=_int32([c + n for c, n in zip(ctx, nodes)]),
                row_starts=_int32(np.concatenate([[0], np.cumsum(nodes)])), mask=torch.from_numpy(mask).cuda(),
                positions=_int32(positions), window=case["window"], longest=max(c + n for c, n in zip(ctx, nodes)), most=n_max)


def _prepare_logprobs(case, seed):
    g = _gen(seed)
    x = torch.randn(case["rows"], case["vocab"], device="cuda", generator=g)
    # A few likely tokens above the rest, as a trained model's rows have them.
    hot = torch.randint(0, case["vocab"], (case["rows"], 12), device="cuda", generator=g)
    x = (2.0 * x).scatter_add_(1, hot, 12.0 * torch.rand(case["rows"], 12, device="cuda", generator=g))
    tokens = torch.where(torch.rand(case["rows"], device="cuda", generator=g) < 0.7, hot[:, 0],
                         torch.randint(0, case["vocab"], (case["rows"],), device="cuda", generator=g))
    return dict(op="logprobs", logits=x.to(DTYPES[case["dtype"]]), tokens=tokens.to(torch.int32), top=min(case["top"], case["vocab"]))


# ---- one pass ---------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    return {"slots": _plain_slots, "qk": _plain_qk, "tree": _plain_tree, "logprobs": _plain_logprobs}[state["op"]](state)


def _run_own(s):
    from cheetah_b200 import runtime as R
    if s["op"] == "slots":
        r = R.page_slots(s["cached"], s["new"], s["free"], s["free_count"], s["table"], s["num_pages"], s["page_tokens"],
                         s["max_tokens"])
        return dict(table=s["table"], row_starts=r.row_starts, seq_lens=r.seq_lens, positions=r.positions,
                    seq_ids=r.seq_ids, slots=r.slots, counts=r.counts)
    if s["op"] == "qk":
        q = R.qk_norm_rope(s["qkv"], s["q_heads"], s["kv_heads"], s["positions"], s["slots"], s["cos"], s["sin"],
                           s["k_pool"], s["v_pool"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=s["eps"])
        return dict(q=q, k_pool=s["k_pool"], v_pool=s["v_pool"])
    if s["op"] == "tree":
        return R.tree_attention(s["q"], s["k_pool"], s["v_pool"], s["table"], s["seq_lens"], s["row_starts"], s["mask"],
                                positions=s["positions"], sliding_window=s["window"])
    r = R.token_logprobs(s["logits"], s["tokens"], top=s["top"])
    out = dict(logprob=r.logprob, entropy=r.entropy, rank=r.rank)
    return dict(out, top_ids=r.top_ids, top_logprobs=r.top_logprobs) if s["top"] else out


def _plain_slots(s):
    pt, width, most = s["page_tokens"], s["table"].shape[1], s["max_tokens"]
    cached, new = s["cached"].long(), s["new"].long()
    fits = (cached >= 0) & (new >= 0) & (cached + new <= width * pt)
    n = torch.where(fits, new, 0)
    ends = torch.cumsum(n, 0)
    fits = fits & (ends <= most)
    have = torch.div(cached + pt - 1, pt, rounding_mode="floor")
    need = torch.where(fits, torch.div(cached + n + pt - 1, pt, rounding_mode="floor") - have, 0)
    taken = torch.cumsum(need, 0)
    got = fits & ((need == 0) | (taken <= s["free_count"]))
    col = torch.arange(width, device="cuda")
    fresh = got[:, None] & (col >= have[:, None]) & (col < (have + need)[:, None])
    at = (taken - need - have)[:, None] + col
    table = torch.where(fresh, s["free"][at.clamp(0, max(0, s["free"].numel() - 1))], s["table"])
    t = torch.arange(most, device="cuda")
    seq = torch.searchsorted(ends, t, right=True)
    live = seq < ends.numel()
    b = seq.clamp(max=ends.numel() - 1)
    live = live & got[b]
    pos = cached[b] + t - (ends - n)[b]
    page = table[b, torch.div(pos, pt, rounding_mode="floor").clamp(0, width - 1)].long()
    good = live & (page >= 0) & (page < s["num_pages"])
    counts = torch.stack([ends[-1], torch.where(got, need, 0).sum(), (~got).sum()])
    i32 = lambda x: x.to(torch.int32)  # noqa: E731
    return dict(table=table, row_starts=i32(torch.cat([ends.new_zeros(1), ends]).clamp(max=most)),
                seq_lens=i32(torch.where(got, cached + n, 0)), positions=i32(torch.where(live, pos, -1)),
                seq_ids=i32(torch.where(seq < ends.numel(), seq, -1)), slots=i32(torch.where(good, page * pt + pos % pt, -1)), counts=i32(counts))


def _normed(x, weight, eps):
    return x if weight is None else x * (torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight.to(x.dtype))


def _rotated(x, cos, sin):
    half = cos.shape[-1]
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _plain_qk(s):
    qh, kh, pt = s["q_heads"], s["kv_heads"], s["k_pool"].shape[2]
    x = s["qkv"].float()
    cos, sin = s["cos"][s["positions"].long()][:, None], s["sin"][s["positions"].long()][:, None]
    q = _rotated(_normed(x[:, :qh], s["q_norm"], s["eps"]), cos, sin)
    k = _rotated(_normed(x[:, qh:qh + kh], s["k_norm"], s["eps"]), cos, sin)
    page, cell = s["slots"].long() // pt, s["slots"].long() % pt
    s["k_pool"][page, :, cell] = k.to(s["k_pool"].dtype)
    s["v_pool"][page, :, cell] = x[:, qh + kh:].to(s["v_pool"].dtype)
    return dict(q=q.to(s["qkv"].dtype), k_pool=s["k_pool"], v_pool=s["v_pool"])


def _plain_tree(s):
    total, qh, d = s["q"].shape
    kh, pt = s["k_pool"].shape[1:3]
    batch, longest, most = s["table"].shape[0], s["longest"], s["most"]
    starts = s["row_starts"].long()
    nodes = starts[1:] - starts[:-1]
    ctx = s["seq_lens"].long() - nodes
    key = torch.arange(longest, device="cuda")
    page = s["table"].long()[:, key // pt].clamp(min=0)
    k = s["k_pool"][page, :, key % pt].float().transpose(1, 2)  # [batch, kv_heads, longest, d]
    v = s["v_pool"][page, :, key % pt].float().transpose(1, 2)
    i = torch.arange(most, device="cuda")
    row = (starts[:-1, None] + i).clamp(max=total - 1)
    q = s["q"][row].float().reshape(batch, most, kh, qh // kh, d).permute(0, 2, 3, 1, 4).reshape(batch, kh, -1, d)
    # Key j of row i: a context position, or node j - ctx when its bit is set.
    node = key[None, :] - ctx[:, None]
    word = s["mask"][row]
    at = node.clamp(0, 64 * word.shape[-1] - 1)[:, None, :].expand(-1, most, -1)
    bit = (torch.gather(word, 2, at // 64) >> (at % 64)) & 1
    seen = (node < 0)[:, None, :] | ((node < nodes[:, None])[:, None, :] & (bit == 1))
    if s["window"]:
        pos = s["positions"].long()[row]
        mine = s["positions"].long()[(starts[:-1, None] + node.clamp(min=0)).clamp(max=total - 1)]
        where = torch.where(node < 0, key[None, :], mine)
        seen = seen & (where[:, None, :] + s["window"] > pos[:, :, None])
    seen = seen[:, None, None]
    score = (q @ k.transpose(2, 3)).reshape(batch, kh, qh // kh, most, longest) / math.sqrt(d)
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total_e = e.sum(-1, keepdim=True)
    p = (e / torch.where(total_e > 0, total_e, 1.0)).reshape(batch, kh, -1, longest)
    v = torch.where((key[None, :] < s["seq_lens"][:, None])[:, None, :, None], v, 0.0)
    o = (p @ v).reshape(batch, kh, qh // kh, most, d).permute(0, 3, 1, 2, 4).reshape(batch, most, qh, d)
    t = torch.arange(total, device="cuda")
    b = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    return o[b, t - starts[b]].to(torch.bfloat16)


def _plain_logprobs(s):
    x = s["logits"].float()
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    lse = m + torch.log(total)
    chosen = torch.gather(x, 1, s["tokens"].long()[:, None])
    gap = torch.where(e > 0, (m - x) * e, 0.0).sum(-1)
    out = dict(logprob=(chosen - lse)[:, 0], entropy=torch.log(total[:, 0]) + gap / total[:, 0],
               rank=(1 + (x > chosen).sum(-1)).to(torch.int32))
    if s["top"]:
        value, index = torch.sort(x, dim=-1, descending=True, stable=True)
        out.update(top_ids=index[:, :s["top"]].to(torch.int32), top_logprobs=value[:, :s["top"]] - lse)
    return out


# ---- the definitions in 64 bits ----------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "slots":
        return None
    return {"qk": _exact_qk, "tree": _exact_tree, "logprobs": _exact_logprobs}[case["op"]](s)


def _exact_qk(s):
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

    q = torch.stack([head(h, s["q_norm"]) for h in range(qh)], 1)
    k_pool, v_pool = s["k_pool"].double(), s["v_pool"].double()
    pt = k_pool.shape[2]
    page, cell = s["slots"].long() // pt, s["slots"].long() % pt
    for h in range(kh):
        k_pool[page, h, cell] = head(qh + h, s["k_norm"])
        v_pool[page, h, cell] = x[:, qh + kh + h]
    return dict(q=q, k_pool=k_pool, v_pool=v_pool)


def _exact_tree(s):
    total, qh, d = s["q"].shape
    kh, pt = s["k_pool"].shape[1:3]
    starts, lens = s["row_starts"].tolist(), s["seq_lens"].tolist()
    out = torch.zeros(total, qh, d, dtype=torch.float64, device="cuda")
    for b, length in enumerate(lens):
        r0, r1 = starts[b], starts[b + 1]
        n = r1 - r0
        c = length - n
        pages = s["table"][b, :-(-length // pt)].long()
        k = s["k_pool"][pages].double().transpose(1, 2).reshape(-1, kh, d)[:length]
        v = s["v_pool"][pages].double().transpose(1, 2).reshape(-1, kh, d)[:length]
        j = torch.arange(n, device="cuda")
        seen = torch.ones(n, length, dtype=torch.bool, device="cuda")
        seen[:, c:] = ((s["mask"][r0:r1][:, j // 64] >> (j % 64)) & 1).bool()
        if s["window"]:
            where = torch.arange(length, device="cuda")
            where[c:] = s["positions"][r0:r1].long()
            seen &= where[None, :] > s["positions"][r0:r1].long()[:, None] - s["window"]
        for h in range(qh):
            a = (s["q"][r0:r1, h].double() @ k[:, h * kh // qh].T / math.sqrt(d)).masked_fill(~seen, -math.inf)
            p = torch.softmax(a, -1).nan_to_num(0.0)
            out[r0:r1, h] = p @ v[:, h * kh // qh]
    return out


def _exact_logprobs(s):
    parts = []
    for r in range(0, s["logits"].shape[0], 256):
        x = s["logits"][r:r + 256].double()
        t = s["tokens"][r:r + 256].long()[:, None]
        lp = torch.log_softmax(x, -1)
        part = dict(logprob=lp.gather(1, t)[:, 0], entropy=-(lp.exp() * lp).nan_to_num(0.0).sum(-1))
        if s["top"]:
            part["top_logprobs"] = lp.topk(s["top"], -1).values
        parts.append(part)
    out = {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
    out["rank"] = None
    if s["top"]:
        out["top_ids"] = None
    return out
