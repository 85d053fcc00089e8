"""The drafted-token operators on the GPU against 64-bit references
(`tests/verify_ref.py`), at the sizes, masks and values where they can go
wrong, and a run of all four as a verification step uses them."""

import math

import numpy as np
import pytest

from tests import verify_ref as V

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from cheetah_b200 import runtime
    runtime.lib()


def i32(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


# ---- page_slots ---------------------------------------------------------------

def _slots_case(cached, new, width, page_tokens, seed=0, free=None, free_count=None, max_tokens=None, num_pages=None, stale=False):
    rng = np.random.default_rng(seed)
    num_pages = num_pages or 4 * len(cached) * width + 8
    ids = rng.permutation(num_pages)
    table = ids[:len(cached) * width].reshape(len(cached), width).copy()
    if stale:
        table[:, ::2] = num_pages + 7  # ids outside the pool
    have = [-(-max(c, 0) // page_tokens) for c in cached]
    need = sum(max(0, -(-(max(c, 0) + max(n, 0)) // page_tokens) - h) for c, n, h in zip(cached, new, have))
    free = list(ids[len(cached) * width:][:need + 2]) if free is None else free
    free_count = len(free) if free_count is None else free_count
    max_tokens = max_tokens or max(1, sum(max(n, 0) for n in new)) + 5
    return dict(cached=list(cached), new=list(new), free=[int(f) for f in free], free_count=free_count, table=table,
                num_pages=num_pages, page_tokens=page_tokens, max_tokens=max_tokens)


def _check_slots(case):
    from cheetah_b200 import runtime as R
    table = i32(case["table"])
    args = (i32(case["cached"]), i32(case["new"]), i32(case["free"]), i32([case["free_count"]]), table,
            case["num_pages"], case["page_tokens"], case["max_tokens"])
    want = V.page_slots(**case)
    for _ in range(2):  # the same call again gives the same result
        got = R.page_slots(*args)
        for name in ("row_starts", "seq_lens", "positions", "seq_ids", "slots", "counts"):
            np.testing.assert_array_equal(getattr(got, name).cpu().numpy(), np.array(want[name]), err_msg=name)
        np.testing.assert_array_equal(table.cpu().numpy(), want["table"])
    return want


@pytest.mark.parametrize("batch,page_tokens,most", [(1, 16, 1), (1, 64, 5000), (3, 1, 9), (31, 64, 17), (64, 48, 200),
                                                    (511, 16, 3), (513, 16, 40), (2049, 128, 5), (16384, 16, 2)])
def test_page_slots_random(batch, page_tokens, most):
    rng = np.random.default_rng(batch + most)
    cached, new = rng.integers(0, 300, batch), rng.integers(0, most + 1, batch)
    _check_slots(_slots_case(cached.tolist(), new.tolist(), -(-(300 + most) // page_tokens), page_tokens, seed=batch))


@pytest.mark.parametrize("name,cached,new,more", [
    ("nothing new", [0, 16, 17], [0, 0, 0], {}),
    ("empty cache", [0, 0], [1, 33], {}),
    ("page borders", [15, 16, 17, 31], [1, 1, 1, 2], {}),
    ("negative lengths", [-1, 5, 5], [3, -2, 4], {}),
    ("past the table", [60, 3, 64, 64], [5, 4, 0, 1], {}),
    ("lengths near 2^31", [2 ** 31 - 1, 1, 2 ** 31 - 1], [2 ** 31 - 1, 2, 0], dict(max_tokens=20)),
    ("free list too short", [0, 10, 0, 16], [20, 3, 17, 9], dict(free=[3, 1, 2])),
    ("free list empty", [0, 10], [1, 3], dict(free=[], free_count=0)),
    ("free count above the list", [0, 0], [16, 17], dict(free=[3, 1], free_count=9)),
    ("free count below the list", [0, 0], [16, 17], dict(free=[3, 1, 5], free_count=1)),
    ("negative free count", [0, 0], [16, 0], dict(free=[3, 1, 5], free_count=-4)),
    ("rows past max_tokens", [0, 5, 0], [10, 10, 10], dict(max_tokens=15)),
    ("page ids outside the pool", [5, 40], [20, 30], dict(stale=True, num_pages=64)),
    ("free ids outside the pool", [0, 0], [16, 16], dict(free=[-1, 1 << 30])),
])
def test_page_slots_edges(name, cached, new, more):
    _check_slots(_slots_case(cached, new, 4, 16, **more))


def test_page_slots_from_two_threads():
    """Host threads whose batches need different amounts of shared memory call
    at the same time (straight through the C-ABI, which runs without Python's
    lock): neither call depends on what the other one asked for."""
    import threading
    from cheetah_b200 import runtime as R
    call, failed = R.lib().cheetah_cuda_op_page_slots, []

    def calls(batch):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            cached, new, table = i32([3] * batch), i32([1] * batch), torch.zeros(batch, 1, dtype=torch.int32, device="cuda")
            free, free_count = i32(range(4)), i32([4])
            outs = [torch.empty(n, dtype=torch.int32, device="cuda") for n in (batch + 1, batch, batch, batch, batch, 3)]
        args = R.PageSlotsArgs(cached.data_ptr(), new.data_ptr(), free.data_ptr(), free_count.data_ptr(), 4, batch,
                               table.data_ptr(), 1, 8, 16, batch, *[o.data_ptr() for o in outs])
        for _ in range(20000):
            if call(args, stream.cuda_stream):
                failed.append((batch, R.lib().cheetah_cuda_last_error()))
                break
        stream.synchronize()
        if outs[5].tolist() != [batch, 0, 0] or not bool((outs[2] == 3).all()):
            failed.append((batch, "wrong rows"))
    threads = [threading.Thread(target=calls, args=(batch,)) for batch in (4200, 16384)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


# ---- qk_norm_rope -------------------------------------------------------------

@pytest.mark.parametrize("q_heads,kv_heads,D,rotary", [(14, 2, 64, 64), (28, 4, 128, 128), (4, 4, 64, 32), (3, 1, 128, 16),
                                                       (8, 4, 128, 96)])
@pytest.mark.parametrize("dtype,kv_dtype", [("bf16", "bf16"), ("f32", "bf16"), ("f32", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("tokens,norm", [(1, True), (7, False), (131, True)])
def test_qk_norm_rope(q_heads, kv_heads, D, rotary, dtype, kv_dtype, tokens, norm):
    from cheetah_b200 import runtime as R
    types = {"bf16": torch.bfloat16, "f32": torch.float32}
    g = torch.Generator().manual_seed(tokens + D + rotary)
    heads, pt, pages, max_pos = q_heads + 2 * kv_heads, 16, 12, 50
    wide = torch.randn(tokens, heads * D + 16, generator=g).to(types[dtype])  # rows lie apart
    x = wide[:, :heads * D]
    slots = torch.randperm(pages * pt, generator=g)[:tokens].to(torch.int32)
    positions = torch.randint(0, max_pos, (tokens,), generator=g).to(torch.int32)
    if tokens > 3:
        slots[1], slots[2], positions[3], positions[4] = -1, pages * pt, -1, max_pos
    angle = torch.rand(max_pos, rotary // 2, generator=g) * 6.0
    cos, sin = angle.cos(), angle.sin()
    w = [1.0 + 0.3 * torch.randn(D, generator=g) if norm else None for _ in range(2)]
    pools = [torch.randn(pages, kv_heads, pt, D, generator=g).to(types[kv_dtype]) for _ in range(2)]
    k_pool, v_pool = pools[0].cuda(), pools[1].cuda()
    q_out = torch.full((tokens, q_heads, D), 7.0, dtype=types[dtype], device="cuda")
    got = R.qk_norm_rope(wide.cuda()[:, :heads * D], q_heads, kv_heads, positions.cuda(), slots.cuda(), cos.cuda(), sin.cuda(),
                         k_pool, v_pool, q_norm=w[0].cuda() if norm else None, k_norm=w[1].cuda() if norm else None,
                         eps=1e-5, q_out=q_out)
    assert got is q_out
    # Sum of squares: D roundings, halved by the square root; then a handful.
    f32 = (D / 2 + 10) * 2.0 ** -24
    step = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}
    want_k, want_v = pools[0].double(), pools[1].clone()
    tol_k = torch.zeros_like(want_k)
    q, k_got = got.cpu().double(), k_pool.cpu().double()
    for t in range(tokens):
        p, s = int(positions[t]), int(slots[t])
        if not 0 <= p < max_pos:
            assert bool((q[t] == 7.0).all())
            continue
        row = x[t].reshape(heads, D)
        for h in range(q_heads):
            z, mag = V.norm_rope_head(row[h], w[0], 1e-5, cos[p], sin[p])
            assert bool(((q[t, h] - z).abs() <= mag * f32 + z.abs() * step[dtype] + 1e-30).all()), (t, h)
        if not 0 <= s < pages * pt:
            continue
        for h in range(kv_heads):
            z, mag = V.norm_rope_head(row[q_heads + h], w[1], 1e-5, cos[p], sin[p])
            want_k[s // pt, h, s % pt] = z
            tol_k[s // pt, h, s % pt] = mag * f32 + z.abs() * step[kv_dtype] + 1e-30
            want_v[s // pt, h, s % pt] = row[q_heads + kv_heads + h].to(types[kv_dtype])
    assert bool(((k_got - want_k).abs() <= tol_k).all())  # cells not named: unchanged
    assert torch.equal(v_pool.cpu(), want_v)


@pytest.mark.parametrize("q_heads,kv_heads,D,rotary,dtype,kv_dtype,tokens", [
    (14, 2, 64, 64, "bf16", "bf16", 2501), (28, 4, 128, 128, "bf16", "bf16", 901), (14, 2, 64, 32, "f32", "bf16", 1503),
    (4, 1, 128, 128, "f32", "f32", 2407), (3, 1, 64, 64, "bf16", "f32", 7205), (32, 8, 64, 64, "bf16", "bf16", 1301)])
def test_qk_norm_rope_rows_that_a_warp_walks_over(q_heads, kv_heads, D, rotary, dtype, kv_dtype, tokens):
    """So many rows that a warp takes all heads of one, up to three groups of
    them and more; some rows are skipped and some append nothing."""
    from cheetah_b200 import runtime as R
    types = {"bf16": torch.bfloat16, "f32": torch.float32}
    g = torch.Generator(device="cuda").manual_seed(tokens)
    heads, pt, max_pos = q_heads + 2 * kv_heads, 16, 70
    pages = -(-tokens // pt) + 2
    x = torch.randn(tokens, heads, D, generator=g, device="cuda").to(types[dtype])
    slots = torch.randperm(pages * pt, generator=g, device="cuda")[:tokens].to(torch.int32)
    positions = torch.randint(0, max_pos, (tokens,), generator=g, device="cuda").to(torch.int32)
    positions[::7], slots[::5] = -1, pages * pt
    angle = torch.rand(max_pos, rotary // 2, generator=g, device="cuda") * 6.0
    cos, sin = angle.cos(), angle.sin()
    w = [1.0 + 0.3 * torch.randn(D, generator=g, device="cuda") for _ in range(2)]
    pools = [torch.randn(pages, kv_heads, pt, D, generator=g, device="cuda").to(types[kv_dtype]) for _ in range(2)]
    k_pool, v_pool = pools[0].clone(), pools[1].clone()
    q_out = torch.full((tokens, q_heads, D), 7.0, dtype=types[dtype], device="cuda")
    R.qk_norm_rope(x, q_heads, kv_heads, positions, slots, cos, sin, k_pool, v_pool, q_norm=w[0], k_norm=w[1], eps=1e-5, q_out=q_out)

    # The formula in 64 bits, and the magnitudes that its last addition joins.
    at = positions.long().clamp(min=0)
    c, s = cos.double()[at][:, None], sin.double()[at][:, None]
    y = x[:, :q_heads + kv_heads].double()
    weight = torch.cat([w[0].expand(q_heads, D), w[1].expand(kv_heads, D)]).double()
    y = y * (weight / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-5))
    half = rotary // 2
    z, mag = y.clone(), y.abs()
    a, b = y[..., :half], y[..., half:rotary]
    z[..., :half], z[..., half:rotary] = a * c - b * s, b * c + a * s
    mag[..., :half], mag[..., half:rotary] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    f32 = (D / 2 + 10) * 2.0 ** -24
    step = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}
    live = positions >= 0
    q, zq = q_out.double(), z[:, :q_heads]
    assert bool(((q - zq).abs() <= mag[:, :q_heads] * f32 + zq.abs() * step[dtype] + 1e-30)[live].all())
    assert bool((q[~live] == 7.0).all())
    kept = live & (slots < pages * pt)
    page, cell = slots[kept].long() // pt, slots[kept].long() % pt
    zk, mk = z[kept, q_heads:], mag[kept, q_heads:]
    assert bool(((k_pool[page, :, cell].double() - zk).abs() <= mk * f32 + zk.abs() * step[kv_dtype] + 1e-30).all())
    pools[0][page, :, cell] = k_pool[page, :, cell]
    pools[1][page, :, cell] = x[kept, q_heads + kv_heads:].to(types[kv_dtype])
    assert torch.equal(k_pool, pools[0]) and torch.equal(v_pool, pools[1])  # cells not named: unchanged

def test_qk_norm_rope_large_values_and_zero_rows():
    """A zero row stays zero, values near the type's limits keep their scale,
    a non-finite value stays in its own head."""
    from cheetah_b200 import runtime as R
    D, pt = 64, 16
    x = torch.zeros(4, 3, D)
    x[1] = 1e18  # squares reach 1e36
    x[2] = 1e-18
    x[3, 0, 5] = math.inf
    x[3, 1:] = 1.0
    one = torch.ones(2, D // 2)
    k, v = torch.zeros(2, 1, pt, D, device="cuda"), torch.zeros(2, 1, pt, D, device="cuda")
    w = torch.ones(D, device="cuda")
    q = R.qk_norm_rope(x.cuda(), 1, 1, i32([0, 0, 0, 0]), i32([0, 1, 2, 3]), one.cuda(), torch.zeros(2, D // 2, device="cuda"),
                       k, v, q_norm=w, k_norm=w, eps=1e-6).cpu()
    assert bool((q[0] == 0).all()) and torch.allclose(q[1], torch.ones(1, D), rtol=1e-5)
    assert torch.allclose(q[2].double(), torch.full((1, D), 1e-15, dtype=torch.float64), rtol=1e-4)
    assert torch.isnan(q[3, 0, 5]) and torch.allclose(k[0, 0, 3].cpu(), torch.ones(D), rtol=1e-5)
    assert bool((v[0, 0, 3] == 1).all())


# ---- tree_attention -----------------------------------------------------------

class Tree:
    """A batch of random trees over a shuffled paged pool, and its reference."""

    def __init__(self, ctx, nodes, q_heads, kv_heads, D, page_tokens=64, window=0, seed=0, words=None, masks=None,
                 scale=1.0, extra_rows=0, fill=float("nan"), width=None):
        rng = np.random.default_rng(seed)
        g = torch.Generator().manual_seed(seed)
        self.window, self.kv_heads, self.group = window, kv_heads, q_heads // kv_heads
        self.ctx, self.nodes = ctx, nodes
        lens = [c + n for c, n in zip(ctx, nodes)]
        per = [-(-n // page_tokens) for n in lens]
        pages = sum(per) + 2
        order = rng.permutation(pages)
        self.table = np.full((len(ctx), width or max(max(per), 1)), -1, np.int32)
        # Cells that hold no position are NaN (a fresh pool holds anything).
        kp = torch.full((pages, kv_heads, page_tokens, D), fill)
        vp = torch.full_like(kp, fill)
        self.k, self.v = [], []
        cursor = 0
        for b, n in enumerate(lens):
            k = torch.randn(n, kv_heads, D, generator=g).bfloat16()
            v = torch.randn(n, kv_heads, D, generator=g).bfloat16()
            for p in range(per[b]):
                page = int(order[cursor])
                cursor += 1
                if p < self.table.shape[1]:
                    self.table[b, p] = page
                lo, hi = p * page_tokens, min(n, (p + 1) * page_tokens)
                kp[page, :, :hi - lo] = k[lo:hi].transpose(0, 1).float()
                vp[page, :, :hi - lo] = v[lo:hi].transpose(0, 1).float()
            self.k.append(k.double())
            self.v.append(v.double())
        self.starts = np.concatenate([[0], np.cumsum(nodes)])
        total = int(self.starts[-1])
        self.rows = max(1, total + extra_rows)
        words = words or max(1, -(-max(nodes + [1]) // 64))
        self.seen, depth = [], []
        for b, n in enumerate(nodes):
            bits, d = V.tree_bits(V.random_tree(rng, n))
            if masks is not None:
                bits = masks(rng, n)
            self.seen.append(bits)
            depth.append(d + ctx[b])
        self.positions = np.concatenate(depth + [np.full(self.rows - total, -1)]).astype(np.int64)
        mask = np.zeros((self.rows, words), np.int64)
        for b, bits in enumerate(self.seen):
            if nodes[b]:
                mask[self.starts[b]:self.starts[b + 1]] = V.pack_bits(bits, words)
        self.words, self.mask = words, mask
        self.q = (torch.randn(self.rows, q_heads, D, generator=g) * scale).bfloat16()
        self.dev = dict(q=self.q.cuda(), k_pool=kp.bfloat16().cuda(), v_pool=vp.bfloat16().cuda(), page_table=i32(self.table),
                        seq_lens=i32(lens), row_starts=i32(self.starts), tree_mask=torch.from_numpy(mask).cuda(),
                        positions=i32(self.positions), sliding_window=window)

    def run(self, **more):
        from cheetah_b200 import runtime as R
        return R.tree_attention(**{**self.dev, **more})

    def visible(self, b, i):
        n, c = self.nodes[b], self.ctx[b]
        seen = np.ones(c + n, bool)
        bits = np.zeros(n, bool)
        w = min(n, 64 * self.words)
        bits[:w] = self.seen[b][i][:w]
        seen[c:] = bits
        if self.window:
            where = np.arange(c + n)
            where[c:] = self.positions[self.starts[b]:self.starts[b + 1]]
            seen &= where > self.positions[self.starts[b] + i] - self.window
        return torch.from_numpy(seen)

    def check(self, out, rows=None):
        out = out.cpu().double()
        rng = np.random.default_rng(1)
        for b, n in enumerate(self.nodes):
            picked = range(n) if n <= 6 else sorted(set([0, 1, n - 1, n // 2]) | set(rng.integers(0, n, 3).tolist()))
            for i in picked:
                seen = self.visible(b, i)
                r = int(self.starts[b]) + i
                for h in range(self.q.shape[1]):
                    kvh = h // self.group
                    want, tol = V.tree_row(self.q[r, h].double(), self.k[b][:, kvh], self.v[b][:, kvh], seen)
                    err = (out[r, h] - want).abs()
                    assert bool((err <= tol).all()), f"sequence {b} node {i} head {h}: {float((err - tol).max())} over"


HEADS = [(14, 2, 64), (28, 4, 128), (4, 4, 64), (16, 1, 128), (8, 4, 128), (6, 2, 64)]


@pytest.mark.parametrize("q_heads,kv_heads,D", HEADS)
@pytest.mark.parametrize("ctx,nodes", [
    ([0], [1]), ([0], [8]), ([1], [1]), ([63], [1]), ([64], [3]), ([127], [2]), ([128], [5]), ([300], [17]),
    ([120, 0, 700], [9, 1, 0]), ([1000, 3, 65], [1, 64, 20]), ([2500], [70]),
])
def test_tree_attention(q_heads, kv_heads, D, ctx, nodes):
    case = Tree(ctx, nodes, q_heads, kv_heads, D, seed=sum(ctx) + sum(nodes))
    case.check(case.run())


@pytest.mark.parametrize("page_tokens", [16, 32, 48, 128, 192])
def test_tree_attention_page_sizes(page_tokens):
    case = Tree([333, 90, 0], [13, 40, 130], 14, 2, 64, page_tokens=page_tokens, seed=page_tokens)
    case.check(case.run())
    case = Tree([333, 16], [13, 5], 8, 4, 128, page_tokens=page_tokens, seed=page_tokens)
    case.check(case.run())


@pytest.mark.parametrize("window", [1, 5, 48, 130, 5000])
@pytest.mark.parametrize("D", [64, 128])
def test_tree_attention_window(window, D):
    case = Tree([400, 1, 129], [20, 70, 3], 8, 2, D, window=window, seed=window)
    case.check(case.run())


def test_tree_attention_long_and_wide():
    case = Tree([9000, 20, 4097], [33, 300, 150], 14, 2, 64, seed=3)
    case.check(case.run())
    case = Tree([5000, 1], [130, 257], 28, 4, 128, seed=4)
    case.check(case.run())


def test_tree_attention_as_many_sequences_as_a_call_takes():
    rng = np.random.default_rng(9)
    case = Tree(rng.integers(0, 150, 4096).tolist(), rng.integers(0, 2, 4096).tolist(), 4, 2, 64, page_tokens=16, seed=9)
    case.check(case.run())
    # All but the last without rows.
    case = Tree([3] * 4095 + [200], [0] * 4095 + [5], 4, 2, 128, page_tokens=16, seed=10)
    case.check(case.run())

@pytest.mark.parametrize("q_heads,kv_heads,D", [(17, 1, 64), (24, 1, 128), (31, 1, 128), (32, 1, 64), (64, 2, 128)])
def test_tree_attention_wide_groups(q_heads, kv_heads, D):
    case = Tree([300, 0, 129], [9, 20, 1], q_heads, kv_heads, D, seed=q_heads)
    case.check(case.run())
    case = Tree([130], [11], q_heads, kv_heads, D, window=70, seed=q_heads)
    case.check(case.run())


@pytest.mark.parametrize("q_heads,kv_heads,D,window", [(14, 2, 64, 0), (8, 4, 128, 0), (4, 4, 64, 100)])
def test_tree_attention_as_many_nodes_as_a_mask_holds(q_heads, kv_heads, D, window):
    """1024 nodes of one sequence, as a tree and as a prompt chunk (a chain)."""
    case = Tree([77, 5], [1024, 3], q_heads, kv_heads, D, window=window, seed=41)
    case.check(case.run())
    case = Tree([200], [1000], q_heads, kv_heads, D, seed=42, masks=lambda rng, n: np.tril(np.ones((n, n), bool)))
    case.check(case.run())

def test_tree_attention_many_sequences():
    rng = np.random.default_rng(8)
    case = Tree(rng.integers(0, 200, 300).tolist(), rng.integers(0, 4, 300).tolist(), 14, 2, 64, seed=8)
    case.check(case.run())


def test_tree_attention_rows_that_see_nothing():
    """Empty mask rows over an empty context give zeros; beside them rows that
    see one node, and NaN in every cell that holds no position."""
    def masks(rng, n):
        bits = np.zeros((n, n), bool)
        bits[1::2, 0] = True
        return bits
    case = Tree([0, 0], [7, 90], 14, 2, 64, masks=masks, seed=5)
    out = case.run()
    assert bool((out[0] == 0).all()) and bool((out[2] == 0).all())
    case.check(out)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("D", [64, 128])
def test_tree_attention_non_finite_cells_reach_only_the_rows_that_see_them(value, D):
    """A node's K and V are non-finite: rows that do not see it are as without
    it; and with a window, so is a context key that has left it."""
    case = Tree([140, 50], [12, 9], 8, 2, D, seed=21)
    for b, j in ((0, 3), (1, 2)):
        pos = case.ctx[b] + j
        page, cell = int(case.table[b, pos // 64]), pos % 64
        case.dev["k_pool"][page, :, cell] = value
        case.dev["v_pool"][page, :, cell] = value
    out = case.run()
    for b, j in ((0, 3), (1, 2)):
        for i in range(case.nodes[b]):
            row = out[int(case.starts[b]) + i]
            if case.seen[b][i][j]:
                assert not bool(torch.isfinite(row).all())
            else:
                assert bool(torch.isfinite(row).all())
    clean = Tree([140, 50], [12, 9], 8, 2, D, seed=21).run()
    for b, j in ((0, 3), (1, 2)):
        for i in range(case.nodes[b]):
            if not case.seen[b][i][j]:
                assert torch.equal(out[int(case.starts[b]) + i], clean[int(case.starts[b]) + i])
    case = Tree([140], [12], 8, 2, D, window=30, seed=22)
    want = case.run()
    first = int(case.positions[:12].max()) - 30  # the deepest node no longer sees it
    page, cell = int(case.table[0, first // 64]), first % 64
    case.dev["v_pool"][page, :, cell] = value
    out = case.run()
    for i in range(12):
        if not bool(case.visible(0, i)[first]):
            assert torch.equal(out[i], want[i])


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("D,ctx", [(64, 400), (128, 400), (128, 9000)])
def test_tree_attention_non_finite_context_beside_a_page_outside_the_pool(value, D, ctx):
    """A context key that every row sees is non-finite, and the page before its
    own lies outside the pool: the key still counts."""
    case = Tree([ctx], [5], 8, 2, D, seed=23)
    page = int(case.table[0, 3])
    case.dev["page_table"][0, 2] = -1
    case.dev["v_pool"][page, :, 5, ::3] = value
    out = case.run()[:5].float()
    hit = torch.zeros(D, dtype=torch.bool, device="cuda")
    hit[::3] = True
    assert bool((torch.isnan(out) if math.isnan(value) else out == value)[..., hit].all())
    assert bool(torch.isfinite(out[..., ~hit]).all())


@pytest.mark.parametrize("extra_rows", [0, 520])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("ctx,nodes", [(300, 12), (300, 40), (9000, 12)])
def test_tree_attention_large_values(ctx, nodes, D, extra_rows):
    """Values up to 2^127 and scores that rise after a row's first keys, by 20
    log2 units and then by 60: the results are averages of the values, so they
    are finite."""
    case = Tree([ctx], [nodes], 8, 2, D, seed=36, extra_rows=extra_rows)
    g = torch.Generator().manual_seed(37)
    n = ctx + nodes
    case.q = torch.zeros(case.rows, 8, D, dtype=torch.bfloat16)
    case.q[:, :, 0] = 8.0
    units = torch.full((n,), 20.0)  # the keys' scores
    units[:64], units[ctx:] = 0.0, 0.0
    for one in (20.0, 80.0):
        units[n * 3 // 4] = one
        k = torch.zeros(n, 2, D)
        k[:, :, 0] = (units * math.log(2.0) * math.sqrt(D) / 8.0)[:, None]
        v = (torch.rand(n, 2, D, generator=g) + 1.0) * 2.0 ** 126
        v[:, :, 1::2] *= -1.0
        k, v = k.bfloat16(), v.bfloat16()
        case.k[0], case.v[0] = k.double(), v.double()
        at = torch.arange(n)
        page = torch.from_numpy(case.table[0])[at // 64].long().cuda()
        case.dev["q"] = case.q.cuda()
        case.dev["k_pool"][page, :, (at % 64).cuda()] = k.cuda()
        case.dev["v_pool"][page, :, (at % 64).cuda()] = v.cuda()
        out = case.run()
        assert bool(torch.isfinite(out[:nodes].float()).all())
        case.check(out)


# Calls of few rows (512 of all heads) multiply P in two parts; with rows behind
# the last sequence the same trees run as a larger call does.

@pytest.mark.parametrize("q_heads,kv_heads,D", HEADS)
@pytest.mark.parametrize("ctx,nodes", [([0], [1]), ([700, 129], [3, 30]), ([1, 64, 300, 0], [1, 17, 40, 5]), ([5000], [12])])
def test_tree_attention_as_a_larger_call(q_heads, kv_heads, D, ctx, nodes):
    case = Tree(ctx, nodes, q_heads, kv_heads, D, seed=31, extra_rows=520)
    case.check(case.run())


@pytest.mark.parametrize("D", [64, 128])
def test_tree_attention_masks_scores_and_cells_as_a_larger_call(D):
    more = dict(q_heads=8, kv_heads=2, D=D, extra_rows=100)
    for window in (5, 130):
        case = Tree([200, 9], [7, 30], window=window, seed=32, **more)
        case.check(case.run())
    case = Tree([300, 40], [10, 70], seed=33, scale=40.0, **more)
    case.check(case.run())
    case = Tree([140, 50], [12, 9], seed=34, **more)
    clean = case.run()
    page, cell = int(case.table[0, 143 // 64]), 143 % 64
    for pool in ("k_pool", "v_pool"):
        case.dev[pool][page, :, cell] = math.inf
    out = case.run()
    for i in range(12):
        if not case.seen[0][i][3]:
            assert torch.equal(out[i], clean[i])


@pytest.mark.parametrize("extra_rows", [0, 520])
@pytest.mark.parametrize("D", [64, 128])
def test_tree_attention_rows_that_see_one_key_return_its_value(D, extra_rows):
    """The only weight of a row is 1 whatever its rounding, in small calls and
    in large ones: nodes that see themselves alone, over an empty context."""
    def masks(rng, n):
        return np.eye(n, dtype=bool)
    case = Tree([0, 0], [30, 9], 8, 2, D, masks=masks, seed=38, extra_rows=extra_rows)
    out = case.run().cpu()
    for b, n in enumerate(case.nodes):
        for i in range(n):
            value = case.v[b][i].bfloat16().repeat_interleave(case.group, 0)
            assert torch.equal(out[int(case.starts[b]) + i], value), (b, i)


@pytest.mark.parametrize("q_heads,kv_heads,D", [(14, 2, 64), (8, 4, 128)])
def test_tree_attention_of_few_rows_rounds_only_its_output(q_heads, kv_heads, D):
    """P enters the products cut to bf16 (off by up to 2^-7) with the rest as
    bf16 beside it (off by half a step of 2^-7): 2^-15, and 2^-23 added."""
    case = Tree([700, 90], [8, 21], q_heads, kv_heads, D, seed=35)
    out = case.run().cpu().double()
    for b, i in ((0, 0), (0, 7), (1, 3), (1, 20)):
        seen, r = case.visible(b, i), int(case.starts[b]) + i
        for h in range(q_heads):
            k, v = case.k[b][:, h // case.group], case.v[b][:, h // case.group]
            want, tol = V.tree_row(case.q[r, h].double(), k, v, seen)
            p = torch.softmax(k[seen] @ case.q[r, h].double() / math.sqrt(D), 0)
            tol = tol - (p @ v[seen].abs()) * (2.0 ** -8 - 2.0 ** -15 - 2.0 ** -23) * 1.01
            assert bool(((out[r, h] - want).abs() <= tol).all())


def test_tree_attention_large_scores():
    """Scores of a few hundred: one weight is 1 and the others underflow."""
    case = Tree([300, 40], [10, 70], 14, 2, 64, seed=9, scale=40.0)
    case.check(case.run())


def test_tree_attention_bad_lengths_pages_and_padding():
    """Sequences without room for their rows give zeros, keys on a page outside
    the pool are unseen, rows behind the last sequence stay."""
    case = Tree([200, 30, 100], [6, 5, 4], 14, 2, 64, seed=11, extra_rows=9)
    case.dev["seq_lens"][1] = 3
    out = torch.full_like(case.dev["q"], 5.0)
    got = case.run(out=out)
    assert got is out
    assert bool((out[6:11] == 0).all()) and bool((out[15:] == 5.0).all())
    case.nodes, starts = [6, 0, 4], case.starts
    case.check(out)
    case.dev["page_table"][0, 1] = 10 ** 6
    case.dev["page_table"][0, 2] = -3
    out = case.run()
    seen = case.visible(0, 2)
    seen[64:192] = False
    for h in range(14):
        want, tol = V.tree_row(case.q[2, h].double(), case.k[0][:, h // 7], case.v[0][:, h // 7], seen)
        assert bool(((out[2, h].cpu().double() - want).abs() <= tol).all())
    assert list(starts) == [0, 6, 11, 15]


def test_tree_attention_mask_words_cut_later_nodes():
    case = Tree([50], [100], 4, 4, 64, words=1, seed=12)
    case.check(case.run())


def test_tree_attention_strided_q_and_table_wider_than_needed():
    case = Tree([500, 77], [20, 30], 14, 2, 64, seed=13, width=40)
    wide = torch.zeros(case.rows, 18, 64, dtype=torch.bfloat16, device="cuda")
    wide[:, :14] = case.dev["q"]
    case.check(case.run(q=wide[:, :14]))


def test_tree_attention_repeats_bit_for_bit():
    case = Tree([3000, 17, 900], [30, 64, 5], 28, 4, 128, seed=14)
    a = case.run()
    for _ in range(3):
        assert torch.equal(a, case.run())


def test_tree_attention_single_nodes_match_decode_attention():
    """One node that sees itself is the decode attention of its position."""
    from cheetah_b200 import runtime as R
    case = Tree([700, 63, 2000], [1, 1, 1], 14, 2, 64, seed=15, fill=0.0)
    d = case.dev
    want = R.decode_attention(d["q"].float(), d["k_pool"], d["v_pool"], d["page_table"], d["seq_lens"], 2001)
    assert (case.run().float() - want).abs().max().item() < 1e-2  # the decode kernel's own contract


def test_tree_attention_on_other_streams_and_in_graphs():
    """Calls that overlap: two streams, and two captured graphs replayed on
    two streams, each with its own workspace."""
    cases = [Tree([4000, 100], [20, 64], 14, 2, 64, seed=s) for s in (31, 32)]
    want = [c.run() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [c.run(stream=s) for _ in range(8) for c, s in zip(cases, streams)]
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 2])
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c.run())
        graphs.append(g)
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)


def test_tree_attention_join_after_a_wait_that_gave_up(tmp_path):
    """The join alone, on a list of split items in which one CTA has given up:
    every row is NaN, those behind the last sequence stay. Without one that has,
    and without anything to join, it writes nothing."""
    import ctypes as C
    import subprocess
    from pathlib import Path
    from cheetah_b200 import build
    here = Path(__file__).resolve().parent
    lib = tmp_path / "tree_join.so"
    subprocess.run([build.nvcc(), *build.ARCH_FLAGS, "-O1", "-std=c++17", "-shared", "-Xcompiler", "-fPIC", "-I", str(build.CSRC),
                    "-I", str(build.INCLUDE), "--expt-relaxed-constexpr", "-o", str(lib), str(here / "tree_join_entry.cu")],
                   check=True, capture_output=True, timeout=300)
    join = C.CDLL(str(lib)).tree_join
    rows, q_heads, ctas = 20, 3, 5
    starts = i32([0, 4, 13])
    splits = torch.zeros(32 * ctas, dtype=torch.uint8, device="cuda")
    for parts, given_up in (([0, 0, -1, 0, 0], True), ([0, 1, 0, 1, 0], False), ([-1] * 5, True)):
        out = torch.full((rows, q_heads, 64), 2.5, dtype=torch.bfloat16, device="cuda")
        rc = join((C.c_int * ctas)(*parts), ctas, C.c_void_p(starts.data_ptr()), 2, rows, q_heads, C.c_void_p(splits.data_ptr()),
                  C.c_void_p(out.data_ptr()), C.c_void_p(torch.cuda.current_stream().cuda_stream))
        torch.cuda.synchronize()
        assert rc == 0
        assert bool(torch.isnan(out[:13]).all()) if given_up else bool((out[:13] == 2.5).all())
        assert bool((out[13:] == 2.5).all())


# ---- token_logprobs -----------------------------------------------------------

def _check_logprobs(x, tokens, top, dtype):
    from cheetah_b200 import runtime as R
    x = x.to({"bf16": torch.bfloat16, "f32": torch.float32}[dtype])
    got = R.token_logprobs(x if x.is_cuda else x.cuda(), i32(tokens), top=top)
    rows = x.cpu()
    for r, token in enumerate(tokens):
        ref = V.logprobs_row(rows[r], token, top)
        lp, h, rank = float(got.logprob[r]), float(got.entropy[r]), int(got.rank[r])
        ids, lps = got.top_ids[r].tolist(), got.top_logprobs[r].cpu().double()
        if ref["bad"]:
            assert math.isnan(lp) and math.isnan(h) and rank == 0 and ids == [-1] * top and bool(torch.isnan(lps).all())
            continue
        assert ids == ref["top_ids"], f"row {r}"
        for a, b in zip(lps.tolist(), ref["top_logprobs"].tolist()):
            assert a == b or abs(a - b) <= V.tol_logprob(ref, b), f"row {r}: {a} vs {b}"
        assert abs(h - ref["entropy"]) <= ref["tol_entropy"], f"row {r}: entropy {h} vs {ref['entropy']}"
        if not ref["known"]:
            assert math.isnan(lp) and rank == 0
            continue
        assert rank == ref["rank"]
        assert lp == ref["logprob"] or abs(lp - ref["logprob"]) <= V.tol_logprob(ref, ref["logprob"])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 2, 0), (3, 7, 7), (5, 33, 32), (2, 1000, 5), (4, 4096, 20), (7, 32001, 32),
                                            (1, 151936, 20), (3, 152064, 5), (40, 20011, 1), (300, 5003, 3)])
def test_token_logprobs(dtype, rows, vocab, top):
    g = torch.Generator().manual_seed(rows + vocab)
    x = torch.randn(rows, vocab, generator=g) * 3.0
    tokens = torch.randint(0, vocab, (rows,), generator=g).tolist()
    _check_logprobs(x, tokens, top, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [100, 5000, 40000])
def test_token_logprobs_orders_that_fill_every_buffer(dtype, vocab):
    """Ascending, descending, all equal, two values, signed zeros: the
    alternatives stay exact whatever order the values come in."""
    up = torch.linspace(-5, 5, vocab)
    equal = torch.full((vocab,), 0.25)
    two = torch.where(torch.arange(vocab) % 3 == 1, 2.0, -1.0)
    zeros = torch.where(torch.arange(vocab) % 2 == 1, 0.0, -0.0)
    late = torch.cat([torch.full((vocab - 40,), -3.0), torch.linspace(0, 1, 40)])
    x = torch.stack([up, up.flip(0), equal, two, zeros, late])
    _check_logprobs(x, [vocab - 1, 0, vocab // 2, 1, 5, vocab - 2], 32, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_token_logprobs_masked_and_broken_rows(dtype):
    """-inf logits have probability 0; NaN, +inf and all -inf rows are refused
    row by row; tokens outside the vocabulary give NaN."""
    vocab = 3001
    g = torch.Generator().manual_seed(3)
    x = torch.randn(10, vocab, generator=g)
    x[0, ::2] = -math.inf
    x[1, 3:] = -math.inf                     # fewer than `top` above -inf
    x[2, :] = -math.inf
    x[3, 17] = math.nan
    x[4, vocab - 1] = math.inf
    x[5, :] = torch.finfo(torch.bfloat16).min  # the type's lowest value throughout
    x[6, 1:] = torch.finfo(torch.bfloat16).min
    x[7] *= 1e30
    _check_logprobs(x, [0, 5, 1, 2, 3, 4, 0, 7, -1, vocab], 8, dtype)


@pytest.mark.parametrize("vocab", [300, 5000, 151936])
@pytest.mark.parametrize("top", [0, 5])
def test_token_logprobs_peaked_rows(vocab, top):
    """Two logits at most count, the rest are 50 below. Then S = 1 + e^-d is
    rounded twice at most (2^-24 each, in a thread and in the join), its log
    once, and e^-d is off by 2^-20 of itself. The entropy adds a few terms of
    at most 2 log2 units with one rounding each."""
    from cheetah_b200 import runtime as R
    gaps = [0.0, 0.5, 0.99, 1.01, 3.0, 7.99, 8.01, 12.0, 25.0]
    places = [(3, vocab - 40), (vocab - 40, 3), (5, vocab // 2), (vocab // 2, vocab // 2 + 1), (vocab // 3, vocab - 1)]
    for base in (0.0, 17.3, -40.2):
        x = torch.full((len(gaps) * len(places), vocab), base - 50.0, dtype=torch.float64)
        low, high = [], []
        for i, d in enumerate(gaps):
            for j, (a, b) in enumerate(places):
                r = i * len(places) + j
                x[r, a], x[r, b] = base, base + d
                low.append(a)
                high.append(b)
        x = x.float()
        exact = torch.log_softmax(x.double(), 1)
        entropy = -(exact.exp() * exact).sum(1)
        u = 2.0 ** -24
        for tokens in (low, high):
            got = R.token_logprobs(x.cuda(), i32(tokens), top=top)
            want = exact.gather(1, torch.tensor(tokens)[:, None])[:, 0]
            lp, h = got.logprob.cpu().double(), got.entropy.cpu().double()
            assert bool((lp <= 0).all()) and bool((h >= 0).all())
            tol = 3 * u + (1 - exact.max(1).values.exp()) * 2.0 ** -20 + 2 * u * want.abs()
            assert bool(((lp - want).abs() <= tol).all()), float(((lp - want).abs() / tol).max())
            assert bool(((h - entropy).abs() <= 15 * u + entropy * 2.0 ** -20).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [700, 40000])
def test_token_logprobs_signs(dtype, vocab):
    """No log probability is above 0 and no entropy below, however far the
    largest logit stands out and wherever it lies."""
    from cheetah_b200 import runtime as R
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn(1000, vocab, generator=g, device="cuda") * 0.3 - 12.0
    at = torch.randint(0, vocab, (1000, 1), generator=g, device="cuda")
    x.scatter_(1, at, torch.rand(1000, 1, generator=g, device="cuda") * 20.0)
    x = x.to({"bf16": torch.bfloat16, "f32": torch.float32}[dtype])
    got = R.token_logprobs(x, at[:, 0].int(), top=2)
    assert bool((got.logprob <= 0).all()) and bool((got.top_logprobs <= 0).all()) and bool((got.entropy >= 0).all())


def test_token_logprobs_strided_unaligned_rows():
    g = torch.Generator().manual_seed(4)
    for dtype in ("f32", "bf16"):
        base = torch.randn(9, 5011, generator=g).to({"bf16": torch.bfloat16, "f32": torch.float32}[dtype]).cuda()
        _check_logprobs(base[:, 3:4998], list(range(9)), 5, dtype)
        _check_logprobs(base[::2, 1:], list(range(5)), 5, dtype)


def test_token_logprobs_captured():
    from cheetah_b200 import runtime as R
    x = torch.randn(6, 30000, device="cuda")
    t = i32(range(6))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = R.token_logprobs(x, t, top=4)
    x.copy_(torch.randn(6, 30000, device="cuda") * 2)
    g.replay()
    want = R.token_logprobs(x, t, top=4)
    for a, b in zip(out, want):
        assert torch.equal(a, b)


# ---- the four together ----------------------------------------------------------

@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("q_heads,kv_heads,D", [(14, 2, 64), (8, 4, 128)])
def test_verification_step(q_heads, kv_heads, D, captured):
    """Slots, append, attention and log probabilities of one step over caches
    that an earlier step of the same operators filled; rows padded to a fixed
    count, one sequence without new rows and one that finds no pages."""
    from cheetah_b200 import runtime as R
    g = torch.Generator().manual_seed(D)
    rng = np.random.default_rng(D)
    pt, width, rows, vocab, B = 16, 24, 64, 1003, 4
    ctx, nodes = [130, 77, 33, 20], [12, 0, 21, 60]
    heads = q_heads + 2 * kv_heads
    num_pages = 1 + sum(-(-c // pt) for c in ctx) + 3
    free = i32(rng.permutation(num_pages)[:num_pages - 1])
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    k_pool = torch.full((num_pages, kv_heads, pt, D), math.nan, dtype=torch.bfloat16, device="cuda")
    v_pool = k_pool.clone()
    angle = torch.rand(400, D // 2, generator=g) * 6.0
    cos, sin = angle.cos().cuda(), angle.sin().cuda()
    w = [(1.0 + 0.2 * torch.randn(D, generator=g)).cuda() for _ in range(2)]

    def step(cached, new, free, count, x, mask, head, tokens, positions=None):
        s = R.page_slots(cached, new, free, count, table, num_pages, pt, x.shape[0])
        pos = s.positions if positions is None else torch.where(s.positions >= 0, positions, -1)
        q = R.qk_norm_rope(x, q_heads, kv_heads, pos, s.slots, cos, sin, k_pool, v_pool, q_norm=w[0], k_norm=w[1])
        o = R.tree_attention(q, k_pool, v_pool, table, s.seq_lens, s.row_starts, mask, positions=pos,
                             out=torch.zeros_like(q))
        return s, q, o, R.token_logprobs(o.float().reshape(x.shape[0], -1) @ head, tokens, top=3)

    # The prompts, as chains.
    total = sum(ctx)
    prompt = torch.randn(total, heads, D, generator=g).bfloat16()
    chain = np.concatenate([np.tril(np.ones((c, 192), bool)) for c in ctx])
    chain = V.pack_bits(chain, 3)
    head = torch.randn(q_heads * D, vocab, generator=g).cuda()
    first = step(i32([0] * B), i32(ctx), free, i32([free.numel()]), prompt.cuda(), torch.from_numpy(chain).cuda(), head,
                 i32(rng.integers(0, vocab, total)))
    used = int(first[0].counts[1])
    assert first[0].counts.tolist() == [total, sum(-(-c // pt) for c in ctx), 0]
    # The drafted trees; the last sequence needs more pages than are left.
    x = torch.randn(rows + 40, heads, D, generator=g).bfloat16()
    trees = [V.tree_bits(V.random_tree(rng, n)) for n in nodes]
    mask = np.zeros((rows + 40, 1), np.int64)
    mask[:sum(nodes)] = np.concatenate([V.pack_bits(t[0], 1) for t in trees if len(t[0])])
    depth = np.full(rows + 40, -1)
    depth[:sum(nodes)] = np.concatenate([t[1] + c for t, c in zip(trees, ctx)])
    tokens = rng.integers(0, vocab, rows + 40)
    args = (i32(ctx), i32(nodes), free[used:].contiguous(), i32([free.numel() - used]), x.cuda(), torch.from_numpy(mask).cuda(),
            head, i32(tokens), i32(depth))
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s, q, o, lp = step(*args)
        graph.replay()
    else:
        s, q, o, lp = step(*args)
    torch.cuda.synchronize()
    assert s.counts.tolist()[2] == 1 and s.seq_lens.tolist() == [142, 77, 54, 0]
    at = np.concatenate([[0], np.cumsum(nodes)])
    # K/V in the pool are what the rows give (checked above); attention over them.
    kc, vc, tab = k_pool.cpu().double(), v_pool.cpu().double(), table.cpu().numpy()
    ocpu = o.cpu().double()
    for b in (0, 2):
        pages = tab[b, :-(-(ctx[b] + nodes[b]) // pt)].astype(np.int64)
        n = ctx[b] + nodes[b]
        kd = kc[pages].transpose(1, 2).reshape(-1, kv_heads, D)[:n]
        vd = vc[pages].transpose(1, 2).reshape(-1, kv_heads, D)[:n]
        assert bool(torch.isfinite(kd).all())
        for i in (0, nodes[b] // 2, nodes[b] - 1):
            seen = torch.from_numpy(np.concatenate([np.ones(ctx[b], bool), trees[b][0][i]]))
            for h in range(q_heads):
                kvh = h * kv_heads // q_heads
                want, tol = V.tree_row(q[at[b] + i, h].cpu().double(), kd[:, kvh], vd[:, kvh], seen)
                assert bool(((ocpu[at[b] + i, h] - want).abs() <= tol).all())
    assert bool((ocpu[at[3]:] == 0).all())  # refused, and the padding as it was
    logits = o.float().reshape(rows + 40, -1) @ head
    again = R.token_logprobs(logits, i32(tokens), top=3)
    assert torch.equal(again.top_ids[:at[3]], lp.top_ids[:at[3]])
    for r in (0, 5, int(at[2]) + 3):
        ref = V.logprobs_row(logits[r].cpu(), int(tokens[r]), 3)
        assert abs(float(lp.logprob[r]) - ref["logprob"]) <= V.tol_logprob(ref, ref["logprob"])
