"""The operators over an 8-bit cache and the test of drafted tokens on the GPU
against 64-bit references (`tests/kv8_ref.py`), at the sizes, masks and values
where they can go wrong, and a run of them as a serving step uses them."""

import math

import numpy as np
import pytest

from tests import kv8_ref as V8
from tests import verify_ref as V

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
E4M3 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from cheetah_b200 import runtime
    runtime.lib()


def i32(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


def random_pool(g, pages, kvh, pt, D, spread=1.0):
    """(codes uint8, scales f32) on the CPU: any code but NaN's, scales over a few powers of two."""
    codes = torch.randint(0, 127, (pages, kvh, pt, D), generator=g).to(torch.uint8)
    codes |= (torch.randint(0, 2, codes.shape, generator=g) << 7).to(torch.uint8)
    e = torch.round(spread * torch.randn(pages, kvh, pt // 16, generator=g)) - 8
    return codes, torch.exp2(e)


def normal_pool(g, pages, kvh, pt, D, spread=0.5):
    """A pool of normal values whose size varies from block to block."""
    x = torch.randn(pages, kvh, pt // 16, 16 * D, generator=g) * torch.exp(spread * torch.randn(pages, kvh, pt // 16, 1, generator=g))
    e = torch.ceil(torch.log2(x.abs().amax(-1) / 448.0))
    return (x / torch.exp2(e)[..., None]).to(E4M3).reshape(pages, kvh, pt, D).view(torch.uint8), torch.exp2(e)


def to_gpu(codes, scales):
    return codes.cuda().view(E4M3), scales.cuda()


# ---- qk_norm_rope_kv8 ----------------------------------------------------------

def check_append(x, q_heads, kvh, positions, slots, cos, sin, w, pools, eps, max_pos, wide=0):
    """One call against the references; returns the GPU pools."""
    from cheetah_b200 import runtime as R
    tokens, heads, D = x.shape
    rows = torch.cat([x.reshape(tokens, heads * D), torch.zeros(tokens, wide, dtype=x.dtype)], 1) if wide else x.reshape(tokens, -1)
    (k_codes, k_scales), (v_codes, v_scales) = to_gpu(*pools[0]), to_gpu(*pools[1])
    q_out = torch.full((tokens, q_heads, D), 7.0, dtype=x.dtype, device="cuda")
    got = R.qk_norm_rope_kv8(rows.cuda()[:, :heads * D], q_heads, kvh, positions.cuda(), slots.cuda(), cos.cuda(), sin.cuda(),
                             k_codes, v_codes, k_scales, v_scales, q_norm=None if w[0] is None else w[0].cuda(),
                             k_norm=None if w[1] is None else w[1].cuda(), eps=eps, q_out=q_out)
    assert got is q_out
    f32, step = (D / 2 + 10) * 2.0 ** -24, 2.0 ** -8 if x.dtype == torch.bfloat16 else 2.0 ** -24
    q = got.cpu().double()
    k_rows = torch.zeros(tokens, kvh, D, dtype=torch.float64)
    live = []
    for t in range(tokens):
        p = int(positions[t])
        if not 0 <= p < max_pos:
            assert bool((q[t] == 7.0).all())
            live.append(-1)
            continue
        live.append(int(slots[t]))
        for h in range(q_heads):
            z, mag = V.norm_rope_head(x[t, h], w[0], eps, cos[p], sin[p])
            assert bool(((q[t, h] - z).abs() <= mag * f32 + z.abs() * step + 1e-30).all()), (t, h)
        for h in range(kvh):
            k_rows[t, h] = V.norm_rope_head(x[t, q_heads + h], w[1], eps, cos[p], sin[p])[0]
    want = [(c.clone(), s.clone()) for c, s in pools]
    V8.append(*want[0], live, k_rows)
    V8.append(*want[1], live, x[:, q_heads + kvh:].double())
    for name, codes, scales, (wc, ws) in (("k", k_codes, k_scales, want[0]), ("v", v_codes, v_scales, want[1])):
        assert torch.equal(scales.cpu(), ws), name + " scales"
        assert torch.equal(codes.view(torch.uint8).cpu(), wc), name + " codes"
    return k_codes, v_codes, k_scales, v_scales


def rope_tables(g, max_pos, rotary):
    angle = torch.rand(max_pos, rotary // 2, generator=g) * 6.0
    return angle.cos(), angle.sin()


@pytest.mark.parametrize("q_heads,kvh,D,rotary", [(14, 2, 64, 64), (28, 4, 128, 128), (4, 4, 64, 32), (3, 1, 128, 16), (8, 4, 128, 96)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("tokens,first,norm", [(1, 0, True), (1, 13, False), (7, 12, True), (37, 5, True), (64, 0, False)])
def test_append_of_a_run(q_heads, kvh, D, rotary, dtype, tokens, first, norm):
    """One sequence's new tokens from position `first` on: whole blocks, the
    ends of two, cells ahead that keep their values."""
    g = torch.Generator().manual_seed(tokens + D + rotary + first)
    pt, pages, max_pos = 32, 6, 90
    x = torch.randn(tokens, q_heads + 2 * kvh, D, generator=g).to(TYPES[dtype])
    order = torch.randperm(pages, generator=g)
    pos = torch.arange(tokens) + first
    slots = (order[pos // pt] * pt + pos % pt).to(torch.int32)
    w = [1.0 + 0.3 * torch.randn(D, generator=g) if norm else None for _ in range(2)]
    pools = [random_pool(g, pages, kvh, pt, D, 2.0) for _ in range(2)]
    check_append(x, q_heads, kvh, pos.to(torch.int32), slots, *rope_tables(g, max_pos, rotary), w, pools, 1e-5, max_pos, wide=16)


@pytest.mark.parametrize("seed", range(4))
def test_append_of_a_ragged_batch(seed):
    """Sequences of 0..20 new tokens in page_slots' order, some rows skipped."""
    g = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed)
    kvh, D, pt, pages, max_pos = 2, 64, 16, 80, 300
    slots, pos, page = [], [], list(rng.permutation(pages))
    for _ in range(20):
        n, cached = int(rng.integers(0, 21)), int(rng.integers(0, 40))
        table = {}
        for i in range(cached, cached + n):
            table.setdefault(i // pt, None)
            if table[i // pt] is None:
                table[i // pt] = int(page.pop())
            slots.append(table[i // pt] * pt + i % pt)
            pos.append(i)
    tokens = len(slots)
    slots, pos = np.array(slots), np.array(pos)
    for i in rng.integers(0, tokens, 12):
        if rng.random() < 0.5:
            slots[i] = rng.choice([-1, pages * pt, 2 ** 31 - 1, -2 ** 31])
        else:
            pos[i] = rng.choice([-1, max_pos, 2 ** 31 - 1])
    x = torch.randn(tokens, 4 + 2 * kvh, D, generator=g).to(torch.bfloat16)
    pools = [random_pool(g, pages, kvh, pt, D, 3.0) for _ in range(2)]
    w = [1.0 + 0.3 * torch.randn(D, generator=g) for _ in range(2)]
    check_append(x, 4, kvh, torch.tensor(pos, dtype=torch.int32), torch.tensor(slots, dtype=torch.int32),
                 *rope_tables(g, max_pos, D), w, pools, 1e-6, max_pos)


@pytest.mark.parametrize("dtype,D,tokens", [("bf16", 128, 2600), ("f32", 64, 2081), ("bf16", 64, 4099)])
def test_append_of_many_rows(dtype, D, tokens):
    """So many rows that a warp looks among sixteen for blocks; the slots of a
    block come in any order within 32 rows."""
    g = torch.Generator().manual_seed(tokens)
    kvh, pt, max_pos = 2, 16, 64
    pages = -(-tokens // pt) + 2
    # Cells of 16 to 24 row windows, shuffled within.
    at = torch.arange(tokens)
    for i in range(5, tokens - 24, 24):
        part = at[i:i + 24].clone()
        at[i:i + 24] = part[torch.randperm(24, generator=g)]
    slots = (torch.randperm(pages, generator=g)[at // pt] * pt + at % pt).to(torch.int32)
    pos = torch.randint(0, max_pos, (tokens,), generator=g).to(torch.int32)
    pos[::17] = -1
    spread = (int(at.max()), [int((at // pt == b).nonzero().max() - (at // pt == b).nonzero().min()) for b in range(tokens // pt)])
    assert max(spread[1]) <= 31 + 24  # blocks that straddle windows
    keep = torch.tensor([b for b, s in enumerate(spread[1]) if s <= 31])
    slots = torch.where(torch.isin(at // pt, keep), slots, torch.full_like(slots, -1))
    x = torch.randn(tokens, 3 * kvh, D, generator=g).to(TYPES[dtype])
    pools = [random_pool(g, pages, kvh, pt, D, 2.0) for _ in range(2)]
    check_append(x, kvh, kvh, pos, slots, *rope_tables(g, max_pos, D), [None, 1.0 + 0.2 * torch.randn(D, generator=g)], pools,
                 1e-6, max_pos)


def test_append_extreme_values():
    """Zeros, tiny, huge and non-finite values, ties between codes, a block's scale at its least."""
    g = torch.Generator().manual_seed(3)
    kvh, D, pt, pages, max_pos = 1, 64, 16, 12, 20
    x = torch.randn(12 * 4, 3, D, generator=g)
    x[0:4] = 0.0
    x[4:8] *= 1e-38
    x[8:12] *= 3e37
    x[12:16] = torch.randint(-448 * 2, 448 * 2, (4, 3, D), generator=g) / 2.0
    x[16:20] = torch.exp2(torch.randint(-20, 8, (4, 3, D), generator=g).float()) * (1 + torch.randint(0, 16, (4, 3, D), generator=g) / 16)
    x[20, 1, 3], x[21, 2, 5], x[22, 2, 6], x[23, 1, 0] = math.nan, math.inf, -math.inf, math.inf
    x[24:28] = 448.0
    x[28:32] = 448.0 * (1 + 2.0 ** -23)
    x[32:36] *= 2.0 ** -62
    x[36:40, :, ::2] = 3.0e38
    slots = torch.cat([torch.arange(4) + 16 * p for p in range(12)]).to(torch.int32)
    pos = torch.zeros(48, dtype=torch.int32)
    cos, sin = torch.ones(max_pos, D // 2), torch.zeros(max_pos, D // 2)  # no rotation: k is x itself
    pools = [random_pool(g, pages, kvh, pt, D) for _ in range(2)]
    check_append(x, 1, kvh, pos, slots, cos, sin, [None, None], pools, 1e-6, max_pos)


@pytest.mark.parametrize("old", [0.0, 2.0 ** -64, 2.0 ** -3, 0.3, 2.0 ** 100])
def test_append_behind_a_scale(old):
    """Cells ahead keep their values while the scale grows, or the scale stays; also one that is no power of two."""
    g = torch.Generator().manual_seed(5)
    kvh, D, pt, pages = 2, 128, 16, 3
    x = torch.randn(3, 6, D, generator=g)
    pools = [random_pool(g, pages, kvh, pt, D) for _ in range(2)]
    for _, s in pools:
        s.fill_(old)
    slots = torch.tensor([16 + 5, 16 + 6, 16 + 7], dtype=torch.int32)
    cos, sin = torch.ones(4, D // 2), torch.zeros(4, D // 2)
    if old == 0.3:
        # Quotients by such a scale round: the nearest of values that lie no nearer to a border than that.
        x = torch.randint(-3, 4, x.shape, generator=g) * 0.3
    check_append(x, 2, kvh, torch.zeros(3, dtype=torch.int32), slots, cos, sin, [None, None], pools, 1e-6, 4)


def test_append_again_changes_nothing():
    from cheetah_b200 import runtime as R
    g = torch.Generator().manual_seed(9)
    kvh, D, pt, pages = 2, 64, 32, 4
    x = torch.randn(20, 8, D, generator=g)
    pools = [random_pool(g, pages, kvh, pt, D) for _ in range(2)]
    slots = (torch.arange(20) + 40).to(torch.int32)
    pos = torch.arange(20).to(torch.int32)
    cos, sin = rope_tables(g, 32, D)
    k_codes, v_codes, k_scales, v_scales = check_append(x, 4, kvh, pos, slots, cos, sin, [None, None], pools, 1e-6, 32)
    before = [t.clone().view(torch.uint8) for t in (k_codes, v_codes, k_scales, v_scales)]
    R.qk_norm_rope_kv8(x.cuda(), 4, kvh, pos.cuda(), slots.cuda(), cos.cuda(), sin.cuda(), k_codes, v_codes, k_scales, v_scales)
    for a, b in zip(before, (k_codes, v_codes, k_scales, v_scales)):
        assert torch.equal(a, b.view(torch.uint8))


# ---- kv8_read ------------------------------------------------------------------

@pytest.mark.parametrize("kvh,D,pt", [(2, 64, 64), (4, 128, 16), (1, 128, 48), (8, 64, 128)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("tokens", [1, 3, 257, 1030])
def test_kv8_read(kvh, D, pt, dtype, tokens):
    from cheetah_b200 import runtime as R
    g = torch.Generator().manual_seed(tokens + D)
    pages = 7
    pools = [random_pool(g, pages, kvh, pt, D, 3.0) for _ in range(2)]
    pools[0][0][2, 0, 3, 5] = 127  # NaN
    pools[1][0][2, 0, 3, 6] = 255
    slots = torch.randint(0, pages * pt, (tokens,), generator=g).to(torch.int32)  # repeated ones among them
    slots[0] = 2 * pt + 3
    if tokens > 2:
        slots[1], slots[2] = -1, pages * pt
    (kc, ks), (vc, vs) = to_gpu(*pools[0]), to_gpu(*pools[1])
    got = R.kv8_read(kc, vc, ks, vs, slots.cuda(), dtype=TYPES[dtype])
    for out, (codes, scales) in zip(got, pools):
        want = torch.zeros(tokens, kvh, D, dtype=torch.float64)
        for t, s in enumerate(slots.tolist()):
            if 0 <= s < pages * pt:
                want[t] = V8.decode(codes[s // pt, :, s % pt]) * scales[s // pt, :, s % pt // 16].double()[:, None]
        assert out.dtype == TYPES[dtype] and out.shape == (tokens, kvh, D)
        # Products of a code and a power of two are exact in either type.
        assert torch.equal(torch.nan_to_num(out.cpu().double(), nan=1e9), torch.nan_to_num(want, nan=1e9))


# ---- attention_kv8 -------------------------------------------------------------

class Attend:
    """A call's inputs, on the CPU as the reference takes them."""

    def __init__(self, seed, ctx, rows, q_heads, kvh, D, pt, window=0, sinks=0, pool=normal_pool, q_scale=1.5, extra_rows=0,
                 wide=0, spread=0.5):
        g = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.kvh, self.D, self.pt, self.window, self.sinks = kvh, D, pt, window, sinks
        need = [-(-(c + n) // pt) for c, n in zip(ctx, rows)]
        self.pages = sum(need) + 2
        order = rng.permutation(self.pages)
        self.table = np.full((len(ctx), max(max(need), 1)), -1)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.k, self.v = pool(g, self.pages, kvh, pt, D, spread), pool(g, self.pages, kvh, pt, D, spread)
        self.lens = [c + n for c, n in zip(ctx, rows)]
        self.starts = [0] + np.cumsum(rows).tolist()
        total = self.starts[-1] + extra_rows
        self.q_wide = (torch.randn(total, q_heads * D + wide, generator=g) * q_scale).to(torch.bfloat16)
        self.q = self.q_wide[:, :q_heads * D].reshape(total, q_heads, D)

    def run(self, out=None, **more):
        from cheetah_b200 import runtime as R
        total, qh, D = self.q.shape
        q = self.q_wide.cuda()[:, :qh * D].unflatten(1, (qh, D))
        (kc, ks), (vc, vs) = to_gpu(*self.k), to_gpu(*self.v)
        return R.attention_kv8(q, kc, vc, ks, vs, i32(self.table), i32(self.lens), i32(self.starts), sliding_window=self.window,
                               sinks=self.sinks, out=out, **more)

    def check(self, got, sample=None):
        """Every row and head (or `sample` sequences) against the reference."""
        got = got.cpu().double()
        qh, group = self.q.shape[1], self.q.shape[1] // self.kvh
        worst = 0.0
        for b in range(len(self.lens)) if sample is None else sample:
            r0, r1, length = self.starts[b], self.starts[b + 1], self.lens[b]
            n = r1 - r0
            if n == 0:
                continue
            if length < n:
                assert bool((got[r0:r1] == 0).all())
                continue
            k, good = V8.cached(*self.k, self.table[b], length)
            v, _ = V8.cached(*self.v, self.table[b], length)
            one = torch.ones(self.pages, self.kvh, self.pt // 16)
            v_codes = V8.cached(self.v[0], one, self.table[b], length)[0]
            zero = torch.zeros_like(self.v[0]) + 56  # the code of 1
            v_scales = V8.cached(zero, self.v[1], self.table[b], length)[0][:, :, 0]
            pos, j = torch.arange(length - n, length)[:, None], torch.arange(length)
            seen = (j <= pos) & good
            if self.window:
                seen &= (j > pos - self.window) | (j < self.sinks)
            any_seen = seen.any(0)
            for h in range(qh):
                kv = h // group
                kk, vv, cc = (torch.where(any_seen[:, None], x[:, kv], torch.zeros_like(x[:, kv])) for x in (k, v, v_codes))
                ss = torch.where(any_seen, v_scales[:, kv], torch.zeros_like(v_scales[:, kv]))
                o, tol = V8.attend(self.q[r0:r1, h].double(), kk, vv, cc, ss, seen)
                err = (got[r0:r1, h] - o).abs()
                assert bool((err <= tol + 1e-30).all()), (b, h, float((err - tol).max()), float((err / (tol + 1e-30)).max()))
                worst = max(worst, float((err / (tol + 1e-30)).max()))
        return worst


HEADS = [(14, 2, 64), (28, 4, 128), (4, 4, 64), (32, 1, 128), (16, 2, 64), (3, 1, 128)]


@pytest.mark.parametrize("q_heads,kvh,D", HEADS)
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 127, 128, 129, 300, 1500])
def test_attention_of_one_token(q_heads, kvh, D, length):
    c = Attend(length, [length - 1], [1], q_heads, kvh, D, 16 if length % 2 else 64)
    c.check(c.run())


@pytest.mark.parametrize("q_heads,kvh,D", HEADS)
@pytest.mark.parametrize("rows", [2, 3, 5, 9, 18, 19, 37, 64, 131, 300])
def test_attention_of_several_rows(q_heads, kvh, D, rows):
    """Drafted tokens and prompt chunks, with and without a context."""
    c = Attend(rows, [0, 77, 129], [rows, 1, max(1, rows - 1)], q_heads, kvh, D, 32)
    c.check(c.run())


@pytest.mark.parametrize("pt", [16, 32, 48, 64, 80, 128, 256])
def test_attention_page_sizes(pt):
    c = Attend(pt, [5, 200, 333, 700], [1, 2, 7, 3], 14, 2, 64, pt)
    c.check(c.run())


@pytest.mark.parametrize("q_heads,kvh,D", [(14, 2, 64), (28, 4, 128)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (48, 4), (127, 1), (128, 128), (129, 130), (300, 17), (64, 5000), (5000, 4),
                                          (2 ** 31 - 1, 2 ** 31 - 1)])
def test_attention_window_and_sinks(q_heads, kvh, D, window, sinks):
    c = Attend(window % 1000 + sinks % 1000, [0, 40, 515, 1300], [3, 1, 40, 9], q_heads, kvh, D, 64, window, sinks)
    c.check(c.run())


@pytest.mark.parametrize("q_heads,kvh,D", [(14, 2, 64), (28, 4, 128)])
def test_attention_window_of_single_tokens(q_heads, kvh, D):
    c = Attend(3, [0, 40, 515, 1300, 2047], [1] * 5, q_heads, kvh, D, 16, 200, 20)
    c.check(c.run())


@pytest.mark.parametrize("rows", [[1] * 70, [1, 0, 3, 0, 0, 2] * 6, [4] * 40])
def test_attention_of_a_batch(rows):
    rng = np.random.default_rng(len(rows))
    ctx = rng.integers(0, 900, len(rows)).tolist()
    c = Attend(len(rows), ctx, rows, 28, 4, 128, 64)
    c.check(c.run())


@pytest.mark.parametrize("rows", [1, 4, 60])
def test_attention_of_a_long_context(rows):
    c = Attend(rows, [9000], [rows], 14, 2, 64, 64)
    c.check(c.run())
    c = Attend(rows, [20011], [rows], 4, 1, 128, 64, 0, 0)
    c.check(c.run())


@pytest.mark.parametrize("q_heads,kvh,D,batch", [(7, 1, 128, 160), (14, 2, 64, 40), (16, 1, 128, 40), (32, 1, 64, 24)])
def test_attention_rings_go_round(q_heads, kvh, D, batch):
    """So many key tiles to a CTA that its rings of tiles go round several times."""
    rng = np.random.default_rng(batch)
    c = Attend(batch, (rng.integers(0, 9000, batch) * (160 / batch)).astype(int).clip(max=18000).tolist(), [1] * batch, q_heads, kvh, D, 64)
    c.check(c.run(), sample=range(0, batch, 7))


def test_attention_codes_of_every_size():
    """Any code and scales that vary over several powers of two: weights and V's scale together set what a row resolves."""
    for seed, rows in ((1, 1), (2, 4), (3, 70)):
        c = Attend(seed, [400, 90], [rows, rows], 8, 2, 64, 32, pool=random_pool, q_scale=0.1, spread=3.0)
        c.check(c.run())


def test_attention_scores_that_grow():
    """Scores rise along the keys, so a row's reference moves again and again; and fall."""
    for rows in (1, 4, 40):
        for sign in (1.0, -1.0):
            c = Attend(rows, [1200], [rows], 8, 2, 64, 64)
            D = 64
            ramp = torch.linspace(0.05, 8.0, 1280)[:, None].expand(1280, D) * sign
            for b in range(-(-c.lens[0] // 64)):
                page = c.table[0, b]
                x = ramp[b * 64:(b + 1) * 64].reshape(1, 4, 16, D).expand(2, 4, 16, D)
                e = torch.ceil(torch.log2(x.abs().amax((-1, -2)) / 448.0))
                c.k[0][page] = (x / torch.exp2(e)[..., None, None]).to(E4M3).reshape(2, 64, D).view(torch.uint8)
                c.k[1][page] = torch.exp2(e)
            c.q = c.q.abs()
            c.q_wide = c.q.reshape(c.q.shape[0], -1)
            c.check(c.run())


def test_attention_of_strided_rows_and_rows_behind_the_last_sequence():
    for rows in (1, 3, 40):
        c = Attend(rows, [100, 300], [rows, rows], 14, 2, 64, 64, extra_rows=5, wide=24)
        out = torch.full((2 * rows + 5, 14, 64), 7.0, dtype=torch.bfloat16, device="cuda")
        assert c.run(out=out) is out
        c.check(out)
        assert bool((out[2 * rows:] == 7.0).all())


def test_attention_of_sequences_without_rows_or_room():
    """No rows; more rows than cached positions (zeros); a length past the table (its pages alone count)."""
    for rows in (1, 5, 40):
        c = Attend(rows, [30, 64, 200, 50], [rows, rows, rows, 0], 14, 2, 64, 16)
        c.lens[0] = rows - 1
        got = c.run()
        c.check(got)
        assert bool((got[:rows] == 0).all())
    c = Attend(2, [64], [1], 14, 2, 64, 16)
    c.table = c.table[:, :3].copy()  # positions 48 .. 64 have no page; 0 .. 47 are seen
    c.check(c.run())


@pytest.mark.parametrize("rows", [1, 4, 40])
def test_attention_pages_outside_the_pool(rows):
    c = Attend(rows, [300, 150, 20], [rows, rows, rows], 28, 4, 128, 16)
    c.table[0, [0, 3, 7, 12]] = [-1, c.pages, 2 ** 31 - 1, -2 ** 31]
    c.table[1, :] = -1  # nothing is seen
    got = c.run()
    c.check(got)
    assert bool((got[rows:2 * rows] == 0).all())


@pytest.mark.parametrize("rows", [1, 4, 9, 40])
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 3)])
def test_attention_cells_that_a_row_does_not_see(rows, window, sinks):
    """NaN codes behind the sequence's end, ahead of the window, in drafted rows
    that earlier ones do not see, and scales of blocks that hold no position."""
    base = Attend(7, [203, 130], [rows, rows], 14, 2, 64, 64, window, sinks)
    want = base.run().clone()
    c = Attend(7, [203, 130], [rows, rows], 14, 2, 64, 64, window, sinks)
    for b in range(2):
        length, low = c.lens[b], c.lens[b] - rows - window + 1 if window else 0
        for j in range(c.table.shape[1] * 64):
            page = c.table[b, j // 64]
            if page < 0:
                continue
            hidden = j >= length or (window and sinks <= j < low)
            for codes, scales in (c.k, c.v):
                if hidden:
                    codes[page, :, j % 64] = 127
                if j % 16 == 0 and (j >= length or (window and j >= sinks and j + 16 <= low)):
                    scales[page, :, j % 64 // 16] = math.nan
    got = c.run()
    assert torch.equal(got, want)
    if rows > 1:  # the last row's own V and K
        for b in range(2):
            j = c.lens[b] - 1
            c.v[0][c.table[b, j // 64], 1, j % 64, 5] = 255
            c.k[0][c.table[b, j // 64], 0, j % 64, 9] = 127
        got = c.run()
        for b in range(2):
            r0, r1 = c.starts[b], c.starts[b + 1]
            assert torch.equal(got[r0:r1 - 1], want[r0:r1 - 1])
            assert bool(torch.isnan(got[r1 - 1, :7]).all())          # K of head 0: the whole row
            assert bool(torch.isnan(got[r1 - 1, 7:, 5]).all())       # V of head 1: one dimension
            rest = [d for d in range(64) if d != 5]
            assert torch.equal(got[r1 - 1, 7:][:, rest], want[r1 - 1, 7:][:, rest])


@pytest.mark.parametrize("ctx", [40, 3000, 30000])
def test_attention_nan_in_the_context_reaches_every_row(ctx):
    for rows in (1, 40):
        c = Attend(ctx, [ctx], [rows], 14, 2, 64, 64)
        j = ctx // 2
        c.v[0][c.table[0, j // 64], 1, j % 64, 5] = 127
        got = c.run()
        assert bool(torch.isnan(got[:, 7:, 5]).all())
        assert not bool(torch.isnan(got[:, :7]).any()) and not bool(torch.isnan(got[:, 7:, 6]).any())


def test_attention_captured_replayed_and_on_another_stream():
    from cheetah_b200 import runtime as R
    for rows in (1, 4, 40):
        c = Attend(rows, [1000, 3000], [rows, rows], 14, 2, 64, 64)
        q = c.q.cuda()
        (kc, ks), (vc, vs) = to_gpu(*c.k), to_gpu(*c.v)
        table, lens, starts = i32(c.table), i32(c.lens), i32(c.starts)
        want = R.attention_kv8(q, kc, vc, ks, vs, table, lens, starts)
        work = torch.full((R.attention_kv8_workspace(64),), 255, dtype=torch.uint8, device="cuda")
        out = torch.empty_like(want)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        other = R.attention_kv8(q, kc, vc, ks, vs, table, lens, starts, workspace=work, stream=s)
        torch.cuda.synchronize()
        assert torch.equal(other, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            R.attention_kv8(q, kc, vc, ks, vs, table, lens, starts, out=out, workspace=work)
        for _ in range(3):
            out.zero_()
            work.fill_(255)
            graph.replay()
            assert torch.equal(out, want)


def test_attention_is_the_same_every_time():
    c = Attend(5, [5000, 100, 9000], [4, 60, 1], 28, 4, 128, 64)
    first = c.run()
    for _ in range(3):
        assert torch.equal(c.run(), first)


@pytest.mark.parametrize("q_heads,kvh,D", [(28, 4, 128), (14, 2, 64), (16, 1, 128), (32, 1, 64)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 5)])
def test_attention_of_a_batch_of_any_rows(q_heads, kvh, D, window, sinks):
    """Items of one row up to two full tiles of rows side by side, whole and cut,
    one without room and some without rows among them."""
    rows = [1, 40, 0, 9, 130, 2, 5, 18, 4, 1, 64, 3]
    ctx = [2000, 0, 70, 513, 1000, 3000, 126, 900, 5, 0, 1, 2500]
    c = Attend(q_heads + window, ctx, rows, q_heads, kvh, D, 64, window, sinks)
    c.lens[6] = 4
    c.check(c.run())


def test_attention_calls_that_overlap():
    """Two captured calls on two streams, each with a workspace of its own."""
    from cheetah_b200 import runtime as R
    calls, keep = [], []
    for rows, D in ((1, 64), (30, 128)):
        c = Attend(rows, [3000, 7000], [rows, rows], 14, 2, D, 64)
        (kc, ks), (vc, vs) = to_gpu(*c.k), to_gpu(*c.v)
        args = (c.q.cuda(), kc, vc, ks, vs, i32(c.table), i32(c.lens), i32(c.starts))
        want = R.attention_kv8(*args)
        out = torch.empty_like(want)
        work = torch.empty(R.attention_kv8_workspace(D), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(4):
                R.attention_kv8(*args, out=out, workspace=work)
        calls.append((graph, torch.cuda.Stream(), out, want))
        keep.append((args, work))
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, stream, _, _ in calls:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, out, want in calls:
        assert torch.equal(out, want)


def test_attention_join_after_a_wait_that_gave_up(tmp_path):
    """The join alone, on a list of split items in which one CTA has given up:
    every row is NaN, those behind the last sequence stay. Without one that has,
    and without anything to join, it writes nothing."""
    import ctypes as C
    import subprocess
    from pathlib import Path
    from cheetah_b200 import build
    here = Path(__file__).resolve().parent
    lib = tmp_path / "kv8_join.so"
    subprocess.run([build.nvcc(), *build.ARCH_FLAGS, "-O1", "-std=c++17", "-shared", "-Xcompiler", "-fPIC", "-I", str(build.CSRC),
                    "-I", str(build.INCLUDE), "--expt-relaxed-constexpr", "-o", str(lib), str(here / "kv8_join_entry.cu")],
                   check=True, capture_output=True, timeout=300)
    join = C.CDLL(str(lib)).kv8_join
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


@pytest.mark.parametrize("rows", [1, 3, 40])
@pytest.mark.parametrize("window,sinks", [(0, 0), (16, 5), (16, 2 ** 31 - 1), (2 ** 31 - 1, 0)])
def test_attention_of_the_largest_length(rows, window, sinks):
    """A length of 2^31 - 1 over a table of 96 positions: the rows see what those of
    length 5000 do: of a short window its sinks alone."""
    outs = []
    for length in (5000, 2 ** 31 - 1):
        c = Attend(rows, [96 - rows], [rows], 14, 2, 64, 32, window, sinks)
        c.lens = [length]
        outs.append(c.run().float())
    # Two roundings of the output and of two orders of f32 sums.
    assert bool(((outs[0] - outs[1]).abs() <= 2.0 ** -7 * outs[0].abs() + 2.0 ** -20).all())
    if window == 16:
        c = Attend(rows, [96 - rows], [rows], 14, 2, 64, 32, window, 0)
        c.lens = [2 ** 31 - 1]
        assert bool((c.run() == 0).all())


# ---- verify_drafts --------------------------------------------------------------

def verify_case(seed, drafts, vocab, given=True, extra=3, wide=0, agree=0.4):
    g = torch.Generator().manual_seed(seed)
    rows = [d + 1 for d in drafts]
    total = sum(rows) + extra
    x = 2.0 * torch.randn(total, vocab, generator=g)
    p = torch.softmax(x, -1)
    q = torch.softmax(x + agree * torch.randn(total, vocab, generator=g), -1)
    drawn = torch.multinomial(q, 1, generator=g)[:, 0]
    tokens = torch.cat([drawn.new_zeros(1), drawn[:-1]]).to(torch.int32)
    return dict(p=p, q=q if given else None, tokens=tokens, row_starts=[0] + np.cumsum(rows).tolist(),
                accept_u=torch.rand(total, generator=g), sample_u=torch.rand(len(drafts), generator=g), wide=wide)


def check_verify(c):
    from cheetah_b200 import runtime as R

    def strided(a):
        if a is None or not c["wide"]:
            return a if a is None else a.cuda()
        return torch.cat([a, torch.full((a.shape[0], c["wide"]), 9.0)], 1).cuda()[:, :a.shape[1]]

    out = torch.full_like(c["tokens"], 77).cuda()
    got = R.verify_drafts(strided(c["p"]), strided(c["q"]), c["tokens"].cuda(), i32(c["row_starts"]), c["accept_u"].cuda(),
                          c["sample_u"].cuda(), out_tokens=out)
    assert got.tokens is out
    accepted, tokens = V8.verify(c["p"].numpy(), None if c["q"] is None else c["q"].numpy(), c["tokens"].tolist(), c["row_starts"],
                                 c["accept_u"].tolist(), c["sample_u"].tolist(), [77] * len(c["tokens"]))
    assert got.accepted.tolist() == accepted
    assert out.tolist() == tokens
    return accepted


@pytest.mark.parametrize("vocab", [1, 2, 3, 31, 1000, 1023, 1025, 4099, 32001, 151936])
@pytest.mark.parametrize("given", [True, False])
def test_verify_drafts(vocab, given):
    check_verify(verify_case(vocab, [4, 0, 1, 7], vocab, given))
    check_verify(verify_case(vocab + 1, [3], vocab, given, extra=0, wide=3))


@pytest.mark.parametrize("batch,vocab", [(70, 5000), (300, 2049), (1100, 700)])
def test_verify_drafts_of_a_batch(batch, vocab):
    rng = np.random.default_rng(batch)
    accepted = check_verify(verify_case(batch, rng.integers(0, 9, batch).tolist(), vocab, wide=1))
    assert min(accepted) == 0 and max(accepted) > 3


def test_verify_drafts_long_runs():
    """More drafts than a warp looks at together; all kept, and one dropped far on."""
    c = verify_case(1, [100, 33, 32, 31], 50, agree=0.0)
    c["accept_u"].fill_(0.5)
    assert check_verify(c) == [100, 33, 32, 31]
    c["accept_u"][70] = 0.999999
    c["q"][70] = c["p"][70].roll(1)
    c["tokens"][71] = int((c["q"][70] / c["p"][70]).argmax())
    assert check_verify(c)[0] == 70


def test_verify_drafts_first_and_last_token():
    """Numbers at the ends of [0, 1): the first and the last token of positive weight."""
    for vocab in (5, 6000):
        c = verify_case(2, [0, 0], vocab)
        c["p"][0, :3] = 0.0
        c["p"][1, -2:] = 0.0
        c["sample_u"] = torch.tensor([0.0, 1.0 - 2.0 ** -24])
        check_verify(c)
        c["sample_u"] = torch.tensor([1.0, math.nan])
        from cheetah_b200 import runtime as R
        got = R.verify_drafts(c["p"].cuda(), None, c["tokens"].cuda(), i32(c["row_starts"]), c["accept_u"].cuda(), c["sample_u"].cuda())
        assert got.tokens[0].item() == vocab - 1 and got.tokens[1].item() == vocab - 3


def test_verify_drafts_exact_comparison():
    """u q = p is dropped, a step below is kept."""
    c = verify_case(3, [1, 1], 8)
    c["p"][0], c["q"][0] = 1 / 8, 1 / 4
    c["p"][2], c["q"][2] = 1 / 8, 1 / 4
    c["accept_u"][0], c["accept_u"][2] = 0.5, 0.5 - 2.0 ** -25
    assert check_verify(c) == [0, 1]


def test_verify_drafts_rows_without_a_distribution():
    """All weights zero (the residual falls back to p), NaN and negative ones, infinities, drafts outside the vocabulary."""
    for given in (True, False):
        c = verify_case(4, [2] * 9, 3000, given)
        c["accept_u"].fill_(1.0 - 2.0 ** -24)
        c["p"][0] = 0.0                                      # token -1
        if given:
            c["q"][3] = 2 * c["p"][3]                        # nothing left: p itself
        c["p"][6] = math.nan
        c["p"][9, ::2] = math.nan
        c["p"][12, ::3] = -1.0
        c["p"][15, 5] = math.inf
        c["tokens"][16] = 4                                  # not the infinite one
        c["tokens"][19], c["tokens"][22] = -1, 3000
        c["p"][24] = 0.0
        c["p"][24, 1234] = 0.25
        c["tokens"][25] = 1234                               # the only weight is the dropped draft's, or kept
        c["accept_u"][24] = 1.0 if not given else 0.5
        check_verify(c)


def test_verify_drafts_sequences_without_rows():
    from cheetah_b200 import runtime as R
    c = verify_case(5, [1, 2], 100, extra=4)
    starts = [0, 0, 2, 2, 5, 5]
    u = torch.rand(5)
    out = torch.full_like(c["tokens"], 77).cuda()
    got = R.verify_drafts(c["p"].cuda(), c["q"].cuda(), c["tokens"].cuda(), i32(starts), c["accept_u"].cuda(), u.cuda(), out_tokens=out)
    accepted, tokens = V8.verify(c["p"].numpy(), c["q"].numpy(), c["tokens"].tolist(), starts, c["accept_u"].tolist(), u.tolist(),
                                 [77] * len(c["tokens"]))
    assert got.accepted.tolist() == accepted and accepted[0] == accepted[2] == accepted[4] == -1
    assert out.tolist() == tokens and tokens[5:] == [77] * 4


def test_verify_drafts_keeps_the_targets_distribution():
    """Over many sequences, the first token behind is distributed as the target says: each frequency within 5 deviations."""
    from cheetah_b200 import runtime as R
    g = torch.Generator(device="cuda").manual_seed(6)
    B, vocab = 60000, 7
    p = torch.tensor([0.3, 0.05, 0.0, 0.25, 0.1, 0.2, 0.1], device="cuda")
    q = torch.tensor([0.1, 0.25, 0.1, 0.05, 0.2, 0.3, 0.0], device="cuda")
    drawn = torch.multinomial(q, B, replacement=True, generator=g)
    tokens = torch.stack([torch.zeros_like(drawn), drawn], 1).flatten().to(torch.int32)
    got = R.verify_drafts(p.repeat(2 * B, 1), q.repeat(2 * B, 1), tokens, i32(np.arange(B + 1) * 2),
                          torch.rand(2 * B, device="cuda", generator=g), torch.rand(B, device="cuda", generator=g))
    counts = torch.bincount(got.tokens[::2].long(), minlength=vocab).double().cpu()
    want = p.double().cpu() * B
    assert bool(((counts - want).abs() <= 5 * torch.sqrt(want * (1 - p.double().cpu())) + 1e-9).all()), counts


# ---- the operators in a row -----------------------------------------------------

def test_a_serving_step_over_an_8_bit_cache():
    """Two steps of page slots, append, attention and the drafts' test, eager and
    captured: each output against its reference on what the step before left."""
    from cheetah_b200 import runtime as R
    g = torch.Generator(device="cuda").manual_seed(11)
    q_heads, kvh, D, pt, vocab = 8, 2, 64, 32, 501
    cached, new = [70, 5, 0], [3, 4, 1]
    num_pages, width, max_tokens = 24, 6, 10
    table = np.full((3, width), -1)
    table[0, :3], table[1, :1] = [4, 9, 2], [7]
    table = i32(table)
    free, free_count = i32([11, 3, 5, 8, 0, 1]), i32([6])
    k_codes = torch.randint(0, 127, (num_pages, kvh, pt, D), generator=g, device="cuda").to(torch.uint8).view(E4M3)
    v_codes = k_codes.clone()
    k_scales = torch.full((num_pages, kvh, pt // 16), 2.0 ** -8, device="cuda")
    v_scales = k_scales.clone()
    qkv = torch.randn(max_tokens, q_heads + 2 * kvh, D, generator=g, device="cuda").to(torch.bfloat16)
    angle = torch.rand(200, D // 2, generator=g, device="cuda") * 6.0
    cos, sin = angle.cos(), angle.sin()
    probs = torch.softmax(torch.randn(max_tokens, vocab, generator=g, device="cuda"), -1)
    draft = torch.softmax(torch.randn(max_tokens, vocab, generator=g, device="cuda"), -1)
    tokens = torch.randint(0, vocab, (max_tokens,), generator=g, device="cuda").to(torch.int32)
    u, us = torch.rand(max_tokens, generator=g, device="cuda"), torch.rand(3, generator=g, device="cuda")
    lens, adds = i32(cached), i32(new)
    work = torch.empty(R.attention_kv8_workspace(D), dtype=torch.uint8, device="cuda")

    def step():
        m = R.page_slots(lens, adds, free, free_count, table, num_pages, pt, max_tokens)
        q = R.qk_norm_rope_kv8(qkv, q_heads, kvh, m.positions, m.slots, cos, sin, k_codes, v_codes, k_scales, v_scales)
        o = R.attention_kv8(q, k_codes, v_codes, k_scales, v_scales, table, m.seq_lens, m.row_starts, workspace=work)
        v = R.verify_drafts(probs, draft, tokens, m.row_starts, u, us)
        k8 = R.kv8_read(k_codes, v_codes, k_scales, v_scales, m.slots, dtype=torch.float32)
        return m, q, o, v, k8

    before = [t.clone() for t in (k_codes.view(torch.uint8), v_codes.view(torch.uint8), k_scales, v_scales, table)]
    m, q, o, v, k8 = step()
    total = sum(new)
    c = Attend(0, cached, new, q_heads, kvh, D, pt)
    c.table, c.pages = table.cpu().numpy(), num_pages
    c.k, c.v = (k_codes.view(torch.uint8).cpu(), k_scales.cpu()), (v_codes.view(torch.uint8).cpu(), v_scales.cpu())
    c.q = q[:total].cpu()
    c.check(o[:total])
    # The appended values read back: within half a step of what was appended.
    x = qkv[:total, q_heads + kvh:].float()
    at = m.slots[:total].long()
    scale = v_scales[at // pt, :, at % pt // 16]
    assert bool(((k8[1][:total] - x).abs() <= x.abs() * 2.0 ** -4 + scale[..., None] * 2.0 ** -10).all())
    assert bool((k8[0][total:] == 0).all())
    accepted, kept = V8.verify(probs.cpu().numpy(), draft.cpu().numpy(), tokens.tolist(), m.row_starts.tolist(), u.tolist(), us.tolist(),
                               v.tokens.tolist())
    assert v.accepted.tolist() == accepted and v.tokens.tolist() == kept

    eager = [t.clone() for t in (q[:total], o[:total], v.accepted, v.tokens[:total], k_codes.view(torch.uint8), v_codes.view(torch.uint8))]
    state = (k_codes.view(torch.uint8), v_codes.view(torch.uint8), k_scales, v_scales, table)
    for t, b in zip(state, before):
        t.copy_(b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m, q, o, v, k8 = step()
    for _ in range(2):
        for t, b in zip(state, before):
            t.copy_(b)
        graph.replay()
        for a, b in zip(eager, (q[:total], o[:total], v.accepted, v.tokens[:total], k_codes.view(torch.uint8), v_codes.view(torch.uint8))):
            assert torch.equal(a, b)
