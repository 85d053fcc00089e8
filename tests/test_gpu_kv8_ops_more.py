"""The operators over an 8-bit cache on the GPU, at what `test_gpu_kv8_ops`
leaves out: ends of short segments, values that only a caller can have set, rows
whose softmax has one heavy key over a long tail."""

import math

import pytest

from tests import kv8_peaked_ref as VP
from tests import kv8_ref as V8
from tests.test_gpu_kv8_ops import Attend, E4M3, _cuda, check_append, random_pool  # noqa: F401  (_cuda is the fixture)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("q_heads,kvh,D", [(7, 1, 128), (14, 2, 64), (16, 1, 128), (16, 1, 64)])
def test_attention_of_segments_whose_last_tile_moves_the_reference(q_heads, kvh, D):
    """A group's first tile of a segment sets its reference. With one to three tiles to
    a sequence every group's last tile does so too, and its maxima and the segment's sums
    come one after the other: many such segments, each time the same rows and right."""
    c = Attend(q_heads + D, [1 + 7 * i % 380 for i in range(300)], [1] * 300, q_heads, kvh, D, 64, q_scale=4.0)
    first = c.run()
    c.check(first, sample=range(0, 300, 9))
    for _ in range(20):
        assert torch.equal(c.run(), first)


@pytest.mark.parametrize("q_heads,kvh,D,rows", [(14, 2, 64, 2), (28, 4, 128, 2), (14, 2, 64, 12), (28, 4, 128, 16), (10, 2, 128, 37), (14, 2, 64, 200)])
@pytest.mark.parametrize("ctx", [30, 4000])
def test_attention_of_rows_beside_lanes_that_hold_none(q_heads, kvh, D, rows, ctx):
    """Items whose tile has lanes without a row, whole and cut, with a NaN in V that only
    some rows see: the lanes of a warp part between the loads of a result's columns."""
    c = Attend(rows + ctx, [ctx, ctx + 3], [rows, rows], q_heads, kvh, D, 64, extra_rows=1)
    base = c.run()
    c.check(base, sample=[0])
    group, at = q_heads // kvh, rows // 2
    for b in range(2):
        j = c.lens[b] - rows + at
        for d in (3, D - 2):
            c.v[0][c.table[b, j // 64], kvh - 1, j % 64, d] = 127
    got = c.run()
    hit = torch.zeros(got.shape, dtype=torch.bool, device="cuda")
    for b in range(2):
        for d in (3, D - 2):
            hit[c.starts[b] + at:c.starts[b + 1], q_heads - group:, d] = True
    hit[c.starts[2]:] = torch.isnan(got[c.starts[2]:])  # rows behind the last sequence are not written
    assert bool(torch.isnan(got[hit]).all())
    assert torch.equal(got[:c.starts[2]][~hit[:c.starts[2]]], base[:c.starts[2]][~hit[:c.starts[2]]])


def peaked(seed, ctx, rows, q_heads, kvh, D, weight, heavy, common, window=0, sinks=0, sink_v=1.0, noise=0.0, extra=0):
    """A call whose every row gives the key `heavy` about `weight` of its softmax and
    spreads the rest over the others; V = common + a normal part, that of the heavy key
    times sink_v."""
    c = Attend(seed, [ctx], [rows], q_heads, kvh, D, 64, window, sinks, extra_rows=extra)
    g = torch.Generator().manual_seed(seed)
    length = c.lens[0]
    # q and the heavy key along one direction, the other keys across it (and some noise).
    u = torch.sign(torch.randn(D, generator=g))
    n = min(length, window + sinks) if window else length
    score = math.log(weight / (1.0 - weight) * n)  # of the heavy key above the others
    c.q = (u * 2.0).expand_as(c.q).to(torch.bfloat16).contiguous()
    c.q_wide = c.q.reshape(c.q.shape[0], -1)
    k = noise * torch.randn(length, kvh, D, generator=g)
    k -= (k @ u)[..., None] * u / D * (0.0 if noise else 1.0)
    k[heavy] = u * (score / (2.0 * math.sqrt(D)))
    v = common + torch.randn(length, kvh, D, generator=g)
    v[heavy] *= sink_v
    for (codes, scales), x in ((c.k, k), (c.v, v)):
        for i in range(-(-length // 64)):
            page = c.table[0, i]
            part = torch.zeros(64, kvh, D)
            part[:min(64, length - i * 64)] = x[i * 64:(i + 1) * 64]
            part = part.transpose(0, 1).reshape(kvh, 4, 16, D)
            e = torch.ceil(torch.log2(part.abs().amax((-1, -2)).clamp(min=2.0 ** -55) / 448.0))
            codes[page] = (part / torch.exp2(e)[..., None, None]).to(E4M3).reshape(kvh, 64, D).view(torch.uint8)
            scales[page] = torch.exp2(e)
    return c


def check_peaked(c, heads, sequences=(0,)):
    """Against the reference, under its own tolerance: relative to each weight. (All
    sequences share pages, length and number of rows.)"""
    got = c.run().cpu().double()
    length, n = c.lens[0], c.starts[1]
    group = c.q.shape[1] // c.kvh
    k, _ = V8.cached(*c.k, c.table[0], length)
    v, _ = V8.cached(*c.v, c.table[0], length)
    codes = V8.cached(c.v[0], torch.ones_like(c.v[1]), c.table[0], length)[0]
    scales = V8.cached(torch.zeros_like(c.v[0]) + 56, c.v[1], c.table[0], length)[0][:, :, 0]
    pos, j = torch.arange(length - n, length)[:, None], torch.arange(length)
    seen = j <= pos
    if c.window:
        seen &= (j > pos - c.window) | (j < c.sinks)
    some = torch.arange(n) if n <= 8 else torch.tensor([r for r in sorted({0, 1, 17, 18, 36, n // 2, n - 2, n - 1}) if r < n])
    for h in heads:
        kv = h // group
        for b in sequences:
            rows = c.starts[b] + some
            o, tol = VP.attend(c.q[rows, h].double(), k[:, kv], v[:, kv], codes[:, kv], scales[:, kv], seen[some])
            err = (got[rows, h] - o).abs()
            assert bool((err <= tol).all()), (h, b, float((err / tol).max()), float((err.norm() / o.norm())))


@pytest.mark.parametrize("rows,q_heads,kvh,D", [(1, 7, 1, 128), (1, 16, 1, 64), (4, 4, 1, 64), (4, 4, 1, 128), (9, 3, 1, 128),
                                                 (12, 4, 1, 64), (40, 7, 1, 128), (300, 7, 1, 64)])
@pytest.mark.parametrize("ctx", [4000, 16300, 32700])
@pytest.mark.parametrize("weight", [0.5, 0.7, 0.9, 0.97])
def test_attention_of_a_heavy_key_and_a_long_tail(rows, q_heads, kvh, D, ctx, weight):
    """The first key holds most of the weight, the others spread the rest: an attention sink."""
    check_peaked(peaked(ctx + rows, ctx, rows, q_heads, kvh, D, weight, 0, 0.5), [0, q_heads - 1])


@pytest.mark.parametrize("rows,D", [(1, 64), (4, 128), (9, 128), (40, 64), (300, 128)])
@pytest.mark.parametrize("weight", [0.8, 0.97])
@pytest.mark.parametrize("window,sinks", [(0, 0), (8192, 4)])
def test_attention_of_a_sink_without_a_value(rows, D, weight, window, sinks):
    """A sink whose V is near zero: the output is the tail's. With a window the sinks stay visible."""
    check_peaked(peaked(rows, 20000, rows, 4, 1, D, weight, 0, 0.3, window, sinks, sink_v=2.0 ** -7, noise=0.4), [1])


@pytest.mark.parametrize("rows,D", [(1, 128), (4, 64), (9, 64), (40, 128), (300, 64)])
@pytest.mark.parametrize("heavy", [5000, 11999])
def test_attention_of_a_heavy_key_behind_the_tail(rows, D, heavy):
    """The heavy key comes after others, the last ahead of the rows: the tail is rescaled, not lost."""
    check_peaked(peaked(rows + heavy, 12000, rows, 4, 1, D, 0.9, heavy, 0.5, noise=0.2), [0, 3])


@pytest.mark.parametrize("rows,q_heads,D", [(1, 7, 128), (1, 16, 64), (4, 7, 128), (9, 7, 64), (18, 7, 128), (36, 7, 64)])
@pytest.mark.parametrize("ctx,weight", [(8000, 0.9), (32700, 0.7), (32700, 0.95)])
def test_attention_of_a_heavy_key_in_items_that_one_cta_walks_through(rows, q_heads, D, ctx, weight):
    """So many sequences (over the same pages) that a CTA has whole items: one reference
    from the heavy key to the end of the tail."""
    c = peaked(rows + D, ctx, rows, q_heads, 1, D, weight, 0, 0.5, noise=0.1)
    copies = 160
    c.table, c.lens, c.starts = c.table.repeat(copies, 0), c.lens * copies, [rows * i for i in range(copies + 1)]
    c.q = c.q.repeat(copies, 1, 1)
    c.q_wide = c.q.reshape(c.q.shape[0], -1)
    check_peaked(c, [0, q_heads - 1], (0, 80, 159))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("old", [2.0 ** 126, 2.0 ** 127])
def test_append_behind_the_largest_scales(old, dtype):
    """A scale that only a caller can have set, whose inverse is the least normal number or none."""
    g = torch.Generator().manual_seed(8)
    kvh, D, pt, pages = 2, 128, 16, 3
    x = (torch.randn(3, 6, D, generator=g) * 1e38).clamp(-3e38, 3e38).to(dtype)
    pools = [random_pool(g, pages, kvh, pt, D) for _ in range(2)]
    for _, s in pools:
        s.fill_(old)
    slots = torch.tensor([16 + 5, 16 + 6, 16 + 7], dtype=torch.int32)
    cos, sin = torch.ones(4, D // 2), torch.zeros(4, D // 2)
    check_append(x, 2, kvh, torch.zeros(3, dtype=torch.int32), slots, cos, sin, [None, None], pools, 1e-6, 4)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_kv8_read_rounds_a_product_once(dtype):
    """Scales that are no powers of two: the product of a code's 4 bits and a scale's 24
    does not fit f32, and bf16 of the rounded product is not always that of the product."""
    from cheetah_b200 import runtime as R
    kvh, D, pt = 1, 64, 16
    # All codes, and scales for which code * scale lies just beside the middle of two bf16:
    # (middle + 2^-20) / 1.125, so that the product rounded to f32 is the middle itself for some.
    g = torch.Generator().manual_seed(4)
    pages = 512
    codes = torch.randint(0, 127, (pages, kvh, pt, D), generator=g).to(torch.uint8)
    odd = 2 * torch.randint(0, 128, (pages,), generator=g) + 257
    scales = (odd.double() / 256 / (1 + torch.randint(1, 8, (pages,), generator=g).double() / 8)).float().reshape(pages, 1, 1)
    want = (codes.view(E4M3).double() * scales.double()[..., None])
    slots = torch.arange(pages * pt, dtype=torch.int32, device="cuda")
    k, v = R.kv8_read(*[codes.cuda().view(E4M3)] * 2, *[scales.cuda()] * 2, slots, dtype=dtype)
    got = k.cpu().reshape(pages, pt, kvh, D).transpose(1, 2)
    # The two neighbours in the output's type: the result is the nearer one.
    step = want.abs() * torch.finfo(dtype).eps
    err = (got.double() - want).abs()
    for other in (torch.nextafter(got, torch.full_like(got, math.inf)), torch.nextafter(got, torch.full_like(got, -math.inf))):
        assert bool((err <= (other.double() - want).abs()).all())
    assert bool((err <= step).all()) and torch.equal(k, v)


@pytest.mark.parametrize("q_heads,kvh,D,rows", [(7, 1, 128, 3), (7, 1, 128, 9), (14, 2, 64, 17)])
def test_attention_of_items_with_one_key_tile(q_heads, kvh, D, rows):
    """One job to a segment, so the second group has none and waits for its end alone:
    many such segments, each time the same rows and right."""
    c = Attend(rows + D, [(5 * i) % (128 - rows) for i in range(200)], [rows] * 200, q_heads, kvh, D, 64, q_scale=4.0)
    first = c.run()
    c.check(first, sample=range(0, 200, 23))
    for _ in range(20):
        assert torch.equal(c.run(), first)


@pytest.mark.parametrize("low,high", [(-100, -100), (100, 100), (-50, 50), (-100, 0), (0, 100)])
@pytest.mark.parametrize("rows,q_heads,kvh,D", [(1, 7, 1, 128), (4, 4, 1, 64), (40, 7, 1, 128), (5, 7, 1, 64)])
def test_attention_of_v_scales_at_the_ends_of_their_range(rows, q_heads, kvh, D, low, high):
    """The sum of the weights counts keys whose V is 2^100 smaller than others', and
    neither end of the range overflows or vanishes."""
    c = Attend(rows + D, [900], [rows], q_heads, kvh, D, 64)
    g = torch.Generator().manual_seed(rows)
    pick = torch.rand(c.v[1].shape, generator=g) < 0.5
    c.v[1][:] = torch.where(pick, torch.tensor(2.0 ** low), torch.tensor(2.0 ** high))
    check_peaked(c, [0, q_heads - 1])
