"""Four-bit operators at the ends of their types' ranges, and where scales and codes are far from even."""
import math

import numpy as np
import pytest

import four_reference as R
from test_gpu_fourbit import Sequences, TYPES, check_product, double, ids, matrix, rng

torch = pytest.importorskip("torch")

from darknet_b200 import fourbit as F  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("n, k, group, rows", [(40, 300, 32, 1), (40, 300, 64, 5), (70, 1000, 128, 13), (8300, 16200, 128, 9)])
def test_products_of_the_largest_rows(dtype, n, k, group, rows):
    """Values of up to 2^127, neighbours of opposite signs, by weights of some 2^-13: what comes out is far inside the type's range."""
    m = matrix(n, k, group, n)
    m.scales.mul_(2.0 ** -13)
    x = torch.rand(rows, k, generator=rng(k)).mul(2.0 ** 127).to(dtype).cuda()
    x[:, 0] = 2.0 ** 127
    x[:, 1::2] = -x[:, :k // 2 * 2:2]
    y = F.forward_connected4(m, x)
    assert torch.isfinite(y).all()
    picked = torch.arange(0, n, max(1, n // 40)).cuda()
    check_product(F.Matrix4(m.codes[picked].contiguous(), m.scales[picked].contiguous(), k, group), x, y[:, picked])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("n, k, group, rows", [(40, 300, 32, 1), (40, 300, 64, 5), (70, 1000, 128, 13), (8300, 16200, 128, 9)])
def test_products_of_the_largest_rows_of_one_sign(dtype, n, k, group, rows):
    """The sum of a group's values is beyond fp32; times weights of both signs, of some 2^-15, nothing is."""
    m = matrix(n, k, group, n)
    m.scales.mul_(2.0 ** -15)
    x = (0.5 + torch.rand(rows, k, generator=rng(k)) / 2).mul(2.0 ** 127).to(dtype).cuda()
    y = F.forward_connected4(m, x)
    assert torch.isfinite(y).all()
    picked = torch.arange(0, n, max(1, n // 40)).cuda()
    check_product(F.Matrix4(m.codes[picked].contiguous(), m.scales[picked].contiguous(), k, group), x, y[:, picked])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=ids)
@pytest.mark.parametrize("group, rows", [(32, 1), (64, 3), (128, 1), (128, 11)])
def test_products_around_the_middle_code(dtype, group, rows):
    """Codes 9 and 7 of neighbours whose values are equal and positive: sums around the middle code never get far from 0, the result, and what
    the tensor cores cut off of them is at most 2^-23 of the 32 that 16 values below 2 come to: after each of 4096 / 16 instructions (twice
    that in two parts).  Sums of codes 0..15 come to 300 a group of 128, and all that is cut off has one sign."""
    n, k = 40, 4096
    codes = torch.full((n, k // 2), 9 | 7 << 4, dtype=torch.uint8)
    scales = torch.tensor([1.0, -8.0]).half().expand(n, k // group, 2).contiguous()
    m = F.Matrix4(codes.cuda(), scales.cuda(), k, group)
    x = (1 + torch.rand(rows, k // 2, generator=rng(group)) * 0.99) * 2.0 ** -torch.randint(0, 11, (rows, k // 2), generator=rng(1)).float()
    x = x.to(dtype).repeat_interleave(2, 1).cuda()
    y = double(F.forward_connected4(m, x))
    assert (np.abs(y) <= (2 if dtype == torch.float32 else 1) * k / 16 * 2.0 ** -23 * 32).all(), np.abs(y).max()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("share, dim, group", [(1, 64, 32), (5, 128, 128), (12, 96, 32)])
def test_attention_of_the_largest_queries(dtype, share, dim, group):
    """Queries of up to 2^126.  The keys of one position point along them and the others do not: that position is all there is.  Keys that are
    all 0: the mean of the values."""
    s = Sequences([70, 40], 1, dim, group, 16, seed=dim)
    c = s.cache
    q = (torch.rand(2, 1, share, dim, generator=rng(1)) + 0.5).mul(2.0 ** 125).to(dtype).cuda()
    c.k_codes.zero_()
    c.k_scales.zero_()
    table, lengths = s.device()
    every = [[(s.table[b][at // 16], at % 16) for at in range(s.lengths[b])] for b in range(2)]
    _, _, v, v_scales = s.buffers()
    held = [np.stack([R.values(v[p, 0, i], v_scales[p, 0, i], group, dim)[0] for p, i in places]) for places in every]
    mean = double(F.attend4(c, q, table, lengths))
    for b in range(2):
        # 70 weights of 1: fp32 sums, and one rounding
        assert (np.abs(mean[b, 0] - held[b].mean(0)) <= np.abs(held[b]).max() * 2.0 ** -8 * (1 if dtype == torch.bfloat16 else 2.0 ** -10)).all()
    for b, at in ((0, 37), (1, 39)):
        page, place = every[b][at]
        c.k_scales[page, 0, place, :, 1] = 2.0 ** -20
    one = double(F.attend4(c, q, table, lengths))
    for b, at in ((0, 37), (1, 39)):
        assert (np.abs(one[b, 0] - held[b][at]) <= np.abs(held[b][at]).max() * 2.0 ** -8 * (1 if dtype == torch.bfloat16 else 2.0 ** -10)).all()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("tokens, share, dim, group", [(1, 8, 64, 32), (1, 3, 128, 128), (5, 5, 128, 64), (1, 2, 256, 64)])
def test_equal_values_average_to_themselves(dtype, tokens, share, dim, group):
    """Whatever the weights are: every output is the type's value next to the values' own.  Errors: a weight times a scale as two fp16 parts
    (2^-22), at most 40 positions' 2^-31 of the largest where fp16 runs out of bits, and fp32 sums of at most 32 links (2^-23 each) of
    |low + 8 s| + s |code - 8|; a value that lies as near as that to the middle of two of the type's may go either way."""
    s = Sequences([40, 9, 3], 2, dim, group, 16, seed=tokens + dim)
    c = s.cache
    for b in range(3):
        pages = [p for p in s.table[b] if p >= 0]
        c.v_codes[pages] = c.v_codes[pages[0], :, :1].clone()
        c.v_scales[pages] = c.v_scales[pages[0], :, :1].clone()
    q = torch.randn(3, tokens, 2 * share, dim, generator=rng(2)).to(dtype).cuda()
    table, lengths = s.device()
    got = F.attend4(c, q, table, lengths).cpu()
    _, _, codes, scales = s.buffers()
    for b in range(3):
        v, size = (torch.from_numpy(x) for x in R.values(codes[s.table[b][0], :, 0], scales[s.table[b][0], :, 0], group, dim, 8))      # [head][dim]
        tolerance = size * (2.0 ** -22 + 40 * 2.0 ** -31 + 32 * 2.0 ** -23)
        low, high = ((v + way * tolerance).to(dtype).repeat_interleave(share, 0) for way in (-1, 1))
        for row in got[b, max(0, tokens - s.lengths[b]):]:
            assert ((row >= low) & (row <= high)).all()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("dim, group, share", [(32, 32, 1), (128, 128, 1), (128, 64, 20), (256, 128, 2)])
def test_long_sums_of_codes_far_from_the_middle(dtype, dim, group, share):
    """60000 positions by one CTA, all of weight 1 (the queries are 0), codes 2 to 4 with low = -3 * scale, as a group has them whose other
    channels are loud: sums around code 8 that come to five scales a position, of which the result is a thousandth.

    Errors: weights and scales are exact.  An fp32 sum that grows evenly to S in n additions is off by at most 2^-23 / sqrt(12) * S * sqrt(n / 3)
    (one standard deviation; every addition rounds to nearest), n = 60000 / 32 / 4 additions of a warp, four of which are averaged: six
    deviations are 1.3e-6 S, below 2^-19 of |low + 8 s| + s |code - 8|.  The sums of low have four times the additions in each of 8 lanes of
    a warp, which is less.  One rounding of the result."""
    batch, kv_heads = 160, 4
    s = Sequences([60000], kv_heads, dim, group, 256, seed=1)
    c = s.cache
    even, odd = (torch.randint(2, 5, c.v_codes.shape, generator=rng(i), dtype=torch.uint8) for i in (1, 2))
    c.v_codes.copy_((even | odd << 4).cuda())
    c.v_scales[..., 1] = -3 * c.v_scales[..., 0]
    table, lengths = s.device()
    q = torch.zeros(batch, 1, kv_heads * share, dim, dtype=dtype, device="cuda")
    got = F.attend4(c, q, table.expand(batch, -1).contiguous(), lengths.expand(batch).contiguous())
    assert (got == got[:1]).all()
    got = double(got[0, 0]).reshape(kv_heads, share, dim)
    codes, scales = (t[torch.tensor(s.table[0]).cuda()].transpose(0, 1).flatten(1, 2)[:, :60000].cpu().numpy() for t in (c.v_codes, c.v_scales))
    for h in range(kv_heads):
        v, size = R.values(codes[h], scales[h], group, dim, 8)
        want, bound = v.mean(0), size.mean(0) * 2.0 ** -19
        off = np.abs(got[h] - want)
        tolerance = bound + np.abs(want) * R.HALF_STEP[dtype] * 1.001 + 2.0 ** -25 * (dtype == torch.float16)
        assert (off <= tolerance).all(), (off / tolerance).max()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("tokens, share, dim, group", [(1, 8, 64, 64), (1, 4, 128, 128), (2, 7, 128, 32), (5, 5, 128, 64), (1, 2, 256, 32)])
def test_scales_that_do_not_count_take_no_bits(dtype, tokens, share, dim, group):
    """Values whose scales differ by up to 2^36, from position to position and from group to group.  Even heads of queries see the large
    ones with weights of 2^-100 and less, odd ones are all theirs.  Errors as for any other values, next to what the column itself sums."""
    s = Sequences([90, 33, 300], 2, dim, group, 16, seed=dim)
    c = s.cache
    size = 2.0 ** torch.randint(-24, 13, c.v_scales.shape[:-1], generator=rng(1)).float()
    loud = torch.rand(c.v_scales.shape[:3], generator=rng(2)) < 0.3
    size = torch.where(loud[..., None], size, size.clamp(max=2.0 ** -12))
    c.v_scales[..., 0] = (size * (1 + torch.rand(size.shape, generator=rng(3)))).half().cuda()
    c.v_scales[..., 1] = -7 * c.v_scales[..., 0]
    c.k_scales[..., 0] *= 0.01
    c.k_scales[..., 1] = torch.where(loud[..., None], 1.0, 0.0).half().cuda()
    q = torch.randn(3, tokens, 2 * share, dim, generator=rng(4))
    q[:, :, 0::2] = -q[:, :, 0::2].abs() * 2000 / dim
    q[:, :, 1::2] = q[:, :, 1::2].abs() * 2000 / dim
    q = q.to(dtype).cuda()
    table, lengths = s.device()
    got = double(F.attend4(c, q, table, lengths, scale=0.1))
    want, _, bound, score = R.attend(double(q), *s.buffers(), s.table, s.lengths, None, group, 0.1, 0, 8 if dtype == torch.float32 else 0)
    assert score.max() < 600
    # as check_attend has it: scores, weights (two parts: 2^-22), sums of at most 300 / 16 + 64 links, one rounding
    weight = 2 * score * (2.0 ** -22 + 24 * 2.0 ** -23) + 2 * 2.0 ** -22 + 2.0 ** -20 + 83 * 2.0 ** -23
    tolerance = bound * weight[..., None] * 1.01 + np.abs(want) * R.HALF_STEP[dtype] * 1.001 + 2.0 ** -25 * (dtype == torch.float16)
    assert (np.abs(got - want) <= tolerance).all(), (np.abs(got - want) / tolerance).max()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("dim, group, share", [(32, 32, 3), (128, 64, 4), (256, 128, 1)])
@pytest.mark.parametrize("far", [-3e4, 3e4, -1e30, 1e30])
def test_scores_far_from_zero(dtype, dim, group, share, far):
    """Scores that are all the same, far below zero or above: every position counts alike.  Errors: 200 weights of 1, fp32 sums of at most 64
    links, one rounding."""
    if dtype == torch.float16 and abs(far) > 1e9:
        pytest.skip("beyond what fp16 queries reach")
    s = Sequences([200, 50], 1, dim, group, 16, seed=3)
    c = s.cache
    c.k_codes.zero_()
    c.k_scales[..., 0] = 0
    c.k_scales[..., 1] = 1.0
    q = torch.full((2, 1, share, dim), far / 64 / dim, dtype=dtype, device="cuda")
    table, lengths = s.device()
    got = double(F.attend4(c, q, table, lengths, scale=64.0))
    _, _, codes, scales = s.buffers()
    for b in range(2):
        at = [(s.table[b][i // 16], i % 16) for i in range(s.lengths[b])]
        v, size = (np.stack(x) for x in zip(*(R.values(codes[p, 0, i], scales[p, 0, i], group, dim, 8) for p, i in at)))
        want, bound = v.mean(0), size.mean(0) * (2.0 ** -22 + 64 * 2.0 ** -23)
        assert (np.abs(got[b, 0] - want) <= bound + np.abs(want) * R.HALF_STEP[dtype] * 1.001 + 2.0 ** -25 * (dtype == torch.float16)).all()


def test_outputs_that_share_memory():
    m = matrix(64, 64, 32, 1)
    whole = torch.randn(6, 160, generator=rng(1)).cuda()
    x = whole[:, :64]
    want = F.forward_connected4(m, x)
    assert torch.equal(F.forward_connected4(m, x, out=whole[:, 64:128]), want)               # side by side
    for out in (x, whole[:, 32:96], whole.view(-1)[100:484].view(6, 64), whole.as_strided((6, 64), (64, 1), 0)):
        with pytest.raises(ValueError, match="memory"):
            F.forward_connected4(m, x, out=out)
    bias = torch.zeros(640, device="cuda")
    with pytest.raises(ValueError, match="memory"):
        F.forward_connected4(m, x, bias[100:164], out=bias[:384].view(6, 64))
    with pytest.raises(ValueError, match="memory"):
        F.forward_connected4(m, x, out=bias.as_strided((6, 64), (63, 1), 0))

    for lengths in ([40, 7], [900, 30]):                     # one CTA, and a cluster of them, a sequence
        s = Sequences(lengths, 2, 64, 32, room=30)
        table, n = s.device()
        qs = torch.randn(2, 3, 12, 64, generator=rng(2)).half().cuda()
        q = qs[:, :, :4]
        want = F.attend4(s.cache, q, table, n)
        assert torch.equal(F.attend4(s.cache, q, table, n, out=qs[:, :, 4:8]), want)
        for out in (qs[:, :, 1:5], qs.as_strided(q.shape, (0, 768, 64, 1), 2000), qs.as_strided(q.shape, q.stride(), 32)):
            with pytest.raises(ValueError, match="memory"):
                F.attend4(s.cache, q, table, n, out=out)
        copy = q.clone()
        assert torch.equal(F.attend4(s.cache, copy, table, n, out=copy), want)               # in the place of the queries
        room = torch.zeros(4096, device="cuda")
        qf = room[:1536].view(2, 3, 4, 64)
        with pytest.raises(ValueError, match="memory"):
            F.attend4(s.cache, qf, table, n, lse=room[1500:1524].view(2, 3, 4))
        with pytest.raises(ValueError, match="memory"):
            F.attend4(s.cache, qf, table, n, out=room[2000:3536].view(2, 3, 4, 64), lse=room[3535:3559].view(2, 3, 4))
        F.attend4(s.cache, qf, table, n, out=room[2000:3536].view(2, 3, 4, 64), lse=room[3536:3560].view(2, 3, 4))
    s = Sequences([6000], 1, 64, 32, 64)                     # more splits than a cluster has
    table, n = s.device()
    q = torch.randn(1, 5, 8, 64, generator=rng(3)).half().cuda()
    want = F.attend4(s.cache, q, table, n)
    assert torch.equal(F.attend4(s.cache, q, table, n, out=q), want)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("lengths, kv_heads, tokens, page", [([90, 50, 70, 33], 16, 1, 16), ([900, 700, 40, 600], 2, 3, 16), ([5000, 3000, 4100, 10], 1, 1, 64)])
def test_a_sequences_results_do_not_depend_on_the_others(dtype, lengths, kv_heads, tokens, page):
    """The first sequence among others of other lengths, pages, queries and counts, of scales that are not finite, and in another place of the
    batch: one CTA a sequence, clusters, and splits that meet in scratch memory."""
    s = Sequences(lengths, kv_heads, 64, 32, page, seed=4, spare=40)
    c = s.cache
    q = torch.randn(4, tokens, 6 * kv_heads, 64, generator=rng(1)).to(dtype).cuda()
    table, n = s.device()
    counts = torch.full((4,), tokens, dtype=torch.int32, device="cuda")
    want = F.attend4(c, q, table, n, counts)[0].clone()
    other = torch.randn(4, tokens, 6 * kv_heads, 64, generator=rng(2)).to(dtype).cuda()
    other[0] = q[0]
    n2, counts2, table2 = n.clone(), counts.clone(), table.clone()
    n2[1:] = torch.tensor([1, 700 % lengths[2], 0], dtype=torch.int32)
    counts2[2] = 0
    table2[3] = -1
    other[1] = math.nan
    for scales in (c.k_scales, c.v_scales):
        scales[table[2][table[2] >= 0].long()] = math.inf
    got = F.attend4(c, other, table2, n2, counts2)
    assert torch.equal(got[0], want) and not got[3].any()
    order = torch.tensor([2, 3, 0, 1]).cuda()
    got = F.attend4(c, other[order], table2[order], n2[order], counts2[order])
    assert torch.equal(got[2], want)


def test_rows_inside_a_table_that_is_too_short_are_read_back():
    s = Sequences([64, 40], 2, 64, 32, 16, seed=5)
    s.lengths = [70, 66]                                     # (of 64 and 48 places: rows 0 and 1 of the first have one)
    table, lengths = s.device()
    k, v = (torch.randn(2, 8, 2, 64, generator=rng(i)).cuda() for i in (3, 4))
    F.append4(s.cache, k, v, table, lengths)
    for given, got in zip((k, v), F.read4(s.cache, table, lengths, 8)):
        codes, scales = R.quantize(double(given[0, :2]), 32)
        want = R.values(R.pack(codes), scales, 32, 64)[0]
        # one fma, rounded to fp32
        assert (np.abs(double(got[0, :2]) - want) <= np.abs(want) * 2.0 ** -23).all()
        assert not got[0, 2:].any() and not got[1].any()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("dim, group, share", [(64, 32, 4), (128, 128, 1), (96, 32, 9), (256, 64, 2)])
def test_a_token_that_sees_one_position_gets_its_values(dtype, dim, group, share):
    """The first token of a sequence, and any behind a window of one: the values as they are, rounded once.  (Scales and lows of few bits, so
    that every step of the sums is exact in fp32; a last bit off would send values half way between two of a type's the wrong way.)"""
    s = Sequences([1, 40, 17, 300], 2, dim, group, 16, seed=7)
    c = s.cache
    c.v_scales[..., 0] = torch.randint(1, 2000, c.v_scales.shape[:-1], generator=rng(1)).mul(2.0 ** -13).half().cuda()
    c.v_scales[..., 1] = torch.randint(-2000, 2000, c.v_scales.shape[:-1], generator=rng(2)).mul(2.0 ** -9).half().cuda()
    q = torch.randn(4, 1, 2 * share, dim, generator=rng(3)).to(dtype).cuda()
    table, lengths = s.device()
    got = F.attend4(c, q, table, lengths, window=1).cpu()
    _, _, codes, scales = s.buffers()
    for b, n in enumerate(s.lengths):
        page, place = s.table[b][(n - 1) // 16], (n - 1) % 16
        v = torch.from_numpy(R.values(codes[page, :, place], scales[page, :, place], group, dim)[0])
        assert torch.equal(got[b, 0], v.to(dtype).repeat_interleave(share, 0))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=ids)
def test_large_products_in_graphs_and_on_two_streams(dtype):
    """Those whose rows are converted by a kernel in front: captured, behind a kernel that writes the rows and one that writes the scales,
    replayed on two streams at a time."""
    n, k, rows = 16384, 8192, 9
    m = [matrix(n, k, 64, i) for i in range(2)]
    base = [x.scales.clone() for x in m]
    xs = [torch.zeros(rows, k, dtype=dtype, device="cuda") for _ in m]
    halves = [torch.zeros(1, dtype=torch.float16, device="cuda") for _ in m]

    def work(i):
        m[i].scales.copy_(base[i] * halves[i])
        return F.forward_connected4(m[i], xs[i] * 2)

    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in m]
    for i in range(2):
        work(i)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(work(i))
    for turn in range(6):
        for i in range(2):
            xs[i].copy_(torch.randn(rows, k, generator=rng(10 * turn + i)))
            halves[i].fill_(0.5 if turn % 2 else 1.0)
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        got = [y.clone() for y in outs]
        for i in range(2):
            assert torch.equal(got[i], work(i))
    picked = torch.arange(0, n, 411).cuda()
    part = F.Matrix4(m[0].codes[picked].contiguous(), m[0].scales[picked].contiguous(), k, 64)
    check_product(part, xs[0] * 2, work(0)[:, picked])
