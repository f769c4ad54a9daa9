"""Four-bit matrices and token caches on the GPU against 64 bits."""
import math

import numpy as np
import pytest

import four_reference as R

torch = pytest.importorskip("torch")

from darknet_b200 import capi, fourbit as F  # noqa: E402

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
ids = {torch.float32: "fp32", torch.float16: "fp16", torch.bfloat16: "bf16"}.get


def double(t):
    return t.detach().cpu().double().numpy()


def rng(seed):
    return torch.Generator().manual_seed(seed)


# ---- packing ------------------------------------------------------------------------------------------------------------------


def check_packed(got_codes, got_scales, rows, group):
    """Scales are the definition's, codes its nearest ones: where a value lies half way between two, to within fp32's rounding of the
    quotient (values up to 15, so 16 * 2^-24), either will do."""
    codes, scales = R.quantize(rows, group)
    np.testing.assert_array_equal(got_scales.view(np.uint16) & 0x7fff, scales.view(np.uint16) & 0x7fff)
    np.testing.assert_array_equal(got_scales.astype(np.float64), scales.astype(np.float64))
    off = got_codes != codes
    if off.any():
        k = rows.shape[-1]
        s, low = (np.repeat(scales[..., i].astype(np.float64), group, -1)[..., :k][off] for i in (0, 1))
        q = (np.clip(rows[off], -65504, 65504) - low) / s
        assert np.abs(np.abs(q - got_codes[off]) - 0.5).max() <= 2.0 ** -19


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("n, k, group", [(1, 1, 32), (3, 31, 32), (5, 32, 128), (7, 33, 64), (2, 129, 128), (33, 1000, 64), (4, 2305, 32), (130, 4608, 128)])
def test_weights_are_packed_as_defined(dtype, n, k, group):
    w = (torch.randn(n, k, generator=rng(n + k)) * torch.logspace(-6, 3, n)[:, None]).to(dtype)
    m = F.quantize_weights4(w.cuda(), group)
    packed = m.codes.cpu().numpy()
    check_packed(R.unpack(packed, k), m.scales.cpu().numpy(), double(w), group)
    np.testing.assert_array_equal(packed, R.pack(R.unpack(packed, k)))                 # bits behind k are 0
    back, _ = R.values(packed, m.scales.cpu().numpy(), group, k)
    step = np.repeat(m.scales.cpu().numpy()[..., 0].astype(np.float64), group, -1)[:, :k]
    assert (np.abs(back - double(w)) <= step * (0.5 + 2.0 ** -19)).all()


def test_weights_of_extreme_values():
    rows = torch.zeros(9, 64)
    rows[1] = 3.25                                          # one value: scale 0
    rows[2] = torch.linspace(-1e6, 1e6, 64)                 # beyond fp16
    rows[3, 5], rows[3, 9] = math.nan, 2.0
    rows[4, 0], rows[4, 1] = math.inf, -math.inf
    rows[5] = torch.linspace(0, 1e-9, 64)                   # below fp16's smallest
    rows[6] = -1e-9
    rows[7] = 1000 + torch.linspace(0, 0.3, 64)             # a range below the step of low
    rows[8] = math.nan
    m = F.quantize_weights4(rows.cuda(), 64)
    check_packed(R.unpack(m.codes.cpu().numpy(), 64), m.scales.cpu().numpy(), double(rows), 64)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_values_next_to_a_half_take_the_nearest_code(group):
    """fp32 values a last bit beside the middle of two codes, whose difference from low has no room for that bit; and the middle itself, which
    takes the even code.  low -1, scale 1/8."""
    rows = torch.full((8, group), -1.0)
    rows[:, 1] = 0.875
    for i, half in enumerate((7.5, 8.5)):
        middle = torch.tensor(-1.0 + half / 8)
        for j, v in enumerate((middle, torch.nextafter(middle, torch.tensor(9.0)), torch.nextafter(middle, torch.tensor(-9.0)))):
            rows[3 * i + j, 2:] = v
    rows[6, 2:] = -1.0 + 0.5 / 8                             # (0: even)
    rows[7, 2:] = torch.nextafter(torch.tensor(-1.0 + 14.5 / 8), torch.tensor(9.0))
    m = F.quantize_weights4(rows.cuda(), group)
    codes, scales = R.quantize(double(rows), group)
    assert codes[:, 2].tolist() == [8, 8, 7, 8, 9, 8, 0, 15]
    np.testing.assert_array_equal(R.unpack(m.codes.cpu().numpy(), group), codes)
    np.testing.assert_array_equal(m.scales.cpu().numpy(), scales)
    s = Sequences([8], 1, 128, group, 16)
    table, lengths = s.device()
    k = rows.repeat(1, 128 // group).view(1, 8, 1, 128).cuda()
    F.append4(s.cache, k, -k, table, lengths)
    got, _ = F.read4(s.cache, table, lengths, 8)
    assert torch.equal(got.view(8, 128)[:, :group].cpu(), torch.from_numpy(-1.0 + codes / 8).float())


def test_random_codes_are_the_definitions_all_of_them():
    """Two million values: some of any such number lie next to a half."""
    rows = torch.randn(4096, 512, generator=rng(12))
    m = F.quantize_weights4(rows.cuda(), 64)
    codes, scales = R.quantize(double(rows), 64)
    np.testing.assert_array_equal(m.scales.cpu().numpy(), scales)
    np.testing.assert_array_equal(R.unpack(m.codes.cpu().numpy(), 512), codes)


@pytest.mark.parametrize("offset, pad", [(0, 0), (1, 3), (3, 8)])
def test_weights_with_strides(offset, pad):
    whole = torch.randn(6, 77 + pad + offset, generator=rng(4), dtype=torch.float32).half().cuda()
    part = whole[:, offset:offset + 77]
    a, b = F.quantize_weights4(part, 32), F.quantize_weights4(part.contiguous(), 32)
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)


# ---- products -----------------------------------------------------------------------------------------------------------------


def matrix(n, k, group, seed, device="cuda"):
    g = rng(seed)
    codes = torch.randint(0, 256, (n, (k + 31) // 32 * 16), generator=g, dtype=torch.uint8)         # bits behind k: anything
    groups = (k + group - 1) // group
    scales = torch.stack((torch.rand(n, groups, generator=g) * 0.1, torch.randn(n, groups, generator=g) * 0.5), -1).half()
    return F.Matrix4(codes.to(device), scales.to(device), k, group)


def centre(dtype):
    return 8 if dtype == torch.float32 else 0


def check_product(m, x, y, biases=None, leaky=False):
    """Errors: x as fp16 parts (2^-22 of it), fp32 sums (each of a chain of additions rounds, or cuts off, by at most 2^-23 of a sum that
    is at most sum |x| (|low| + scale * code), for fp32 around code 8; a chain has 2 * 16 products of a group, a group's two terms, the blocks and the slices),
    one rounding of the result."""
    v, size = R.values(m.codes.cpu().numpy(), m.scales.cpu().numpy(), m.group, m.k, centre(x.dtype))
    xd = double(x)
    want, bound = xd @ v.T, np.abs(xd) @ size.T
    if biases is not None:
        want, bound = want + double(biases), bound + np.abs(double(biases))
    if leaky:
        want = np.where(want > 0, want, 0.1 * want)
    links = 32 + 2 * (m.k // m.group + 1) + 2 * (m.k // 256 + 1) + 16
    tolerance = bound * (2.0 ** -22 + links * 2.0 ** -23) + np.abs(want) * R.HALF_STEP[x.dtype] * 1.001 + 2.0 ** -25 * (x.dtype == torch.float16)
    off = np.abs(double(y) - want)
    assert (off <= tolerance).all(), (off - tolerance).max()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n, k, rows", [(1, 1, 1), (15, 31, 2), (64, 256, 1), (65, 257, 3), (200, 1000, 8), (130, 2305, 9), (70, 4608, 16), (33, 700, 17), (40, 513, 40)])
def test_products(dtype, group, n, k, rows):
    m = matrix(n, k, group, n + k)
    x = torch.randn(rows, k, generator=rng(k)).to(dtype).cuda()
    check_product(m, x, F.forward_connected4(m, x))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_product_of_a_long_row(dtype):
    m = matrix(20, 70001, 128, 6)
    x = torch.randn(2, 70001, generator=rng(1)).to(dtype).cuda()
    check_product(m, x, F.forward_connected4(m, x))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("n, k, group, rows", [(16500, 8200, 64, 9), (8300, 16200, 128, 16), (16384, 8192, 32, 35)])
def test_large_products_of_many_rows(dtype, n, k, group, rows):
    """Those convert x beforehand.  What they give is compared with calls of eight rows, which do not, filter by filter: both are within
    check_product's bound of the same value; the bound itself is looked at for some filters."""
    m = matrix(n, k, group, rows)
    whole = torch.randn(rows, k + 8, generator=rng(k)).to(dtype).cuda()
    for x in (whole[:, :k], whole[:, 3:k + 3]):
        y = F.forward_connected4(m, x)
        assert capi.lib().xnor_b200_w4_scratch_bytes(capi.W4Desc(n, k, group, 0), 1, rows) > 0
        picked = torch.arange(0, n, 211)
        part = F.Matrix4(m.codes[picked.cuda()].contiguous(), m.scales[picked.cuda()].contiguous(), k, group)
        check_product(part, x, y[:, picked.cuda()])
        few = torch.cat([F.forward_connected4(m, x[i:i + 8]) for i in range(0, rows, 8)])
        assert ((y.float() - few.float()).abs() <= few.float().abs() * 2 * R.HALF_STEP[dtype] + 2e-3).all()
        for _ in range(2):
            assert torch.equal(F.forward_connected4(m, x), y)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_product_with_bias_and_leaky(dtype):
    m = matrix(100, 300, 32, 1)
    x, b = torch.randn(3, 300, generator=rng(2)).to(dtype).cuda(), torch.randn(100, generator=rng(3)).cuda()
    check_product(m, x, F.forward_connected4(m, x, b), b)
    check_product(m, x, F.forward_connected4(m, x, b, capi.LEAKY), b, True)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_product_of_values_of_any_size(dtype):
    """Rows, and stretches of a row, of very different magnitudes: each block of 256 has a power of two of its own."""
    m = matrix(50, 1024, 64, 5)
    x = torch.randn(4, 1024, generator=rng(8))
    high, small = (4.0, 1e-4) if dtype == torch.float16 else (30.0, 1e-25)
    x[0] *= 10 ** high
    x[1] *= small
    x[2, ::3] *= small
    x[3, 256:512] = 0
    x = x.to(dtype).cuda()
    v, size = R.values(m.codes.cpu().numpy(), m.scales.cpu().numpy(), m.group, m.k)
    xd = double(x)
    y = F.forward_connected4(m, x)
    fits = np.isfinite(double(y))
    want, bound = xd @ v.T, np.abs(xd) @ size.T
    assert (fits | (np.abs(want) > torch.finfo(dtype).max * 0.99)).all()
    tolerance = bound * 120 * 2.0 ** -23 + np.abs(want) * R.HALF_STEP[dtype] * 1.001 + float(torch.finfo(dtype).smallest_normal)
    assert (np.abs(double(y) - want)[fits] <= tolerance[fits]).all()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows", [5, 13])
def test_a_row_that_is_not_finite_gives_nan_and_no_other_does(dtype, rows):
    m = matrix(70, 600, 64, 2)
    for bad in (math.inf, -math.inf, math.nan):
        x = torch.randn(rows, 600, generator=rng(1)).to(dtype).cuda()
        x[1, 300] = bad
        y = F.forward_connected4(m, x)
        assert torch.isnan(y[1]).all()
        rest = [i for i in range(rows) if i != 1]
        check_product(m, x[rest], y[rest])


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("offset", [0, 1, 8])
def test_product_with_strides_writes_its_rows_only(dtype, offset):
    m = matrix(77, 200, 32, 3)
    whole = torch.randn(4, 240, generator=rng(4)).to(dtype).cuda()
    x = whole[:, offset:offset + 200]
    room = torch.full((4, 100), 7.0, dtype=dtype, device="cuda")
    y = F.forward_connected4(m, x, out=room[:, 5:82])
    assert y.data_ptr() == room[:, 5:82].data_ptr()
    check_product(m, x, y)
    assert (room[:, :5] == 7).all() and (room[:, 82:] == 7).all()
    one = x[:1].expand(3, -1)                                # the same row three times
    y = F.forward_connected4(m, one)
    assert torch.equal(y[0], y[1]) and torch.equal(y[0], y[2])


def test_products_repeat_bit_for_bit_and_do_not_depend_on_other_rows():
    m = matrix(300, 4096, 128, 9)
    x = torch.randn(16, 4096, generator=rng(5)).cuda()
    y = F.forward_connected4(m, x)
    for _ in range(3):
        assert torch.equal(F.forward_connected4(m, x), y)
    order = torch.randperm(16, generator=rng(6)).cuda()
    assert torch.equal(F.forward_connected4(m, x[order]), y[order])


# ---- the cache ------------------------------------------------------------------------------------------------------------------


class Sequences:
    """A cache of random rows, with sequences in it."""

    def __init__(self, lengths, kv_heads, dim, group, page=16, seed=0, room=0, spare=2):
        g = rng(seed)
        per = [-(-n // page) for n in lengths]
        self.pages, self.group, self.dim, self.kv_heads, self.page = sum(per) + spare, group, dim, kv_heads, page
        order = torch.randperm(self.pages, generator=g).tolist()
        width = max(max(per), 1) + room
        self.table = [[order.pop() for _ in range(n)] + [-1] * (width - n) for n in per]
        self.lengths = list(lengths)
        codes = [torch.randint(0, 256, (self.pages, kv_heads, page, dim // 2), generator=g, dtype=torch.uint8) for _ in "kv"]
        shape = (self.pages, kv_heads, page, dim // group)
        scales = [torch.stack((torch.rand(*shape, generator=g) * 0.2, torch.randn(*shape, generator=g)), -1).half() for _ in "kv"]
        self.cache = F.Cache4(codes[0].cuda(), scales[0].cuda(), codes[1].cuda(), scales[1].cuda(), group)

    def device(self):
        return torch.tensor(self.table, dtype=torch.int32, device="cuda"), torch.tensor(self.lengths, dtype=torch.int32, device="cuda")

    def buffers(self):
        c = self.cache
        return [t.cpu().numpy() for t in (c.k_codes, c.k_scales, c.v_codes, c.v_scales)]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("dim, group, kv_heads, page", [(32, 32, 1, 16), (64, 64, 3, 32), (96, 32, 5, 48), (128, 128, 8, 64), (192, 64, 2, 16), (256, 32, 9, 16), (256, 128, 1, 256)])
def test_append_and_read(dtype, dim, group, kv_heads, page):
    s = Sequences([0, 1, 17, 40, 70, 33], kv_heads, dim, group, page, seed=dim)
    s.table[3][0] = -1                                       # a page that the cache does not have
    s.table[5][-1] = s.pages
    counts = [0, 1, 5, 40, 3, 50]                            # the last sequence holds 33: 17 of its rows come before its start
    tokens = 45
    before = s.buffers()
    k, v = (torch.randn(6, tokens, kv_heads, dim, generator=rng(i)).to(dtype).cuda() for i in (1, 2))
    table, lengths = s.device()
    n = torch.tensor(counts, dtype=torch.int32, device="cuda")
    F.append4(s.cache, k, v, table, lengths, n)
    after = s.buffers()
    rows = R.find(s.table, s.lengths, counts, tokens, page, s.pages)
    assert len(rows) > 5
    got = F.read4(s.cache, table, lengths, tokens, n, dtype)
    touched = np.zeros((s.pages, page), bool)
    for i, x in enumerate((k, v)):
        back = double(got[i])
        for (b, r), (p, place) in rows.items():
            check_packed(R.unpack(after[2 * i][p, :, place], dim), after[2 * i + 1][p, :, place], double(x[b, r]), group)
            want, size = R.values(after[2 * i][p, :, place], after[2 * i + 1][p, :, place], group, dim)
            # one rounding to fp32, one to the type
            assert (np.abs(back[b, r] - want) <= np.abs(want) * (R.HALF_STEP[dtype] + 2.0 ** -23) + 2.0 ** -25 * (dtype == torch.float16)).all()
            touched[p, place] = True
        for b in range(6):
            for r in range(tokens):
                assert (b, r) in rows or not back[b, r].any()
    for x, y in zip(before, after):                          # all other places are as they were
        np.testing.assert_array_equal(x.transpose(0, 2, 1, 3, *range(4, x.ndim))[~touched], y.transpose(0, 2, 1, 3, *range(4, x.ndim))[~touched])


def test_append_takes_strides():
    s = Sequences([20, 9], 4, 64, 32)
    table, lengths = s.device()
    qkv = torch.randn(2, 3, 13, 64, generator=rng(1)).half().cuda()          # heads of queries, keys and values side by side
    odd = torch.randn(2, 3, 4, 67, generator=rng(2)).half().cuda()[..., 3:]  # rows that start on no 16 bytes
    for k, v in ((qkv[:, :, 5:9], qkv[:, :, 9:13]), (odd, odd.transpose(0, 1).contiguous().transpose(0, 1))):
        F.append4(s.cache, k, v, table, lengths)
        a = s.buffers()
        F.append4(s.cache, k.contiguous(), v.contiguous(), table, lengths)
        for x, y in zip(a, s.buffers()):
            np.testing.assert_array_equal(x, y)


# ---- attention ------------------------------------------------------------------------------------------------------------------


def check_attend(s, q, counts=None, scale=None, window=0, out=None, with_lse=True):
    """Errors.  A score: q as fp16 parts (2^-22), 24 fp32 operations on sums of at most scale * sum |q| (|low| + s * code): by delta =
    (2^-22 + 24 * 2^-23) * score in all, and its weight by twice that (the maximum's too).  A weight: 2^-22 of the exponential, for bf16
    2^-11 of rounding it with the value's scale to fp16 (2^-21 in two parts), at most 2^-30 of the largest where fp16 runs out of bits.
    Sums: a step a link, three where parts meet.  One rounding of the result."""
    table, lengths = s.device()
    scale = 1 / math.sqrt(s.dim) if scale is None else scale
    n = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    lse = torch.full(q.shape[:3], 5.0, device="cuda") if with_lse else None
    got = F.attend4(s.cache, q, table, lengths, n, scale=scale, window=window, out=out, lse=lse)
    want, want_lse, size, score = R.attend(double(q), *s.buffers(), s.table, s.lengths, counts, s.group, scale, window, centre(q.dtype))
    delta = score * (2.0 ** -22 + 24 * 2.0 ** -23)
    links = max(s.lengths) / 16 + 64
    weight = 2 * delta + 2.0 ** -22 + (2.0 ** -11 if q.dtype == torch.bfloat16 else 2.0 ** -21) + 2.0 ** -20 + links * 2.0 ** -23
    tolerance = size * weight[..., None] * 1.01 + np.abs(want) * R.HALF_STEP[q.dtype] * 1.001 + 2.0 ** -25 * (q.dtype == torch.float16)
    off = np.abs(double(got) - want)
    assert (off <= tolerance).all(), (off - tolerance).max()
    if with_lse:
        seen = np.isfinite(want_lse)
        assert (np.isneginf(double(lse)) == ~seen).all()
        assert (np.abs(double(lse)[seen] - want_lse[seen]) <= (weight[seen] + np.abs(want_lse[seen]) * 2.0 ** -22 + 2.0 ** -20)).all()
        assert not double(got)[~seen].any()
    return got


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("dim, group", [(32, 32), (64, 32), (64, 64), (96, 32), (128, 32), (128, 64), (128, 128), (160, 32), (192, 64), (224, 32), (256, 32), (256, 64), (256, 128)])
@pytest.mark.parametrize("share", [1, 3, 8, 11])
def test_attention_of_one_token(dtype, dim, group, share):
    s = Sequences([0, 1, 2, 15, 16, 17, 31, 63, 64, 65, 200], 2, dim, group, 16, seed=dim + share)
    q = torch.randn(len(s.lengths), 1, 2 * share, dim, generator=rng(share)).to(dtype).cuda()
    check_attend(s, q)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("tokens, share, window", [(2, 1, 0), (3, 4, 0), (5, 7, 5), (4, 8, 1), (9, 2, 33), (33, 1, 16), (40, 3, 0)])
def test_attention_of_several_tokens(dtype, tokens, share, window):
    s = Sequences([0, 1, tokens - 1, tokens, 50, 130], 3, 128, 64, 32, seed=tokens)
    q = torch.randn(6, tokens, 3 * share, 128, generator=rng(tokens)).to(dtype).cuda()
    check_attend(s, q, window=window)
    check_attend(s, q, counts=[0, 1, tokens, 1, max(1, tokens // 2), tokens], window=window)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("dim, group", [(32, 32), (64, 32), (64, 64), (96, 32), (128, 32), (128, 128), (192, 32), (256, 128)])
@pytest.mark.parametrize("tokens, share", [(2, 6), (4, 6), (5, 5)])
def test_columns_of_every_width(dtype, dim, group, tokens, share):
    """12, 24 and 25 columns of a head of keys: two and three tiles of eight, and one more than fits."""
    s = Sequences([150, 3, 64, 0], 2, dim, group, 16, seed=dim + tokens)
    q = torch.randn(4, tokens, 2 * share, dim, generator=rng(tokens)).to(dtype).cuda()
    check_attend(s, q, counts=[tokens, 2, 1, 1], window=90)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_scales_below_zero(dtype):
    s = Sequences([200, 33], 2, 64, 32, 16, seed=6)
    for scales in (s.cache.k_scales, s.cache.v_scales):
        scales[..., 0] *= torch.where(torch.rand(scales.shape[:-1], generator=rng(1)) < 0.5, -1.0, 1.0).half().cuda()
    check_attend(s, torch.randn(2, 1, 6, 64, generator=rng(2)).to(dtype).cuda())
    m = matrix(90, 500, 32, 2)
    m.scales[..., 0] *= -1
    x = torch.randn(4, 500, generator=rng(3)).to(dtype).cuda()
    check_product(m, x, F.forward_connected4(m, x))


def test_lengths_beyond_the_table():
    """A sequence that is longer than its table has pages for: the positions behind them are nowhere."""
    s = Sequences([64, 40], 2, 64, 32, 16, seed=5)
    s.lengths = [70, 2 ** 31 - 1]
    check_attend(s, torch.randn(2, 3, 4, 64, generator=rng(2)).cuda())
    s.lengths = [70, 66]
    table, lengths = s.device()
    before = s.buffers()
    k = torch.randn(2, 8, 2, 64, generator=rng(3)).cuda()
    F.append4(s.cache, k, k, table, lengths)
    rows = R.find(s.table, s.lengths, None, 8, 16, s.pages)
    assert sorted(rows) == [(0, 0), (0, 1)]
    got, _ = F.read4(s.cache, table, lengths, 8)
    assert got[0, :2].abs().min() >= 0 and not got[0, 2:].any() and not got[1].any()
    changed = (before[0] != s.buffers()[0]).any((1, 3))
    assert {(p, i) for p, i in zip(*np.nonzero(changed))} <= set(rows.values())
    s.lengths = [-3, 0]
    out = F.attend4(s.cache, torch.randn(2, 3, 4, 64).cuda(), *s.device())
    assert not out.any()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("length, batch, kv_heads, page, room", [(513, 1, 8, 64, 0), (2000, 3, 2, 16, 0), (5000, 1, 1, 128, 0), (3001, 2, 1, 48, 400)])
def test_attention_over_long_sequences(dtype, length, batch, kv_heads, page, room):
    """Few sequences, split over clusters and over scratch memory; tables with room for much more than there is."""
    s = Sequences([length - 700 * i for i in range(batch)], kv_heads, 64, 32, page, seed=length, room=room)
    q = torch.randn(batch, 1, 4 * kv_heads, 64, generator=rng(1)).to(dtype).cuda()
    check_attend(s, q)
    check_attend(s, q, window=300)
    q = torch.randn(batch, 3, 4 * kv_heads, 64, generator=rng(1)).to(dtype).cuda()
    check_attend(s, q, counts=[3, 2, 1][:batch])


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_long_sums_lose_nothing(dtype):
    """Equal weights over 20000 positions by one CTA: sums whose result is a hundredth of what goes into them.  Sequences enough that
    none is split, all of them one and the same."""
    batch, kv_heads = 60, 16
    s = Sequences([20000], kv_heads, 32, 32, 256, seed=1)
    s.cache.v_scales[..., 1] = -7.5 * s.cache.v_scales[..., 0]
    q = 0.01 * torch.randn(1, 1, kv_heads, 32, generator=rng(1)).to(dtype).cuda()
    want, _, size, score = R.attend(double(q), *s.buffers(), s.table, s.lengths, None, 32, 0.1, 0, centre(dtype))
    table, lengths = s.device()
    got = double(F.attend4(s.cache, q.expand(batch, -1, -1, -1), table.expand(batch, -1).contiguous(), lengths.expand(batch).contiguous(), scale=0.1))
    assert (got == got[:1]).all()
    # as check_attend has it, but for the sums: a link of a sum adds a rounding of what the sum has come to, which stays within a few times
    # the square root of the links' own sizes
    links = 20000 / 16 / 4
    weight = 2 * score * (2.0 ** -22 + 24 * 2.0 ** -23) + 2.0 ** -22 + (2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -21)
    tolerance = size * (weight[..., None] / 8 + 4 * links ** 0.5 * 2.0 ** -23) + np.abs(want) * R.HALF_STEP[dtype] * 1.001 + 2.0 ** -25 * (dtype == torch.float16)
    assert (np.abs(got - want) <= tolerance).all(), (np.abs(got - want) / tolerance).max()


@pytest.mark.parametrize("dim, group", [(64, 64), (128, 128), (256, 64)])
def test_pages_that_are_not_there_are_not_seen(dim, group):
    s = Sequences([100, 64, 40], 2, dim, group, 16, seed=3)
    s.table[0][2] = -1
    s.table[0][4] = s.pages
    s.table[1] = [-1] * len(s.table[1])                      # nothing left of the second
    s.table[2][0] = -2 ** 31
    check_attend(s, torch.randn(3, 2, 4, dim, generator=rng(1)).cuda())


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_what_is_not_seen_never_counts_whatever_it_is(dtype):
    """NaN and infinities behind a sequence's end, in front of its window, and in places that later tokens of the call see."""
    s = Sequences([37, 100], 2, 64, 32, 32, seed=8)
    c = s.cache
    q = torch.randn(2, 1, 6, 64, generator=rng(2)).to(dtype).cuda()
    clean = check_attend(s, q, window=20).clone()
    for scales in (c.k_scales, c.v_scales):
        for b, (first, behind) in enumerate(((0, 17), (37, 64)), 0):
            for at in list(range(0, s.lengths[b] - 20)) + list(range(s.lengths[b], len(s.table[b]) * 32)):
                if at // 32 < len(s.table[b]) and s.table[b][at // 32] >= 0:
                    scales[s.table[b][at // 32], :, at % 32] = (math.nan, math.inf, -math.inf)[at % 3]
    table, lengths = s.device()
    assert torch.equal(F.attend4(c, q, table, lengths, window=20), clean)
    # two tokens: the newest place holds an infinity, which only the second token sees
    t = Sequences([30], 1, 64, 32, 16, seed=4)
    q = torch.randn(1, 2, 4, 64, generator=rng(3)).to(dtype).cuda()
    table, lengths = t.device()
    want = F.attend4(t.cache, q, table, lengths)
    t.cache.v_scales[t.table[0][1], :, 13] = math.inf
    got = F.attend4(t.cache, q, table, lengths)
    assert torch.equal(got[:, 0], want[:, 0]) and not torch.isfinite(got[:, 1]).any()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("q_size, v_size, scale", [(100.0, 1.0, 1.0), (1e-3, 1e-3, None), (1.0, 60000.0, None), (1.0, 1.0, 0.0), (1.0, 1.0, -0.3), (30.0, 1e-6, 0.5)])
def test_attention_of_values_of_any_size(dtype, q_size, v_size, scale):
    s = Sequences([150, 40], 2, 64, 32, 16, seed=9)
    s.cache.v_scales.mul_(v_size * 5 if v_size > 1 else v_size).nan_to_num_(posinf=65504.0, neginf=-65504.0)
    if v_size > 1:
        s.cache.v_scales.clamp_(-4000, 4000)                 # values of fp16 calls stay in its range
    q = (q_size * torch.randn(2, 1, 4, 64, generator=rng(5))).to(dtype).cuda()
    check_attend(s, q, scale=scale)


def test_scores_that_rise_all_the_way_and_scales_that_grow():
    """The running maximum and the unit of the values' scales move at nearly every step."""
    s = Sequences([400], 1, 32, 32, 16, seed=1)
    c = s.cache
    for at in range(400):
        place = (s.table[0][at // 16], 0, at % 16)
        c.k_codes[place] = 0
        c.k_scales[place] = torch.tensor([[0.0, at * 0.35]], dtype=torch.float16)
        c.v_scales[place][0, 0] = 2.0 ** (at / 25 - 12)
    for dtype in TYPES:
        q = torch.full((1, 1, 2, 32), 0.125, dtype=dtype, device="cuda")
        q[0, 0, 1] = -0.125
        check_attend(s, q, scale=1.0)


def test_a_query_that_is_not_finite_gives_nan_and_no_other_does():
    s = Sequences([70], 1, 64, 64, 16, seed=1)
    table, lengths = s.device()
    for bad in (math.inf, math.nan):
        q = torch.randn(1, 1, 5, 64, generator=rng(1)).cuda()
        want = F.attend4(s.cache, q, table, lengths)
        q[0, 0, 2, 7] = bad
        got = F.attend4(s.cache, q, table, lengths)
        assert torch.isnan(got[0, 0, 2]).all()
        keep = [0, 1, 3, 4]
        assert torch.equal(got[0, 0, keep], want[0, 0, keep])


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_attention_takes_strides(dtype):
    s = Sequences([60, 33, 5], 2, 96, 32, 16, seed=2)
    table, lengths = s.device()
    wide = torch.randn(3, 2, 10, 100, generator=rng(1)).to(dtype).cuda()
    for q in (wide[:, :, 1:7, :96], wide[:, :, ::2, 3:99][:, :, :4], torch.randn(2, 3, 4, 96, generator=rng(2)).to(dtype).cuda().transpose(0, 1)):
        want = F.attend4(s.cache, q.contiguous(), table, lengths)
        assert torch.equal(F.attend4(s.cache, q, table, lengths), want)
        room = torch.full((3, 2, q.shape[2] + 2, 99), 9.0, dtype=dtype, device="cuda")
        F.attend4(s.cache, q, table, lengths, out=room[:, :, 1:-1, 2:98])
        assert torch.equal(room[:, :, 1:-1, 2:98], want)
        assert (room[:, :, 0] == 9).all() and (room[:, :, -1] == 9).all() and (room[..., :2] == 9).all() and (room[..., 98:] == 9).all()


def test_attention_repeats_bit_for_bit_and_does_not_depend_on_other_sequences():
    s = Sequences([3000, 700], 2, 128, 64, 64, seed=2)
    table, lengths = s.device()
    q = torch.randn(2, 1, 8, 128, generator=rng(1)).half().cuda()
    y = F.attend4(s.cache, q, table, lengths)
    for _ in range(3):
        assert torch.equal(F.attend4(s.cache, q, table, lengths), y)


def test_offsets_beyond_32_bits():
    """Pages that lie 4 GB and more behind the start of their buffer."""
    pages, heads, page, dim = 70000, 8, 128, 128
    c = F.Cache4(*(torch.empty(pages, heads, page, *last, dtype=t, device="cuda") for last, t in (((64,), torch.uint8), ((1, 2), torch.float16)) * 2), 128)
    small = F.new_cache4(4, heads, page, dim, 128)
    far = torch.tensor([[pages - 1, 65537, pages - 3]], dtype=torch.int32, device="cuda")
    near = torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([300], dtype=torch.int32, device="cuda")
    k, v = (torch.randn(1, 300, heads, dim, generator=rng(i)).half().cuda() for i in (1, 2))
    q = torch.randn(1, 1, 16, dim, generator=rng(3)).half().cuda()
    for cache, table in ((c, far), (small, near)):
        F.append4(cache, k, v, table, lengths)
    assert torch.equal(F.attend4(c, q, far, lengths), F.attend4(small, q, near, lengths))
    for x, y in zip(F.read4(c, far, lengths, 300), F.read4(small, near, lengths, 300)):
        assert torch.equal(x, y)


# ---- as they are used -------------------------------------------------------------------------------------------------------------


class Block:
    """One attention block of a decoder: three products, the cache, a product."""

    def __init__(self, width, heads, kv_heads, dim, group, batch, longest, dtype, seed=0):
        g = rng(seed)
        self.heads, self.kv_heads, self.dim, self.batch = heads, kv_heads, dim, batch
        self.qkv = F.quantize_weights4((torch.randn((heads + 2 * kv_heads) * dim, width, generator=g) * width ** -0.5).to(dtype).cuda(), group)
        self.back = F.quantize_weights4((torch.randn(width, heads * dim, generator=g) * width ** -0.5).to(dtype).cuda(), group)
        per = -(-longest // 16)
        self.cache = F.new_cache4(batch * per, kv_heads, 16, dim, 32)
        self.table = torch.randperm(batch * per, generator=g).to(torch.int32).reshape(batch, per).cuda()
        self.lengths = torch.zeros(batch, dtype=torch.int32, device="cuda")

    def step(self, x):
        y = F.forward_connected4(self.qkv, x).view(self.batch, 1, self.heads + 2 * self.kv_heads, self.dim)
        q, k, v = y.split((self.heads, self.kv_heads, self.kv_heads), 2)
        self.lengths += 1
        F.append4(self.cache, k, v, self.table, self.lengths)
        a = F.attend4(self.cache, q, self.table, self.lengths)
        return q, k, v, a, F.forward_connected4(self.back, a.view(self.batch, -1))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_a_decoder_answers_token_by_token(dtype):
    block = Block(200, 6, 2, 64, 64, 3, 40, dtype)
    for i in range(35):
        x = torch.randn(3, 200, generator=rng(i)).to(dtype).cuda()
        q, k, v, a, y = block.step(x)
        if i in (0, 1, 16, 34):
            check_product(block.qkv, x, torch.cat((q, k, v), 2).reshape(3, -1))
            s = Sequences.__new__(Sequences)
            s.cache, s.table, s.lengths, s.group, s.dim = block.cache, block.table.tolist(), block.lengths.tolist(), 32, 64
            check_attend(s, q)
            check_product(block.back, a.reshape(3, -1), y)
            kept = F.read4(block.cache, block.table, block.lengths, 1, dtype=torch.float32)
            for stored, given in zip(kept, (k, v)):
                # half a step of a range of at most twice the largest value, and fp16's rounding of its ends
                assert (stored - given.float()).abs().max() <= given.float().abs().max() * (2 / 30 + 2.0 ** -9)


def test_a_step_in_a_graph_and_on_another_stream():
    eager, captured = (Block(128, 4, 2, 32, 32, 2, 64, torch.float16) for _ in range(2))
    x = torch.zeros(2, 128, dtype=torch.float16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        captured.step(x)                                     # first launches outside the capture
        captured.lengths.zero_()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = captured.step(x)
    for i in range(40):
        x.copy_(torch.randn(2, 128, generator=rng(i)))
        want = eager.step(x)
        graph.replay()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        again = eager.step(x)
    torch.cuda.current_stream().wait_stream(side)
    graph.replay()
    assert torch.equal(out[-1], again[-1])


def test_two_graphs_of_long_sequences_side_by_side():
    """Calls that need scratch memory, replayed at the same time: each graph has its own."""
    sets = []
    for seed in (1, 2):
        s = Sequences([6000], 1, 64, 32, 64, seed=seed)
        q = torch.randn(1, 1, 4, 64, generator=rng(seed)).half().cuda()
        table, lengths = s.device()
        want = F.attend4(s.cache, q, table, lengths)
        c = s.cache
        assert capi.lib().xnor_b200_kv4_attend_scratch_bytes(
            capi.Kv4Cache(*(t.data_ptr() for t in c._native[:4]), c.pages, c.kv_heads, c.page, c.dim, c.group),
            capi.Kv4Rows(1, 1, table.shape[1], table.data_ptr(), lengths.data_ptr(), None), 4, 0) > 0
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = F.attend4(s.cache, q, table, lengths)
        sets.append((graph, out, want, torch.cuda.Stream(), (s, q, table, lengths)))
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, _, _, stream, _ in sets:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, out, want, _, _ in sets:
        assert torch.equal(out, want)


def test_handles_keep_what_they_were_made_with():
    m, s = matrix(30, 64, 32, 0), Sequences([20, 3], 2, 64, 32)
    for handle, name in ((m, "codes"), (m, "k"), (s.cache, "v_scales"), (s.cache, "pages")):
        with pytest.raises(AttributeError):
            setattr(handle, name, getattr(handle, name))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_a_whole_prompt(dtype):
    """Hundreds of new tokens of ragged sequences at once, appended and attended to, with and without a window."""
    s = Sequences([0, 330, 301, 300, 7, 640], 2, 64, 32, 48, seed=3)
    counts = [0, 300, 300, 300, 7, 120]
    n = torch.tensor(counts, dtype=torch.int32, device="cuda")
    table, lengths = s.device()
    k, v = (torch.randn(6, 300, 2, 64, generator=rng(i)).to(dtype).cuda() for i in (1, 2))
    F.append4(s.cache, k, v, table, lengths, n)
    q = torch.randn(6, 300, 6, 64, generator=rng(3)).to(dtype).cuda()
    check_attend(s, q, counts=counts)
    check_attend(s, q, counts=counts, window=77)


def test_a_graph_that_forks():
    """Calls on two streams of one capture, each behind the other's: launches that overlap their predecessor wait for all they depend on."""
    m = [matrix(256, 256, 64, i) for i in range(4)]
    s = Sequences([900, 40], 2, 64, 32, 64, seed=2)
    table, lengths = s.device()
    x = torch.randn(2, 256, generator=rng(1)).half().cuda()
    side = torch.cuda.Stream()

    def work(fork):
        a = F.forward_connected4(m[0], x)
        if fork:
            side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side if fork else torch.cuda.current_stream()):
            b = F.attend4(s.cache, a.view(2, 1, 4, 64), table, lengths)
            b = F.forward_connected4(m[1], b.view(2, 256))
        c = F.forward_connected4(m[2], a * 0.5)
        if fork:
            torch.cuda.current_stream().wait_stream(side)
        return F.forward_connected4(m[3], (b + c) * 0.01)

    work(False)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work(True)
    for i in range(20):
        x.copy_(torch.randn(2, 256, generator=rng(i)))
        graph.replay()
        got = out.clone()
        assert torch.equal(got, work(False))


def test_calls_behind_one_another_see_what_was_written():
    """A long chain of short calls, each of which reads what the one before wrote, against the same calls one at a time."""
    m = [matrix(192, 192, 32, i) for i in range(3)]
    s = Sequences([64], 1, 64, 32, 16, seed=1)
    table, lengths = s.device()

    def chain(wait):
        x = torch.randn(1, 192, generator=rng(7)).cuda()
        for i in range(200):
            x = F.forward_connected4(m[i % 3], x) * 0.05
            kv = x[:, :128].view(1, 1, 2, 64)
            F.append4(s.cache, kv[:, :, :1], kv[:, :, 1:], table, lengths)
            k, v = F.read4(s.cache, table, lengths, 1)
            a = F.attend4(s.cache, x[:, 128:].view(1, 1, 1, 64), table, lengths)
            x = torch.cat((k.view(1, 64), v.view(1, 64), a.view(1, 64)), 1)
            if wait:
                torch.cuda.synchronize()
        return x

    want = chain(True)
    for _ in range(3):
        assert torch.equal(chain(False), want)


def test_refusals_name_the_fault():
    m = matrix(8, 64, 32, 0)
    x = torch.zeros(2, 64, device="cuda")
    s = Sequences([20, 3], 2, 64, 32)
    table, lengths = s.device()
    q, k = torch.zeros(2, 1, 4, 64, device="cuda"), torch.zeros(2, 1, 2, 64, device="cuda")
    for wrong in (lambda: F.forward_connected4(m, x.double()), lambda: F.forward_connected4(m, x[:, :63]), lambda: F.forward_connected4(m, x.cpu()),
                  lambda: F.forward_connected4(m, x, torch.zeros(7, device="cuda")), lambda: F.forward_connected4(m, x, activation=5),
                  lambda: F.forward_connected4(m, x, out=torch.zeros(2, 9, device="cuda")), lambda: F.forward_connected4(m, x.t().contiguous().t()),
                  lambda: F.append4(s.cache, k, k.half(), table, lengths), lambda: F.append4(s.cache, k[:, :, :1], k[:, :, :1], table, lengths),
                  lambda: F.append4(s.cache, k, k, table.long(), lengths), lambda: F.append4(s.cache, k, k, table, lengths[:1]),
                  lambda: F.append4(s.cache, k, k, table.cpu(), lengths), lambda: F.attend4(s.cache, q[:, :, :3], table, lengths),
                  lambda: F.attend4(s.cache, q, table[:1], lengths), lambda: F.attend4(s.cache, q, table, lengths, window=-1),
                  lambda: F.attend4(s.cache, q, table, lengths, out=q[:, :, :, :32]), lambda: F.attend4(s.cache, q[..., :32], table, lengths),
                  lambda: F.attend4(s.cache, q, table, lengths, out=q[:, :, :1].expand(-1, -1, 4, -1)),
                  lambda: F.attend4(s.cache, q, table, lengths, window=0.5), lambda: F.read4(s.cache, table, lengths, -1),
                  lambda: F.read4(s.cache, table, lengths, 1, dtype=torch.float64), lambda: F.forward_connected4(m, x, biases=x[0, :8].half()),
                  lambda: F.attend4(s.cache, q.transpose(2, 3).contiguous().transpose(2, 3), table, lengths),
                  lambda: F.attend4(s.cache, q, table, lengths, lse=torch.zeros(2, 1, 4, device="cuda").half())):
        with pytest.raises(ValueError):
            wrong()
    with pytest.raises(capi.XnorError, match="invalid size"):
        F.attend4(s.cache, q, table, lengths, scale=math.inf)
    assert F.forward_connected4(m, x[:0]).shape == (0, 8)
    assert F.attend4(s.cache, q[:, :0], table, lengths).shape == (2, 0, 4, 64)
    F.append4(s.cache, k[:, :0], k[:, :0], table, lengths)
