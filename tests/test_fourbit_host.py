"""Four-bit operators without a GPU: the format's reference, sizes, and refusals that answer before anything is launched."""
import ctypes as C

import numpy as np
import pytest

import four_reference as R

torch = pytest.importorskip("torch")

from darknet_b200 import build, capi, fourbit as F  # noqa: E402


@pytest.fixture(scope="module")
def L():
    build.build()
    return capi.lib()


def test_the_format_clips_nothing():
    rows = np.random.default_rng(1).standard_normal((50, 96)) * np.logspace(-7, 4, 50)[:, None]
    codes, scales = R.quantize(rows, 32)
    back, size = R.values(R.pack(codes), scales, 32, 96)
    step = np.repeat(scales[..., 0].astype(np.float64), 32, -1)
    assert (np.abs(back - rows) <= step * 0.5 * (1 + 1e-12)).all() and (size >= np.abs(back) * (1 - 1e-12)).all()
    assert codes.min() == 0 and codes.max() == 15
    np.testing.assert_array_equal(R.unpack(R.pack(codes), 96), codes)


def test_sizes(L):
    def sizes(n, k, group):
        d = capi.W4Desc(n, k, group, 0)
        return L.xnor_b200_w4_code_bytes(C.byref(d)), L.xnor_b200_w4_scale_bytes(C.byref(d))
    assert sizes(10, 256, 64) == (10 * 128, 10 * 4 * 4)
    assert sizes(3, 33, 32) == (3 * 32, 3 * 2 * 4)
    assert sizes(3, 1, 128) == (3 * 16, 3 * 4)
    assert sizes(1 << 20, 1 << 20, 32) == (1 << 39, 1 << 37)
    for wrong in ((0, 8, 32), (8, 0, 32), (8, 8, 16), (8, -1, 64)):
        assert sizes(*wrong) == (0, 0)
    assert L.xnor_b200_w4_code_bytes(None) == 0 and L.xnor_b200_w4_scale_bytes(None) == 0


def test_products_refuse(L):
    d = capi.W4Desc(16, 64, 32, 0)

    def forward(d=d, x=256, dtype=0, rows=1, ldx=64, codes=256, scales=256, biases=None, out=256, ldo=16, scratch=None, nbytes=0):
        return L.xnor_b200_w4_forward(None if d is None else C.byref(d), x, dtype, rows, ldx, codes, scales, biases, out, ldo, scratch, nbytes, None)

    for null in ("d", "x", "codes", "scales", "out"):
        assert forward(**{null: None}) == 2
    for wrong in (dict(dtype=3), dict(dtype=-1), dict(rows=0), dict(rows=-4), dict(ldx=-1), dict(ldo=15), dict(d=capi.W4Desc(0, 64, 32, 0)),
                  dict(d=capi.W4Desc(16, 64, 48, 0)), dict(d=capi.W4Desc(16, 64, 32, 2)), dict(d=capi.W4Desc(16, -5, 32, 0))):
        assert forward(**wrong) == 1, wrong
    for odd in (dict(codes=264), dict(scales=258), dict(x=258), dict(out=258), dict(biases=257)):
        assert forward(**odd) == 5, odd
    assert forward(rows=(1 << 16) + 1) == 6
    assert forward(d=capi.W4Desc(16, (1 << 24) + 1, 32, 0)) == 6
    # a large product of many rows converts x once, into scratch memory
    large, small = capi.W4Desc(1 << 14, 1 << 13, 64, 0), capi.W4Desc(1 << 14, 1 << 12, 64, 0)
    need = L.xnor_b200_w4_scratch_bytes(C.byref(large), 1, 9)
    assert need >= 9 * (1 << 13) * 2 and L.xnor_b200_w4_scratch_bytes(C.byref(large), 2, 17) > 2 * need
    assert L.xnor_b200_w4_scratch_bytes(C.byref(large), 1, 8) == 0 and L.xnor_b200_w4_scratch_bytes(C.byref(small), 1, 16) == 0
    assert L.xnor_b200_w4_scratch_bytes(C.byref(large), 5, 16) == 0 and L.xnor_b200_w4_scratch_bytes(None, 1, 16) == 0
    many = dict(d=large, dtype=1, rows=9, ldx=1 << 13, ldo=1 << 14)
    assert forward(**many) == 2 and forward(**many, scratch=256, nbytes=need - 1) == 3 and forward(**many, scratch=264, nbytes=need) == 5
    assert L.xnor_b200_w4_quantize(C.byref(d), None, 0, 64, 256, 256, None) == 2
    assert L.xnor_b200_w4_quantize(C.byref(d), 256, 7, 64, 256, 256, None) == 1
    assert L.xnor_b200_w4_quantize(C.byref(d), 256, 0, 64, 264, 256, None) == 5


def cache(pages=4, kv_heads=2, page=16, dim=64, group=32, **pointers):
    at = dict(k_codes=256, k_scales=256, v_codes=256, v_scales=256) | pointers
    return capi.Kv4Cache(at["k_codes"], at["k_scales"], at["v_codes"], at["v_scales"], pages, kv_heads, page, dim, group)


def rows(batch=1, tokens=1, max_pages=2, table=256, lengths=256, counts=None):
    return capi.Kv4Rows(batch, tokens, max_pages, table, lengths, counts)


def tensor(data=256, dtype=0):
    return capi.Kv4Tensor(data, dtype, 64, 64, 64)


def test_caches_refuse(L):
    def every(c, r):
        t = tensor()
        return {L.xnor_b200_kv4_append(c, r, t, t, None), L.xnor_b200_kv4_read(c, r, t, t, None),
                L.xnor_b200_kv4_attend(c, r, t, 4, 1.0, 0, t, None, None, 0, None)}

    for c in (cache(pages=0), cache(page=8), cache(page=24), cache(dim=48), cache(group=16), cache(dim=96, group=64), cache(kv_heads=0), cache(dim=0)):
        assert every(c, rows()) == {1}
    for r in (rows(batch=0), rows(tokens=-1), rows(max_pages=0)):
        assert every(cache(), r) == {1}
    for name in ("k_codes", "k_scales", "v_codes", "v_scales"):
        assert every(cache(**{name: None}), rows()) == {2}
        assert every(cache(**{name: 264}), rows()) == {5}
    assert every(cache(), rows(table=None)) == {2} and every(cache(), rows(lengths=None)) == {2}
    assert every(cache(), rows(table=258)) == {5} and every(cache(), rows(counts=257)) == {5}
    assert every(cache(dim=288), rows()) == {6} and every(cache(), rows(batch=1 << 16, tokens=1 << 16)) == {6}


def test_attention_refuses(L):
    def attend(c=cache(), r=rows(), q=tensor(), heads=4, scale=1.0, window=0, out=tensor(), lse=None, scratch=None, nbytes=0):
        return L.xnor_b200_kv4_attend(c, r, q, heads, scale, window, out, lse, scratch, nbytes, None)

    for wrong in (dict(heads=3), dict(heads=0), dict(window=-1), dict(scale=float("inf")), dict(scale=float("nan")), dict(q=tensor(dtype=1)), dict(q=tensor(dtype=4), out=tensor(dtype=4))):
        assert attend(**wrong) == 1, wrong
    assert attend(q=tensor(None)) == 2 and attend(out=None) == 2
    assert attend(q=tensor(258)) == 5 and attend(lse=258) == 5
    assert attend(r=rows(batch=65536)) == 6
    # a long table of one sequence is split over CTAs that leave their sums in scratch memory
    c, r = cache(pages=100000), rows(max_pages=4096)
    need = L.xnor_b200_kv4_attend_scratch_bytes(c, r, 4, 0)
    assert need > 0 and need % 4 == 0
    assert attend(c=c, r=r) == 2
    assert attend(c=c, r=r, scratch=256, nbytes=need - 1) == 3
    assert attend(c=c, r=r, scratch=264, nbytes=need) == 5
    assert L.xnor_b200_kv4_attend_scratch_bytes(c, rows(), 4, 0) == 0                   # a short one is not
    assert L.xnor_b200_kv4_attend_scratch_bytes(c, r, 4, 100) == 0                      # nor a short window
    assert L.xnor_b200_kv4_attend_scratch_bytes(c, r, 3, 0) == 0


def test_a_missing_binding_fails_loudly(L, monkeypatch):
    import sys
    calls = F._Calls()
    monkeypatch.setitem(sys.modules, "darknet_b200._fourbit", None)
    monkeypatch.delattr("darknet_b200._fourbit", raising=False)
    with pytest.raises(FileNotFoundError, match="no CPU or PyTorch fallback"):
        calls.product


def test_bindings_take_nothing_else(L):
    from darknet_b200 import _fourbit
    t = torch.zeros(2, 2)
    for f in (_fourbit.product, _fourbit.append, _fourbit.read, _fourbit.attend):
        assert f() is None and f(t) is None and f(None, None, None, None, None, None) is None
        for n in (5, 6, 9):
            assert f(*["x"] * n) is None and f(*[t] * n) is None and f((t,) * 5, *[t] * (n - 1)) is None
            assert f((t, t, 2, 32), *[None] * (n - 1)) is None


def test_tensors_off_the_gpu_are_refused(L):
    codes, scales = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, 2, dtype=torch.float16)
    m = F.Matrix4(codes, scales, 64, 32)
    with pytest.raises(ValueError, match="CUDA device"):
        F.forward_connected4(m, torch.zeros(1, 64))
    with pytest.raises(ValueError, match="CUDA device"):
        F.quantize_weights4(torch.zeros(4, 64), 32)
    c = F.new_cache4(3, 2, 16, 64, 32, device="cpu")
    i32 = dict(dtype=torch.int32)
    table, lengths, x = torch.zeros(1, 2, **i32), torch.zeros(1, **i32), torch.zeros(1, 1, 2, 64)
    for call in (lambda: F.append4(c, x, x, table, lengths), lambda: F.read4(c, table, lengths, 1), lambda: F.attend4(c, x, table, lengths)):
        with pytest.raises(ValueError, match="CUDA device"):
            call()


@pytest.mark.parametrize("what", ["codes", "scales", "group", "k", "dtype"])
def test_matrices_of_other_shapes_are_refused(what):
    args = dict(codes=torch.zeros(4, 32, dtype=torch.uint8), scales=torch.zeros(4, 2, 2, dtype=torch.float16), k=64, group=32)
    F.Matrix4(**args)
    args |= dict(codes=dict(codes=torch.zeros(4, 33, dtype=torch.uint8)), scales=dict(scales=torch.zeros(4, 3, 2, dtype=torch.float16)),
                 group=dict(group=48), k=dict(k=0), dtype=dict(scales=torch.zeros(4, 2, 2)))[what]
    with pytest.raises(ValueError):
        F.Matrix4(**args)


@pytest.mark.parametrize("shape", [(3, 2, 8, 64, 32), (3, 2, 16, 48, 32), (3, 2, 16, 96, 64), (3, 2, 16, 288, 32), (0, 2, 16, 64, 32), (3, 2, 16, 64, 16)])
def test_caches_of_other_shapes_are_refused(shape):
    with pytest.raises(ValueError):
        F.new_cache4(*shape, device="cpu")


@pytest.mark.parametrize("n, k", [(2 ** 32 + 5, 32), (2 ** 28 + 1, 8), (1, 2 ** 24 + 1), (2, 2 ** 32 + 64)])
def test_matrices_beyond_an_int_are_refused(n, k):
    """(Sizes that the C ABI's ints would have cut down to other, valid ones.)"""
    on = dict(device="meta")
    codes, scales = torch.empty(n, (k + 31) // 32 * 16, dtype=torch.uint8, **on), torch.empty(n, (k + 31) // 32, 2, dtype=torch.float16, **on)
    with pytest.raises(ValueError, match="at most"):
        F.Matrix4(codes, scales, k, 32)
    with pytest.raises(ValueError, match="at most"):
        F.quantize_weights4(torch.empty(n, k, **on), 32)
    F.Matrix4(torch.empty(2 ** 28, 16, dtype=torch.uint8, **on), torch.empty(2 ** 28, 1, 2, dtype=torch.float16, **on), 32, 32)
    F.Matrix4(torch.empty(2, 2 ** 23, dtype=torch.uint8, **on), torch.empty(2, 2 ** 19, 2, dtype=torch.float16, **on), 2 ** 24, 32)


def test_caches_beyond_an_int_are_refused():
    with pytest.raises(ValueError, match="below 2"):
        F.new_cache4(2 ** 32 + 1, 1, 16, 32, 32, device="meta")
    F.new_cache4(2 ** 31 - 1, 1, 16, 32, 32, device="meta")


def test_the_limits_are_the_headers():
    import os
    import re
    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "xnor_b200.h")).read()
    for name in ("W4_MAX_K", "W4_MAX_N", "KV4_MAX_DIM"):
        value = re.search(rf"#define XNOR_B200_{name}\s+(.*)", header)[1]
        assert eval(value) == getattr(capi, name)


def test_memory_in_common_is_found(L):
    """Views of one buffer against what their entries' numbers say."""
    import random
    from darknet_b200 import _fourbit
    r = random.Random(5)
    buffer = torch.arange(600, dtype=torch.int16)
    found = {True: 0, False: 0}
    for i in range(4000):
        def view(like=None):
            if like is not None and r.random() < 0.5:
                size, stride = like.size(), like.stride()
            else:
                size = [r.choice((1, 1, 2, 3, 4)) for _ in range(r.choice((1, 2, 3)))] + [r.choice((1, 2, 5))]
                stride = [r.choice((0, 1, 3, 5, 6, 10, 20, 40)) for _ in size[:-1]] + [r.choice((1, 1, 1, 2))]
            room = 600 - sum((n - 1) * s for n, s in zip(size, stride))
            return buffer.as_strided(size, stride, r.randrange(min(60, room)))
        a = view()
        b = view(a)
        entries = a.flatten().tolist()
        assert _fourbit.shares(a) == (len(set(entries)) < len(entries)), (a.size(), a.stride())
        want = bool(set(entries) & set(b.flatten().tolist()))
        assert _fourbit.shares(a, b) == want, (a.size(), a.stride(), b.size(), b.stride(), a.storage_offset(), b.storage_offset())
        found[want] += 1
    assert min(found.values()) > 500
    wide = buffer.view(torch.int32)                          # entries of another size
    assert _fourbit.shares(wide[3:5], buffer[9:20]) and not _fourbit.shares(wide[3:5], buffer[10:20])
    assert not _fourbit.shares(buffer[:0], buffer) and _fourbit.shares(torch.zeros(2, 2)) is False
    qkv = torch.zeros(64, 512, 24, 128, device="cpu", dtype=torch.float16)
    assert not _fourbit.shares(qkv[:, :, :8], qkv[:, :, 8:16]) and _fourbit.shares(qkv[:, :, :9], qkv[:, :, 8:17])


def test_attention_over_prompts_has_the_limit_that_the_header_names(L):
    """65535 tiles of columns in a call's grid: of 8 columns, up to dim 128 of 24.  (Refusals only: nothing is launched.)"""
    def attend(tokens, heads, kv_heads, dim):
        c, r, t = cache(dim=dim, kv_heads=kv_heads), rows(tokens=tokens), tensor()
        return L.xnor_b200_kv4_attend(c, r, t, heads, 1.0, 0, t, None, None, 0, None)
    assert attend(65535 // 8 * 2 + 2, 32, 8, 256) == 6 and attend(65535 // 8 * 6 + 6, 32, 8, 128) == 6
    assert attend(1, 32, 65536, 64) in (1, 6) and attend((1 << 31) - 1, 64, 1, 64) == 6


def test_handles_whose_buffers_have_changed_are_refused(L):
    """The attributes are fixed, the tensors are the caller's: one that has been resized would be read and written beyond its end."""
    i32 = dict(dtype=torch.int32)
    x = torch.zeros(1, 64)
    for change in (lambda m: m.codes.resize_(9, 32), lambda m: m.scales.resize_(4, 1, 2), lambda m: m.scales.set_(torch.zeros(1, dtype=torch.float16)),
                   lambda m: m.codes.t_()):
        m = F.Matrix4(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, 2, dtype=torch.float16), 64, 32)
        change(m)
        with pytest.raises(ValueError, match="made with"):
            F.forward_connected4(m, x)
    kv, table, lengths = torch.zeros(1, 1, 2, 64), torch.zeros(1, 2, **i32), torch.zeros(1, **i32)
    for change in (lambda c: c.k_codes.resize_(4, 2, 16, 32), lambda c: c.v_codes.resize_(1, 2, 16, 32), lambda c: c.k_scales.resize_(3, 2, 16, 1, 2),
                   lambda c: c.v_scales.set_(torch.zeros(5, dtype=torch.float16)), lambda c: c.v_codes.transpose_(0, 1)):
        c = F.new_cache4(3, 2, 16, 64, 32, device="cpu")
        change(c)
        for call in (lambda: F.append4(c, kv, kv, table, lengths), lambda: F.read4(c, table, lengths, 1), lambda: F.attend4(c, kv, table, lengths)):
            with pytest.raises(ValueError, match="made with"):
                call()
