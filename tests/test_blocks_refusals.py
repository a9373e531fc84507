"""The ops of decoder layers in 8 and 4 bits say no to what they cannot compute,
before anything reaches a GPU."""
import numpy as np
import pytest


@pytest.fixture(scope="module")
def om():
    import om_mi355x
    om_mi355x.load()
    return om_mi355x


def f8(om, *shape):
    return np.zeros(shape, om.float8_e4m3fn)


def f32(*shape):
    return np.zeros(shape, np.float32)


def refused(om, what, call):
    with pytest.raises(om.RuntimeError_, match=what):
        call()


def test_quantize_blocks_refuses(om):
    Q = om.DynamicQuantizeBlocks
    refused(om, "expected f32, f16 or bf16 x", lambda: Q(np.zeros((2, 128), np.int8)))
    refused(om, "block_rows must be 1, or 128", lambda: Q(f32(2, 128), 64))
    refused(om, "block_rows must be 1, or 128", lambda: Q(f32(2, 2, 128), 128, out=(f8(om, 2, 2, 128), f32(1, 1))))
    refused(om, "y_scale has 2 entries, expected 4", lambda: Q(f32(2, 129), out=(f8(om, 2, 129), f32(2, 1))))
    refused(om, "f8e4m3fn y of x's shape", lambda: Q(f32(2, 128), out=(f8(om, 128, 2), f32(2, 1))))
    refused(om, "f8e4m3fn y of x's shape", lambda: Q(f32(2, 128), out=(np.zeros((2, 128), np.uint8), f32(2, 1))))


def test_matmul_blocks_refuses(om):
    def product(a=(4, 200), a_scale=(4, 2), b=(130, 200), b_scale=(2, 2), **kw):
        return om.MatMulBlocks(f8(om, *a), f32(*a_scale), f8(om, *b), f32(*b_scale), **kw)

    refused(om, "inner dimensions differ \\(200 vs 128\\)", lambda: product(b=(130, 128)))
    refused(om, "b_scale \\[2, 2\\]", lambda: product(b_scale=(1, 2)))
    refused(om, "a_scale \\[.., 2\\]", lambda: product(a_scale=(4, 1)))
    refused(om, "expected f8e4m3fn a", lambda: om.MatMulBlocks(np.zeros((4, 200), np.int8), f32(4, 2), f8(om, 130, 200), f32(2, 2)))
    refused(om, "expected f8e4m3fn a", lambda: product(dtype=np.int32))
    refused(om, "output has 8 elements, expected 520", lambda: product(out=f32(4, 2)))
    refused(om, "bias must be f32, scalar or", lambda: product(bias=f32(7)))
    refused(om, "activation 5 is not", lambda: product(activation=5))


def test_a_product_of_too_many_elements_is_refused(om):
    """Offsets within a tile's rows are counted in 32 bits (nothing is read)."""
    K = 2 ** 22 + 128
    a, b = (om.DeviceArray.wrap(4096, (n, K), om.float8_e4m3fn) for n in (1, 128))
    sa, sb = (om.DeviceArray.wrap(4096, (1, K // 128), np.dtype(np.float32)) for _ in range(2))
    y = om.DeviceArray.wrap(4096, (1, 128), np.dtype(np.float32))
    refused(om, "too large|2\\^22", lambda: om.MatMulBlocks(a, sa, b, sb, out=y))


@pytest.mark.parametrize("M,N", [(1, 2 ** 27 - 127), (2 ** 30 + 1, 1), (2 ** 30, 1), (2 ** 18, 2 ** 19)])
def test_a_product_of_too_many_results_is_refused(om, M, N):
    """A launch has fewer than 2^32 threads (nothing is read)."""
    wrap = lambda shape, dtype: om.DeviceArray.wrap(4096, shape, np.dtype(dtype))
    a, b = wrap((M, 128), om.float8_e4m3fn), wrap((N, 128), om.float8_e4m3fn)
    sa, sb = wrap((M, 1), np.float32), wrap((-(-N // 128), 1), np.float32)
    refused(om, "too large", lambda: om.MatMulBlocks(a, sa, b, sb, out=wrap((M, N), np.float32)))


def test_rotary_refuses(om):
    R = om.RotaryEmbedding
    x, t, p = f32(2, 3, 5, 64), f32(10, 32), np.zeros((2, 5), np.int64)
    refused(om, "x must be \\[B, H, S, D\\]", lambda: R(f32(5, 64), t, t, p))
    refused(om, "do not divide into heads", lambda: R(f32(2, 5, 190), t, t, p, num_heads=3))
    refused(om, "do not divide into heads", lambda: R(f32(2, 5, 192), t, t, p))
    refused(om, "cannot be rotated", lambda: R(x, t, t, p, rotary_embedding_dim=66))
    refused(om, "cannot be rotated", lambda: R(x, t, t, p, rotary_embedding_dim=33))
    refused(om, "tables must be f32 \\[positions, 16\\]", lambda: R(x, t, t, p, rotary_embedding_dim=32))
    refused(om, "tables must be", lambda: R(x, t, f32(9, 32), p))
    refused(om, "tables must be", lambda: R(x, t, t))
    refused(om, "position_ids must be i64 \\[2, 5\\]", lambda: R(x, t, t, np.zeros((2, 4), np.int64)))
    refused(om, "y of x's type and shape", lambda: R(x, t, t, p, out=np.zeros(x.shape, np.float16)))
    refused(om, "interleaved 0 or 1", lambda: R(x, t, t, p, interleaved=2))


def i32(*v):
    return np.array(v, np.int32)


def test_cache_append_refuses(om):
    c = om.Cache4(4, 2, 16, 64)
    k = f32(2, 2, 3, 64)
    A = om.CacheAppend4
    past = i32(0, 0)
    refused(om, "k is \\[.., 3 heads, .., 64\\]", lambda: A(c, f32(2, 3, 3, 64), f32(2, 3, 3, 64), past))
    refused(om, "do not divide into heads", lambda: A(c, f32(2, 3, 130), f32(2, 3, 130), past))
    refused(om, "v of k's type and shape", lambda: A(c, k, f32(2, 2, 4, 64), past))
    refused(om, "past must be i32 \\[2\\]", lambda: A(c, k, k, i32(0)))
    refused(om, "counts must be i32 \\[2\\]", lambda: A(c, k, k, past, counts=i32(1, 1, 1)))
    refused(om, "5 sequences without a page table, and 4 pages", lambda: A(c, f32(5, 2, 3, 64), f32(5, 2, 3, 64), i32(0, 0, 0, 0, 0)))
    refused(om, "page_table must be i32", lambda: A(c, k, k, past, np.zeros((1, 2), np.int32)))
    refused(om, "page_size must be a multiple of 16", lambda: A(om.Cache4(4, 2, 24, 64), k, k, past, np.zeros((2, 1), np.int32)))
    refused(om, "heads of 80 elements", lambda: A(om.Cache4(4, 2, 16, 80), k, k, past))
    refused(om, "past\\[1\\] is 14", lambda: A(c, k, k, i32(13, 14)))
    refused(om, "past\\[0\\] is -1", lambda: A(c, k, k, i32(-1, 0)))
    refused(om, "counts\\[1\\] is 4, of 3 rows", lambda: A(c, k, k, past, counts=i32(1, 4)))
    bad = np.array([[0, 1], [2, 4]], np.int32)
    refused(om, "page_table\\[1, 1\\] is 4, of 4 pages", lambda: A(c, k, k, i32(0, 14), bad))
    refused(om, "page_table\\[0, 0\\] is -1", lambda: A(c, k, k, i32(0, 0), np.array([[-1, 1], [2, 3]], np.int32)))
    small = om.Cache4(4, 2, 16, 64)
    small.v_scales = np.zeros((4, 2, 16, 2, 2), np.float32)
    refused(om, "scales must be f16", lambda: A(small, k, k, past))
    small = om.Cache4(4, 2, 16, 64)
    small.v_codes = np.zeros((4, 2, 16, 64), np.uint8)
    refused(om, "codes must be ui8", lambda: A(small, k, k, past))


def test_cache_attention_refuses(om):
    c = om.Cache4(4, 2, 16, 64)
    q, past = f32(2, 4, 1, 64), i32(3, 3)
    A = om.CacheAttention4
    refused(om, "5 query heads on 2 heads of keys", lambda: A(f32(2, 5, 1, 64), c, past))
    refused(om, "do not divide into heads", lambda: A(f32(2, 1, 100), c, past))
    refused(om, "q is \\[.., 4 heads, .., 128\\]", lambda: A(f32(2, 4, 1, 128), c, past))
    refused(om, "y of q's type and shape", lambda: A(q, c, past, out=f32(2, 4, 2, 64)))
    refused(om, "starts must be i32 \\[2\\]", lambda: A(q, c, past, starts=i32(1)))
    refused(om, "scale must be an f32 scalar", lambda: A(q, c, past, scale=f32(2)))
    refused(om, "causal must be 0 or 1", lambda: A(q, c, past, causal=2))
    refused(om, "window not negative", lambda: A(q, c, past, window=-1))
    refused(om, "past\\[0\\] is 16", lambda: A(q, c, i32(16, 0)))
    refused(om, "page_table\\[0, 0\\] is 9", lambda: A(q, c, past, np.array([[9], [0]], np.int32)))
    refused(om, "the cache has no room", lambda: A(q, om.Cache4(2, 2, 0, 64), i32(0, 0), counts=i32(0, 0)))


def test_a_cache_of_too_many_rows_is_refused(om):
    """Rows are counted in 32 bits (nothing is allocated, and nothing read)."""
    c = om.Cache4(1, 1, 16, 64)
    shape = (2 ** 20, 64, 64)
    c.k_codes, c.v_codes = (om.DeviceArray.wrap(4096, shape + (32,), np.dtype(np.uint8)) for _ in range(2))
    c.k_scales, c.v_scales = (om.DeviceArray.wrap(4096, shape + (2, 2), np.dtype(np.float16)) for _ in range(2))
    k = om.DeviceArray.wrap(4096, (1, 64, 1, 64), np.dtype(np.float32))
    past = om.DeviceArray.wrap(4096, (1,), np.dtype(np.int32))
    refused(om, "2\\^32 rows", lambda: om.CacheAppend4(c, k, k, past))
    refused(om, "2\\^32 rows", lambda: om.CacheAttention4(k, c, past, out=k))


def test_types_that_numpy_lacks_keep_their_bits(om):
    x = np.array([1.0, -2.5, 3.0e38, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, np.inf, -0.0, 0.0], np.float32)
    b = om.from_float32(x, om.bfloat16)
    assert b.dtype == om.bfloat16 and b.shape == x.shape
    v = om.to_float32(b)
    assert np.all(np.abs(v[:5] - x[:5]) <= 2.0 ** -8 * np.abs(x[:5])) and v[3] == 1 and v[4] == 1 + 2.0 ** -6
    assert v[5] == np.inf and np.signbit(v[6]) and not np.signbit(v[7])
    assert np.isnan(om.to_float32(om.from_float32(np.float32([np.nan]), om.bfloat16)))[0]
    codes = np.arange(256, dtype=np.uint8).view(om.float8_e4m3fn)
    e = om.to_float32(codes)
    assert e[0x38] == 1 and e[0x7E] == 448 and e[0x01] == 2.0 ** -9 and e[0xB8] == -1
    assert np.isnan(e[0x7F]) and np.isnan(e[0xFF]) and np.isfinite(np.delete(e, [0x7F, 0xFF])).all()


def test_rotary_tables(om):
    cos, sin = om.rotary_tables(50, 8)
    p, i = 49, 3
    assert cos.shape == sin.shape == (50, 4) and cos.dtype == np.float32
    assert cos[p, i] == np.float32(np.cos(p * 10000.0 ** (-2 * i / 8)))
    assert sin[p, 0] == np.float32(np.sin(49.0))
    lin, _ = om.rotary_tables(50, 8, scaling="linear", factor=2.0)
    assert np.array_equal(lin[2::2], cos[1:25])
    # (from the sines: a cosine near 1 says nothing of its angle in f32)
    ntk = np.arcsin(om.rotary_tables(2, 8, scaling="ntk", factor=4.0)[1][1].astype(np.float64))
    own = np.arcsin(sin[1].astype(np.float64))
    assert abs(ntk[0] - own[0]) < 1e-6 and abs(ntk[3] / own[3] * 4 - 1) < 1e-3
    c, s = om.rotary_tables(2, 64, scaling="yarn", factor=8.0, trained=4096)
    gain = 0.1 * np.log(8.0) + 1
    rate = np.arctan2(s[1].astype(np.float64), c[1].astype(np.float64))
    base = 10000.0 ** (-np.arange(0, 64, 2) / 64)
    assert np.allclose(np.hypot(c, s), gain, rtol=2e-7)
    assert abs(rate[0] / base[0] - 1) < 1e-6 and abs(rate[-1] / base[-1] * 8 - 1) < 1e-5
    for bad in (dict(dim=7), dict(dim=8, factor=0.5), dict(dim=8, scaling="yarn"), dict(dim=8, scaling="other")):
        with pytest.raises(ValueError):
            om.rotary_tables(4, **{"factor": 2.0, **bad})


def test_from_float32_refuses_types_that_it_does_not_round_to(om):
    for dtype in (om.float8_e4m3fn, np.uint8, np.int32, np.float64):
        with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
            om.from_float32(np.float32([1.5, 300.0]), dtype)
    assert om.from_float32(np.float32([1.5]), "float16").dtype == np.float16


def test_scales_the_other_way_round_are_refused(om):
    """As many entries, but not blocks of a row beside one another."""
    a, b = f8(om, 4, 200), f8(om, 300, 200)
    refused(om, "a_scale \\[.., 2\\]", lambda: om.MatMulBlocks(a, f32(2, 4), b, f32(3, 2)))
    refused(om, "b_scale \\[3, 2\\]", lambda: om.MatMulBlocks(a, f32(4, 2), b, f32(2, 3)))
    refused(om, "y_scale must be \\[.., 2\\]", lambda: om.DynamicQuantizeBlocks(f32(4, 200), out=(a, f32(2, 4))))
    refused(om, "y_scale must be \\[.., 2\\]", lambda: om.DynamicQuantizeBlocks(f32(300, 200), 128, out=(b, f32(2, 3))))
