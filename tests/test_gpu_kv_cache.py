"""GPU: the 8-bit key/value cache (append, read, attention, eviction) against plain 64-bit torch."""

import math

import pytest
import torch

import dtorch_b200 as dt
from tests import kv_oracle as ko

pytestmark = pytest.mark.gpu
INT8, E4M3 = torch.int8, torch.float8_e4m3fn
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def tokens(gen, n, h, t, e, dtype):
    x = torch.randn((n, h, t, e), generator=gen) * torch.exp(torch.randn((1, h, 1, e), generator=gen))
    x = x * (1 + 5 * (torch.rand((n, h, t, 1), generator=gen) > 0.9))
    return x.to(dtype)


def junk(cache, lengths):
    """Fill what lies behind the lengths: float8 NaN / -128 codes, and NaN scales of blocks that hold nothing."""
    for i, l in enumerate(lengths):
        l = min(max(l, 0), cache.capacity)
        for c, s in ((cache.key, cache.key_scale), (cache.value, cache.value_scale)):
            c.view(torch.int8)[i, :, l:] = 127 if cache.dtype == E4M3 else -128
            s[i, :, -(-l // cache.block):] = math.nan


def filled(gen, lengths, h, cap, e, code, block, dtype=BF16):
    """A cache that holds lengths[i] tokens (appended at once), junk behind them, and its oracle."""
    n = len(lengths)
    cache = dt.QuantizedKVCache(n, h, cap, e, dtype=code, block=block)
    most = max(max(min(l, cap) for l in lengths), 0)
    k, v = tokens(gen, n, h, most, e, dtype), tokens(gen, n, h, most, e, dtype)
    counts = [min(max(l, 0), cap) for l in lengths]
    if most:
        dt.kv_cache_append(cache, k.cuda(), v.cuda(), ints([0] * n), counts=ints(counts))
    ok, ov = ko.Cache(n, h, cap, e, code, block), ko.Cache(n, h, cap, e, code, block)
    ok.append(k, [0] * n, counts)
    ov.append(v, [0] * n, counts)
    junk(cache, lengths)
    return cache, ok, ov


def same_cache(cache, ok, ov, lengths):
    for codes, scale, o in ((cache.key, cache.key_scale, ok), (cache.value, cache.value_scale, ov)):
        for i, l in enumerate(lengths):
            l = min(max(l, 0), cache.capacity)
            nb = -(-l // cache.block)
            assert torch.equal(codes[i, :, :l].float().cpu().double(), o.codes[i, :, :l])
            got, want = scale[i, :, :nb].cpu().double(), o.scale[i, :, :nb]
            assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("code", [INT8, E4M3])
@pytest.mark.parametrize("dtype,block,e,t", [(BF16, 64, 128, 1), (BF16, 32, 64, 3), (FP16, 64, 80, 64), (FP16, 128, 256, 131),
                                             (BF16, 128, 16, 300), (BF16, 32, 128, 65)])
def test_append_in_steps(code, dtype, block, e, t):
    gen = torch.Generator().manual_seed(t * 7 + e)
    n, h, cap = 5, 3, 640
    cache = dt.QuantizedKVCache(n, h, cap, e, dtype=code, block=block)
    ok, ov = ko.Cache(n, h, cap, e, code, block), ko.Cache(n, h, cap, e, code, block)
    lengths = [0, 1, block - 1, block, 2 * block + 5]
    for step in range(3):  # the second and third enter blocks that are filling, with larger tokens
        k, v = (tokens(gen, n, h, t, e, dtype) * (1 + 2 * step) for _ in range(2))
        counts = None if step != 1 else [t, 0, t // 2, t, max(t - 1, 0)]
        dt.kv_cache_append(cache, k.cuda(), v.cuda(), ints(lengths), counts=None if counts is None else ints(counts))
        ok.append(k, lengths, counts)
        ov.append(v, lengths, counts)
        start = lengths
        lengths = [min(l + (t if counts is None else counts[i]), cap) for i, l in enumerate(lengths)]
    del start
    # tokens before the first append were never written: zeros in both
    same_cache(cache, ok, ov, lengths)


def test_append_at_the_end_of_the_capacity_and_bad_lengths():
    gen = torch.Generator().manual_seed(3)
    n, h, cap, e = 6, 2, 128, 32
    cache = dt.QuantizedKVCache(n, h, cap, e, block=32)
    ok, ov = ko.Cache(n, h, cap, e, INT8, 32), ko.Cache(n, h, cap, e, INT8, 32)
    lengths = [120, 127, 128, 4000, -5, 0]
    k, v = tokens(gen, n, h, 40, e, BF16), tokens(gen, n, h, 40, e, BF16)
    dt.kv_cache_append(cache, k.cuda(), v.cuda(), ints(lengths), counts=ints([40, 40, 40, 40, 99, -3]))
    ok.append(k, lengths, [40, 40, 40, 40, 40, 0])
    ov.append(v, lengths, [40, 40, 40, 40, 40, 0])
    same_cache(cache, ok, ov, [128, 128, 128, 128, 40, 0])
    assert not cache.key[5].any() and not cache.key[2].any()


@pytest.mark.parametrize("layout", ["heads_last", "unaligned", "broadcast", "inner_strided"])
def test_append_of_strided_tokens(layout):
    gen = torch.Generator().manual_seed(5)
    n, h, t, e, cap = 2, 4, 37, 48, 64
    k, v = tokens(gen, n, h, t, e, BF16).cuda(), tokens(gen, n, h, t, e, BF16).cuda()

    def lay(x):
        if layout == "heads_last":
            return x.transpose(1, 2).contiguous().transpose(1, 2)
        if layout == "unaligned":
            flat = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")
            flat[1:] = x.reshape(-1)
            return flat[1:].view(x.shape)
        if layout == "broadcast":
            return x[:, :1].expand(n, h, t, e)
        return torch.stack([x, x], -1)[..., 0]

    k, v = lay(k), lay(v)
    cache = dt.QuantizedKVCache(n, h, cap, e, dtype=E4M3, block=64)
    dt.kv_cache_append(cache, k, v, ints([3, 0]))
    ok, ov = ko.Cache(n, h, cap, e, E4M3, 64), ko.Cache(n, h, cap, e, E4M3, 64)
    ok.append(k.cpu(), [3, 0])
    ov.append(v.cpu(), [3, 0])
    same_cache(cache, ok, ov, [40, 37])


@pytest.mark.parametrize("code", [INT8, E4M3])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_non_finite_value_marks_its_block(code, bad):
    gen = torch.Generator().manual_seed(6)
    k, v = tokens(gen, 1, 2, 100, 32, BF16), tokens(gen, 1, 2, 100, 32, BF16)
    k[0, 1, 40, 7] = bad
    v[0, 0, 99, 0] = bad
    cache = dt.QuantizedKVCache(1, 2, 128, 32, dtype=code, block=32)
    dt.kv_cache_append(cache, k.cuda(), v.cuda(), ints([0]))
    ok, ov = ko.Cache(1, 2, 128, 32, code, 32), ko.Cache(1, 2, 128, 32, code, 32)
    ok.append(k, [0])
    ov.append(v, [0])
    more = tokens(gen, 1, 2, 8, 32, BF16) * 3  # the last block stays marked
    dt.kv_cache_append(cache, more.cuda(), more.cuda(), ints([100]))
    ok.append(more, [100])
    ov.append(more, [100])
    same_cache(cache, ok, ov, [108])
    rk, rv = dt.kv_cache_read(cache, ints([108]), dtype=torch.float32)
    assert rk[0, 1, 32:64].isnan().all() and not rk[0, 1, :32].isnan().any() and not rk[0, 0].isnan().any()
    assert rv[0, 0, 96:108].isnan().all() and not rv[0, 0, 108:].any()


def test_extreme_sizes_of_values():
    for dtype, big, small in ((BF16, 3.38e38, 1e-40), (FP16, 65504.0, 6e-8)):
        for code in (INT8, E4M3):
            x = torch.zeros((1, 3, 64, 32), dtype=dtype)
            x[0, 0], x[0, 1, 5, 3] = big, -small
            x[0, 0, :, ::3] = -big / 2
            cache = dt.QuantizedKVCache(1, 3, 64, 32, dtype=code)
            dt.kv_cache_append(cache, x.cuda(), x.cuda(), ints([0]))
            o = ko.Cache(1, 3, 64, 32, code, 64)
            o.append(x, [0])
            same_cache(cache, o, o, [64])


@pytest.mark.parametrize("code,block,e", [(INT8, 64, 128), (E4M3, 32, 48), (INT8, 128, 256)])
def test_read(code, block, e):
    gen = torch.Generator().manual_seed(7)
    lengths = [0, 1, 200, 256]
    cache, ok, ov = filled(gen, lengths, 2, 256, e, code, block)
    for dtype in (torch.float32, BF16, FP16):
        for first, count in ((0, None), (100, 57), (250, 20), (ints([0, 5, 190, 256]), 33), (ints([-3, 0, 1, 2]), None)):
            got = dt.kv_cache_read(cache, ints(lengths), first=first, count=count, dtype=dtype)
            f = [first] * 4 if isinstance(first, int) else first.tolist()
            c = count if count is not None else 256 - first if isinstance(first, int) else 256
            for x, o in zip(got, (ok, ov)):
                want = torch.zeros((4, 2, c, e), dtype=torch.float64)
                for i in range(4):
                    for j in range(c):
                        if 0 <= f[i] + j < lengths[i]:
                            want[i, :, j] = o.values()[i, :, f[i] + j]
                assert torch.equal(x.cpu(), want.to(torch.float32).to(dtype))


def check_attention(cache, ok, ov, lengths, q, counts=None, causal=True, scale=None, weights=True):
    n, h, cap = cache.batch, cache.kv_heads, cache.capacity
    before = torch.rand((n, h, cap), generator=torch.Generator().manual_seed(1)).cuda()
    w = before.clone()
    out, lse = dt.kv_cache_attention(q, cache, ints(lengths), counts=None if counts is None else ints(counts),
                                     is_causal=causal, scale=scale, weights=w if weights else None, return_lse=True)
    eo, el, ew, mag, size = ko.attention(q.cpu().double(), ok.values(), ov.values(), lengths, counts, causal, scale)
    bound = ko.attention_bounds(eo, mag, size, q.dtype)
    off = (out.cpu().double() - eo).abs() - bound
    assert not out.isnan().any() and off.max() <= 0, f"output off by {off.max():g} over its bound"
    empty = torch.isinf(el)
    assert torch.equal(torch.isinf(lse.cpu()), empty) and not lse.isnan().any()
    d = 2.0 ** -19 * size
    off = ((lse.cpu().double() - el).abs() - (d + 2.0 ** -21 * el.abs() + 2.0 ** -20))[~empty]
    assert off.numel() == 0 or off.max() <= 0, f"lse off by {off.max():g} over its bound"
    if weights:
        # a weight's error: the score's and the sum's (2 d), 2^-19 of it; the sum with what was there: fp32's half step
        dmax = d.amax(dim=(1, 2))[:, None, None]
        want = before.cpu().double() + ew
        off = (w.cpu().double() - want).abs() - ((2 * dmax + 2.0 ** -18) * ew + 2.0 ** -23 * want)
        held = torch.arange(cap) < torch.tensor([min(max(l, 0), cap) for l in lengths])[:, None]
        held = held[:, None].expand(n, h, cap)
        assert off[held].numel() == 0 or off[held].max() <= 0, f"weights off by {off[held].max():g} over their bound"
        assert torch.equal(w.cpu()[~held], before.cpu()[~held]), "a slot behind a length was written"
        w2 = before.clone()
        out2 = dt.kv_cache_attention(q, cache, ints(lengths), counts=None if counts is None else ints(counts),
                                     is_causal=causal, scale=scale, weights=w2, accumulate=False)
        assert torch.equal(out2, out)
        # fp32's exponentials flush below 2^-126: at most that much from each of a key head's query rows
        flush = q.shape[1] // h * q.shape[2] * 2.0 ** -126
        off = ((w2.cpu().double() - ew).abs() - (2 * dmax + 2.0 ** -18) * ew - flush)[held]
        assert off.numel() == 0 or off.max() <= 0, f"written weights off by {off.max():g}"
        assert torch.equal(w2.cpu()[~held], before.cpu()[~held])


LENGTHS = [0, 1, 31, 32, 33, 127, 128, 129, 300, 511]


@pytest.mark.parametrize("code", [INT8, E4M3])
@pytest.mark.parametrize("dtype,e,block,h,g,t", [
    (BF16, 128, 64, 2, 8, 1), (FP16, 64, 32, 3, 1, 1), (BF16, 16, 64, 1, 2, 1), (BF16, 80, 128, 2, 3, 2),
    (FP16, 96, 64, 2, 4, 5), (BF16, 256, 64, 1, 2, 1), (FP16, 192, 32, 2, 5, 7), (BF16, 128, 64, 1, 16, 3),
    (BF16, 128, 128, 2, 1, 130), (FP16, 64, 64, 1, 4, 70), (BF16, 48, 32, 2, 4, 40), (FP16, 128, 32, 1, 7, 61)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention(code, dtype, e, block, h, g, t, causal):
    gen = torch.Generator().manual_seed(e + t)
    cache, ok, ov = filled(gen, LENGTHS, h, 512, e, code, block, dtype)
    q = (torch.randn((len(LENGTHS), h * g, t, e), generator=gen) * 1.5).to(dtype).cuda()
    check_attention(cache, ok, ov, LENGTHS, q, causal=causal)


@pytest.mark.parametrize("t", [1, 4, 40])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_of_a_padded_batch(t, causal):
    gen = torch.Generator().manual_seed(t)
    lengths = [5, 200, 64, 0, 300, -7, 9999]
    counts = [0, t, t - 1, t, max(t // 2, 1), 1, t + 50]
    cache, ok, ov = filled(gen, lengths, 2, 384, 64, INT8, 32)
    q = (torch.randn((7, 6, t, 64), generator=gen)).to(FP16).cuda()
    q[0] = math.nan  # a row behind its count is not read as a query
    check_attention(cache, ok, ov, lengths, q, counts=counts, causal=causal)


@pytest.mark.parametrize("layout", ["heads_last", "unaligned", "inner_strided", "broadcast"])
@pytest.mark.parametrize("t", [2, 70])
def test_attention_of_strided_queries(layout, t):
    gen = torch.Generator().manual_seed(11)
    cache, ok, ov = filled(gen, [150, 77], 2, 192, 96, E4M3, 64)
    q = torch.randn((2, 4, t, 96), generator=gen).to(BF16).cuda()
    if layout == "heads_last":
        q = q.transpose(1, 2).contiguous().transpose(1, 2)
    elif layout == "unaligned":
        flat = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")
        flat[1:] = q.reshape(-1)
        q = flat[1:].view(q.shape)
    elif layout == "inner_strided":
        q = torch.stack([q, q], -1)[..., 0]
    else:
        q = q[:, :1].expand(2, 4, t, 96)
    check_attention(cache, ok, ov, [150, 77], q)


@pytest.mark.parametrize("t", [1, 66])
@pytest.mark.parametrize("scale", [0.0, -0.3, 0.05, 2.0])
def test_attention_scales(scale, t):
    gen = torch.Generator().manual_seed(12)
    cache, ok, ov = filled(gen, [150, 3], 2, 192, 64, INT8, 64)
    q = torch.randn((2, 4, t, 64), generator=gen).to(BF16).cuda()
    check_attention(cache, ok, ov, [150, 3], q, scale=scale)


@pytest.mark.parametrize("t", [1, 66])
def test_attention_of_values_of_very_different_size(t):
    # blocks whose scales differ by 2^20, the larger ones with the smaller weights and the other way round
    gen = torch.Generator().manual_seed(13)
    for order in (1, -1):
        n, h, cap, e = 1, 1, 256, 64
        k, v = tokens(gen, n, h, cap, e, BF16), torch.randn((n, h, cap, e), generator=gen).to(BF16)
        for b in range(4):
            v[:, :, b * 64:(b + 1) * 64] *= 2.0 ** (order * (b * 7 - 10))
        cache = dt.QuantizedKVCache(n, h, cap, e, dtype=E4M3, block=64)
        dt.kv_cache_append(cache, k.cuda(), v.cuda(), ints([0]))
        ok, ov = ko.Cache(n, h, cap, e, E4M3, 64), ko.Cache(n, h, cap, e, E4M3, 64)
        ok.append(k, [0])
        ov.append(v, [0])
        q = torch.randn((n, 4, t, e), generator=gen).to(BF16).cuda()
        check_attention(cache, ok, ov, [256], q, causal=False)


@pytest.mark.parametrize("t", [1, 66])
def test_attention_with_a_marked_block(t):
    gen = torch.Generator().manual_seed(14)
    cache, _, _ = filled(gen, [100, 100], 2, 128, 64, E4M3, 32)
    cache.value_scale[0, 1, 1] = math.nan
    cache.key_scale[1, 0, 0] = math.nan
    q = torch.randn((2, 4, t, 64), generator=gen).to(BF16).cuda()
    out, lse = dt.kv_cache_attention(q, cache, ints([100, 100]), is_causal=False, return_lse=True)
    assert out[0, 2:].isnan().all() and not lse[0].isnan().any()  # heads 2 and 3 read key head 1
    assert out[1, :2].isnan().all() and lse[1, :2].isnan().all()
    assert not out[0, :2].isnan().any() and not out[1, 2:].isnan().any()


def test_attention_in_long_caches_and_ragged_batches():
    # oracle on the GPU, in 64 bits: one long sequence among short ones, split over many CTAs
    gen = torch.Generator().manual_seed(15)
    lengths = [20000, 3, 0, 777]
    n, h, g, e, cap = 4, 2, 4, 128, 20032
    cache = dt.QuantizedKVCache(n, h, cap, e, dtype=INT8, block=64)
    k, v = (torch.randn((n, h, cap, e), generator=gen).to(BF16).cuda() for _ in range(2))
    dt.kv_cache_append(cache, k, v, ints([0] * n), counts=ints(lengths))
    kk, vv = (x.double() for x in dt.kv_cache_read(cache, ints(lengths), dtype=torch.float32))
    for t in (1, 3, 33):
        q = torch.randn((n, h * g, t, e), generator=gen).to(FP16).cuda()
        w = torch.zeros((n, h, cap), device="cuda")
        out = dt.kv_cache_attention(q, cache, ints(lengths), weights=w)
        for i, l in enumerate(lengths):
            s = torch.einsum("hgte,hle->hgtl", q[i].double().view(h, g, t, e), kk[i, :, :l]) / math.sqrt(e)
            ban = torch.arange(l, device="cuda") > (l - t + torch.arange(t, device="cuda"))[:, None]
            p = torch.softmax(s.masked_fill(ban, -math.inf), -1).nan_to_num()
            want = torch.einsum("hgtl,hle->hgte", p, vv[i, :, :l]).reshape(h * g, t, e)
            mag = torch.einsum("hgtl,hle->hgte", p, vv[i, :, :l].abs()).reshape(h * g, t, e)
            size = torch.full((h * g, t), 15.0, device="cuda", dtype=torch.float64)  # scale * sum |q k| is about 7
            assert ((out[i].double() - want).abs() <= ko.attention_bounds(want, mag, size, FP16)).all()
            ew = p.sum(dim=(1, 2))
            assert ((w[i, :, :l].double() - ew).abs() <= (2.0 ** -18 + 2 * 15 * 2.0 ** -19) * ew).all()
            assert not w[i, :, l:].any()


@pytest.mark.parametrize("n,h,g,t,lo,hi,cap,e", [
    (40, 3, 4, 9, 1, 40, 64, 64),        # many items of one tile, rows in one of the two row tiles
    (24, 4, 2, 100, 90, 700, 65536, 128),  # short sequences in a large cache, rows in both
    (3, 1, 1, 129, 0, 1000, 1024, 96), (1, 2, 3, 400, 399, 399, 512, 128), (70, 1, 4, 33, 0, 3, 128, 32)])
@pytest.mark.parametrize("causal", [True, False])
def test_many_items_for_a_cta(n, h, g, t, lo, hi, cap, e, causal):
    # oracle on the GPU, in 64 bits
    gen = torch.Generator().manual_seed(n + t)
    lengths = [lo + (hi - lo) * (i * 7 % n) // max(n - 1, 1) for i in range(n)]
    cache = dt.QuantizedKVCache(n, h, cap, e, dtype=E4M3, block=32)
    k, v = (torch.randn((n, h, max(lengths), e), generator=gen).to(BF16).cuda() for _ in range(2))
    dt.kv_cache_append(cache, k, v, ints([0] * n), counts=ints(lengths))
    kk, vv = (x.double() for x in dt.kv_cache_read(cache, ints(lengths), count=max(lengths), dtype=torch.float32))
    q = torch.randn((n, h * g, t, e), generator=gen).to(FP16).cuda()
    w = torch.full((n, h, cap), 7.0, device="cuda")
    out = dt.kv_cache_attention(q, cache, ints(lengths), is_causal=causal, weights=w, accumulate=False)
    pos = torch.arange(max(lengths), device="cuda")
    s = torch.einsum("nhgte,nhle->nhgtl", q.double().view(n, h, g, t, e), kk) / math.sqrt(e)
    lim = ints(lengths)[:, None] - (t - 1 - torch.arange(t, device="cuda") if causal else 0 * torch.arange(t, device="cuda"))
    s = s.masked_fill((pos >= lim[..., None])[:, None, None], -math.inf)
    p = torch.softmax(s, -1).nan_to_num()
    want = torch.einsum("nhgtl,nhle->nhgte", p, vv).reshape(out.shape)
    mag = torch.einsum("nhgtl,nhle->nhgte", p, vv.abs()).reshape(out.shape)
    size = torch.full(out.shape[:3], 25.0, device="cuda", dtype=torch.float64)  # scale * sum |q k| is 4 to 8, and spreads
    assert ((out.double() - want).abs() <= ko.attention_bounds(want, mag, size, FP16)).all()
    ew = p.sum(dim=(2, 3))
    for i, l in enumerate(lengths):
        off = (w[i, :, :l].double() - ew[i, :, :l]).abs() - (2.0 ** -18 + 2 * 25 * 2.0 ** -19) * ew[i, :, :l]
        assert l == 0 or off.max() <= g * t * 2.0 ** -126
        assert (w[i, :, l:] == 7.0).all()


def test_offsets_beyond_32_bits():
    # two heads of 2^24 + 64 tokens of 128 elements: the second head's codes begin behind 2^31 bytes
    cap, e = (1 << 24) + 64, 128
    cache = dt.QuantizedKVCache(1, 2, cap, e, dtype=INT8, block=64)
    gen = torch.Generator().manual_seed(16)
    k, v = tokens(gen, 1, 2, 70, e, BF16), tokens(gen, 1, 2, 70, e, BF16)
    dt.kv_cache_append(cache, k.cuda(), v.cuda(), ints([cap - 70]))
    o = ko.Cache(1, 2, 128, e, INT8, 64)
    ov = ko.Cache(1, 2, 128, e, INT8, 64)
    o.append(k, [128 - 70])
    ov.append(v, [128 - 70])
    rk, rv = dt.kv_cache_read(cache, ints([cap]), first=cap - 128, count=128, dtype=torch.float32)
    assert torch.equal(rk.cpu().double(), o.values()) and torch.equal(rv.cpu().double(), ov.values())
    for t in (1, 70):
        q = (torch.randn((1, 4, t, e), generator=gen)).to(BF16).cuda()
        w = torch.zeros((1, 2, cap), device="cuda")
        out, lse = dt.kv_cache_attention(q, cache, ints([cap]), weights=w, return_lse=True)
        # the tokens before are zero: score 0 and value 0 each
        s = torch.einsum("hgte,hle->hgtl", q.cpu().double().view(2, 2, t, e), o.values()[0, :, 58:]) / math.sqrt(e)
        lim = torch.arange(70) > (70 - t + torch.arange(t))[:, None]
        s = s.masked_fill(lim, -math.inf)
        lead = torch.full(s.shape[:-1] + (1,), math.log(cap - 70.0), dtype=torch.float64)
        p = torch.softmax(torch.cat([lead, s], -1), -1)
        want = torch.einsum("hgtl,hle->hgte", p[..., 1:], ov.values()[0, :, 58:]).reshape(4, t, e)
        mag = torch.einsum("hgtl,hle->hgte", p[..., 1:], ov.values()[0, :, 58:].abs()).reshape(4, t, e)
        size = torch.full((4, t), 60.0, dtype=torch.float64)
        # 2^24 equal weights: fp16 subnormals are not met (weights are 2^10 of the largest), the sum is fp32 in parts
        bound = ko.attention_bounds(want, mag, size, BF16)
        assert ((out[0].cpu().double() - want).abs() <= bound).all()
        ew = p[..., 1:].sum(dim=(1, 2))
        assert ((w[0, :, cap - 70:].cpu().double() - ew).abs() <= (2.0 ** -16 + 120 * 2.0 ** -19) * ew).all()


@pytest.mark.parametrize("t", [1, 90])
def test_attention_is_the_same_bits_again_and_on_another_stream(t):
    gen = torch.Generator().manual_seed(17)
    cache, _, _ = filled(gen, [3000, 11, 513], 2, 3008, 128, INT8, 64)
    q = torch.randn((3, 8, t, 128), generator=gen).to(BF16).cuda()
    lengths = ints([3000, 11, 513])
    runs = []
    for k in range(4):
        s = torch.cuda.Stream() if k % 2 else torch.cuda.current_stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            w = torch.zeros((3, 2, 3008), device="cuda")
            runs.append((dt.kv_cache_attention(q, cache, lengths, weights=w), w))
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for out, w in runs[1:]:
        assert torch.equal(out, runs[0][0]) and torch.equal(w, runs[0][1])


def test_two_calls_at_once():
    gen = torch.Generator().manual_seed(18)
    caches = [filled(gen, [2000, 100], 2, 2048, 128, code, 64)[0] for code in (INT8, E4M3)]
    qs = [torch.randn((2, 8, t, 128), generator=gen).to(BF16).cuda() for t in (1, 3)]
    lengths = ints([2000, 100])
    alone = [dt.kv_cache_attention(q, c, lengths) for q, c in zip(qs, caches)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(dt.kv_cache_attention(qs[i], caches[i], lengths))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, alone[i]) for x in got[i])


def evict_case(gen, lengths, h, cap, e, code, block, budget, recent, weights):
    cache, ok, ov = filled(gen, lengths, h, cap, e, code, block)
    out, l2, w2, kept = dt.kv_cache_evict(cache, ints(lengths), weights.cuda(), budget, recent)
    want = ko.keep(weights, lengths, budget, recent)
    assert torch.equal(kept.cpu(), want)
    assert l2.tolist() == [min(max(l, 0), cap, budget) for l in lengths]
    same_cache(out, ko.evict(ok, want, out.capacity), ko.evict(ov, want, out.capacity), l2.tolist())
    full = torch.nn.functional.pad(want, (0, out.capacity - budget), value=-1)
    ew = torch.where(full >= 0, torch.gather(weights, 2, full.clamp(min=0).long()), torch.zeros(()))
    assert torch.equal(w2.cpu().nan_to_num(-1), ew.nan_to_num(-1))
    # the slots behind the last kept token of its block hold zeros
    for i, l in enumerate(l2.tolist()):
        assert not out.key[i, :, l:-(-l // block) * block].float().any()


@pytest.mark.parametrize("code", [INT8, E4M3])
@pytest.mark.parametrize("budget,recent", [(0, 0), (1, 1), (64, 0), (100, 100), (130, 37), (256, 5), (600, 200)])
def test_evict(code, budget, recent):
    gen = torch.Generator().manual_seed(budget)
    lengths = [0, 1, 64, 129, 500, 576]
    w = torch.randn((6, 2, 576), generator=gen)
    w[3] = 0  # ties
    w[4, 0, 100:300] = 1.0
    evict_case(gen, lengths, 2, 576, 80, code, 64, budget, recent, w)


def test_evict_order_of_odd_weights():
    gen = torch.Generator().manual_seed(1)
    w = torch.randn((3, 1, 2500), generator=gen)
    w[0, 0, ::7] = -0.0
    w[0, 0, 1::7] = 0.0
    w[1, 0, 5:50] = math.nan
    w[1, 0, 60:70] = math.inf
    w[1, 0, 80:2000] = -math.inf
    w[2] = -w[2].abs() * 1e-39  # subnormal
    evict_case(gen, [2500, 2500, 2499], 1, 2560, 16, INT8, 128, 1100, 3, torch.nn.functional.pad(w, (0, 60)))


def test_evict_of_a_marked_block_and_into_a_larger_cache():
    gen = torch.Generator().manual_seed(2)
    cache, ok, ov = filled(gen, [200, 90], 2, 256, 32, INT8, 32)
    cache.key_scale[0, 1, 2] = math.nan
    ok.scale[0, 1, 2] = math.nan
    w = torch.rand((2, 2, 256), generator=gen)
    into = dt.QuantizedKVCache(2, 2, 512, 32, block=32)
    into.key.fill_(9)
    into.key_scale.fill_(7)
    out, l2, w2, kept = dt.kv_cache_evict(cache, ints([200, 90]), w.cuda(), 100, 10, out=into)
    assert out is into and l2.tolist() == [100, 90] and w2.shape == (2, 2, 512) and not w2[0, :, 100:].any()
    want = ko.keep(w, [200, 90], 100, 10)
    assert torch.equal(kept.cpu(), want)
    same_cache(out, ko.evict(ok, want, 512), ko.evict(ov, want, 512), [100, 90])
    assert (into.key[:, :, 128:] == 9).all() and (into.key_scale[:, :, 4:] == 7).all()  # left as they were


def test_a_run_of_them_together():
    """A prompt, two parts of it with weights, a cut to the budget, single tokens, captured and replayed."""
    gen = torch.Generator().manual_seed(19)
    n, h, g, e, block, cap = 2, 2, 4, 64, 32, 320
    cache = dt.QuantizedKVCache(n, h, cap, e, dtype=E4M3, block=block)
    ok, ov = ko.Cache(n, h, cap, e, E4M3, block), ko.Cache(n, h, cap, e, E4M3, block)
    lengths, seen = ints([0, 0]), torch.zeros((n, h, cap), device="cuda")
    held, eseen = [0, 0], torch.zeros((n, h, cap), dtype=torch.float64)

    def step(t, counts=None):
        nonlocal cache, lengths, seen, held, eseen
        k, v = tokens(gen, n, h, t, e, BF16), tokens(gen, n, h, t, e, BF16)
        q = torch.randn((n, h * g, t, e), generator=gen).to(BF16)
        cc = None if counts is None else ints(counts)
        dt.kv_cache_append(cache, k.cuda(), v.cuda(), lengths, counts=cc)
        lengths += t if counts is None else cc
        out = dt.kv_cache_attention(q.cuda(), cache, lengths, counts=cc, weights=seen)
        ok.append(k, held, counts)
        ov.append(v, held, counts)
        held = [l + (t if counts is None else counts[i]) for i, l in enumerate(held)]
        eo, _, ew, mag, size = ko.attention(q.double(), ok.values(), ov.values(), held, counts)
        eseen += ew
        assert ((out.cpu().double() - eo).abs() <= ko.attention_bounds(eo, mag, size, BF16)).all()
        assert ((seen.cpu().double() - eseen).abs() <= 1e-4 * eseen + 1e-9).all()

    step(150, counts=[150, 97])
    step(80)
    step(1)
    cache, lengths, seen, kept = dt.kv_cache_evict(cache, lengths, seen, 128, 32,
                                                   out=dt.QuantizedKVCache(n, h, cap, e, dtype=E4M3, block=block))
    # the oracle follows the same choice: two weights closer than their error may be ordered either way
    want = kept.cpu()
    ok, ov = ko.evict(ok, want, cap), ko.evict(ov, want, cap)
    held = [128, 128]
    eseen = torch.nn.functional.pad(torch.gather(eseen, 2, want.long()), (0, cap - 128))
    same_cache(cache, ok, ov, held)
    step(1)
    step(1)

    # the same step captured: the lengths grow on the device between replays
    k, v = tokens(gen, n, h, 1, e, BF16), tokens(gen, n, h, 1, e, BF16)
    q = torch.randn((n, h * g, 1, e), generator=gen).to(BF16).cuda()
    gk, gv = k.cuda(), v.cuda()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        dt.kv_cache_attention(q, cache, lengths)  # allocations settle before the capture
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dt.kv_cache_append(cache, gk, gv, lengths)
        lengths += 1
        out = dt.kv_cache_attention(q, cache, lengths, weights=seen)
    for i in range(40):
        k, v = tokens(gen, n, h, 1, e, BF16), tokens(gen, n, h, 1, e, BF16)
        gk.copy_(k)
        gv.copy_(v)
        graph.replay()
        ok.append(k, held)
        ov.append(v, held)
        held = [l + 1 for l in held]
        eo, _, ew, mag, size = ko.attention(q.cpu().double(), ok.values(), ov.values(), held)
        assert ((out.cpu().double() - eo).abs() <= ko.attention_bounds(eo, mag, size, BF16)).all(), i
    assert lengths.tolist() == held
    same_cache(cache, ok, ov, held)


def test_nothing_to_do():
    cache = dt.QuantizedKVCache(2, 2, 64, 32)
    lengths = ints([0, 0])
    empty = torch.empty((2, 2, 0, 32), dtype=BF16, device="cuda")
    dt.kv_cache_append(cache, empty, empty, lengths)
    assert dt.kv_cache_attention(empty, cache, lengths).shape == (2, 2, 0, 32)
    assert dt.kv_cache_read(cache, lengths, count=0)[0].shape == (2, 2, 0, 32)
    none = dt.QuantizedKVCache(0, 2, 64, 32)
    q = torch.empty((0, 4, 3, 32), dtype=BF16, device="cuda")
    assert dt.kv_cache_attention(q, none, ints([])).shape == (0, 4, 3, 32)
    w = torch.empty((0, 2, 64), device="cuda")
    assert dt.kv_cache_evict(none, ints([]), w, 10)[3].shape == (0, 2, 10)


@pytest.fixture(params=["same", "peer"])
def mode(request, monkeypatch):
    if request.param == "same":
        monkeypatch.setenv("DTORCH_DTENSOR_IN_SAME_DEVICE", "1")
    else:
        if torch.cuda.device_count() < 2:
            pytest.skip("peer mode needs 2 GPUs")
        monkeypatch.delenv("DTORCH_DTENSOR_IN_SAME_DEVICE", raising=False)
    monkeypatch.setenv("DTORCH_COMM_TIMEOUT_SECOND", "30")
    dt.clear()
    yield request.param
    dt.clear()


@pytest.mark.parametrize("group", [1, 3])
def test_context_parallel_attention_with_a_cache(mode, group):
    """A sequence-sharded prompt, a head-sharded token, an eviction and another token through
    scaled_dot_product_attention_with_cp, against one device's cache."""
    n, h, e, cap = 2, 4, 64, 256
    mesh = dt.init_device_mesh("cuda", (2,), mesh_dim_names=["cp"])
    gen = torch.Generator().manual_seed(23)
    cache = dt.DistributedKVCache(mesh, [dt.Shard(1)], n, h, cap, e, block=32, track_weights=True)
    one = dt.QuantizedKVCache(n, h, cap, e, block=32)
    lengths, seen = ints([0, 0]), torch.zeros((n, h, cap), device="cuda")

    def step(t, place):
        q = torch.randn((n, h * group, t, e), generator=gen).to(BF16)
        k, v = tokens(gen, n, h, t, e, BF16), tokens(gen, n, h, t, e, BF16)
        dq, dk, dv = (dt.DTensor.from_torch(x, mesh, [place]) for x in (q, k, v))
        out = dt.scaled_dot_product_attention_with_cp(dq, dk, dv, is_causal=True, ulysses_cp_dim="cp", kv_cache=cache)
        assert out.placements == [place] and out.shape == q.shape
        nonlocal lengths
        dt.kv_cache_append(one, k.cuda(), v.cuda(), lengths)
        lengths = lengths + t
        want = dt.kv_cache_attention(q.cuda(), one, lengths, weights=seen)
        torch.cuda.synchronize()
        # how the tiles are shared out depends on the number of heads: sums differ in their order
        assert torch.allclose(out.to_torch().float(), want.float().cpu(), rtol=2.0 ** -7, atol=2.0 ** -9)
        for gid in mesh.ids:
            part = seen[:, gid * 2:gid * 2 + 2].cpu()
            assert torch.allclose(cache.weights[gid].cpu(), part, rtol=1e-5, atol=1e-8)

    step(101, dt.Shard(2))
    step(1, dt.Shard(1))
    cache.evict(64, 16)
    assert cache.max_length == 64
    for gid in mesh.ids:
        assert cache.locals[gid].capacity == cap and cache.lengths[gid].tolist() == [64, 64]
    # the same choice on one device: the distributed weights
    w = torch.cat([cache.weights[g].cpu() for g in mesh.ids], 1)
    both = [torch.cat([getattr(cache.locals[g], k).cpu() for g in mesh.ids], 1).cuda()
            for k in ("key", "value", "key_scale", "value_scale")]
    one, lengths, seen = dt.QuantizedKVCache.from_tensors(*both), ints([64, 64]), w.cuda()
    step(1, dt.Shard(1))
    step(6, dt.Shard(2))
    with pytest.raises(ValueError, match="evict"):
        step(250, dt.Shard(1))


def test_two_captured_graphs_side_by_side():
    """A prompt with weights and a token, captured apart and replayed at once and again, with other lengths each time."""
    gen = torch.Generator().manual_seed(31)
    cap, h, g, e = 1024, 2, 4, 128
    made = []
    for t, code in ((96, E4M3), (1, INT8)):
        cache, _, _ = filled(gen, [700, 900], h, cap, e, code, 64)
        cache.key_scale.nan_to_num_(0.01)  # other lengths come to lie on what was junk
        cache.value_scale.nan_to_num_(0.01)
        if code == E4M3:
            cache.key.view(torch.int8)[:, :, 700:] = 3
            cache.value.view(torch.int8)[:, :, 700:] = 5
        q = torch.randn((2, h * g, t, e), generator=gen).to(BF16).cuda()
        lengths, w = ints([700, 900]), torch.zeros((2, h, cap), device="cuda")
        dt.kv_cache_attention(q, cache, lengths, weights=w, accumulate=False)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = dt.kv_cache_attention(q, cache, lengths, weights=w, accumulate=False)
            kept = dt.kv_cache_evict(cache, lengths, w, 128, 16)
        made.append((graph, cache, q, lengths, w, out, kept))
    streams = [torch.cuda.Stream() for _ in made]
    for lens in ([700, 900], [1, 64], [1024, 0], [333, 1000]):
        for m in made:
            m[3].copy_(ints(lens))
        torch.cuda.synchronize()
        for _ in range(3):
            for s, m in zip(streams, made):
                with torch.cuda.stream(s):
                    m[0].replay()
        torch.cuda.synchronize()
        for _, cache, q, lengths, w, out, kept in made:
            w2 = w.clone()
            want = dt.kv_cache_attention(q, cache, lengths, weights=w2, accumulate=False)
            assert torch.equal(out, want) and torch.equal(w, w2)
            want = dt.kv_cache_evict(cache, lengths, w, 128, 16)
            assert torch.equal(kept[1], want[1]) and torch.equal(kept[3], want[3])
            a, b = (dt.kv_cache_read(c[0], c[1], dtype=torch.float32) for c in (kept, want))
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_c_abi_calls():
    """The entry points by pointers, without kept positions and with a workspace, against the Python calls."""
    from dtorch_b200 import capi

    gen = torch.Generator().manual_seed(33)
    n, h, cap, e, t = 2, 2, 256, 64, 40
    cache = dt.QuantizedKVCache(n, h, cap, e, block=32)
    same = dt.QuantizedKVCache(n, h, cap, e, block=32)
    abi = capi.KvCache(cache.key.data_ptr(), cache.value.data_ptr(), cache.key_scale.data_ptr(), cache.value_scale.data_ptr(),
                       n, h, cap, e, 32, capi.DT_KV_INT8)
    k, v = tokens(gen, n, h, 150, e, FP16).cuda(), tokens(gen, n, h, 150, e, FP16).cuda()
    q = torch.randn((n, 4, t, e), generator=gen).to(FP16).cuda()
    zero, lengths = ints([0, 0]), ints([150, 150])
    stream = torch.cuda.current_stream().cuda_stream
    capi.kv_append(abi, k.data_ptr(), v.data_ptr(), 150, k.stride()[:3], v.stride()[:3], capi.DT_FLOAT16, zero.data_ptr(), None,
                   stream)
    dt.kv_cache_append(same, k, v, zero)
    assert torch.equal(cache.key, same.key) and torch.equal(cache.value_scale, same.value_scale)
    out, w = torch.empty_like(q), torch.zeros((n, h, cap), device="cuda")
    nbytes = capi.kv_attention_workspace(abi, 4, t, True)
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    with pytest.raises(capi.DtError, match="workspace"):
        capi.kv_attention(abi, q.data_ptr(), 4, t, q.stride()[:3], capi.DT_FLOAT16, lengths.data_ptr(), None, 0.125,
                          capi.DT_KV_CAUSAL, out.data_ptr(), None, w.data_ptr(), ws.data_ptr(), nbytes - 1, stream)
    capi.kv_attention(abi, q.data_ptr(), 4, t, q.stride()[:3], capi.DT_FLOAT16, lengths.data_ptr(), None, 0.125,
                      capi.DT_KV_CAUSAL, out.data_ptr(), None, w.data_ptr(), ws.data_ptr(), nbytes, stream)
    w2 = torch.zeros_like(w)
    assert torch.equal(out, dt.kv_cache_attention(q, same, lengths, weights=w2)) and torch.equal(w, w2)
    value = torch.empty((n, h, 10, e), device="cuda")
    capi.kv_read(abi, lengths.data_ptr(), None, 145, 10, None, value.data_ptr(), capi.DT_FLOAT32, stream)
    assert torch.equal(value, dt.kv_cache_read(same, lengths, first=145, count=10, dtype=torch.float32)[1])
    into = dt.QuantizedKVCache(n, h, 64, e, block=32)
    abi2 = capi.KvCache(into.key.data_ptr(), into.value.data_ptr(), into.key_scale.data_ptr(), into.value_scale.data_ptr(),
                        n, h, 64, e, 32, capi.DT_KV_INT8)
    l2 = torch.empty_like(lengths)
    ws = torch.empty(capi.kv_evict_workspace(abi, 50), dtype=torch.uint8, device="cuda")
    capi.kv_evict(abi, abi2, lengths.data_ptr(), w.data_ptr(), 50, 7, l2.data_ptr(), None, None, ws.data_ptr(), ws.numel(), stream)
    want = dt.kv_cache_evict(same, lengths, w, 50, 7)
    assert l2.tolist() == [50, 50]
    assert torch.equal(into.key[:, :, :50], want[0].key[:, :, :50]) and torch.equal(into.value_scale, want[0].value_scale)
