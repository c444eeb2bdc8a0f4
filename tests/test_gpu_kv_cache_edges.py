"""GPU: attention over the 8-bit key/value cache where masks, marked blocks, large scores and block scales far apart
meet, and calls that are refused as a whole."""

import math

import pytest
import torch

import dtorch_b200 as dt
from tests import kv_oracle as ko
from tests.test_gpu_kv_cache import BF16, E4M3, FP16, INT8, check_attention, evict_case, filled, ints, tokens

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def appended(k, v, cap, code, block):
    """A cache that holds k and v (N, H, cap, E) whole, and its oracle."""
    n, h, _, e = k.shape
    cache = dt.QuantizedKVCache(n, h, cap, e, dtype=code, block=block)
    dt.kv_cache_append(cache, k.cuda(), v.cuda(), ints([0] * n))
    ok, ov = ko.Cache(n, h, cap, e, code, block), ko.Cache(n, h, cap, e, code, block)
    ok.append(k, [0] * n)
    ov.append(v, [0] * n)
    return cache, ok, ov


def check_with_nan(cache, ok, ov, lengths, q, counts, causal):
    """As check_attention, for oracles that hold NaN: NaN where the oracle has one and nowhere else."""
    w = torch.zeros((cache.batch, cache.kv_heads, cache.capacity), device="cuda")
    out, lse = dt.kv_cache_attention(q, cache, ints(lengths), counts=None if counts is None else ints(counts),
                                     is_causal=causal, weights=w, return_lse=True)
    eo, el, ew, mag, size = ko.attention(q.cpu().double(), ok.values(), ov.values(), lengths, counts, causal)
    out, lse, w = out.cpu().double(), lse.cpu().double(), w.cpu().double()
    assert torch.equal(out.isnan(), eo.isnan()), "outputs that are NaN"
    good = ~eo.isnan()
    assert ((out - eo).abs() <= ko.attention_bounds(eo, mag, size, q.dtype))[good].all()
    assert torch.equal(lse.isnan(), el.isnan()), "log-sum-exps that are NaN"
    good = ~el.isnan() & ~el.isinf()
    assert torch.equal(lse.isinf(), el.isinf())
    assert ((lse - el).abs() <= 2.0 ** -19 * size + 2.0 ** -21 * el.abs() + 2.0 ** -20)[good].all()
    assert torch.equal(w.isnan(), ew.isnan()), "weights that are NaN"
    good = ~ew.isnan()
    dmax = size.nan_to_num().amax()
    assert ((w - ew).abs() <= (2 * 2.0 ** -19 * dmax + 2.0 ** -18) * ew + 2.0 ** -100)[good].all()


@pytest.mark.parametrize("which", ["value", "key"])
@pytest.mark.parametrize("code,e,g,t", [(E4M3, 64, 2, 1), (INT8, 128, 2, 5), (INT8, 128, 1, 24), (E4M3, 128, 2, 66),
                                        (INT8, 64, 1, 66), (INT8, 256, 1, 5), (E4M3, 192, 1, 40)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("padded", [False, True])
def test_a_marked_block_reaches_only_queries_that_see_it(which, code, e, g, t, causal, padded):
    # blocks of 32; in sequence i block i is marked: in front of all queries' limits, across them, behind the first ones,
    # behind some of the padded batch's
    gen = torch.Generator().manual_seed(t + e)
    lengths = [70, 96, 100, 130, 158, 160, 161, 200]
    marked = [0, 2, 3, 4, 4, 4, 5, 4]
    counts = [t, 0, t, max(t // 2, 1), t, 1, t - 1, t] if padded else None
    cache, ok, ov = filled(gen, lengths, 2, 224, e, code, 32)
    for i, b in enumerate(marked):
        (cache.value_scale if which == "value" else cache.key_scale)[i, 1, b] = math.nan
        (ov if which == "value" else ok).scale[i, 1, b] = math.nan
    q = torch.randn((len(lengths), 2 * g, t, e), generator=gen).to(BF16).cuda()
    check_with_nan(cache, ok, ov, lengths, q, counts, causal)


@pytest.mark.parametrize("t", [8, 70])
def test_a_marked_block_in_a_sequence_that_many_ctas_share(t):
    # the last block is marked; most queries end before it, and their parts come from many CTAs
    gen = torch.Generator().manual_seed(t)
    l = 6000 - 6000 % 32 + 2
    cache, ok, ov = filled(gen, [l], 1, 6016, 64, INT8, 32)
    cache.value_scale[0, 0, l // 32] = math.nan
    ov.scale[0, 0, l // 32] = math.nan
    q = torch.randn((1, 2, t, 64), generator=gen).to(BF16).cuda()
    check_with_nan(cache, ok, ov, [l], q, None, True)
    assert dt.kv_cache_attention(q, cache, ints([l])).isnan().any(-1).sum() == 2 * 2


@pytest.mark.parametrize("t", [1, 12, 66])
@pytest.mark.parametrize("size", [3000.0, -3000.0, 6000.0, -6000.0, 10000.0, -10000.0, 50000.0])
@pytest.mark.parametrize("code,e", [(INT8, 64), (E4M3, 128)])
def test_attention_of_large_scores(t, size, code, e):
    # Scores of one size and sign in all tokens, apart by up to about 8: the products of one channel are nearly all of
    # a score, so sum |q k| is little above |score| and the bound stays tight enough to tell (2^-18 of the size: 4 % of
    # a weight at 10000). Every query has another size, so that the largest score is anywhere between two bfloat16.
    gen = torch.Generator().manual_seed(int(abs(size)) + t)
    n, h, cap = 2, 1, 320
    k = torch.zeros((n, h, cap, e))
    k[..., 0] = 1.0
    k[..., 1:9] = (torch.rand((n, h, cap, 8), generator=gen) - 0.5) * 2
    v = torch.randn((n, h, cap, e), generator=gen)
    cache, ok, ov = appended(k.to(BF16), v.to(BF16), cap, code, 64)
    q = torch.zeros((n, 2, t, e))
    q[..., 0] = size * (1 + torch.rand((n, 2, t), generator=gen))
    q[..., 1:9] = torch.randn((n, 2, t, 8), generator=gen)
    check_attention(cache, ok, ov, [cap, 300], q.to(BF16).cuda(), scale=1.0)


@pytest.mark.parametrize("t", [3, 66])
@pytest.mark.parametrize("power", [24, 30, 36, 100])
@pytest.mark.parametrize("code,e", [(INT8, 64), (E4M3, 128)])
def test_values_far_larger_behind_a_querys_limit(t, power, code, e):
    # the last block's values are 2^power larger than the others; only the last query sees one token of it
    gen = torch.Generator().manual_seed(power)
    n, h, cap = 2, 1, 416
    k, v = torch.randn((n, h, cap, e), generator=gen), torch.randn((n, h, cap, e), generator=gen)
    v[:, :, 384:] *= 2.0 ** power
    cache, ok, ov = appended(k.to(BF16), v.to(BF16), cap, code, 32)
    q = torch.randn((n, 2, t, e), generator=gen).to(BF16).cuda()
    check_attention(cache, ok, ov, [385, 400], q)


@pytest.mark.parametrize("t", [1, 12, 66])
@pytest.mark.parametrize("down,up", [(20, 18), (40, 30), (60, 60), (90, 85), (100, 90)])
@pytest.mark.parametrize("where", ["other_tile", "same_tile"])
@pytest.mark.parametrize("code,e", [(INT8, 64), (E4M3, 128)])
def test_small_weights_of_large_values(t, down, up, where, code, e):
    # one block has weights of about 2^-down and values 2^up larger: its part of the output is 2^(up - down) of the others'
    gen = torch.Generator().manual_seed(down)
    n, h, cap = 1, 1, 512
    k, v = torch.randn((n, h, cap, e), generator=gen) * 0.25, torch.randn((n, h, cap, e), generator=gen)
    b = 64 if where == "same_tile" else 256
    k[..., 0] = 1.0
    k[:, :, b:b + 32, 0] = -1.0
    v[:, :, b:b + 32] *= 2.0 ** up
    # a part of a tile that holds nothing but the small weights must not set the others' scale, nor the other way round
    k[:, :, 480:, 0] = -1.0
    cache, ok, ov = appended(k.to(BF16), v.to(BF16), cap, code, 32)
    q = torch.randn((n, 2, t, e), generator=gen) * 0.2
    q[..., 0] = down * math.log(2) / 2
    check_attention(cache, ok, ov, [cap], q.to(BF16).cuda(), causal=False, scale=1.0)


@pytest.mark.parametrize("t", [1, 9])
@pytest.mark.parametrize("down,up", [(40, 38), (100, 98)])
@pytest.mark.parametrize("code,e", [(INT8, 64), (E4M3, 128), (INT8, 256)])
def test_small_weights_of_large_values_behind_others_in_a_stretch(t, down, up, code, e):
    # as many tiles as make a CTA take several of a sequence: the same tokens of each tile, block by block, share a state
    gen = torch.Generator().manual_seed(down + t)
    n, cap = 160, 512
    k, v = torch.randn((n, 1, cap, e), generator=gen) * 0.25, torch.randn((n, 1, cap, e), generator=gen)
    k[..., 0] = 1.0
    for b in (128, 384 + 32):
        k[:, :, b:b + 32, 0] = -1.0
        v[:, :, b:b + 32] *= 2.0 ** up
    cache, ok, ov = appended(k.to(BF16), v.to(BF16), cap, code, 32)
    q = torch.randn((n, 2, t, e), generator=gen) * 0.2
    q[..., 0] = down * math.log(2) / 2
    check_attention(cache, ok, ov, [cap] * n, q.to(BF16).cuda(), causal=False, scale=1.0)


@pytest.mark.parametrize("t", [1, 12, 66])
@pytest.mark.parametrize("code,e", [(INT8, 64), (E4M3, 128)])
def test_the_largest_scores_on_values_of_zero(t, code, e):
    # a first block that takes nearly all of the weight and holds zeros: the output is the others', 2^-60 of their size
    gen = torch.Generator().manual_seed(5)
    n, h, cap = 1, 1, 256
    k, v = torch.randn((n, h, cap, e), generator=gen) * 0.25, torch.randn((n, h, cap, e), generator=gen) * 2.0 ** 60
    k[..., 0] = -1.0
    k[:, :, :32, 0] = 1.0
    v[:, :, :32] = 0
    cache, ok, ov = appended(k.to(BF16), v.to(BF16), cap, code, 32)
    q = torch.randn((n, 2, t, e), generator=gen) * 0.2
    q[..., 0] = 60 * math.log(2) / 2
    check_attention(cache, ok, ov, [cap], q.to(BF16).cuda(), causal=False, scale=1.0)


@pytest.mark.parametrize("e,t", [(64, 1), (128, 9), (64, 40), (256, 3)])
@pytest.mark.parametrize("bad_value", [math.inf, -math.inf, math.nan])
def test_queries_of_infinities(e, t, bad_value):
    # all scores of a query are +infinity, or all -infinity: its softmax is not defined, and says so; others are not touched
    gen = torch.Generator().manual_seed(e + t)
    k, v = torch.rand((2, 1, 96, e), generator=gen) + 0.5, torch.randn((2, 1, 96, e), generator=gen)
    cache, ok, ov = appended(k.to(BF16), v.to(BF16), 96, INT8, 32)
    q = torch.randn((2, 2, t, e), generator=gen).to(BF16)
    q[0, 1, t // 2] = 0
    q[0, 1, t // 2, 3] = bad_value
    w = torch.zeros((2, 1, 96), device="cuda")
    # the second sequence holds nothing that its queries see
    out, lse = dt.kv_cache_attention(q.cuda(), cache, ints([90, 0]), is_causal=False, weights=w, return_lse=True)
    bad = torch.zeros((2, 2, t), dtype=torch.bool)
    bad[0, 1, t // 2] = True
    assert torch.equal(out.cpu().isnan().all(-1), bad) and torch.equal(out.cpu().isnan().any(-1), bad)
    assert w[0, 0, :90].isnan().all() and not w[0, 0, 90:].any() and not w[1].any()
    assert not out[1].any() and (lse[1] == -math.inf).all() and lse.cpu()[0][~bad[0]].isfinite().all()
    q[0, 1, t // 2] = 0
    check_attention(cache, ok, ov, [90, 0], q.cuda(), causal=False)


@pytest.mark.parametrize("e", [64, 256])
def test_weights_of_no_queries(e):
    cache = dt.QuantizedKVCache(3, 2, 96, e, block=32)
    none = torch.empty((3, 4, 0, e), dtype=BF16, device="cuda")
    w = torch.full((3, 2, 96), 7.0, device="cuda")
    dt.kv_cache_attention(none, cache, ints([0, 5, 200]), weights=w)
    assert (w == 7).all()
    dt.kv_cache_attention(none, cache, ints([0, 5, 200]), weights=w, accumulate=False)
    assert (w[0] == 7).all() and not w[1, :, :5].any() and (w[1, :, 5:] == 7).all() and not w[2].any()


@pytest.fixture
def mesh(monkeypatch):
    monkeypatch.setenv("DTORCH_DTENSOR_IN_SAME_DEVICE", "1")
    monkeypatch.setenv("DTORCH_COMM_TIMEOUT_SECOND", "30")
    dt.clear()
    yield dt.init_device_mesh("cuda", (2,), mesh_dim_names=["cp"])
    dt.clear()


def untouched(cache, length):
    torch.cuda.synchronize()
    return cache.max_length == length and all(l.tolist() == [length] * 2 for l in cache.lengths.values())


@pytest.mark.parametrize("place", [1, 2])
def test_a_refused_step_leaves_the_distributed_cache_as_it_was(mesh, place):
    n, h, e, cap = 2, 4, 64, 128
    place = dt.Shard(place)
    gen = torch.Generator().manual_seed(3)
    cache = dt.DistributedKVCache(mesh, [dt.Shard(1)], n, h, cap, e, block=32, track_weights=True)

    def made(heads=h, dtype=BF16, e=e, n=n):
        return dt.DTensor.from_torch(torch.randn((n, heads, 6, e), generator=gen).to(dtype), mesh, [place])

    def step(q, k, v, **kw):
        return dt.scaled_dot_product_attention_with_cp(q, k, v, is_causal=True, ulysses_cp_dim="cp", kv_cache=cache, **kw)

    k, v = made(), made()
    step(made(), k, v)
    assert untouched(cache, 6)
    grad = made()
    for t in grad.locals.values():
        t.requires_grad_()
    refused = [(ValueError, made(heads=6), {}), (ValueError, made(e=32), {}), (ValueError, made(n=4), {}),
               (TypeError, made(dtype=torch.float32), {}), (ValueError, made(), dict(scale=math.inf)),
               (ValueError, made(), dict(scale=math.nan)), (TypeError, made(), dict(scale="a quarter")),
               (RuntimeError, grad, {})]
    before = {g: c.key.clone() for g, c in cache.locals.items()}
    for error, q, kw in refused:
        with pytest.raises(error):
            step(q, k, v, **kw)
        assert untouched(cache, 6)
    for bad in (made(dtype=torch.float32), made(dtype=FP16)):
        with pytest.raises(TypeError):
            step(made(), k, bad)
        assert untouched(cache, 6)
    assert all(torch.equal(c.key.view(torch.int8), before[g].view(torch.int8)) for g, c in cache.locals.items())
    step(made(heads=8), k, v)  # the retry, with two query heads a key head
    assert untouched(cache, 12)


def test_append_checks_every_device_before_the_first_write(mesh):
    n, h, e = 2, 4, 64
    cache = dt.DistributedKVCache(mesh, [dt.Shard(1)], n, h, 128, e, block=32)
    k = dt.DTensor.from_torch(torch.ones((n, h, 6, e), dtype=BF16), mesh, [dt.Shard(1)])
    last = max(mesh.ids)
    odd = {g: k.local(g).float() if g == last else k.local(g) for g in mesh.ids}
    odd = dt.DTensor(odd, mesh, [dt.Shard(1)], (n, h, 6, e))
    with pytest.raises(TypeError):
        cache.append(k, odd)
    assert untouched(cache, 0) and not any(c.key.any() or c.value.any() for c in cache.locals.values())
    cache.append(k, k)
    assert untouched(cache, 6)


def test_the_tracked_weights_are_float32_under_another_default_type(mesh):
    torch.set_default_dtype(BF16)
    try:
        cache = dt.DistributedKVCache(mesh, [dt.Shard(1)], 2, 4, 128, 64, block=32, track_weights=True)
        x = dt.DTensor.from_torch(torch.ones((2, 4, 40, 64), dtype=BF16), mesh, [dt.Shard(1)])
        dt.scaled_dot_product_attention_with_cp(x, x, x, is_causal=True, ulysses_cp_dim="cp", kv_cache=cache)
        cache.evict(16, 4)
        assert all(w.dtype == torch.float32 for w in cache.weights.values()) and untouched(cache, 16)
    finally:
        torch.set_default_dtype(torch.float32)


@pytest.mark.parametrize("code", [INT8, E4M3])
@pytest.mark.parametrize("block", [32, 64, 128])
@pytest.mark.parametrize("e", range(16, 257, 16))
def test_evict_of_every_head_size_and_block(code, block, e):
    # 128 tokens of 192 elements: keys and values together are 48 KB, to which the kernel's own shared memory comes
    gen = torch.Generator().manual_seed(e)
    evict_case(gen, [300, 70], 1, 384, e, code, block, 150, 20, torch.randn((2, 1, 384), generator=gen))


@pytest.mark.parametrize("t", [1, 66])
def test_captured_behind_copies_fills_and_joined_streams(t):
    """A graph whose calls follow a memory fill, a copy and the join of two streams with calls of their own, replayed with
    other lengths, queries and caches."""
    gen = torch.Generator().manual_seed(41)
    cap, h, g, e = 512, 2, 2, 128
    caches = [filled(gen, [300, 511], h, cap, e, code, 64)[0] for code in (INT8, E4M3)]
    for c in caches:
        for s in (c.key_scale, c.value_scale):
            s.nan_to_num_(0.01)
        c.key.view(torch.int8)[:, :, 300:] = 3
        c.value.view(torch.int8)[:, :, 300:] = 5
    new_q = torch.randn((2, h * g, t, e), generator=gen).to(BF16).cuda()
    q, lengths = torch.empty_like(new_q), ints([300, 511])
    w = [torch.ones((2, h, cap), device="cuda") for _ in caches]
    side = torch.cuda.Stream()

    def calls():
        main = torch.cuda.current_stream()
        q.copy_(new_q)
        for x in w:
            x.zero_()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            a = dt.kv_cache_attention(q, caches[0], lengths, weights=w[0])
        b = dt.kv_cache_attention(q, caches[1], lengths, weights=w[1])
        main.wait_stream(side)
        both = w[0] + w[1]
        side.wait_stream(main)
        with torch.cuda.stream(side):
            first = dt.kv_cache_evict(caches[0], lengths, both, 128, 16)
        second = dt.kv_cache_evict(caches[1], lengths, both, 100, 0)
        main.wait_stream(side)
        k = dt.kv_cache_read(second[0], second[1], count=100, dtype=torch.float32)[0]
        dt.kv_cache_append(first[0], k[:, :, :20].to(BF16), k[:, :, 20:40].to(BF16), first[1] - 20)
        return a, b, both, first[3], second[3], k, *dt.kv_cache_read(first[0], first[1], dtype=torch.float32)

    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = calls()
    for lens in ([300, 511], [0, 130], [512, 64], [150, 151]):
        lengths.copy_(ints(lens))
        new_q.copy_(torch.randn(new_q.shape, generator=gen).to(BF16))
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        kept = [x.clone() for x in got]
        for x, y in zip(kept, calls()):
            torch.cuda.synchronize()
            assert torch.equal(x, y)


@pytest.mark.parametrize("shape,places", [((2,), [dt.Shard(0)]), ((2,), [dt.Replicate()]),
                                          ((2, 2), [dt.Shard(0), dt.Shard(1)]), ((2, 2), [dt.Shard(1), dt.Replicate()])])
def test_other_placements_of_a_distributed_cache(monkeypatch, shape, places):
    monkeypatch.setenv("DTORCH_DTENSOR_IN_SAME_DEVICE", "1")
    dt.clear()
    mesh = dt.init_device_mesh("cuda", shape)
    gen = torch.Generator().manual_seed(7)
    n, h, e, cap = 4, 4, 64, 128
    cache = dt.DistributedKVCache(mesh, places, n, h, cap, e, block=32, track_weights=True)
    one = dt.QuantizedKVCache(n, h, cap, e, block=32)
    lengths, seen = ints([0] * n), torch.zeros((n, h, cap), device="cuda")
    for t in (70, 1, 9):
        q, k, v = (tokens(gen, n, heads, t, e, BF16) for heads in (2 * h, h, h))
        out = dt.scaled_dot_product_attention_with_cp(*(dt.DTensor.from_torch(x, mesh, places) for x in (q, k, v)),
                                                      is_causal=True, kv_cache=cache)
        dt.kv_cache_append(one, k.cuda(), v.cuda(), lengths)
        lengths += t
        want = dt.kv_cache_attention(q.cuda(), one, lengths, weights=seen)
        torch.cuda.synchronize()
        # the tiles are shared out by the numbers of sequences and heads: sums differ in their order
        assert torch.allclose(out.to_torch().float(), want.float().cpu(), rtol=2.0 ** -7, atol=2.0 ** -9)
    full = dt.DTensor(cache.weights, mesh, places, (n, h, cap)).to_torch()
    assert torch.allclose(full.cpu(), seen.cpu(), rtol=1e-5, atol=1e-8)
    for g in mesh.ids:
        assert cache.lengths[g].tolist() == [80] * cache.locals[g].batch
    codes = dt.DTensor({g: c.key for g, c in cache.locals.items()}, mesh, places, (n, h, cap, e)).to_torch()
    assert torch.equal(codes.cpu(), one.key.cpu())
    cache.evict(32, 8)
    assert cache.max_length == 32 and all((l == 32).all() for l in cache.lengths.values())
    dt.clear()


def test_a_captured_step_of_a_distributed_cache(mesh):
    gen = torch.Generator().manual_seed(9)
    n, h, e, cap = 2, 4, 64, 128
    place = [dt.Shard(1)]
    cache = dt.DistributedKVCache(mesh, place, n, h, cap, e, block=32, track_weights=True)
    one = dt.QuantizedKVCache(n, h, cap, e, block=32)
    lengths, seen = ints([0] * n), torch.zeros((n, h, cap), device="cuda")
    new = [dt.DTensor.from_torch(torch.zeros((n, heads, 1, e), dtype=BF16), mesh, place) for heads in (2 * h, h, h)]

    def step():
        return dt.scaled_dot_product_attention_with_cp(*new, is_causal=True, ulysses_cp_dim="cp", kv_cache=cache)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            cache.evict(16)
    with torch.cuda.graph(graph):
        out = step()
    assert cache.max_length == 2  # the second of them by the first replay
    for l in cache.lengths.values():
        l.zero_()
    for w in cache.weights.values():
        w.zero_()
    for i in range(40):
        x = [tokens(gen, n, heads, 1, e, BF16) for heads in (2 * h, h, h)]
        for t, y in zip(new, x):
            for g in mesh.ids:
                t.local(g).copy_(y[:, g * y.shape[1] // 2:(g + 1) * y.shape[1] // 2])
        graph.replay()
        dt.kv_cache_append(one, x[1].cuda(), x[2].cuda(), lengths)
        lengths += 1
        want = dt.kv_cache_attention(x[0].cuda(), one, lengths, weights=seen)
        torch.cuda.synchronize()
        assert torch.allclose(out.to_torch().float(), want.float().cpu(), rtol=2.0 ** -7, atol=2.0 ** -9), i
    cache.max_length = 40
    cache.evict(16, 4)
    assert untouched(cache, 16)


@pytest.mark.parametrize("code,e,g,t", [(INT8, 64, 8, 4096), (E4M3, 128, 1, 20001), (INT8, 256, 8, 4096), (E4M3, 192, 3, 5003)])
def test_weights_of_many_equal_rows(code, e, g, t):
    # Scores of 0: every row gives every token the same weight, whose sum over up to 32768 rows is known. Adding n equal
    # numbers one after another in fp32 is off by up to n 2^-26 of the sum (each addition by half a step of what there is).
    # 64 rows, or 32 pairs of rows, at a time and then 128 of those: 2^-18 of the sum, as for few rows.
    lengths = [43, 1, 96]
    cache, _, _ = filled(torch.Generator().manual_seed(1), lengths, 1, 96, e, code, 32)
    q = torch.zeros((3, g, t, e), dtype=BF16, device="cuda")
    w = torch.zeros((3, 1, 96), device="cuda")
    dt.kv_cache_attention(q, cache, ints(lengths), is_causal=False, weights=w)
    for i, l in enumerate(lengths):
        want = g * t / l
        assert ((w[i, 0, :l].double() - want).abs() <= 2.0 ** -18 * want).all() and not w[i, 0, l:].any()


def test_weights_of_many_equal_rows_over_many_tokens():
    # As above where a CTA has all rows of its tokens. To the rows' sum comes that of the tokens' weights, 157 tiles one
    # after another, and the log-sum-exp, rounded to 2^-21 at log2(20000): 2^-18 + 2^-18 + 2^-20 of a weight.
    l, rows = 20000, 8 * 4096
    cache, _, _ = filled(torch.Generator().manual_seed(1), [l], 1, 20032, 64, INT8, 64)
    w = torch.zeros((1, 1, 20032), device="cuda")
    dt.kv_cache_attention(torch.zeros((1, 8, 4096, 64), dtype=BF16, device="cuda"), cache, ints([l]), is_causal=False,
                          weights=w)
    assert ((w[0, 0, :l].double() - rows / l).abs() <= (2.0 ** -17 + 2.0 ** -20) * rows / l).all() and not w[0, 0, l:].any()
