"""CPU: what the 8-bit key/value cache refuses, before any CUDA call, through the Python API and the C ABI."""

import ctypes
import math

import pytest
import torch

import dtorch_b200 as dt
from dtorch_b200 import capi
from tests import kv_oracle as ko

BF16 = torch.bfloat16


def cache(n=2, h=2, cap=128, e=64, **kw):
    return dt.QuantizedKVCache(n, h, cap, e, device="cpu", **kw)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def rows(n=2, h=2, t=3, e=64, dtype=BF16):
    return torch.zeros((n, h, t, e), dtype=dtype)


@pytest.mark.parametrize("kw", [dict(cap=100), dict(cap=0), dict(e=24), dict(e=272), dict(e=0), dict(block=16), dict(block=48),
                                dict(h=0)])
def test_caches_that_cannot_be(kw):
    with pytest.raises(ValueError):
        cache(**kw)


def test_cache_types_and_tensors():
    with pytest.raises(TypeError):
        cache(dtype=torch.float16)
    c = cache(dtype=torch.float8_e4m3fn, block=32)
    assert (c.batch, c.kv_heads, c.capacity, c.head_dim, c.block) == (2, 2, 128, 64, 32)
    again = dt.QuantizedKVCache.from_tensors(c.key, c.value, c.key_scale, c.value_scale)
    assert again.block == 32 and again.key.data_ptr() == c.key.data_ptr()
    with pytest.raises(ValueError):
        dt.QuantizedKVCache.from_tensors(c.key, c.value[:, :1], c.key_scale, c.value_scale)
    with pytest.raises(ValueError):
        dt.QuantizedKVCache.from_tensors(c.key, c.value, c.key_scale[:, :, :3], c.value_scale[:, :, :3])
    with pytest.raises(ValueError):
        dt.QuantizedKVCache.from_tensors(c.key.transpose(0, 1), c.value.transpose(0, 1), c.key_scale, c.value_scale)
    with pytest.raises(TypeError):
        dt.QuantizedKVCache.from_tensors(c.key.float(), c.value.float(), c.key_scale, c.value_scale)


def test_append_refuses():
    c, l = cache(), ints(0, 0)
    for k, v in ((rows(h=1), rows(h=1)), (rows(e=32), rows(e=32)), (rows(n=1), rows(n=1)), (rows(), rows(t=2)),
                 (rows()[0], rows()[0])):
        with pytest.raises(ValueError):
            dt.kv_cache_append(c, k, v, l)
    with pytest.raises(TypeError):
        dt.kv_cache_append(c, rows(dtype=torch.float32), rows(dtype=torch.float32), l)
    with pytest.raises(TypeError):
        dt.kv_cache_append(c, rows(), rows(dtype=torch.float16), l)
    for bad in (ints(0), torch.zeros(2, dtype=torch.int64), ints(0, 0, 0, 0)[::2]):
        with pytest.raises(ValueError):
            dt.kv_cache_append(c, rows(), rows(), bad)
        with pytest.raises(ValueError):
            dt.kv_cache_append(c, rows(), rows(), l, counts=bad)
    with pytest.raises(RuntimeError, match="backward"):
        dt.kv_cache_append(c, rows().requires_grad_(), rows(), l)
    with pytest.raises(ValueError, match="cuda"):  # everything else is right
        dt.kv_cache_append(c, rows(), rows(), l)


def test_attention_refuses():
    c, l = cache(), ints(0, 0)
    for q in (rows(h=3), rows(h=0), rows(e=32), rows(n=3), rows()[0]):
        with pytest.raises(ValueError):
            dt.kv_cache_attention(q, c, l)
    with pytest.raises(TypeError):
        dt.kv_cache_attention(rows(dtype=torch.float32), c, l)
    for w in (torch.zeros((2, 2, 64)), torch.zeros((2, 4, 128)), torch.zeros((2, 2, 128), dtype=torch.float64),
              torch.zeros((2, 2, 256))[..., ::2]):
        with pytest.raises(ValueError):
            dt.kv_cache_attention(rows(h=4), c, l, weights=w)
    with pytest.raises(RuntimeError, match="backward"):
        dt.kv_cache_attention(rows(h=4).requires_grad_(), c, l)
    with pytest.raises(ValueError, match="cuda"):
        dt.kv_cache_attention(rows(h=4), c, l)


def test_read_and_evict_refuse():
    c, l, w = cache(), ints(0, 0), torch.zeros((2, 2, 128))
    with pytest.raises(ValueError):
        dt.kv_cache_read(c, l, first=-1)
    with pytest.raises(ValueError):
        dt.kv_cache_read(c, l, count=-1)
    with pytest.raises(TypeError):
        dt.kv_cache_read(c, l, dtype=torch.float64)
    for budget, recent in ((-1, 0), (129, 0), (64, 65), (64, -1)):
        with pytest.raises(ValueError):
            dt.kv_cache_evict(c, l, w, budget, recent, out=cache())
    with pytest.raises(ValueError):
        dt.kv_cache_evict(c, l, w[:, :, :64], 64)
    with pytest.raises(ValueError, match="cuda"):
        dt.kv_cache_evict(c, l, w, 64, 8)


def abi(**kw):
    c = dict(key=4096, value=8192, key_scale=4096, value_scale=4096, batch=1, kv_heads=2, capacity=64, head_dim=32,
             block=32, code=capi.DT_KV_INT8)
    c.update(kw)
    return capi.KvCache(**c)


@pytest.mark.parametrize("kw", [dict(code=2), dict(block=8), dict(head_dim=20), dict(head_dim=512), dict(capacity=65),
                                dict(batch=-1), dict(kv_heads=0), dict(key=None), dict(value_scale=None), dict(key=4100),
                                dict(capacity=1 << 31), dict(capacity=0)])
def test_c_abi_refuses_caches(kw):
    L, c, ptr = capi.lib(), abi(**kw), 4096
    s = capi.i64_array([1, 1, 1])
    n = ctypes.c_size_t()
    r = ctypes.byref(c)
    assert L.dt_kv_append(r, ptr, ptr, 1, s, s, capi.DT_BFLOAT16, ptr, None, None) == capi.DT_ERR_INVALID
    assert L.dt_kv_read(r, ptr, None, 0, 1, ptr, ptr, capi.DT_BFLOAT16, None) == capi.DT_ERR_INVALID
    assert L.dt_kv_attention(r, ptr, 2, 1, s, capi.DT_BFLOAT16, ptr, None, 1.0, 0, ptr, None, None, ptr, 1 << 30,
                             None) == capi.DT_ERR_INVALID
    assert L.dt_kv_attention_workspace(r, 2, 1, 0, ctypes.byref(n)) == capi.DT_ERR_INVALID
    assert L.dt_kv_evict_workspace(r, 1, ctypes.byref(n)) == capi.DT_ERR_INVALID
    assert L.dt_kv_evict(r, ctypes.byref(abi()), ptr, ptr, 1, 0, ptr, ptr, ptr, None, 0, None) == capi.DT_ERR_INVALID
    assert L.dt_last_error_message()


def test_c_abi_refuses_arguments():
    L, c, ptr = capi.lib(), abi(), 4096
    r, s = ctypes.byref(c), capi.i64_array([1, 1, 1])
    bad = capi.DT_ERR_INVALID
    assert L.dt_kv_append(None, ptr, ptr, 1, s, s, capi.DT_BFLOAT16, ptr, None, None) == bad
    assert L.dt_kv_append(r, ptr, ptr, 1, s, s, capi.DT_FLOAT32, ptr, None, None) == bad
    assert L.dt_kv_append(r, ptr, ptr, -1, s, s, capi.DT_BFLOAT16, ptr, None, None) == bad
    assert L.dt_kv_append(r, None, ptr, 1, s, s, capi.DT_BFLOAT16, ptr, None, None) == bad
    assert L.dt_kv_append(r, ptr, ptr, 1, s, None, capi.DT_BFLOAT16, ptr, None, None) == bad
    assert L.dt_kv_append(r, ptr, ptr, 0, s, s, capi.DT_BFLOAT16, ptr, None, None) == capi.DT_OK  # nothing to do
    assert L.dt_kv_read(r, ptr, None, 0, 1, ptr, ptr, 7, None) == bad
    assert L.dt_kv_read(r, None, None, 0, 1, ptr, ptr, capi.DT_BFLOAT16, None) == bad
    assert L.dt_kv_read(r, ptr, None, 0, 1, ptr + 2, ptr, capi.DT_BFLOAT16, None) == bad

    def attend(q=ptr, heads=2, t=1, dtype=capi.DT_BFLOAT16, scale=1.0, flags=0, out=ptr):
        return L.dt_kv_attention(r, q, heads, t, s, dtype, ptr, None, scale, flags, out, None, None, ptr, 1 << 30, None)

    assert attend(q=None) == bad and attend(heads=3) == bad and attend(heads=0) == bad and attend(t=-1) == bad
    assert attend(dtype=capi.DT_FLOAT32) == bad and attend(scale=math.inf) == bad and attend(scale=math.nan) == bad
    assert attend(flags=4) == bad and attend(out=None) == bad and attend(out=ptr + 2) == bad
    assert attend(t=0) == capi.DT_OK

    def evict(dst, budget=8, recent=0, kept=4096, lengths=1 << 20, dst_lengths=1 << 21, w=1 << 22, dst_w=1 << 23):
        return L.dt_kv_evict(r, ctypes.byref(dst), lengths, w, budget, recent, dst_lengths, dst_w, kept, None, 0, None)

    far = dict(key=1 << 24, value=1 << 25, key_scale=1 << 26, value_scale=1 << 27)
    assert evict(abi()) == bad and b"overlap" in L.dt_last_error_message()
    assert evict(abi(**far, head_dim=64)) == bad and evict(abi(**far, code=1)) == bad and evict(abi(**far, batch=2)) == bad
    assert evict(abi(**far), budget=65) == bad and evict(abi(**far), recent=9) == bad
    assert evict(abi(**far), kept=None) == bad and b"workspace" in L.dt_last_error_message()
    assert evict(abi(**far), dst_lengths=1 << 20) == bad and evict(abi(**far), dst_w=1 << 22) == bad


def test_oracle_rounds_as_torch_does():
    # the oracle's e4m3 codes against torch's cast, its scales against bfloat16's neighbours
    y = torch.cat([torch.linspace(-448, 448, 4001), torch.linspace(-0.02, 0.02, 401)]).double()
    assert torch.equal(ko.round_code(y, torch.float8_e4m3fn), y.float().to(torch.float8_e4m3fn).double())
    a = torch.rand(1000, generator=torch.Generator().manual_seed(0)).to(BF16).double() + 2.0 ** -8
    for dtype in (torch.int8, torch.float8_e4m3fn):
        s = ko.scale_of(a, dtype)
        assert torch.equal(s, s.to(BF16).double()) and (s * ko.LIMIT[dtype] >= a).all()
        assert (s * ko.LIMIT[dtype] <= a * (1 + 2.0 ** -7)).all()


def test_distributed_cache_refuses():
    mesh = dt.init_device_mesh("cuda", (2,))
    for placements, shape in (([dt.Shard(2)], (2, 2)), ([dt.Shard(3)], (2, 2)), ([dt.Partial()], (2, 2)),
                              ([dt.Shard(1, 3)], (2, 4)), ([dt.Shard(1)], (2, 3)), ([dt.Shard(0)], (3, 2))):
        with pytest.raises(ValueError):
            dt.DistributedKVCache(mesh, placements, shape[0], shape[1], 64, 32)


def test_attention_with_cp_refuses_what_the_cache_does_not_serve():
    mesh = dt.init_device_mesh("cuda", (2,))
    x = dt.DTensor({0: rows(h=2), 1: rows(h=2)}, mesh, [dt.Shard(1)], (2, 4, 3, 64))
    s0 = dt.DTensor({0: rows(n=1), 1: rows(n=1)}, mesh, [dt.Shard(0)], (2, 2, 3, 64))
    odd = dt.DTensor({0: rows(h=2), 1: rows(h=1)}, mesh, [dt.Shard(1)], (2, 3, 3, 64))
    fake = object()  # never reached
    for kw in (dict(dropout_p=0.1), dict(ring_cp_dim=0), dict(ulysses_overlap_groups=2)):
        with pytest.raises(ValueError, match="kv_cache"):
            dt.scaled_dot_product_attention_with_cp(x, x, x, kv_cache=fake, **{"ulysses_cp_dim": 0, **kw})
    with pytest.raises(ValueError, match="Shard"):
        dt.scaled_dot_product_attention_with_cp(s0, s0, s0, kv_cache=fake, ulysses_cp_dim=0)
    with pytest.raises(ValueError, match="divided"):
        dt.scaled_dot_product_attention_with_cp(odd, odd, odd, kv_cache=fake, ulysses_cp_dim=0)


def test_a_step_on_a_mesh_is_refused_before_it_begins():
    mesh = dt.init_device_mesh("cuda", (2,))
    c = object.__new__(dt.DistributedKVCache)  # on CPU tensors: nothing behind the checks can run
    c.device_mesh, c.placements, c.shape, c.max_length = mesh, [dt.Shard(1)], (2, 4, 64, 64), 60
    c.locals = {g: cache(cap=64) for g in mesh.ids}
    c.lengths, c.weights = {g: ints(60, 60) for g in mesh.ids}, {}

    def made(n=2, h=4, t=3, e=64, dtype=BF16, last=None, place=1):
        local = {g: rows(n, h // 2, t, e, dtype) if place == 1 else rows(n, h, t // 2, e, dtype) for g in mesh.ids}
        local[mesh.ids[-1]] = local[mesh.ids[-1]].to(last or dtype)
        return dt.DTensor(local, mesh, [dt.Shard(place)], (n, h, t, e))

    def step(q, k, v, **kw):
        return dt.scaled_dot_product_attention_with_cp(q, k, v, is_causal=True, ulysses_cp_dim=0, kv_cache=c, **kw)

    grad = made()
    grad.local(mesh.ids[-1]).requires_grad_()
    wrong = made()
    wrong._locals[mesh.ids[0]] = rows(2, 2, 2, 64)
    for error, q, k, v, kw in (
            (ValueError, made(h=6), made(), made(), {}), (ValueError, made(e=32), made(), made(), {}),
            (ValueError, made(n=4), made(), made(), {}), (TypeError, made(dtype=torch.float32), made(), made(), {}),
            (TypeError, made(last=torch.float32), made(), made(), {}), (RuntimeError, grad, made(), made(), {}),
            (ValueError, wrong, made(), made(), {}), (ValueError, made(), wrong, made(), {}),
            (TypeError, made(), made(), made(last=torch.float16), {}), (RuntimeError, made(), made(), grad, {}),
            (ValueError, made(), made(t=5), made(t=5), {}), (ValueError, made(), made(h=8), made(h=8), {}),
            (ValueError, made(), made(), made(t=2), {}), (ValueError, made(), made(), made(), dict(scale=math.inf)),
            (ValueError, made(), made(), made(), dict(scale=1e39)), (TypeError, made(), made(), made(), dict(scale="1")),
            (ValueError, made(h=6, t=4, place=2), made(t=4, place=2), made(t=4, place=2), {}),
            (TypeError, made(t=4, place=2), made(t=4, place=2), made(t=4, place=2, last=torch.float32), {})):
        with pytest.raises(error) as e:
            step(q, k, v, **kw)
        assert "served on cuda" not in str(e.value)
        assert c.max_length == 60 and all(l.tolist() == [60, 60] for l in c.lengths.values())
    with pytest.raises(ValueError, match="cuda"):  # everything is right
        step(made(h=8), made(), made())
    assert c.max_length == 60


def test_no_forward_mode_derivatives():
    import torch.autograd.forward_ad as fwd

    c, l = cache(), ints(0, 0)
    with fwd.dual_level():
        x = fwd.make_dual(rows(), torch.ones_like(rows()))
        q = fwd.make_dual(rows(h=4), torch.ones_like(rows(h=4)))
        for call in (lambda: dt.kv_cache_append(c, x, rows(), l), lambda: dt.kv_cache_append(c, rows(), x, l),
                     lambda: dt.kv_cache_attention(q, c, l)):
            with pytest.raises(RuntimeError, match="derivative"):
                call()
        with torch.no_grad(), pytest.raises(ValueError, match="cuda"):  # values alone are asked for
            dt.kv_cache_append(c, fwd.unpack_dual(x).primal, rows(), l)
