"""The operators of the 8-bit key/value cache, as cases to be timed and compared.

The cache holds keys and values in 8 bits (int8 or float8_e4m3fn), layout (N, H_kv, capacity, E), with one float32
scale for each block of `block` consecutive tokens of a head: a value is code * scale. Four operators work on it:

* append: new tokens are written behind those that a sequence holds; a block's scale is the largest
  |value| / limit of its tokens (limit 127 for int8, 448 for e4m3), rounded up to 8 significant bits, and the codes of
  a block that is still filling are rounded again when its scale grows;
* read: tokens as values again, in the model's type;
* attention: T queries of each sequence, its last T tokens, over all tokens that it holds, causal or not, grouped
  heads, with the sum over queries of each cached token's softmax weight where it is asked for;
* evict: the last `recent` tokens and, of the others, those of the largest accumulated weight move to another cache
  that holds `budget` tokens, in order; blocks are scaled anew.

`own` False: elementary torch operations. `own` True: dtorch_b200's operators.
"""

import math

import numpy as np
import torch

own = False

LIMIT = {"int8": 127.0, "e4m3": 448.0}
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TYPE = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _case(name, op, **kw):
    c = {"op": op, "N": 1, "Hq": 8, "Hkv": 8, "E": 128, "T": 1, "lo": 0, "hi": 1024, "code": "int8", "type": "bf16",
         "block": 64, "causal": True, "weights": False, "budget": 0, "recent": 0}
    c.update(kw)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token of each of 32 sequences goes behind what it holds: the write of a decode step
        _case("append_token", "append", N=32, lo=1000, hi=8000, code="e4m3"),
        # two prompts of an odd length enter behind a shared opening that ends inside a block
        _case("append_prompt", "append", N=2, T=8191, lo=37, hi=90),
        # one short conversation, small heads, each with its own key head: latency counts
        _case("attend_token_small", "attend", N=1, Hq=12, Hkv=12, E=64, lo=301, hi=301, block=32),
        # a serving batch of ragged lengths, eight query heads to a key head
        _case("attend_token_batch", "attend", N=32, Hq=64, Hkv=8, lo=1, hi=8192, code="e4m3"),
        # one long document, with the weights that eviction goes by
        _case("attend_token_long", "attend", N=1, Hq=64, Hkv=8, lo=131071, hi=131071, weights=True),
        # a few drafted tokens are verified at once
        _case("attend_draft", "attend", N=8, Hq=32, Hkv=8, T=5, lo=900, hi=6001, code="e4m3", type="fp16", block=128),
        # a part of a long prompt over what came before it
        _case("attend_prompt", "attend", N=1, Hq=32, Hkv=8, T=4096, lo=16384, hi=16384),
        # whole prompts of odd lengths, with the weights that eviction goes by
        _case("attend_prompt_weights", "attend", N=2, Hq=16, Hkv=4, T=2001, lo=1501, hi=2001, code="e4m3",
              type="fp16", weights=True),
        # a decode step as a program runs it: the token is appended, then attends, and weights are kept
        _case("decode_step", "step", N=16, Hq=32, Hkv=8, lo=2000, hi=4095, weights=True),
        # one conversation is cut back to its budget
        _case("evict_small", "evict", N=1, Hkv=8, E=64, lo=700, hi=700, budget=512, recent=64, block=32),
        # a batch of long prompts is cut back before decoding
        _case("evict_batch", "evict", N=8, Hkv=8, lo=3000, hi=32768, budget=4096, recent=511, code="e4m3"),
        # one long document
        _case("evict_long", "evict", N=1, Hkv=8, lo=131072, hi=131072, budget=8192, recent=1024),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "step", "evict"])
    hkv, group, e = rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 64, 128, 128, 128, 96])
    kw = {"Hkv": hkv, "E": e, "code": rng.choice(["int8", "e4m3"]), "type": rng.choice(["bf16", "bf16", "fp16"]),
          "block": rng.choice([32, 64, 64, 128]), "Hq": hkv}
    if op == "append":
        kw["T"] = rng.choice([1, 1, _log(rng, 2, 8000)])
        kw["N"] = _log(rng, 1, max(1, 16000 // kw["T"]) if kw["T"] > 1 else 64)
        kw["lo"] = rng.randrange(0, 1000)
        kw["hi"] = kw["lo"] + rng.randrange(0, 3000)
    elif op in ("attend", "step"):
        kw["Hq"] = hkv * group
        kind = "token" if op == "step" else rng.choice(["token", "token", "draft", "prompt"])
        kw["T"] = 1 if kind == "token" else rng.randrange(2, 20) if kind == "draft" else _log(rng, 64, 3000)
        kw["hi"] = max(kw["T"], _log(rng, 64, 100000 if kind != "prompt" else 12000))
        kw["lo"] = rng.randrange(kw["T"], kw["hi"] + 1) if kind != "prompt" else max(kw["T"], kw["hi"] // 2)
        kw["N"] = _log(rng, 1, max(1, min(48, (200000 if kind != "prompt" else 16000) // kw["hi"])))
        kw["causal"] = rng.random() < 0.8
        kw["weights"] = op == "step" or rng.random() < 0.4
    else:
        kw["hi"] = _log(rng, 300, 100000)
        kw["lo"] = rng.randrange(kw["hi"] // 3, kw["hi"] + 1)
        kw["N"] = _log(rng, 1, max(1, min(16, 250000 // kw["hi"])))
        kw["budget"] = _log(rng, 64, max(65, kw["hi"] // 2))
        kw["recent"] = rng.randrange(0, kw["budget"] + 1)
    return _case(None, op, **kw)


def _lengths(c):
    """The tokens that each sequence holds, spread evenly from lo to hi in a fixed order that is not sorted. With
    appended tokens: before them for op append, with them otherwise."""
    n = c["N"]
    return [c["hi"] if n == 1 else c["lo"] + (c["hi"] - c["lo"]) * ((i * 7 + n // 2) % n) // (n - 1) for i in range(n)]


def _capacity(c):
    most = c["hi"] + (c["T"] if c["op"] == "append" else 0)
    return -(-most // c["block"]) * c["block"]


def _read_count(c):
    return c["T"] + c["block"] - 1  # the appended tokens and the others of the block that was filling


# -- the definition in elementary operations ---------------------------------------------------------------------


def _round_up(s):
    """Up to 8 significant bits: the next bfloat16 that is not below."""
    return ((s.view(torch.int32) + 0xFFFF) & -65536).view(torch.float32)


def _scale_of(amax, code):
    amax = amax.float()
    # a true division: torch multiplies by the reciprocal where the divisor is a number, which is off next to a border
    return _round_up(amax / torch.full_like(amax, LIMIT[code]))


def _encode(x, scale, code):
    """x / scale in 8 bits; x float32, scale float32 broadcast over it (0: all of it is 0)."""
    y = x / torch.where(scale > 0, scale, torch.ones_like(scale))
    if code == "int8":
        return torch.round(y).clamp(-127, 127).to(torch.int8)
    return y.clamp(-448, 448).to(torch.float8_e4m3fn)


def _values(codes, scale):
    """float32 values of (N, H, L, E) codes with (N, H, L / block) scales; L a multiple of block."""
    n, h, l, e = codes.shape
    nb = scale.shape[2]
    return (codes.float().view(n, h, nb, l // nb, e) * scale[..., None, None]).view(n, h, l, e)


def _quantize(x, block, code):
    """(codes, scales) of whole blocks of float32 (N, H, L, E)."""
    n, h, l, e = x.shape
    xb = x.view(n, h, l // block, block, e)
    s = _scale_of(xb.abs().amax(dim=(3, 4)), code)
    return _encode(xb, s[..., None, None], code).view(n, h, l, e), s


def _append(codes, scale, new, start, c):
    """Writes `new` (N, H, T, E) at `start` (N,) into codes / scale, in place."""
    n, h, t, e = new.shape
    block = c["block"]
    first = start // block * block  # the block that is filling
    span = -(-(t + block - 1) // block) * block
    pos = first[:, None] + torch.arange(span, device=new.device)  # (N, span)
    held = pos < start[:, None]
    fresh = (pos >= start[:, None]) & (pos < start[:, None] + t)
    inside = pos < codes.shape[2]
    at = pos.clamp(max=codes.shape[2] - 1).long()[:, None, :, None].expand(n, h, span, e)
    blk = at[:, :, ::block, 0] // block  # (N, H, span / block)
    old_scale = torch.where(held[:, None, ::block], torch.gather(scale, 2, blk), torch.zeros_like(scale[:, :1, :1]))
    raw = codes.view(torch.int8)
    there = torch.gather(raw, 2, at)
    old = there.view(codes.dtype).float().view(n, h, -1, block, e) * old_scale[..., None, None]
    take = (pos - start[:, None]).clamp(0, t - 1).long()[:, None, :, None].expand(n, h, span, e)
    x = torch.gather(new.float(), 2, take)
    x = torch.where(fresh[:, None, :, None], x, torch.zeros_like(x)).view(n, h, -1, block, e)
    s = torch.maximum(old_scale, _scale_of(x.abs().amax(dim=(3, 4)), c["code"]))
    x = torch.where(held.view(n, 1, -1, block, 1), old, x)
    y = _encode(x, s[..., None, None], c["code"]).view(n, h, span, e).view(torch.int8)
    keep = (held | fresh)[:, None, :, None]
    # slots outside the cache, and those that hold nothing, keep what they have
    y = torch.where(keep & inside[:, None, :, None], y, there)
    ok = inside.nonzero(as_tuple=True)
    raw[ok[0], :, pos[ok].long()] = y[ok[0], :, ok[1]]
    touched = (fresh & inside).view(n, -1, block).any(dim=2).nonzero(as_tuple=True)
    scale[touched[0], :, blk[:, 0][touched]] = s[touched[0], :, touched[1]]


def _read(codes, scale, lengths, first, count, c):
    n, h, cap, e = codes.shape
    pos = first[:, None] + torch.arange(count, device=codes.device)
    at = pos.clamp(max=cap - 1).long()[:, None, :].expand(n, h, count)
    x = torch.gather(codes.view(torch.int8), 2, at[..., None].expand(n, h, count, e)).view(codes.dtype).float()
    x = x * torch.gather(scale, 2, at // c["block"])[..., None]
    return torch.where((pos < lengths[:, None])[:, None, :, None], x, torch.zeros_like(x)).to(TYPE[c["type"]])


def _attend(q, kc, ks, vc, vs, lengths, c):
    n, hq, t, e = q.shape
    hkv, cap = kc.shape[1], kc.shape[2]
    g = hq // hkv
    pos = torch.arange(cap, device=q.device)
    held = pos < lengths[:, None]  # (N, L)
    k = _values(kc, ks).masked_fill(~held[:, None, :, None], 0.0)
    v = _values(vc, vs).masked_fill(~held[:, None, :, None], 0.0)
    s = torch.matmul(q.float().reshape(n, hkv, g * t, e), k.transpose(2, 3)).view(n, hkv, g, t, cap)
    s = s * (1.0 / math.sqrt(e))
    last = lengths[:, None] - (t - 1 if c["causal"] else 0) + torch.arange(t, device=q.device) * int(c["causal"])
    s = s.masked_fill(~(pos < last[:, :, None])[:, None, None], -math.inf)
    m = s.amax(dim=-1, keepdim=True)
    p = torch.exp(s - m.clamp(min=-3e38))
    l = p.sum(dim=-1, keepdim=True)
    p = p / torch.where(l > 0, l, torch.ones_like(l))
    out = torch.matmul(p.view(n, hkv, g * t, cap), v).view(n, hq, t, e).to(q.dtype)
    lse = (m + torch.log(l)).view(n, hq, t)
    return {"out": out, "lse": lse, **({"weights": p.sum(dim=(2, 3))} if c["weights"] else {})}


def _evict(codes, scale, kept, c):
    """The kept tokens (N, H, budget rounded up to blocks; -1: none) of one of keys or values, scaled anew."""
    n, h, cap, e = codes.shape
    at = kept.clamp(min=0).long()
    x = torch.gather(codes.view(torch.int8), 2, at[..., None].expand(*at.shape, e)).view(codes.dtype).float()
    x = x * torch.gather(scale, 2, at // c["block"])[..., None]
    return _quantize(torch.where((kept >= 0)[..., None], x, torch.zeros_like(x)), c["block"], c["code"])


def _keep(weights, lengths, c):
    """(N, H, budget) positions that stay, ascending, -1 behind the last."""
    n, h, cap = weights.shape
    budget, recent = c["budget"], c["recent"]
    pos = torch.arange(cap, device=weights.device)
    held = (pos < lengths[:, None])[:, None]
    late = held & (pos >= (lengths[:, None] - recent))[:, None]
    rank = torch.where(late, math.inf, torch.where(held, weights, -math.inf))
    order = torch.sort(rank, dim=2, descending=True, stable=True).indices[:, :, :budget]
    kept = torch.sort(torch.where(torch.gather(held.expand(n, h, cap), 2, order), order, cap), dim=2).values
    return torch.nn.functional.pad(torch.where(kept < cap, kept, -1), (0, budget - kept.shape[2]), value=-1).int()


# -- what perf calls ---------------------------------------------------------------------------------------------


def _tokens(c, gen, length):
    """Keys or values as a model makes them: channels of different size, and a few tokens much larger."""
    shape = (c["N"], c["Hkv"], length, c["E"])
    x = torch.randn(shape, generator=gen, device="cuda")
    x *= torch.exp(0.5 * torch.randn((1, c["Hkv"], 1, c["E"]), generator=gen, device="cuda"))
    return x * (1 + 3 * (torch.rand((c["N"], c["Hkv"], length, 1), generator=gen, device="cuda") > 0.98))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    c = dict(case)
    dt, cap = TYPE[c["type"]], _capacity(c)
    lengths = torch.tensor(_lengths(c), dtype=torch.int32, device="cuda")
    st = {"case": c, "lengths": lengths}
    held = lengths - c["T"] if c["op"] == "step" else lengths
    for name in ("k", "v"):
        x = _tokens(c, gen, cap).to(dt).float()
        x = torch.where((torch.arange(cap, device="cuda") < held[:, None])[:, None, :, None], x, torch.zeros_like(x))
        st[name], st[name + "s"] = _quantize(x, c["block"], c["code"])
        del x
    if c["op"] in ("append", "step"):
        st["new_k"], st["new_v"] = (_tokens(c, gen, c["T"]).to(dt) for _ in range(2))
        st["held"] = held
        st["after"] = held + c["T"]
        st["first"] = held // c["block"] * c["block"]
    if c["op"] in ("attend", "step"):
        q = torch.randn((c["N"], c["Hq"], c["T"], c["E"]), generator=gen, device="cuda")
        st["q"] = (q * 1.5).to(dt)
        st["w"] = torch.zeros((c["N"], c["Hkv"], cap), device="cuda")
    if c["op"] == "evict":
        # weights as attention leaves them: most are small, a few carry the mass, some were never seen
        w = torch.exp(2 * torch.randn((c["N"], c["Hkv"], cap), generator=gen, device="cuda"))
        st["w"] = w * (torch.rand(w.shape, generator=gen, device="cuda") > 0.05)
    if own:  # the handles that a program keeps: they hold the tensors above, and nothing that is computed
        import dtorch_b200 as dt2

        st["cache"] = dt2.QuantizedKVCache.from_tensors(st["k"], st["v"], st["ks"], st["vs"])
        if c["op"] == "evict":
            most = -(-c["budget"] // c["block"]) * c["block"]
            st["into"] = dt2.QuantizedKVCache(c["N"], c["Hkv"], most, c["E"], dtype=CODE[c["code"]], block=c["block"],
                                              device="cuda")
    return st


def _run_own(st):
    import dtorch_b200 as dt2

    c, cache, got = st["case"], st["cache"], {}
    if c["op"] in ("append", "step"):
        dt2.kv_cache_append(cache, st["new_k"], st["new_v"], st["held"])
        got["key"], got["value"] = dt2.kv_cache_read(cache, st["after"], first=st["first"], count=_read_count(c),
                                                     dtype=TYPE[c["type"]])
        got["key_scale"], got["value_scale"] = cache.key_scale, cache.value_scale
    if c["op"] in ("attend", "step"):
        w = st["w"] if c["weights"] else None
        got["out"], got["lse"] = dt2.kv_cache_attention(st["q"], cache, st["lengths"], is_causal=c["causal"],
                                                        weights=w, accumulate=False, return_lse=True)
        if w is not None:
            got["weights"] = w
    if c["op"] == "evict":
        into, lengths, weights, kept = dt2.kv_cache_evict(cache, st["lengths"], st["w"], c["budget"], c["recent"],
                                                          out=st["into"])
        got["key"], got["value"] = dt2.kv_cache_read(into, lengths, dtype=TYPE[c["type"]])
        got.update(key_scale=into.key_scale, value_scale=into.value_scale, lengths=lengths, weights=weights, kept=kept)
    return got


def run(st):
    if own:
        return _run_own(st)
    c, got = st["case"], {}
    if c["op"] in ("append", "step"):
        _append(st["k"], st["ks"], st["new_k"], st["held"], c)
        _append(st["v"], st["vs"], st["new_v"], st["held"], c)
        got["key"] = _read(st["k"], st["ks"], st["after"], st["first"], _read_count(c), c)
        got["value"] = _read(st["v"], st["vs"], st["after"], st["first"], _read_count(c), c)
        got["key_scale"], got["value_scale"] = st["ks"], st["vs"]
    if c["op"] in ("attend", "step"):
        got.update(_attend(st["q"], st["k"], st["ks"], st["v"], st["vs"], st["lengths"], c))
    if c["op"] == "evict":
        kept = _keep(st["w"], st["lengths"], c)
        got["kept"], got["lengths"] = kept, st["lengths"].clamp(max=c["budget"])
        most = -(-c["budget"] // c["block"]) * c["block"]
        full = torch.nn.functional.pad(kept, (0, most - c["budget"]), value=-1)
        got["weights"] = torch.where(full >= 0, torch.gather(st["w"], 2, full.clamp(min=0).long()), 0.0)
        zero = torch.zeros_like(st["lengths"])
        for name, k in (("key", "k"), ("value", "v")):
            codes, scale = _evict(st[k], st[k + "s"], full, c)
            got[name] = _read(codes, scale, got["lengths"], zero, most, c)
            got[name + "_scale"] = scale
    return got


def work(case):
    c = case
    n, hq, hkv, e, t = c["N"], c["Hq"], c["Hkv"], c["E"], c["T"]
    lens = _lengths(c)
    flops = bytes_ = 0
    if c["op"] in ("append", "step"):
        bytes_ += 2 * n * hkv * e * (t * (2 + 1) + _read_count(c) * (1 + 2))  # K and V: in, codes out; codes in, out
        flops += 2 * n * hkv * e * (3 * t + _read_count(c))
    if c["op"] in ("attend", "step"):
        pairs = sum(l * t - (t * (t - 1) // 2 if c["causal"] else 0) for l in lens)
        bytes_ += 2 * sum(lens) * hkv * (e + 4 / c["block"]) + n * hq * t * (4 * e + 4)
        bytes_ += 4 * sum(lens) * hkv * int(c["weights"])
        flops += 4 * hq * e * pairs
    if c["op"] == "evict":
        kept = sum(min(l, c["budget"]) for l in lens)
        bytes_ += 4 * sum(lens) * hkv + kept * hkv * (4 + 4 + 2 * e * (1 + 1)) + 2 * n * c["budget"] * hkv * e * (1 + 2)
        flops += 6 * kept * hkv * e
    return {"bytes": bytes_, "flops": flops}


# -- the same from the definition, in 64 bits ---------------------------------------------------------------------


def _exact_scale(amax, code):
    """amax / limit up to 8 significant bits, in float64."""
    s = amax / torch.full_like(amax, LIMIT[code])
    mant, ex = torch.frexp(s)
    return torch.ldexp(torch.ceil(mant * 256) / 256, ex)


def _exact_code(x, s, code):
    """x / s to the nearest code (ties to even), both float64, as float64."""
    y = torch.where(s > 0, x / s.clamp(min=1e-300), torch.zeros_like(x))
    if code == "int8":
        return torch.round(y)
    ex = torch.frexp(y.abs().clamp(min=2.0 ** -6)).exponent - 1  # normal numbers begin at 2^-6, 3 bits behind the point
    step = torch.ldexp(torch.ones_like(y), ex - 3)
    return torch.round(y / step) * step


def _exact_tokens(codes, scale, length, block):
    """float64 values of the first `length` tokens of one head."""
    s = scale.double().repeat_interleave(block)[:length, None]
    return codes[:length].double() * s if codes.dtype == torch.int8 else codes[:length].float().double() * s


def exact(case, seed):
    global own
    before, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = before
    c = st["case"]
    lens, blk, code = st["lengths"].tolist(), c["block"], c["code"]
    dt, got = TYPE[c["type"]], {}
    n, hkv = c["N"], c["Hkv"]
    vals = {}  # (name, sequence, head): float64 values of what the cache holds at the end
    if c["op"] in ("append", "step"):
        span = _read_count(c)
        for name, k in (("key", "k"), ("value", "v")):
            scales = st[k + "s"].double().clone()
            out = torch.zeros((n, hkv, span, c["E"]), dtype=torch.float64, device="cuda")
            for i, held in enumerate(st["held"].tolist()):
                first = held // blk * blk
                x = torch.zeros((hkv, span, c["E"]), dtype=torch.float64, device="cuda")
                x[:, held - first:held - first + c["T"]] = st["new_" + k][i].double()
                old = st[k][i, :, first:held].float().double() * scales[i, :, first // blk:first // blk + 1, None] \
                    if held > first else x[:, :0]
                for b in range(0, held - first + c["T"], blk):
                    part = x[:, b:b + blk]
                    s = _exact_scale(part.abs().amax(dim=(1, 2)), code)
                    if b == 0 and held > first:
                        s = torch.maximum(s, scales[i, :, first // blk])
                        part = torch.cat([old, part[:, held - first:]], 1)
                    out[i, :, b:b + blk] = _exact_code(part, s[:, None, None], code) * s[:, None, None]
                    scales[i, :, (first + b) // blk] = s
                out[i, :, held - first + c["T"]:] = 0
                if c["op"] == "step":
                    for h in range(hkv):
                        v = _exact_tokens(st[k][i, h], st[k + "s"][i, h], first, blk)
                        vals[k, i, h] = torch.cat([v, out[i, h, :held - first + c["T"]]])
            got[name], got[name + "_scale"] = out, scales
    if c["op"] in ("attend", "step"):
        t, g = c["T"], c["Hq"] // hkv
        if 4.0 * c["Hq"] * c["E"] * t * sum(lens) > 2e13:
            return None
        out = torch.zeros((n, c["Hq"], t, c["E"]), dtype=torch.float64, device="cuda")
        lse = torch.full((n, c["Hq"], t), -math.inf, dtype=torch.float64, device="cuda")
        wts = torch.zeros(st["w"].shape, dtype=torch.float64, device="cuda")
        for i, l in enumerate(lens):
            for h in range(hkv):
                k, v = (vals[x, i, h] if c["op"] == "step" else _exact_tokens(st[x][i, h], st[x + "s"][i, h], l, blk)
                        for x in ("k", "v"))
                for j in range(g * h, g * h + g):
                    s = st["q"][i, j].double() @ k.T / math.sqrt(c["E"])
                    if c["causal"]:
                        ban = torch.arange(l, device="cuda")[None] > (l - t + torch.arange(t, device="cuda"))[:, None]
                        s = s.masked_fill(ban, -math.inf)
                    lse[i, j] = torch.logsumexp(s, 1)
                    p = torch.softmax(s, 1).nan_to_num()  # queries before the sequence's first token see nothing
                    out[i, j] = p @ v
                    wts[i, h, :l] += p.sum(0)
        got.update({"out": out, "lse": lse, **({"weights": wts} if c["weights"] else {})})
    if c["op"] == "evict":
        budget, recent = c["budget"], c["recent"]
        most = -(-budget // blk) * blk
        kept = np.full((n, hkv, budget), -1, dtype=np.int32)
        weights = st["w"].cpu().numpy()
        for i, l in enumerate(lens):
            for h in range(hkv):
                old = max(0, l - recent)
                take = np.argsort(-weights[i, h, :old], kind="stable")[:max(0, budget - min(recent, l))]
                pos = np.concatenate([np.sort(take), np.arange(old, l)])
                kept[i, h, :len(pos)] = pos
        full = np.pad(kept, ((0, 0), (0, 0), (0, most - budget)), constant_values=-1)
        got["kept"] = kept
        got["lengths"] = np.minimum(np.array(lens, dtype=np.int32), budget)
        got["weights"] = np.where(full >= 0, np.take_along_axis(weights, np.maximum(full, 0), 2), 0.0).astype(np.float64)
        for name, k in (("key", "k"), ("value", "v")):
            x = torch.zeros((n, hkv, most, c["E"]), dtype=torch.float64, device="cuda")
            for i in range(n):
                for h in range(hkv):
                    at = torch.from_numpy(full[i, h][full[i, h] >= 0]).long().to("cuda")
                    x[i, h, :len(at)] = _exact_tokens(st[k][i, h], st[k + "s"][i, h], st[k].shape[2], blk)[at]
            xb = x.view(n, hkv, -1, blk, c["E"])
            s = _exact_scale(xb.abs().amax(dim=(3, 4)), code)
            got[name] = (_exact_code(xb, s[..., None, None], code) * s[..., None, None]).view(x.shape)
            got[name + "_scale"] = s
    return {k: v.cpu().numpy() if isinstance(v, torch.Tensor) else v for k, v in got.items()}
