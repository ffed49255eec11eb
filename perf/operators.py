"""Cases of the operators that make a KV cache smaller: a cache held in 4 bits (its rows written and read back, decode
attention and prompt attention over it) and a cache of a bounded number of rows (the attention weight that each row
has drawn, and the eviction of the rows that drew least).

``run`` computes a case either with elementary torch operations in float32 (``own`` false) or with the calls a user
makes of ``glake_amd._custom_ops`` (``own`` true); ``exact`` gives the same outputs from the definitions in float64.

A 4-bit row of ``kv_heads`` heads of ``head`` values: head / 2 bytes of codes per head (value 2i in the low half of
byte i), then per head a bfloat16 scale and a bfloat16 zero, padded to 16 bytes; a value is code * scale + zero."""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------------------ cases
def _case(name, kind, **kw):
    base = {"name": name, "kind": kind, "type": "bf16", "heads": 32, "kv_heads": 8, "head": 128}
    base.update(kw)
    return base


def listed():
    return [
        # one decode step's new rows of 64 sequences, one layer: a launch's latency
        _case("write_step", "write", seqs=64, lo=1, hi=1),
        # the rows of eight prompts of up to 2048 tokens
        _case("write_prompts", "write", seqs=8, lo=1900, hi=2048),
        # a single request with a short context: the smallest decode call
        _case("decode_single", "decode", seqs=1, lo=777, hi=777, alibi=False),
        # the batch of the benchmark's c2: 64 sequences of 512 to 4096 rows
        _case("decode_batch", "decode", seqs=64, lo=512, hi=4096, alibi=False),
        # the batch of the benchmark's c3: four long sequences, work split along the rows
        _case("decode_long", "decode", seqs=4, lo=32768, hi=131072, alibi=False),
        # one kv head per query head, a head size that is no power of two, fp16, ALiBi, odd lengths
        _case("decode_mha", "decode", seqs=17, lo=3, hi=2501, heads=32, kv_heads=32, head=80, type="fp16", alibi=True),
        # eight prompts, each attending to itself
        _case("prompt_whole", "prompt", seqs=8, qlo=2048, qhi=2048, lo=0, hi=0, alibi=False),
        # chunks of prompts behind prefixes that are cached already
        _case("prompt_chunk", "prompt", seqs=4, qlo=301, qhi=700, lo=2000, hi=7200, heads=64, alibi=False),
        # the attention weight of one decode step added to its rows, 16-bit cache, the batch of c2
        _case("weights_batch", "weights", seqs=64, lo=512, hi=4096, cache="auto"),
        # the same over a 4-bit cache, with a larger group of query heads and longer sequences
        _case("weights_int4", "weights", seqs=24, lo=1024, hi=8192, heads=64, cache="int4"),
        # full caches give up one row per head for the next token
        _case("evict_step", "evict", seqs=64, lo=2049, hi=2049, keep=2048, recent=256),
        # caches that have grown to twice their budget are cut back to it
        _case("evict_half", "evict", seqs=32, lo=3001, hi=4096, keep=2048, recent=512),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "decode", "decode", "prompt", "weights", "evict"])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 8, 16])
    group = rng.choice([1, 2, 3, 4, 7, 8, 16])
    head = rng.choice([64, 80, 96, 112, 128, 128, 256])
    c = {"kind": kind, "type": rng.choice(["bf16", "bf16", "fp16"]), "heads": kv_heads * group, "kv_heads": kv_heads, "head": head}
    wide = kv_heads * head / 1024.0  # a row, against the listed cases' rows
    if kind == "write":
        hi = rng.choice([1, _log(rng, 2, 2048)])
        c.update(seqs=_log(rng, 1, 200 if hi == 1 else 8), lo=max(1, hi * rng.randint(3, 10) // 10), hi=hi)
    elif kind == "decode":
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 2, max(40, min(131072, int(250000 / (seqs * max(wide, 0.5))))))
        c.update(seqs=seqs, lo=max(1, hi // rng.randint(1, 9)), hi=hi, alibi=rng.random() < 0.3)
    elif kind == "prompt":
        seqs = _log(rng, 1, 8)
        q = _log(rng, 1, 1500)
        most = 1.0e9 / (seqs * c["heads"] * q) / max(1.0, head / 128)
        hi = rng.choice([0, _log(rng, 16, max(17, min(8192, int(most) - q)))])
        if q * q * seqs * c["heads"] > 9.0e8:
            q = int(math.sqrt(9.0e8 / (seqs * c["heads"])))
        c.update(seqs=seqs, qlo=max(1, q // rng.randint(1, 4)), qhi=q, lo=hi // 3, hi=hi, alibi=rng.random() < 0.3)
    elif kind == "weights":
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 2, max(40, min(65536, int(120000 / (seqs * max(wide, 0.5))))))
        c.update(seqs=seqs, lo=max(1, hi // rng.randint(1, 6)), hi=hi, cache=rng.choice(["auto", "int4"]))
    else:
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 32, max(64, min(32768, int(90000 / (seqs * max(wide, 0.5))))))
        keep = max(8, int(hi * rng.uniform(0.3, 1.0)))
        c.update(seqs=seqs, lo=max(1, hi * 2 // 3), hi=hi, keep=keep, recent=int(keep * rng.uniform(0.0, 0.6)))
    return c


def _spread(n, lo, hi):
    """n lengths between lo and hi, the same for every seed, spread evenly and out of order."""
    return [hi if n == 1 else lo + int((hi - lo + 0.999) * (((i + 1) * 0.6180339887498949) % 1.0)) for i in range(n)]


def _row_bytes(kv_heads, head):
    return (kv_heads * (head // 2 + 4) + 15) // 16 * 16


def work(case):
    h, hk, d = case["heads"], case["kv_heads"], case["head"]
    kind = case["kind"]
    if kind == "prompt":
        ql = _spread(case["seqs"], case["qlo"], case["qhi"])
        cached = _spread(case["seqs"], case["lo"], case["hi"])
        pairs = sum(q * c + q * (q + 1) // 2 for q, c in zip(ql, cached))
        rows = sum(q + c for q, c in zip(ql, cached))
        return {"bytes": 2 * rows * _row_bytes(hk, d) + 2 * sum(ql) * h * d * 2, "flops": 4.0 * pairs * h * d}
    lens = _spread(case["seqs"], case["lo"], case["hi"])
    rows = sum(lens)
    if kind == "write":  # values in, 4-bit rows out, values back
        return {"bytes": 2 * rows * (2 * hk * d * 2 + _row_bytes(hk, d)), "flops": 8.0 * rows * hk * d}
    if kind == "decode":
        return {"bytes": 2 * rows * _row_bytes(hk, d) + 2 * case["seqs"] * h * d * 2, "flops": 4.0 * rows * h * d}
    if kind == "weights":
        row = _row_bytes(hk, d) if case["cache"] == "int4" else hk * d * 2
        return {"bytes": rows * (row + 8 * hk) + case["seqs"] * h * d * 2, "flops": 2.0 * rows * h * d}
    # eviction: every weight is read; the recent rows, and the rows that fill the places of evicted ones, move
    moved = 0
    for n in lens:
        if n > case["keep"]:
            heavy = case["keep"] - case["recent"]
            old = n - case["recent"]
            moved += case["recent"] + heavy * (old - heavy) // max(1, old)
    return {"bytes": rows * hk * 4 + moved * hk * (2 * d * 2 + 4) * 2, "flops": 4.0 * rows * hk}


# ------------------------------------------------------------------------------------------------ the plain forms
def _quantise(x):
    """x [..., head] -> codes (uint8, one per value), scale and zero (float32 that bfloat16 holds).  In 64 bits: 16-bit
    values lie on the border between two codes often enough for a rounded quotient to show."""
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    zero = lo.to(torch.bfloat16).double()
    scale = ((hi.double() - zero) / torch.full_like(zero, 15.0)).float().to(torch.bfloat16).double()
    scale = torch.where(scale < 2.0 ** -126, torch.zeros_like(scale), scale)
    steps = (x.double() - zero) / torch.where(scale > 0, scale, torch.ones_like(scale))
    codes = torch.where(scale > 0, torch.floor(steps + 0.5).clamp_(0, 15), torch.zeros_like(steps)).to(torch.uint8)
    return codes, scale.float(), zero.float()


def _pack(codes, scale, zero):
    """... -> rows [..., row bytes] uint8, from codes [..., kv_heads, head] and scale, zero [..., kv_heads, 1]."""
    hk, d = codes.shape[-2:]
    half = codes[..., 0::2] | (codes[..., 1::2] << 4)
    tail = torch.cat([scale, zero], -1).to(torch.bfloat16).view(torch.uint8)
    rows = torch.cat([half.flatten(-2), tail.flatten(-2)], -1)
    return torch.nn.functional.pad(rows, (0, _row_bytes(hk, d) - rows.shape[-1]))


def _unpack(rows, hk, d):
    """rows [..., row bytes] -> values [..., kv_heads, head] float32."""
    n = hk * d // 2
    half = rows[..., :n].unflatten(-1, (hk, d // 2))
    codes = torch.stack([half & 15, half >> 4], -1).flatten(-2).float()
    tail = rows[..., n:n + 4 * hk].contiguous().view(torch.bfloat16).unflatten(-1, (hk, 2)).float()
    return codes * tail[..., 0:1] + tail[..., 1:2]


def _values(s, cache, longest):
    """The first `longest` rows of every sequence of the batch, [seqs, rows, kv_heads, head] float32."""
    rows = cache[s["slots"], :longest]
    return rows.float() if rows.dtype != torch.uint8 else _unpack(rows, s["hk"], s["d"])


def _probabilities(s, q, k, limit, positions=None):
    """Softmax over the rows: q [seqs, tokens, heads, head], k [seqs, rows, kv_heads, head], limit [seqs, tokens] rows
    visible to a token -> [seqs, kv_heads, group * tokens, rows]."""
    b, t, h, d = q.shape
    hk = s["hk"]
    q = q.view(b, t, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    x = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) * s["scale"]
    at = torch.arange(k.shape[1], device=k.device)
    x = x.view(b, hk, h // hk, t, -1)
    if s["slopes"] is not None:
        x = x + s["slopes"].view(1, hk, -1, 1, 1) * (at - limit[:, None, None, :, None] + 1).float()
    x = x.masked_fill(at >= limit[:, None, None, :, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    return (x / x.sum(-1, keepdim=True)).flatten(2, 3)


def _plain_attention(s, q, limit, longest):
    b, t, h, d = q.shape
    hk = s["hk"]
    p = _probabilities(s, q, _values(s, s["k"], longest), limit)
    o = torch.matmul(p, _values(s, s["v"], longest).permute(0, 2, 1, 3).contiguous())
    return o.view(b, hk, h // hk, t, d).permute(0, 3, 1, 2, 4).reshape(b, t, h, d)


def _plain_write(s):
    out = []
    for name, cache in (("key", s["k"]), ("value", s["v"])):
        codes, scale, zero = _quantise(s[name])
        cache[s["tok_slot"], s["tok_row"]] = _pack(codes, scale, zero)
        out.append((codes.float() * scale + zero).to(s[name].dtype))
    return out


def _plain_prompt(s):
    q = torch.zeros(s["b"], s["longest_query"], s["h"], s["d"], device="cuda")
    q[s["tok_seq"], s["tok_at"]] = s["query"].float()
    at = torch.arange(s["longest_query"], device="cuda")
    limit = s["lens"].long()[:, None] - s["query_lens"][:, None] + at + 1
    o = _plain_attention(s, q, limit, s["longest"])
    return o[s["tok_seq"], s["tok_at"]].to(s["query"].dtype)


def _plain_weights(s):
    p = _probabilities(s, s["query"].float()[:, None], _values(s, s["k"], s["longest"]), s["lens"].long()[:, None])
    s["weights"][s["slots"], :, :s["longest"]] += p.sum(2)
    return s["weights"]


def _plain_evict(s, weights, case):
    keep, recent, longest = case["keep"], case["recent"], s["longest"]
    heavy = keep - recent
    n = s["lens"].long()[:, None, None]
    at = torch.arange(longest, device="cuda").expand(s["b"], s["hk"], longest)
    w = weights[s["slots"], :, :longest]
    full = n > keep
    old = at < n - recent
    # the heaviest `heavy` of the rows that are not recent stay, equal ones from the lowest index on
    order = torch.sort(w.masked_fill(~old, -math.inf), dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, at.contiguous())
    stays = old & (rank < heavy)
    hole, mover = ~stays & (at < heavy), stays & (at >= heavy)
    movers = torch.sort(torch.where(mover, at, longest), dim=-1).values
    nth = (hole.cumsum(-1) - 1).clamp_min(0)
    src = torch.where(hole, movers.gather(-1, nth), at)
    src = torch.where((at >= heavy) & (at < keep), n - recent + at - heavy, src)
    src = torch.where(full & (at < keep), src, at)
    for cache in (s["k"], s["v"]):
        rows = cache[s["slots"], :longest]
        cache[s["slots"], :longest] = rows.gather(1, src.permute(0, 2, 1)[..., None].expand(rows.shape))
    w = w.gather(-1, src)
    weights[s["slots"], :, :longest] = torch.where(full & (at >= keep) & (at < n), 0.0, w)
    return torch.clamp(s["lens"], max=keep)


# ------------------------------------------------------------------------------------------------ inputs
def _rows(g, slots, rows, hk, d, dtype):
    """Keys or values of a model's distribution: normal, a few channels wider than the rest and off centre."""
    x = torch.randn(slots, rows, hk, d, generator=g, device="cuda", dtype=torch.float32)
    wide = (torch.rand(hk, d, generator=g, device="cuda") < 0.04).float()
    x.mul_(1 + 2 * wide).add_(wide * torch.randn(hk, d, generator=g, device="cuda"))
    return x.to(dtype)


def _int4_cache(g, slots, rows, hk, d, dtype):
    cache = torch.empty(slots, rows, _row_bytes(hk, d), dtype=torch.uint8, device="cuda")
    for i in range(slots):
        cache[i] = _pack(*_quantise(_rows(g, 1, rows, hk, d, dtype)[0]))
    return cache


def _pointers(cache):
    step = cache.stride(0) * cache.element_size()
    return torch.tensor([cache.data_ptr() + i * step for i in range(cache.shape[0])], dtype=torch.int64, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype = case["kind"], TYPES[case["type"]]
    b, h, hk, d = case["seqs"], case["heads"], case["kv_heads"], case["head"]
    slots = b + 1
    s = {"case": case, "b": b, "h": h, "hk": hk, "d": d, "scale": d ** -0.5, "slopes": None}
    s["slots"] = torch.randperm(slots, generator=g, device="cuda")[:b]
    if case.get("alibi"):
        s["slopes"] = 0.02 * torch.rand(h, generator=g, device="cuda") + 0.001
    lens = _spread(b, case["lo"], case["hi"])
    if kind == "write":
        row = _row_bytes(hk, d)
        rows = sum(lens)
        at = 0 if case["hi"] > 1 else 300  # a step appends behind rows that are there
        s["k"], s["v"] = (torch.zeros(slots, at + case["hi"], row, dtype=torch.uint8, device="cuda") for _ in range(2))
        s["key"], s["value"] = (_rows(g, 1, rows, hk, d, dtype)[0] for _ in range(2))
        starts = [sum(lens[:i]) for i in range(b)]
        s["slot_m"] = torch.full((b,), at * row, dtype=torch.int64, device="cuda")
        s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        s["tok_slot"] = torch.repeat_interleave(s["slots"], torch.tensor(lens, device="cuda"))
        s["tok_row"] = torch.tensor([at + t for n in lens for t in range(n)], device="cuda")
    else:
        if kind == "prompt":
            ql = _spread(b, case["qlo"], case["qhi"])
            lens = [q + c for q, c in zip(ql, lens)]
            s["host_query_lens"], s["longest_query"] = ql, max(ql)
            s["query_lens"] = torch.tensor(ql, dtype=torch.int64, device="cuda")
            s["tok_seq"] = torch.tensor([i for i, q in enumerate(ql) for _ in range(q)], device="cuda")
            s["tok_at"] = torch.tensor([t for q in ql for t in range(q)], device="cuda")
            queries = sum(ql)
        else:
            queries = b
        s["longest"] = max(lens)
        room = s["longest"]
        if kind in ("decode", "prompt") or case.get("cache") == "int4":
            s["k"], s["v"] = (_int4_cache(g, slots, room, hk, d, dtype) for _ in range(2))
        else:
            s["k"], s["v"] = (_rows(g, slots, room, hk, d, dtype) for _ in range(2))
        s["query"] = (1.5 * torch.randn(queries, h, d, generator=g, device="cuda")).to(dtype)
        if kind in ("weights", "evict"):
            # the accumulators as earlier steps have left them: mostly small, a few rows with much
            s["weights"] = torch.rand(slots, hk, room, generator=g, device="cuda").pow_(8).mul_(4)
            s["kept"] = s["weights"].clone()
    s["host_lens"] = lens
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["kp"], s["vp"] = _pointers(s["k"]), _pointers(s["v"])
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        from glake_amd import _custom_ops as ops
    if kind == "write":
        if not own:
            return _plain_write(s)
        ops.reshape_and_cache(s["key"], s["value"], s["kp"], s["vp"], s["slot_m"], s["slots"], s["lens"], s["starts"],
                              case["hi"], s["hk"], s["d"], "int4")
        key, value = torch.empty_like(s["key"]), torch.empty_like(s["value"])
        ops.read_cached_rows(key, value, s["kp"], s["vp"], s["slot_m"], s["slots"], s["lens"], s["starts"], case["hi"],
                             s["hk"], s["d"], "int4")
        return [key, value]
    if kind == "decode":
        if not own:
            o = _plain_attention(s, s["query"].float()[:, None], s["lens"].long()[:, None], s["longest"])
            return o[:, 0].to(s["query"].dtype)
        out = torch.empty_like(s["query"])
        ops.paged_attention_v1(out, s["query"], s["kp"], s["vp"], s["hk"], s["scale"], s["lens"], 1, s["longest"],
                               s["slopes"], "int4", 1.0, s["slots"])
        return out
    if kind == "prompt":
        if not own:
            return _plain_prompt(s)
        out = torch.empty_like(s["query"])
        ops.prefill_attention(out, s["query"], s["kp"], s["vp"], s["hk"], s["scale"], s["host_query_lens"],
                              s["host_lens"], s["slots"], s["slopes"], "int4")
        return out
    if kind == "weights":
        if not own:
            return _plain_weights(s)
        ops.accumulate_attention_weights(s["weights"], s["query"], s["kp"], s["hk"], s["scale"], s["lens"],
                                         s["longest"], s["slots"], None, case["cache"])
        return s["weights"]
    # an eviction empties the accumulators of the rows it frees: the next pass starts from the same ones again
    s["weights"].copy_(s["kept"])
    if own:
        lens = torch.empty_like(s["lens"])
        ops.evict_rows(s["kp"], s["vp"], s["weights"], s["lens"], lens, case["keep"], case["recent"], s["longest"],
                       s["slots"], s["hk"], s["d"], "auto", s["query"].dtype)
    else:
        lens = _plain_evict(s, s["weights"], case)
    return {"k": s["k"], "v": s["v"], "weights": s["weights"], "lens": lens}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_values(rows, hk, d):
    """A sequence's 4-bit rows [n, row bytes] as float64 [n, kv_heads, head]."""
    n = rows.shape[0]
    byte = rows[:, :hk * d // 2].to(torch.int32).reshape(n, hk, d // 2)
    v = torch.empty(n, hk, d, dtype=torch.float64, device=rows.device)
    v[:, :, 0::2] = byte % 16
    v[:, :, 1::2] = torch.div(byte, 16, rounding_mode="floor")
    pair = rows[:, hk * d // 2:hk * d // 2 + 4 * hk].to(torch.int32).reshape(n, hk, 2, 2)
    bits = ((pair[..., 1] * 256 + pair[..., 0]) * 65536).to(torch.int64)
    bits = torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).to(torch.int32)
    scale_zero = bits.view(torch.float32).double()
    return v * scale_zero[:, :, :1] + scale_zero[:, :, 1:]


def _exact_softmax(s, b, q, limit):
    """Weights of sequence b's rows for q [heads, tokens, head] (float64), limit [tokens]: [heads, tokens, rows]."""
    n = s["host_lens"][b]
    rows = s["k"][s["slots"][b], :n]
    k = _exact_values(rows, s["hk"], s["d"]) if rows.dtype == torch.uint8 else rows.double()
    group = s["h"] // s["hk"]
    k = k.transpose(0, 1).contiguous()
    x = torch.empty(s["h"], q.shape[1], n, dtype=torch.float64, device="cuda")
    at = torch.arange(n, device="cuda", dtype=torch.float64)
    for head in range(s["h"]):
        x[head] = (q[head] @ k[head // group].T) / math.sqrt(s["d"])
        if s["slopes"] is not None:
            x[head] += s["slopes"][head].double() * (at[None] + 1 - limit[:, None])
    x.masked_fill_(at[None, None] >= limit[None, :, None], -math.inf)
    return torch.softmax(x, -1)


def _exact_written(x):
    """What x [tokens, kv_heads, head] reads back as."""
    x = x.double()
    zero = x.min(-1).values.float().to(torch.bfloat16).double()
    scale = ((x.max(-1).values - zero) / 15).float().to(torch.bfloat16).double()
    safe = torch.where(scale > 0, scale, torch.ones_like(scale))
    codes = torch.floor((x - zero[..., None]) / safe[..., None] + 0.5).clamp(0, 15)
    return torch.where(scale[..., None] > 0, codes * scale[..., None] + zero[..., None], zero[..., None])


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "write":
        return [_exact_written(s["key"]), _exact_written(s["value"])]
    group = s["h"] // s["hk"]
    if kind in ("decode", "prompt"):
        out = torch.empty(s["query"].shape, dtype=torch.float64, device="cuda")
        at = 0
        for b, n in enumerate(s["host_lens"]):
            t = s["host_query_lens"][b] if kind == "prompt" else 1
            q = s["query"][at:at + t].double().transpose(0, 1).contiguous()
            limit = torch.arange(n - t + 1, n + 1, device="cuda", dtype=torch.float64)
            p = _exact_softmax(s, b, q, limit)
            v = _exact_values(s["v"][s["slots"][b], :n], s["hk"], s["d"]).transpose(0, 1).contiguous()
            for head in range(s["h"]):
                out[at:at + t, head] = p[head] @ v[head // group]
            at += t
        return out
    if kind == "weights":
        w = s["weights"].double()
        for b, n in enumerate(s["host_lens"]):
            limit = torch.full((1,), n, device="cuda", dtype=torch.float64)
            p = _exact_softmax(s, b, s["query"][b].double()[:, None], limit)[:, 0]
            w[s["slots"][b], :, :n] += p.view(s["hk"], group, n).sum(1)
        return w
    keep, recent = case["keep"], case["recent"]
    heavy = keep - recent
    out = {"k": s["k"].clone().double(), "v": s["v"].clone().double(), "weights": s["kept"].double(), "lens": None}
    weights = s["kept"].cpu().numpy()
    slots = s["slots"].tolist()
    for b, n in enumerate(s["host_lens"]):
        if n <= keep:
            continue
        for head in range(s["hk"]):
            w = weights[slots[b], head, :n - recent]
            chosen = sorted((-w).argsort(kind="stable")[:heavy].tolist())
            within = set(i for i in chosen if i < heavy)
            movers = iter([i for i in chosen if i >= heavy])
            src = [i if i in within else next(movers) for i in range(heavy)] + list(range(n - recent, n))
            index = torch.tensor(src, device="cuda")
            for name in ("k", "v"):
                out[name][slots[b], :keep, head] = s[name][slots[b], index, head].double()
            out["weights"][slots[b], head, :keep] = s["kept"][slots[b], head, index].double()
            out["weights"][slots[b], head, keep:n] = 0
    return out
