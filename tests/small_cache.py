"""Test-side forms, in float64 on the host, of the operators that make a cache smaller: 4-bit rows, attention over them,
the attention weight drawn by each row, eviction.  Written from the definitions, apart from the kernels."""
from __future__ import annotations

import numpy as np


def to_bf16(x):
    """float64 -> the nearest bfloat16 value (by way of float32, ties to even), as float64."""
    u = np.asarray(x, np.float32).view(np.uint32)
    r = (u + 0x7FFF + ((u >> 16) & 1)) & np.uint32(0xFFFF0000)
    return r.astype(np.uint32).view(np.float32).astype(np.float64)


def bf16_bits(x):
    return (np.asarray(x, np.float32).view(np.uint32) >> 16).astype(np.uint16)


def row_bytes(hkv, d):
    return (hkv * (d // 2 + 4) + 15) // 16 * 16


def quantise(x):
    """x [..., d] -> codes, scale [..., 1], zero [..., 1]."""
    x = np.asarray(x, np.float64)
    zero = to_bf16(x.min(-1, keepdims=True))
    scale = to_bf16((x.max(-1, keepdims=True) - zero) / 15.0)
    scale = np.where(scale < 2.0 ** -126, 0.0, scale)
    steps = (x - zero) / np.where(scale > 0, scale, 1.0)
    codes = np.where(scale > 0, np.clip(np.floor(steps + 0.5), 0, 15), 0)
    return codes.astype(np.uint8), scale, zero


def pack(codes, scale, zero):
    """codes [rows, hkv, d] -> [rows, row_bytes] uint8"""
    rows, hkv, d = codes.shape
    out = np.zeros((rows, row_bytes(hkv, d)), np.uint8)
    out[:, :hkv * d // 2] = (codes[..., 0::2] | (codes[..., 1::2] << 4)).reshape(rows, hkv * d // 2)
    pair = np.concatenate([bf16_bits(scale), bf16_bits(zero)], -1)  # [rows, hkv, 2] uint16
    out[:, hkv * d // 2:hkv * d // 2 + 4 * hkv] = np.ascontiguousarray(pair.reshape(rows, 2 * hkv)).view(np.uint8)
    return out


def values(codes, scale, zero):
    return codes.astype(np.float64) * scale + zero


def softmax(q, k, scale, limit=None, slopes=None):
    """q [t, h, d], k [n, hkv, d], limit [t] (rows a token sees) -> weights [t, h, n]; all zero where a token sees none."""
    t, h, d = q.shape
    n, hkv, _ = k.shape
    group = h // hkv
    x = np.einsum("tkgd,nkd->tkgn", q.reshape(t, hkv, group, d), k).reshape(t, h, n) * scale
    limit = np.full(t, n) if limit is None else np.asarray(limit)
    at = np.arange(n)
    if slopes is not None:
        x = x + np.asarray(slopes, np.float64)[None, :, None] * (at[None] + 1 - limit[:, None])[:, None]
    x = np.where(at[None, None] < limit[:, None, None], x, -np.inf)
    top = np.where(limit[:, None, None] > 0, x.max(-1, keepdims=True, initial=-np.inf), 0.0)
    e = np.exp(x - top)
    s = e.sum(-1, keepdims=True)
    return np.divide(e, s, out=np.zeros_like(e), where=s > 0)


def attention(q, k, v, scale, limit=None, slopes=None):
    p = softmax(q, k, scale, limit, slopes)
    t, h, n = p.shape
    hkv, d = v.shape[1:]
    return np.einsum("tkgn,nkd->tkgd", p.reshape(t, hkv, h // hkv, n), v).reshape(t, h, d)


def evicted_sources(weights, n, keep, recent):
    """weights [n] of one head -> the row that ends up at each of the first min(n, keep) places."""
    if n <= keep:
        return list(range(n))
    heavy = keep - recent
    order = sorted(range(n - recent), key=lambda i: (-weights[i], i))
    stays = set(order[:heavy])
    movers = [i for i in sorted(stays) if i >= heavy]
    src, at = [], 0
    for i in range(heavy):
        if i in stays:
            src.append(i)
        else:
            src.append(movers[at])
            at += 1
    return src + list(range(n - recent, n))


class Ranges:
    """Ranges of `slots` sequences with `rows` rows of `row` bytes each, as plain GPU memory, and their pointer tables."""

    def __init__(self, slots, rows, row, fill=0xFF):
        import torch

        self.row = row
        self.k = torch.full((slots, rows, row), fill, dtype=torch.uint8, device="cuda")
        self.v = torch.full((slots, rows, row), fill, dtype=torch.uint8, device="cuda")

        def table(t):
            return torch.tensor([t.data_ptr() + i * t.stride(0) for i in range(slots)], dtype=torch.int64, device="cuda")

        self.kp, self.vp = table(self.k), table(self.v)


def model_values(rng, shape):
    """Values of a model's keys: normal, with a few wide channels off centre."""
    x = rng.standard_normal(shape)
    wide = rng.random(shape[-2:]) < 0.05
    return x * (1 + 2 * wide) + wide * rng.standard_normal(shape[-2:])


def as_type(x, dtype):
    """x (float64) rounded to a torch dtype: (torch tensor on the GPU, its values as float64)."""
    import torch

    t = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(dtype)
    return t.cuda(), t.double().numpy()


def step_metadata(engine, slots, seq_lens, prompts):
    """Metadata of a batch that holds all prompts (every row of seq_lens new) or all decode tokens."""
    import torch

    from glake_amd.attention.backends.vtensor import VTensorBackend

    n = len(slots)
    meta = VTensorBackend.make_metadata(
        num_prefills=n if prompts else 0, num_prefill_tokens=sum(seq_lens) if prompts else 0,
        num_decode_tokens=0 if prompts else n, slot_mapping=torch.tensor(slots, dtype=torch.int64, device="cuda"),
        seq_lens=list(seq_lens), seq_lens_tensor=torch.tensor(seq_lens, dtype=torch.int32, device="cuda"),
        max_query_len=max(seq_lens) if prompts else None, max_prefill_seq_len=max(seq_lens) if prompts else 0,
        max_decode_seq_len=0 if prompts else max(seq_lens), query_start_loc=None, seq_start_loc=None,
        context_lens_tensor=None, block_tables=None, is_extend=0, kv_batch_stride=engine.kv_batch_stride,
        kv_num_heads=engine.num_kv_heads, kv_head_size=engine.head_size, max_seq_len=max(seq_lens),
        slot_mapping_list=list(slots), set_used_size=[0] * n, extend_seq_list=[-1] * n, use_cuda_graph=False)
    meta.k_cache_segment_ptr_list = engine.k_cache_ptr
    meta.v_cache_segment_ptr_list = engine.v_cache_ptr
    meta.kvcache_segment = [engine.vmm_kvcache_segment[s] for s in slots]
    return meta
