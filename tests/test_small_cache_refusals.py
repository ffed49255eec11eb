"""What the 4-bit cache and the eviction refuse, on the CPU: every bad call is turned away before a kernel is launched."""
import ctypes as C

import pytest
import torch

from glake_amd import _C, _custom_ops as ops
from glake_amd.worker.step import kv_row_bytes

P = C.c_void_p(4096)  # never followed: the call is refused before
N = C.c_void_p(0)


def refused(rc, *words):
    assert rc < 0
    for w in words:
        assert w in _C.last_error()


def test_row_bytes():
    lib = _C.lib()
    for hkv, d, want in ((8, 128, 544), (1, 128, 80), (1, 64, 48), (3, 80, 144), (5, 112, 304), (32, 256, 4224)):
        assert lib.vtkv_kv_row_bytes(hkv, d, _C.INT4) == kv_row_bytes(hkv, d, "int4") == want
    assert lib.vtkv_kv_row_bytes(8, 128, _C.BF16) == kv_row_bytes(8, 128) == 2048
    assert lib.vtkv_kv_row_bytes(8, 128, _C.FP8_E4M3) == kv_row_bytes(8, 128, "fp8") == 1024
    assert lib.vtkv_kv_row_bytes(8, 100, _C.INT4) == 0 and lib.vtkv_kv_row_bytes(0, 128, _C.INT4) == 0


def write(**kw):
    a = dict(k=P, v=P, kp=P, vp=P, sm=P, si=P, sl=P, cs=P, b=1, m=2, h=2, d=128, ks=256, vs=256, src=_C.BF16)
    a.update(kw)
    return _C.lib().vtkv_reshape_and_cache(*[a[x] for x in ("k", "v", "kp", "vp", "sm", "si", "sl", "cs", "b", "m", "h", "d",
                                                            "ks", "vs", "src")], _C.INT4, 1.0, 1.0, N)


def test_write_refusals():
    refused(write(d=72), "head sizes")
    refused(write(src=_C.F32), "float16")
    refused(write(ks=255), "stride")
    refused(write(sl=N), "seq_lens")
    refused(write(k=N), "null")
    refused(write(m=0))
    refused(write(m=70000), "65535")
    assert write(b=0) == 0


def read(**kw):
    a = dict(k=P, v=P, kp=P, vp=P, sm=P, si=P, sl=P, cs=P, b=1, m=2, h=2, d=128, ks=256, vs=256, dst=_C.BF16, kv=_C.INT4)
    a.update(kw)
    return _C.lib().vtkv_read_cached_rows(*[a[x] for x in ("k", "v", "kp", "vp", "sm", "si", "sl", "cs", "b", "m", "h", "d",
                                                           "ks", "vs", "dst", "kv")], N)


def test_read_refusals():
    refused(read(kv=_C.BF16), "4-bit")
    refused(read(dst=_C.FP8_E4M3))
    refused(read(d=100))
    refused(read(vs=1))
    assert read(b=0) == 0


def decode(**kw):
    a = dict(out=P, q=P, kp=P, vp=P, si=P, sl=P, b=2, h=8, hk=2, d=128, qs=1024, sc=0.1, m=64, al=N, qd=_C.BF16, od=_C.BF16,
             kv=_C.INT4, ws=N, wn=0)
    a.update(kw)
    return _C.lib().vtkv_decode_attention(a["out"], a["q"], a["kp"], a["vp"], a["si"], a["sl"], a["b"], a["h"], a["hk"], a["d"],
                                          a["qs"], a["sc"], a["m"], a["al"], a["qd"], a["od"], a["kv"], 1.0, 1.0, a["ws"],
                                          a["wn"], 0, N)


def test_decode_refusals():
    refused(decode(d=72), "head_size")
    refused(decode(h=7), "multiple")
    refused(decode(qd=_C.F32, od=_C.F32), "bfloat16 and float16")
    refused(decode(od=_C.F16), "out_dtype")
    refused(decode(qs=1023), "aligned")
    refused(decode(qs=512), "apart")
    refused(decode(m=0), "max_seq_len")
    refused(decode(sl=N), "null")
    assert decode(b=0) == 0


def test_entry_points_without_4_bit_rows():
    lib = _C.lib()
    refused(lib.vtkv_decode_attention_v2(P, P, P, P, P, P, P, P, P, 1, 8, 2, 128, 1024, 0.1, 64, 1, N, _C.BF16, _C.BF16, _C.INT4,
                                         1.0, 1.0, P, 1 << 20, N), "split-K")
    refused(lib.vtkv_decode_append_attention(P, P, P, P, 256, 256, P, P, P, P, None, 1, 8, 2, 128, 1024, 0.1, 64, N, _C.BF16,
                                             _C.BF16, _C.INT4, 1.0, 1.0, P, 1 << 20, 0, N), "reshape_and_cache")


def prompt(**kw):
    a = dict(d=128, h=8, hk=2, qs=1024, m=64, qd=_C.BF16, od=_C.BF16, sc=0.1, n=1, units=P)
    a.update(kw)
    return _C.lib().vtkv_prefill_attention(P, P, P, P, P, a["units"], a["n"], a["h"], a["hk"], a["d"], a["qs"], a["sc"], a["m"], N,
                                           a["qd"], a["od"], _C.INT4, 1.0, 1.0, N)


def test_prompt_refusals():
    refused(prompt(d=72))
    refused(prompt(qd=_C.F32, od=_C.F32))
    refused(prompt(od=_C.F16), "out_dtype")
    refused(prompt(qs=100))
    refused(prompt(m=0))
    refused(prompt(units=N))
    assert prompt(n=0) == 0


def weigh(**kw):
    a = dict(w=P, ss=128, hs=64, ns=4, q=P, kp=P, si=P, sl=P, b=1, h=8, hk=2, d=128, qs=1024, m=64, qd=_C.BF16, kv=_C.BF16, ks=1.0,
             ws=P, wn=1 << 30)
    a.update(kw)
    return _C.lib().vtkv_accumulate_attention_weights(
        a["w"], a["ss"], a["hs"], a["ns"], a["q"], a["kp"], a["si"], a["sl"], a["b"], a["h"], a["hk"], a["d"], a["qs"], 0.1, a["m"],
        N, a["qd"], a["kv"], a["ks"], a["ws"], a["wn"], N)


def test_weight_refusals():
    refused(weigh(w=N), "null")
    refused(weigh(d=72), "head_size")
    refused(weigh(h=9), "multiple")
    refused(weigh(qd=_C.F32, kv=_C.F32), "BF16 or F16")
    refused(weigh(kv=_C.F16), "kv_dtype")
    refused(weigh(kv=_C.FP8_E4M3, ks=0.0), "positive")
    refused(weigh(qs=1020))
    refused(weigh(m=0))
    refused(weigh(ns=0))
    assert weigh(b=0) == 0


def evict(**kw):
    a = dict(kp=P, vp=P, w=P, ns=4, si=P, sl=P, nl=P, b=1, hk=2, d=128, kv=_C.BF16, keep=10, recent=5, m=64, ws=P, wn=1 << 20)
    a.update(kw)
    return _C.lib().vtkv_evict_rows(a["kp"], a["vp"], a["w"], 128, 64, a["ns"], a["si"], a["sl"], a["nl"], a["b"], a["hk"], a["d"],
                                    a["kv"], a["keep"], a["recent"], a["m"], a["ws"], a["wn"], N)


def test_evict_refusals():
    refused(evict(nl=N), "null")
    refused(evict(keep=0), "keep_rows")
    refused(evict(recent=11), "recent_rows")
    refused(evict(recent=-1), "recent_rows")
    refused(evict(d=72))
    refused(evict(kv=9), "kv_dtype")
    refused(evict(m=0))
    assert evict(wn=8) == _C.ENOMEM and evict(ws=N) == _C.ENOMEM
    assert evict(b=0) == 0


def test_python_refusals():
    key = torch.zeros(2, 2, 128, dtype=torch.bfloat16)
    i64, i32 = torch.zeros(2, dtype=torch.int64), torch.ones(2, dtype=torch.int32)
    with pytest.raises(_C.VtkvError, match="GPU"):
        ops.reshape_and_cache(key, key, 0, 0, i64, i64, None, None, 1, 2, 128, "int4")
    with pytest.raises(_C.VtkvError, match="int4"):
        ops.read_cached_rows(key, key, 0, 0, i64, i64, None, None, 1, 2, 128, "fp8")
    with pytest.raises(_C.VtkvError, match="GPU"):
        ops.accumulate_attention_weights(torch.zeros(2, 2, 8), key, 0, 2, 0.1, i32, 8, i64)
    with pytest.raises(_C.VtkvError, match="GPU"):
        ops.evict_rows(0, 0, torch.zeros(2, 2, 8), i32, i32, 4, 2, 8, i64, 2, 128)
    with pytest.raises(_C.VtkvError, match="scales"):
        ops._int4_scales("int4", 0.5)
    with pytest.raises(_C.VtkvError, match="kv cache"):
        ops._kv_dtype("int3", _C.BF16)
    for bad in (torch.zeros(2, 3, 8), torch.zeros(2, 2, 7), torch.zeros(2, 2, 8, dtype=torch.float64), torch.zeros(2, 2, 16)[..., ::2]):
        with pytest.raises(_C.VtkvError, match="weights"):
            ops._weights_of(bad, 2, 8)


def test_pointer_tables():
    ops._pointer_tables(0, 123)
    for bad in (torch.zeros(4, dtype=torch.int64), torch.zeros(4, dtype=torch.int32)):
        with pytest.raises(_C.VtkvError, match="pointer table"):
            ops._pointer_tables(0, bad)
    weights = torch.zeros(5, 2, 8)
    assert ops._num_slots(weights, 0) == 5 and ops._num_slots(weights, torch.zeros(3, dtype=torch.int64), 0) == 3


def test_cache_engine_refusals():
    from glake_amd.worker.cache_engine import CacheEngine

    for dtype, kind in ((torch.bfloat16, "int3"), (torch.bfloat16, "fp8"), (torch.uint8, "auto")):
        with pytest.raises(_C.VtkvError):
            CacheEngine(1, 2, 128, dtype, 1, 64, kv_cache_dtype=kind)
    assert CacheEngine.get_cache_block_size(16, 8, 128, 2, torch.bfloat16, "int4") == 2 * 2 * 16 * 544
