"""The 4-bit cache on the GPU against float64 forms on the host: rows written and read back, decode attention, prompt
attention, and the paths that lead there (backend, step plan, cache engine).

Tolerances.  Rows: byte for byte.  Decode attention before its rounding: a logit is off by less than 2^-14 (fp32 sums
of at most 256 products whose magnitudes add up to less than 2^9), so a weight by 2^-13 of itself, and the weights are
carried with 16 bits or more: 2^-12 of the largest value in all.  Prompt attention rounds weights and values to fp16,
half a step being 2^-11 of each, and adds the same logit error: 2^-10 + 2^-11 of the largest value.  The output's own
rounding is half a step of its type, finfo.eps / 2 of the value."""
import numpy as np
import pytest

import small_cache as S

pytestmark = pytest.mark.gpu

HEADS = [(32, 8), (8, 8), (8, 1), (15, 5), (28, 4), (12, 6), (16, 1), (71, 1), (40, 2), (64, 8), (96, 32)]


@pytest.fixture(scope="module")
def env():
    import torch

    from glake_amd import _custom_ops as ops

    assert torch.cuda.is_available()
    torch.cuda.set_device(0)
    return torch, ops


def dtypes(torch):
    return {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def filled(rng, lens, hkv, d, slots, room=0):
    """Ranges with the lens[i] rows of sequence i in its slot; what lies behind them is NaN."""
    import torch

    r = S.Ranges(len(lens) + 2, max(lens) + 1 + room, S.row_bytes(hkv, d))
    k, v = [], []
    for n, slot in zip(lens, slots):
        for values, cache in ((k, r.k), (v, r.v)):
            x = S.quantise(S.to_bf16(S.model_values(rng, (n, hkv, d))))
            values.append(S.values(*x))
            cache[slot, :n] = torch.from_numpy(S.pack(*x)).cuda()
    return r, k, v


# ------------------------------------------------------------------------------------------------ rows
def write_case(env, seed, lens, hkv, d, dtype, change=None, stride=0, offset=5):
    torch, ops = env
    rng = np.random.default_rng(seed)
    b, t = len(lens), sum(lens)
    x = [S.model_values(rng, (t, hkv, d)) for _ in range(2)]
    if change is not None:
        change(x)
    tensors, want = [], []
    for a in x:
        dev, host = S.as_type(a, dtype)
        if stride:
            wide = torch.zeros(t, hkv * d + stride, dtype=dtype, device="cuda")
            wide[:, :hkv * d] = dev.view(t, -1)
            dev = wide[:, :hkv * d].view(t, hkv, d) if stride % 8 == 0 else wide[:, :hkv * d].unflatten(1, (hkv, d))
        tensors.append(dev)
        want.append(host)
    row = S.row_bytes(hkv, d)
    r = S.Ranges(b + 2, offset + max(lens) + 2, row, fill=0xA5)
    slots = rng.permutation(b + 2)[:b]
    starts = np.concatenate([[0], np.cumsum(lens)[:-1]])
    i32 = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")  # noqa: E731
    slot_m = torch.tensor([offset * row] * b, dtype=torch.int64, device="cuda")
    slot_t = torch.tensor(slots, dtype=torch.int64, device="cuda")
    args = (r.kp, r.vp, slot_m, slot_t, i32(lens), i32(starts), max(lens), hkv, d, "int4")
    ops.reshape_and_cache(*tensors, *args)
    back = [torch.full((t, hkv, d), 77.0, dtype=torch.float32, device="cuda") for _ in range(2)]
    ops.read_cached_rows(*back, *args)
    rounded = [torch.empty(t, hkv, d, dtype=dtype, device="cuda") for _ in range(2)]
    ops.read_cached_rows(*rounded, *args)
    torch.cuda.synchronize()
    for cache, host, got, got16 in ((r.k, want[0], back[0], rounded[0]), (r.v, want[1], back[1], rounded[1])):
        expect = np.full(cache.shape, 0xA5, np.uint8)
        codes, scale, zero = S.quantise(host)
        packed = S.pack(codes, scale, zero)
        for i, n in enumerate(lens):
            expect[slots[i], offset:offset + n] = packed[starts[i]:starts[i] + n]
        assert np.array_equal(cache.cpu().numpy(), expect)
        v = S.values(codes, scale, zero).astype(np.float32)
        assert np.array_equal(got.cpu().numpy(), v)
        assert torch.equal(got16.cpu(), torch.from_numpy(v).to(dtype))


@pytest.mark.parametrize("d", [64, 80, 96, 112, 128, 256])
@pytest.mark.parametrize("hkv", [1, 3, 8])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_rows_written_and_read_back(env, d, hkv, dtype):
    write_case(env, d + hkv, [1, 17, 2], hkv, d, dtypes(env[0])[dtype])
    write_case(env, d + hkv + 1, [1, 1, 1, 1, 1], hkv, d, dtypes(env[0])[dtype])


def test_rows_of_equal_tiny_and_large_values(env):
    def change(x):
        for a in x:
            a[0] = 0.0
            a[1] = -3.25
            a[2] = 1e-30 * a[2]
            a[3] = 1e-38 * a[3]
            a[4] = 1e30 * a[4]
            a[5] = 100.0 + 1e-3 * a[5]
            a[6, :, ::2] = 0.0
            a[7, :, 0] = 3e38

    write_case(env, 3, [9, 4], 4, 128, env[0].bfloat16, change)

    def change16(x):
        for a in x:
            a[0] = -0.0
            a[1] = 2049.0  # no bfloat16: the zero is rounded, above every value of the row
            a[2] = 6e-8 * np.round(a[2])
            a[3] = np.clip(30000 * a[3], -65504, 65504)
            a[4] = 2049.0 + a[4]

    write_case(env, 4, [9, 4], 4, 128, env[0].float16, change16)


def test_rows_on_the_border_between_two_codes(env):
    # whole and half steps of a power-of-two scale: every second value lies exactly on a border
    def change(x):
        for a in x:
            a[:] = np.random.default_rng(9).integers(0, 31, a.shape) / 2.0 - 7.5
            a[..., 0], a[..., 1] = -7.5, 7.5

    write_case(env, 5, [33, 8], 2, 64, env[0].bfloat16, change)


@pytest.mark.parametrize("stride", [8, 3])
def test_rows_from_strided_tensors(env, stride):
    write_case(env, 6, [3, 5], 8, 128, env[0].bfloat16, stride=stride)


def test_rows_that_are_not_finite_read_back_as_nan(env):
    torch, ops = env
    rng = np.random.default_rng(8)
    key = torch.from_numpy(rng.standard_normal((4, 4, 80)).astype(np.float32)).bfloat16().cuda()
    key[0, 1, 7], key[1, 3, 79], key[2, 0, 0] = float("nan"), float("inf"), float("-inf")
    key[3, 2, 0], key[3, 2, 1] = 3e38, -3e38
    r = S.Ranges(4, 2, S.row_bytes(4, 80))
    slots = torch.arange(4, device="cuda")
    at = torch.zeros(4, dtype=torch.int64, device="cuda")
    at[1] = -1  # skipped
    ops.reshape_and_cache(key, key, r.kp, r.vp, at, slots, None, None, 1, 4, 80, "int4")
    got = torch.zeros(4, 4, 80, device="cuda")
    ops.read_cached_rows(got, torch.empty_like(got), r.kp, r.vp, at, slots, None, None, 1, 4, 80)
    nan = torch.isnan(got).all(-1).cpu().numpy()
    want = np.zeros((4, 4), bool)
    want[0, 1] = want[2, 0] = want[3, 2] = True
    assert np.array_equal(nan, want) and not torch.isnan(got[~torch.isnan(got).all(-1)]).any()
    assert (r.k[1] == 0xFF).all() and (got[1] == 0).all()


# ------------------------------------------------------------------------------------------------ decode
def check(got, want, v_max, dtype_eps, bound):
    err = np.abs(got - want)
    lim = bound * v_max + dtype_eps / 2 * np.abs(want)
    assert np.isfinite(got).all() and (err <= lim).all(), f"max err {err.max():.3e}, {(err / lim).max():.2f} of the bound"


def decode_case(env, seed, lens, hq, hkv, d=128, dtype="bf16", alibi=False, q_scale=1.5, extra=0, change=None):
    torch, ops = env
    rng = np.random.default_rng(seed)
    b = len(lens)
    slots = rng.permutation(b + 2)[:b]
    r, k, v = filled(rng, lens, hkv, d, slots)
    if change is not None:
        change(r, slots)
    q, q_host = S.as_type(rng.standard_normal((b, hq, d)) * q_scale, dtypes(torch)[dtype])
    slopes = np.abs(rng.standard_normal(hq)).astype(np.float32) * 0.05 if alibi else None
    args = (r.kp, r.vp, hkv, d ** -0.5, torch.tensor(lens, dtype=torch.int32, device="cuda"), 1, max(lens) + extra,
            None if slopes is None else torch.from_numpy(slopes).cuda(), "int4", 1.0,
            torch.tensor(slots, dtype=torch.int64, device="cuda"))
    out32 = torch.full((b, hq, d), 55.0, device="cuda")
    out16 = torch.full((b, hq, d), 55.0, dtype=q.dtype, device="cuda")
    ops.paged_attention_v1(out32, q, *args)
    ops.paged_attention_v1(out16, q, *args)
    torch.cuda.synchronize()
    for i in range(b):
        want = S.attention(q_host[i:i + 1], k[i], v[i], d ** -0.5, [lens[i]], slopes)[0]
        v_max = np.abs(v[i]).max() if lens[i] else 0.0
        check(out32[i].double().cpu().numpy(), want, v_max, 0.0, 2.0 ** -12)
        check(out16[i].double().cpu().numpy(), want, v_max, torch.finfo(q.dtype).eps, 2.0 ** -12)
    assert torch.equal(out32.to(q.dtype), out16)


@pytest.mark.parametrize("hq,hkv", HEADS)
def test_decode_heads(env, hq, hkv):
    decode_case(env, hq + hkv, [1, 15, 16, 17, 63, 64, 65, 257, 1030], hq, hkv)


@pytest.mark.parametrize("d", [64, 80, 96, 112, 256])
@pytest.mark.parametrize("hq,hkv", [(32, 8), (8, 8), (7, 1), (12, 3)])
def test_decode_head_sizes(env, d, hq, hkv):
    decode_case(env, d, [1, 2, 31, 129, 500, 777], hq, hkv, d, dtype="fp16" if hq == 8 else "bf16")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_decode_alibi(env, dtype):
    decode_case(env, 1, [3, 100, 513], 16, 4, 128, dtype, alibi=True)
    decode_case(env, 2, [3, 100, 513], 8, 8, 80, dtype, alibi=True)
    decode_case(env, 2, [3, 100, 513], 26, 2, 64, dtype, alibi=True)


def test_decode_empty_sequences_and_a_loose_bound(env):
    decode_case(env, 3, [0, 40, 0, 0, 700, 1, 0], 8, 2, extra=1000)
    decode_case(env, 3, [0, 0], 8, 2, extra=5)


def test_decode_large_logits(env):
    decode_case(env, 4, [300, 1500], 32, 8, q_scale=12.0)


def test_decode_many_and_long_sequences(env):
    decode_case(env, 5, list(np.random.default_rng(1).integers(1, 90, 1100)), 2, 1, 64)
    decode_case(env, 6, [20011], 32, 8)
    decode_case(env, 7, [9001, 5], 4, 1, 256)


def test_decode_ragged_batches(env):
    """Sequences of a few rows between empty and long ones: workgroups with several sequences, spans that begin or end before
    a sequence's first row."""
    rng = np.random.default_rng(14)
    decode_case(env, 15, [1] * 70, 8, 8, 80)
    decode_case(env, 16, [0, 1] * 60 + [3000], 8, 2)
    decode_case(env, 17, list(rng.integers(0, 300, 40)) + [9000] + list(rng.integers(0, 20, 40)), 16, 16, 64, "fp16")
    decode_case(env, 18, list(rng.integers(1, 600, 33)), 24, 1, 128)


@pytest.mark.parametrize("factor", [1e6, 1e-12])
def test_decode_large_and_small_values(env, factor):
    torch, ops = env
    rng = np.random.default_rng(19)
    lens, hq, hkv, d = [200, 33], 8, 2, 128
    r, k, v = filled(rng, lens, hkv, d, [0, 1])
    for i, n in enumerate(lens):
        x = S.quantise(S.to_bf16(factor * S.model_values(rng, (n, hkv, d))))
        v[i] = S.values(*x)
        r.v[i, :n] = torch.from_numpy(S.pack(*x)).cuda()
    q, q_host = S.as_type(rng.standard_normal((2, hq, d)) * 1.5, torch.bfloat16)
    out = torch.full((2, hq, d), 55.0, device="cuda")
    ops.paged_attention_v1(out, q, r.kp, r.vp, hkv, d ** -0.5, torch.tensor(lens, dtype=torch.int32, device="cuda"), 1, 200,
                           None, "int4", 1.0, torch.tensor([0, 1], device="cuda"))
    for i in range(2):
        want = S.attention(q_host[i:i + 1], k[i], v[i], d ** -0.5)[0]
        # (weights times scales below 2^-57 lose bits, 2^-53 at most per row)
        check(out[i].double().cpu().numpy() / factor, want / factor, np.abs(v[i]).max() / factor, 0.0,
              2.0 ** -12 + lens[i] * 15 * 2.0 ** -53 / np.abs(v[i]).max())


def test_decode_without_a_workspace(env):
    """The entry point that takes no workspace, against the one that does."""
    import ctypes as C

    from glake_amd import _C

    torch, _ = env
    rng = np.random.default_rng(20)
    for lens, hq, hkv, d in (([700, 1, 33, 0, 5000], 32, 8, 128), ([90, 400], 128, 8, 256)):
        b = len(lens)
        r, _, _ = filled(rng, lens, hkv, d, list(range(b)))
        q = torch.from_numpy(rng.standard_normal((b, hq, d)).astype(np.float32)).bfloat16().cuda()
        lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
        slots = torch.arange(b, device="cuda")
        outs = [torch.full((b, hq, d), 55.0, device="cuda") for _ in range(2)]
        lib = _C.lib()
        p = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
        stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
        ws = torch.zeros(lib.vtkv_decode_attention_workspace_bytes(b, hq, d, max(lens), 0), dtype=torch.uint8, device="cuda")
        for out, tail, entry in ((outs[0], (), lib.vtkv_decode_attention_noalloc),
                                 (outs[1], (p(ws), ws.numel(), 0), lib.vtkv_decode_attention)):
            _C.check(entry(p(out), p(q), p(r.kp), p(r.vp), p(slots), p(lens_t), b, hq, hkv, d, hq * d, d ** -0.5, max(lens), None,
                           _C.BF16, _C.F32, _C.INT4, 1.0, 1.0, *tail, stream))
        torch.cuda.synchronize()
        # (the spans may differ with the workspace, and with them the order of the sums: 2^-12 of the values each)
        assert torch.isfinite(outs[0]).all() and (outs[0] - outs[1]).abs().max() <= 2.0 ** -11 * 10
        assert (outs[0][3] == 0).all() if len(lens) == 5 else True


def test_decode_strided_queries(env):
    torch, ops = env
    rng = np.random.default_rng(11)
    lens, hq, hkv, d = [30, 90], 8, 2, 128
    r, k, v = filled(rng, lens, hkv, d, [0, 1])
    wide = torch.from_numpy(rng.standard_normal((2, 3 * hq * d)).astype(np.float32)).bfloat16().cuda()
    q = wide[:, hq * d:2 * hq * d].unflatten(1, (hq, d))
    out = torch.empty(2, hq, d, dtype=torch.bfloat16, device="cuda")
    ops.paged_attention_v1(out, q, r.kp, r.vp, hkv, d ** -0.5, torch.tensor(lens, dtype=torch.int32, device="cuda"), 1, 90,
                           None, "int4", 1.0, torch.tensor([0, 1], device="cuda"))
    for i in range(2):
        want = S.attention(q[i:i + 1].double().cpu().numpy(), k[i], v[i], d ** -0.5)[0]
        check(out[i].double().cpu().numpy(), want, np.abs(v[i]).max(), 2.0 ** -7, 2.0 ** -12)


def test_decode_a_row_that_is_not_finite_stays_with_its_head(env):
    torch, ops = env
    rng = np.random.default_rng(12)
    lens, hq, hkv, d = [70, 90], 8, 2, 128
    r, k, v = filled(rng, lens, hkv, d, [0, 1])
    r.k[1, 33, hkv * d // 2:hkv * d // 2 + 4] = torch.tensor([0xC0, 0x7F, 0xC0, 0x7F], dtype=torch.uint8)  # head 0
    q = torch.from_numpy(rng.standard_normal((2, hq, d)).astype(np.float32)).bfloat16().cuda()
    out = torch.empty(2, hq, d, dtype=torch.float32, device="cuda")
    ops.paged_attention_v1(out, q, r.kp, r.vp, hkv, d ** -0.5, torch.tensor(lens, dtype=torch.int32, device="cuda"), 1, 90,
                           None, "int4", 1.0, torch.tensor([0, 1], device="cuda"))
    out = out.double().cpu().numpy()
    assert np.isnan(out[1, :4]).all()
    for i, heads in ((0, slice(0, 8)), (1, slice(4, 8))):
        want = S.attention(q[i:i + 1].double().cpu().numpy(), k[i], v[i], d ** -0.5)[0]
        check(out[i, heads], want[heads], np.abs(v[i]).max(), 0.0, 2.0 ** -12)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_a_query_that_is_not_finite_stays_with_its_head(env, dtype, value):
    """Decode and prompt attention: the other heads of the same kv head and the other tokens are as without it."""
    torch, ops = env
    rng = np.random.default_rng(22)
    lens, hq, hkv, d = [70, 90], 8, 2, 128
    r, k, v = filled(rng, lens, hkv, d, [0, 1])
    q, q_host = S.as_type(rng.standard_normal((2, hq, d)), dtypes(torch)[dtype])
    q[1, 1, 5] = value
    slots = torch.tensor([0, 1], device="cuda")
    out = torch.empty(2, hq, d, dtype=torch.float32, device="cuda")
    ops.paged_attention_v1(out, q, r.kp, r.vp, hkv, d ** -0.5, torch.tensor(lens, dtype=torch.int32, device="cuda"), 1, 90,
                           None, "int4", 1.0, slots)
    prompt = torch.empty(2, hq, d, dtype=torch.float32, device="cuda")
    ops.prefill_attention(prompt, q, r.kp, r.vp, hkv, d ** -0.5, [1, 1], lens, slots, None, "int4")
    for got, bound in ((out, 2.0 ** -12), (prompt, 2.0 ** -8)):  # (a unit with such a query is computed with bfloat16 values)
        got = got.double().cpu().numpy()
        assert np.isnan(got[1, 1]).all()
        for i in range(2):
            want = S.attention(q_host[i:i + 1], k[i], v[i], d ** -0.5)[0]
            heads = [h for h in range(hq) if (i, h) != (1, 1)]
            check(got[i, heads], want[heads], np.abs(v[i]).max(), 0.0, bound)


def test_decode_in_a_graph_and_on_two_streams(env):
    torch, ops = env
    rng = np.random.default_rng(13)
    lens, hq, hkv, d = [900, 257, 64], 32, 8, 128
    r, k, v = filled(rng, lens, hkv, d, [0, 1, 2])
    q = torch.from_numpy(rng.standard_normal((3, hq, d)).astype(np.float32)).bfloat16().cuda()
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    slots = torch.tensor([0, 1, 2], device="cuda")

    def call(out):
        ops.paged_attention_v1(out, q, r.kp, r.vp, hkv, d ** -0.5, lens_t, 1, 900, None, "int4", 1.0, slots)

    want = torch.empty(3, hq, d, dtype=torch.float32, device="cuda")
    call(want)
    outs = [torch.zeros_like(want) for _ in range(2)]
    graphs = []
    for o in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(o)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for n in ([900, 257, 64], [1, 256, 3], [899, 0, 64]):
        lens_t.copy_(torch.tensor(n, dtype=torch.int32))
        call(want)
        torch.cuda.synchronize()
        for g, s, o in zip(graphs, streams, outs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o, want)
    eager = [torch.zeros_like(want) for _ in range(2)]
    for s, o in zip(streams, eager):
        with torch.cuda.stream(s):
            for _ in range(5):
                call(o)
    torch.cuda.synchronize()
    assert torch.equal(eager[0], want) and torch.equal(eager[1], want)


# ------------------------------------------------------------------------------------------------ prompts
def prompt_case(env, seed, query_lens, cached, hq, hkv, d=128, dtype="bf16", alibi=False, v_mul=1.0):
    torch, ops = env
    rng = np.random.default_rng(seed)
    lens = [a + c for a, c in zip(query_lens, cached)]
    b = len(lens)
    slots = rng.permutation(b + 2)[:b]
    r, k, v = filled(rng, lens, hkv, d, slots)
    if v_mul != 1.0:
        for i, (n, slot) in enumerate(zip(lens, slots)):
            x = S.quantise(S.to_bf16(v_mul * S.model_values(rng, (n, hkv, d))))
            v[i] = S.values(*x)
            r.v[slot, :n] = torch.from_numpy(S.pack(*x)).cuda()
    t = sum(query_lens)
    q, q_host = S.as_type(rng.standard_normal((t, hq, d)) * 1.5, dtypes(torch)[dtype])
    slopes = np.abs(rng.standard_normal(hq)).astype(np.float32) * 0.05 if alibi else None
    slopes_t = None if slopes is None else torch.from_numpy(slopes).cuda()
    out32 = torch.full((t, hq, d), 55.0, device="cuda")
    out16 = torch.full((t, hq, d), 55.0, dtype=q.dtype, device="cuda")
    for o in (out32, out16):
        ops.prefill_attention(o, q, r.kp, r.vp, hkv, d ** -0.5, query_lens, lens,
                              torch.tensor(slots, dtype=torch.int64, device="cuda"), slopes_t, "int4")
    torch.cuda.synchronize()
    at = 0
    for i, n in enumerate(query_lens):
        limit = np.arange(cached[i], lens[i]) + 1
        want = S.attention(q_host[at:at + n], k[i], v[i], d ** -0.5, limit, slopes)
        bound = 2.0 ** -10 + 2.0 ** -11
        if v_mul != 1.0:
            bound = 2.0 ** -8  # values beyond the fp16 range are carried as bfloat16: half a step is 2^-8 of them
        v_max = np.abs(v[i]).max() if n else 0.0
        check(out32[at:at + n].double().cpu().numpy(), want, v_max, 0.0, bound)
        check(out16[at:at + n].double().cpu().numpy(), want, v_max, torch.finfo(q.dtype).eps, bound)
        at += n


@pytest.mark.parametrize("hq,hkv", [(32, 8), (8, 8), (8, 1), (15, 5), (28, 4), (40, 2), (16, 1)])
def test_prompt_heads(env, hq, hkv):
    prompt_case(env, hq, [1, 33, 130], [0, 0, 70], hq, hkv)


@pytest.mark.parametrize("d", [64, 80, 96, 112, 128, 256])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_prompt_head_sizes(env, d, dtype):
    prompt_case(env, d, [47, 1, 65], [0, 31, 200], 8, 2, d, dtype)


def test_prompt_alibi(env):
    prompt_case(env, 1, [100, 3], [0, 400], 16, 4, alibi=True)
    prompt_case(env, 2, [100, 3], [0, 400], 6, 6, 80, "fp16", alibi=True)


def test_prompt_without_tokens_and_behind_a_long_prefix(env):
    prompt_case(env, 3, [0, 5, 0], [10, 5000, 0], 32, 8)


def test_prompt_values_beyond_the_fp16_range(env):
    prompt_case(env, 4, [70], [20], 8, 2, v_mul=1e6)


def test_prompt_scales_from_128_on(env):
    prompt_case(env, 6, [70, 40], [20, 0], 8, 2, v_mul=1e3)
    prompt_case(env, 7, [40], [0], 8, 2, dtype="fp16", v_mul=1e3)


@pytest.mark.parametrize("kind", ["bf16", "int4"])
@pytest.mark.parametrize("column", [0, 1, 2, 3, 6, 61, 127])
def test_prompt_one_value_beyond_the_fp16_range(env, kind, column):
    """A single value of V, in whichever column it lies."""
    torch, ops = env
    rng = np.random.default_rng(column)
    n, hq, hkv, d = 50, 4, 2, 128
    k, v = S.to_bf16(rng.standard_normal((n, hkv, d))), S.to_bf16(rng.standard_normal((n, hkv, d)))
    v[7, 1, column] = S.to_bf16(np.float64(3e5))
    r = S.Ranges(1, n, S.row_bytes(hkv, d) if kind == "int4" else 2 * hkv * d)
    for x, cache in ((k, r.k), (v, r.v)):
        if kind == "int4":
            codes = S.quantise(x)
            x[:] = S.values(*codes)
            cache[0] = torch.from_numpy(S.pack(*codes)).cuda()
        else:
            cache[0] = torch.from_numpy(S.bf16_bits(x).reshape(n, -1).view(np.uint8)).cuda()
    q, q_host = S.as_type(rng.standard_normal((n, hq, d)), torch.bfloat16)
    out = torch.full((n, hq, d), 55.0, device="cuda")
    ops.prefill_attention(out, q, r.kp, r.vp, hkv, d ** -0.5, [n], [n], torch.tensor([0], device="cuda"), None,
                          "int4" if kind == "int4" else "auto")
    torch.cuda.synchronize()
    want = S.attention(q_host, k, v, d ** -0.5, np.arange(n) + 1)
    # (carried as bfloat16: half a step is 2^-8 of a value; the weights' own rounding a fraction of that)
    check(out.double().cpu().numpy(), want, np.abs(v).max(), 0.0, 2.0 ** -8)


@pytest.mark.parametrize("side", ["k", "v"])
def test_prompt_a_row_that_is_not_finite_stays_with_the_tokens_that_see_it(env, side):
    torch, ops = env
    rng = np.random.default_rng(31)
    query_lens, cached, hq, hkv, d, bad = [90, 50], [0, 40], 8, 2, 128, 61
    lens = [a + c for a, c in zip(query_lens, cached)]
    r, k, v = filled(rng, lens, hkv, d, [1, 0])
    cache = r.k if side == "k" else r.v
    cache[0, bad, hkv * d // 2 + 4:hkv * d // 2 + 8] = torch.tensor([0xC0, 0x7F, 0xC0, 0x7F], dtype=torch.uint8)  # head 1
    q, q_host = S.as_type(rng.standard_normal((sum(query_lens), hq, d)), torch.bfloat16)
    out = torch.full((sum(query_lens), hq, d), 55.0, device="cuda")
    ops.prefill_attention(out, q, r.kp, r.vp, hkv, d ** -0.5, query_lens, lens, torch.tensor([1, 0], device="cuda"), None, "int4")
    out = out.double().cpu().numpy()
    sees = bad - cached[1]  # the first token of the second sequence that sees the row
    assert np.isnan(out[90 + sees:, 4:]).all()
    for i, at in ((0, 0), (1, 90)):
        want = S.attention(q_host[at:at + query_lens[i]], k[i], v[i], d ** -0.5, np.arange(cached[i], lens[i]) + 1)
        got = out[at:at + query_lens[i]]
        v_max = np.abs(v[i]).max()
        # (the tokens before it may have been computed with bfloat16 values: half a step is 2^-8 of a value)
        check(got[:, :4], want[:, :4], v_max, 0.0, 2.0 ** -8)
        check(got[:sees if i else None, 4:], want[:sees if i else None, 4:], v_max, 0.0, 2.0 ** -8)


# ------------------------------------------------------------------------------------------------ the paths
def test_backend_engine_and_step_plan_on_an_int4_cache(env, gpu_pool):
    """Prompts and two decode steps through VTensorImpl over a CacheEngine with kv_cache_dtype="int4", a swap in
    between, then a DecodeStepPlan: every result against attention over the rows as they read back."""
    torch, ops = env
    from glake_amd.attention.backends.vtensor import VTensorImpl
    from glake_amd.worker.cache_engine import CacheEngine
    from glake_amd.worker.step import DecodeStepPlan, kv_row_bytes, prepare_step

    rng = np.random.default_rng(20)
    hq, hkv, d, lens = 8, 2, 128, [37, 300]
    eng = CacheEngine(1, hkv, d, torch.bfloat16, 3, 4096, swap_space_bytes=1 << 20, kv_cache_dtype="int4")
    assert eng.token_size == kv_row_bytes(hkv, d, "int4") == S.row_bytes(hkv, d)
    impl = VTensorImpl(hq, d, d ** -0.5, hkv, kv_cache_dtype="int4")
    slots = [2, 0]
    rows = [[], []]  # K and V of each sequence, as quantised

    def new_rows(n):
        k, kh = S.as_type(S.model_values(rng, (n, hkv, d)), torch.bfloat16)
        v, vh = S.as_type(S.model_values(rng, (n, hkv, d)), torch.bfloat16)
        return k, v, S.values(*S.quantise(kh)), S.values(*S.quantise(vh))

    def step(n_new, prompt):
        k, v, kh, vh = new_rows(sum(n_new))
        at = 0
        for i, n in enumerate(n_new):
            rows[i].append((kh[at:at + n], vh[at:at + n]))
            at += n
        now = [sum(len(x[0]) for x in rows[i]) for i in range(2)]
        q, qh = S.as_type(rng.standard_normal((sum(n_new), hq, d)), torch.bfloat16)
        meta = S.step_metadata(eng, slots, now, prompt)
        prepare_step(meta, eng.gpu_cache)
        out = impl.forward(q.view(-1, hq * d), k.view(-1, hkv * d), v.view(-1, hkv * d), *eng.gpu_cache[0], meta)
        compare(out.view(-1, hq, d), qh, n_new, now, 2.0 ** -10 + 2.0 ** -11)

    def compare(out, qh, n_new, now, bound):
        at = 0
        for i, n in enumerate(n_new):
            kk, vv = (np.concatenate([x[s] for x in rows[i]]) for s in range(2))
            want = S.attention(qh[at:at + n], kk, vv, d ** -0.5, np.arange(now[i] - n, now[i]) + 1)
            check(out[at:at + n].double().cpu().numpy(), want, np.abs(vv).max(), 2.0 ** -7, bound)
            at += n

    step(lens, True)
    step([1, 1], False)
    moved = eng.swap_out(slots)
    assert moved == 2 * sum(n + 1 for n in lens) * eng.token_size
    eng.swap_in(slots)
    step([1, 1], False)
    plan = DecodeStepPlan([eng.vmm_kvcache_segment[s] for s in slots], slots, eng.k_cache_ptr[0], eng.v_cache_ptr[0], hq, hkv,
                          d, d ** -0.5, kv_cache_dtype="int4")
    for _ in range(3):
        k, v, kh, vh = new_rows(2)
        for i in range(2):
            rows[i].append((kh[i:i + 1], vh[i:i + 1]))
        q, qh = S.as_type(rng.standard_normal((2, hq, d)), torch.bfloat16)
        out = torch.empty_like(q)
        longest = plan.run(q, k, v, out)
        now = [sum(len(x[0]) for x in rows[i]) for i in range(2)]
        assert longest == max(now)
        compare(out, qh, [1, 1], now, 2.0 ** -12)
    eng.close()
