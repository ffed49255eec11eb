"""The 4-bit cache, the attention weights and the eviction at the edges of what they take: values, queries, lengths and slots
that the ordinary cases do not meet, on the GPU against float64 forms on the host.  Each tolerance is derived where it stands."""
import numpy as np
import pytest

import small_cache as S

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch

    from glake_amd import _custom_ops as ops

    assert torch.cuda.is_available()
    torch.cuda.set_device(0)
    return torch, ops


def i32(values):
    import torch

    return torch.tensor(values, dtype=torch.int32, device="cuda")


def i64(values):
    import torch

    return torch.tensor(values, dtype=torch.int64, device="cuda")


def put(cache, slot, codes, scale, zero):
    """Rows with these codes [n, hkv, d], scales and zeros (numbers, or [n, hkv, 1]) into a slot, from its first row on."""
    import torch

    n, hkv = codes.shape[:2]
    pair = [np.broadcast_to(np.asarray(x, np.float64), (n, hkv, 1)) for x in (scale, zero)]
    cache[slot, :n] = torch.from_numpy(S.pack(codes.astype(np.uint8), *pair)).cuda()


# ------------------------------------------------------------------------------------------------ how weights are carried
@pytest.mark.parametrize("hq,d", [(8, 128), (16, 128), (4, 80), (13, 256)])
def test_decode_weights_are_not_cut_off(env, hq, d):
    """Every value is 15, so the result is 15 whatever the weights are, up to how p s is carried: rounded twice to bfloat16
    it is off by 2^-18 of itself at most (half a step of 2^-8, twice, and the tail's own), the sums of 31 rows (two products
    each) by 62 * 2^-24 < 2^-18, the normaliser and the quotient by less than half of that.  The weight of all rows but the
    first is one that loses 0.9 * 2^-15 of itself when head and tail are cut off instead."""
    torch, ops = env
    n = 31
    p = 0.5 * (1 + 2.0 ** -8 * (2 - 0.1 * 2.0 ** -7))
    r = S.Ranges(1, n, S.row_bytes(1, d))
    put(r.k, 0, np.zeros((n, 1, d)), 0.0, np.where(np.arange(n) > 0, -1.0, 0.0)[:, None, None])
    put(r.v, 0, np.full((n, 1, d), 15), 1.0, 0.0)
    q = torch.zeros(1, hq, d, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = 1.0
    out = torch.full((1, hq, d), 55.0, device="cuda")
    ops.paged_attention_v1(out, q, r.kp, r.vp, 1, -np.log(p), i32([n]), 1, n, None, "int4", 1.0, i64([0]))
    err = np.abs(out.double().cpu().numpy() / 15.0 - 1.0)
    assert err.max() <= 2.5 * 2.0 ** -18, f"{err.max() * 2.0 ** 18:.2f} * 2^-18"


# ------------------------------------------------------------------------------------------------ queries far apart
def filled(rng, lens, hkv, d, k_factor=1.0, v_factor=1.0):
    """Ranges with lens[i] rows of sequence i in slot i, and the rows' values."""
    r = S.Ranges(len(lens), max(lens), S.row_bytes(hkv, d))
    k, v = [], []
    for i, n in enumerate(lens):
        for values, cache, f in ((k, r.k, k_factor), (v, r.v, v_factor)):
            x = S.quantise(S.to_bf16(f * S.model_values(rng, (n, hkv, d))))
            values.append(S.values(*x))
            put(cache, i, *x)
    return r, k, v


@pytest.mark.parametrize("value", [2.0 ** 26, 1e30])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (16, 1, 80), (8, 8, 64), (6, 2, 256), (40, 2, 112)])
def test_a_large_query_stays_with_its_head(env, value, hq, hkv, d):
    """One large finite number in one head of one token: decode, prompts and weights are, everywhere else, as they are
    without it, and that head attends to the one row that is largest there.  Tolerances as for ordinary values: 2^-12 of the
    largest value (decode), 2^-10 + 2^-11 (prompts), 2^-12 of a weight (a sum over the heads of a kv head)."""
    torch, ops = env
    rng = np.random.default_rng(40)
    lens, query_lens = [70, 90], [40, 33]
    r, k, v = filled(rng, lens, hkv, d)
    scale, slots = d ** -0.5, i64([0, 1])
    v_max = [np.abs(x).max() for x in v]

    x = rng.standard_normal((2, hq, d))
    x[1, 1, 5] = value
    q, qh = S.as_type(x, torch.bfloat16)
    out = torch.empty(2, hq, d, device="cuda")
    ops.paged_attention_v1(out, q, r.kp, r.vp, hkv, scale, i32(lens), 1, 90, None, "int4", 1.0, slots)
    weights = torch.zeros(2, hkv, 90, device="cuda")
    ops.accumulate_attention_weights(weights, q, r.kp, hkv, scale, i32(lens), 90, slots, None, "int4")
    for i, n in enumerate(lens):
        want = S.attention(qh[i:i + 1], k[i], v[i], scale)[0]
        assert (np.abs(out[i].double().cpu().numpy() - want) <= 2.0 ** -12 * v_max[i]).all()
        p = S.softmax(qh[i:i + 1], k[i], scale)[0].reshape(hkv, hq // hkv, n).sum(1)
        assert (np.abs(weights[i, :, :n].double().cpu().numpy() - p) <= 2.0 ** -12 * p + 1e-30).all()

    x = rng.standard_normal((sum(query_lens), hq, d))
    x[query_lens[0] + 9, 1, 5] = value
    q, qh = S.as_type(x, torch.bfloat16)
    out = torch.empty(q.shape, device="cuda")
    ops.prefill_attention(out, q, r.kp, r.vp, hkv, scale, query_lens, lens, slots, None, "int4")
    at = 0
    for i, n in enumerate(query_lens):
        want = S.attention(qh[at:at + n], k[i], v[i], scale, np.arange(lens[i] - n, lens[i]) + 1)
        assert (np.abs(out[at:at + n].double().cpu().numpy() - want) <= (2.0 ** -10 + 2.0 ** -11) * v_max[i]).all()
        at += n


# ------------------------------------------------------------------------------------------------ large and small numbers
def attend(ops, r, q, hkv, lens, out_dtype=None):
    import torch

    b, hq, d = q.shape
    out = torch.full(q.shape, 55.0, dtype=out_dtype or torch.float32, device="cuda")
    ops.paged_attention_v1(out, q, r.kp, r.vp, hkv, d ** -0.5, i32(lens), 1, max(lens), None, "int4", 1.0, i64(list(range(b))))
    return out


@pytest.mark.parametrize("lens", [[200, 33], [9001]])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (16, 1, 80), (8, 8, 256)])
@pytest.mark.parametrize("factor", [1e18, 1e20, 1e30, 1e37])
def test_decode_of_large_finite_values(env, lens, hq, hkv, d, factor):
    """Results of spans that hold a whole sequence (200, 33 rows) and of several spans (9001).  The tolerance of ordinary
    values, relative to the largest value."""
    torch, ops = env
    rng = np.random.default_rng(41)
    r, k, v = filled(rng, lens, hkv, d, v_factor=factor)
    q, qh = S.as_type(rng.standard_normal((len(lens), hq, d)), torch.bfloat16)
    got, rounded = attend(ops, r, q, hkv, lens), attend(ops, r, q, hkv, lens, torch.bfloat16)
    for i in range(len(lens)):
        want = S.attention(qh[i:i + 1], k[i], v[i], d ** -0.5)[0]
        assert (np.abs(got[i].double().cpu().numpy() - want) <= 2.0 ** -12 * np.abs(v[i]).max()).all()
    assert torch.equal(got.bfloat16(), rounded)



@pytest.mark.parametrize("hq,hkv,d", [(40, 2, 128), (71, 1, 64), (8, 8, 96)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_decode_of_large_values_with_alibi_and_many_heads(env, dtype, hq, hkv, d):
    torch, ops = env
    rng = np.random.default_rng(46)
    lens = [500, 1, 0, 257]
    r, k, v = filled(rng, [max(n, 1) for n in lens], hkv, d, v_factor=1e32)
    q, qh = S.as_type(rng.standard_normal((4, hq, d)), torch.float16 if dtype == "fp16" else torch.bfloat16)
    slopes = np.abs(rng.standard_normal(hq)).astype(np.float32) * 0.05
    out = torch.full(q.shape, 55.0, device="cuda")
    ops.paged_attention_v1(out, q, r.kp, r.vp, hkv, d ** -0.5, i32(lens), 1, 900, torch.from_numpy(slopes).cuda(), "int4", 1.0,
                           i64([0, 1, 2, 3]))
    for i, n in enumerate(lens):
        if n == 0:
            assert (out[i] == 0).all()
            continue
        want = S.attention(qh[i:i + 1], k[i][:n], v[i][:n], d ** -0.5, [n], slopes)[0]
        assert (np.abs(out[i].double().cpu().numpy() - want) <= 2.0 ** -12 * np.abs(v[i]).max()).all()


@pytest.mark.parametrize("n", [100, 7000])
def test_decode_of_one_large_row_without_weight(env, n):
    """A row of 1e25 that no query pays anything to (2^-200), among ordinary ones: the result is theirs."""
    torch, ops = env
    rng = np.random.default_rng(42)
    hq, hkv, d, at = 8, 2, 128, 77
    r, k, v = filled(rng, [n], hkv, d)
    k[0][at], v[0][at] = 0.0, 0.0
    big = S.quantise(S.to_bf16(1e25 * rng.standard_normal((1, hkv, d))))
    r.v[0, at] = torch.from_numpy(S.pack(*big)).cuda()[0]
    low = S.quantise(np.full((1, hkv, d), -1600.0))  # (queries are positive: far below every other row)
    r.k[0, at] = torch.from_numpy(S.pack(*low)).cuda()[0]
    q, qh = S.as_type(np.abs(rng.standard_normal((1, hq, d))) * 0.2, torch.bfloat16)
    k[0][at] = -1600.0
    got = attend(ops, r, q, hkv, [n])
    want = S.attention(qh, k[0], v[0], d ** -0.5)[0]
    assert (np.abs(got[0].double().cpu().numpy() - want) <= 2.0 ** -12 * np.abs(v[0]).max()).all()


@pytest.mark.parametrize("factor", [1e30, 1e-30])
def test_large_keys_of_small_queries_and_the_other_way_round(env, factor):
    """Keys and queries whose products are ordinary numbers: decode, prompt and weights as for ordinary ones."""
    torch, ops = env
    rng = np.random.default_rng(43)
    lens, hq, hkv, d = [300, 90], 8, 2, 128
    r, k, v = filled(rng, lens, hkv, d, k_factor=factor)
    q, qh = S.as_type(rng.standard_normal((sum(lens), hq, d)) / factor, torch.bfloat16)
    out = torch.empty(q.shape, device="cuda")
    ops.prefill_attention(out, q, r.kp, r.vp, hkv, d ** -0.5, lens, lens, i64([0, 1]), None, "int4")
    ends = [lens[0] - 1, sum(lens) - 1]
    last = attend(ops, r, q[ends], hkv, lens)
    weights = torch.zeros(2, hkv, 300, device="cuda")
    ops.accumulate_attention_weights(weights, q[ends], r.kp, hkv, d ** -0.5, i32(lens), 300, i64([0, 1]), None, "int4")
    at = 0
    for i, n in enumerate(lens):
        want = S.attention(qh[at:at + n], k[i], v[i], d ** -0.5, np.arange(n) + 1)
        top = np.abs(v[i]).max()
        assert (np.abs(out[at:at + n].double().cpu().numpy() - want) <= (2.0 ** -10 + 2.0 ** -11) * top).all()
        assert (np.abs(last[i].double().cpu().numpy() - want[-1]) <= 2.0 ** -12 * top).all()
        p = S.softmax(qh[ends[i]:ends[i] + 1], k[i], d ** -0.5)[0].reshape(hkv, hq // hkv, n).sum(1)
        assert (np.abs(weights[i, :, :n].double().cpu().numpy() - p) <= 2.0 ** -12 * p).all()
        at += n


@pytest.mark.parametrize("factor", [1e-6, 1e-9, 1e-15, 1e-18])
def test_decode_of_small_values(env, factor):
    """Down to 1e-18 values keep the relative tolerance of ordinary ones."""
    torch, ops = env
    rng = np.random.default_rng(44)
    lens, hq, hkv, d = [200, 1033], 8, 2, 128
    r, k, v = filled(rng, lens, hkv, d, v_factor=factor)
    q, qh = S.as_type(rng.standard_normal((2, hq, d)) * 1.5, torch.bfloat16)
    got = attend(ops, r, q, hkv, lens)
    for i in range(2):
        want = S.attention(qh[i:i + 1], k[i], v[i], d ** -0.5)[0]
        assert (np.abs(got[i].double().cpu().numpy() - want) <= 2.0 ** -12 * np.abs(v[i]).max()).all()


@pytest.mark.parametrize("factor", [1e6, 1e30, 1e37])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_prompt_of_large_finite_values(env, dtype, factor):
    """Values that a unit's second pass holds as bfloat16: half a step, 2^-8 of the largest value at most."""
    torch, ops = env
    rng = np.random.default_rng(45)
    lens, hq, hkv, d = [130, 60], 8, 2, 128
    r, k, v = filled(rng, lens, hkv, d, v_factor=factor)
    q, qh = S.as_type(rng.standard_normal((sum(lens), hq, d)) * 3, torch.float16 if dtype == "fp16" else torch.bfloat16)
    out = torch.empty(q.shape, device="cuda")
    ops.prefill_attention(out, q, r.kp, r.vp, hkv, d ** -0.5, lens, lens, i64([0, 1]), None, "int4")
    at = 0
    for i, n in enumerate(lens):
        want = S.attention(qh[at:at + n], k[i], v[i], d ** -0.5, np.arange(n) + 1)
        assert (np.abs(out[at:at + n].double().cpu().numpy() - want) <= 2.0 ** -8 * np.abs(v[i]).max()).all()
        at += n


# ------------------------------------------------------------------------------------------------ slots
@pytest.mark.parametrize("alias", [False, True])
@pytest.mark.parametrize("kind", ["auto", "int4"])
def test_evict_leaves_sequences_of_foreign_slots_alone(env, kind, alias):
    """Slots outside the weights (slot 3 has ranges but no weights) and outside everything: rows, weights and lengths stay."""
    torch, ops = env
    rng = np.random.default_rng(50)
    hkv, d, keep, recent, lens, slots = 2, 64, 40, 10, [90, 60, 100, 30, 75], [1, 3, -1, 1 << 40, 0]
    r = S.Ranges(4, 100, S.row_bytes(hkv, d) if kind == "int4" else hkv * d * 2)
    for t in (r.k, r.v):
        t.copy_(torch.from_numpy(rng.integers(0, 256, t.shape, dtype=np.uint8)).cuda())
    w = torch.rand(2, hkv, 100, device="cuda")
    before = [x.clone() for x in (r.k, r.v, w)]
    lens_t = i32(lens)
    new = lens_t if alias else torch.full_like(lens_t, -7)
    ops.evict_rows(r.kp, r.vp, w, lens_t, new, keep, recent, 100, i64(slots), hkv, d, kind)
    assert new.tolist() == [40, 60, 100, 30, 40]
    for a, b in zip((r.k, r.v), before):
        assert torch.equal(a[2:], b[2:]) and not torch.equal(a[0, :40], b[0, :40]) and not torch.equal(a[1, :40], b[1, :40])
    assert (w[1, :, 40:90] == 0).all() and (w[0, :, 40:75] == 0).all() and torch.equal(w[:, :, 90:], before[2][:, :, 90:])


def test_empty_sequences_may_have_any_slot(env):
    """Padded entries (length 0) whose slots lie in no table, below and above 256 sequences: zeros, and nobody else notices;
    a step's write skips them by their byte offset, the weights by their length."""
    torch, ops = env
    rng = np.random.default_rng(51)
    hq, hkv, d, b = 8, 2, 128, 300
    lens = [0] * b
    for i, n in ((0, 40), (7, 1), (255, 90), (256, 33), (299, 5)):
        lens[i] = n
    held = [n for n in lens if n]
    r, k, v = filled(rng, held, hkv, d)
    slots, at = [], 0
    for i, n in enumerate(lens):
        slots.append(at if n else [-1, 1 << 40, -(1 << 40)][i % 3])
        at += n > 0
    q, qh = S.as_type(rng.standard_normal((b, hq, d)), torch.bfloat16)
    out = torch.full((b, hq, d), 55.0, device="cuda")
    ops.paged_attention_v1(out, q, r.kp, r.vp, hkv, d ** -0.5, i32(lens), 1, 100, None, "int4", 1.0, i64(slots))
    weights = torch.zeros(len(held), hkv, 100, device="cuda")
    ops.accumulate_attention_weights(weights, q, r.kp, hkv, d ** -0.5, i32(lens), 100, i64(slots), None, "int4")
    at = 0
    for i, n in enumerate(lens):
        if not n:
            assert (out[i] == 0).all()
            continue
        want = S.attention(qh[i:i + 1], k[at], v[at], d ** -0.5)[0]
        assert (np.abs(out[i].double().cpu().numpy() - want) <= 2.0 ** -12 * np.abs(v[at]).max()).all()
        p = S.softmax(qh[i:i + 1], k[at], d ** -0.5)[0].reshape(hkv, hq // hkv, n).sum(1)
        assert (np.abs(weights[at, :, :n].double().cpu().numpy() - p) <= 2.0 ** -12 * p).all() and (weights[at, :, n:] == 0).all()
        at += 1
    key = torch.zeros(b, hkv, d, dtype=torch.bfloat16, device="cuda")
    before = r.k.clone()
    ops.reshape_and_cache(key, key, r.kp, r.vp, i64([-1] * b), i64([-1] * b), None, None, 1, hkv, d, "int4")
    assert torch.equal(r.k, before)


def test_decode_of_a_batch_that_takes_several_launches(env):
    """A loose bound on the lengths and many chunks of kv heads: the units of all sequences together pass 32 bits, so the
    batch runs in parts."""
    torch, ops = env
    rng = np.random.default_rng(52)
    hkv, d, b = 37, 64, 25
    lens = [int(n) for n in rng.integers(0, 60, b)]
    r, k, v = filled(rng, lens, hkv, d)
    q, qh = S.as_type(rng.standard_normal((b, hkv, d)), torch.bfloat16)
    out = torch.full(q.shape, 55.0, device="cuda")
    ops.paged_attention_v1(out, q, r.kp, r.vp, hkv, d ** -0.5, i32(lens), 1, 100_000_000, None, "int4", 1.0, i64(list(range(b))))
    for i, n in enumerate(lens):
        want = S.attention(qh[i:i + 1], k[i], v[i], d ** -0.5)[0] if n else np.zeros((hkv, d))
        top = np.abs(v[i]).max() if n else 0.0
        assert (np.abs(out[i].double().cpu().numpy() - want) <= 2.0 ** -12 * top).all()


# ------------------------------------------------------------------------------------------------ the attention weights
@pytest.mark.parametrize("kind", ["auto", "fp8", "int4"])
@pytest.mark.parametrize("fit", [1, 2, 4])
def test_weights_through_a_workspace_of_a_few_sequences(env, kind, fit):
    """A workspace that holds some of the batch's sequences: the parts run one after the other through it, bit for bit as all
    at once."""
    import ctypes as C

    from glake_amd import _C

    torch, _ = env
    rng = np.random.default_rng(60)
    lens, hq, hkv, d = [300, 1, 0, 129, 700, 64, 65], 8, 2, 128
    b, most = len(lens), max(lens)
    if kind == "int4":
        r, _, _ = filled(rng, [max(n, 1) for n in lens], hkv, d)
    else:
        r = S.Ranges(b, most, hkv * d * (1 if kind == "fp8" else 2))
        x = torch.from_numpy(rng.standard_normal((b, most, hkv * d)).astype(np.float32))
        r.k[:] = x.to(torch.float8_e4m3fn if kind == "fp8" else torch.bfloat16).view(torch.uint8).view(r.k.shape).cuda()
    q = torch.from_numpy(rng.standard_normal((b, hq, d)).astype(np.float32)).bfloat16().cuda()
    lib = _C.lib()
    slots, lens_t = i64(list(reversed(range(b)))), i32(list(reversed(lens)))
    one = lib.vtkv_accumulate_attention_weights_workspace_bytes(1, hq, most)
    got = []
    for nbytes in (one * b, one * fit + 16):
        w = torch.zeros(b, hkv, most, device="cuda")
        ws = torch.full((nbytes,), 0xFF, dtype=torch.uint8, device="cuda")
        p = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
        _C.check(lib.vtkv_accumulate_attention_weights(
            p(w), w.stride(0), w.stride(1), b, p(q), p(r.kp), p(slots), p(lens_t), b, hq, hkv, d, hq * d, d ** -0.5, most, None,
            _C.BF16, {"auto": _C.BF16, "fp8": _C.FP8_E4M3, "int4": _C.INT4}[kind], 1.0, p(ws), nbytes,
            C.c_void_p(torch.cuda.current_stream().cuda_stream)))
        got.append(w)
    assert torch.equal(*got)
    sums = got[0].double().sum(-1).cpu().numpy()  # (each query head pays 1 in all: 700 rows within 2^-12 of themselves)
    assert (np.abs(sums - np.array([hq // hkv if n else 0 for n in lens])[:, None]) <= hq // hkv * 2.0 ** -11).all()


# ------------------------------------------------------------------------------------------------ a bounded cache, served
@pytest.mark.parametrize("kind", ["auto", "int4"])
@pytest.mark.parametrize("path", ["plan", "backend"])
def test_a_bounded_cache_on_the_engine(env, gpu_pool, kind, path):
    """Prompts through the backend, then decode steps through a DecodeStepPlan or the backend over a CacheEngine's ranges,
    weights after each step, evictions when a sequence is four rows over its budget.  The lengths that the calls take are
    numbers of rows, not of tokens, from the first eviction on."""
    torch, ops = env
    from glake_amd.attention.backends.vtensor import VTensorImpl
    from glake_amd.worker.cache_engine import CacheEngine
    from glake_amd.worker.step import DecodeStepPlan, prepare_step

    rng = np.random.default_rng(61)
    hq, hkv, d, keep, recent, slack, room = 8, 2, 128, 40, 12, 4, 64
    slots, lens = [2, 0], [39, 30]
    eng = CacheEngine(1, hkv, d, torch.bfloat16, 3, 4096, kv_cache_dtype=kind)
    impl = VTensorImpl(hq, d, d ** -0.5, hkv, kv_cache_dtype=kind)
    segments = [eng.vmm_kvcache_segment[s] for s in slots]
    tables = eng.k_cache_ptr[0], eng.v_cache_ptr[0]
    weights = torch.zeros(3, hkv, room, device="cuda")
    held = [[[np.zeros((0, d))] * hkv for _ in range(2)] for _ in slots]  # [sequence][K, V][head] -> rows

    def batch(n_new):
        out = []
        for _ in range(2):
            t, h = S.as_type(S.model_values(rng, (sum(n_new), hkv, d)), torch.bfloat16)
            out.append((t, S.values(*S.quantise(h)) if kind == "int4" else h))
        at = 0
        for i, n in enumerate(n_new):
            for side in range(2):
                held[i][side] = [np.concatenate([x, out[side][1][at:at + n, h]]) for h, x in enumerate(held[i][side])]
            at += n
        q, qh = S.as_type(rng.standard_normal((sum(n_new), hq, d)), torch.bfloat16)
        return q, qh, out[0][0], out[1][0]

    def through_backend(q, k, v, rows, prompt):
        meta = S.step_metadata(eng, slots, rows, prompt)
        prepare_step(meta, eng.gpu_cache)
        return impl.forward(q.view(-1, hq * d), k.view(-1, hkv * d), v.view(-1, hkv * d), *eng.gpu_cache[0], meta).view(-1, hq, d)

    def compare(out, qh, n_new, bound):
        at = 0
        for i, n in enumerate(n_new):
            kk, vv = (np.stack(held[i][s], 1) for s in range(2))
            want = S.attention(qh[at:at + n], kk, vv, d ** -0.5, np.arange(len(kk) - n, len(kk)) + 1)
            err = np.abs(out[at:at + n].double().cpu().numpy() - want)
            assert (err <= bound * np.abs(vv).max() + 2.0 ** -8 * np.abs(want)).all()
            at += n

    q, qh, k, v = batch(lens)
    compare(through_backend(q, k, v, lens, True), qh, lens, 2.0 ** -10 + 2.0 ** -11)
    plan = DecodeStepPlan(segments, slots, *tables, hq, hkv, d, d ** -0.5, kv_cache_dtype=kind)
    evictions = 0
    for _ in range(30):
        q, qh, k, v = batch([1, 1])
        rows = [len(held[i][0][0]) for i in range(2)]
        if path == "plan":
            out = torch.empty_like(q)
            assert plan.run(q, k, v, out) == max(rows) and plan.seq_lens.tolist() == rows
        else:
            out = through_backend(q, k, v, rows, False)
        compare(out, qh, [1, 1], 2.0 ** -12)
        lens_t = i32(rows)
        ops.accumulate_attention_weights(weights, q, tables[0], hkv, d ** -0.5, lens_t, max(rows), i64(slots), None, kind)
        if max(rows) < keep + slack:
            continue
        evictions += 1
        before = weights.double().cpu().numpy()
        ops.evict_rows(*tables, weights, lens_t, lens_t, keep, recent, max(rows), i64(slots), hkv, d, kind)
        for i, n in enumerate(lens_t.tolist()):
            assert n == min(rows[i], keep)
            segments[i].set_used_size(n * eng.token_size)
            for h in range(hkv):
                src = S.evicted_sources(before[slots[i], h, :rows[i]], rows[i], keep, recent)
                for side in range(2):
                    held[i][side][h] = held[i][side][h][src]
    assert evictions >= 4 and all(s.used_size == len(held[i][0][0]) * eng.token_size for i, s in enumerate(segments))
    torch.cuda.synchronize()
    eng.close()
