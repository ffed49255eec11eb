"""Attention weight per cached row and the eviction of rows, on the GPU against float64 forms on the host.

Tolerance of the weights: a logit is off by less than 2^-14 (fp32 sums of at most 256 products whose magnitudes add up
to less than 2^9), so a softmax weight by 2^-13 of itself and the same again for its sum; what is added is therefore
within 2^-12 of itself, and the accumulator rounds at 2^-24 of its value per query head.  An eviction moves bytes: exact."""
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


def rows_of(rng, kind, n, hkv, d):
    """n cached rows of a kind of cache: (bytes [n, row bytes], values [n, hkv, d] float64)."""
    import torch

    if n == 0:  # (torch gives an empty tensor strides that its views refuse)
        raw, v = rows_of(rng, kind, 1, hkv, d)
        return raw[:0], v[:0]
    x = S.model_values(rng, (n, hkv, d))
    if kind == "int4":
        q = S.quantise(S.to_bf16(x))
        return S.pack(*q), S.values(*q)
    if kind == "fp8":
        t = torch.from_numpy(x.astype(np.float32)).to(torch.float8_e4m3fn)
        return t.view(torch.uint8).reshape(n, hkv * d).numpy(), t.double().numpy() * 0.75
    t = torch.from_numpy(x.astype(np.float32)).to({"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[kind])
    return t.view(torch.uint8).reshape(n, hkv * d * t.element_size()).numpy(), t.double().numpy()


def row_size(kind, hkv, d):
    return S.row_bytes(hkv, d) if kind == "int4" else hkv * d * {"fp8": 1, "fp32": 4}.get(kind, 2)


# ------------------------------------------------------------------------------------------------ weights
def weights_case(env, seed, lens, hq, hkv, d=128, kind="bf16", alibi=False, q_scale=1.5, extra=0):
    torch, ops = env
    rng = np.random.default_rng(seed)
    b = len(lens)
    slots = rng.permutation(b + 2)[:b]
    r = S.Ranges(b + 2, max(lens) + 1, row_size(kind, hkv, d))
    k = []
    for n, slot in zip(lens, slots):
        raw, v = rows_of(rng, kind, n, hkv, d)
        r.k[slot, :n] = torch.from_numpy(raw.copy()).cuda()
        k.append(v)
    dtype = torch.float16 if kind == "fp16" else torch.bfloat16
    q, q_host = S.as_type(rng.standard_normal((b, hq, d)) * q_scale, dtype)
    slopes = np.abs(rng.standard_normal(hq)).astype(np.float32) * 0.05 if alibi else None
    room = max(lens) + extra
    wide = torch.rand(b + 2, hkv, room + 7, device="cuda")
    before = wide.double().cpu().numpy()
    weights = wide[:, :, 3:3 + room]
    ops.accumulate_attention_weights(
        weights, q, r.kp, hkv, d ** -0.5, torch.tensor(lens, dtype=torch.int32, device="cuda"), room,
        torch.tensor(slots, dtype=torch.int64, device="cuda"), None if slopes is None else torch.from_numpy(slopes).cuda(),
        {"int4": "int4", "fp8": "fp8"}.get(kind, "auto"), 0.75 if kind == "fp8" else 1.0)
    torch.cuda.synchronize()
    got = wide.double().cpu().numpy()
    want, added = before.copy(), np.zeros_like(before)
    for i, n in enumerate(lens):
        if n:
            p = S.softmax(q_host[i:i + 1], k[i], d ** -0.5, [n], slopes)[0]
            added[slots[i], :, 3:3 + n] = p.reshape(hkv, hq // hkv, n).sum(1)
    want += added
    touched = added > 0
    assert np.array_equal(got[~touched], before[~touched])  # other slots, rows behind the sequences
    lim = 2.0 ** -12 * added + 2.0 ** -23 * want * max(1, hq // hkv)
    assert (np.abs(got - want) <= lim)[touched].all(), f"{(np.abs(got - want)[touched] / lim[touched]).max():.2f} of the bound"


@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp8", "int4"])
@pytest.mark.parametrize("hq,hkv", [(32, 8), (8, 8), (8, 1), (15, 5), (48, 4), (71, 1), (40, 2)])
def test_weights_heads(env, kind, hq, hkv):
    weights_case(env, hq, [1, 16, 63, 64, 65, 300, 1025], hq, hkv, kind=kind)


@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp8", "int4"])
@pytest.mark.parametrize("d", [64, 80, 96, 112, 256])
def test_weights_head_sizes(env, kind, d):
    weights_case(env, d, [1, 130, 517], 12, 3, d, kind)


@pytest.mark.parametrize("kind", ["bf16", "int4"])
def test_weights_alibi_empty_sequences_and_a_loose_bound(env, kind):
    weights_case(env, 1, [0, 200, 0, 31], 16, 4, kind=kind, alibi=True, extra=900)
    weights_case(env, 2, [0, 0, 1], 4, 2, kind=kind, extra=3)


@pytest.mark.parametrize("kind", ["bf16", "int4"])
def test_weights_large_logits_and_long_sequences(env, kind):
    weights_case(env, 3, [700], 8, 2, kind=kind, q_scale=12.0)
    weights_case(env, 4, [9001, 40], 8, 2, kind=kind)
    weights_case(env, 5, list(np.random.default_rng(1).integers(1, 70, 1100)), 2, 1, 64, kind=kind)


def test_weights_add_up_and_skip_foreign_slots(env):
    torch, ops = env
    rng = np.random.default_rng(6)
    raw, _ = rows_of(rng, "bf16", 50, 2, 64)
    r = S.Ranges(3, 50, row_size("bf16", 2, 64))
    r.k[:] = torch.from_numpy(raw.copy()).cuda()
    q = torch.randn(2, 4, 64, device="cuda").bfloat16()
    weights = torch.zeros(2, 2, 50, device="cuda")
    lens = torch.tensor([50, 50], dtype=torch.int32, device="cuda")
    for _ in range(3):  # slot 2 has ranges but no accumulators
        ops.accumulate_attention_weights(weights, q, r.kp, 2, 0.125, lens, 50, torch.tensor([1, 2], device="cuda"))
    sums = weights.double().sum(-1).cpu().numpy()
    assert np.allclose(sums[1], 6.0, rtol=2.0 ** -11) and (sums[0] == 0).all()  # three steps of two heads each


def test_weights_in_a_graph(env):
    torch, ops = env
    rng = np.random.default_rng(7)
    r = S.Ranges(2, 400, row_size("bf16", 2, 128))
    for s in range(2):
        r.k[s] = torch.from_numpy(rows_of(rng, "bf16", 400, 2, 128)[0].copy()).cuda()
    q = torch.randn(2, 8, 128, device="cuda").bfloat16()
    lens = torch.tensor([400, 100], dtype=torch.int32, device="cuda")
    slots = torch.tensor([1, 0], device="cuda")
    a, b = (torch.zeros(2, 2, 400, device="cuda") for _ in range(2))

    def call(w):
        ops.accumulate_attention_weights(w, q, r.kp, 2, 0.1, lens, 400, slots)

    call(a)
    a.zero_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(b)
    b.zero_()
    for n in ([400, 100], [1, 399], [300, 0]):
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        call(a)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------ eviction
def evict_case(env, seed, lens, keep, recent, hkv=2, d=64, kind="bf16", weights=None, alias=False, extra=0):
    torch, ops = env
    rng = np.random.default_rng(seed)
    b = len(lens)
    slots = rng.permutation(b + 2)[:b]
    rows = max(lens) + 3
    r = S.Ranges(b + 2, rows, row_size(kind, hkv, d))
    for t in (r.k, r.v):
        t.copy_(torch.from_numpy(rng.integers(0, 256, t.shape, dtype=np.uint8)).cuda())
    max_len = max(lens) + extra
    w = rng.random((b + 2, hkv, max_len + 2)).astype(np.float32)
    if weights is not None:
        w = weights(rng, w.shape).astype(np.float32)
    w_t = torch.from_numpy(w).cuda()
    k0, v0 = r.k.cpu().numpy(), r.v.cpu().numpy()
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    new = lens_t if alias else torch.full_like(lens_t, -7)
    model = {"fp32": torch.float32, "fp16": torch.float16}.get(kind, torch.bfloat16)
    ops.evict_rows(r.kp, r.vp, w_t, lens_t, new, keep, recent, max_len, torch.tensor(slots, dtype=torch.int64, device="cuda"),
                   hkv, d, {"int4": "int4", "fp8": "fp8"}.get(kind, "auto"), model)
    torch.cuda.synchronize()
    assert new.tolist() == [min(n, keep) for n in lens]
    k1, v1, w1 = k0.copy(), v0.copy(), w.copy()
    size = row_size(kind, hkv, d)
    for i, n in enumerate(lens):
        for h in range(hkv):
            src = S.evicted_sources(w[slots[i], h], n, keep, recent)
            m = len(src)
            if kind == "int4":
                cols = list(range(h * d // 2, (h + 1) * d // 2)) + [hkv * d // 2 + 4 * h + j for j in range(4)]
            else:
                hb = size // hkv
                cols = list(range(h * hb, (h + 1) * hb))
            for a, a0 in ((k1, k0), (v1, v0)):
                a[slots[i], np.arange(m)[:, None], np.array(cols)] = a0[slots[i]][src][:, cols]
            w1[slots[i], h, :m] = w[slots[i], h, src]
            if n > keep:
                w1[slots[i], h, keep:n] = 0
    assert np.array_equal(w_t.cpu().numpy(), w1, equal_nan=True)
    assert np.array_equal(r.k.cpu().numpy(), k1) and np.array_equal(r.v.cpu().numpy(), v1)


@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32", "fp8", "int4"])
@pytest.mark.parametrize("d", [64, 80, 96, 112, 128, 256])
def test_evict_types_and_head_sizes(env, kind, d):
    evict_case(env, d, [100, 41, 39, 40], 40, 13, 3, d, kind)


@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (64, 0), (64, 64), (64, 63), (300, 200), (1000, 1), (500, 499)])
def test_evict_budgets(env, keep, recent):
    evict_case(env, keep + recent, [keep + 1, keep + 2, 2 * keep + 5, 1, keep, 1500], keep, recent)


@pytest.mark.parametrize("kind", ["bf16", "int4"])
def test_evict_one_row_of_many(env, kind):
    evict_case(env, 3, [2049, 2048, 2049], 2048, 256, 8, 128, kind)


@pytest.mark.parametrize("kind", ["bf16", "int4"])
def test_evict_long_sequences(env, kind):
    evict_case(env, 4, [70001, 33000], 20000, 3000, 2, 64, kind)
    evict_case(env, 5, [40000], 39000, 30000, 1, 64, kind)


def test_evict_equal_weights_keep_the_first(env):
    evict_case(env, 6, [500, 130], 64, 16, weights=lambda rng, s: np.zeros(s))
    evict_case(env, 7, [900, 700], 200, 50, weights=lambda rng, s: rng.integers(0, 3, s))
    evict_case(env, 8, [900, 700], 200, 50, weights=lambda rng, s: np.where(rng.random(s) < 0.5, -0.0, 0.0))
    evict_case(env, 9, [5000], 1000, 10, weights=lambda rng, s: (rng.random(s) < 0.01) * 1.0)


def test_evict_weights_in_order(env):
    evict_case(env, 10, [600], 200, 50, weights=lambda rng, s: np.broadcast_to(np.arange(s[-1]), s).copy())
    evict_case(env, 11, [600], 200, 50, weights=lambda rng, s: np.broadcast_to(-1.0 * np.arange(s[-1]), s).copy())
    evict_case(env, 12, [600], 200, 50, weights=lambda rng, s: rng.standard_normal(s) * 10.0 ** rng.integers(-40, 38, s))
    evict_case(env, 13, [600], 200, 50, weights=lambda rng, s: np.where(rng.random(s) < 0.2, np.inf, rng.random(s)))


def test_evict_lengths_in_place_and_a_loose_bound(env):
    evict_case(env, 14, [90, 0, 300, 20], 50, 10, alias=True)
    evict_case(env, 15, [90, 0, 300, 20], 50, 10, extra=800)
    evict_case(env, 16, [5, 0, 3], 50, 10, alias=True)


def test_evict_lengths_in_place_for_many_heads(env):
    """Every kv head of a sequence sees the length as it was, however late it runs."""
    evict_case(env, 19, [50 + i % 7 for i in range(150)], 50, 10, 16, 64, alias=True)


def test_evict_moves_of_many_steps(env):
    """More moved rows, and more recent ones, than a step of the kernel covers, with and without overlap of the recent rows'
    old and new places."""
    evict_case(env, 21, [3000, 2101, 2500], 2100, 2000, 2, 128)
    evict_case(env, 22, [3000, 2101, 2500], 2100, 700, 2, 112, "int4")
    evict_case(env, 23, [17000, 16500], 8000, 500, 1, 64)  # (16384 old rows and a few more)
    evict_case(env, 24, [16884, 9000], 8000, 500, 1, 64)  # (16384)


def test_evict_negative_nan_stays(env):
    torch, ops = env
    w = torch.rand(1, 1, 100, device="cuda")
    w[0, 0, 17] = torch.tensor([-4194304], dtype=torch.int32).view(torch.float32)[0]  # 0xffc00000
    w[0, 0, 20] = float("inf")
    r = S.Ranges(1, 100, 128)
    r.k[0, :, 0] = torch.arange(100, dtype=torch.uint8, device="cuda")
    lens = torch.tensor([100], dtype=torch.int32, device="cuda")
    ops.evict_rows(r.kp, r.vp, w, lens, lens, 11, 10, 100, torch.tensor([0], device="cuda"), 1, 64)
    assert r.k[0, :11, 0].tolist() == [17] + list(range(90, 100)) and lens.item() == 11


def test_evict_many_sequences(env):
    evict_case(env, 17, list(np.random.default_rng(2).integers(0, 60, 700)), 20, 5, 1)


def test_evict_nan_stays(env):
    torch, ops = env
    w = torch.rand(1, 1, 100, device="cuda")
    w[0, 0, 17] = float("nan")
    r = S.Ranges(1, 100, 128)
    r.k[0, :, 0] = torch.arange(100, dtype=torch.uint8, device="cuda")
    lens = torch.tensor([100], dtype=torch.int32, device="cuda")
    ops.evict_rows(r.kp, r.vp, w, lens, lens, 11, 10, 100, torch.tensor([0], device="cuda"), 1, 64)
    assert r.k[0, :11, 0].tolist() == [17] + list(range(90, 100)) and torch.isnan(w[0, 0, 0]) and lens.item() == 11


def test_evict_in_a_graph(env):
    torch, ops = env
    rng = np.random.default_rng(18)
    base = torch.from_numpy(rng.integers(0, 256, (2, 300, 256), dtype=np.uint8)).cuda()
    w0 = torch.rand(2, 2, 300, device="cuda")
    lens = torch.tensor([300, 200], dtype=torch.int32, device="cuda")
    slots = torch.tensor([1, 0], device="cuda")
    sides = []
    for _ in range(2):
        r = S.Ranges(2, 300, 256)
        sides.append((r, w0.clone(), torch.zeros_like(lens)))

    def call(r, w, new):
        ops.evict_rows(r.kp, r.vp, w, lens, new, 100, 30, 300, slots, 2, 64)

    def reset():
        for r, w, _ in sides:
            r.k.copy_(base)
            r.v.copy_(base)
            w.copy_(w0)

    reset()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(*sides[1])
    for n in ([300, 200], [101, 99], [150, 300]):
        reset()
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        call(*sides[0])
        g.replay()
        torch.cuda.synchronize()
        (a, wa, na), (b, wb, nb) = sides
        assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v) and torch.equal(wa, wb) and torch.equal(na, nb)


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("kind", ["bf16", "int4"])
def test_decode_steps_on_a_bounded_cache(env, kind):
    """Steps of a serving loop: write the row, attend, accumulate, and cut back to the budget whenever a sequence is
    eight rows over it; every step's attention against the rows that a host model of the cache holds."""
    torch, ops = env
    rng = np.random.default_rng(30)
    hq, hkv, d, keep, recent, slack = 8, 2, 128, 48, 16, 8
    lens = [40, 55]
    cache_dtype = "int4" if kind == "int4" else "auto"
    row = row_size(kind, hkv, d)
    r = S.Ranges(2, 64, row)
    weights = torch.zeros(2, hkv, 64, device="cuda")
    slots = torch.tensor([1, 0], device="cuda")
    k = [[np.zeros((0, d))] * hkv for _ in range(2)]  # per sequence and head: its rows in their places
    v = [[np.zeros((0, d))] * hkv for _ in range(2)]
    acc = [[np.zeros(0)] * hkv for _ in range(2)]

    def append(n_new):
        t = sum(n_new)
        kt, kh = S.as_type(S.model_values(rng, (t, hkv, d)), torch.bfloat16)
        vt, vh = S.as_type(S.model_values(rng, (t, hkv, d)), torch.bfloat16)
        if kind == "int4":
            kh, vh = S.values(*S.quantise(kh)), S.values(*S.quantise(vh))
        at = 0
        starts = []
        for i, n in enumerate(n_new):
            starts.append(at)
            for h in range(hkv):
                k[i][h] = np.concatenate([k[i][h], kh[at:at + n, h]])
                v[i][h] = np.concatenate([v[i][h], vh[at:at + n, h]])
                acc[i][h] = np.concatenate([acc[i][h], np.zeros(n)])
            at += n
        held = [len(k[i][0]) - n for i, n in enumerate(n_new)]
        i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
        ops.reshape_and_cache(kt, vt, r.kp, r.vp, torch.tensor([n * row for n in held], dtype=torch.int64, device="cuda"),
                              slots, i32(n_new), i32(starts), max(n_new), hkv, d, cache_dtype)

    append(lens)
    evictions = 0
    for step in range(20):
        append([1, 1])
        now = [len(k[i][0]) for i in range(2)]
        lens_t = torch.tensor(now, dtype=torch.int32, device="cuda")
        q, qh = S.as_type(rng.standard_normal((2, hq, d)) * 1.5, torch.bfloat16)
        out = torch.empty(2, hq, d, dtype=torch.float32, device="cuda")
        ops.paged_attention_v1(out, q, r.kp, r.vp, hkv, d ** -0.5, lens_t, 1, max(now), None, cache_dtype, 1.0, slots)
        ops.accumulate_attention_weights(weights, q, r.kp, hkv, d ** -0.5, lens_t, max(now), slots, None, cache_dtype)
        got, got_w = out.double().cpu().numpy(), weights.double().cpu().numpy()
        for i in range(2):
            kk, vv = np.stack(k[i], 1), np.stack(v[i], 1)
            want = S.attention(qh[i:i + 1], kk, vv, d ** -0.5)[0]
            assert (np.abs(got[i] - want) <= 2.0 ** -11 * np.abs(vv).max()).all()
            p = S.softmax(qh[i:i + 1], kk, d ** -0.5)[0].reshape(hkv, hq // hkv, -1).sum(1)
            for h in range(hkv):
                acc[i][h] = acc[i][h] + p[h]
                assert (np.abs(got_w[1 - i, h, :now[i]] - acc[i][h]) <= 2.0 ** -11 * acc[i][h] + 1e-9).all()
                assert (got_w[1 - i, h, now[i]:] == 0).all()
        if max(now) >= keep + slack:
            evictions += 1
            ops.evict_rows(r.kp, r.vp, weights, lens_t, lens_t, keep, recent, max(now), slots, hkv, d, cache_dtype)
            for i in range(2):
                for h in range(hkv):
                    # (by the GPU's own sums: two that are nearly equal may order either way in float64)
                    src = S.evicted_sources(got_w[1 - i, h, :now[i]], now[i], keep, recent)
                    k[i][h], v[i][h], acc[i][h] = k[i][h][src], v[i][h][src], acc[i][h][src]
            assert lens_t.tolist() == [len(k[i][0]) for i in range(2)]
    assert evictions >= 2
