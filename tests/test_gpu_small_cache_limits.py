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
