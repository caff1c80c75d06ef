"""Values and calls at the edges of the batched-serving operators, against their
definitions in 64 bits.

Tolerances are those of ``tests/test_serving_gpu.py``: |got - want| <= u (|o| +
sum(p |v|) / sum(p)), u the unit roundoff of the 16-bit type. Where a value that a row
sees is infinite or NaN, the definition gives an infinity or NaN in that column of the
row and in no other place."""
import math

import pytest
import torch

import megakernel_b200 as mk
from test_serving_gpu import BF, DEV, FP, U, Cache, attend, cu_of, prompts, rand, seeded

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan


def attend_any(q, k, v):
    """One request as ``attend``, with V that need not be finite: what a row does not see
    does not reach it, and what it sees is added with a positive weight."""
    n, hq, d = q.shape
    m, hk = k.shape[:2]
    o, size = attend(q, k, torch.where(v.isfinite(), v, 0))
    sees = (torch.arange(m, device=DEV) <= (m - n + torch.arange(n, device=DEV))[:, None]).double()

    def any_of(bad):  # [n, hq, d]: some key that the row sees has it
        return (torch.einsum("qk,khd->qhd", sees, bad.double()) > 0).repeat_interleave(hq // hk, 1)

    up, down, nan = (any_of(b) for b in (v == INF, v == -INF, v.isnan()))
    o = torch.where(up, INF, o)
    o = torch.where(down, torch.where(up, NAN, -INF), o)
    return torch.where(nan, NAN, o), size


def check_any(got, want, size, dtype):
    assert got.dtype == dtype and got.shape == want.shape
    g = got.double()
    assert torch.equal(g.isnan(), want.isnan())
    assert torch.equal(g == INF, want == INF) and torch.equal(g == -INF, want == -INF)
    fin = want.isfinite()
    off = (g - want).abs()[fin] - U[dtype] * (want.abs() + size)[fin]
    assert off.numel() == 0 or float(off.max()) <= 0, float(off.max())


def plant(cache, b, key, head, dim, value):
    """Value ``dim`` of one V row, in the pages and in the plain copy."""
    cache.v[b][key, head, dim] = value
    page = cache.kc.shape[2]
    cache.vc[int(cache.table[b, key // page]), head, key % page, dim] = value


def want_of(cache, q, q_lens):
    got, at = [], 0
    for b, n in enumerate(q_lens):
        got.append(attend_any(q[at:at + n], cache.k[b], cache.v[b]))
        at += n
    return torch.cat([a for a, _ in got]), torch.cat([s for _, s in got])


# ---- V that is not finite ----------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("hq,hk,d", [(16, 8, 128), (2, 1, 128), (12, 4, 64)])
@pytest.mark.parametrize("n", [1, 2])
def test_decode_with_infinite_values(n, hq, hk, d, dtype):
    """One key, a few, and lengths that warps and CTAs share: an infinity with a weight of
    exactly 1, with a rounded one, of both signs in a column, NaN beside them."""
    kv = [n, 33, 300, 5000]
    c = Cache(kv, hk, d, 16, dtype, seed=n)
    plant(c, 0, 0, 0, 5, INF)
    plant(c, 0, n - 1, hk - 1, 6, -INF)
    for b in (1, 2, 3):
        m = kv[b]
        plant(c, b, 0, 0, 0, INF)
        plant(c, b, m - 1, 0, 1, -INF)          # the last key: not every new token sees it
        plant(c, b, m // 2, 0, 2, NAN)
        plant(c, b, m // 3, hk - 1, 63, INF)
        plant(c, b, m // 3 + 1, hk - 1, 63, -INF)
        plant(c, b, m - 1, hk - 1, d - 1, NAN)
    q = rand(seeded(21), 4, n, hq, d, dtype=dtype, scale=0.25)  # (weights of every key far from underflow)
    got = mk.paged_attention(q if n > 1 else q[:, 0], c.kc, c.vc, c.table, c.lens)
    check_any(got.view(-1, hq, d), *want_of(c, q.flatten(0, 1), [n] * 4), dtype)


@pytest.mark.parametrize("n", [2, 4])
def test_decode_of_several_tokens_with_values_that_some_do_not_see(n):
    """Non-finite rows of V at the new tokens' own positions, in one tile of keys and across two."""
    kv = [160, 161, 162, 163, 17, n, 4000]
    c = Cache(kv, 8, 128, 16, seed=n)
    for b, m in enumerate(kv):
        for i in range(n):
            plant(c, b, m - 1 - i, b % 8, 10 + i, (INF, NAN, -INF, INF)[i])
    q = rand(seeded(22), len(kv), n, 16, 128)
    got = mk.paged_attention(q, c.kc, c.vc, c.table, c.lens)
    check_any(got.flatten(0, 1), *want_of(c, q.flatten(0, 1), [n] * len(kv)), BF)
