"""The batched-serving operators against their definitions in 64 bits.

Tolerances come from the roundings a kernel may make, with u the unit roundoff of the
16-bit type (2^-8 for BF16, 2^-11 for FP16): the output's own rounding gives u |o|, and
the probabilities enter the second product in the 16-bit type, u sum(p |v|) / sum(p).
The FP32 arithmetic is far below either (a score is off by at most D 2^-24 sum |q||k|
scale, under 2^-13 at these sizes): |got - want| <= u (|o| + sum(p |v|) / sum(p))."""
import math

import pytest
import torch

import megakernel_b200 as mk

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float16
U = {BF: 2.0 ** -8, FP: 2.0 ** -11}  # unit roundoff of the type
HEADS = [(16, 8, 128), (2, 1, 128), (8, 8, 64), (24, 8, 64), (14, 2, 128), (16, 1, 128), (20, 1, 64)]


def rand(gen, *shape, dtype=BF, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEV) * scale).to(dtype)


def seeded(seed=0):
    return torch.Generator(device=DEV).manual_seed(seed)


def cu_of(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).to(DEV)


def attend(q, k, v, scale=None):
    """FP64, one request: q [n, Hq, D] at the last n of k's positions -> (o, sum p|v| / sum p)."""
    n, hq, d = q.shape
    m, hk = k.shape[:2]
    q, k, v = (x.double() for x in (q, k, v))
    k, v = (x.repeat_interleave(hq // hk, 1) for x in (k, v))
    s = torch.einsum("qhd,khd->hqk", q, k) * (d ** -0.5 if scale is None else scale)
    sees = torch.arange(m, device=DEV) <= (m - n + torch.arange(n, device=DEV))[:, None]
    s = s.masked_fill(~sees, -math.inf)
    p = torch.softmax(s, -1).masked_fill(~sees.any(-1)[:, None], 0.0)
    p = p.masked_fill(~sees, 0.0)
    return torch.einsum("hqk,khd->qhd", p, v), torch.einsum("hqk,khd->qhd", p, v.abs())


def check(got, want, size, dtype):
    assert got.dtype == dtype and got.shape == want.shape
    off = (got.double() - want).abs() - U[dtype] * (want.abs() + size)
    assert not torch.isnan(got).any()
    assert float(off.max()) <= 0 if off.numel() else True, float(off.max())


def prompts(lens, hq, hk, d, dtype=BF, seed=0, spread=2.0):
    g = seeded(seed)
    t = sum(lens)
    return rand(g, t, hq, d, dtype=dtype, scale=spread), rand(g, t, hk, d, dtype=dtype), rand(g, t, hk, d, dtype=dtype)


def want_prompts(q, k, v, lens, scale=None):
    got, at = [], 0
    for n in lens:
        got.append(attend(q[at:at + n], k[at:at + n], v[at:at + n], scale))
        at += n
    return torch.cat([a for a, _ in got]), torch.cat([b for _, b in got])


class Cache:
    """A paged cache of known keys; what no key fills is NaN."""

    def __init__(self, kv_lens, hk, d, page, dtype=BF, seed=0, width=None, layout="hs", spare=3):
        g = seeded(seed + 100)
        self.k = [rand(g, n, hk, d, dtype=dtype) for n in kv_lens]
        self.v = [rand(g, n, hk, d, dtype=dtype) for n in kv_lens]
        need = [-(-n // page) for n in kv_lens]
        pool = sum(need) + spare
        shape = {"hs": (pool, hk, page, d), "sh": (pool, page, hk, d)}.get(layout)
        if layout == "kv":  # one allocation, K and V side by side within a page
            both = torch.full((pool, 2, hk, page, d), math.nan, dtype=dtype, device=DEV)
            self.kc, self.vc = both[:, 0], both[:, 1]
        else:
            self.kc, self.vc = (torch.full(shape, math.nan, dtype=dtype, device=DEV) for _ in range(2))
            if layout == "sh":
                self.kc, self.vc = self.kc.transpose(1, 2), self.vc.transpose(1, 2)
        order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).tolist()
        width = max(need + [1]) if width is None else width
        self.table = torch.full((len(kv_lens), width), -1, dtype=torch.int32)
        for b, n in enumerate(kv_lens):
            for e in range(need[b]):
                pg = order.pop()
                self.table[b, e] = pg
                rows = slice(e * page, min(n, (e + 1) * page))
                self.kc[pg, :, : rows.stop - rows.start] = self.k[b][rows].transpose(0, 1)
                self.vc[pg, :, : rows.stop - rows.start] = self.v[b][rows].transpose(0, 1)
        self.table = self.table.to(DEV)
        self.lens = torch.tensor(kv_lens, dtype=torch.int32, device=DEV)

    def want(self, q, q_lens, scale=None):
        got, at = [], 0
        for b, n in enumerate(q_lens):
            m = self.k[b].shape[0]
            o, size = attend(q[at + max(0, n - m):at + n], self.k[b], self.v[b], scale)
            zero = torch.zeros((max(0, n - m), *q.shape[1:]), dtype=torch.float64, device=DEV)
            got.append((torch.cat((zero, o)), torch.cat((zero, size))))
            at += n
        return torch.cat([a for a, _ in got]), torch.cat([b for _, b in got])


# ---- packed prompts -------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("hq,hk,d", HEADS)
def test_prompt_heads_and_types(hq, hk, d, dtype):
    lens = [1, 130, 64, 2, 257]
    q, k, v = prompts(lens, hq, hk, d, dtype)
    check(mk.prompt_attention(q, k, v, cu_of(lens)), *want_prompts(q, k, v, lens), dtype)


@pytest.mark.parametrize("lens", [[1], [1, 1, 1], [127], [128], [129], [255, 256, 257], [0, 5, 0, 0, 31, 0], [1023, 3],
                                  [33] * 40, [1500, 2, 700, 1, 1]])
def test_prompt_lengths(lens):
    q, k, v = prompts(lens, 8, 4, 128, seed=len(lens))
    check(mk.prompt_attention(q, k, v, cu_of(lens)), *want_prompts(q, k, v, lens), BF)


@pytest.mark.parametrize("hq,hk,d", [(4, 2, 128), (3, 1, 64)])
def test_prompt_long(hq, hk, d):
    lens = [4500]
    q, k, v = prompts(lens, hq, hk, d, seed=3)
    check(mk.prompt_attention(q, k, v, cu_of(lens)), *want_prompts(q, k, v, lens), BF)


def test_prompt_strides_scale_and_out():
    lens = [200, 77]
    g = seeded(5)
    qkv = rand(g, 277, 8, 128)  # 4 q, 2 k, 2 v heads of one projection
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    wide = torch.full((277, 6, 128), 7.0, dtype=BF, device=DEV)
    got = mk.prompt_attention(q, k, v, cu_of(lens), scale=0.3, out=wide[:, 1:5])
    assert got.data_ptr() == wide[:, 1:5].data_ptr()
    check(got, *want_prompts(q, k, v, lens, 0.3), BF)
    assert bool((wide[:, 0] == 7).all()) and bool((wide[:, 5] == 7).all())
    heads_first = rand(g, 4, 277, 128).transpose(0, 1)
    check(mk.prompt_attention(heads_first, k, v, cu_of(lens)), *want_prompts(heads_first, k, v, lens), BF)


def test_prompt_large_scores_and_growing_maximum():
    """Scores of several hundred, the largest key last: every rescaling of the sums is taken."""
    lens = [700]
    q, k, v = prompts(lens, 4, 2, 128, seed=8)
    k *= (1 + torch.arange(700, device=DEV) / 50)[:, None, None]
    q, k = q.to(BF), k.to(BF)
    check(mk.prompt_attention(q, k, v, cu_of(lens)), *want_prompts(q, k, v, lens), BF)
    k = -k.flip(0)
    check(mk.prompt_attention(q, k.contiguous(), v, cu_of(lens)), *want_prompts(q, k, v, lens), BF)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("where", ["k", "v"])
def test_prompt_future_and_foreign_values_do_not_matter(bad, where):
    """A token that cannot see position j does not depend on it, whatever stands there."""
    lens, j = [150, 60, 300], 90  # position 90 of the first prompt, 17 of the third
    q, k, v = prompts(lens, 4, 2, 128, seed=9)
    clean = mk.prompt_attention(q, k, v, cu_of(lens))
    x = {"k": k, "v": v}[where]
    x[j] = bad
    x[210 + 17, 1, 5] = bad
    got = mk.prompt_attention(q, k, v, cu_of(lens))
    same = torch.ones(510, dtype=torch.bool, device=DEV)
    same[j:150] = False
    same[227:510] = False
    want, size = want_prompts(q[:90], k[:90], v[:90], [90])
    check(got[:90], want, size, BF)
    check(got[150:210], *want_prompts(q[150:210], k[150:210], v[150:210], [60]), BF)
    check(got[210:227], *want_prompts(q[210:227], k[210:227], v[210:227], [17]), BF)
    assert torch.equal(got[same].isfinite(), clean[same].isfinite())
    if where == "v":
        assert not got[j:150].isfinite().any()
        assert not got[227:510, 2:, 5].isfinite().any() and got[227:510, :2].isfinite().all()


def test_prompt_is_reproducible_and_runs_on_other_streams():
    lens = [900, 45, 1300]
    q, k, v = prompts(lens, 16, 8, 128, seed=4)
    cu = cu_of(lens)
    first = mk.prompt_attention(q, k, v, cu)
    side = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for i in range(6):
        with torch.cuda.stream(side[i % 3]):
            got.append(mk.prompt_attention(q, k, v, cu))
    torch.cuda.synchronize()
    assert all(torch.equal(first, x) for x in got)


# ---- over the paged cache ---------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("hq,hk,d", HEADS)
def test_decode_heads_and_types(hq, hk, d, dtype):
    kv = [1, 17, 400, 64, 33]
    c = Cache(kv, hk, d, 16, dtype)
    q = rand(seeded(1), 5, hq, d, dtype=dtype, scale=2.0)
    check(mk.paged_attention(q, c.kc, c.vc, c.table, c.lens), *c.want(q, [1] * 5), dtype)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("layout", ["hs", "sh", "kv"])
def test_pages_and_layouts(page, layout):
    kv, new = [300, 1, 128, 129, 1000], [3, 1, 128, 60, 200]
    c = Cache(kv, 2, 128, page, layout=layout, seed=page)
    q = rand(seeded(2), sum(new), 4, 128, scale=2.0)
    check(mk.paged_attention(q, c.kc, c.vc, c.table, c.lens, cu_of(new)), *c.want(q, new), BF)
    last = cu_of(new)[1:].long() - 1
    check(mk.paged_attention(q[last], c.kc, c.vc, c.table, c.lens), *c.want(q[last], [1] * 5), BF)


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("hq,hk,d", [(4, 2, 128), (6, 3, 64)])
@pytest.mark.parametrize("gaps", [(0, 24), (40, 0), (8, 8)])
def test_pages_and_heads_with_gaps(gaps, hq, hk, d, page):
    """Page and KV head strides of which neither is a multiple of the other (or one is)."""
    new, kv = [1, 90, 200, 1], [1, 333, 200, 700]
    c = Cache(kv, hk, d, page, seed=page)
    q = rand(seeded(12), sum(new), hq, d, scale=2.0)
    want = c.want(q, new)
    pool = c.kc.shape[0]
    hs = page * d + gaps[0]
    ps = hk * hs + gaps[1]
    caches = []
    for x in (c.kc, c.vc):
        store = torch.full((pool * ps,), math.nan, dtype=BF, device=DEV)
        caches.append(torch.as_strided(store, (pool, hk, page, d), (ps, hs, d, 1)))
        caches[-1].copy_(x)
    check(mk.paged_attention(q, *caches, c.table, c.lens, cu_of(new)), *want, BF)
    one = [1] * 4
    check(mk.paged_attention(q[:4], *caches, c.table, c.lens), *c.want(q[:4], one), BF)


@pytest.mark.parametrize("kv", [[1], [5000], [1, 9000, 2], [257] * 70, [int(1.13 ** i) for i in range(2, 66)]])
@pytest.mark.parametrize("hq,hk", [(16, 8), (2, 1), (5, 1)])
def test_decode_lengths(kv, hq, hk):
    c = Cache(kv, hk, 128, 16, seed=len(kv))
    q = rand(seeded(3), len(kv), hq, 128, scale=2.0)
    check(mk.paged_attention(q, c.kc, c.vc, c.table, c.lens), *c.want(q, [1] * len(kv)), BF)


@pytest.mark.parametrize("hq,hk,d,dtype", [(16, 8, 128, BF), (16, 1, 128, BF), (24, 8, 64, FP), (7, 7, 128, FP)])
@pytest.mark.parametrize("n", [2, 4, 9])
def test_several_tokens_each(n, hq, hk, d, dtype):
    kv = [n, 40, 1000, 129]
    c = Cache(kv, hk, d, 32, dtype, seed=n)
    q = rand(seeded(4), 4, n, hq, d, dtype=dtype, scale=2.0)
    got = mk.paged_attention(q, c.kc, c.vc, c.table, c.lens)
    check(got.flatten(0, 1), *c.want(q.flatten(0, 1), [n] * 4), dtype)


@pytest.mark.parametrize("hq,hk,d,dtype", [(16, 8, 128, BF), (14, 2, 128, BF), (24, 8, 64, FP), (16, 1, 64, BF)])
@pytest.mark.parametrize("new,kv", [([300], [300]), ([1, 257, 1, 31], [700, 1025, 40, 8000]), ([512, 512], [4000, 513]),
                                    ([0, 4, 0, 130], [50, 4, 0, 4097]), ([1] * 30 + [600], [99 * i + 1 for i in range(31)]),
                                    ([5], [20000])])
def test_chunks(new, kv, hq, hk, d, dtype):
    kv = [max(a, b) for a, b in zip(new, kv)]
    c = Cache(kv, hk, d, 16, dtype, seed=len(kv))
    q = rand(seeded(5), sum(new), hq, d, dtype=dtype, scale=2.0)
    check(mk.paged_attention(q, c.kc, c.vc, c.table, c.lens, cu_of(new)), *c.want(q, new), dtype)


def test_no_keys_give_zeros():
    c = Cache([0, 20, 0, 3], 2, 128, 16, seed=1)
    q = rand(seeded(6), 4, 4, 128)
    got = mk.paged_attention(q, c.kc, c.vc, c.table, c.lens)
    check(got, *c.want(q, [1] * 4), BF)
    assert bool((got[0] == 0).all()) and bool((got[2] == 0).all())
    new = [2, 5, 1, 9]  # more new tokens than keys: the first of them stand before position 0
    q = rand(seeded(7), 17, 4, 128)
    got = mk.paged_attention(q, c.kc, c.vc, c.table, c.lens, cu_of(new))
    check(got, *c.want(q, new), BF)
    assert bool((got[:2] == 0).all()) and bool((got[8:14] == 0).all())
    assert mk.serving_status() == (0, "ok")
    empty = mk.paged_attention(q[:0], c.kc, c.vc, c.table[:0], c.lens[:0])
    assert empty.shape == (0, 4, 128)


@pytest.mark.parametrize("new", [[1], [150]])
def test_offsets_past_32_bits(new):
    """Pages 2^26 elements apart: the last ones lie past 2^32 elements."""
    kv, page, hk, d = [150], 16, 2, 128
    stride, pool = 2 ** 26, 72
    store = torch.empty((pool - 1) * stride + hk * page * d, dtype=BF, device=DEV)
    c = Cache(kv, hk, d, page, seed=4)
    big = torch.as_strided(store, (pool, hk, page, d), (stride, page * d, d, 1))
    ids = torch.tensor([71, 64, 3, 70, 69, 66, 68, 67, 65, 0], device=DEV)
    q = rand(seeded(8), sum(new), 4, d, scale=2.0)
    table = ids.to(torch.int32)[None]
    big[ids] = c.kc[c.table[0].long()]
    vbig = c.vc.new_zeros((pool, hk, page, d))
    vbig[ids] = c.vc[c.table[0].long()]
    got = mk.paged_attention(q, big, vbig, table, c.lens, cu_of(new) if new != [1] else None)
    check(got, *c.want(q, new), BF)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_masked_values_do_not_matter_over_pages(bad):
    new, kv = [70, 1], [200, 64]
    c = Cache(kv, 2, 128, 16, seed=3)
    q = rand(seeded(9), 71, 4, 128)
    want, size = c.want(q, new)
    j = 160  # seen by the last 40 of the first request's 70 tokens
    c.vc[c.table[0, j // 16].long(), :, j % 16] = bad
    got = mk.paged_attention(q, c.kc, c.vc, c.table, c.lens, cu_of(new))
    check(got[:30], want[:30], size[:30], BF)
    check(got[70:], want[70:], size[70:], BF)
    assert not got[30:70].isfinite().any()


def test_wrong_pages_and_lengths_are_reported():
    for new in ([1, 1, 1], [1, 40, 1]):
        c = Cache([30, 40, 50], 2, 128, 16, seed=2)
        q = rand(seeded(10), sum(new), 4, 128)
        cu = cu_of(new) if max(new) > 1 else None
        want, size = c.want(q, new)
        ok = torch.ones(sum(new), dtype=torch.bool)
        ok[1:-1] = False
        good = c.table.clone()
        for page in (-1, c.kc.shape[0], 2 ** 31 - 1):
            c.table[1, 1] = page
            got = mk.paged_attention(q, c.kc, c.vc, c.table, c.lens, cu)
            check(got[ok], want[ok], size[ok], BF)
            assert got[1:-1].isnan().any()
            assert mk.serving_status()[0] == 1 and mk.serving_status()[0] == 0
        c.table = good
        c.lens[1] = 16 * c.table.shape[1] + 1
        got = mk.paged_attention(q, c.kc, c.vc, c.table, c.lens, cu)
        check(got[ok], want[ok], size[ok], BF)
        assert got[1:-1].isnan().all()
        assert mk.serving_status()[0] == 2


@pytest.mark.parametrize("new", [[1, 1, 1], [1, 40, 1]])
def test_pool_without_pages(new):
    """No page is inside it: requests with keys are reported, those without get zeros."""
    pool = torch.empty((0, 2, 16, 128), dtype=BF, device=DEV)
    table = torch.zeros((3, 4), dtype=torch.int32, device=DEV)
    lens = torch.tensor([0, 50, 0], dtype=torch.int32, device=DEV)
    q = rand(seeded(11), sum(new), 4, 128)
    got = mk.paged_attention(q, pool, pool, table, lens, cu_of(new) if max(new) > 1 else None)
    assert bool((got[0] == 0).all()) and bool((got[-1] == 0).all())
    assert got[1:-1].isnan().all()
    assert mk.serving_status()[0] == 1


def test_paged_is_reproducible_across_streams_and_in_graphs():
    kv, new = [3000, 50, 7000, 1], [1, 30, 1, 1]
    c = Cache(kv, 8, 128, 16, seed=6)
    q = rand(seeded(11), sum(new), 16, 128)
    cu = cu_of(new)
    one, many = q[:4].clone(), q
    calls = [lambda: mk.paged_attention(one, c.kc, c.vc, c.table, c.lens),
             lambda: mk.paged_attention(many, c.kc, c.vc, c.table, c.lens, cu)]
    for call in calls:
        first = call()
        side = [torch.cuda.Stream() for _ in range(3)]
        torch.cuda.synchronize()
        got = []
        for i in range(9):
            with torch.cuda.stream(side[i % 3]):
                got.append(call())
        torch.cuda.synchronize()
        assert all(torch.equal(first, x) for x in got)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        for _ in range(3):
            out.zero_()
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)


# ---- the append ---------------------------------------------------------------------------

def want_append(qkv, hk, positions, cos, sin, q_norm, k_norm, eps=1e-6):
    x = qkv.double()
    hq, d = x.shape[1] - 2 * hk, x.shape[2]

    def turn(y, w):
        if w is not None:
            y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * w.double()
        rot = torch.cat((-y[..., d // 2:], y[..., :d // 2]), -1)
        c, s = cos.double()[positions][:, None], sin.double()[positions][:, None]
        return y * c + rot * s

    return turn(x[:, :hq], q_norm), turn(x[:, hq:hq + hk], k_norm), x[:, hq + hk:]


def close(got, want, dtype):
    """One rounding, and FP32 arithmetic on values of a few units (cancellation in the rotation)."""
    assert float(((got.double() - want).abs() - U[dtype] * want.abs() - 2e-5 * (1 + want.abs().amax())).max()) <= 0


@pytest.mark.parametrize("source", [BF, FP, torch.float32])
@pytest.mark.parametrize("hq,hk,d", HEADS)
@pytest.mark.parametrize("dtype", [BF, FP])
def test_append(source, hq, hk, d, dtype):
    new, kv, page = [1, 7, 0, 33, 1], [5, 7, 9, 100, 64], 16
    c = Cache(kv, hk, d, page, dtype, seed=1)
    g = seeded(12)
    qkv = rand(g, sum(new), hq + 2 * hk, d, dtype=source)
    cos, sin = torch.rand((128, d), generator=g, device=DEV) * 2 - 1, torch.rand((128, d), generator=g, device=DEV)
    norms = [dict(), dict(q_norm=rand(g, d, dtype=dtype), k_norm=rand(g, d, dtype=dtype)),
             dict(k_norm=rand(g, d, dtype=dtype))]
    pos = torch.cat([torch.arange(m - n, m) for n, m in zip(new, kv)]).to(DEV)
    req = torch.repeat_interleave(torch.arange(5), torch.tensor(new)).to(DEV)
    page_of, slot = c.table[req, pos // page].long(), pos % page
    for norm in norms:
        kc, vc = c.kc.clone(), c.vc.clone()
        q, k = mk.paged_append(qkv, kc, vc, c.table, c.lens, cos, sin, cu_of(new), return_k=True, **norm)
        wq, wk, wv = want_append(qkv, hk, pos, cos, sin, norm.get("q_norm"), norm.get("k_norm"))
        close(q, wq, dtype)
        close(k, wk, dtype)
        assert torch.equal(kc[page_of, :, slot], k)
        assert torch.equal(vc[page_of, :, slot], wv.to(torch.float32).to(dtype))
        untouched = torch.ones(kc.shape[:1] + kc.shape[2:3], dtype=torch.bool, device=DEV)
        untouched[page_of, slot] = False
        for x, y in ((kc, c.kc), (vc, c.vc)):
            a, b = x.transpose(1, 2)[untouched], y.transpose(1, 2)[untouched]
            assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


def test_append_one_token_each_strided_16_bit_tables():
    kv = [1, 200, 16, 17]
    c = Cache(kv, 8, 128, 32, layout="sh", seed=2)
    g = seeded(13)
    wide = rand(g, 4, 40, 128)
    qkv = wide[:, 4:36]
    cos, sin = mk.rope_tables(200, DEV, BF)
    w = rand(g, 128)
    q = mk.paged_append(qkv, c.kc, c.vc, c.table, c.lens, cos, sin, q_norm=w, k_norm=w, eps=1e-5)
    pos = torch.tensor(kv, device=DEV) - 1
    wq, wk, wv = want_append(qkv, 8, pos, cos, sin, w, w, 1e-5)
    close(q, wq, BF)
    pg = c.table[torch.arange(4, device=DEV), pos // 32].long()
    close(c.kc[pg, :, pos % 32], wk, BF)
    assert torch.equal(c.vc[pg, :, pos % 32], wv.to(BF))
    both = mk.paged_append(wide[:, None, 4:36].expand(4, 1, 32, 128), c.kc, c.vc, c.table, c.lens, cos, sin, q_norm=w,
                           k_norm=w, eps=1e-5)
    assert both.shape == (4, 1, 16, 128) and torch.equal(both[:, 0], q)


def test_append_wrong_positions_are_reported():
    c = Cache([30, 40, 50], 2, 128, 16, seed=2)
    g = seeded(14)
    qkv = rand(g, 3, 8, 128)
    cos, sin = mk.rope_tables(96, DEV)
    before = c.kc.clone()

    def call(cos=cos, sin=sin):
        return mk.paged_append(qkv, c.kc, c.vc, c.table, c.lens, cos, sin)

    good = call()
    after = c.kc.clone()
    assert mk.serving_status() == (0, "ok") and not torch.equal(before.nan_to_num(), after.nan_to_num())
    q = call(cos[:45].contiguous(), sin[:45].contiguous())
    assert mk.serving_status()[0] == 3
    assert torch.equal(q[:2], good[:2]) and q[2].isnan().all()
    keep = c.table.clone()
    c.table[1, 2] = c.kc.shape[0]
    q = call()
    assert mk.serving_status()[0] == 1 and q[1].isnan().all() and torch.equal(q[::2], good[::2])
    c.table = keep
    c.lens[0] = 16 * c.table.shape[1] + 1
    assert call()[0].isnan().all() and mk.serving_status()[0] == 2
    c.lens[0] = 0  # its one token stands before position 0: nothing to write, zeros
    assert bool((call()[0] == 0).all()) and mk.serving_status() == (0, "ok")
    assert torch.equal(c.kc.nan_to_num(), after.nan_to_num())


# ---- refusals -------------------------------------------------------------------------------

def test_refusals():
    q, k, v = prompts([40], 4, 2, 128)
    cu = cu_of([40])
    c = Cache([20, 30], 2, 128, 16)
    one = q[:2]
    cos, sin = mk.rope_tables(64, DEV)
    qkv = rand(seeded(0), 2, 8, 128)

    def prompt(**kw):
        a = dict(q=q, k=k, v=v, cu_seqlens=cu)
        a.update(kw)
        return mk.prompt_attention(**a)

    def paged(**kw):
        a = dict(q=one, k_cache=c.kc, v_cache=c.vc, block_table=c.table, kv_lens=c.lens)
        a.update(kw)
        return mk.paged_attention(**a)

    def append(**kw):
        a = dict(qkv=qkv, k_cache=c.kc, v_cache=c.vc, block_table=c.table, kv_lens=c.lens, cos=cos, sin=sin)
        a.update(kw)
        return mk.paged_append(**a)

    odd = torch.empty(40 * 4 * 128 + 8, dtype=BF, device=DEV)[1:-7].view(40, 4, 128)
    small = torch.zeros((5, 2, 8, 128), dtype=BF, device=DEV)
    refused = [
        (prompt, dict(q=q.float())), (prompt, dict(q=q.cpu())), (prompt, dict(k=k.half())), (prompt, dict(k=k[:39])),
        (prompt, dict(v=v[:, :1])), (prompt, dict(q=q[:, :3])), (prompt, dict(q=q[:, :, :96].contiguous())),
        (prompt, dict(q=q[:, :, ::2])), (prompt, dict(q=odd)), (prompt, dict(cu_seqlens=cu.long())),
        (prompt, dict(cu_seqlens=cu.cpu())), (prompt, dict(scale=0.0)), (prompt, dict(scale=-1.0)),
        (prompt, dict(scale=math.inf)), (prompt, dict(out=q[:39])), (prompt, dict(out=q.half())),
        (prompt, dict(cu_seqlens=cu[:1])),
        (paged, dict(q=q[:3])), (paged, dict(q=one.half())), (paged, dict(v_cache=c.vc[:-1])),
        (paged, dict(k_cache=small, v_cache=small)), (paged, dict(kv_lens=c.lens[:1])),
        (paged, dict(block_table=c.table.long())), (paged, dict(kv_lens=c.lens.cpu())), (paged, dict(cu_q=cu)),
        (paged, dict(q=one[:, :3])), (paged, dict(q=one[:, :, :64].contiguous())), (paged, dict(scale=math.nan)),
        (append, dict(qkv=qkv[:, :5])), (append, dict(cos=cos[:, :64])), (append, dict(sin=sin[:10])),
        (append, dict(q_norm=cos[0])), (append, dict(k_norm=q[0, 0, :64])), (append, dict(eps=-1.0)),
        (append, dict(qkv=qkv.double())), (append, dict(cos=cos.half(), sin=sin.half())),
        (append, dict(k_cache=c.kc.float(), v_cache=c.vc.float())),
    ]
    for i, (call, kw) in enumerate(refused):
        with pytest.raises(ValueError):
            call(**kw)
            pytest.fail(f"case {i} of {call.__name__} ({list(kw)}) was not refused")
    prompt()
    paged()
    append()
    assert mk.serving_status() == (0, "ok")
