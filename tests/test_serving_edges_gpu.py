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


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("hq,hk,d,n", [(14, 2, 128, 1), (16, 2, 64, 1), (5, 1, 128, 1), (6, 2, 128, 2), (2, 1, 64, 4)])
def test_five_to_eight_rows_over_a_table_for_long_requests(n, hq, hk, d, dtype):
    """Room for 16,384 keys or more, of which the requests use any part."""
    kv = [n, 40, 16384, 700]
    c = Cache(kv, hk, d, 16, dtype, seed=n, width=1100)
    for b, m in enumerate(kv):
        plant(c, b, m - 1, 0, 3, INF)
        plant(c, b, m // 2, hk - 1, 4, (NAN, -INF)[b % 2])
    q = rand(seeded(25), 4, n, hq, d, dtype=dtype, scale=0.25)
    got = mk.paged_attention(q, c.kc, c.vc, c.table, c.lens)
    check_any(got.flatten(0, 1), *want_of(c, q.flatten(0, 1), [n] * 4), dtype)


def test_few_short_requests_of_eight_rows_take_no_longer_than_with_offsets():
    """With offsets the tensor-core tiles run: where they are faster they run without, too."""
    c = Cache([500, 700, 1000], 8, 128, 16)
    q, cu = rand(seeded(26), 12, 16, 128), cu_of([4, 4, 4])

    def times(call):
        graph, _ = captured(call, 20)
        return elapsed(graph.replay, 5)

    direct = times(lambda: mk.paged_attention(q.view(3, 4, 16, 128), c.kc, c.vc, c.table, c.lens))
    assert direct < 1.2 * times(lambda: mk.paged_attention(q, c.kc, c.vc, c.table, c.lens, cu))


def spoil(v, at):
    """Values at (key, head, dim) of v, in place."""
    for key, head, dim, value in at:
        v[key, head, dim] = value


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("hq,hk,d", [(16, 8, 128), (8, 8, 64), (6, 2, 128), (16, 1, 64), (128, 1, 128)])
@pytest.mark.parametrize("lens", [[300, 1, 70], [1000, 255, 130], [2, 3, 129, 64]])
def test_prompts_with_values_that_some_rows_do_not_see(lens, hq, hk, d, dtype):
    """At the first and last key, at both sides of a tile's border, of both signs in a column."""
    q, k, v = prompts(lens, hq, hk, d, dtype, seed=len(lens), spread=0.25)
    at = 0
    for n in lens:
        keys = sorted({0, 1, 63, 64, 127, 128, 200, n // 2, n - 2, n - 1} & set(range(n)))
        spoil(v[at:at + n], [(j, i % hk, (7 * i) % d, (INF, -INF, NAN)[i % 3]) for i, j in enumerate(keys)])
        spoil(v[at:at + n], [(n // 3, 0, 1, INF), (2 * n // 3, 0, 1, -INF)])
        at += n
    got = mk.prompt_attention(q, k, v, cu_of(lens))
    want, at = [], 0
    for n in lens:
        want.append(attend_any(q[at:at + n], k[at:at + n], v[at:at + n]))
        at += n
    check_any(got, torch.cat([a for a, _ in want]), torch.cat([b for _, b in want]), dtype)


@pytest.mark.parametrize("hq,hk,d,page", [(16, 8, 128, 16), (4, 2, 64, 32), (14, 2, 128, 128)])
@pytest.mark.parametrize("new,kv", [([70, 1, 5], [200, 64, 5]), ([130], [9000]), ([300, 40], [4000, 12000]),
                                    ([1, 2], [20000, 30]), ([20, 9], [7, 0])])
def test_chunks_with_values_that_some_rows_do_not_see(new, kv, hq, hk, d, page):
    """Over pages: whole rows, rows whose keys are split, and tokens that stand before position 0."""
    c = Cache(kv, hk, d, page, seed=len(new))
    for b, m in enumerate(kv):
        for i, j in enumerate(sorted({0, m // 2, m - 1, m - 2, m - 5, m - 69, m - 130} & set(range(m)))):
            plant(c, b, j, i % hk, (5 * i) % d, (INF, -INF, NAN)[i % 3])
            plant(c, b, j, 0, d - 1, (INF, -INF)[i % 2])
    q = rand(seeded(23), sum(new), hq, d, scale=0.25)
    got = mk.paged_attention(q, c.kc, c.vc, c.table, c.lens, cu_of(new))
    want, at = [], 0
    for b, n in enumerate(new):
        m, blind = kv[b], max(0, n - kv[b])
        zero = torch.zeros((blind, hq, d), dtype=torch.float64, device=DEV)
        o, size = attend_any(q[at + blind:at + n], c.k[b], c.v[b]) if m else (zero[:0], zero[:0])
        want += [(zero, zero), (o, size)]
        at += n
    check_any(got, torch.cat([a for a, _ in want]), torch.cat([b for _, b in want]), BF)


def elapsed(call, n=3):
    call()
    best = INF
    for _ in range(n):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        call()
        end.record()
        end.synchronize()
        best = min(best, start.elapsed_time(end))
    return best


def test_values_that_are_not_finite_cost_little():
    """A NaN that every row sees is no reason to look at any row again; one that only some see
    takes a look at the few keys they differ in. A pass over all keys of every row, key by key,
    takes a hundred times as long."""
    n = 4000
    q, k, v = prompts([n], 16, 8, 128, seed=5, spread=0.25)
    cu = cu_of([n])
    clean = elapsed(lambda: mk.prompt_attention(q, k, v, cu))
    v[0] = NAN
    got = mk.prompt_attention(q, k, v, cu)
    assert got.isnan().all()
    assert elapsed(lambda: mk.prompt_attention(q, k, v, cu)) < 4 * clean
    v[:] = INF
    assert (mk.prompt_attention(q, k, v, cu) == INF).all()
    assert elapsed(lambda: mk.prompt_attention(q, k, v, cu)) < 20 * clean
    assert mk.serving_status() == (0, "ok")


@pytest.mark.parametrize("new,kv", [([1, 1, 1], [300, 5000, 40]), ([90, 1, 700], [300, 5000, 700])])
def test_output_in_place_of_q(new, kv):
    """Every row of q is read before its row of the output is written, whatever V holds."""
    c = Cache(kv, 2, 128, 16, seed=9)
    plant(c, 0, kv[0] - 1, 0, 3, INF)
    plant(c, 2, kv[2] // 2, 1, 4, NAN)
    q = rand(seeded(24), sum(new), 16, 128, scale=0.25)
    cu = cu_of(new) if max(new) > 1 else None
    want = mk.paged_attention(q, c.kc, c.vc, c.table, c.lens, cu)
    check_any(want, *want_of(c, q, new), BF)
    got = mk.paged_attention(q, c.kc, c.vc, c.table, c.lens, cu, out=q)
    assert got.data_ptr() == q.data_ptr()
    assert torch.equal(got.nan_to_num(7.0, 8.0, 9.0), want.nan_to_num(7.0, 8.0, 9.0))


# ---- small weights ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("gap", [12, 20, 25.3, 27])
@pytest.mark.parametrize("n", [1, 3])
def test_many_small_weights_beside_a_large_one(n, gap, dtype):
    """One key far ahead (by ``gap`` powers of two) of 40,000 that together still count. A 16-bit
    weight holds 2^-32 of the largest at least (FP16: its smallest value 2^-24, half of that in
    rounding, and 2^7 of headroom), so the error may be that of every value on top."""
    m, d = 40000, 64
    c = Cache([m], 1, d, 16, dtype)
    lead = gap * math.log(2) * d ** 0.5
    k, v = torch.zeros((m, 1, d), device=DEV), rand(seeded(31), m, 1, d).float().abs()
    k[0, 0, 0] = 1
    v[0] = 0
    c.k[0], c.v[0] = k.to(dtype), v.to(dtype)
    ids = c.table[0].long()
    c.kc[ids, 0], c.vc[ids, 0] = (x.view(-1, 16, d) for x in (c.k[0][:, 0], c.v[0][:, 0]))
    q = torch.zeros((n, 2, d), dtype=dtype, device=DEV)
    q[:, :, 0] = lead
    want, size = attend(q, c.k[0], c.v[0])
    for cu in (None, cu_of([n])):
        got = mk.paged_attention(q[None] if cu is None else q, c.kc, c.vc, c.table, c.lens, cu).view(n, 2, d)
        low = 2.0 ** -32 * c.v[0].double().abs().sum(0) if dtype == FP else 0
        off = (got.double() - want).abs() - U[dtype] * (want.abs() + size) - low
        assert float(off.max()) <= 0, (cu is None, float(off.max()))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("gap", [12, 20, 25.3, 27])
def test_many_small_weights_beside_a_large_one_in_a_long_prompt(gap, dtype):
    m, d = 16000, 64
    k, v = torch.zeros((m, 8, d), dtype=dtype, device=DEV), rand(seeded(32), m, 8, d).abs().to(dtype)
    k[0, :, 0] = 1
    v[0] = 0
    q = torch.zeros((m, 16, d), dtype=dtype, device=DEV)
    q[:, :, 0] = gap * math.log(2) * d ** 0.5
    got = mk.prompt_attention(q, k, v, cu_of([m]))[-64:]
    want, size = attend(q[-64:], k, v)
    low = 2.0 ** -32 * v.double().abs().sum(0).repeat_interleave(2, 0) if dtype == FP else 0
    off = (got.double() - want).abs() - U[dtype] * (want.abs() + size) - low
    assert float(off.max()) <= 0, float(off.max())


# ---- a wait that runs out ------------------------------------------------------------------

@pytest.fixture
def withhold():
    """Makes a CTA of the calls that follow stop loading, so that its waits run out."""
    from megakernel_b200 import _lib
    lib = _lib.load()
    yield lib.mkb_attn_withhold
    lib.mkb_attn_withhold(-1, 0)
    mk.serving_status()


def calls_to_stop():
    lens = [900, 45, 1300, 1]
    q, k, v = prompts(lens, 16, 8, 128, seed=4)
    many = prompts([33] * 300, 8, 4, 64, seed=5)
    c = Cache([30000, 50, 7000, 1], 2, 128, 16, seed=6)
    few, cu = rand(seeded(11), 33, 16, 128), cu_of([1, 30, 1, 1])
    long = Cache([1500] * 60, 8, 128, 16, seed=7)
    one = rand(seeded(12), 60, 16, 128)
    return {"prompts": (mk.prompt_attention, (q, k, v, cu_of(lens))),
            "many prompts": (mk.prompt_attention, (*many, cu_of([33] * 300))),
            "split rows": (mk.paged_attention, (few, c.kc, c.vc, c.table, c.lens, cu)),
            "decode": (mk.paged_attention, (one, long.kc, long.vc, long.table, long.lens))}


@pytest.mark.parametrize("name,cta,start", [(name, cta, 0) for cta in (3, -2) for name in
                                            ("prompts", "many prompts", "split rows", "decode")] +
                         [("prompts", -2, 1), ("many prompts", 0, 1), ("many prompts", -2, 1), ("many prompts", -2, 3)])
def test_a_wait_that_runs_out_leaves_rows_right_or_nan_and_the_next_call_right(name, cta, start, withhold):
    """With a CTA that loads nothing, or nothing after its first piece of work, and with all of them."""
    call, args = calls_to_stop()[name]
    want = call(*args)
    assert mk.serving_status() == (0, "ok") and not want.isnan().any()
    out = torch.full_like(want, 7.0)
    withhold(cta, start)
    call(*args, out=out)
    withhold(-1, 0)
    after = call(*args)  # on the same workspace
    lost = out.isnan()
    assert torch.equal(out[~lost], want[~lost])
    assert torch.equal(after, want)
    assert lost.all() if cta == -2 and start == 0 else lost.any() and (cta == -2 or not lost.all())
    assert mk.serving_status()[0] == 4 and mk.serving_status()[0] == 0


# ---- calls ----------------------------------------------------------------------------------

@pytest.mark.parametrize("which", ["k_cache", "v_cache"])
def test_append_refuses_a_cache_whose_heads_are_one(which):
    c = Cache([20, 30], 2, 128, 16)
    cos, sin = mk.rope_tables(64, DEV)
    caches = {"k_cache": c.kc, "v_cache": c.vc}
    caches[which] = caches[which][:, :1].expand(-1, 2, -1, -1)
    with pytest.raises(ValueError, match=which):
        mk.paged_append(rand(seeded(0), 2, 8, 128), **caches, block_table=c.table, kv_lens=c.lens, cos=cos, sin=sin)


def captured(call, n):
    """A graph of n calls; the pool's memory is the graph's."""
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [call() for _ in range(n)]
    return graph, out


def test_a_captured_call_clears_no_more_than_its_counters():
    """A captured attention call has a workspace of its own, of tens of MB: clearing it all would
    take longer than the call."""
    c = Cache([33], 8, 128, 16)
    q = rand(seeded(1), 1, 16, 128)
    want = mk.paged_attention(q, c.kc, c.vc, c.table, c.lens)
    n = 28

    def layers():
        for _ in range(n):
            mk.paged_attention(q, c.kc, c.vc, c.table, c.lens)

    graph, out = captured(lambda: mk.paged_attention(q, c.kc, c.vc, c.table, c.lens), n)
    direct, replayed = elapsed(layers), elapsed(graph.replay)
    assert all(torch.equal(x, want) for x in out)
    assert replayed < direct + n * 6e-3, (direct, replayed)  # ms: 6 us a call


def test_append_from_fp32_with_strides_of_four_elements():
    """16 bytes are four FP32 values: strides need be no more."""
    c = Cache([20, 30], 2, 128, 16)
    cos, sin = mk.rope_tables(64, DEV)
    wide = rand(seeded(3), 2, 9, 132, dtype=torch.float32)
    qkv = wide[:, 1:, 4:]
    assert qkv.stride(0) % 8 and qkv.stride(1) % 8
    q = mk.paged_append(qkv, c.kc, c.vc, c.table, c.lens, cos, sin)
    want = mk.paged_append(qkv.contiguous(), c.kc, c.vc, c.table, c.lens, cos, sin)
    assert torch.equal(q, want)


def test_more_tokens_and_requests_than_can_be_counted_are_refused():
    n = 2 ** 20
    pool = torch.zeros((1, 8, 16, 64), dtype=BF, device=DEV)
    table, lens, cu = (torch.zeros(s, dtype=torch.int32, device=DEV) for s in ((n, 1), (n,), (n + 1,)))
    with pytest.raises(ValueError, match="tokens"):
        mk.paged_attention(torch.zeros((1, 1024, 64), dtype=BF, device=DEV), pool, pool, table, lens, cu)


def test_errors_are_kept_where_the_first_call_of_a_process_is_captured():
    import os
    import subprocess
    import sys
    code = """if True:
        import torch
        import megakernel_b200 as mk
        pool = torch.zeros((3, 2, 16, 128), dtype=torch.bfloat16, device="cuda")
        table, lens = (torch.full(s, 7, dtype=torch.int32, device="cuda") for s in ((2, 1), (2,)))
        q = torch.zeros((2, 4, 128), dtype=torch.bfloat16, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = mk.paged_attention(q, pool, pool, table, lens)
        assert mk.serving_status() == (0, "ok")
        graph.replay()
        assert out.isnan().all()
        code = mk.serving_status()[0]
        assert code == 1, code
        lens.fill_(0)
        graph.replay()
        assert bool((out == 0).all()) and mk.serving_status()[0] == 0
        print("kept")
    """
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "kept" in r.stdout, r.stderr[-2000:]


def test_append_to_a_pool_without_pages_or_a_table_without_entries():
    """Nothing can be stored: what needs a page is reported, what needs none is not."""
    cos, sin = mk.rope_tables(64, DEV)
    qkv = rand(seeded(4), 2, 8, 128)
    pool = torch.empty((0, 2, 16, 128), dtype=BF, device=DEV)
    some = torch.zeros((3, 2, 16, 128), dtype=BF, device=DEV)
    table = torch.zeros((2, 4), dtype=torch.int32, device=DEV)
    lens = torch.tensor([0, 5], dtype=torch.int32, device=DEV)
    for caches, entries, code in ((pool, table, 1), (some, table[:, :0], 2)):
        q = mk.paged_append(qkv, caches, caches.clone(), entries, lens, cos, sin)
        assert bool((q[0] == 0).all()) and q[1].isnan().all()
        assert mk.serving_status()[0] == code
    q = mk.paged_append(qkv, some, some.clone(), table, lens, cos[:0], sin[:0])
    assert bool((q[0] == 0).all()) and q[1].isnan().all() and mk.serving_status()[0] == 3


@pytest.mark.parametrize("bad", [NAN, INF])
def test_append_before_position_0_gives_zeros_whatever_the_token_holds(bad):
    c = Cache([0, 30], 2, 128, 16)
    cos, sin = mk.rope_tables(64, DEV)
    w = rand(seeded(6), 128)
    for norm in (dict(), dict(q_norm=w, k_norm=w)):
        qkv = rand(seeded(5), 2, 8, 128)
        qkv[0, 0, 3] = qkv[0, 5, 100] = bad
        q, k = mk.paged_append(qkv, c.kc, c.vc, c.table, c.lens, cos, sin, return_k=True, **norm)
        assert bool((q[0] == 0).all()) and bool((k[0] == 0).all()) and q[1].isfinite().all()


@pytest.mark.parametrize("new", [1, 40])
def test_lengths_past_two_to_the_thirty_are_reported(new):
    """A table may list a page many times; keys are counted in 32 bits, with room for a tile."""
    pool = torch.zeros((1, 1, 2 ** 16, 64), dtype=BF, device=DEV)
    table = torch.zeros((2, 2 ** 15), dtype=torch.int32, device=DEV)
    q = torch.zeros((2 * new, 1, 64), dtype=BF, device=DEV)
    cu = None if new == 1 else cu_of([new, new])
    for n in (2 ** 31 - 1, 2 ** 30 + 1):
        lens = torch.tensor([50, n], dtype=torch.int32, device=DEV)
        got = mk.paged_attention(q, pool, pool, table, lens, cu)
        assert bool((got[:new] == 0).all()) and got[new:].isnan().all()
        assert mk.serving_status()[0] == 2
    lens = torch.tensor([50, -2 ** 31], dtype=torch.int32, device=DEV)  # no keys: tokens before position 0
    assert bool((mk.paged_attention(q, pool, pool, table, lens, cu) == 0).all())
    cos = torch.ones((64, 64), device=DEV)
    qkv = torch.ones((2 * new, 3, 64), dtype=BF, device=DEV)
    got = mk.paged_append(qkv, pool, pool.clone(), table, lens, cos, cos, cu)
    assert bool((got[new:] == 0).all()) and mk.serving_status() == (0, "ok")
