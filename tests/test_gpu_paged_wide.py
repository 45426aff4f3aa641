"""aarh_paged_attention where a call has much to do (tiles of 128 rows) or many sequences (two column tiles a workgroup), and the
paged operators' rarer legal calls: pools past 4 GiB, shared pages, odd scales and prefixes, a captured chain."""
import numpy as np
import pytest
import torch

import aarambh_hip as A
import paged_util as U
from test_gpu_paged import DEV, TYPES, f64, run_attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    m = U.context()
    yield m
    m.close()


def much(rows, n_kv, nh, hd, kv):
    """A bound on the cached tokens with which the call's work (rows of a kv head x kv heads x 32-token blocks) is past
    what tiles of 16 or 32 rows are taken for: 540000, twice as much at head_dim 64, eight times over INT8."""
    most = 540000 * (2 if hd == 64 else 1) * (8 if kv == "int8" else 1)
    return 32 * (most // (max(rows) * (nh // n_kv) * len(rows) * n_kv) + 2)


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_wide_tiles(ctx, act, kv, hd):
    rows = [131, 70, 40]
    run_attention(ctx, np.random.default_rng(112), act, kv, 2, 6, hd, 64, [131, 200, 77], rows, extra_rows=5, strided=True,
                  max_kv=much(rows, 2, 6, hd, kv))
    # whole blocks behind and in front of the rows, one sequence without rows, one with a single row
    rows = [33, 0, 1, 64]
    run_attention(ctx, np.random.default_rng(113), act, kv, 1, 4, hd, 32, [700, 50, 257, 64], rows, grouped=True,
                  max_kv=much(rows, 1, 4, hd, kv))


@pytest.mark.parametrize("act,kv", [("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "int8")])
@pytest.mark.parametrize("how", [
    dict(window=40, prefix=[0, 0, 0, 0]), dict(window=1, prefix=[0, 0, 0, 0]), dict(window=64, prefix=[0, 5, 40, 200]),
    dict(prefix=[1, 0, 64, 1000]), dict(softcap=5.0), dict(softcap=30.0, scale=0.5), dict(slopes=[0.5, 0.25, 0.0, -0.01]),
    dict(slopes=[1.0, 0.1, 0.03, 0.01], softcap=10.0, window=50, prefix=[3, 3, 3, 3], grouped=True)])
def test_wide_tiles_with_masks(ctx, act, kv, how):
    rows = [90, 40, 70, 33]
    run_attention(ctx, np.random.default_rng(114), act, kv, 2, 4, 64, 32, [90, 47, 170, 225], rows,
                  max_kv=much(rows, 2, 4, 64, kv), **how)


def test_wide_tiles_with_a_window_alone(ctx):
    run_attention(ctx, np.random.default_rng(115), "f16", "f16", 8, 8, 128, 32, [70 + 9 * i for i in range(16)], [70] * 16, window=40)


def test_wide_tiles_peaked_and_shifted_scores(ctx):
    for seed, how in ((116, dict(q_scale=30.0)), (117, dict(q_scale=1e-6)), (118, dict(q_scale=1e6, scale=1e-6))):
        act = "f16" if how["q_scale"] == 30.0 else "f32"
        run_attention(ctx, np.random.default_rng(seed), act, "f16", 1, 2, 64, 32, [700], [150], max_kv=much([150], 1, 2, 64, "f16"), **how)


def test_wide_tiles_with_bad_pages(ctx):
    rows = [40, 70]
    run_attention(ctx, np.random.default_rng(119), "f16", "f16", 2, 4, 64, 32, [100, 150], rows, bad=[(0, 1), (1, 0), (1, 3)],
                  max_kv=much(rows, 2, 4, 64, "f16"))
    rows = [20, 70]
    run_attention(ctx, np.random.default_rng(120), "f16", "int8", 2, 4, 64, 32, [20, 150], rows, bad=[(0, 0)],
                  max_kv=much(rows, 2, 4, 64, "int8"))


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("hd,nseq,tokens", [(128, 17, 5), (128, 9, 20), (64, 33, 7), (64, 16, 20)])
def test_many_sequences(ctx, act, kv, hd, nseq, tokens):
    """Two 16-row tiles a workgroup, one workgroup a kv head and several."""
    lens = [tokens + 13 * i % 90 for i in range(nseq)]
    run_attention(ctx, np.random.default_rng(121), act, kv, 8, 32, hd, 32, lens, [tokens] * nseq)


@pytest.mark.parametrize("rows,wide", [([1, 2], False), ([40, 60], False), ([40, 60], True)])
@pytest.mark.parametrize("how", [dict(scale=-0.2), dict(scale=0.0), dict(scale=-0.2, softcap=4.0), dict(prefix=[-5, 2 ** 31 - 1]),
                                 dict(window=2 ** 31 - 1), dict(window=7, prefix=[3, -1])])
def test_odd_scales_windows_and_prefixes(ctx, rows, how, wide):
    run_attention(ctx, np.random.default_rng(122), "f16", "f16", 2, 4, 64, 32, [50, 130], rows,
                  max_kv=much(rows, 2, 4, 64, "f16") if wide else None, **how)


@pytest.mark.parametrize("kv", ["f16", "int8"])
def test_pools_past_4_gib(ctx, kv):
    """The last pages of a pool whose keys alone pass 4 GiB (elements too, for INT8) are written and read like the first."""
    rng = np.random.default_rng(123)
    n_kv, hd, page = 8, 128, 256
    n = (1 << 32) // (n_kv * hd * page) + 40 if kv == "int8" else (1 << 32) // (n_kv * hd * page * 2) + 40
    big, small = A.PagePool.allocate(n, n_kv, hd, page, U.KV[kv]), A.PagePool.allocate(4, n_kv, hd, page, U.KV[kv])
    act = torch.float16
    total, heads = 300, 8
    q = torch.from_numpy(rng.standard_normal((total, heads, hd)).astype(np.float32)).to(DEV).to(act)
    k, v = (torch.from_numpy(rng.standard_normal((total, n_kv, hd)).astype(np.float32)).to(DEV).to(act) for _ in range(2))
    inv = torch.from_numpy(A.rope_frequencies(hd)[0]).to(DEV)
    one = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    outs = []
    for pool, pages in ((big, [n - 1, n - 3]), (small, [1, 2])):
        bt = A.PageBatch(one(*pages)[None], one(total), one(0, total), rows=total, max_rows=total, max_kv=512)
        r = ctx.rope_append(pool, bt, q, k, v, inv)
        step = A.PageBatch(one(*pages)[None], one(total), one(0, 1), rows=1, max_rows=1, max_kv=512)
        outs.append([r, ctx.paged_attention(pool, step, r[-1:].contiguous()), ctx.paged_attention(pool, bt, r)] + pool.read(pages))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    # the tiles of 128 rows too (a wide table: the bound makes the call large)
    bound = much([total], n_kv, heads, hd, kv)
    for pool, pages in ((big, [n - 1, n - 3]), (small, [1, 2])):
        table = torch.full((1, -(-bound // page)), -1, dtype=torch.int32, device=DEV)
        table[0, :2] = one(*pages)
        outs.append(ctx.paged_attention(pool, A.PageBatch(table, one(total), one(0, total), rows=total, max_rows=total, max_kv=bound), q))
    assert torch.equal(outs[-1], outs[-2])


def test_sequences_share_pages(ctx):
    """A prompt's full pages in two tables (one of them twice in a table): read like copies."""
    cache = U.Cache(np.random.default_rng(124), "f16", 2, 64, 32, [96, 70, 70])
    cache.tables[1, :2] = cache.tables[0, :2]
    cache.tables[2, 1] = cache.tables[2, 0]
    q = torch.randn((6, 4, 64), device=DEV, dtype=torch.float16, generator=torch.Generator(DEV).manual_seed(2))
    # the tail of the second sequence lies in a page of its own
    bt = cache.batch([2, 2, 2])
    got = ctx.paged_attention(cache.pool, bt, q)
    want, mag, err = U.attention_reference(cache, f64(q), [2, 2, 2], 64 ** -0.5)
    assert np.all(np.abs(f64(got) - want) <= U.attention_bound(want, mag, err, "f16", "f16", 96))
    # one table for several sequences has to be laid out: a row stride of 0 cannot hold them
    t = torch.from_numpy(cache.tables[:1]).to(DEV).expand(3, -1)
    one = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    with pytest.raises(A.ShapeError):
        ctx.paged_attention(cache.pool, A.PageBatch(t, one(90, 80, 70), one(0, 2, 4, 6), rows=6, max_rows=2, max_kv=96), q)


def test_a_captured_decode_step(ctx):
    """rope_append, paged_attention and process_logits in one graph, whose inputs move on between the replays (lengths, rows, history
    on the device; bounds of the longest): every replay gives what eager calls on a copy of the cache give."""
    rng = np.random.default_rng(125)
    nseq, nh, n_kv, hd, V, steps = 3, 8, 2, 64, 512, 40
    start = [31, 1, 70]
    most = max(start) + steps
    caches = [U.Cache(np.random.default_rng(126), "f16", n_kv, hd, 32, [n + steps for n in start], max_kv=most) for _ in range(2)]
    dev = lambda a, dt: torch.from_numpy(np.ascontiguousarray(a)).to(dt).to(DEV)  # noqa: E731
    tables = dev(caches[0].tables, torch.int32)
    lens, off = torch.zeros(nseq, dtype=torch.int32, device=DEV), dev(np.arange(nseq + 1), torch.int32)
    qkv = torch.zeros((nseq, (nh + 2 * n_kv) * hd), device=DEV, dtype=torch.float16)
    hist, gain = torch.zeros((nseq, most), dtype=torch.int32, device=DEV), torch.randn(V, device=DEV) * 5
    pen, plen = dev([[1.3, 0.5, 0.2]] * nseq, torch.float32), dev(start, torch.int32)
    inv = torch.from_numpy(A.rope_frequencies(hd)[0]).to(DEV)

    def step(cache, bt):
        q, k, v = (t.unflatten(1, (-1, hd)) for t in qkv.split([nh * hd, n_kv * hd, n_kv * hd], 1))
        q = ctx.rope_append(cache.pool, bt, q, k, v, inv)
        o = ctx.paged_attention(cache.pool, bt, q, window=50)
        y = o.float().reshape(nseq, V) * gain  # (a library's reduction may record memory sets, which replays get wrong)
        return o, y, ctx.process_logits(y, hist, lens, plen, pen)

    bts = [A.PageBatch(tables, lens, off, rows=nseq, max_rows=1, max_kv=most) for _ in range(2)]
    lens.copy_(dev([n + 1 for n in start], torch.int32))
    step(caches[1], bts[1])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(caches[0], bts[0])
    for i in range(steps):
        lens.copy_(dev([n + 1 + i for n in start], torch.int32))
        qkv.copy_(dev(rng.standard_normal(tuple(qkv.shape)), torch.float16))
        hist[:, i] = dev(rng.integers(0, V, nseq), torch.int32)
        want = step(caches[1], bts[1])
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), i
    for a, b in zip(caches[0].t, caches[1].t):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("wide,how", [(False, {}), (False, dict(window=6)), (True, {}), (True, dict(window=20, prefix=[0, 3])),
                                      (False, dict(prefix=[9, 0]))])
def test_infinities_and_nan_reach_only_the_rows_that_see_them(ctx, act, kv, hd, wide, how):
    """Keys and values of tokens that some rows of a call see and others, beside them in a tile, do not."""
    rows = [60, 45] if wide else [7, 5]
    lens = [75, 45 + 64]
    cache = U.Cache(np.random.default_rng(128), kv, 2, hd, 32, lens)
    inf, nan = float("inf"), float("nan")

    def plant(which, b, tok, h, dim, value):
        page, at = int(cache.tables[b, tok // 32]), tok % 32
        if kv == "int8":
            cache.st[which][page, h, at] = value
        else:
            cache.t[which][page, h, int((cache.v_at if which else cache.k_at)[at, dim])] = value

    # 16-bit pools: single elements; INT8: a token's scale.  (row of the token, kv head, dimension, value)
    r0 = [n - r for n, r in zip(lens, rows)]
    plant(1, 0, r0[0] + 3, 0, 5, inf)
    plant(1, 0, r0[0] + 5, 0, hd - 1, nan)
    plant(1, 0, r0[0] + 5, 1, 17, -inf)
    plant(1, 1, r0[1] + 2, 1, 40, -inf)
    plant(1, 1, r0[1] + 4, 1, 40, inf)
    plant(0, 1, r0[1] + 3, 0, 8, nan)
    nh = 8
    q = torch.randn((sum(rows), nh, hd), device=DEV, generator=torch.Generator(DEV).manual_seed(3)).to(U.DT[act])
    args = dict(how)
    if "prefix" in args:
        args["prefix"] = torch.tensor(args["prefix"], dtype=torch.int32, device=DEV)
    bt = cache.batch(rows, max_kv=much(rows, 2, nh, hd, kv) if wide else None)
    if wide:
        table = torch.full((2, bt._c.max_kv // 32 + 1), -1, dtype=torch.int32, device=DEV)
        table[:, :cache.tables.shape[1]] = bt.tables
        bt = A.PageBatch(table, bt.kv_len, bt.row_off, rows=sum(rows), max_rows=max(rows), max_kv=bt._c.max_kv)
    got = f64(ctx.paged_attention(cache.pool, bt, q, **args))
    with np.errstate(invalid="ignore"):
        want, mag, err = U.attention_reference(cache, f64(q), rows, hd ** -0.5, **how)
        fine = np.isfinite(want)
        assert 0 < fine.sum() < fine.size
        bound = U.attention_bound(want, mag, err, act, kv, max(lens))
        assert np.all(np.isfinite(got[fine]))
        off = np.abs(got - want)
        live = fine & np.isfinite(bound)
        assert np.all(off[live] <= bound[live]), (off[live] / bound[live]).max()
        assert not np.any(np.isfinite(got[~fine]))
        # (f32 rows have weights of two halves, of which the second may be zero or negative: with an infinity that makes NaN)
        if kv != "int8" and act != "f32":
            assert np.array_equal(got[~fine], want[~fine], equal_nan=True)


def test_grids_past_their_bound_are_refused(ctx):
    pool = A.PagePool.allocate(1, 8, 64, 32)
    n, rows = 60000, 2300
    zeros = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=DEV)  # noqa: E731
    q = torch.ones((rows, 8, 64), dtype=torch.float16, device=DEV)
    out = torch.full_like(q, 5.0)
    with pytest.raises(A.ShapeError):
        ctx.paged_attention(pool, A.PageBatch(zeros(n, 72), zeros(n), zeros(n + 1), rows=rows, max_rows=rows, max_kv=2300), q, out=out)
    # as many sequences without rows, in a call made for one row each: nothing to do
    ctx.paged_attention(pool, A.PageBatch(zeros(n, 1), zeros(n), zeros(n + 1), rows=rows, max_rows=1, max_kv=32), q, out=out)
    assert torch.all(out == 5.0)


@pytest.mark.parametrize("act,kv,hd,rows,lens", [("f16", "f16", 128, [300], [900]), ("bf16", "bf16", 64, [300, 280], [700, 900]),
                                                 ("f32", "f16", 128, [290], [1500])])
def test_many_rows_over_a_few_splits(ctx, act, kv, hd, rows, lens):
    cache, q, out = run_attention(ctx, np.random.default_rng(127), act, kv, 8, 32, hd, 64, lens, rows, max_kv=2500)
    bt = cache.batch(rows, max_kv=2500)
    assert torch.equal(ctx.paged_attention(cache.pool, bt, q), out)
    splits = next(iter(bt._workspace.values())) / (sum(rows) * 32 * (hd + 2) * 4)
    assert 2 <= splits <= 512 // hd, splits


def test_calls_from_two_threads(ctx):
    """One context, two threads with streams and batches of their own: the results of calls one after another."""
    import threading
    made = []
    for seed in (129, 130):
        cache = U.Cache(np.random.default_rng(seed), "f16", 2, 64, 32, [400, 90])
        q = torch.randn((6, 8, 64), device=DEV, generator=torch.Generator(DEV).manual_seed(seed)).half()
        want = ctx.paged_attention(cache.pool, cache.batch([3, 3]), q)
        made.append((cache, q, want, []))
    torch.cuda.synchronize()

    def work(cache, q, want, got):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            bt = cache.batch([3, 3])
            stream.synchronize()
            for _ in range(50):
                got.append(ctx.paged_attention(cache.pool, bt, q))
        stream.synchronize()

    threads = [threading.Thread(target=work, args=m) for m in made]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for _, _, want, got in made:
        assert len(got) == 50 and all(torch.equal(g, want) for g in got)
