"""aarh_rope_append and aarh_paged_attention against their definitions in 64 bits: types, head layouts, lengths from one
token on, pages that end inside a block, strided rows, masks, bad pages and lengths, streams, graphs, and a run of
decode steps as a server makes them."""
import math

import numpy as np
import pytest
import torch

import aarambh_hip as A
import paged_util as U

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "int8"), ("f16", "int8")]


@pytest.fixture(scope="module")
def ctx():
    m = U.context()
    yield m
    m.close()


def f64(t):
    return t.double().cpu().numpy()


# ---------------------------------------------------------------------------
# rope + append
# ---------------------------------------------------------------------------
def run_rope(ctx, rng, act, kv, n_kv, nh, hd, page, rot, interleaved, lens, rows, strided=False, attn_factor=1.0,
             extra_rows=0, bad=(), theta=10000.0):
    """One call; checks queries, stored tokens, and that everything else stayed as it was."""
    cache = U.Cache(rng, kv, n_kv, hd, page, lens)
    for b, place in bad:
        cache.tables[b, place] = cache.n_pages + 3 if place % 2 else -1
    total = sum(rows) + extra_rows
    w = (nh + 2 * n_kv) * hd
    if strided:  # views of a fused projection with a gap behind each row
        buf = torch.from_numpy(rng.standard_normal((total, w + 64)).astype(np.float32)).to(DEV).to(U.DT[act])
        q, k, v = (x.unflatten(1, (-1, hd)) for x in buf[:, :w].split([nh * hd, n_kv * hd, n_kv * hd], 1))
    else:
        mk = lambda h: torch.from_numpy(rng.standard_normal((total, h, hd)).astype(np.float32)).to(DEV).to(U.DT[act])  # noqa: E731
        q, k, v = mk(nh), mk(n_kv), mk(n_kv)
    inv, _ = A.rope_frequencies(rot, theta) if rot else (None, 1.0)
    status = torch.zeros(len(rows), dtype=torch.int32, device=DEV)
    before = [t.clone() for t in cache.t] + [None if s is None else s.clone() for s in cache.st]
    out = torch.full((total, nh, hd), 7.0, dtype=U.DT[act], device=DEV)
    got = ctx.rope_append(cache.pool, cache.batch(rows, total=total, status=status), q, k, v,
                          None if inv is None else torch.from_numpy(inv).to(DEV), attn_factor, interleaved, out=out)
    torch.cuda.synchronize()
    assert got is out
    pos = np.concatenate([np.arange(n - r, n) for n, r in zip(lens, rows)]).astype(np.int64)
    seq = np.repeat(np.arange(len(rows)), rows)
    m = len(pos)
    ident = lambda x: (x, np.abs(x))  # noqa: E731
    turn = (lambda x: U.rope_reference(x, pos, inv, attn_factor, rot, interleaved)) if rot else ident
    want, size = turn(f64(q)[:m])
    # cos and sin are each off by 3 units at most and take one rounding with attn_factor; two products, one sum
    slack = lambda s: 8 * 2.0 ** -24 * s  # noqa: E731
    err = np.abs(f64(out)[:m] - want)
    assert np.all(err <= U.HALF[act] * np.abs(want) * 1.001 + slack(size) + U.TINY[act]), err.max()
    assert torch.all(out[m:] == 7.0)
    untouched = np.ones((cache.n_pages, page), bool)
    for which, x in ((0, turn(f64(k)[:m])), (1, ident(f64(v)[:m]))):
        x, size = x
        pages = cache.values(which)
        for r in range(m):
            place = pos[r] // page
            if (seq[r], place) in bad:
                continue
            got_row = pages[cache.tables[seq[r], place], :, pos[r] % page]
            untouched[cache.tables[seq[r], place], pos[r] % page] = False
            if kv == "int8":
                top = np.abs(x[r]).max(-1, keepdims=True) + slack(size[r]).max(-1, keepdims=True)
                unit = np.where(top <= U.EPS32, 1.0, top / 127)
                # half a code, the fp16 scale's rounding on up to 127 codes, the f32 errors before it
                bound = unit * (0.5 + 127 * 2.0 ** -11 + 2.0 ** -14) * 1.001 + slack(size[r]) + 2.0 ** -24
            else:
                bound = U.HALF[kv] * np.abs(x[r]) * 1.001 + slack(size[r]) + U.TINY[kv]
            assert np.all(np.abs(got_row - x[r]) <= bound), (which, r, np.abs(got_row - x[r]).max())
    # nothing else in the pool moved (NaN included)
    same = lambda a, b: torch.equal(a.view(torch.uint8), b.view(torch.uint8))  # noqa: E731
    for which in range(2):
        at = cache.v_at if which else cache.k_at
        a, b = cache.t[which][:, :, torch.from_numpy(at).to(DEV)], before[which][:, :, torch.from_numpy(at).to(DEV)]
        keep = torch.from_numpy(untouched).to(DEV)
        assert same(a.transpose(1, 2)[keep].contiguous(), b.transpose(1, 2)[keep].contiguous())
        if cache.st[which] is not None:
            assert same(cache.st[which].transpose(1, 2)[keep].contiguous(), before[2 + which].transpose(1, 2)[keep].contiguous())
    want_status = [1 if any((b, p // page) in bad for p in range(n - r, n)) else 0
                   for b, (n, r) in enumerate(zip(lens, rows))]
    assert status.tolist() == want_status
    return cache


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("hd,rot,interleaved", [(128, 128, False), (128, 32, True), (64, 64, True), (64, 16, False), (128, 0, False)])
def test_rope_append_types_and_layouts(ctx, act, kv, hd, rot, interleaved):
    rng = np.random.default_rng(1)
    run_rope(ctx, rng, act, kv, 2, 6, hd, 32, rot, interleaved, [1, 33, 70, 97], [1, 2, 5, 66], attn_factor=1.25)


@pytest.mark.parametrize("page", [32, 64, 128, 256])
def test_rope_append_pages_and_lengths(ctx, page):
    rng = np.random.default_rng(2)
    # one token, whole blocks, ends inside a block, no rows, rows behind the last sequence, far positions
    run_rope(ctx, rng, "f16", "f16", 3, 7, 64, page, 32, False, [1, 64, 95, 40, 31, 300], [1, 64, 95, 0, 1, 3],
             strided=True, extra_rows=4)


@pytest.mark.parametrize("act,kv", TYPES)
def test_rope_append_strided_and_one_head(ctx, act, kv):
    rng = np.random.default_rng(3)
    run_rope(ctx, rng, act, kv, 1, 1, 128, 64, 128, True, [50], [50], strided=True, extra_rows=1)


def test_rope_angles_of_far_positions(ctx):
    """Position 10^9 - 1 in 64-bit angles: an angle rounded to f32 is off by up to 32 radians there.  The page table
    reaches there through a table whose rows hold only the last page (entries before it are read by nothing)."""
    rng = np.random.default_rng(4)
    n, page = 1_000_000_000, 256
    places = -(-n // page)
    tables = torch.full((1, places), -1, dtype=torch.int32, device=DEV)
    tables[0, -1] = 0
    k = torch.randn((2, 2, 64), dtype=torch.float32, device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    pool = A.PagePool.allocate(1, 2, 64, page)
    one = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    bt = A.PageBatch(tables, one(n), one(0, 2), rows=2, max_rows=2, max_kv=n)
    inv, _ = A.rope_frequencies(64, 10000.0)
    got = ctx.rope_append(pool, bt, k, k, k, torch.from_numpy(inv).to(DEV))
    want, size = U.rope_reference(f64(k), np.array([n - 2, n - 1]), inv, 1.0, 64, False)
    # position * inv_freq / 2 pi in f64 is off by 1.5e-8 turns at most (two roundings of 1.6e8 turns); the reference's own
    # angle by one rounding of 1e9 radians
    slack = 2 * math.pi * 3.6e8 * 2.0 ** -53 + 1e9 * 2.0 ** -53 + 8 * 2.0 ** -24
    assert np.all(np.abs(f64(got) - want) <= slack * size + 2.0 ** -24 * np.abs(want))
    kk, vv = pool.read([0])
    at = (n - 2) % page
    assert np.all(np.abs(f64(kk)[at:at + 2] - want) <= U.HALF["f16"] * np.abs(want) + slack * size + 2.0 ** -24)
    assert torch.equal(vv[at:at + 2], k.half().float())


def test_rope_append_bad_pages_and_lengths(ctx):
    rng = np.random.default_rng(5)
    run_rope(ctx, rng, "f16", "f16", 2, 4, 64, 32, 64, False, [70, 40], [70, 40], bad=[(0, 1), (1, 0)])
    # contradictory sequences are left out, the others are not
    cache = U.Cache(rng, "f16", 2, 64, 32, [40, 40, 40, 40])
    before = [t.clone() for t in cache.t]
    q = torch.randn((12, 4, 64), device=DEV, dtype=torch.float16)
    k = torch.randn((12, 2, 64), device=DEV, dtype=torch.float16)
    status = torch.zeros(4, dtype=torch.int32, device=DEV)
    bt = A.PageBatch(torch.from_numpy(cache.tables).to(DEV), torch.tensor([2, 40, 41, 40], dtype=torch.int32, device=DEV),
                     torch.tensor([0, 3, 6, 9, 13], dtype=torch.int32, device=DEV), rows=12, max_rows=3, max_kv=40, status=status)
    out = torch.full_like(q, 3.0)
    ctx.rope_append(cache.pool, bt, q, k, k, out=out)
    assert status.tolist() == [2, 0, 2, 2]
    assert torch.all(out[:3] == 3) and torch.all(out[6:] == 3) and torch.equal(out[3:6], q[3:6])
    for b in (0, 2, 3):
        pages = torch.from_numpy(cache.tables[b]).long().to(DEV)
        for t, old in zip(cache.t, before):
            assert torch.equal(t[pages].view(torch.int16), old[pages].view(torch.int16))
    o = ctx.paged_attention(cache.pool, bt, q, out=out)
    assert torch.all(o[:3] == 3) and torch.all(o[6:] == 3) and torch.isfinite(o[3:6]).all()


def test_rope_in_place_and_without_queries(ctx):
    rng = np.random.default_rng(6)
    cache, other = (U.Cache(np.random.default_rng(6), "f16", 2, 64, 32, [5, 9]) for _ in range(2))
    q = torch.randn((6, 4, 64), device=DEV, dtype=torch.float16)
    k = torch.randn((6, 2, 64), device=DEV, dtype=torch.float16)
    inv = torch.from_numpy(A.rope_frequencies(64)[0]).to(DEV)
    bt = cache.batch([2, 4])
    want = ctx.rope_append(cache.pool, bt, q, k, k, inv)
    assert ctx.rope_append(cache.pool, bt, None, k, k, inv) is None
    for t, o in zip(cache.t, other.t):
        assert not torch.equal(t.view(torch.int16), o.view(torch.int16))
    ctx.rope_append(other.pool, bt, None, k, k, inv)
    for t, o in zip(cache.t, other.t):
        assert torch.equal(t.view(torch.int16), o.view(torch.int16))
    ctx.rope_append(cache.pool, bt, q, k, k, inv, out=q)
    assert torch.equal(q, want)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def run_attention(ctx, rng, act, kv, n_kv, nh, hd, page, lens, rows, extra_rows=0, strided=False, bad=(), q_scale=1.0,
                  max_rows=None, max_kv=None, **how):
    cache = U.Cache(rng, kv, n_kv, hd, page, lens, max_kv=max_kv)
    total = sum(rows) + extra_rows
    buf = torch.from_numpy((rng.standard_normal((total, nh * hd + (64 if strided else 0))) * q_scale).astype(np.float32))
    q = buf.to(DEV).to(U.DT[act])[:, :nh * hd].unflatten(1, (nh, hd))
    o_buf = torch.full((total, nh * hd + (128 if strided else 0)), 7.0, dtype=U.DT[act], device=DEV)
    out = o_buf[:, :nh * hd].unflatten(1, (nh, hd))
    for b, place in bad:
        cache.tables[b, place] = cache.n_pages if place % 2 else -2
    status = torch.zeros(len(rows), dtype=torch.int32, device=DEV)
    args = dict(how)
    for name, dt in (("slopes", np.float32), ("prefix", np.int32)):
        if args.get(name) is not None:
            args[name] = torch.from_numpy(np.asarray(args[name], dt)).to(DEV)
    bt = cache.batch(rows, total=total, max_rows=max_rows, max_kv=max_kv, status=status)
    ctx.paged_attention(cache.pool, bt, q, out=out, **args)
    torch.cuda.synchronize()
    for b, place in bad:
        cache.tables[b, place] = 0  # the reference's tokens() looks there and drops what it finds
    m = sum(rows)
    ref = {k: v for k, v in how.items() if k != "scale"}
    want, mag, err = U.attention_reference(cache, f64(q)[:m], rows, how.get("scale", hd ** -0.5), skip_pages=set(bad), **ref)
    off = np.abs(f64(out)[:m] - want)
    bound = U.attention_bound(want, mag, err, act, kv, max(lens))
    assert np.all(off <= bound), (off.max(), (off / bound).max(), np.unravel_index((off / bound).argmax(), off.shape))
    # far inside the bound as a whole: the norm of the error goes by the roundings' mean square
    norm = np.linalg.norm(want)
    tight = {"f32": 2e-6, "f16": 6e-4, "bf16": 5e-3}[act]
    assert np.linalg.norm(off) <= tight * norm, np.linalg.norm(off) / norm
    assert torch.all(out[m:] == 7.0) and torch.all(o_buf[:, nh * hd:] == 7.0)
    bits = [0] * len(rows)
    for b, place in bad:
        bits[b] = 1
    assert status.tolist() == bits
    return cache, q, out


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("n_kv,nh,hd", [(2, 8, 128), (2, 6, 64), (1, 7, 64), (3, 3, 128)])
def test_attention_types_and_heads(ctx, act, kv, n_kv, nh, hd):
    # single tokens: contexts of one token, inside a block, block and page edges, several pages
    run_attention(ctx, np.random.default_rng(10), act, kv, n_kv, nh, hd, 64, [1, 2, 31, 32, 33, 64, 65, 130, 300], [1] * 9)


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_verify_rows(ctx, act, kv, hd):
    run_attention(ctx, np.random.default_rng(11), act, kv, 2, 8, hd, 32, [5, 40, 97, 200, 33, 64], [5, 4, 1, 9, 0, 12],
                  extra_rows=3, strided=True, grouped=True)


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_chunks(ctx, act, kv, hd):
    # a prompt from nothing, a chunk behind cached tokens, odd ends
    run_attention(ctx, np.random.default_rng(12), act, kv, 2, 6, hd, 64, [131, 200, 77], [131, 70, 40])


@pytest.mark.parametrize("act,kv", [("f16", "f16"), ("bf16", "bf16"), ("f32", "int8")])
@pytest.mark.parametrize("how", [
    dict(window=1), dict(window=40), dict(window=64, prefix=[0, 5, 40, 200]), dict(prefix=[1, 0, 64, 1000]),
    dict(softcap=5.0), dict(softcap=30.0, scale=0.5), dict(slopes=[0.5, 0.25, 0.0, -0.01]),
    dict(slopes=[1.0, 0.1, 0.03, 0.01], softcap=10.0, window=50, prefix=[3, 3, 3, 3], grouped=True)])
@pytest.mark.parametrize("rows", [[1, 1, 1, 1], [3, 5, 2, 4], [90, 40, 70, 33]])
def test_attention_masks(ctx, act, kv, how, rows):
    run_attention(ctx, np.random.default_rng(13), act, kv, 2, 4, 64, 32, [90, 47, 170, 225], rows, **how)


@pytest.mark.parametrize("act,kv", TYPES)
def test_attention_split_over_long_contexts(ctx, act, kv):
    run_attention(ctx, np.random.default_rng(14), act, kv, 1, 4, 128, 256, [4100, 1, 2300], [2, 1, 3], max_kv=5000)


def test_attention_peaked_and_shifted_scores(ctx):
    # scores of some hundreds: one key takes all, and the running maximum moves late
    run_attention(ctx, np.random.default_rng(15), "f16", "f16", 1, 2, 64, 32, [700], [3], q_scale=30.0)
    run_attention(ctx, np.random.default_rng(16), "f32", "f16", 1, 2, 64, 32, [700], [150], q_scale=1e-6)
    run_attention(ctx, np.random.default_rng(17), "f32", "f16", 1, 2, 64, 32, [200], [70], q_scale=1e6, scale=1e-6)


@pytest.mark.parametrize("rows", [[1, 1], [40, 70]])
def test_attention_bad_pages_count_as_absent(ctx, rows):
    run_attention(ctx, np.random.default_rng(18), "f16", "f16", 2, 4, 64, 32, [100, 150], rows, bad=[(0, 1), (1, 0), (1, 3)])
    run_attention(ctx, np.random.default_rng(19), "f16", "int8", 2, 4, 64, 32, [20, 150], rows if rows[0] == 1 else [20, 70],
                  bad=[(0, 0)])  # nothing left for the first sequence: zeros


@pytest.mark.parametrize("rows,window", [(1, 0), (4, 0), (100, 0), (1, 40)])
def test_attention_on_other_streams_and_in_graphs(ctx, rows, window):
    """Two captured calls replayed on two streams at once, between eager calls."""
    made = []
    for seed in (20, 21):
        rng = np.random.default_rng(seed)
        cache = U.Cache(rng, "f16", 2, 128, 64, [1500, 900])
        q = torch.from_numpy(rng.standard_normal((2 * rows, 8, 128)).astype(np.float32)).to(DEV).half()
        bt = cache.batch([rows, rows])
        want = ctx.paged_attention(cache.pool, bt, q, window=window)
        made.append((cache, q, bt, want))
    torch.cuda.synchronize()
    graphs = []
    for cache, q, bt, want in made:
        g = torch.cuda.CUDAGraph()
        out = torch.empty_like(want)
        with torch.cuda.graph(g):
            ctx.paged_attention(cache.pool, bt, q, window=window, out=out)
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    for rep in range(4):
        for (g, out), st in zip(graphs, streams):
            out.zero_()
        torch.cuda.synchronize()
        for (g, out), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        eager = ctx.paged_attention(made[0][0].pool, made[0][2], made[0][1], window=window)
        torch.cuda.synchronize()
        for (g, out), m in zip(graphs, made):
            assert torch.equal(out, m[3]), rep
        assert torch.equal(eager, made[0][3])


def test_operators_refuse_wrong_tensors(ctx):
    rng = np.random.default_rng(22)
    cache = U.Cache(rng, "f16", 2, 64, 32, [10])
    bt = cache.batch([2])
    q = torch.zeros((2, 4, 64), dtype=torch.float16, device=DEV)
    k = q[:, :2]
    with pytest.raises(A.ConfigError):
        ctx.paged_attention(cache.pool, bt, q.cpu())
    with pytest.raises(A.ShapeError):
        ctx.paged_attention(cache.pool, bt, q[:1])
    with pytest.raises(A.ShapeError):
        ctx.paged_attention(cache.pool, bt, q[:, :3])
    with pytest.raises(A.UnsupportedError):
        ctx.paged_attention(cache.pool, bt, q.double())
    with pytest.raises(A.UnsupportedError):
        ctx.paged_attention(cache.pool, bt, q.bfloat16())
    with pytest.raises(A.UnsupportedError):
        ctx.paged_attention(cache.pool, bt, q.transpose(0, 1).contiguous().transpose(0, 1))
    with pytest.raises(A.ShapeError):
        ctx.paged_attention(cache.pool, bt, q, slopes=torch.zeros(3, device=DEV))
    with pytest.raises(A.ShapeError):
        ctx.paged_attention(cache.pool, cache.batch([2], max_kv=33), q)
    with pytest.raises(A.UnsupportedError):
        ctx.rope_append(cache.pool, bt, q, k.contiguous(), k.float().contiguous())
    with pytest.raises(A.ShapeError):
        ctx.rope_append(cache.pool, bt, q, q, q)
    with pytest.raises(A.UnsupportedError):
        ctx.rope_append(cache.pool, bt, q, k.contiguous(), k.contiguous(), torch.zeros(4, dtype=torch.float64, device=DEV))
    with pytest.raises(A.UnsupportedError):
        ctx.rope_append(cache.pool, bt, q, k.contiguous(), k.contiguous(), torch.zeros(8, device=DEV))
    with pytest.raises(A.UnsupportedError):
        A.PagePool(cache.t[0].float(), cache.t[1].float(), 2, 64, 32)
    with pytest.raises(A.ShapeError):
        A.PagePool(cache.t[0], cache.t[1], 2, 64, 64)


def test_pool_read_gives_tokens(ctx):
    for kv in ("f16", "int8"):
        cache = U.Cache(np.random.default_rng(23), kv, 2, 128, 64, [100])
        got = cache.pool.read(cache.tables[0, :2])
        for which in range(2):
            assert np.array_equal(f64(got[which])[:100].astype(np.float32), cache.tokens(which, 0).astype(np.float32))


# ---------------------------------------------------------------------------
# a run of them together
# ---------------------------------------------------------------------------
def test_prompt_then_decode_steps_then_sampling(ctx):
    """Two requests of a one-layer attention model: prompts in chunks, then decode steps (rope_append, paged_attention,
    LM head, process_logits, accept_sample), in f32 rows over fp16 pages.  The tokens are those of a plain f64
    run of the same model over its whole history at every step."""
    rng = np.random.default_rng(30)
    nh, n_kv, hd, page, V, H = 4, 2, 64, 32, 256, 256
    embed = rng.standard_normal((V, H)) * 0.5
    wqkv = rng.standard_normal((H, (nh + 2 * n_kv) * hd)) * H ** -0.5
    head = rng.standard_normal((nh * hd, V)) * 4 * (nh * hd) ** -0.5
    inv, _ = A.rope_frequencies(hd, 10000.0)
    prompts = [rng.integers(1, V, 45), rng.integers(1, V, 7)]
    pen = np.array([[1.3, 0.2, 0.1], [1.1, 0.0, 0.4]], np.float32)
    dev = lambda a, dt: torch.from_numpy(np.ascontiguousarray(a)).to(dt).to(DEV)  # noqa: E731

    def plain(tokens, b):
        """Processed logits after `tokens` from the definitions."""
        x = embed[tokens].astype(np.float32).astype(np.float64) @ wqkv
        n = len(tokens)
        q, k, v = np.split(x.reshape(n, nh + 2 * n_kv, hd), [nh, nh + n_kv], 1)
        pos = np.arange(n)
        q, k = U.rope_reference(q, pos, inv, 1.0, hd, False)[0], U.rope_reference(k, pos, inv, 1.0, hd, False)[0]
        o = np.zeros((nh, hd))
        for h in range(nh):
            s = k[:, h % n_kv] @ q[-1, h] / math.sqrt(hd)
            w = np.exp(s - s.max())
            o[h] = w @ v[:, h % n_kv] / w.sum()
        y = o.reshape(1, -1) @ head
        P = len(prompts[b])
        return U.logits_reference(y, 1, np.array([tokens]), [n], [P], pen[b:b + 1], None, None, None, None)[0][0]

    tables = torch.tensor([[3, 0, 5], [1, 4, 2]], dtype=torch.int32, device=DEV)
    pool = A.PagePool.allocate(6, n_kv, hd, page)
    w_dev, head_dev, inv_dev = dev(wqkv, torch.float32), dev(head, torch.float32), dev(inv, torch.float64)

    def forward(new, lens):
        rows = [len(t) for t in new]
        x = dev(embed[np.concatenate(new)], torch.float32) @ w_dev
        q, k, v = (t.unflatten(1, (-1, hd)) for t in x.split([nh * hd, n_kv * hd, n_kv * hd], 1))
        bt = A.PageBatch(tables, dev(np.array(lens), torch.int32), dev(np.concatenate([[0], np.cumsum(rows)]), torch.int32),
                         rows=sum(rows), max_rows=max(rows), max_kv=96)
        q = ctx.rope_append(pool, bt, q, k, v, inv_dev)
        o = ctx.paged_attention(pool, bt, q)
        return o.reshape(sum(rows), -1) @ head_dev, np.cumsum(rows) - 1

    done = [0, 0]
    seqs = [list(p) for p in prompts]
    for lo, hi in ((0, 20), (20, 45)):  # prompt chunks: the second request has its prompt in the first
        new = [p[lo:hi] for p in prompts]
        done = [min(len(p), hi) for p in prompts]
        last_logits, last = forward(new, done)
        if lo == 0:
            keep = last_logits[last[1]].clone()
    logits = torch.stack([last_logits[last[0]], keep])
    hist = np.zeros((2, 96), np.int32)
    for step in range(12):
        for b in range(2):
            hist[b, :len(seqs[b])] = seqs[b]
        y = ctx.process_logits(logits, dev(hist, torch.int32), dev([len(s) for s in seqs], torch.int32),
                               dev([len(p) for p in prompts], torch.int32), dev(pen, torch.float32))
        got = ctx.accept_sample(y[:, None].contiguous(), None, None, A.Sampler.greedy_sampler(), True,
                                seeds=torch.zeros(2, dtype=torch.int64, device=DEV))
        assert got["status"].tolist() == [0, 0]
        for b in range(2):
            want = plain(seqs[b], b)
            # fp16 keys and values: 2^-11 relative on each moves a logit by some 1e-3 of its size
            assert np.abs(f64(y)[b] - want).max() < 2e-2 * np.abs(want).max()
            order = np.sort(want)
            tok = int(got["token"][b])
            assert tok == int(np.argmax(want)) or want[tok] > order[-1] - 4e-2 * np.abs(want).max()
            seqs[b].append(tok)
        logits, _ = forward([s[-1:] for s in seqs], [len(s) for s in seqs])
