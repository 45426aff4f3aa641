"""aarh_process_logits against its definition in 64 bits: sizes and strides, histories with repeated tokens, verify rows, the
same token twice in a bias list, masks that leave a row empty, values that are not finite, in place, graphs."""
import numpy as np
import pytest
import torch

import aarambh_hip as A
import paged_util as U

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ctx():
    m = U.context()
    yield m
    m.close()


def make(rng, B, R, V, n, bias=0, masks=0, draft=True, pad=0):
    c = dict(R=R, x=rng.standard_normal((B * R, V)).astype(np.float32) * 4)
    c["hist"] = rng.integers(0, max(1, min(V, 2 * n)), (B, n)).astype(np.int32) if n else None
    c["hist_len"] = rng.integers(0, n + 1, B).astype(np.int32) if n else None
    c["prompt_len"] = (c["hist_len"] // 2).astype(np.int32) if n else None
    c["pen"] = np.stack([0.8 + rng.random(B), rng.random(B) - 0.3, rng.random(B)], 1).astype(np.float32)
    c["draft"] = rng.integers(0, V, (B, R - 1)).astype(np.int32) if draft and R > 1 else None
    if c["draft"] is not None and R > 2:
        c["draft"][:, 1] = c["draft"][:, 0]  # the same proposal twice
    c["bias"] = [(rng.integers(0, V, bias - b % 2), (rng.standard_normal(bias - b % 2) * 5).astype(np.float32))
                 for b in range(B)] if bias else None
    c["masks"] = rng.integers(0, 1 << 32, (masks, -(-V // 32)), dtype=np.uint32) if masks else None
    c["mask_of_row"] = rng.integers(-1, masks, B * R).astype(np.int32) if masks else None
    return c


def call(ctx, c, out=None, x=None):
    dev = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(DEV)  # noqa: E731
    b = c["bias"]
    ids = vals = off = None
    if b is not None:
        ids = np.concatenate([i for i, _ in b]).astype(np.int64).astype(np.uint32).view(np.int32)
        vals = np.concatenate([v for _, v in b]).astype(np.float32)
        off = np.concatenate([[0], np.cumsum([len(i) for i, _ in b])]).astype(np.int32)
    return ctx.process_logits(dev(c["x"]) if x is None else x, dev(c["hist"]), dev(c["hist_len"]), dev(c["prompt_len"]),
                              dev(c["pen"]), rows_per_seq=c["R"], draft=dev(c["draft"]), bias_off=dev(off), bias_ids=dev(ids),
                              bias_vals=dev(vals), masks=None if c["masks"] is None else dev(c["masks"].view(np.int32)),
                              mask_of_row=dev(c["mask_of_row"]), out=out)


def check(c, got):
    want, size = U.logits_reference(c["x"], c["R"], c["hist"], c["hist_len"], c["prompt_len"], c["pen"], c["draft"], c["bias"],
                                    c["masks"], c["mask_of_row"])
    got = got.double().cpu().numpy()
    live = np.isfinite(want)
    assert np.array_equal(got[~live], want[~live], equal_nan=True)
    # a quotient or product, two products and differences, a sum: five roundings of at most 2^-24 of the terms
    assert np.all(np.abs(got - want)[live] <= 6 * 2.0 ** -24 * size[live] + 2.0 ** -149)


@pytest.mark.parametrize("B,R,V,n", [(1, 1, 1, 1), (1, 1, 5, 3), (2, 1, 31, 0), (3, 2, 33, 7), (1, 4, 1000, 500),
                                     (5, 3, 4099, 100), (2, 6, 50257, 2000), (64, 1, 257, 40), (1, 2, 128001, 300)])
@pytest.mark.parametrize("bias,masks", [(0, 0), (9, 3)])
def test_rows(ctx, B, R, V, n, bias, masks):
    c = make(np.random.default_rng([B, R, V]), B, R, V, n, bias, masks)
    check(c, call(ctx, c))


def test_each_part_alone(ctx):
    for drop in (("hist", "hist_len", "prompt_len"), ("prompt_len",), ("pen",), ("draft",), ("bias",), ("masks", "mask_of_row")):
        c = make(np.random.default_rng(3), 3, 4, 777, 50, 6, 2)
        for k in drop:
            c[k] = None
        check(c, call(ctx, c))


def test_ids_and_lengths_outside_are_cut(ctx):
    c = make(np.random.default_rng(4), 3, 3, 300, 20, 5, 2)
    c["hist"][:, ::3] = [[-1], [300], [1 << 30]]
    c["hist"][:, 1] = -2147483648
    c["hist_len"][:] = [1000, -5, 20]
    c["prompt_len"][:] = [-3, 50, 2000]
    c["draft"][0, 0], c["draft"][1, 1] = -1, 300
    c["bias"][0][0][1] = 4_000_000_000
    c["bias"][2][0][0] = 300
    check(c, call(ctx, c))


def test_bias_lists_with_a_token_twice_use_the_last_value(ctx):
    c = make(np.random.default_rng(5), 2, 2, 64, 0, 0, 0)
    ids = np.array([7, 9, 7, 63, 7, 9] * 100)
    vals = np.arange(600).astype(np.float32)
    c["bias"] = [(ids, vals), (ids[::-1].copy(), vals)]
    got = call(ctx, c)
    check(c, got)
    for _ in range(5):
        assert torch.equal(call(ctx, c), got)
    # offsets past the arrays are cut, not read
    off = torch.tensor([-4, 2, 1 << 20], dtype=torch.int32, device=DEV)
    x = torch.zeros((4, 64), device=DEV)
    y = ctx.process_logits(x, rows_per_seq=2, bias_off=off, bias_ids=torch.tensor([1, 2, 3], dtype=torch.int32, device=DEV),
                           bias_vals=torch.tensor([1.0, 2.0, 3.0], device=DEV))
    want = torch.zeros((4, 64))
    want[:2, 1], want[:2, 2], want[2:, 3] = 1, 2, 3
    assert torch.equal(y.cpu(), want)


def test_masks_that_leave_nothing_and_values_that_are_not_finite(ctx):
    c = make(np.random.default_rng(6), 2, 3, 100, 10, 4, 3)
    c["masks"][0] = 0
    c["masks"][1] = 0xFFFFFFFF
    c["mask_of_row"][:] = [0, 1, 2, -1, 3, -2]  # the last two are no masks: everything masked
    c["x"][:, 5], c["x"][:, 6], c["x"][:, 7] = np.inf, -np.inf, np.nan
    got = call(ctx, c).cpu().numpy()
    want, size = U.logits_reference(c["x"], 3, c["hist"], c["hist_len"], c["prompt_len"], c["pen"], c["draft"], c["bias"],
                                    c["masks"], c["mask_of_row"])
    for r in (0, 4, 5):
        assert np.all(got[r] == -np.inf)
    live = np.isfinite(want)
    assert np.array_equal(got[~live], want[~live].astype(np.float32), equal_nan=True)
    assert np.all(np.abs(got - want)[live] <= 6 * 2.0 ** -24 * size[live])
    status = ctx.accept_sample(torch.from_numpy(got[:1][:, None]).to(DEV), None, None, A.Sampler.top_k_top_p(1.0), True,
                               seeds=torch.zeros(1, dtype=torch.int64, device=DEV))["status"]
    assert status.tolist() == [1]  # an empty row is no distribution


@pytest.mark.parametrize("V,ld", [(1000, 1024), (1001, 1003), (64, 65)])
def test_strided_and_in_place(ctx, V, ld):
    c = make(np.random.default_rng(7), 3, 2, V, 60, 5, 2)
    buf = torch.full((6, ld), 9.0, device=DEV)
    buf[:, :V] = torch.from_numpy(c["x"]).to(DEV)
    want = call(ctx, c)
    out = torch.full((6, ld + 3), 5.0, device=DEV)
    assert torch.equal(call(ctx, c, out=out[:, :V], x=buf[:, :V]), want)
    assert torch.all(out[:, V:] == 5) and torch.all(buf[:, V:] == 9)
    call(ctx, c, out=buf[:, :V], x=buf[:, :V])
    assert torch.equal(buf[:, :V], want) and torch.all(buf[:, V:] == 9)
    shifted = torch.full((6 * ld + 1,), 9.0, device=DEV)[1:].view(6, ld)  # rows that are 4-byte aligned only
    shifted[:, :V] = torch.from_numpy(c["x"]).to(DEV)
    assert torch.equal(call(ctx, c, x=shifted[:, :V]), want)


def test_graph_replays_with_new_histories(ctx):
    c = make(np.random.default_rng(8), 4, 3, 5000, 200, 10, 2)
    x = torch.from_numpy(c["x"]).to(DEV)
    hist, n = torch.from_numpy(c["hist"]).to(DEV), torch.from_numpy(c["hist_len"]).to(DEV)
    draft, pen = torch.from_numpy(c["draft"]).to(DEV), torch.from_numpy(c["pen"]).to(DEV)
    out = torch.empty_like(x)
    run = lambda o: ctx.process_logits(x, hist, n, None, pen, rows_per_seq=3, draft=draft, out=o)  # noqa: E731
    run(out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run(out)
    for rep in range(4):
        hist.copy_(torch.randint(0, 5000, hist.shape, device=DEV, dtype=torch.int32))
        n.copy_(torch.randint(0, 201, n.shape, device=DEV, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, run(None))
        c["hist"], c["hist_len"], c["prompt_len"] = hist.cpu().numpy(), n.cpu().numpy(), None
        c["bias"] = c["masks"] = c["mask_of_row"] = None
        check(c, got)


def test_wrong_tensors_refused(ctx):
    x = torch.zeros((4, 50), device=DEV)
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)  # noqa: E731
    with pytest.raises(A.ShapeError):
        ctx.process_logits(x, rows_per_seq=3)
    with pytest.raises(A.UnsupportedError):
        ctx.process_logits(x.half())
    with pytest.raises(A.ConfigError):
        ctx.process_logits(x.cpu())
    with pytest.raises(A.UnsupportedError):
        ctx.process_logits(x.T)
    with pytest.raises(A.ShapeError):
        ctx.process_logits(x, i(3, 5), i(4))
    with pytest.raises(A.ConfigError):
        ctx.process_logits(x, i(4, 5))
    with pytest.raises(A.ShapeError):
        ctx.process_logits(x, rows_per_seq=2, draft=i(2, 0))
    with pytest.raises(A.ShapeError):
        ctx.process_logits(x, masks=i(1, 1), mask_of_row=i(4))
    with pytest.raises(A.ConfigError):
        ctx.process_logits(x, bias_off=i(5))
    with pytest.raises(A.UnsupportedError):
        ctx.process_logits(x, penalties=torch.zeros((4, 3), dtype=torch.float64, device=DEV))
    assert ctx.process_logits(x[:0]).shape == (0, 50)
