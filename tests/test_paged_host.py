"""The paged-cache operators without a GPU: csrc/paged_rule.hpp on the host, the argument checks of every entry
(which come before anything touches a device) and the frequency tables against the formulas in f64."""
import ctypes as C
import math
import os
import shutil
import subprocess

import numpy as np
import pytest

import aarambh_hip as A

HERE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "host")
PTR = 0x10000  # stands for a device array: never read before the checks are through


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_layouts_sequences_and_pages(tmp_path):
    exe = str(tmp_path / "paged_rule")
    subprocess.run(["g++", "-O2", "-std=c++17", "-o", exe, os.path.join(HERE, "paged_rule.cpp")], check=True)
    n, wrong = map(int, subprocess.run([exe], check=True, capture_output=True, text=True, timeout=60).stdout.split())
    assert n > 12000 and wrong == 0, (n, wrong)


@pytest.fixture(scope="module")
def ctx():
    """A context that has no device behind it (its number does not exist), good for its error text."""
    cfg = A._Cfg(128, 128, 128, 1, 1, 1, 16, 10000.0, 1e-5, 0, 0, 0, 0, 1, 16, 0)
    h = A._P()
    assert A.lib().aarh_create(1 << 20, C.byref(cfg), C.byref(h)) == 4 and h
    yield h
    A.lib().aarh_destroy(h)


def pool(**kw):
    p = dict(kv_format=A.KV_F16, n_kv_heads=2, head_dim=128, page_tokens=64, n_pages=4, k=PTR, v=PTR, k_scale=None,
             v_scale=None)
    p.update(kw)
    return A._PagePool(**p)


def batch(**kw):
    p = dict(nseq=2, rows=3, max_rows=2, max_kv=100, row_off=PTR, kv_len=PTR, tables=PTR, table_ld=2, status=None)
    p.update(kw)
    return A._PageBatch(**p)


def rope(**kw):
    p = dict(act=A.A_F16, n_heads=4, q=PTR, k=PTR, v=PTR, q_ld=512, k_ld=256, v_ld=256, q_out=PTR, q_out_ld=512,
             inv_freq=PTR, rot_dim=128, interleaved=0, attn_factor=1.0)
    p.update(kw)
    return A._RopeArgs(**p)


def attn(**kw):
    p = dict(act=A.A_F16, n_heads=4, grouped=0, q=PTR, q_ld=512, out=PTR, out_ld=512, scale=0.1, softcap=0.0, window=0,
             slopes=None, prefix=None, workspace=PTR, workspace_bytes=1 << 40)
    p.update(kw)
    return A._PagedAttnArgs(**p)


BAD_POOL = [(dict(kv_format=A.KV_F32), 3), (dict(kv_format=9), 3), (dict(head_dim=96), 3), (dict(head_dim=0), 3),
            (dict(page_tokens=48), 3), (dict(page_tokens=512), 3), (dict(page_tokens=16), 3), (dict(n_pages=0), 2),
            (dict(n_kv_heads=0), 2), (dict(k=None), 1), (dict(v=PTR + 8), 3), (dict(kv_format=A.KV_INT8), 1),
            (dict(kv_format=A.KV_BF16), 3)]  # (bf16 pages under fp16 rows)
BAD_BATCH = [(dict(nseq=-1), 2), (dict(nseq=70000), 2), (dict(rows=-1), 2), (dict(max_kv=-1), 2),
             (dict(max_kv=(1 << 30) + 1, table_ld=1 << 30), 2), (dict(row_off=None), 1), (dict(kv_len=None), 1),
             (dict(tables=None), 1), (dict(max_kv=129), 2)]


@pytest.mark.parametrize("kw,code", BAD_POOL)
def test_pools_refused(ctx, kw, code):
    L, n = A.lib(), C.c_int64()
    assert L.aarh_rope_append(ctx, pool(**kw), batch(), rope(), None) == code
    assert L.aarh_paged_attention(ctx, pool(**kw), batch(), attn(), None) == code
    assert L.aarh_paged_attention_workspace(ctx, pool(**kw), batch(), attn(), C.byref(n)) == code
    assert A.lib().aarh_last_error(ctx)


@pytest.mark.parametrize("kw,code", BAD_BATCH)
def test_batches_refused(ctx, kw, code):
    assert A.lib().aarh_rope_append(ctx, pool(), batch(**kw), rope(), None) == code
    assert A.lib().aarh_paged_attention(ctx, pool(), batch(**kw), attn(), None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(act=A.A_BF16), 3), (dict(act=7), 3), (dict(n_heads=-1), 2), (dict(rot_dim=8), 3), (dict(rot_dim=144), 3),
    (dict(rot_dim=-16), 3), (dict(inv_freq=None), 1), (dict(k=None), 1), (dict(q=None), 1), (dict(q_out=None), 1),
    (dict(q_ld=511), 2), (dict(k_ld=255), 2), (dict(v_ld=260), 3), (dict(q=PTR + 2), 3), (dict(q_out_ld=516), 3)])
def test_rope_arguments_refused(ctx, kw, code):
    assert A.lib().aarh_rope_append(ctx, pool(), batch(), rope(**kw), None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(act=A.A_BF16), 3), (dict(n_heads=3), 2), (dict(n_heads=0), 2), (dict(scale=math.nan), 1),
    (dict(scale=math.inf), 1), (dict(softcap=-1.0), 1), (dict(softcap=math.nan), 1), (dict(window=-1), 1),
    (dict(q=None), 1), (dict(out=None), 1), (dict(q_ld=500), 2), (dict(out=PTR + 8), 3), (dict(out_ld=516), 3)])
def test_attention_arguments_refused(ctx, kw, code):
    assert A.lib().aarh_paged_attention(ctx, pool(), batch(), attn(**kw), None) == code


def logits(**kw):
    p = dict(nseq=2, rows_per_seq=3, vocab=100, logits=PTR, ld=100, out=PTR, out_ld=100, history=PTR, history_ld=5,
             history_len=PTR, prompt_len=None, penalties=PTR, draft=PTR, draft_ld=2, bias_off=PTR, bias_ids=PTR,
             bias_vals=PTR, n_bias=4, masks=PTR, mask_ld=4, n_masks=1, mask_of_row=PTR)
    p.update(kw)
    return A._LogitsArgs(**p)


@pytest.mark.parametrize("kw,code", [
    (dict(nseq=-1), 2), (dict(nseq=70000), 2), (dict(rows_per_seq=-1), 2), (dict(vocab=-1), 2), (dict(logits=None), 1),
    (dict(out=None), 1), (dict(ld=99), 2), (dict(out_ld=99), 2), (dict(out_ld=101), 2), (dict(out=PTR + 2), 3),
    (dict(history_len=None), 1), (dict(history_ld=-1), 1), (dict(draft_ld=1), 2), (dict(bias_ids=None), 1),
    (dict(n_bias=-1), 1), (dict(mask_ld=3), 2), (dict(mask_of_row=None), 2), (dict(n_masks=-1), 2)])
def test_logits_arguments_refused(ctx, kw, code):
    assert A.lib().aarh_process_logits(ctx, logits(**kw), None) == code


def test_null_blocks_and_empty_calls(ctx):
    L, n = A.lib(), C.c_int64(-1)
    assert L.aarh_rope_append(None, pool(), batch(), rope(), None) == 1
    assert L.aarh_rope_append(ctx, None, batch(), rope(), None) == 1
    assert L.aarh_paged_attention(ctx, pool(), batch(), None, None) == 1
    assert L.aarh_process_logits(ctx, None, None) == 1
    # nothing to do: no launch, no array looked at
    for empty in (dict(nseq=0, row_off=None, kv_len=None, tables=None), dict(rows=0)):
        assert L.aarh_rope_append(ctx, pool(), batch(**empty), rope(k=None, v=None, q=None), None) == 0
        assert L.aarh_paged_attention(ctx, pool(), batch(**empty), attn(q=None, out=None), None) == 0
        assert L.aarh_paged_attention_workspace(ctx, pool(), batch(**empty), attn(), C.byref(n)) == 0 and n.value == 0
    for empty in (dict(nseq=0), dict(rows_per_seq=0), dict(vocab=0)):
        assert L.aarh_process_logits(ctx, logits(logits=None, **empty), None) == 0


@pytest.mark.parametrize("scaling", [None, A.RopeScaling("linear", 4.0, 4096), A.RopeScaling("ntk", 2.0, 4096),
                                     A.RopeScaling("yarn", 8.0, 4096, attn_factor=1.2)])
@pytest.mark.parametrize("rot,theta", [(128, 10000.0), (64, 500000.0), (16, 10000.0)])
def test_frequencies(scaling, rot, theta):
    inv, attn_factor = A.rope_frequencies(rot, theta, scaling, 1 << 17)
    i = np.arange(rot // 2)
    th = theta * (scaling.factor ** (rot / (rot - 2)) if scaling and scaling.method == "ntk" else 1.0)
    want = th ** (-2.0 * i / rot)
    if scaling and scaling.method == "linear":
        want = want / 4.0
    if scaling and scaling.method == "yarn":
        turns = 4096 * want / (2 * math.pi)  # rotations over the original context
        fast, slow = turns >= 32, turns <= 1
        np.testing.assert_allclose(inv[fast][:-1], want[fast][:-1], rtol=1e-13)
        np.testing.assert_allclose(inv[slow][1:], want[slow][1:] / 8, rtol=1e-13)
        assert np.all(inv <= want * (1 + 1e-13)) and np.all(inv >= want / 8 * (1 - 1e-13))
    else:
        np.testing.assert_allclose(inv, want, rtol=1e-13)
    assert attn_factor == np.float32(scaling.attn_factor if scaling else 1.0)


def test_frequencies_refused():
    for kw in (dict(rot_dim=0), dict(rot_dim=7), dict(rot_dim=1 << 20)):
        with pytest.raises(A.ShapeError):
            A.rope_frequencies(**kw)
    for kw in (dict(theta=0.0), dict(theta=math.nan), dict(theta=math.inf)):
        with pytest.raises(A.ConfigError):
            A.rope_frequencies(64, **kw)
    with pytest.raises(A.ConfigError, match="factor"):
        A.rope_frequencies(64, 10000.0, A.RopeScaling("linear", 1.0, 4096), 8192)
    with pytest.raises(A.ConfigError, match="max_seq_len"):
        A.rope_frequencies(64, 10000.0, A.RopeScaling("linear", 2.0, 4096), 1000)
