"""Inputs and 64-bit references of the paged-cache operators and the logits processor (numpy, on the CPU)."""
import math

import numpy as np
import torch

import aarambh_hip as A

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
KV = {"f16": A.KV_F16, "bf16": A.KV_BF16, "int8": A.KV_INT8}
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step of a rounding, relative
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}  # smallest step
EPS32 = 1.1920928955078125e-07


def context():
    return A.HipModel(A.ModelConfig(vocab_size=128, hidden_dim=128, ffn_dim=128, n_layers=1, n_heads=1, n_kv_heads=1,
                                    max_seq_len=16), max_batch=1, max_rows=16)


def k_index(page, hd, i8):
    """Place of (token, dim) in a page of keys / values, from the documented orders."""
    n = 32 * hd
    blocks = np.arange(page // 32) * n
    if i8:
        k = np.arange(n).reshape(2, hd // 64, 4, 4, 4, 2, 8).transpose(3, 0, 4, 1, 2, 5, 6)  # a s b c g h j
        v = np.arange(n).reshape(hd // 32, 4, 16, 2, 8).transpose(1, 4, 0, 3, 2)  # g j p h r
    else:
        k = np.arange(n).reshape(2, hd // 64, 2, 4, 4, 4, 8).transpose(4, 0, 5, 1, 3, 2, 6)
        v = np.arange(n).reshape(hd, 32).T
    full = lambda x: (blocks[:, None, None] + x.reshape(32, hd)).reshape(page, hd)  # noqa: E731
    return full(k), full(v)


class Cache:
    """A pool and page tables for sequences of `lens` tokens, filled with random values (NaN where no token lies)."""

    def __init__(self, rng, kv, n_kv, hd, page, lens, extra_pages=2, max_kv=None, fill=True, spread=1.0):
        self.kv, self.n_kv, self.hd, self.page, self.lens = kv, n_kv, hd, page, list(lens)
        self.i8 = kv == "int8"
        used = [-(-n // page) for n in lens]
        self.n_pages = sum(used) + extra_pages
        ids = rng.permutation(self.n_pages).astype(np.int32)
        most = max(max(used), -(-(max_kv or 0) // page), 1)
        self.tables = np.full((len(lens), most), -7, np.int32)
        at = 0
        for b, n in enumerate(used):
            self.tables[b, :n] = ids[at:at + n]
            at += n
        self.k_at, self.v_at = k_index(page, hd, self.i8)
        shape = (self.n_pages, n_kv, page * hd)
        nat = (self.n_pages, n_kv, page, hd)
        self.scales = [None, None]
        if self.i8:
            data = [rng.integers(-127, 128, nat).astype(np.int8) for _ in range(2)]
            # scales of tokens that no sequence has are NaN
            self.scales = [(0.005 + 0.02 * rng.random(nat[:3])).astype(np.float16) for _ in range(2)]
        else:
            data = [rng.standard_normal(nat).astype(np.float32) * spread for _ in range(2)]
        live = np.zeros((self.n_pages, page), bool)
        for b, n in enumerate(lens):
            for t in range(n):
                live[self.tables[b, t // page], t % page] = True
        self.live = live
        if fill:
            for x, sc in zip(data, self.scales):
                if self.i8:
                    sc.transpose(0, 2, 1)[~live] = np.nan
                else:
                    x.transpose(0, 2, 1, 3)[~live] = np.nan
        dev = torch.device("cuda:0")
        self.t = []
        for x, at_ in zip(data, (self.k_at, self.v_at)):
            flat = np.empty(shape, x.dtype)
            flat[:, :, at_.reshape(-1)] = x.reshape(self.n_pages, n_kv, -1)
            t = torch.from_numpy(flat).to(dev)
            self.t.append(t if self.i8 else t.to(DT[kv]))
        self.st = [None if s is None else torch.from_numpy(s).to(dev) for s in self.scales]
        self.pool = A.PagePool(self.t[0], self.t[1], n_kv, hd, page, self.st[0], self.st[1])

    def values(self, which):
        """All pages as f64 [n_pages, n_kv, page, hd] from the device."""
        at = self.v_at if which else self.k_at
        x = self.t[which].double().cpu().numpy()[:, :, at]
        if self.i8:
            x = x * self.st[which].double().cpu().numpy()[..., None]
        return x

    def tokens(self, which, b, n=None):
        """Keys or values of a sequence's tokens, [n, n_kv, hd] f64."""
        n = self.lens[b] if n is None else n
        x = self.values(which)
        return np.stack([x[self.tables[b, t // self.page], :, t % self.page] for t in range(n)]) if n else \
            np.zeros((0, self.n_kv, self.hd))

    def batch(self, rows, total=None, max_rows=None, max_kv=None, status=None, lens=None):
        off = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        lens = self.lens if lens is None else lens
        dev = torch.device("cuda:0")
        return A.PageBatch(torch.from_numpy(self.tables).to(dev), torch.tensor(lens, dtype=torch.int32, device=dev),
                           torch.from_numpy(off).to(dev), rows=int(off[-1]) if total is None else total,
                           max_rows=max(rows, default=0) if max_rows is None else max_rows,
                           max_kv=max(lens, default=0) if max_kv is None else max_kv, status=status)


def attention_reference(cache, q, rows, scale, softcap=0.0, window=0, slopes=None, prefix=None, grouped=False,
                        skip_pages=()):
    """o and, per output, sum_j p_j |v_j| and the largest score error of f32 arithmetic (f64, [rows, heads, hd] / [rows,
    heads, 1]): q f64 [rows, heads, hd].  Tokens of table places in skip_pages [(b, place)] are absent."""
    nh, hd = q.shape[1:]
    G = nh // cache.n_kv
    out, mag, err = np.zeros(q.shape), np.zeros(q.shape), np.zeros((q.shape[0], nh, 1))
    r0 = 0
    for b, r in enumerate(rows):
        n = cache.lens[b]
        k, v = cache.tokens(0, b), cache.tokens(1, b)
        j = np.arange(n)
        here = np.array([(b, t // cache.page) not in skip_pages for t in range(n)], bool)
        for h in range(nh):
            g = h // G if grouped else h % cache.n_kv
            for i in range(r):
                p = n - r + i
                seen = (j <= p) & ((window == 0) | (p - j < window))
                if prefix is not None:
                    seen |= j < prefix[b]
                seen &= here
                if not seen.any():
                    continue
                prod = q[r0 + i, h] * k[seen, g]
                s = prod.sum(1) * scale
                size = np.abs(prod).sum(1) * abs(scale)
                if softcap:
                    s = softcap * np.tanh(s / softcap)
                if slopes is not None:
                    s = s + slopes[h] * (j[seen] - p)
                # dot products of hd f32 terms (the split of f32 queries loses 2^-22 of each), then a few
                # roundings of the score, its bias and the exponent's argument
                err[r0 + i, h] = ((hd + 8) * 2.0 ** -24 + 2.0 ** -22) * size.max() + 2.0 ** -21 * (np.abs(s).max() + abs(
                    softcap) + (0 if slopes is None else abs(slopes[h]) * (p + n)) + 1)
                w = np.exp(s - s.max())
                w /= w.sum()
                out[r0 + i, h] = w @ v[seen, g]
                mag[r0 + i, h] = w @ np.abs(v[seen, g])
        r0 += r
    return out, mag, err


def attention_bound(out, mag, err, act, kv, n):
    """How far the operator may be off: a score error e moves every weight by exp(2 e) at most; weights are
    rounded to the pool's 16 bits for the product with V (f32 queries keep two such halves: 2^-21);
    sums over n tokens in f32; the result is rounded once."""
    w = 2.0 ** -21 if act == "f32" else HALF["bf16" if kv == "bf16" else "f16"]
    return 1.001 * HALF[act] * np.abs(out) + mag * (np.expm1(2 * err) + w * 1.01 + (n + 64) * 2.0 ** -24) + TINY[act]


def rope_reference(x, pos, inv, attn, rot, interleaved):
    """x f64 [rows, heads, hd] rotated, and the size |x| + |y| that its roundings go by."""
    y, size = x.copy(), np.abs(x)
    ang = pos[:, None].astype(np.float64) * inv
    c, s = (np.cos(ang) * attn)[:, None], (np.sin(ang) * attn)[:, None]
    i = np.arange(rot // 2)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    both = (np.abs(a) + np.abs(b)) * attn
    size[..., first] = size[..., second] = both
    return y, size


def logits_reference(x, R, hist, hist_len, prompt_len, pen, draft, bias, masks, mask_of_row):
    """Rows in f64 and the size that their f32 roundings go by.  bias: list of (ids, values) per sequence."""
    x = x.astype(np.float64)
    out, size = x.copy(), np.abs(x)
    V = x.shape[1]
    for row in range(x.shape[0]):
        b, t = divmod(row, R)
        n = 0 if hist is None else min(max(int(hist_len[b]), 0), hist.shape[1])
        h = hist[b, :n].astype(np.int64) & 0xFFFFFFFF if n else np.zeros(0, np.int64)
        cut = 0 if prompt_len is None else min(max(int(prompt_len[b]), 0), n)
        new = np.concatenate([h[cut:], draft[b, :t].astype(np.int64) & 0xFFFFFFFF if draft is not None else h[:0]])
        r, p, f = (1.0, 0.0, 0.0) if pen is None else pen[b].astype(np.float64)
        seen = np.zeros(V, bool)
        seen[[w for w in np.concatenate([h[:cut], new]) if w < V]] = True
        count = np.bincount(new[new < V], minlength=V)
        y = np.where(seen, np.where(x[row] > 0, x[row] / r, x[row] * r), x[row])
        s = np.abs(y) + np.where(count > 0, abs(p), 0) + abs(f) * count
        y = y - np.where(count > 0, p, 0) - f * count
        if bias is not None:
            table = dict(zip([int(u) for u in bias[b][0]], [float(v) for v in bias[b][1]]))
            for w, val in table.items():
                if 0 <= w < V:
                    y[w] += val
                    s[w] += abs(val)
        if masks is not None:
            m = int(mask_of_row[row])
            if m != -1:
                bits = np.zeros(V, bool) if not 0 <= m < masks.shape[0] else np.unpackbits(
                    np.ascontiguousarray(masks[m]).view(np.uint8), bitorder="little")[:V].astype(bool)
                y = np.where(bits, y, -math.inf)
        out[row], size[row] = y, s
    return out, size
