"""Plain float64 forms of the paged cache's operators, row by row, and batches
of ragged sequences to run them on (torch, on the tensors' own device)."""
import math

import numpy as np
import torch

F32, BF16 = torch.float32, torch.bfloat16
NAN = float("nan")


class Batch:
    """Sequences of (positions after the append, new tokens) on shuffled pages.

    The pools hold NaN except where fill() puts keys and values; the table
    names no page (-1, or far out of range) for pages without a position in
    use. pad: rows behind the last sequence; slack: how far the host's bounds
    lie above the lengths."""

    def __init__(self, seqs, H, KH, hd, page, q=F32, kv=F32, seed=0, pad=0, slack=0, dev="cuda",
                 extra_pages=3):
        self.seqs, self.H, self.KH, self.hd, self.P = seqs, H, KH, hd, page
        self.g = torch.Generator(device="cpu").manual_seed(seed)
        self.dev, self.qt, self.kt = dev, q, kv
        r = np.random.default_rng(seed)
        lens = np.array([a for a, _ in seqs], np.int32)
        toks = np.array([b for _, b in seqs], np.int32)
        held = -(-lens // page)
        self.n = len(seqs)
        self.max_q, self.max_kv = int(toks.max()) + slack, int(lens.max()) + slack
        self.ld = max(1, -(-self.max_kv // page))
        self.n_pages = max(1, int(held.sum())) + extra_pages
        order = r.permutation(self.n_pages)[:int(held.sum())]
        self.table_np = np.full((self.n, self.ld), -1, np.int32)
        at = 0
        for s in range(self.n):
            self.table_np[s, :held[s]] = order[at:at + held[s]]
            at += held[s]
        self.start_np = np.concatenate([[0], np.cumsum(toks)]).astype(np.int32)
        self.used = int(self.start_np[-1])
        self.rows = self.used + pad
        self.start, self.kv_len = self.put(self.start_np), self.put(lens)
        self.table = self.put(self.table_np)
        self.k = torch.full((self.n_pages, KH, page, hd), NAN, dtype=kv, device=dev)
        self.v = torch.full_like(self.k, NAN)

    def put(self, a):
        return torch.from_numpy(np.ascontiguousarray(a)).to(self.dev)

    def normal(self, *shape, dtype=F32, std=1.0):
        return (torch.randn(*shape, generator=self.g) * std).to(dtype).to(self.dev)

    def visible(self, s, window, sinks):
        """[new tokens, positions] of sequence s: which key each row sees."""
        T, n = self.seqs[s]
        p = torch.arange(T - n, T)[:, None]
        j = torch.arange(T)[None, :]
        m = j <= p
        if window:
            m = m & ((j > p - window) | (j < sinks))
        return m.to(self.dev)

    def fill(self, window=0, sinks=0, drop_pages=True):
        """Keys and values where some row sees them; pages that none sees leave the table."""
        for s, (T, n) in enumerate(self.seqs):
            if n == 0 or T == 0:
                if drop_pages:
                    self.table_np[s] = -1
                continue
            seen = self.visible(s, window, sinks).any(0).cpu().numpy()
            for i in range(-(-T // self.P)):
                here = np.flatnonzero(seen[i * self.P:(i + 1) * self.P])
                if here.size == 0:
                    if drop_pages:
                        self.table_np[s, i] = self.n_pages + 7
                    continue
                pg = int(self.table_np[s, i])
                slot = torch.from_numpy(here).to(self.dev)
                for t in (self.k, self.v):
                    t[pg, :, slot] = self.normal(self.KH, here.size, self.hd, dtype=self.kt)
        self.table = self.put(self.table_np)

    def history(self, pool, s):
        """[KH, positions, hd] float64 of sequence s; NaN where nothing was put."""
        T = self.seqs[s][0]
        n = -(-T // self.P)
        pg = torch.from_numpy(np.where(self.table_np[s, :n] < self.n_pages, self.table_np[s, :n], 0)
                              .clip(0).astype(np.int64)).to(self.dev)
        return pool[pg].double().transpose(0, 1).reshape(self.KH, n * self.P, self.hd)[:, :T]

    def attention(self, q, scale=None, window=0, sinks=0):
        """(out, sum_j p_j |v_j|, max_j scale sum |q||k_j|) in float64, [rows, H, hd] and [rows, H]."""
        hd, G = self.hd, self.H // self.KH
        scale = 1.0 / math.sqrt(hd) if scale is None else scale
        out = torch.zeros(self.rows, self.H, hd, dtype=torch.float64, device=self.dev)
        mag, dot = torch.zeros_like(out), torch.zeros(self.rows, self.H, dtype=torch.float64, device=self.dev)
        q = q.double().reshape(self.rows, self.H, hd)
        for s, (T, n) in enumerate(self.seqs):
            if n == 0 or T == 0:
                continue
            m = self.visible(s, window, sinks)
            K, V = (torch.nan_to_num(self.history(t, s), nan=0.0) for t in (self.k, self.v))
            a, z = int(self.start_np[s]), int(self.start_np[s + 1])
            for h in range(self.H):
                x, key, val = q[a:z, h], K[h // G], V[h // G]
                sc = (x @ key.t().contiguous()) * scale
                sc = sc.masked_fill(~m, -math.inf)
                top = sc.amax(-1, keepdim=True)
                e = torch.where(m, torch.exp(sc - torch.where(top > -math.inf, top, 0.0)), 0.0)
                l = e.sum(-1, keepdim=True)
                p = torch.where(l > 0, e / l.clamp(min=1e-300), 0.0)
                out[a:z, h] = p @ val
                mag[a:z, h] = p @ val.abs()
                big = (x.abs() @ key.abs().t().contiguous()) * scale
                dot[a:z, h] = torch.where(m, big, 0.0).amax(-1)
        return out, mag, dot


def attn_tolerance(out, mag, dot, hd, longest, bf16):
    """How far a row's outputs may be off. A score is a sum of hd products (times
    six term products) in fp32, each addition off by 2^-24 of what it has:
    |ds| <= (hd + 32) 2^-24 dot, and its place below the maximum is rounded once
    more; a weight exp(s) is then off by |ds| + 2^-22 (exp2's own error), and so
    is their sum, hence twice; the sums over the keys add (longest + 64) 2^-24.
    bf16 rows: the weights are rounded once (2^-8) and so is the output."""
    ds = (hd + 32) * 2.0 ** -24 * dot[..., None]
    t = (2 * ds + 2.0 ** -21 + (longest + 64) * 2.0 ** -24) * mag
    return t + (2.0 ** -8 * (mag + out.abs()) if bf16 else 0.0) + 1e-30


def append_rows(b, qkv, cos, sin, norm, eps, wq, wk, interleaved=False):
    """(q [rows, H, hd], k, v [rows, KH, hd]) in float64, and each row's (sequence, position)."""
    H, KH, hd = b.H, b.KH, b.hd
    x = qkv.double().reshape(b.rows, H + 2 * KH, hd)
    if interleaved:
        x = torch.cat([x[..., 0::2], x[..., 1::2]], -1)
    q, k, v = x[:, :H].clone(), x[:, H:H + KH].clone(), x[:, H + KH:]
    if norm:
        q = q / torch.sqrt((q * q).mean(-1, keepdim=True) + eps)
        k = k / torch.sqrt((k * k).mean(-1, keepdim=True) + eps)
        q = q if wq is None else q * wq.double()
        k = k if wk is None else k * wk.double()
    where = [(-1, -1)] * b.rows
    for s, (T, n) in enumerate(b.seqs):
        for i in range(n):
            where[int(b.start_np[s]) + i] = (s, T - n + i)
    if cos is not None:
        pos = torch.tensor([max(0, p) for _, p in where], device=b.dev)
        c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
        h = hd // 2
        q, k = (torch.cat([t[..., :h] * c + t[..., h:] * s, t[..., h:] * c - t[..., :h] * s], -1)
                for t in (q, k))
    return q, k, v, where


def draw_row(x, temp, top_k, top_p, min_p, u):
    """(id, probability) of one row from the definition, float64 on the host."""
    x = np.asarray(x, np.float64)
    ok = x > -math.inf  # (False for NaN)
    if not ok.any():
        return -1, 0.0
    first = int(np.flatnonzero(ok & (x == x[ok].max()))[0])
    if temp <= 0:
        return first, 1.0
    temp = 1.0 if math.isnan(temp) else temp
    m = x[first]
    e = np.zeros(len(x))
    with np.errstate(invalid="ignore"):
        e[ok] = np.where(x[ok] == m, 1.0, np.exp(np.where(x[ok] == m, 0.0, (x[ok] - m) / temp)))
    order = np.flatnonzero(ok)
    order = order[np.argsort(-x[order], kind="stable")]
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        c = np.cumsum(e[order])
        keep = np.concatenate([[0.0], c[:-1]]) < max(top_p, 0.0) * c[-1]
        keep[0] = True
        order = order[keep]
    if min_p > 0:
        order = order[e[order] >= min(min_p, 1.0)]
    kept = np.sort(order)
    c = np.cumsum(e[kept])
    u = min(max(u, 0.0), 1.0) if u == u else 0.0
    at = int(np.searchsorted(c, u * c[-1], side="right"))
    if at >= len(kept):  # u of 1 or more: the last id with mass
        at = int(np.flatnonzero(e[kept] > 0)[-1])
    return int(kept[at]), float(e[kept[at]] / c[-1])
