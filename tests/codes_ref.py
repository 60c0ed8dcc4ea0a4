"""Batches on 8-bit pages: pools of bytes (rows of codes, then their scales, a head
and page) beside the float64 values that they stand for."""
import torch

from autoresearch_amd import engine

from . import paged_ref as R

TYPES = {"i8": engine.FG_I8, "e4m3": engine.FG_E4M3}
TOP = {"i8": 127.0, "e4m3": 448.0}
TINY = 2.0 ** -126


def quantise(x, kind):
    """(codes as bytes, scales, float64 values) of fp32 rows, by the definition in fp32."""
    finite = torch.isfinite(x).all(-1, keepdim=True)
    top = torch.where(finite, x, 0.0).abs().amax(-1, keepdim=True)
    s = top / torch.full_like(top, TOP[kind])  # (by a number, torch multiplies with its rounded inverse on the GPU)
    s = torch.where(s < TINY, 0.0, s)
    y = torch.where(finite, x, 0.0) * torch.where(s > 0, 1.0 / s, 0.0)
    y = y.clamp(-TOP[kind], TOP[kind])
    y = y.round().to(torch.int8) if kind == "i8" else y.to(torch.float8_e4m3fn)
    s = torch.where(finite, s, R.NAN)
    return y.view(torch.uint8), s[..., 0], values(y.view(torch.uint8), kind) * s.double()


def values(codes, kind):
    return codes.view(torch.int8 if kind == "i8" else torch.float8_e4m3fn).float().double()


def views(pool, P, hd):
    """Codes [pages, heads, P, hd] and scales [pages, heads, P] of a pool."""
    return pool[..., :P * hd].unflatten(-1, (P, hd)), pool[..., P * hd:].view(torch.float32)


class Batch(R.Batch):
    """paged_ref's batch: k and v are the float64 values, kq and vq the pools. Rows that
    nobody filled have NaN scales and codes that stand for NaN or lie out of range."""

    def __init__(self, seqs, H, KH, hd, page, q=R.F32, kind="i8", **kw):
        super().__init__(seqs, H, KH, hd, page, q, R.F32, **kw)
        self.kind = kind
        self.kq, self.vq = self.pool(), self.pool()

    def pool(self, n_pages=None):
        p = torch.empty(n_pages or self.n_pages, self.KH, self.P * (self.hd + 4), dtype=torch.uint8, device=self.dev)
        codes, scales = views(p, self.P, self.hd)
        codes.fill_(0x80 if self.kind == "i8" else 0x7F)
        scales.fill_(R.NAN)
        return p

    def fill(self, *a, **kw):
        self.k = torch.full((self.n_pages, self.KH, self.P, self.hd), R.NAN, device=self.dev)
        self.v = torch.full_like(self.k, R.NAN)
        super().fill(*a, **kw)
        self.kq, self.vq = self.pool(), self.pool()
        for name in ("k", "v"):
            x = getattr(self, name)
            put = ~torch.isnan(x[..., 0])
            c, s, val = quantise(x[put], self.kind)
            codes, scales = views(getattr(self, name + "q"), self.P, self.hd)
            codes[put], scales[put] = c, s
            full = torch.full(x.shape, R.NAN, dtype=torch.float64, device=self.dev)
            full[put] = val
            setattr(self, name, full)

    def pages(self):
        return engine.pages(self.kq.data_ptr(), self.vq.data_ptr(), self.kq.shape[0], self.P, self.KH, self.hd,
                            type=TYPES[self.kind])

    def ragged(self):
        return engine.ragged(self.start.data_ptr(), self.kv_len.data_ptr(), self.table.data_ptr(), self.n, self.rows,
                             self.max_q, self.max_kv, self.ld)


def attn_tolerance(out, mag, dot, hd, longest, bf16):
    """paged_ref's, and what the scales add: a score is rounded once more at its
    key's scale (2^-24 of it, so of its weight, and of the weights' sum: twice),
    a weight once at its value's (2^-24)."""
    more = (2 * 2.0 ** -24 * dot[..., None] + 2.0 ** -24) * mag
    return R.attn_tolerance(out, mag, dot, hd, longest, bf16) + more
