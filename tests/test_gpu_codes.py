"""8-bit pages on the GPU: append, reading back and attention against the float64
values of codes and scales (tests/codes_ref.py)."""
import math

import numpy as np
import pytest
import torch

from autoresearch_amd import engine

from . import codes_ref as Q
from . import paged_ref as R
from .paged_ref import BF16, F32, NAN

pytestmark = pytest.mark.gpu

SHAPES = {"mha128": (3, 3, 128), "gqa5": (10, 2, 128), "gqa4_64": (8, 2, 64), "mqa24": (24, 1, 128)}
KINDS = sorted(Q.TYPES)
ROWS = {"f32": F32, "bf16": BF16}


def run_attn(b, q, window=0, sinks=0, scale=0.0, out=None, stream=0):
    cfg = engine.attn_cfg(b.H, window=window, sinks=sinks, scale=scale, bf16=b.qt == BF16)
    out = torch.full((b.rows, b.H * b.hd), 7.0, dtype=b.qt, device="cuda") if out is None else out
    n = engine.paged_attn_work(b.pages(), b.ragged(), cfg)
    work = torch.full((max(n, 16),), 255, dtype=torch.uint8, device="cuda")  # (NaN)
    engine.paged_attn(b.pages(), b.ragged(), cfg, q.data_ptr(), out.data_ptr(), work.data_ptr(), n, stream)
    torch.cuda.synchronize()
    return out


def check_attn(b, q, got, window=0, sinks=0, scale=None):
    out, mag, dot = b.attention(q, scale, window, sinks)
    got = got.double().reshape(b.rows, b.H, b.hd)
    used = got[:b.used]
    assert torch.isfinite(used).all()
    longest = max(t for t, _ in b.seqs)
    tol = Q.attn_tolerance(out, mag, dot, b.hd, longest, b.qt == BF16)[:b.used]
    over = ((used - out[:b.used]).abs() / tol).max() if b.used else torch.tensor(0.0)
    assert over <= 1.0, float(over)
    assert (got[b.used:] == 7.0).all()  # rows behind the last sequence
    if b.qt == F32 and b.used and out.norm() > 0:
        # roundings of independent sums add in quadrature (as in test_gpu_paged.py)
        rel = float((used - out[:b.used]).norm() / out[:b.used].norm())
        assert rel <= math.sqrt(b.hd + longest + 66) * 2.0 ** -24 * 4, rel


# ------------------------------------------------------------------ reading back

def read(b, pages, bf16, k=True, v=True, ld=0, width=None):
    w = width or b.KH * b.hd
    outs = [torch.full((b.rows, w), 7.0, dtype=BF16 if bf16 else F32, device="cuda") for _ in range(2)]
    engine.pages_read(pages, b.ragged() if isinstance(b, Q.Batch) else engine.ragged(
        b.start.data_ptr(), b.kv_len.data_ptr(), b.table.data_ptr(), b.n, b.rows, b.max_q, b.max_kv, b.ld),
        outs[0].data_ptr() if k else 0, outs[1].data_ptr() if v else 0, bf16=bf16, ld=ld)
    torch.cuda.synchronize()
    return outs


def check_read(b, outs, rt):
    for pool, got in zip((b.k, b.v), outs):
        for s, (T, n) in enumerate(b.seqs):
            a, z, m = int(b.start_np[s]), int(b.start_np[s + 1]), min(n, T)
            want = b.history(pool, s)[:, T - m:].transpose(0, 1).reshape(m, b.KH * b.hd)
            # a product of an 8-bit and a 24-bit significand: fp32 rounds it once, then bf16 does
            assert torch.equal(got[z - m:z], want.float().to(rt)), s
            assert (got[a:z - m] == 7.0).all()  # positions below 0
        assert (got[b.used:] == 7.0).all()


LENGTHS = [(70, 70), (1, 1), (300, 17), (20, 0), (2, 5), (128, 1), (0, 0), (513, 513)]


@pytest.mark.parametrize("rt", sorted(ROWS))
@pytest.mark.parametrize("kind", KINDS + ["f32", "bf16"])
@pytest.mark.parametrize("shape,page", [("mha128", 16), ("gqa4_64", 64), ("gqa5", 256)])
@pytest.mark.parametrize("many", [False, True], ids=["few", "many"])
def test_read(shape, page, kind, rt, many):
    H, KH, hd = SHAPES[shape]
    seqs = LENGTHS + [(1500, 1500)] * many
    if kind in Q.TYPES:
        b = Q.Batch(seqs, H, KH, hd, page, kind=kind, seed=1, pad=3)
        b.fill()
        check_read(b, read(b, b.pages(), rt == "bf16"), ROWS[rt])
    else:
        b = R.Batch(seqs, H, KH, hd, page, F32, ROWS[kind], seed=1, pad=3)
        b.fill()
        pg = engine.pages(b.k.data_ptr(), b.v.data_ptr(), b.n_pages, page, KH, hd, bf16=kind == "bf16")
        check_read(b, read(b, pg, rt == "bf16"), ROWS[rt])


@pytest.mark.parametrize("kind", KINDS)
def test_read_strides_and_bad_pages(kind):
    """A wider row distance, one of the two alone, and NaN where a page is not there."""
    b = Q.Batch([(90, 4), (33, 33), (40, 20)], 4, 2, 128, 16, kind=kind, seed=2)
    b.fill()
    outs = read(b, b.pages(), False, v=False, ld=3 * 128, width=3 * 128)
    assert (outs[0][:, 256:] == 7.0).all() and (outs[1] == 7.0).all()
    whole = read(b, b.pages(), False)
    assert torch.equal(outs[0][:, :256], whole[0])
    b.table_np[1, 1] = -3   # positions 16 .. 31 of the second sequence
    b.table_np[2, 2] = b.n_pages  # 32 .. 39 of the third
    b.table = b.put(b.table_np)
    outs = read(b, b.pages(), False)
    gone = torch.zeros(b.rows, dtype=torch.bool, device="cuda")
    gone[4 + 16:4 + 32] = True
    gone[37 + 12:] = True
    for got, want in zip(outs, whole):
        assert torch.isnan(got[gone]).all() and torch.equal(got[~gone], want[~gone])


def test_read_far_pages():
    """Byte offsets past 2^32."""
    b = Q.Batch([(600, 3), (300, 40)], 2, 1, 128, 256, kind="i8", seed=3)
    b.fill()
    n = (1 << 32) // (256 * 132) + 50
    far = n - b.n_pages
    pools = [torch.empty(n, 1, 256 * 132, dtype=torch.uint8, device="cuda") for _ in range(2)]
    for p, q in zip(pools, (b.kq, b.vq)):
        p[far:] = q
    q = b.normal(b.rows, 256)
    want = run_attn(b, q), read(b, b.pages(), False)
    b.kq, b.vq = pools
    b.table_np = np.where(b.table_np >= 0, b.table_np + far, b.table_np).astype(np.int32)
    b.table = b.put(b.table_np)
    got = run_attn(b, q), read(b, b.pages(), False)
    assert torch.equal(got[0], want[0]) and all(torch.equal(a, w) for a, w in zip(got[1], want[1]))


# ------------------------------------------------------------------ append

def tables(n, hd):
    th = 10000.0 ** (-2.0 * np.arange(hd // 2) / hd)
    a = np.arange(n)[:, None] * th
    return [torch.from_numpy(f(a).astype(np.float32)).cuda() for f in (np.cos, np.sin)]


def append(b, qkv, cos=None, norm=False, w=None, interleaved=False):
    out = torch.full((b.rows, b.H * b.hd), 7.0, dtype=b.qt, device="cuda")
    ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    c, s = cos or (None, None)
    cfg = engine.append_cfg(b.H, ptr(c), ptr(s), b.max_kv if cos else 0, norm=norm, eps=1e-5,
                            wq=ptr(w[0]) if w else 0, wk=ptr(w[1]) if w else 0, bf16=b.qt == BF16,
                            interleaved=interleaved)
    engine.qk_append(b.pages(), b.ragged(), cfg, qkv.data_ptr(), out.data_ptr())
    torch.cuda.synchronize()
    return out


def places(b):
    """Rows with a position, their pages and slots."""
    rows, pages, slots = [], [], []
    for s, (T, n) in enumerate(b.seqs):
        for i in range(n):
            p = T - n + i
            if p >= 0:
                rows.append(int(b.start_np[s]) + i)
                pages.append(int(b.table_np[s, p // b.P]))
                slots.append(p % b.P)
    return [torch.tensor(a, device="cuda") for a in (rows, pages, slots)]


@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("norm", [None, "plain", "weights"])
@pytest.mark.parametrize("rows", sorted(ROWS))
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape,page", [("mha128", 16), ("gqa4_64", 64), ("gqa5", 256)])
def test_append(shape, page, kind, rows, norm, interleaved):
    check_append([(70, 70), (1, 1), (300, 17), (20, 0), (2, 3), (128, 1), (0, 0)] + [(9, 1)] * 70, shape,
                 page, kind, rows, norm, interleaved)


@pytest.mark.parametrize("rows", sorted(ROWS))
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", ["mha128", "gqa4_64"])
def test_append_many_rows(shape, kind, rows):
    check_append([(901, 901), (2, 3), (1200, 1147), (30, 1), (31, 1), (1, 1)], shape, 32, kind, rows, "weights", False)


def check_append(seqs, shape, page, kind, rows, norm, interleaved):
    H, KH, hd = SHAPES[shape]
    qt = ROWS[rows]
    b = Q.Batch(seqs, H, KH, hd, page, qt, kind=kind, seed=11, pad=5)
    cos = tables(b.max_kv, hd)
    w = [1 + 0.3 * b.normal(hd) for _ in range(2)] if norm == "weights" else None
    qkv = b.normal(b.rows, (H + 2 * KH) * hd, dtype=qt, std=2.0)
    before = b.kq.clone()
    out = append(b, qkv, cos, norm is not None, w, interleaved)
    q, k, v, _ = R.append_rows(b, qkv, *cos, norm is not None, 1e-5, *(w or (None, None)), interleaved=interleaved)
    at, pg, slot = places(b)
    # fp32 error of a normed and rotated value, as test_gpu_paged.py derives it
    noise = lambda x: (hd / 2 + 8) * 2.0 ** -24 * x.abs().amax(-1, keepdim=True) * 2  # noqa: E731
    err = (out.reshape(b.rows, H, hd).double() - q).abs()
    assert (err <= noise(q) + (2.0 ** -8 * q.abs() if qt == BF16 else 0))[at].all()
    for pool, want in ((b.kq, k[at]), (b.vq, v[at])):
        codes, scales = Q.views(pool, page, hd)
        c, s = Q.values(codes[pg, :, slot].contiguous(), kind), scales[pg, :, slot].double()[..., None]
        top = want.abs().amax(-1, keepdim=True)
        assert ((s - top / Q.TOP[kind]).abs() <= noise(want) / Q.TOP[kind] + 2.0 ** -23 * s).all()
        # a value is at most half a step of its code off the value it was made of: of
        # integers 1/2, of three bits behind the leading one 2^-4 of it or, below 2^-6, 2^-10
        step = 0.5 if kind == "i8" else torch.maximum(c.abs() * 2.0 ** -4, torch.full_like(c, 2.0 ** -10))
        # (x * (1 / s): two roundings before the code's)
        assert ((c * s - want).abs() <= (step + Q.TOP[kind] * 2.0 ** -22) * s + noise(want)).all()
    # v goes through no arithmetic: its codes and scales are the definition's, bit for bit
    codes, scales = Q.views(b.vq, page, hd)
    c, s, _ = Q.quantise(v[at].float(), kind)
    assert torch.equal(codes[pg, :, slot], c) and torch.equal(scales[pg, :, slot], s)
    # nothing else was written
    unseen = torch.ones(b.n_pages, page, dtype=torch.bool, device="cuda")
    unseen[pg, slot] = False
    for x, y in zip(Q.views(b.kq, page, hd), Q.views(before, page, hd)):
        x, y = x.transpose(1, 2)[unseen], y.transpose(1, 2)[unseen]
        assert torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))


@pytest.mark.parametrize("rows", sorted(ROWS))
@pytest.mark.parametrize("kind", KINDS)
def test_append_extreme_rows(kind, rows):
    """Zeros, the smallest and largest values, infinities and NaN, a row each."""
    qt = ROWS[rows]
    b = Q.Batch([(9, 9)], 2, 1, 64, 16, qt, kind=kind, seed=12)
    qkv = b.normal(9, 4 * 64, dtype=qt)
    v = qkv[:, 192:]
    v[0] = 0.0
    v[1] = -0.0
    v[2] = 1e-42 if qt == F32 else 1e-39   # below the smallest scale
    v[3, 5] = float("inf")
    v[4, 63] = NAN
    v[5] *= 1e36
    v[6, 0] = 3.3e38
    v[7] *= 1e-35
    v[8, 1:] = 0.0
    append(b, qkv)
    codes, scales = Q.views(b.vq, 16, 64)
    pg = int(b.table_np[0, 0])
    c, s, val = Q.quantise(v.float(), kind)
    assert torch.equal(scales[pg, 0, :9].isnan(), s.isnan()) and s.isnan().sum() == 2
    ok = ~s.isnan()
    same = lambda x: x[ok].view(torch.int8)  # noqa: E731
    assert torch.equal(scales[pg, 0, :9][ok], s[ok])
    got = Q.values(codes[pg, 0, :9].contiguous(), kind)
    assert torch.equal(got[ok], Q.values(c, kind)[ok])
    assert (got[~ok] == 0).all() and (scales[pg, 0, :3] == 0).all() and same(codes[pg, 0, :9])[:3].eq(0).all()
    out = read(b, b.pages(), False)[1]
    assert torch.equal(out.isnan().all(-1), s.isnan()) and torch.equal(out[ok], val[ok].float())


# ------------------------------------------------------------------ attention

ATTN = {
    "one": [(1, 1)],
    "short": [(5, 5), (16, 1), (17, 3)],
    "empty": [(0, 0), (33, 0), (31, 2), (4, 0)],
    "tile_ends": [(32, 32), (33, 33), (64, 1), (65, 2), (127, 16), (128, 17), (129, 129)],
    "decode": [(700, 1), (1, 1), (300, 1), (1025, 1), (40, 0), (512, 1)],
    "long": [(5003, 1), (4096, 7)],
    "mixed": [(900, 200), (901, 1), (257, 257), (64, 3)],
    "below_zero": [(3, 5), (40, 40), (0, 4)],
}


@pytest.mark.parametrize("lengths", sorted(ATTN))
@pytest.mark.parametrize("rows", sorted(ROWS))
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape,page", [("mha128", 16), ("gqa5", 64), ("gqa4_64", 32), ("mqa24", 256)])
def test_attention(shape, page, kind, rows, lengths):
    H, KH, hd = SHAPES[shape]
    b = Q.Batch(ATTN[lengths], H, KH, hd, page, ROWS[rows], kind=kind, seed=len(lengths) + page, pad=3)
    b.fill()
    q = b.normal(b.rows, H * hd, dtype=b.qt, std=1.5)
    check_attn(b, q, run_attn(b, q))


@pytest.mark.parametrize("rows", sorted(ROWS))
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", ["mha128", "gqa4_64"])
@pytest.mark.parametrize("T", [127, 128, 129, 255, 257, 385, 511, 512, 513, 545])
def test_where_parts_begin(T, shape, kind, rows):
    """Up to 512 positions at most, two key tiles for each of eight wavefronts, one part takes them."""
    H, KH, hd = SHAPES[shape]
    b = Q.Batch([(T, 1), (1, 1), (T // 2, 2), (0, 0)], H, KH, hd, 16, ROWS[rows], kind=kind, seed=24)
    b.fill()
    q = b.normal(b.rows, H * hd, dtype=ROWS[rows])
    at = engine.attn_cfg(H, bf16=rows == "bf16")
    assert (engine.paged_attn_work(b.pages(), b.ragged(), at) == 0) == (T <= 512)
    check_attn(b, q, run_attn(b, q))


@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 3), (33, 70), (100, 32), (640, 5), (5000, 4)])
@pytest.mark.parametrize("rows", sorted(ROWS))
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape,page", [("gqa5", 16), ("gqa4_64", 64), ("mha128", 32)])
def test_window(shape, page, kind, rows, window, sinks):
    """Keys that no row sees have NaN scales, their pages gone from the table."""
    H, KH, hd = SHAPES[shape]
    b = Q.Batch([(1500, 1), (2000, 9), (90, 90), (400, 130), (3, 1), (50, 0)], H, KH, hd, page, ROWS[rows],
                kind=kind, seed=window + sinks, pad=1)
    b.fill(window, sinks)
    q = b.normal(b.rows, H * hd, dtype=b.qt)
    check_attn(b, q, run_attn(b, q, window, sinks), window, sinks)


@pytest.mark.parametrize("rows", sorted(ROWS))
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", sorted(SHAPES))
def test_large_batches(shape, kind, rows):
    """Rows and keys enough for the 128-row tiles whole, part tiles among them."""
    H, KH, hd = SHAPES[shape]
    b = Q.Batch([(700, 700), (650, 1), (900, 300), (33, 33), (500, max(1, 100 // (H // KH))), (1, 1)], H, KH, hd,
                64, ROWS[rows], kind=kind, seed=24, pad=7)
    for w, s in ((0, 0), (150, 5)):
        b.fill(w, s, drop_pages=False)
        q = b.normal(b.rows, H * hd, dtype=b.qt)
        check_attn(b, q, run_attn(b, q, w, s), w, s)


@pytest.mark.parametrize("rows", sorted(ROWS))
@pytest.mark.parametrize("kind", KINDS)
def test_large_scores_and_scale(kind, rows):
    b = Q.Batch([(700, 3), (200, 60)], 4, 4, 64, 32, ROWS[rows], kind=kind, seed=4)
    b.fill()
    q = b.normal(b.rows, 4 * 64, dtype=b.qt, std=30.0)
    check_attn(b, q, run_attn(b, q))
    check_attn(b, q, run_attn(b, q, scale=0.01), scale=float(np.float32(0.01)))


@pytest.mark.parametrize("kind", KINDS)
def test_scales_of_many_sizes(kind):
    """Keys of very different lengths, values too: each has its own scale."""
    b = Q.Batch([(300, 40), (900, 1)], 6, 2, 128, 16, kind=kind, seed=5)
    b.fill()
    for name in ("k", "v"):
        f = torch.exp2(torch.randint(-8, 3, b.k.shape[:3], generator=b.g).double()).cuda()
        _, scales = Q.views(getattr(b, name + "q"), b.P, b.hd)
        scales.mul_(f.float())
        setattr(b, name, getattr(b, name) * f[..., None])
    q = b.normal(b.rows, 6 * 128)
    check_attn(b, q, run_attn(b, q))


@pytest.mark.parametrize("rows", sorted(ROWS))
@pytest.mark.parametrize("kind", KINDS)
def test_nan_rows(kind, rows):
    """A key or value of NaN (its scale) that a row sees makes it NaN; a bad page too."""
    b = Q.Batch([(300, 2), (100, 20), (40, 1), (64, 1)], 4, 2, 128, 16, ROWS[rows], kind=kind, seed=6)
    b.fill()
    Q.views(b.kq, 16, 128)[1][int(b.table_np[0, 9]), :, 3] = NAN
    Q.views(b.vq, 16, 128)[1][int(b.table_np[1, 0]), :, 0] = NAN
    b.table_np[2, 0] = -5
    b.table = b.put(b.table_np)
    got = run_attn(b, b.normal(b.rows, 4 * 128, dtype=b.qt))
    assert torch.isnan(got[:23]).all() and torch.isfinite(got[23:]).all()


@pytest.mark.parametrize("kind", KINDS)
def test_repeats_streams_and_place(kind):
    """The same bits twice, on another stream, in the place of q; pages that moved by a copy."""
    b = Q.Batch([(3000, 1), (200, 70)], 10, 2, 128, 64, F32, kind=kind, seed=9)
    b.fill()
    q = b.normal(b.rows, 1280)
    one = run_attn(b, q)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    assert torch.equal(one, run_attn(b, q)) and torch.equal(one, run_attn(b, q, stream=s.cuda_stream))
    page = engine.page_bytes(64, 2, 128, Q.TYPES[kind])
    assert page == b.kq.stride(0)
    free = np.setdiff1d(np.arange(b.n_pages), b.table_np)[:3].astype(np.int32)
    src = b.table_np[0, [0, 7, 46]].copy()
    for pool in (b.kq, b.vq):
        engine.pages_copy(pool.data_ptr(), 1, page * b.n_pages, b.n_pages, page, src, free)
    torch.cuda.synchronize()
    b.table_np[0, [0, 7, 46]] = free
    b.table = b.put(b.table_np)
    assert torch.equal(one, run_attn(b, q))
    assert torch.equal(one, run_attn(b, q, out=q))


@pytest.mark.parametrize("rows", sorted(ROWS))
@pytest.mark.parametrize("kind", KINDS)
def test_append_read_attend_captured(kind, rows):
    """Append, reading back and attention in one graph: every replay is the eager calls'."""
    H, KH, hd, P = 10, 2, 128, 32
    b = Q.Batch([(700, 1), (90, 40), (33, 2)], H, KH, hd, P, ROWS[rows], kind=kind, seed=10)
    b.fill()
    cos = tables(b.max_kv, hd)
    qkv = b.normal(b.rows, (H + 2 * KH) * hd, dtype=b.qt)
    q = torch.zeros(b.rows, H * hd, dtype=b.qt, device="cuda")
    k, v = (torch.zeros(b.rows, KH * hd, device="cuda") for _ in range(2))
    out = torch.zeros_like(q)
    ap = engine.append_cfg(H, cos[0].data_ptr(), cos[1].data_ptr(), b.max_kv, norm=True, bf16=b.qt == BF16)
    at = engine.attn_cfg(H, bf16=b.qt == BF16)
    n = engine.paged_attn_work(b.pages(), b.ragged(), at)
    work = torch.empty(max(16, n), dtype=torch.uint8, device="cuda")

    def calls(stream):
        engine.qk_append(b.pages(), b.ragged(), ap, qkv.data_ptr(), q.data_ptr(), stream)
        engine.pages_read(b.pages(), b.ragged(), k.data_ptr(), v.data_ptr(), stream=stream)
        engine.paged_attn(b.pages(), b.ragged(), at, q.data_ptr(), out.data_ptr(), work.data_ptr(), n, stream)

    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
        calls(torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        qkv.copy_(b.normal(b.rows, (H + 2 * KH) * hd, dtype=b.qt))
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (q, k, v, out)]
        for t in (q, k, v, out):
            t.zero_()
        calls(0)
        torch.cuda.synchronize()
        assert all(torch.equal(a, w) for a, w in zip(got, (q, k, v, out))) and torch.isfinite(out).all()
