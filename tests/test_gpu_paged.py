"""The paged cache's operators on the GPU against plain float64 forms
(tests/paged_ref.py), on pools that hold NaN wherever no row may look."""
import math

import numpy as np
import pytest
import torch

from autoresearch_amd import engine

from . import paged_ref as R
from .paged_ref import BF16, F32, NAN

pytestmark = pytest.mark.gpu

SHAPES = {"mha128": (3, 3, 128), "gqa5": (10, 2, 128), "gqa4_64": (8, 2, 64), "mqa24": (24, 1, 128)}
TYPES = {"f32": (F32, F32), "f32_kv16": (F32, BF16), "bf16": (BF16, BF16)}


def pages_of(b):
    return engine.pages(b.k.data_ptr(), b.v.data_ptr(), b.n_pages, b.P, b.KH, b.hd, bf16=b.kt == BF16)


def ragged_of(b):
    return engine.ragged(b.start.data_ptr(), b.kv_len.data_ptr(), b.table.data_ptr(), b.n, b.rows,
                         b.max_q, b.max_kv, b.ld)


def run_attn(b, q, window=0, sinks=0, scale=0.0, out=None, q_ld=0, out_ld=0, stream=0):
    cfg = engine.attn_cfg(b.H, window=window, sinks=sinks, scale=scale, bf16=b.qt == BF16, q_ld=q_ld,
                          out_ld=out_ld)
    out = torch.full((b.rows, b.H * b.hd), 7.0, dtype=b.qt, device="cuda") if out is None else out
    n = engine.paged_attn_work(pages_of(b), ragged_of(b), cfg)
    work = torch.full((max(n, 16),), 255, dtype=torch.uint8, device="cuda")  # (NaN)
    engine.paged_attn(pages_of(b), ragged_of(b), cfg, q.data_ptr(), out.data_ptr(), work.data_ptr(), n,
                      stream)
    torch.cuda.synchronize()
    return out


def check_attn(b, q, got, window=0, sinks=0, scale=None):
    out, mag, dot = b.attention(q, scale, window, sinks)
    got = got.double().reshape(b.rows, b.H, b.hd)
    used = got[:b.used]
    assert torch.isfinite(used).all()
    longest = max(t for t, _ in b.seqs)
    tol = R.attn_tolerance(out, mag, dot, b.hd, longest, b.qt == BF16)[:b.used]
    over = ((used - out[:b.used]).abs() / tol).max() if b.used else torch.tensor(0.0)
    assert over <= 1.0, float(over)
    assert (got[b.used:] == 7.0).all()  # rows behind the last sequence
    if b.qt == F32 and b.used and out.norm() > 0:
        # roundings of independent sums add in quadrature: (hd + longest + 64)
        # of them of 2^-24 at most (operands in two terms would leave 2^-17)
        rel = float((used - out[:b.used]).norm() / out[:b.used].norm())
        assert rel <= math.sqrt(b.hd + longest + 64) * 2.0 ** -24 * 4, rel


LENGTHS = {
    "one": [(1, 1)],
    "short": [(5, 5), (16, 1), (17, 3)],
    "empty": [(0, 0), (33, 0), (31, 2), (4, 0)],
    "tile_ends": [(32, 32), (33, 33), (64, 1), (65, 2), (127, 16), (128, 17), (129, 129)],
    "decode": [(700, 1), (1, 1), (300, 1), (1025, 1), (40, 0), (512, 1)],
    "long": [(5003, 1), (4096, 7)],
    "mixed": [(900, 200), (901, 1), (257, 257), (64, 3)],
}


@pytest.mark.parametrize("lengths", sorted(LENGTHS))
@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("shape,page", [("mha128", 16), ("gqa5", 64), ("gqa4_64", 32), ("mqa24", 256)])
def test_attention(shape, page, types, lengths):
    H, KH, hd = SHAPES[shape]
    qt, kt = TYPES[types]
    b = R.Batch(LENGTHS[lengths], H, KH, hd, page, qt, kt, seed=len(lengths) + page, pad=3)
    b.fill()
    q = b.normal(b.rows, H * hd, dtype=qt, std=1.5)
    check_attn(b, q, run_attn(b, q))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (16, 4), (33, 70), (100, 0), (100, 32),
                                          (640, 5), (5000, 4)])
@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("shape,page", [("gqa5", 16), ("gqa4_64", 64), ("mha128", 32)])
def test_window(shape, page, types, window, sinks):
    """Keys that no row sees are NaN, their pages gone from the table."""
    H, KH, hd = SHAPES[shape]
    qt, kt = TYPES[types]
    b = R.Batch([(1500, 1), (2000, 9), (90, 90), (400, 130), (3, 1), (50, 0)], H, KH, hd, page, qt, kt,
                seed=window + sinks, pad=1)
    b.fill(window, sinks)
    q = b.normal(b.rows, H * hd, dtype=qt)
    check_attn(b, q, run_attn(b, q, window, sinks), window, sinks)


@pytest.mark.parametrize("types", sorted(TYPES))
def test_rows_without_a_key(types):
    """More new tokens than positions: the first ones sit below 0 and see nothing."""
    qt, kt = TYPES[types]
    b = R.Batch([(3, 5), (40, 40), (0, 4)], 4, 2, 128, 16, qt, kt, seed=3)
    b.fill()
    q = b.normal(b.rows, 4 * 128, dtype=qt)
    got = run_attn(b, q)
    check_attn(b, q, got)
    assert (got[:2] == 0).all() and (got[45:] == 0).all()


@pytest.mark.parametrize("types", sorted(TYPES))
def test_large_scores_and_scale(types):
    """Scores in the hundreds (one key takes all) and a scale of the caller's."""
    qt, kt = TYPES[types]
    b = R.Batch([(700, 3), (200, 60)], 4, 4, 64, 32, qt, kt, seed=4)
    b.fill()
    q = b.normal(b.rows, 4 * 64, dtype=qt, std=30.0)
    check_attn(b, q, run_attn(b, q))
    check_attn(b, q, run_attn(b, q, scale=0.01), scale=float(np.float32(0.01)))


def test_strided_rows():
    """q as a slice of QKV rows, out with a wider row distance."""
    b = R.Batch([(90, 4), (33, 33)], 6, 2, 128, 16, seed=5)
    b.fill()
    wide = b.normal(b.rows, 10 * 128)
    out = torch.full((b.rows, 8 * 128), 7.0, device="cuda")
    run_attn(b, wide, out=out, q_ld=10 * 128, out_ld=8 * 128)
    q = wide[:, :6 * 128].contiguous()
    check_attn(b, q, out[:, :6 * 128].contiguous())
    assert (out[:, 6 * 128:] == 7.0).all()


@pytest.mark.parametrize("types", sorted(TYPES))
def test_bad_page_gives_nan_rows(types):
    qt, kt = TYPES[types]
    b = R.Batch([(300, 2), (100, 20), (40, 1)], 4, 2, 128, 16, qt, kt, seed=6)
    b.fill()
    b.table_np[0, 9] = b.n_pages
    b.table_np[1, 0] = -5
    b.table = b.put(b.table_np)
    got = run_attn(b, b.normal(b.rows, 4 * 128, dtype=qt))
    assert torch.isnan(got[:22]).all() and torch.isfinite(got[22:]).all()


def test_far_pages():
    """Page offsets past 2^31 elements (a pool of 4.4 GB)."""
    H, KH, hd, P = 2, 1, 128, 256
    b = R.Batch([(600, 3), (300, 40)], H, KH, hd, P, BF16, BF16, seed=7)
    n_pages = (1 << 31) // (P * hd) + 50
    k = torch.empty(n_pages, KH, P, hd, dtype=BF16, device="cuda")
    v = torch.empty_like(k)
    b.fill()
    want = b.attention(q := b.normal(b.rows, H * hd, dtype=BF16))[0]
    shift = n_pages - b.n_pages
    k[shift:], v[shift:] = b.k, b.v
    b.k, b.v, b.n_pages = k, v, n_pages
    b.table_np = np.where(b.table_np >= 0, b.table_np + shift, b.table_np).astype(np.int32)
    b.table = b.put(b.table_np)
    got = run_attn(b, q).double().reshape(want.shape)
    assert torch.allclose(got, want, rtol=2.0 ** -6, atol=2.0 ** -6)


def test_capture_replays_other_lengths():
    """One captured call serves any batch within its bounds; two graphs with a
    workspace each, on a stream of the caller's, with eager work between."""
    H, KH, hd, P = 10, 2, 128, 32
    batches = [R.Batch(s, H, KH, hd, P, F32, BF16, seed=i, pad=p, slack=0)
               for i, (s, p) in enumerate([([(2000, 1), (100, 40), (5, 5)], 4),
                                           ([(1999, 30), (40, 1), (0, 0)], 19),
                                           ([(7, 7), (1500, 3), (900, 40)], 0)])]
    rows, ld = 50, 63
    n_pages = max(b.n_pages for b in batches)
    st = dict(start=torch.zeros(4, dtype=torch.int32, device="cuda"),
              kv=torch.zeros(3, dtype=torch.int32, device="cuda"),
              table=torch.full((3, ld), -1, dtype=torch.int32, device="cuda"),
              q=torch.zeros(rows, H * hd, device="cuda"))
    k = torch.zeros(n_pages, KH, P, hd, dtype=BF16, device="cuda")
    v = torch.zeros_like(k)
    pg = engine.pages(k.data_ptr(), v.data_ptr(), n_pages, P, KH, hd, bf16=True)
    bt = engine.ragged(st["start"].data_ptr(), st["kv"].data_ptr(), st["table"].data_ptr(), 3, rows, 40,
                       2016, ld)
    cfg = engine.attn_cfg(H)
    n = engine.paged_attn_work(pg, bt, cfg)
    assert n > 0
    outs, graphs, works = [], [], []
    for _ in range(2):
        out = torch.full((rows, H * hd), 7.0, device="cuda")
        work = torch.empty(n, dtype=torch.uint8, device="cuda")
        g = torch.cuda.CUDAGraph()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
            engine.paged_attn(pg, bt, cfg, st["q"].data_ptr(), out.data_ptr(), work.data_ptr(), n,
                              torch.cuda.current_stream().cuda_stream)
        outs.append(out)
        graphs.append(g)
        works.append(work)
    for b in batches + batches[:1]:
        b.fill()
        k[:b.n_pages], v[:b.n_pages] = b.k, b.v
        st["start"].copy_(b.start)
        st["kv"].copy_(b.kv_len)
        st["table"].fill_(-1)
        st["table"][:, :b.ld].copy_(b.table)
        q = b.normal(b.rows, H * hd)
        st["q"][:b.rows].copy_(q)
        for o in outs:
            o.fill_(7.0)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1])
        check_attn(b, q, outs[0][:b.rows])


def test_repeats_are_equal():
    """The same call twice, and on another stream: the same bits."""
    b = R.Batch([(3000, 1), (200, 70)], 10, 2, 128, 64, F32, F32, seed=9)
    b.fill()
    q = b.normal(b.rows, 1280)
    one = run_attn(b, q)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    assert torch.equal(one, run_attn(b, q)) and torch.equal(one, run_attn(b, q, stream=s.cuda_stream))


def test_two_streams_at_once():
    """Calls on two streams with a workspace each, queued behind each other's work."""
    bs = [R.Batch([(4000, 1), (900, 30)], 10, 2, 128, 32, F32, BF16, seed=21),
          R.Batch([(64 + 50 * i, 1) for i in range(40)], 6, 6, 128, 16, F32, F32, seed=22)]
    qs = []
    for b in bs:
        b.fill()
        qs.append(b.normal(b.rows, b.H * b.hd))
    alone = [run_attn(b, q) for b, q in zip(bs, qs)]
    outs, keep = [], []
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for b, q in zip(bs, qs):
        cfg = engine.attn_cfg(b.H)
        n = engine.paged_attn_work(pages_of(b), ragged_of(b), cfg)
        keep.append((cfg, n, torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")))
        outs.append([torch.zeros(b.rows, b.H * b.hd, device="cuda") for _ in range(6)])
    torch.cuda.synchronize()
    for i in range(6):
        for k, b in enumerate(bs):
            cfg, n, work = keep[k]
            engine.paged_attn(pages_of(b), ragged_of(b), cfg, qs[k].data_ptr(), outs[k][i].data_ptr(),
                              work.data_ptr(), n, streams[k].cuda_stream)
    torch.cuda.synchronize()
    for a, o in zip(alone, outs):
        assert all(torch.equal(a, x) for x in o)


@pytest.mark.parametrize("types", sorted(TYPES))
def test_out_in_place(types):
    qt, kt = TYPES[types]
    b = R.Batch([(3000, 2), (200, 90)], 10, 2, 128, 32, qt, kt, seed=23)
    b.fill()
    q = b.normal(b.rows, 1280, dtype=qt)
    want = run_attn(b, q)
    assert torch.equal(run_attn(b, q, out=q), want)


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("shape", sorted(SHAPES))
def test_large_batches(shape, types):
    """Rows and keys enough for the 128-row tiles whole (no parts), part tiles
    and wavefronts without rows among them."""
    H, KH, hd = SHAPES[shape]
    qt, kt = TYPES[types]
    G = H // KH
    b = R.Batch([(700, 700), (650, 1), (900, 300), (33, 33), (500, max(1, 100 // G)), (1, 1)], H, KH, hd, 64,
                qt, kt, seed=24, pad=7)
    for w, s in ((0, 0), (150, 5)):
        b.k.fill_(NAN)
        b.v.fill_(NAN)
        b.fill(w, s, drop_pages=False)
        q = b.normal(b.rows, H * hd, dtype=qt)
        check_attn(b, q, run_attn(b, q, w, s), w, s)


# ------------------------------------------------------------------ append

def tables(n, hd):
    th = 10000.0 ** (-2.0 * np.arange(hd // 2) / hd)
    a = np.arange(n)[:, None] * th
    return [torch.from_numpy(f(a).astype(np.float32)).cuda() for f in (np.cos, np.sin)]


@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("norm", [None, "plain", "weights"])
@pytest.mark.parametrize("types", ["f32", "f32_kv16", "bf16", "bf16_kv32"])
@pytest.mark.parametrize("shape,page", [("mha128", 16), ("gqa4_64", 64), ("gqa5", 256)])
def test_append(shape, page, types, norm, interleaved):
    check_append([(70, 70), (1, 1), (300, 17), (20, 0), (2, 3), (128, 1), (0, 0)] + [(9, 1)] * 70, shape,
                 page, types, norm, interleaved)


@pytest.mark.parametrize("norm", [None, "weights"])
@pytest.mark.parametrize("types", ["f32", "bf16"])
@pytest.mark.parametrize("shape", ["mha128", "gqa4_64"])
def test_append_many_rows(shape, types, norm):
    """From 2048 rows on, four a workgroup (some of them of different sequences)."""
    check_append([(901, 901), (2, 3), (1200, 1147), (30, 1), (31, 1), (1, 1)], shape, 32, types, norm, False)


def check_append(seqs, shape, page, types, norm, interleaved):
    H, KH, hd = SHAPES[shape]
    qt, kt = {**TYPES, "bf16_kv32": (BF16, F32)}[types]
    b = R.Batch(seqs, H, KH, hd, page, qt, kt, seed=11, pad=5)
    cos, sin = tables(b.max_kv, hd)
    w = [1 + 0.3 * b.normal(hd) for _ in range(2)] if norm == "weights" else [None, None]
    qkv = b.normal(b.rows, (H + 2 * KH) * hd, dtype=qt, std=2.0)
    out = torch.full((b.rows, H * hd), 7.0, dtype=qt, device="cuda")
    cfg = engine.append_cfg(H, cos.data_ptr(), sin.data_ptr(), b.max_kv, norm=norm is not None, eps=1e-5,
                            wq=w[0].data_ptr() if norm == "weights" else 0,
                            wk=w[1].data_ptr() if norm == "weights" else 0, bf16=qt == BF16,
                            interleaved=interleaved)
    engine.qk_append(pages_of(b), ragged_of(b), cfg, qkv.data_ptr(), out.data_ptr())
    torch.cuda.synchronize()
    q, k, v, where = R.append_rows(b, qkv, cos, sin, norm is not None, 1e-5, *w, interleaved=interleaved)
    real = torch.tensor([p >= 0 for _, p in where], device="cuda")
    pg = torch.tensor([int(b.table_np[s, p // page]) for s, p in where if p >= 0], device="cuda")
    slot = torch.tensor([p % page for _, p in where if p >= 0], device="cuda")
    # fp32: a rotation adds two products of rounded factors (the norm's sum of hd
    # squares, root and quotient: hd / 2 + 4 halves of 2^-23 of x in all); bf16 adds one rounding
    for got, want, h0, dt in ((out.reshape(b.rows, H, hd), q, 0, qt), (b.k, k, H, kt), (b.v, v, H + KH, kt)):
        size = want.abs().amax(-1, keepdim=True) * 2
        tol = (hd / 2 + 8) * 2.0 ** -24 * size + (2.0 ** -8 * want.abs() if dt == BF16 else 0)
        if h0 == 0:
            assert ((got.double() - want).abs() <= tol)[real].all() and (got[~real] == 7.0).all()
            continue
        assert ((got[pg, :, slot].double() - want[real]).abs() <= tol[real]).all()
        unseen = torch.ones(b.n_pages, page, dtype=torch.bool, device="cuda")
        unseen[pg, slot] = False
        assert torch.isnan(got.transpose(1, 2)[unseen]).all()  # nothing else was written


def test_append_without_rotation_and_bad_pages():
    b = R.Batch([(40, 4), (20, 2)], 2, 2, 64, 16, F32, F32, seed=12)
    b.table_np[0, 2] = b.n_pages  # positions 32.. of the first sequence
    b.table_np[1, 1] = -1
    b.table = b.put(b.table_np)
    wide = b.normal(b.rows, 8 * 64)
    out = torch.full((b.rows, 4 * 64), 7.0, device="cuda")
    cfg = engine.append_cfg(2, qkv_ld=8 * 64, q_ld=4 * 64)
    engine.qk_append(pages_of(b), ragged_of(b), cfg, wide.data_ptr(), out.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(out[:, :128], wide[:, :128]) and (out[:, 128:] == 7.0).all()
    assert torch.isnan(b.k).all() and torch.isnan(b.v).all()


# ------------------------------------------------------------------ page copies

@pytest.mark.parametrize("planes,page_bytes,pages,n", [(1, 16, 4, 1), (3, 48, 9, 4), (24, 49152, 40, 19),
                                                       (2, 16400, 1000, 499), (5, 4096, 1200, 600)])
def test_pages_copy(planes, page_bytes, pages, n):
    g = torch.Generator(device="cuda").manual_seed(n)
    gap = 64
    pool = torch.randint(0, 255, (planes, pages * page_bytes + gap), generator=g, device="cuda",
                         dtype=torch.uint8)
    pick = np.random.default_rng(n).permutation(pages)[:2 * n].astype(np.int32)
    src, dst = pick[:n].copy(), pick[n:].copy()
    src[-1] = src[0]  # one page to two places
    want = pool.clone()
    w = want[:, :pages * page_bytes].unflatten(1, (pages, page_bytes))
    w[:, torch.from_numpy(dst).long().cuda()] = w[:, torch.from_numpy(src).long().cuda()]
    engine.pages_copy(pool.data_ptr(), planes, pages * page_bytes + gap, pages, page_bytes, src, dst)
    src[:] = 0  # (the list is the caller's again)
    dst[:] = 0
    torch.cuda.synchronize()
    assert torch.equal(pool, want)


# ------------------------------------------------------------------ draws

def run_draw(x, temp=None, top_k=None, top_p=None, min_p=None, u=None):
    rows, V = x.shape
    dev = lambda a, t: None if a is None else torch.from_numpy(np.asarray(a, t)).cuda()  # noqa: E731
    ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    lg = torch.full((rows, V + 5), 99.0, device="cuda")
    lg[:, :V] = torch.from_numpy(x).cuda()
    temp, top_p, min_p, u = (dev(a, np.float32) for a in (temp, top_p, min_p, u))
    top_k = dev(top_k, np.int32)
    ids = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    probs = torch.full((rows,), -7.0, device="cuda")
    n = engine.draw_rows_work(rows, V)
    work = torch.full((max(n, 16),), 255, dtype=torch.uint8, device="cuda")
    engine.draw_rows(lg.data_ptr(), rows, V, V + 5, ptr(u), ids.data_ptr(), probs.data_ptr(), temp=ptr(temp),
                     top_k=ptr(top_k), top_p=ptr(top_p), min_p=ptr(min_p), work=work.data_ptr(), work_bytes=n)
    torch.cuda.synchronize()
    return ids.cpu().numpy(), probs.cpu().numpy()


def check_draw(x, got, temp, top_k, top_p, min_p, u):
    ids, probs = got
    # (the settings as the kernel has them: 0.7 of 150 equal ids is id 105, fp32(0.7) of them 104)
    temp, top_p, min_p, u = (np.asarray(a, np.float32) for a in (temp, top_p, min_p, u))
    for r in range(len(x)):
        want = R.draw_row(x[r], float(temp[r]), int(top_k[r]), float(top_p[r]), float(min_p[r]), float(u[r]))
        assert ids[r] == want[0], (r, ids[r], want)
        # (a mass is off by 2^-45 of the largest; the quotient is rounded once)
        assert abs(probs[r] - want[1]) <= 2.0 ** -23 * want[1] + len(x[r]) * 2.0 ** -44, (r, probs[r], want)


def settings(rng, rows, V):
    off = lambda a, o, p: np.where(rng.random(rows) < p, o, a)  # noqa: E731
    temp = off(rng.uniform(0.2, 2.0, rows), rng.choice([0.0, -1.0, 1.0]), 0.15).astype(np.float32)
    top_k = off(rng.integers(1, max(2, min(V, 300)), rows), rng.choice([0, -3, V, V + 9]), 0.4)
    top_p = off(rng.uniform(0.05, 0.999, rows), rng.choice([1.0, 2.0, np.nan]), 0.4).astype(np.float32)
    min_p = off(rng.uniform(1e-4, 0.5, rows), rng.choice([0.0, -1.0, np.nan]), 0.5).astype(np.float32)
    return temp, top_k.astype(np.int32), top_p, min_p, (rng.integers(0, 1 << 24, rows) / 2.0 ** 24).astype(np.float32)


@pytest.mark.parametrize("kind", ["normal", "ties", "levels", "flat", "peaked"])
@pytest.mark.parametrize("V,rows", [(1, 3), (2, 9), (63, 9), (64, 9), (65, 9), (1000, 40), (8192, 64),
                                    (50257, 7), (131073, 3), (262144, 2)])
def test_draw(V, rows, kind):
    rng = np.random.default_rng(V + len(kind))
    x = rng.normal(0, 3, (rows, V)).astype(np.float32)
    if kind == "ties":  # 8 significant bits
        x = (x.view(np.uint32) & 0xFFFF0000).view(np.float32)
    elif kind == "levels":
        x = rng.integers(-2, 2, (rows, V)).astype(np.float32) * np.float32(0.7)
    elif kind == "flat":
        x[:] = np.float32(-1.25)
    elif kind == "peaked":
        x -= 30
        x[np.arange(rows), rng.integers(0, V, rows)] = 40
    for k in range(2):
        s = settings(rng, rows, V)
        check_draw(x, run_draw(x, *s[:4], u=s[4]), *s)


def test_draw_many_rows_of_many_ids():
    """More rows than the slices are for: a workgroup a row past 8192 ids."""
    rng = np.random.default_rng(4)
    x = rng.normal(0, 2.5, (600, 9001)).astype(np.float32)
    s = settings(rng, 600, 9001)
    check_draw(x, run_draw(x, *s[:4], u=s[4]), *s)


def test_draw_edges():
    """NaN, infinities and -0 among the logits; settings and u at and past their ends."""
    V = 300
    rng = np.random.default_rng(1)
    base = rng.normal(0, 2, V).astype(np.float32)
    rows = []
    def add(x, temp=1.0, top_k=0, top_p=1.0, min_p=0.0, u=0.5):  # noqa: E306
        rows.append((np.asarray(x, np.float32), temp, top_k, top_p, min_p, u))
    nan = base.copy()
    nan[::3] = np.nan
    nan[1::3] = -np.inf
    for u in (0.0, 0.5, 1 - 2.0 ** -24, 1.0, 3.0, -1.0, np.nan):
        add(base, u=u)
        add(nan, u=u, top_k=20)
        add(nan, u=u, top_k=250)  # (more than can be drawn)
        add(nan, u=u, top_p=0.7)
    add(np.full(V, np.nan))
    add(np.full(V, -np.inf))
    one = np.full(V, -np.inf)
    one[77] = -3e38
    add(one, u=0.9)
    add(one, temp=0.0)
    inf = base.copy()
    inf[[5, 250]] = np.inf
    for u in (0.0, 0.4, 0.6):
        add(inf, u=u)
        add(inf, u=u, top_k=1)
        add(inf, temp=0.0, u=u)
    zero = np.zeros(V)
    zero[::2] = -0.0
    for u in (0.0, 0.3, 0.7):
        add(zero, u=u, top_k=3)
        add(zero, u=u, top_p=0.5)
    for kw in (dict(top_p=0.0), dict(top_p=-1.0), dict(min_p=1.0), dict(min_p=5.0), dict(top_k=1),
               dict(temp=1e-30), dict(temp=np.inf), dict(temp=np.nan), dict(top_k=V - 1), dict(top_k=1 << 30)):
        add(base, u=0.8, **kw)
    big = base * 1e37
    add(big, temp=1e36, u=0.9)
    x = np.stack([r[0] for r in rows])
    cols = [np.array([r[i] for r in rows]) for i in range(1, 6)]
    check_draw(x, run_draw(x, *cols[:4], u=cols[4]), *cols)


@pytest.mark.parametrize("V", [8193, 30000])
@pytest.mark.parametrize("n", [1, 2, 64, 65, 128, 129, 400, 511, 512, 513, 2000])
def test_draw_cut_among_near_equal_ids(n, V):
    """Rows in slices whose cut lies among n ids of nearly one logit (some of
    them equal), behind 40 likelier ones: by top_k, by top_p, by both, at the
    first of them, at the last and between."""
    rng = np.random.default_rng(n + V)
    rows = 24
    x = np.full((rows, V), -7.0, np.float32) - rng.random((rows, V)).astype(np.float32)
    s = [np.ones(rows, np.float32), np.zeros(rows, np.int32), np.ones(rows, np.float32),
         np.zeros(rows, np.float32), rng.random(rows).astype(np.float32)]
    for r in range(rows):
        ids = rng.permutation(V)
        x[r, ids[:40]] = -0.2 * rng.random(40)
        x[r, ids[40:40 + n]] = -1 - np.round(rng.random(n) * 0.01, 3)
        x[r, ids[-3:]] = np.nan, -np.inf, np.nan
        s[0][r] = (1.0, 0.6, 1.7)[r % 3]
        e = np.where(x[r] > -np.inf, np.exp((x[r].astype(np.float64)) / s[0][r]), 0)
        front, group = e[ids[:40]].sum(), e[ids[40:40 + n]].sum()
        at = (0.001, 0.999, rng.random())[(r // 3) % 3]
        if r % 4 != 1:
            s[1][r] = 40 + max(1, round(at * n))
        if r % 4 == 1:
            s[2][r] = (front + at * group) / np.nansum(e)
        elif r % 4 == 2:
            s[2][r] = (front + 0.5 * at * group) / (front + at * group)
    check_draw(x, run_draw(x, *s[:4], u=s[4]), *s)


def test_draw_defaults_and_repeats():
    """Every setting absent: one draw from softmax(x); the same call gives the same ids."""
    rng = np.random.default_rng(2)
    x = rng.normal(0, 2, (300, 777)).astype(np.float32)
    u = rng.random(300).astype(np.float32)
    got = run_draw(x, u=u)
    n = np.ones(300)
    check_draw(x, got, n, 0 * n, n, 0 * n, u)
    assert np.array_equal(got[0], run_draw(x, u=u)[0])


# ------------------------------------------------------------------ together

def test_a_server_of_its_own():
    """The operators as a caller's own program uses them: a pool's pages, QKV
    rows normed, rotated and appended, attention, an id drawn from each
    sequence's last row; prompts first, then a fork, then single tokens through
    one captured step whose arrays change between replays."""
    H, KH, hd, P, V, n_pages, S = 6, 2, 64, 16, 300, 60, 5
    g = torch.Generator().manual_seed(31)
    normal = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    pool = engine.Pool(n_pages, P, S)
    kv = torch.full((2, n_pages, KH, P, hd), NAN, device="cuda")
    wq, wk = 1 + 0.2 * normal(hd), 1 + 0.2 * normal(hd)
    head = 0.3 * normal(V, H * hd)
    cos, sin = tables(200, hd)
    pg = engine.pages(kv[0].data_ptr(), kv[1].data_ptr(), n_pages, P, KH, hd)
    ap = engine.append_cfg(H, cos.data_ptr(), sin.data_ptr(), 200, norm=True, wq=wq.data_ptr(), wk=wk.data_ptr())
    at = engine.attn_cfg(H)
    ld, rows = 13, 128
    dev = dict(start=torch.zeros(S + 1, dtype=torch.int32).cuda(), kv=torch.zeros(S, dtype=torch.int32).cuda(),
               table=torch.full((S, ld), -1, dtype=torch.int32).cuda(), qkv=torch.zeros(rows, 10 * hd).cuda(),
               q=torch.zeros(rows, H * hd).cuda(), o=torch.zeros(rows, H * hd).cuda(),
               u=torch.zeros(S).cuda(), temp=torch.full((S,), 0.8).cuda(),
               top_k=torch.full((S,), 40, dtype=torch.int32).cuda(), top_p=torch.full((S,), 0.95).cuda(),
               lg=torch.zeros(S, V).cuda(), ids=torch.zeros(S, dtype=torch.int32).cuda())
    bt = {m: engine.ragged(dev["start"].data_ptr(), dev["kv"].data_ptr(), dev["table"].data_ptr(), S, m and rows or S,
                           m or 1, 200, ld) for m in (0, 90)}
    work = torch.empty(max(engine.paged_attn_work(pg, b, at) for b in bt.values()) + 16, dtype=torch.uint8, device="cuda")
    history = {s: [] for s in range(S)}  # QKV rows a sequence was given

    def launch(b, last):
        st = torch.cuda.current_stream().cuda_stream
        engine.qk_append(pg, b, ap, dev["qkv"].data_ptr(), dev["q"].data_ptr(), st)
        engine.paged_attn(pg, b, at, dev["q"].data_ptr(), dev["o"].data_ptr(), work.data_ptr(), work.numel(), st)
        torch.mm(dev["o"][last], head.t(), out=dev["lg"])
        engine.draw_rows(dev["lg"].data_ptr(), S, V, V, dev["u"].data_ptr(), dev["ids"].data_ptr(),
                         temp=dev["temp"].data_ptr(), top_k=dev["top_k"].data_ptr(),
                         top_p=dev["top_p"].data_ptr(), stream=st)

    def put(counts):
        """New rows for the sequences: the pool's pages, copies, the step's arrays."""
        new = {s: normal(n, 10 * hd) for s, n in counts.items()}
        start, copies = [0], []
        for s in range(S):
            n = counts.get(s, 0)
            c = pool.extend(s, n)
            if c:
                copies.append(c)
            t = pool.table(s)
            dev["table"][s].fill_(-1)
            dev["table"][s, :len(t)] = torch.from_numpy(t).cuda()
            if n:
                dev["qkv"][start[-1]:start[-1] + n] = new[s]
                history[s] = history[s] + list(new[s])
            start.append(start[-1] + n)
        if copies:
            engine.pages_copy(kv.data_ptr(), 2, kv.stride(0) * 4, n_pages, KH * P * hd * 4,
                              [a for a, _ in copies], [b for _, b in copies])
        dev["start"].copy_(torch.tensor(start, dtype=torch.int32))
        dev["kv"].copy_(torch.tensor([pool.len(s) for s in range(S)], dtype=torch.int32))
        dev["u"].copy_(torch.rand(S, generator=g))
        return start

    def check(seqs, at_row):
        for s in seqs:
            x = torch.stack(history[s]).double().reshape(-1, 10, hd)
            n = len(x)
            nrm = lambda t, w: t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-5) * w.double()  # noqa: E731
            def rot(t):  # noqa: E306
                c, sn = cos[:n, None].double(), sin[:n, None].double()
                a, b = t.chunk(2, -1)
                return torch.cat([a * c + b * sn, b * c - a * sn], -1)
            q, k, v = rot(nrm(x[:, :H], wq)), rot(nrm(x[:, H:H + KH], wk)), x[:, H + KH:]
            for h in range(H):
                p = torch.softmax((k[:, h // 3] @ q[-1, h]) / math.sqrt(hd), 0)
                want = p @ v[:, h // 3].contiguous()
                got = dev["o"][at_row[s], h * hd:(h + 1) * hd].double()
                # (attention's bound with the append's roundings of q, k and v in it)
                assert (got - want).abs().max() <= 2.0 ** -17 * v.abs().max()
            r = R.draw_row(dev["lg"][s].cpu().numpy(), float(np.float32(0.8)), 40, float(np.float32(0.95)), 0.0,
                           float(dev["u"][s]))
            assert int(dev["ids"][s]) == r[0]

    start = put({0: 50, 1: 7, 2: 1, 3: 33})
    last = torch.tensor([max(0, start[s + 1] - 1) for s in range(S)], device="cuda")
    launch(bt[90], last)
    torch.cuda.synchronize()
    check(range(4), last.tolist())
    pool.fork(0, 4, 40)
    history[4] = history[0][:40]
    one = torch.arange(S, device="cuda")
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    put({s: 1 for s in range(S)})
    launch(bt[0], one)  # (eager once, as a caller warms up)
    torch.cuda.synchronize()
    check(range(S), list(range(S)))
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        launch(bt[0], one)
    for _ in range(20):
        put({s: 1 for s in range(S)})
        graph.replay()
        torch.cuda.synchronize()
        check(range(S), list(range(S)))
    src, dst = (pool.trim(1), pool.trim(2), pool.compact())[2]
    assert len(src)
    engine.pages_copy(kv.data_ptr(), 2, kv.stride(0) * 4, n_pages, KH * P * hd * 4, src, dst)
    history[1], history[2] = [], []
    put({0: 1, 1: 1, 2: 1, 3: 1, 4: 1})
    graph.replay()
    torch.cuda.synchronize()
    check(range(S), list(range(S)))
    pool.close()


# ------------------------------------------------------------------ precision of bf16 rows

@pytest.mark.parametrize("window,sinks", [(0, 0), (600, 4)])
@pytest.mark.parametrize("shape,page", [("gqa5", 64), ("gqa4_64", 16), ("mqa24", 32)])
def test_few_bf16_rows_lose_the_output_rounding_alone(shape, page, window, sinks):
    """Single tokens and short chunks: probabilities in two bf16 terms, each off
    by half a step of what it rounds (2^-16 of a weight in all), so what is left
    is the output's own rounding (2^-8 of it)."""
    H, KH, hd = SHAPES[shape]
    b = R.Batch([(900, 1), (1300, 1), (40, 1), (2500, 1), (700, 1)], H, KH, hd, page, BF16, BF16, seed=41)
    b.fill(window, sinks)
    q = b.normal(b.rows, H * hd, dtype=BF16, std=1.5)
    out, mag, dot = b.attention(q, None, window, sinks)
    got = run_attn(b, q, window, sinks).double().reshape(out.shape)
    tol = R.attn_tolerance(out, mag, dot, hd, 2500, False) + 2.0 ** -16 * mag
    assert ((got - out).abs() <= tol + 2.0 ** -8 * (out.abs() + tol)).all()


# ------------------------------------------------------------------ loose bounds

@pytest.mark.parametrize("max_q", [50, 1 << 29, (1 << 31) - 1])
@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("shape", ["gqa4_64", "gqa5", "mqa24"])
@pytest.mark.parametrize("lengths", ["tokens", "chunks", "prompts"])
def test_bounds_above_the_lengths(lengths, shape, types, max_q):
    """max_q and max_kv are bounds: loose ones, up to the largest that the type
    holds, change nothing (16-row and 128-row tiles, one tile a sequence and
    several)."""
    H, KH, hd = SHAPES[shape]
    qt, kt = TYPES[types]
    b = R.Batch({"tokens": [(700, 1), (40, 1), (0, 0), (1300, 1)], "chunks": [(300, 20), (90, 1), (64, 33)],
                 "prompts": [(900, 900), (1200, 400), (5, 1), (700, 690)]}[lengths], H, KH, hd, 32, qt, kt, seed=51,
                pad=6, slack=77)
    b.max_q = max(b.max_q, max_q)
    b.fill()
    q = b.normal(b.rows, H * hd, dtype=qt)
    check_attn(b, q, run_attn(b, q))


@pytest.mark.parametrize("types", sorted(TYPES))
def test_no_position_at_all(types):
    """Rows of sequences whose cache is empty (max_kv 0): zeros, and nothing appended."""
    qt, kt = TYPES[types]
    b = R.Batch([(0, 3), (0, 0), (0, 40)], 4, 2, 128, 16, qt, kt, seed=52, pad=2)
    assert b.max_kv == 0
    got = run_attn(b, b.normal(b.rows, 4 * 128, dtype=qt))
    assert (got[:43] == 0).all() and (got[43:] == 7.0).all()
    out = torch.full((b.rows, 4 * 128), 7.0, dtype=qt, device="cuda")
    qkv = b.normal(b.rows, 8 * 128, dtype=qt)
    engine.qk_append(pages_of(b), ragged_of(b), engine.append_cfg(4, bf16=qt == BF16), qkv.data_ptr(), out.data_ptr())
    torch.cuda.synchronize()
    assert (out == 7.0).all() and torch.isnan(b.k).all() and torch.isnan(b.v).all()


# ------------------------------------------------------------------ draws: min_p above 1

@pytest.mark.parametrize("rows,V", [(12, 300), (12, 8192), (12, 30000), (600, 9001)])
def test_min_p_above_one_keeps_the_first_largest_id(rows, V):
    """Several ids at the maximum (or, at a large temp, of the same mass as it):
    min_p 1 leaves them all, above 1 the first of the largest alone."""
    rng = np.random.default_rng(V)
    x = rng.normal(0, 1, (rows, V)).astype(np.float32)
    top = np.stack([np.sort(rng.permutation(V)[:5]) for _ in range(rows)])
    for r in range(rows):
        x[r, top[r]] = np.inf if r % 4 == 3 else 9.0
    n = np.ones(rows, np.float32)
    u = ((np.arange(rows) % 10) / 10).astype(np.float32)
    temp = np.where(np.arange(rows) % 3 == 1, 1e30, 1.0).astype(np.float32)
    for min_p in (1.5, 5.0, np.inf, np.nextafter(np.float32(1), np.float32(2))):
        for more in ({}, dict(top_k=0 * n + 4, top_p=0.9 * n), dict(top_p=0.99 * n)):
            ids, probs = run_draw(x, temp=temp, min_p=min_p * n, u=u, **more)
            assert np.array_equal(ids, top[:, 0]) and (probs == 1).all()
    ids, probs = run_draw(x, temp=n, min_p=n, u=u)
    assert np.array_equal(ids, top[np.arange(rows), (u * np.float32(5)).astype(int)])
    assert np.allclose(probs, 0.2, rtol=2.0 ** -23)


# ------------------------------------------------------------------ infinities and NaN that are seen

@pytest.mark.parametrize("bad", [math.inf, -math.inf, NAN], ids=["inf", "-inf", "nan"])
@pytest.mark.parametrize("where", ["key", "value"])
@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("seqs,window", [(((300, 1), (120, 3), (50, 1)), 0), (((700, 500), (400, 300), (90, 20)), 0),
                                         (((700, 500), (400, 300), (90, 20)), 64)], ids=["few", "many", "many_window"])
def test_infinities_stay_in_their_sequence(seqs, window, types, where, bad):
    """One key or value of the second sequence holds it: rows of that sequence
    are the formula's or NaN (also where they do not see it), other sequences
    unchanged."""
    H, KH, hd, dim = 8, 2, 64, 13
    qt, kt = TYPES[types]
    b = R.Batch(list(seqs), H, KH, hd, 32, qt, kt, seed=61)
    b.fill(window, drop_pages=False)
    q = b.normal(b.rows, H * hd, dtype=qt)
    clean = run_attn(b, q, window).double().reshape(b.rows, H, hd)
    exact, mag, dot = b.attention(q, window=window)
    tol = R.attn_tolerance(exact, mag, dot, hd, 700, qt == BF16)
    T, n = seqs[1]
    a = int(b.start_np[1])
    j = T - (n + 1) // 2  # (the chunk's first half does not see it)
    (b.k if where == "key" else b.v)[int(b.table_np[1, j // 32]), 0, j % 32, dim] = bad
    got = run_attn(b, q, window).double().reshape(b.rows, H, hd)
    mine = torch.zeros(b.rows, dtype=torch.bool, device="cuda")
    sees = mine.clone()
    mine[a:a + n] = True
    sees[a:a + n] = b.visible(1, window, 0)[:, j]
    assert torch.equal(got[~mine], clean[~mine])
    assert torch.equal(got[:, H // KH:], clean[:, H // KH:])  # (the other key head's)
    # (not the same bits: rows of a wavefront move their running maxima together,
    # and this one's score or NaN moves them; the bound holds for any maxima)
    assert (((got - exact).abs() <= tol) | torch.isnan(got))[~sees].all()
    at = got[sees][:, :H // KH]
    if where == "value":
        assert (torch.isnan(at[..., dim]) | (at[..., dim] == bad)).all()
        assert torch.equal(*(t[sees][..., [d for d in range(hd) if d != dim]] for t in (got, clean)))
        return
    # a score of -inf leaves the key out, any other one is NaN
    x = q.double().reshape(b.rows, H, hd)
    K, V = (torch.nan_to_num(b.history(t, 1)[0], nan=0.0, posinf=0.0, neginf=0.0) for t in (b.k, b.v))
    see = b.visible(1, window, 0).clone()
    see[:, j] = False
    rest = torch.softmax(((x[a:a + n, :H // KH].reshape(-1, hd) @ K.t().contiguous()) / math.sqrt(hd))
                         .masked_fill(~see.repeat_interleave(H // KH, 0), -math.inf), -1) @ V
    rest = rest.reshape(n, H // KH, hd)[sees[a:a + n]]
    out = (x[sees][:, :H // KH, dim] * bad < 0)[..., None]  # (False for NaN)
    # (as check_attn has it, with sum_j p_j |v_j| and the scores' sizes at their bounds)
    near = (at - rest).abs() <= (2.0 ** -7 if qt == BF16 else 2.0 ** -12) * V.abs().max()
    assert (torch.isnan(at) | (out & near)).all()
