"""Attention with shared prefixes (fg_prefix_attn) on the GPU against the plain
float64 attention of every sequence alone, on pages of every type; rows that nobody
sees are NaN, pages that nobody sees are gone from the tables."""
import numpy as np
import pytest
import torch

from autoresearch_amd import engine

from . import codes_ref as Q
from . import paged_ref as R
from . import test_gpu_codes as TC
from . import test_gpu_paged as TP
from .paged_ref import BF16, F32

pytestmark = pytest.mark.gpu

SHAPES = {"mha128": (3, 3, 128), "gqa5": (10, 2, 128), "gqa4_64": (8, 2, 64), "mqa24": (24, 1, 128)}
TYPES = {"f32": (F32, "f32"), "f32_kv16": (F32, "bf16"), "bf16": (BF16, "bf16"), "f32_i8": (F32, "i8"),
         "bf16_i8": (BF16, "i8"), "f32_e4m3": (F32, "e4m3"), "bf16_e4m3": (BF16, "e4m3")}


def make(groups, shape, page, types, window=0, sinks=0, seed=0, pad=2, slack=0):
    """A batch of groups (shared positions, [(own positions, new tokens), ..]); the
    group None shares nothing and is not among the call's."""
    H, KH, hd = SHAPES[shape]
    qt, kv = TYPES[types]
    seqs = [((sh or 0) + own, n) for sh, members in groups for own, n in members]
    kw = dict(seed=seed, pad=pad, slack=slack)
    if kv in Q.TYPES:
        b = Q.Batch(seqs, H, KH, hd, page, qt, kind=kv, **kw)
    else:
        b = R.Batch(seqs, H, KH, hd, page, qt, F32 if kv == "f32" else BF16, **kw)
    starts, shared, at = [0], [], 0
    for sh, members in groups:
        for s in range(at + 1, at + len(members)):
            b.table_np[s, :(sh or 0) // page] = b.table_np[at, :(sh or 0) // page]
        at += len(members)
        if sh is not None:
            starts.append(at)
            shared.append(sh)
    b.fill(window, sinks, drop_pages=False)
    # a page that no row sees is gone
    seen = np.zeros(b.table_np.shape, bool)
    for s, (T, n) in enumerate(seqs):
        if n and T:
            some = b.visible(s, window, sinks).any(0).cpu().numpy()
            some = np.pad(some, (0, b.ld * page - T))
            seen[s] = some.reshape(b.ld, page).any(1)
    at = 0
    for sh, members in groups:
        k = (sh or 0) // page
        seen[at:at + len(members), :k] = seen[at:at + len(members), :k].any(0)
        at += len(members)
    b.table_np = np.where(seen, b.table_np, b.n_pages + 9).astype(np.int32)
    b.table = b.put(b.table_np)
    b.starts, b.shared_np = np.asarray(starts, np.int32), np.asarray(shared, np.int32)
    b.seq_start, b.shared = b.put(b.starts), b.put(b.shared_np)
    b.max_shared = int(max(shared, default=0))
    return b


def pages_of(b):
    return b.pages() if isinstance(b, Q.Batch) else TP.pages_of(b)


def run(b, q, window=0, sinks=0, scale=0.0, out=None, q_ld=0, out_ld=0, stream=0, max_shared=None):
    cfg = engine.attn_cfg(b.H, window=window, sinks=sinks, scale=scale, bf16=b.qt == BF16, q_ld=q_ld, out_ld=out_ld)
    out = torch.full((b.rows, b.H * b.hd), 7.0, dtype=b.qt, device="cuda") if out is None else out
    pre = engine.prefix(b.seq_start.data_ptr(), b.shared.data_ptr(), len(b.shared_np),
                        b.max_shared if max_shared is None else max_shared)
    n = engine.prefix_attn_work(pages_of(b), TP.ragged_of(b), pre, cfg)
    work = torch.full((max(n, 16),), 255, dtype=torch.uint8, device="cuda")  # (NaN)
    engine.prefix_attn(pages_of(b), TP.ragged_of(b), pre, cfg, q.data_ptr(), out.data_ptr(), work.data_ptr(), n,
                       stream)
    torch.cuda.synchronize()
    return out


def check(b, q, got, window=0, sinks=0, scale=None):
    # (the parts' join adds the same terms in another order, which the tolerances count)
    (TC if isinstance(b, Q.Batch) else TP).check_attn(b, q, got, window, sinks, scale)


def normal_q(b, std=1.5):
    return b.normal(b.rows, b.H * b.hd, dtype=b.qt, std=std)


GROUPS = {
    "tokens": [(512, [(1, 1), (40, 1), (7, 1), (33, 1)])],
    "one_member": [(256, [(5, 5)]), (512, [(64, 1)])],
    "beside_others": [(768, [(20, 1), (300, 1)]), (0, [(9, 1), (70, 3)]), (256, [(1, 1)] * 5), (None, [(600, 1), (4, 4)])],
    "below_a_tile": [(16, [(20, 1), (3, 1)]), (48, [(1, 1), (2, 2), (30, 1)])],
    "without_tokens": [(256, [(30, 0), (40, 1), (0, 0), (1, 1), (50, 2)]), (512, [(9, 0), (8, 0)]), (256, [(3, 1)])],
    "chunks": [(1024, [(40, 40), (200, 7), (130, 1), (90, 90)]), (512, [(17, 16)] * 3)],
    "many": [(1536, [(30 + 7 * i, 1 + i % 3) for i in range(70)]), (256, [(200, 150), (150, 150)])],
    "long": [(6144, [(100, 1), (2000, 1)])],
}


@pytest.mark.parametrize("groups", sorted(GROUPS))
@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("shape,page", [("mha128", 16), ("gqa5", 16), ("gqa4_64", 16), ("mqa24", 16), ("gqa5", 256)])
def test_groups(shape, page, types, groups):
    g = GROUPS[groups]
    if any((sh or 0) % page for sh, _ in g):
        g = [(sh if sh is None else sh * 16, m) for sh, m in g]
    b = make(g, shape, page, types, seed=len(groups))
    q = normal_q(b)
    check(b, q, run(b, q))


@pytest.mark.parametrize("window,sinks", [(1, 0), (30, 4), (200, 0), (200, 300), (700, 70), (5000, 1)])
@pytest.mark.parametrize("types", ["f32", "bf16", "f32_i8", "bf16_e4m3"])
@pytest.mark.parametrize("shape,page", [("gqa5", 16), ("gqa4_64", 32), ("mha128", 64)])
@pytest.mark.parametrize("groups", ["tokens", "chunks", "beside_others"])
def test_window(shape, page, types, window, sinks, groups):
    b = make(GROUPS[groups], shape, page, types, window, sinks, seed=window)
    q = normal_q(b)
    check(b, q, run(b, q, window, sinks), window, sinks)


@pytest.mark.parametrize("types", sorted(TYPES))
def test_large_scores_and_scale(types):
    """Scores in the hundreds: one part holds all of the mass."""
    b = make(GROUPS["chunks"], "gqa4_64", 32, types, seed=4)
    q = normal_q(b, 30.0)
    check(b, q, run(b, q))
    check(b, q, run(b, q, scale=0.01), scale=float(np.float32(0.01)))


@pytest.mark.parametrize("bound", [0, 31, 100, 700])
def test_less_shared_than_said(bound):
    """max_shared below a group's shared positions; more groups than share anything."""
    b = make(GROUPS["beside_others"], "gqa5", 16, "f32_kv16", seed=5)
    q = normal_q(b)
    check(b, q, run(b, q, max_shared=bound))


def test_group_bounds_outside():
    """Group bounds outside the sequences are taken as the nearest."""
    b = make([(256, [(5, 1), (40, 1)]), (512, [(33, 1), (2, 2)])], "gqa5", 16, "f32", seed=6)
    q = normal_q(b)
    want = run(b, q)
    b.seq_start = b.put(np.asarray([-7, 2, 1 << 30], np.int32))
    assert torch.equal(want, run(b, q))
    b.shared = b.put(np.asarray([-5, -(1 << 30)], np.int32))  # nothing shared
    check(b, q, run(b, q))


@pytest.mark.parametrize("types", sorted(TYPES))
def test_bad_page_gives_nan_rows(types):
    b = make([(256, [(30, 1), (40, 2)]), (512, [(9, 1), (8, 1)]), (256, [(3, 1)])], "gqa5", 16, types, seed=7)
    b.table_np[0, 9] = b.n_pages
    b.table_np[3, 32] = -5  # an own page of the second group's second member
    b.table_np[3, 0] = b.n_pages + 1  # (shared: the first member's is read)
    b.table = b.put(b.table_np)
    got = run(b, normal_q(b))
    bad = torch.zeros(b.rows, dtype=torch.bool, device="cuda")
    bad[[0, 1, 2, 4]] = True
    assert torch.isnan(got[bad]).all() and torch.isfinite(got[~bad]).all()


def test_strided_rows_and_place():
    b = make(GROUPS["chunks"], "gqa5", 16, "f32_kv16", seed=8)
    wide = b.normal(b.rows, 14 * 128)
    out = torch.full((b.rows, 12 * 128), 7.0, device="cuda")
    run(b, wide, out=out, q_ld=14 * 128, out_ld=12 * 128)
    q = wide[:, :1280].contiguous()
    check(b, q, out[:, :1280].contiguous())
    assert (out[:, 1280:] == 7.0).all()
    want = run(b, q)
    q2 = q.clone()
    q2[b.used:] = 7.0
    assert torch.equal(run(b, q2, out=q2), want)


@pytest.mark.parametrize("types", ["f32", "bf16_e4m3"])
def test_repeats_and_streams(types):
    """The same bits twice, on another stream, and behind each other on two."""
    bs = [make(GROUPS[n], "gqa5", 16, types, seed=9) for n in ("many", "tokens")]
    qs = [normal_q(b) for b in bs]
    want = [run(b, q) for b, q in zip(bs, qs)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    calls = []
    for b, q in zip(bs, qs):
        cfg = engine.attn_cfg(b.H, bf16=b.qt == BF16)
        pre = engine.prefix(b.seq_start.data_ptr(), b.shared.data_ptr(), len(b.shared_np), b.max_shared)
        n = engine.prefix_attn_work(pages_of(b), TP.ragged_of(b), pre, cfg)
        calls.append((b, cfg, pre, n, torch.empty(n, dtype=torch.uint8, device="cuda"), q,
                      [torch.full_like(q, 7.0) for _ in range(5)]))
    torch.cuda.synchronize()
    for i in range(5):
        for k, (b, cfg, pre, n, work, q, outs) in enumerate(calls):
            engine.prefix_attn(pages_of(b), TP.ragged_of(b), pre, cfg, q.data_ptr(), outs[i].data_ptr(),
                               work.data_ptr(), n, streams[k].cuda_stream)
    torch.cuda.synchronize()
    for w, c in zip(want, calls):
        assert all(torch.equal(w, o) for o in c[-1])


def test_capture_replays_other_groups():
    """One captured call serves other lengths, groups and shared positions within its
    bounds; two graphs with a workspace each, eager work between the replays."""
    H, KH, hd, P = 10, 2, 128, 32
    batches = [make(g, "gqa5", P, "f32_kv16", seed=i, pad=0)
               for i, g in enumerate([[(1024, [(1, 1), (200, 4), (3, 3)]), (256, [(50, 1)])],
                                      [(64, [(300, 9), (8, 1)]), (512, [(1, 1), (40, 30)])],
                                      [(0, [(700, 1)]), (1024, [(2, 2), (90, 1), (7, 0)])]])]
    rows, ld, max_kv = 44, 42, 1344
    n_pages = max(b.n_pages for b in batches)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    st = dict(start=i32(5), kv=i32(4), table=i32(4, ld), seq_start=i32(3), shared=i32(2),
              q=torch.zeros(rows, H * hd, device="cuda"))
    k, v = (torch.zeros(n_pages, KH, P, hd, dtype=BF16, device="cuda") for _ in range(2))
    pg = engine.pages(k.data_ptr(), v.data_ptr(), n_pages, P, KH, hd, bf16=True)
    bt = engine.ragged(st["start"].data_ptr(), st["kv"].data_ptr(), st["table"].data_ptr(), 4, rows, 30, max_kv, ld)
    pre = engine.prefix(st["seq_start"].data_ptr(), st["shared"].data_ptr(), 2, 1024)
    cfg = engine.attn_cfg(H)
    n = engine.prefix_attn_work(pg, bt, pre, cfg)
    outs, graphs, works = [], [], []
    for _ in range(2):
        out = torch.full((rows, H * hd), 7.0, device="cuda")
        work = torch.empty(n, dtype=torch.uint8, device="cuda")
        g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
            engine.prefix_attn(pg, bt, pre, cfg, st["q"].data_ptr(), out.data_ptr(), work.data_ptr(), n,
                               torch.cuda.current_stream().cuda_stream)
        outs.append(out)
        graphs.append(g)
        works.append(work)
    for b in batches + batches[:1]:
        k[:b.n_pages], v[:b.n_pages] = b.k, b.v
        for name, t in (("start", b.start), ("kv", b.kv_len), ("seq_start", b.seq_start), ("shared", b.shared)):
            st[name].copy_(t)
        st["table"].fill_(-1)
        st["table"][:, :b.ld].copy_(b.table)
        q = normal_q(b)
        st["q"][:b.rows].copy_(q)
        for o in outs:
            o.fill_(7.0)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1])
        check(b, q, outs[0][:b.rows])
        assert (outs[0][b.rows:] == 7.0).all()


def test_far_pages():
    """Shared pages past 2^31 elements of a pool."""
    b = make([(512, [(3, 1), (70, 2)])], "gqa5", 256, "bf16", seed=10)
    q = normal_q(b)
    want = run(b, q)
    n_pages = (1 << 31) // (256 * 2 * 128) + 40
    k = torch.empty(n_pages, 2, 256, 128, dtype=BF16, device="cuda")
    v = torch.empty_like(k)
    far = n_pages - b.n_pages
    k[far:], v[far:] = b.k, b.v
    b.k, b.v, b.n_pages = k, v, n_pages
    b.table_np = (b.table_np + far).astype(np.int32)
    b.table = b.put(b.table_np)
    assert torch.equal(run(b, q), want)


@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 3)])
@pytest.mark.parametrize("types", ["f32", "bf16_i8"])
def test_tokens_among_the_shared(types, window, sinks):
    """Sequences with a new token below shared[g] read all of their keys themselves;
    the others of their group are as they were."""
    g = [(512, [(1, 1), (10, 30), (3, 500), (200, 2)]), (512, [(5, 511), (7, 1)])]
    b = make(g, "gqa5", 16, types, window, sinks, seed=11)
    q = normal_q(b)
    check(b, q, run(b, q, window, sinks), window, sinks)
