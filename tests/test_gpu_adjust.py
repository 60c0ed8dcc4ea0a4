"""fg_adjust_rows on the GPU: every step is one fp32 operation, so the results are
those of the same steps in numpy, bit for bit; and within their roundings of the
definition in float64."""
import numpy as np
import pytest
import torch

from autoresearch_amd import engine

pytestmark = pytest.mark.gpu
F = np.float32
NAN, INF = float("nan"), float("inf")


def reference(x, hist=None, count_from=None, rep=None, pres=None, freq=None, bias=None, mask=None, mask_row=None,
              real=F):
    """The definition row by row; hist, bias: a list (of ids, of (id, value)) a row."""
    out = x.astype(real)
    rows, V = x.shape
    for r in range(rows):
        get = lambda a, off: off if a is None or np.isnan(a[r]) else a[r]  # noqa: E731
        y = out[r]
        with np.errstate(all="ignore"):
            if hist is not None and not (rep is None and pres is None and freq is None):
                h = np.asarray(hist[r], np.int64)
                late = h[max(0, 0 if count_from is None else int(count_from[r])):]
                h, late = (a[(a >= 0) & (a < V)] for a in (h, late))
                ids, n = np.unique(late, return_counts=True)
                p, f, t = real(get(pres, 0)), real(get(freq, 0)), real(get(rep, 1))
                t = t if t > 0 else real(1)
                y[ids] = (y[ids] - p) - f * n.astype(real)
                ids = np.unique(h)
                y[ids] = np.where(y[ids] > 0, y[ids] / t, y[ids] * t)
            if bias is not None:
                for i, v in bias[r]:
                    if 0 <= i < V:
                        y[i] = y[i] + real(v)
        if mask is not None:
            m = r if mask_row is None else int(mask_row[r])
            if 0 <= m < len(mask):
                bits = np.unpackbits(mask[m].view(np.uint8), bitorder="little")[:V]
                y[bits == 0] = -INF
    return out


def lists(parts, dtype):
    start = np.concatenate([[0], np.cumsum([len(p) for p in parts])]).astype(np.int32)
    flat = [v for p in parts for v in p]
    return start, np.asarray(flat, dtype)


def run(x, hist=None, count_from=None, rep=None, pres=None, freq=None, bias=None, mask=None, mask_row=None, pad=3,
        in_place=False, stream=0, out_pad=1):
    rows, V = x.shape
    keep = []

    def put(a, t):
        if a is None:
            return 0
        keep.append(torch.from_numpy(np.ascontiguousarray(np.asarray(a, t))).cuda())
        return keep[-1].data_ptr()

    kw = {}
    if hist is not None:
        start, flat = lists(hist, np.int32)
        kw.update(hist=put(flat, np.int32), hist_start=put(start, np.int32), n_hist=flat.size)
    if bias is not None:
        start, ids = lists([[i for i, _ in p] for p in bias], np.int32)
        _, val = lists([[v for _, v in p] for p in bias], F)
        kw.update(bias=put(val, F), bias_id=put(ids, np.int32), bias_start=put(start, np.int32), n_bias=ids.size)
    if mask is not None:
        wide = np.pad(mask, ((0, 0), (0, 2)))
        kw.update(mask=put(wide.view(np.int32), np.int32), n_mask=len(mask), mask_ld=wide.shape[1],
                  mask_row=put(mask_row, np.int32))
    cfg = engine.adjust_cfg(count_from=put(count_from, np.int32), rep=put(rep, F), pres=put(pres, F),
                            freq=put(freq, F), **kw)
    lg = torch.full((rows, V + pad), 99.0, device="cuda")
    lg[:, :V] = torch.from_numpy(x).cuda()
    out = lg if in_place else torch.full((rows, V + out_pad), 99.0, device="cuda")
    torch.cuda.synchronize()
    engine.adjust_rows(lg.data_ptr(), rows, V, V + pad, cfg, out.data_ptr(), out.shape[1], stream)
    torch.cuda.synchronize()
    assert (out[:, V:] == 99.0).all()
    if not in_place:
        assert np.array_equal(lg[:, :V].cpu().numpy(), x, equal_nan=True)
    return out[:, :V].cpu().numpy()


def same(a, b):
    number = ~np.isnan(b)  # (NaN have no sign here)
    return np.array_equal(a, b, equal_nan=True) and np.array_equal(np.signbit(a[number]), np.signbit(b[number]))


def settings(rng, rows, V, hist=200, bias=30, masks=3):
    ids = lambda n: (rng.pareto(0.6, n) * 3).astype(np.int64) % (V + 2) - 1  # noqa: E731 (-1 and V too)
    word = rng.integers(0, 1 << 32, (masks, (V + 31) // 32), dtype=np.uint64).astype(np.uint32)
    off = lambda a: np.where(rng.random(rows) < 0.2, NAN, a).astype(F)  # noqa: E731
    return dict(hist=[ids(rng.integers(0, hist + 1)) for _ in range(rows)],
                count_from=rng.integers(-3, hist + 5, rows), rep=off(rng.uniform(0.8, 1.6, rows)),
                pres=off(rng.uniform(-0.5, 1, rows)), freq=off(rng.uniform(-0.2, 0.5, rows)),
                bias=[[(int(i), float(F(v))) for i, v in zip(rng.integers(-1, V + 1, n), rng.normal(0, 3, n))]
                      for n in rng.integers(0, bias + 1, rows)],
                mask=word, mask_row=rng.integers(-2, masks + 2, rows))


@pytest.mark.parametrize("V,rows", [(1, 3), (2, 9), (31, 5), (33, 5), (1000, 40), (1023, 2), (1025, 2), (4095, 9),
                                    (4097, 9), (8192, 64), (8192, 300), (50257, 7), (131073, 20), (262144, 9)])
def test_everything(V, rows):
    rng = np.random.default_rng(V + rows)
    x = rng.normal(0, 3, (rows, V)).astype(F)
    s = settings(rng, rows, V)
    got = run(x, **s)
    assert same(got, reference(x, **s))
    # float64: a difference of three terms, a quotient and a sum, each rounded once
    want = reference(x, **s, real=np.float64)
    fin = np.isfinite(want)
    assert np.array_equal(fin, np.isfinite(got))
    big = np.abs(x) + 1 + 0.5 * 200 + np.max([sum(abs(v) for _, v in p) for p in s["bias"]] + [0.0])
    assert (np.abs(got[fin] - want[fin]) <= (2.0 ** -24 * 40 * 2 * big)[fin]).all()


@pytest.mark.parametrize("names", [("hist", "rep"), ("hist", "pres"), ("hist", "freq", "count_from"), ("hist",),
                                   ("bias",), ("mask",), ("mask", "mask_row"), ("hist", "rep", "bias"), ()])
@pytest.mark.parametrize("rows", [1, 4, 200])
def test_steps_alone(names, rows):
    rng = np.random.default_rng(rows + len(names))
    x = rng.normal(0, 3, (rows, 5000)).astype(F)
    s = settings(rng, rows, 5000, masks=rows)
    s = {k: v for k, v in s.items() if k in names}
    assert same(run(x, **s), reference(x, **s))
    assert same(run(x, in_place=True, **s), reference(x, **s))


def test_odd_settings():
    """rep of 0, below 0, infinite; infinite penalties; infinities and NaN among the logits."""
    rng = np.random.default_rng(5)
    rows, V = 12, 70
    x = rng.normal(0, 3, (rows, V)).astype(F)
    x[:, 3], x[:, 5], x[:, 7], x[:, 9] = INF, -INF, NAN, -0.0
    s = settings(rng, rows, V, hist=100)
    s["hist"] = [np.arange(V).repeat(2)] * rows
    s["rep"] = np.array([0, -1, INF, NAN, 1e-30, 1e30, 1, 2, 1.5, -0.0, 3, 1.0001], F)
    s["pres"] = np.array([INF, 0, 0, -INF, 1, 1e30, 0, NAN, 2, 0, 0, 0], F)
    s["freq"] = np.array([0, INF, 0, 0, 0, 1e38, NAN, 0, 0, -1, 0, 0], F)
    assert same(run(x, **s), reference(x, **s))


@pytest.mark.parametrize("V", [600, 9000])
@pytest.mark.parametrize("rows", [2, 300])
def test_biases_named_often(V, rows):
    """Ids named twice, in one piece of the list and far apart, and a thousand times:
    they are added in the list's order, whoever runs first."""
    rng = np.random.default_rng(6)
    x = rng.normal(0, 3, (rows, V)).astype(F)
    bias = []
    for r in range(rows):
        ids = np.concatenate([[4] * 1000, rng.integers(0, 40, 300), [V - 1, V - 1], rng.integers(0, V, 400)])
        rng.shuffle(ids)
        bias.append([(int(i), float(F(v))) for i, v in zip(ids, rng.normal(0, 100, ids.size))])
    bias[0] = [(3, 1e30), (3, -1e30), (3, 1.0), (5, INF), (5, 1.0), (6, -INF), (6, INF)]
    one = run(x, bias=bias)
    assert same(one, reference(x, bias=bias))
    assert same(one, run(x, bias=bias))


def test_lists_cut_off():
    """Starts that fall, lie below 0 or past the lists' ends; ids far outside."""
    x = torch.zeros(5, 50, device="cuda")
    out = torch.full_like(x, 9.0)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    hist, start = i32([1, 2, 3, 2 ** 31 - 1, -2 ** 31, 4]), i32([-8, 2, 1, 100, 5, 2 ** 31 - 1])
    ids, bstart = i32([7, -2 ** 31, 2 ** 31 - 1, 50, 8]), i32([4, 9, -1, 2, 2, 1])
    val, pres = torch.ones(5, device="cuda"), torch.ones(5, device="cuda")
    cfg = engine.adjust_cfg(hist=hist.data_ptr(), hist_start=start.data_ptr(), n_hist=6, pres=pres.data_ptr(),
                            bias=val.data_ptr(), bias_id=ids.data_ptr(), bias_start=bstart.data_ptr(), n_bias=5,
                            count_from=i32([0, 0, 0, 0, -2 ** 31]).data_ptr())
    engine.adjust_rows(x.data_ptr(), 5, 50, 50, cfg, out.data_ptr(), 50)
    torch.cuda.synchronize()
    want = torch.zeros(5, 50)
    want[0, [1, 2]] = -1   # [0, 2)
    want[2, [2, 3, 4]] = -1  # [1, 6)
    want[4, 4] = -1        # [5, 6)
    want[0, 8] = 1         # [4, 5)
    want[2, 7] = 1         # [0, 2)
    assert torch.equal(out.cpu(), want)


def test_long_history():
    rng = np.random.default_rng(8)
    V, rows = 3000, 3
    x = rng.normal(0, 3, (rows, V)).astype(F)
    s = dict(hist=[rng.integers(0, V, 100000) % (r * 1000 + 5) for r in range(rows)],
             count_from=np.array([0, 99999, 5000]), freq=np.full(rows, 0.001, F), rep=np.full(rows, 1.1, F))
    assert same(run(x, **s), reference(x, **s))


def test_adjusted_draws_in_a_graph():
    """Adjust and draw in one graph on a stream of the caller's, other histories and
    masks each replay: equal to the eager calls', and masked ids are never drawn."""
    rows, V, L = 17, 8192, 300
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(rows, V, generator=g, device="cuda") * 3
    hist = torch.randint(0, V, (rows * L,), generator=g, device="cuda", dtype=torch.int32)
    start = torch.arange(rows + 1, device="cuda", dtype=torch.int32) * L
    pen = torch.full((rows,), 0.7, device="cuda")
    mask = torch.randint(-2 ** 31, 2 ** 31 - 1, (rows, V // 32), generator=g, device="cuda", dtype=torch.int32)
    u = torch.rand(rows, generator=g, device="cuda")
    out, ids = torch.zeros_like(x), torch.zeros(rows, dtype=torch.int32, device="cuda")
    cfg = engine.adjust_cfg(hist=hist.data_ptr(), hist_start=start.data_ptr(), n_hist=rows * L, pres=pen.data_ptr(),
                            freq=pen.data_ptr(), mask=mask.data_ptr(), n_mask=rows)
    n = engine.draw_rows_work(rows, V)
    work = torch.empty(max(16, n), dtype=torch.uint8, device="cuda")

    def calls(stream):
        engine.adjust_rows(x.data_ptr(), rows, V, V, cfg, out.data_ptr(), V, stream)
        engine.draw_rows(out.data_ptr(), rows, V, V, u.data_ptr(), ids.data_ptr(), work=work.data_ptr(), work_bytes=n,
                         stream=stream)

    gr, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s), torch.cuda.graph(gr, stream=s):
        calls(torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        hist.random_(0, V, generator=g)
        mask.random_(-2 ** 31, 2 ** 31 - 1, generator=g)
        u.uniform_(generator=g)
        gr.replay()
        torch.cuda.synchronize()
        got = out.clone(), ids.clone()
        out.zero_(), ids.zero_()
        calls(0)
        torch.cuda.synchronize()
        assert torch.equal(got[0], out) and torch.equal(got[1], ids)
        bit = mask.gather(1, (ids[:, None] // 32).long())[:, 0] >> (ids % 32) & 1
        assert (bit == 1).all()


def test_mask_of_nothing_draws_nothing():
    x = np.zeros((2, 100), F)
    mask = np.array([[0, 0, 0, 0], [0, 8, 0, 0xFFFFFFF0]], np.uint32)  # (bits past V count for nothing)
    got = run(x, mask=mask)
    assert np.isneginf(got[0]).all() and np.flatnonzero(got[1] == 0).tolist() == [35]
    lg = torch.from_numpy(got).cuda()
    ids, u = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(2, device="cuda")
    engine.draw_rows(lg.data_ptr(), 2, 100, 100, u.data_ptr(), ids.data_ptr())
    assert ids.tolist() == [-1, 35]
