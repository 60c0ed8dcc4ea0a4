"""A model's paged cache in 8 bits, with shared prefixes, and steps that draw from
adjusted logits: against the float64 model of test_gpu_paged_step.py, whose bars hold
(5e-5 x max|logit| on an fp32 cache)."""
import math

import numpy as np
import pytest
import torch

from autoresearch_amd import engine
from autoresearch_amd.weights import rope_tables, seeded_weights, uniform_ids

from . import codes_ref as Q
from . import paged_ref as R
from . import test_gpu_adjust as TA
from . import test_gpu_paged_step as TS

pytestmark = pytest.mark.gpu

MAX = TS.MAX
setup = TS.setup
relerr = TS.relerr


class Exact(TS.Exact):
    """The float64 model, keys and values as the 8-bit type holds them."""

    kind = None

    def hold(self, x):
        """[n, KH, hd] float64 -> the values of its codes, by the definition in float64."""
        if self.kind is None:
            return x
        top = Q.TOP[self.kind]
        s = x.abs().amax(-1, keepdim=True) / top
        y = (x / s.clamp(min=1e-300)).clamp(-top, top)
        if self.kind == "i8":
            return y.round() * s
        return y.float().to(torch.float8_e4m3fn).double() * s

    def logits(self, ids, window=0, sinks=0):
        d, w = self.d, self.w
        n, H, KH, hd = len(ids), d.n_head, d.n_kv_head, d.head_dim
        p, j = torch.arange(n)[:, None], torch.arange(n)[None, :]
        seen = j <= p
        if window:
            seen = seen & ((j > p - window) | (j < sinks))
        x = self.norm(w["wte"][torch.from_numpy(np.asarray(ids, np.int64))])
        kvs = []
        for l in range(d.n_layer):
            y = self.norm(x)
            q = self.rot((y @ w["q"][l].T).view(n, H, hd))
            k, v = self.rot((y @ w["k"][l].T).view(n, KH, hd)), (y @ w["v"][l].T).view(n, KH, hd)
            kvs.append((k, v))
            k, v = (self.hold(t).repeat_interleave(H // KH, 1) for t in (k, v))
            sc = torch.einsum("nhd,mhd->hnm", q, k) / math.sqrt(hd)
            a = torch.softmax(sc.masked_fill(~seen, -math.inf), -1)
            x = x + torch.einsum("hnm,mhd->nhd", a, v).reshape(n, -1) @ w["p"][l].T
            h = (self.norm(x) @ w["f"][l].T).clamp(min=0)
            x = x + (h * h) @ w["g"][l].T
        return (self.norm(x) @ w["lm"].T).numpy(), kvs


# A value next to a border between two codes may get the other one: one of a row's hd
# values is then off by a code's step, 1/127 of the row's largest or 1/8 of itself. Borders
# are met by fp32 noise (2^-16 of the largest, the linears') in a share of about 127 2^-16 or
# 8 2^-16 = 2^-9 or 2^-13 of the values: a row's relative error is at most sqrt(2^-9) / 127
# or sqrt(2^-13) / 8 = 2^-11.5 or 2^-9.5 then, and attention averages over rows. Two layers
# of it, and a factor of two:
BARS = {"i8": 2 * 2 * 2.0 ** -11.5, "e4m3": 2 * 2 * 2.0 ** -9.5}


def exact_of(ex, kind):
    e = Exact.__new__(Exact)
    e.__dict__.update(ex.__dict__)
    e.kind = kind
    return e


@pytest.mark.parametrize("kind", sorted(Q.TYPES))
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3)], ids=["all", "window"])
def test_ragged_passes_in_8_bits(setup, kind, window, sinks):
    d, m, ex = setup
    ex = exact_of(ex, kind)
    pc = m.paged(80, 16, 8, type=Q.TYPES[kind], window=window, sinks=sinks)
    text = {s: uniform_ids(100 + s, MAX, d.vocab) for s in range(8)}
    at = {s: 0 for s in range(8)}

    def step(counts):
        lg, nxt = pc.step({s: text[s][at[s]:at[s] + n] for s, n in counts.items()})
        for i, (s, n) in enumerate(counts.items()):
            at[s] += n
            want, _ = ex.logits(text[s][:at[s]], window, sinks)
            assert relerr(lg[i], want[-1]) < BARS[kind], (s, at[s], relerr(lg[i], want[-1]))
            assert nxt[i] == int(lg[i].argmax())

    step({3: 1})
    step({1: 37, 3: 1, 2: 16, 0: 3})
    step({5: 150, 6: 200, 1: 1, 7: 5})
    step({s: 1 for s in (7, 6, 5, 3, 2, 1, 0)})
    pc.trim(5)
    pc.fork(6, 5, 150 if not window else 200)
    at[5], text[5] = pc.len(5), np.concatenate([text[6][:pc.len(5)], uniform_ids(300, 100, d.vocab)])
    step({5: 3, 6: 2})
    pc.trim(2)
    pc.compact()
    step({6: 1, 5: 1, 0: 40})
    # what is held is the keys and values, to half a step of a code
    for s in (0, 6):
        k, v = pc.read(s)
        _, kvs = ex.logits(text[s][:at[s]], window, sinks)
        lost = (k[0] == 0).all(-1)
        assert window or not lost.any()
        first = kvs[0]  # (later layers see the errors of earlier ones)
        for got, want in zip((k[0], v[0]), first):
            got = torch.from_numpy(got).double().reshape(want.shape)
            top = want.abs().amax(-1, keepdim=True)
            step_ = top / 127 / 2 if kind == "i8" else torch.maximum(want.abs() * 2.0 ** -4, top * 2.0 ** -10 / 448)
            assert ((got - want).abs() <= 1.02 * step_ + 1e-4 * top)[torch.from_numpy(~lost)].all()
    pc.close()


def taken(m, pc, f, saved):
    """f()'s answer; whether its step read the shared keys once (its bytes say so)."""
    m.timing(True)
    out = f()
    got = m.timing_read()
    m.timing(False)
    return out, saved and got["attn_decode"][3] + got["attn_chunk"][3] < saved


@pytest.mark.parametrize("type,window,sinks", [(engine.FG_F32, 0, 0), (engine.FG_F32, 200, 5), (engine.FG_BF16, 0, 0),
                                               (engine.FG_E4M3, 0, 0)])
def test_shared_prefixes(setup, type, window, sinks):
    """Many forks of two prompts, beside others, tokens and chunks: each sequence's
    logits are near those of a cache that reads every sequence alone, and a sample of
    them are the float64 model's."""
    d, m, ex = setup
    ex = exact_of(ex, "e4m3" if type == engine.FG_E4M3 else None)
    bar = {engine.FG_F32: 5e-5, engine.FG_BF16: 2e-3, engine.FG_E4M3: BARS["e4m3"]}[type]
    pcs = [m.paged(900, 16, 256, type=type, window=window, sinks=sinks, prefix=p) for p in (True, False)]
    prompts = [uniform_ids(7, 300, d.vocab), uniform_ids(8, 260, d.vocab), uniform_ids(9, 50, d.vocab)]
    B = 190  # the second prompt's first
    for pc in pcs:
        pc.step({0: prompts[0], B: prompts[1], 255: prompts[2]}, want_logits=False)
        for s in range(1, B):
            pc.fork(0, s, 300 - (s % 4) if not window else 300)
        for s in range(B + 1, 250):
            pc.fork(B, s)
    text = {s: prompts[0][:pcs[0].len(s)] for s in range(B)} | {s: prompts[1] for s in range(B, 250)}
    text[255] = prompts[2]
    for k in range(3):
        new = {s: uniform_ids(1000 * k + s, 1 if k < 2 else 1 + s % 4, d.vocab) for s in text}
        if k == 1:  # another order, a sequence left out
            new = {s: new[s] for s in [255, *range(B - 1, 5, -1), *range(0, 5), *range(249, B - 1, -1)]}
        row = {engine.FG_F32: 4.0, engine.FG_BF16: 2.0, engine.FG_E4M3: (d.head_dim + 4) / d.head_dim}[type]
        alone = 2 * row * d.n_kv_head * d.head_dim * d.n_layer * sum(len(text[s]) for s in new)
        (lg, _), once = taken(m, pcs[0], lambda: pcs[0].step(new), 0 if window else 0.5 * alone)
        assert window or once
        lg2, _ = pcs[1].step(new)
        assert relerr(lg, lg2) < 2 * bar
        for i, s in enumerate(new):
            text[s] = np.concatenate([text[s], new[s]])
            if s % 25 == 0 or s in (255, 249, B - 1):
                want, _ = ex.logits(text[s], window, sinks)
                assert relerr(lg[i], want[-1]) < bar, (k, s, relerr(lg[i], want[-1]))
    for pc in pcs:
        pc.close()


def test_steps_that_adjust(setup):
    """Ids are the draw's definition on the adjusted logits' definition; the logits that
    come back are the model's own."""
    d, m, ex = setup
    pcs = [m.paged(60, 16, 6) for _ in range(2)]
    prompts = {s: uniform_ids(30 + s, 20 + 9 * s, d.vocab) for s in range(6)}
    for pc in pcs:
        pc.step(prompts, want_logits=False)
    rng = np.random.default_rng(4)
    text = {s: list(prompts[s]) for s in range(6)}
    allowed = [None if s % 3 == 0 else rng.random(d.vocab) < 0.1 for s in range(6)]
    for k in range(5):
        new = {s: [int(rng.integers(d.vocab))] for s in range(6)}
        for s in range(6):
            text[s] += new[s]
        u = rng.random(6).astype(np.float32)
        s = dict(history=[np.asarray(t, np.int32) for t in text.values()],
                 count_from=[prompts[i].size for i in range(6)], rep=np.float32(1.3),
                 pres=rng.uniform(0, 1, 6).astype(np.float32), freq=np.float32(0.2),
                 bias=[{i: 2.0, d.vocab - 1 - i: -3.0} if i % 2 else None for i in range(6)], allowed=allowed)
        draw = dict(u=u, temp=0.8, top_k=50) if k < 3 else {}
        lg, ids = pcs[0].step(new, **s, **draw)
        assert np.array_equal(lg, pcs[1].step(new)[0])
        mask = np.stack([np.packbits(np.ones(d.vocab, bool) if a is None else a, bitorder="little").view(np.uint32)
                         for a in allowed])
        full = lambda v: np.broadcast_to(np.asarray(v, np.float32), (6,))  # noqa: E731
        want = TA.reference(lg, hist=s["history"], count_from=np.asarray(s["count_from"]), rep=full(s["rep"]),
                            pres=full(s["pres"]), freq=full(s["freq"]),
                            bias=[list((b or {}).items()) for b in s["bias"]], mask=mask)
        for i in range(6):
            if draw:
                one = R.draw_row(want[i], float(np.float32(0.8)), 50, 1.0, 0.0, float(u[i]))[0]
            else:
                one = int(want[i].argmax())
            assert ids[i] == one, (k, i)
    # a mask that leaves nothing
    _, ids = pcs[0].step({0: [1], 1: [2]}, allowed=[np.zeros(d.vocab, bool), None])
    assert ids[0] == -1 and ids[1] >= 0
    for f in (dict(rep=1.2), dict(history=[[1]]), dict(allowed=[None]), dict(bias=[{}, {}, {}])):
        with pytest.raises(ValueError):
            pcs[0].step({0: [1], 1: [2]}, **f)
    lib = engine.load_library()
    i32 = lambda *v: (engine.C.c_int32 * len(v))(*v)  # noqa: E731
    cfg = engine.adjust_cfg(n_hist=1)
    n = pcs[0].len(0)
    for c, nx in ((cfg, i32(0)), (engine.adjust_cfg(), None)):
        assert lib.fg_paged_step_adjust(m.handle, pcs[0]._h, 1, i32(0), i32(1), i32(1), c, None, None, nx) == -1
    assert pcs[0].len(0) == n
    for pc in pcs:
        pc.close()


@pytest.mark.parametrize("kind", sorted(Q.TYPES))
def test_a_served_run(setup, kind):
    """All of it as a server has it: an 8-bit cache, forks of one prompt that draw
    under penalties and a mask, ends and new forks among them, a compaction. Every
    step's ids are the definition's on its logits, and a sample of the sequences'
    logits the float64 model's on their own ids."""
    d, m, ex = setup
    ex = exact_of(ex, kind)
    pc = m.paged(600, 16, 256, type=Q.TYPES[kind], prefix=True)
    prompt = uniform_ids(3, 320, d.vocab)
    pc.step({0: prompt}, want_logits=False)
    rng = np.random.default_rng(6)
    text = {s: list(prompt) for s in range(250)}
    for s in range(1, 250):
        pc.fork(0, s)
    banned = rng.random(d.vocab) < 0.3
    last = {s: 5 + s for s in range(250)}
    for k in range(6):
        if k == 3:
            for s in (1, 4, 5, 130):
                pc.trim(s)
                del text[s], last[s]
            pc.compact()
            pc.fork(0, 251, 320)
            text[251], last[251] = list(prompt), 9
        new = {s: [last[s]] for s in text}
        for s in new:
            text[s] += new[s]
        u = rng.random(len(new)).astype(np.float32)
        alone = 2 * (d.head_dim + 4) * d.n_kv_head * d.n_layer * sum(len(t) for t in text.values())
        (lg, ids), once = taken(m, pc, lambda: pc.step(
            new, u=u, temp=0.9, top_p=0.95, history=list(text.values()), count_from=320, pres=0.5, freq=0.1, rep=1.1,
            allowed=[~banned] * len(new)), 0.5 * alone)
        assert once
        mask = np.packbits(~banned, bitorder="little").view(np.uint32)[None]
        full = lambda v: np.full(len(new), v, np.float32)  # noqa: E731
        adj = TA.reference(lg, hist=[np.asarray(t) for t in text.values()], count_from=np.full(len(new), 320),
                           rep=full(1.1), pres=full(0.5), freq=full(0.1), mask=mask, mask_row=np.zeros(len(new), int))
        for i, s in enumerate(new):
            if s % 40 == 0 or s in (251, 6):
                assert relerr(lg[i], ex.logits(np.asarray(text[s]))[0][-1]) < BARS[kind], (k, s)
            assert ids[i] == R.draw_row(adj[i], float(np.float32(0.9)), 0, float(np.float32(0.95)), 0.0, float(u[i]))[0]
            assert not banned[ids[i]]
            last[s] = int(ids[i])
    pc.close()


def test_cache_types_refused(setup):
    d, m, _ = setup
    lib = engine.load_library()
    out = engine.C.c_void_p()
    for flags in (3, 5, 6, 7, 16, 32, -1):
        assert lib.fg_paged_create(m.handle, 4, 16, 1, flags, 0, 0, engine.C.byref(out)) == -1
    for flags in (0, 1, 2, 4, 8, 9, 10, 12):
        assert lib.fg_paged_create(m.handle, 4, 16, 1, flags, 0, 0, engine.C.byref(out)) == 0
        assert lib.fg_paged_destroy(out) == 0
    assert lib.fg_kv_create_ex(m.handle, 1, 16, engine.FG_KV_I8, engine.C.byref(out)) == -1
