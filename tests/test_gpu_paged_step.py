"""fg_paged_step: a model's passes over ragged batches on its paged cache,
against a float64 form of the model and the contiguous cache's passes.

Bars: logits within 5e-5 x max|logit| of the float64 model on an fp32 cache
(the linears carry ~16 bits of an activation, which the engine's other passes
show as 5e-6); on a bf16 cache within 2e-3 (K and V rounded to 8 bits)."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from autoresearch_amd import engine
from autoresearch_amd.weights import Dims, rope_tables, seeded_weights, uniform_ids

from . import paged_ref as R

pytestmark = pytest.mark.gpu

GQA = Dims(n_layer=2, d_model=640, n_head=5, n_kv_head=1, head_dim=128, vocab=1024)
MHA64 = Dims(n_layer=3, d_model=256, n_head=4, n_kv_head=4, head_dim=64, vocab=512)
MAX = 400


class Exact:
    """The model in float64, a sequence from scratch, with an optional window."""

    def __init__(self, d, seed):
        self.d = d
        w = seeded_weights(d, seed)
        t = lambda n, *s: torch.from_numpy(np.asarray(w[n], np.float64)).reshape(*s)  # noqa: E731
        L, D, qd, kd, V = d.n_layer, d.d_model, d.n_head * d.head_dim, d.n_kv_head * d.head_dim, d.vocab
        self.w = dict(wte=t("wte", V, D), lm=t("lm_head", V, D), q=t("c_q", L, qd, D), k=t("c_k", L, kd, D),
                      v=t("c_v", L, kd, D), p=t("c_proj", L, D, qd), f=t("c_fc", L, 4 * D, D),
                      g=t("c_proj2", L, D, 4 * D))
        c, s = rope_tables(MAX, d.head_dim)
        self.c, self.s = (torch.from_numpy(np.asarray(a, np.float64).reshape(MAX, 1, -1)) for a in (c, s))

    def norm(self, x):
        return x / torch.sqrt((x * x).mean(-1, keepdim=True) + self.d.eps)

    def rot(self, x):
        n, h = x.shape[0], x.shape[-1] // 2
        c, s = self.c[:n], self.s[:n]
        a, b = x[..., :h], x[..., h:]
        return torch.cat([a * c + b * s, b * c - a * s], -1)

    def logits(self, ids, window=0, sinks=0, bf16=False):
        """[len, V] logits and the layers' rotated keys and values."""
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
            k = self.rot((y @ w["k"][l].T).view(n, KH, hd))
            v = (y @ w["v"][l].T).view(n, KH, hd)
            if bf16:
                k, v = k.bfloat16().double(), v.bfloat16().double()
            kvs.append((k.reshape(n, -1).numpy(), v.reshape(n, -1).numpy()))
            k, v = (t.repeat_interleave(H // KH, 1) for t in (k, v))
            sc = torch.einsum("nhd,mhd->hnm", q, k) / math.sqrt(hd)
            a = torch.softmax(sc.masked_fill(~seen, -math.inf), -1)
            x = x + torch.einsum("hnm,mhd->nhd", a, v).reshape(n, -1) @ w["p"][l].T
            h = (self.norm(x) @ w["f"][l].T).clamp(min=0)
            x = x + (h * h) @ w["g"][l].T
        return (self.norm(x) @ w["lm"].T).numpy(), kvs


@pytest.fixture(scope="module", params=["gqa", "mha64"])
def setup(request):
    d = {"gqa": GQA, "mha64": MHA64}[request.param]
    m = engine.Model(d, stacks=seeded_weights(d, 5))
    c, s = rope_tables(MAX, d.head_dim)
    m.set_rope(c.reshape(-1), s.reshape(-1))
    yield d, m, Exact(d, 5)
    m.close()


def relerr(a, b):
    return float(np.abs(np.asarray(a, np.float64) - b).max() / np.abs(b).max())


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3)], ids=["all", "window"])
def test_ragged_passes(setup, bf16, window, sinks):
    """Prompts of several lengths, chunks beside single tokens, one token, many
    rows and few (each linear's path), sequences that end and start."""
    d, m, ex = setup
    bar = 2e-3 if bf16 else 5e-5
    pc = m.paged(80, 16, 12, bf16=bf16, window=window, sinks=sinks)
    text = {s: uniform_ids(100 + s, MAX, d.vocab) for s in range(12)}
    at = {s: 0 for s in range(12)}

    def step(counts):
        lg, nxt = pc.step({s: text[s][at[s]:at[s] + n] for s, n in counts.items()})
        for i, (s, n) in enumerate(counts.items()):
            at[s] += n
            assert pc.len(s) == at[s]
            want, _ = ex.logits(text[s][:at[s]], window, sinks, bf16)
            assert relerr(lg[i], want[-1]) < bar, (s, at[s], relerr(lg[i], want[-1]))
            assert nxt[i] == int(lg[i].argmax())

    step({3: 1})
    step({3: 1, 0: 1, 7: 1})
    step({1: 37, 3: 1, 2: 16, 0: 3})
    step({5: 150, 6: 200, 1: 1, 7: 5})
    step({s: 1 for s in (7, 6, 5, 3, 2, 1, 0)})
    pc.trim(5)
    at[5] = 0
    text[5] = uniform_ids(300, MAX, d.vocab)
    step({5: 33, 6: 2, 11: 1})
    pc.compact()
    step({6: 1, 5: 1, 11: 40, 0: 1})
    for s in (0, 6):
        k, v = pc.read(s)
        _, kvs = ex.logits(text[s][:at[s]], window, sinks, bf16)
        lost = (k[0] == 0).all(-1)
        # (a row a later token could see is there)
        assert window or not lost.any()
        for l in range(d.n_layer):
            for got, want in zip((k[l], v[l]), kvs[l]):
                tol = (2.0 ** -7 if bf16 else 1e-4) * np.abs(want).max()
                assert np.abs(got - want)[~lost].max() <= tol
        if window:
            assert not lost[:sinks].any() and not lost[max(0, at[s] - window + 1):].any()
    if window:  # pages behind the window are free again
        assert pc.free >= 80 - 9 * (window // 16 + 4)
    for s in range(12):
        pc.trim(s)
    assert pc.free == 80
    pc.close()


def test_forks(setup):
    """Sequences that share a prompt, and the page it ends in, go on apart."""
    d, m, ex = setup
    pc = m.paged(40, 32, 6)
    prompt = uniform_ids(1, 70, d.vocab)
    pc.step({0: prompt}, want_logits=False)
    for s, n in ((1, 70), (2, 70), (3, 41), (4, 64)):
        pc.fork(0, s, n)
    assert pc.free == 40 - 3
    text = {0: prompt, 1: prompt, 2: prompt, 3: prompt[:41], 4: prompt[:64]}
    for k in range(3):
        new = {s: uniform_ids(10 * k + s, 1 + (s + k) % 3, d.vocab) for s in range(5)}
        lg, _ = pc.step(new)
        for i, s in enumerate(new):
            text[s] = np.concatenate([text[s], new[s]])
            want, _ = ex.logits(text[s])
            assert relerr(lg[i], want[-1]) < 5e-5, (k, s)
    used = 40 - pc.free
    assert used == 2 + 3 + 1 + 1 + 0  # two shared pages, the third of 0, 1, 2, the second of 3, 4's third
    pc.close()


def test_rolled_back_tokens_are_gone(setup):
    d, m, ex = setup
    pc = m.paged(10, 16, 2)
    a, b = uniform_ids(1, 40, d.vocab), uniform_ids(2, 9, d.vocab)
    pc.step({0: a}, want_logits=False)
    pc.trim(0, 30)
    lg, _ = pc.step({0: b})
    want, _ = ex.logits(np.concatenate([a[:30], b]))
    assert relerr(lg[0], want[-1]) < 5e-5
    pc.close()


def test_greedy_and_drawn_ids(setup):
    """Greedy ids against the contiguous cache's loop; drawn ones are the draw's
    definition on the logits that came back."""
    d, m, _ = setup
    prompts = [uniform_ids(40 + s, 20 + 7 * s, d.vocab) for s in range(3)]
    pc = m.paged(30, 16, 3, bf16=False)
    lg, nxt = pc.step(dict(enumerate(prompts)))
    got, margins = [nxt], [np.sort(lg, -1)[:, -1] - np.sort(lg, -1)[:, -2]]
    for _ in range(12):
        lg, nxt = pc.step({s: [nxt[s]] for s in range(3)})
        got.append(nxt)
        margins.append(np.sort(lg, -1)[:, -1] - np.sort(lg, -1)[:, -2])
    got, margins = np.stack(got, 1), np.stack(margins, 1)
    for s in range(3):
        kv = m.kv(1, MAX)
        kv.step_multi(prompts[s][None, :-1], want_logits=False)
        ids, _ = kv.decode_greedy(prompts[s][-1:], 13)
        kv.close()
        diff = np.flatnonzero(ids[:, 0] != got[s])
        assert diff.size == 0 or margins[s, diff[0]] < 1e-4 * np.abs(lg).max()
    rng = np.random.default_rng(3)
    for k in range(6):
        temp = rng.uniform(0.5, 1.5, 3).astype(np.float32)
        u = rng.random(3).astype(np.float32)
        lg, nxt = pc.step({s: [k + s] for s in range(3)}, u=u, temp=temp, top_k=[5, 0, 100], top_p=0.9)
        for s in range(3):
            want = R.draw_row(lg[s], float(temp[s]), [5, 0, 100][s], float(np.float32(0.9)), 0.0, float(u[s]))
            assert nxt[s] == want[0]
    pc.close()


def test_refusals(setup):
    d, m, ex = setup
    pc = m.paged(6, 16, 4)
    a = uniform_ids(1, 60, d.vocab)
    pc.step({0: a[:60]}, want_logits=False)

    def code(f):
        with pytest.raises(engine.FgptError) as e:
            f()
        return e.value.code

    # 4 pages held; 2 free: three more sequences do not fit, and nothing happens
    assert code(lambda: pc.step({1: a[:1], 2: a[:1], 3: a[:1]})) == -5
    assert [pc.len(s) for s in range(4)] == [60, 0, 0, 0] and pc.free == 2
    lib = engine.load_library()
    i32 = lambda *v: (C.c_int32 * len(v))(*v)  # noqa: E731
    call = lambda n, s, c, i, dr=None, nx=None: lib.fg_paged_step(m.handle, pc._h, n, s, c, i, dr, None, nx)  # noqa: E731
    assert call(2, i32(1, 1), i32(1, 1), i32(1, 2)) == -1      # named twice
    assert call(1, i32(4), i32(1), i32(1)) == -1               # no such sequence
    assert call(1, i32(-1), i32(1), i32(1)) == -1
    assert call(1, i32(1), i32(0), i32(1)) == -1               # no token
    assert call(0, i32(1), i32(1), i32(1)) == -1
    assert call(1, i32(1), i32(1), i32(d.vocab)) == -1         # no such id
    assert call(1, None, i32(1), i32(1)) == -1
    assert call(1, i32(1), i32(1), i32(1), engine._DrawCfg(), i32(0)) == -1  # a draw without u
    assert code(lambda: pc.fork(0, 0)) == -1 and code(lambda: pc.trim(0, 61)) == -1
    assert code(lambda: m.paged(6, 16, 4, window=-1)) == -1 and code(lambda: m.paged(6, 17, 4)) == -1
    with pytest.raises(ValueError):
        pc.step({0: [1]}, temp=0.5)
    big = m.paged(60, 16, 1)
    assert code(lambda: big.step({0: uniform_ids(1, MAX + 1, d.vocab)})) == -6  # RoPE rows
    assert big.len(0) == 0
    big.close()
    lg, _ = pc.step({0: a[:3]})  # the sequence went through all of that unchanged
    assert relerr(lg[0], ex.logits(np.concatenate([a, a[:3]]))[0][-1]) < 5e-5
    # its last page is full now but shared: two holders that go on need one copy
    pc.trim(0, 20)
    pc.fork(0, 1)
    assert pc.free == 4
    pc.step({0: a[:1], 1: a[:1]})
    assert pc.free == 3
    pc.close()


def hip_error_pending():
    """Leaves an error behind as a failed HIP call of this thread does: the
    engine's next check after a launch then finds one (the launch itself runs)."""
    assert engine.load_library().hipSetDevice(1 << 20) != 0


def test_a_failed_compaction_moves_nothing(setup):
    """The sequences name the new pages only after the copies have succeeded."""
    d, m, ex = setup
    pc = m.paged(20, 16, 3)
    a, b = uniform_ids(1, 60, d.vocab), uniform_ids(2, 75, d.vocab)
    pc.step({0: a}, want_logits=False)
    pc.step({1: b}, want_logits=False)
    pc.trim(0)
    before = pc.read(1)
    hip_error_pending()
    with pytest.raises(engine.FgptError) as e:
        pc.compact()
    assert e.value.code == -4 and pc.len(1) == 75 and pc.free == 20 - 5
    for x, y in zip(before, pc.read(1)):
        assert np.array_equal(x, y)
    pc.step({2: a[:50]}, want_logits=False)  # (into the pages that the copies wrote to)
    for x, y in zip(before, pc.read(1)):
        assert np.array_equal(x, y)
    pc.trim(2)
    assert pc.compact() == 4
    lg, _ = pc.step({1: a[:2]})
    assert relerr(lg[0], ex.logits(np.concatenate([b, a[:2]]))[0][-1]) < 5e-5
    pc.close()


def test_a_step_whose_page_copies_fail_changes_nothing(setup):
    """Forks that go on from one partly filled page share it as before."""
    d, m, ex = setup
    pc = m.paged(20, 16, 4)
    a = uniform_ids(1, 70, d.vocab)
    pc.step({0: a}, want_logits=False)
    pc.fork(0, 1, 70)
    pc.fork(0, 2, 67)
    before, free = [pc.read(s) for s in range(3)], pc.free
    for _ in range(2):
        hip_error_pending()
        with pytest.raises(engine.FgptError) as e:
            pc.step({0: a[:2], 1: a[:20], 2: a[:1]})
        assert e.value.code == -4 and [pc.len(s) for s in range(4)] == [70, 70, 67, 0] and pc.free == free
    pc.step({3: a[:free * 16]}, want_logits=False)  # (into the pages that were given out and back)
    for s in range(3):
        for x, y in zip(before[s], pc.read(s)):
            assert np.array_equal(x, y)
    pc.trim(3)
    lg, _ = pc.step({0: a[:2], 1: a[:20], 2: a[:1]})
    for s, (n, k) in enumerate(((70, 2), (70, 20), (67, 1))):
        assert relerr(lg[s], ex.logits(np.concatenate([a[:n], a[:k]]))[0][-1]) < 5e-5
    for s in range(3):
        pc.trim(s)
    assert pc.free == 20
    pc.close()


@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3), (64, 70), (1, 0), (399, 4)])
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_timed_attention_counts_what_its_rows_see(setup, window, sinks, bf16):
    """fg_timing's operations and bytes of the attention: pairs of a query and a
    key that it sees, and each visible key and value once."""
    d, m, _ = setup
    pc = m.paged(80, 16, 4, bf16=bf16, window=window, sinks=sinks)

    def seen(T, n):
        p, j = np.arange(T - n, T)[:, None], np.arange(T)[None, :]
        return (j <= p) & ((j > p - window) | (j < sinks) if window else True)

    lens = {}
    for counts in ({0: 150, 1: 3, 2: 64}, {0: 1, 1: 1, 2: 1}, {1: 90, 0: 2, 3: 20}):
        m.timing(True)
        pc.step({s: uniform_ids(s, n, d.vocab) for s, n in counts.items()}, want_logits=False)
        got = m.timing_read()
        m.timing(False)
        for s, n in counts.items():
            lens[s] = lens.get(s, 0) + n
        rows, cut = sum(counts.values()), sum(counts.values()) > len(counts)
        want = {"attn_chunk": [0, 0.0, 0.0], "attn_decode": [0, 0.0, 0.0]}
        for layer in range(d.n_layer):
            last = cut and layer == d.n_layer - 1
            see = [seen(lens[s], 1 if last else n) for s, n in counts.items()]
            w = want["attn_chunk" if cut and not last else "attn_decode"]
            w[0] += 1
            w[1] += 4.0 * d.head_dim * d.n_head * sum(int(x.sum()) for x in see)
            w[2] += 8.0 * (len(counts) if last else rows) * d.n_head * d.head_dim \
                + 2 * (2 if bf16 else 4) * d.n_kv_head * d.head_dim * sum(int(x.any(0).sum()) for x in see)
        for kind, w in want.items():
            assert (got[kind][0], got[kind][2], got[kind][3]) == tuple(w), kind
    pc.close()


def test_a_model_that_is_closed_first():
    """Its caches go with it; closing them afterwards, or calling them, is no fault."""
    m = engine.Model(MHA64, stacks=seeded_weights(MHA64, 5))
    c, s = rope_tables(MAX, MHA64.head_dim)
    m.set_rope(c.reshape(-1), s.reshape(-1))
    pc, kv = m.paged(10, 16, 2), m.kv(1, 64)
    pc.step({0: [1, 2]})
    m.close()
    for call in (lambda: pc.step({0: [3]}), lambda: pc.len(0), pc.compact, lambda: kv.len):
        with pytest.raises(engine.FgptError) as e:
            call()
        assert e.value.code == -1
    pc.close()
    kv.close()
    m.close()
