"""The paged cache's operators as cases that a timing program can run and check.

Four kinds of call, each through autoresearch_amd.engine where `own` is set
and in elementary torch operations where it is not:

  attn    attention of ragged new tokens over a paged KV cache (paged_attn):
          chunks and single tokens, grouped heads, sliding window with sinks
  append  heads normed and rotated, keys and values put into their pages
          (qk_append)
  copy    pages of every layer copied by a list, as fork and compaction do
          (pages_copy)
  draw    an id a row under temperature, top-k, top-p and min-p from given
          uniform numbers (draw_rows)

Shapes are those of the two models the repository serves (6 heads of 128 with
their own keys, 10 heads of 128 on 2 key heads, vocabulary 8192) and generic
ones of grouped heads and larger vocabularies.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-5
HEADS = {  # query heads, key heads, head dim
    "d12": (6, 6, 128),
    "gqa20": (10, 2, 128),
    "h64": (16, 4, 64),
    "g8": (32, 4, 128),
}


def listed():
    return [
        # chat: one sequence's next token on the default cache
        dict(name="attn_one", kind="attn", mix=1, heads="d12", q="f32", kv="f32", n=1, lo=300, hi=300,
             q_lo=1, q_hi=1, page=16, window=0, sinks=0),
        # batched serving: 64 sequences of about a thousand positions on the bf16 cache
        dict(name="attn_decode_64", kind="attn", mix=2, heads="d12", q="f32", kv="bf16", n=64, lo=700,
             hi=1300, q_lo=1, q_hi=1, page=64, window=0, sinks=0),
        # prompt chunks beside decoding sequences, long contexts, grouped heads, default cache
        dict(name="attn_mixed_gqa20", kind="attn", mix=3, heads="gqa20", q="f32", kv="f32", n=9, lo=1200,
             hi=3900, q_lo=1, q_hi=130, page=32, window=0, sinks=0),
        # whole prompts
        dict(name="attn_prefill", kind="attn", mix=4, heads="g8", q="bf16", kv="bf16", n=4, lo=1500,
             hi=4000, q_lo=1500, q_hi=4000, page=64, window=0, sinks=0),
        # endless streams: a window and the first tokens of a long history
        dict(name="attn_window_32", kind="attn", mix=5, heads="g8", q="bf16", kv="bf16", n=32, lo=6000,
             hi=16000, q_lo=1, q_hi=4, page=16, window=2048, sinks=4),
        # one decoding step's rows into the bf16 cache
        dict(name="append_64", kind="append", mix=6, heads="d12", q="f32", kv="bf16", n=64, lo=700,
             hi=1300, q_lo=1, q_hi=1, page=64, norm=False, weights=False),
        # whole prompts with weighted head norms
        dict(name="append_prefill", kind="append", mix=7, heads="g8", q="bf16", kv="bf16", n=6, lo=1000,
             hi=2600, q_lo=1000, q_hi=2600, page=32, norm=True, weights=True),
        # a fork's partly filled page in every layer
        dict(name="copy_fork", kind="copy", planes=24, page_bytes=16 * 6 * 128 * 4, pages=257, n=1),
        # a compaction
        dict(name="copy_compact", kind="copy", planes=40, page_bytes=32 * 2 * 128 * 4, pages=2000,
             n=701),
        # batched serving at the models' vocabulary
        dict(name="draw_64", kind="draw", rows=64, V=8192, ties=False, mode="all"),
        # the smallest draw, logits rounded to 8 bits (ties)
        dict(name="draw_one", kind="draw", rows=1, V=8192, ties=True, mode="all"),
        # a large vocabulary, nucleus only (a whole row's mass counts)
        dict(name="draw_wide", kind="draw", rows=48, V=131073, ties=False, mode="topp"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "attn", "append", "copy", "draw", "draw"])
    if kind in ("attn", "append"):
        q, kv = rng.choice([("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")])
        c = dict(kind=kind, heads=rng.choice(sorted(HEADS)), q=q, kv=kv,
                 page=rng.choice([16, 32, 64, 128, 256]), mix=rng.randint(100, 1 << 30))
        form = rng.choice(["one", "chunk", "prompt"])
        if form == "one":  # decoding
            c["n"] = _log_int(rng, 1, 64)
            c["hi"] = _log_int(rng, 1, 8000 if c["n"] <= 16 else 2000)
            c["q_lo"], c["q_hi"] = 1, rng.choice([1, 1, 1, 2, 5])
        elif form == "chunk":  # prompt chunks after a context
            c["n"] = _log_int(rng, 1, 12)
            c["hi"] = _log_int(rng, 200, 4000)
            c["q_hi"] = _log_int(rng, 1, 200)
            c["q_lo"] = rng.randint(1, c["q_hi"])
        else:
            c["n"] = rng.randint(1, 3)
            c["hi"] = c["q_hi"] = _log_int(rng, 6, 2500)
            c["q_lo"] = max(1, c["q_hi"] // 2)
        c["hi"] = max(c["hi"], c["q_hi"])
        c["lo"] = c["q_lo"] if form == "prompt" else max(1, c["hi"] // 2)
        if kind == "append":
            c["norm"] = rng.random() < 0.5
            c["weights"] = c["norm"] and rng.random() < 0.5
        else:
            c["window"] = rng.choice([0, 0, _log_int(rng, 1, 2000)])
            c["sinks"] = rng.choice([0, 1, 4, 70]) if c["window"] else 0
        return c
    if kind == "copy":
        planes = rng.choice([1, 2, 24, 40])
        page_bytes = rng.choice([16, 32, 64]) * rng.choice([64, 256, 768]) * rng.choice([2, 4])
        n = _log_int(rng, 1, max(1, min(600, int(1.5e9 / planes / page_bytes))))
        return dict(kind=kind, planes=planes, page_bytes=page_bytes,
                    pages=2 * n + rng.randint(1, 50), n=n)
    V = rng.choice([rng.randint(2, 500), 8192, 8192, _log_int(rng, 500, 120000)])
    return dict(kind=kind, rows=_log_int(rng, 1, 128 if V <= 16384 else 24), V=V,
                ties=rng.random() < 0.4, mode=rng.choice(["all", "topk", "topp", "minp", "plain"]))


# ------------------------------------------------------------------ inputs

def _type(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _lengths(case):
    """Positions after the append and new tokens of each sequence (host)."""
    r = np.random.default_rng(case["mix"])
    n = case["n"]
    kv = r.integers(case["lo"], case["hi"] + 1, n)
    q = np.minimum(r.integers(case["q_lo"], case["q_hi"] + 1, n), kv)
    if case["lo"] == case["q_lo"] and case["hi"] == case["q_hi"]:  # whole prompts
        q = kv
    return kv.astype(np.int32), q.astype(np.int32)


def _batch(case, seed):
    """The batch's device arrays: shuffled pages, as a cache in use has them."""
    kv, q = _lengths(case)
    P = case["page"]
    held = -(-kv // P)
    ld, total = int(held.max()), int(held.sum())
    n_pages = total + total // 8 + 1
    order = np.random.default_rng(seed).permutation(n_pages)[:total].astype(np.int32)
    table = np.full((len(kv), ld), -1, np.int32)
    table[np.arange(ld)[None, :] < held[:, None]] = order
    start = np.concatenate([[0], np.cumsum(q)]).astype(np.int32)
    return dict(case=case, n=len(kv), rows=int(start[-1]), max_q=int(q.max()), max_kv=int(kv.max()),
                n_pages=n_pages, ld=ld, start=torch.from_numpy(start).cuda(),
                kv_len=torch.from_numpy(kv).cuda(), table=torch.from_numpy(table).cuda())


def _rope(n, hd):
    """(n, hd/2) fp32 tables, as an app builds them."""
    theta = 10000.0 ** (-2.0 * np.arange(hd // 2) / hd)
    ang = np.arange(n)[:, None] * theta[None, :]
    return [torch.from_numpy(f(ang).astype(np.float32)).cuda() for f in (np.cos, np.sin)]


MODES = {"all": (1, 1, 1), "topk": (1, 0, 0), "topp": (0, 1, 0), "minp": (0, 0, 1), "plain": (0, 0, 0)}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * seed + 17)

    def normal(*shape, dtype=torch.float32, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(dtype)

    k = case["kind"]
    if k in ("attn", "append"):
        H, KH, hd = HEADS[case["heads"]]
        st = _batch(case, seed)
        qt, kt = _type(case["q"]), _type(case["kv"])
        pool = (st["n_pages"], KH, case["page"], hd)
        st["k"], st["v"] = normal(*pool, dtype=kt), normal(*pool, dtype=kt)
        if k == "attn":
            st["q"] = normal(st["rows"], H * hd, dtype=qt, std=1.5)
            st["out"] = torch.empty_like(st["q"])
        else:
            st["qkv"] = normal(st["rows"], (H + 2 * KH) * hd, dtype=qt, std=2.0)
            st["q"] = torch.empty(st["rows"], H * hd, dtype=qt, device="cuda")
            st["cos"], st["sin"] = _rope(st["max_kv"], hd)
            if case["weights"]:
                st["wq"], st["wk"] = 1 + normal(hd, std=0.1), 1 + normal(hd, std=0.1)
        return st
    if k == "copy":
        words = case["page_bytes"] // 2
        pool = torch.randint(-30000, 30000, (case["planes"], case["pages"], words), generator=g,
                             device="cuda", dtype=torch.int16)
        pick = np.random.default_rng(seed).permutation(case["pages"])[:2 * case["n"]].astype(np.int32)
        return dict(case=case, pool=pool, src=pick[:case["n"]].copy(), dst=pick[case["n"]:].copy())
    rows, V = case["rows"], case["V"]
    x = normal(rows, V, std=2.5)
    x += 4.0 * (torch.rand(rows, V, generator=g, device="cuda") < 4.0 / V)  # a few likely ids
    if case["ties"]:
        x = x.bfloat16().float()
    r = np.random.default_rng(seed + 5)
    tk, tp, mp = MODES[case["mode"]]
    f32 = lambda a: torch.from_numpy(np.asarray(a, np.float32)).cuda()  # noqa: E731
    return dict(case=case, x=x, temp=f32(r.uniform(0.5, 1.3, rows)),
                top_k=torch.from_numpy(r.integers(1, 200, rows).astype(np.int32)).cuda() if tk else None,
                top_p=f32(r.uniform(0.5, 0.99, rows)) if tp else None,
                min_p=f32(r.uniform(0.001, 0.1, rows)) if mp else None,
                u=f32(r.integers(0, 1 << 24, rows) / float(1 << 24)),
                ids=torch.empty(rows, dtype=torch.int32, device="cuda"),
                probs=torch.empty(rows, dtype=torch.float32, device="cuda"))


# ------------------------------------------------------------------ the framework's calls

def _own(st):
    from autoresearch_amd import engine
    case = st["case"]
    stream = torch.cuda.current_stream().cuda_stream
    if case["kind"] == "copy":
        pool = st["pool"]
        engine.pages_copy(pool.data_ptr(), case["planes"], pool.stride(0) * 2, case["pages"],
                          case["page_bytes"], st["src"], st["dst"], stream)
        return pool
    if case["kind"] == "draw":
        ptr = lambda n: 0 if st[n] is None else st[n].data_ptr()  # noqa: E731
        rows, V = case["rows"], case["V"]
        if "work" not in st:
            st["work"] = torch.empty(engine.draw_rows_work(rows, V), dtype=torch.uint8, device="cuda")
        engine.draw_rows(st["x"].data_ptr(), rows, V, V, st["u"].data_ptr(), st["ids"].data_ptr(),
                         st["probs"].data_ptr(), temp=ptr("temp"), top_k=ptr("top_k"),
                         top_p=ptr("top_p"), min_p=ptr("min_p"), work=st["work"].data_ptr(),
                         work_bytes=st["work"].numel(), stream=stream)
        return st["ids"], st["probs"]
    H, KH, hd = HEADS[case["heads"]]
    pages = engine.pages(st["k"].data_ptr(), st["v"].data_ptr(), st["n_pages"], case["page"], KH, hd,
                         bf16=case["kv"] == "bf16")
    batch = engine.ragged(st["start"].data_ptr(), st["kv_len"].data_ptr(), st["table"].data_ptr(),
                          st["n"], st["rows"], st["max_q"], st["max_kv"], st["ld"])
    if case["kind"] == "append":
        w = case["weights"]
        cfg = engine.append_cfg(H, st["cos"].data_ptr(), st["sin"].data_ptr(), st["max_kv"],
                                norm=case["norm"], eps=EPS, wq=st["wq"].data_ptr() if w else 0,
                                wk=st["wk"].data_ptr() if w else 0, bf16=case["q"] == "bf16")
        engine.qk_append(pages, batch, cfg, st["qkv"].data_ptr(), st["q"].data_ptr(), stream)
        return st["q"], st["k"], st["v"]
    cfg = engine.attn_cfg(H, window=case["window"], sinks=case["sinks"], bf16=case["q"] == "bf16")
    if "work" not in st:
        st["work"] = torch.empty(engine.paged_attn_work(pages, batch, cfg), dtype=torch.uint8,
                                 device="cuda")
    engine.paged_attn(pages, batch, cfg, st["q"].data_ptr(), st["out"].data_ptr(),
                      st["work"].data_ptr(), st["work"].numel(), stream)
    return st["out"]


# ------------------------------------------------------------------ the plain form

def _rows_of(st):
    """Sequence and position of every row."""
    at = torch.arange(st["rows"], device="cuda", dtype=torch.int32)
    seq = torch.bucketize(at, st["start"][1:], right=True)
    return seq, st["kv_len"][seq] - st["start"][seq + 1] + at


def _head_norm(x, w):
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x if w is None else x * w


def _rotate(x, c, s):
    a, b = x.chunk(2, -1)
    return torch.cat([a * c + b * s, b * c - a * s], -1)


def _append(st, real):
    """Rotated q, k and v of every row in the type `real`, unrounded."""
    case = st["case"]
    H, KH, hd = HEADS[case["heads"]]
    q, k, v = st["qkv"].to(real).view(st["rows"], -1, hd).split([H, KH, KH], 1)
    if case["norm"]:
        q = _head_norm(q, st["wq"].to(real) if case["weights"] else None)
        k = _head_norm(k, st["wk"].to(real) if case["weights"] else None)
    seq, pos = _rows_of(st)
    c, s = (t[pos][:, None, :].to(real) for t in (st["cos"], st["sin"]))
    page = st["table"][seq, pos // case["page"]]
    return _rotate(q, c, s).reshape(st["rows"], -1), _rotate(k, c, s), v, page, pos % case["page"]


def _plain_attn(st):
    case = st["case"]
    H, KH, hd = HEADS[case["heads"]]
    n, Q, T, G = st["n"], st["max_q"], st["max_kv"], H // KH
    pages = st["table"].clamp(min=0)
    K, V = (t[pages].float().transpose(1, 2).reshape(n, KH, -1, hd)[:, :, :T] for t in (st["k"], st["v"]))
    seq, pos = _rows_of(st)
    slot = torch.arange(st["rows"], device="cuda") - st["start"][seq]
    q = torch.zeros(n, Q, KH, G, hd, device="cuda")
    q[seq, slot] = st["q"].float().view(-1, KH, G, hd)
    where = torch.full((n, Q), -1, device="cuda", dtype=pos.dtype)
    where[seq, slot] = pos
    s = q.permute(0, 2, 3, 1, 4).reshape(n, KH, G * Q, hd) @ K.transpose(2, 3).contiguous()
    s = s.view(n, KH, G, Q, T) * (1.0 / math.sqrt(hd))
    j = torch.arange(T, device="cuda")
    at = where[:, :, None]
    seen = j <= at
    if case["window"]:
        seen &= (j > at - case["window"]) | (j < case["sinks"])
    s = s.masked_fill_(~seen[:, None, None], -1e30)
    s = (s - s.amax(-1, keepdim=True)).exp_()
    total = s.sum(-1, keepdim=True)
    o = s.view(n, KH, G * Q, T) @ V
    o = (o.view(n, KH, G, Q, hd) / total).permute(0, 3, 1, 2, 4)
    return o[seq, slot].reshape(st["rows"], H * hd).to(st["q"].dtype)


def _plain_draw(st):
    x, V = st["x"].double(), st["case"]["V"]
    x, order = x.sort(dim=-1, descending=True, stable=True)
    e = ((x - x[:, :1]) / st["temp"].double()[:, None]).exp()
    keep = torch.ones_like(e, dtype=torch.bool)
    if st["top_k"] is not None:
        keep &= torch.arange(V, device="cuda") < st["top_k"][:, None]
    if st["top_p"] is not None:
        w = e * keep
        c = w.cumsum(-1)
        keep &= (c - w) < st["top_p"].double()[:, None] * c[:, -1:]
    if st["min_p"] is not None:
        keep &= e >= st["min_p"].double()[:, None]
    w = torch.zeros_like(e).scatter_(1, order, e * keep)
    c = w.cumsum(-1)
    ids = (c <= st["u"].double()[:, None] * c[:, -1:]).sum(-1)
    return ids.int(), (w.gather(1, ids[:, None]) / c[:, -1:])[:, 0].float()


@torch.no_grad()
def run(st):
    if own:
        return _own(st)
    k = st["case"]["kind"]
    if k == "attn":
        return _plain_attn(st)
    if k == "draw":
        return _plain_draw(st)
    if k == "copy":
        pool = st["pool"]
        src, dst = (torch.from_numpy(st[n]).long().cuda() for n in ("src", "dst"))
        pool[:, dst] = pool[:, src]
        return pool
    q, key, v, page, slot = _append(st, torch.float32)
    st["k"][page, :, slot] = key.to(st["k"].dtype)
    st["v"][page, :, slot] = v.to(st["v"].dtype)
    return q.to(st["q"].dtype), st["k"], st["v"]


# ------------------------------------------------------------------ what a call cannot do without

def _seen(case, kv, q):
    """(query, key) pairs and distinct visible keys of a sequence (averages over the ranges)."""
    w, s = case["window"], case["sinks"]
    if not w:
        return q * (kv - q) + q * (q + 1) / 2, kv
    pos = np.arange(int(kv - q), int(kv))
    first = np.maximum(0, pos - w + 1)
    pairs = (pos + 1 - first + np.minimum(first, s)).sum()
    lo = max(0, int(kv - q) - w + 1)
    return float(pairs), kv - lo + min(lo, s)


def work(case):
    k = case["kind"]
    if k == "copy":
        return {"bytes": 2.0 * case["planes"] * case["page_bytes"] * case["n"], "flops": 0.0}
    if k == "draw":
        return {"bytes": case["rows"] * (4.0 * case["V"] + 28), "flops": 4.0 * case["rows"] * case["V"]}
    H, KH, hd = HEADS[case["heads"]]
    eq, ek = (2 if case[n] == "bf16" else 4 for n in ("q", "kv"))
    kv, q = (a.astype(np.float64) for a in _lengths(case))
    rows = q.sum()
    if k == "append":
        by = rows * hd * ((2 * H + 2 * KH) * eq + 2 * KH * ek) + kv.max() * hd * 4
        return {"bytes": float(by), "flops": float(rows * hd * 8 * (H + KH))}
    seen = [_seen(case, a, b) for a, b in zip(kv, q)]
    pairs, keys = sum(a for a, _ in seen), sum(b for _, b in seen)
    return {"bytes": float(2 * rows * H * hd * eq + 2 * keys * KH * hd * ek),
            "flops": float(4.0 * hd * H * pairs)}


# ------------------------------------------------------------------ 64 bits

def _exact_attn(st):
    case = st["case"]
    H, KH, hd = HEADS[case["heads"]]
    G, P = H // KH, case["page"]
    start, lens, table = (st[n].cpu().numpy() for n in ("start", "kv_len", "table"))
    out = torch.zeros(st["rows"], H, hd, device="cuda", dtype=torch.float64)
    for b in range(st["n"]):
        a, z, T = int(start[b]), int(start[b + 1]), int(lens[b])
        pages = torch.from_numpy(table[b, :-(-T // P)].astype(np.int64)).cuda()
        p = torch.arange(T - (z - a), T, device="cuda")[:, None]
        j = torch.arange(T, device="cuda")[None, :]
        hidden = j > p
        if case["window"]:
            hidden = hidden | ((j <= p - case["window"]) & (j >= case["sinks"]))
        for h in range(H):
            K = st["k"][pages, h // G].reshape(-1, hd)[:T].double()
            V = st["v"][pages, h // G].reshape(-1, hd)[:T].double()
            q = st["q"][a:z, h * hd:(h + 1) * hd].double()
            for r in range(0, z - a, 1024):
                s = (q[r:r + 1024] @ K.t().contiguous()) / math.sqrt(hd)
                s = s.masked_fill(hidden[r:r + 1024], -math.inf)
                out[a + r:a + r + s.shape[0], h] = torch.softmax(s, -1) @ V
    return out.reshape(st["rows"], H * hd)


def _exact_draw(st):
    """Row by row on the host, from the definition."""
    x = st["x"].cpu().numpy().astype(np.float64)
    get = lambda n: None if st[n] is None else st[n].cpu().numpy()  # noqa: E731
    temp, top_k, top_p, min_p, u = (get(n) for n in ("temp", "top_k", "top_p", "min_p", "u"))
    ids, probs = [], []
    for r in range(len(x)):
        e = np.exp((x[r] - x[r].max()) / float(temp[r]))
        order = np.argsort(-x[r], kind="stable")
        if top_k is not None:
            order = order[:top_k[r]]
        if top_p is not None:
            c = np.cumsum(e[order])
            before = np.concatenate([[0.0], c[:-1]])
            order = order[before < float(top_p[r]) * c[-1]]
        if min_p is not None:
            order = order[e[order] >= float(min_p[r])]
        kept = np.sort(order)
        c = np.cumsum(e[kept])
        at = min(int(np.searchsorted(c, float(u[r]) * c[-1], side="right")), len(kept) - 1)
        ids.append(kept[at])
        probs.append(e[kept[at]] / c[-1])
    return np.asarray(ids, np.int32), np.asarray(probs, np.float64)


@torch.no_grad()
def exact(case, seed):
    st = prepare(case, seed)
    k = case["kind"]
    if k == "attn":
        return _exact_attn(st)
    if k == "draw":
        return _exact_draw(st)
    if k == "copy":
        want = st["pool"].cpu().numpy()
        want[:, st["dst"]] = want[:, st["src"]]
        return want
    H, KH, hd = HEADS[case["heads"]]
    x = st["qkv"].double().reshape(st["rows"], H + 2 * KH, hd)
    start, lens, table = (st[n].cpu().numpy() for n in ("start", "kv_len", "table"))
    q = torch.empty(st["rows"], H * hd, device="cuda", dtype=torch.float64)
    pools = [st["k"].double(), st["v"].double()]
    h2 = hd // 2
    for b in range(st["n"]):
        a, z, T = int(start[b]), int(start[b + 1]), int(lens[b])
        pos = torch.arange(T - (z - a), T, device="cuda")
        page = torch.from_numpy(table[b].astype(np.int64)).cuda()[pos // case["page"]]
        c, s = st["cos"][pos].double()[:, None], st["sin"][pos].double()[:, None]
        y = x[a:z, :H + KH]
        if case["norm"]:
            y = y / ((y ** 2).sum(-1, keepdim=True) / hd + EPS).sqrt()
            if case["weights"]:
                y = torch.cat([y[:, :H] * st["wq"].double(), y[:, H:] * st["wk"].double()], 1)
        y = torch.cat([y[..., :h2] * c + y[..., h2:] * s, y[..., h2:] * c - y[..., :h2] * s], -1)
        q[a:z] = y[:, :H].reshape(z - a, -1)
        for pool, rows in zip(pools, (y[:, H:], x[a:z, H + KH:])):
            pool[page, :, pos % case["page"]] = rows
    return q, pools[0], pools[1]
