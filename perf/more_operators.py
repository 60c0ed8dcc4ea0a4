"""8-bit pages, shared prefixes and logit adjustments as cases that a timing program can run and check.

Five kinds of call, each through autoresearch_amd.engine where `own` is set and
in elementary torch operations where it is not:

  append  heads normed and rotated, keys and values quantised into 8-bit pages
          (qk_append), and the appended tokens read back (pages_read)
  read    keys and values of whole sequences read back from 8-bit pages
          (pages_read)
  attn    attention of ragged new tokens over 8-bit pages (paged_attn)
  prefix  the same for sequences that share the pages of their first positions
          (prefix_attn), on pages of any type
  adjust  penalties over each row's history, biases and grammar masks on a
          batch's logits (adjust_rows)

A page of an 8-bit type holds, per key head, page_size rows of head_dim codes
and then page_size fp32 scales; a value is its code times its row's scale.

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
TOP = {"i8": 127.0, "e4m3": 448.0}  # the largest code
TINY = 2.0 ** -126


def listed():
    return [
        # one decoding step's rows of a batch into the int8 cache
        dict(name="append_64", kind="append", mix=1, heads="d12", q="f32", kv="i8", n=64, lo=700, hi=1300,
             q_lo=1, q_hi=1, page=64, norm=False, weights=False),
        # whole prompts with weighted head norms into the e4m3 cache
        dict(name="append_prefill", kind="append", mix=2, heads="g8", q="bf16", kv="e4m3", n=6, lo=1000,
             hi=2600, q_lo=1000, q_hi=2600, page=32, norm=True, weights=True),
        # one chat read back, to go on in a cache of another type
        dict(name="read_one", kind="read", mix=3, heads="gqa20", q="f32", kv="i8", n=1, lo=777, hi=777,
             page=16),
        # long sequences of a batch handed over in bf16
        dict(name="read_long", kind="read", mix=4, heads="g8", q="bf16", kv="e4m3", n=12, lo=3000, hi=9000,
             page=64),
        # chat: one sequence's next token
        dict(name="attn_one", kind="attn", mix=5, heads="d12", q="f32", kv="i8", n=1, lo=300, hi=300, q_lo=1,
             q_hi=1, page=16, window=0, sinks=0),
        # batched serving: 64 sequences of about a thousand positions
        dict(name="attn_decode_64", kind="attn", mix=6, heads="d12", q="f32", kv="e4m3", n=64, lo=700,
             hi=1300, q_lo=1, q_hi=1, page=64, window=0, sinks=0),
        # whole prompts
        dict(name="attn_prefill", kind="attn", mix=7, heads="g8", q="bf16", kv="i8", n=4, lo=1500, hi=4000,
             q_lo=1500, q_hi=4000, page=64, window=0, sinks=0),
        # a few answers to one question side by side, on the default cache
        dict(name="prefix_4", kind="prefix", mix=8, heads="d12", q="f32", kv="f32", groups=1, n=4, shared=512,
             lo=20, hi=90, q_lo=1, q_hi=1, page=16, window=0, sinks=0),
        # 64 users of one long instruction, each some hundred tokens into an answer
        dict(name="prefix_64", kind="prefix", mix=9, heads="gqa20", q="f32", kv="bf16", groups=1, n=64,
             shared=3900, lo=50, hi=500, q_lo=1, q_hi=1, page=64, window=0, sinks=0),
        # three instructions, drafts and short questions of several tokens on the 8-bit cache
        dict(name="prefix_groups", kind="prefix", mix=10, heads="g8", q="bf16", kv="e4m3", groups=3, n=48,
             shared=6000, lo=40, hi=700, q_lo=1, q_hi=9, page=32, window=0, sinks=0),
        # one row of the models' vocabulary
        dict(name="adjust_one", kind="adjust", mix=11, rows=1, V=8192, hist=200, bias=20, masks=0),
        # a large vocabulary, long histories, grammars shared by the rows
        dict(name="adjust_wide", kind="adjust", mix=12, rows=48, V=131073, hist=4000, bias=300, masks=7),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "read", "attn", "attn", "attn", "prefix", "prefix", "prefix", "adjust",
                       "adjust"])
    mix = rng.randint(100, 1 << 30)
    if kind == "adjust":
        V = rng.choice([rng.randint(2, 500), 8192, _log_int(rng, 500, 131073)])
        return dict(kind=kind, mix=mix, rows=_log_int(rng, 1, 128 if V <= 16384 else 40), V=V,
                    hist=rng.choice([0, _log_int(rng, 1, 4000)]), bias=rng.choice([0, _log_int(rng, 1, 300)]),
                    masks=rng.choice([0, 1, 5]))
    c = dict(kind=kind, mix=mix, heads=rng.choice(sorted(HEADS)), q=rng.choice(["f32", "bf16"]),
             kv=rng.choice(["i8", "e4m3"]), page=rng.choice([16, 32, 64, 128, 256]))
    if kind == "read":
        c["n"] = _log_int(rng, 1, 24)
        c["hi"] = _log_int(rng, 1, 60000 // c["n"])
        c["lo"] = max(1, c["hi"] // 3)
        return c
    if kind == "prefix":
        c["kv"] = rng.choice(["f32", "bf16", "i8", "e4m3"])
        if c["kv"] == "f32":
            c["q"] = "f32"
        c["groups"] = rng.choice([1, 1, 2, 4])
        c["n"] = max(c["groups"], _log_int(rng, 2, 64))
        c["shared"] = _log_int(rng, 16, 4000)
        c["hi"] = _log_int(rng, 1, 800)
        c["q_lo"], c["q_hi"] = 1, min(c["hi"], rng.choice([1, 1, 1, 5, _log_int(rng, 1, 100 if c["n"] < 16 else 20)]))
    else:
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
        if form == "prompt":
            c["lo"] = c["q_lo"]
    c.setdefault("lo", max(1, c["hi"] // 2))
    if kind == "append":
        c["norm"] = rng.random() < 0.5
        c["weights"] = c["norm"] and rng.random() < 0.5
    else:
        c["window"] = rng.choice([0, 0, _log_int(rng, 1, 2000)])
        c["sinks"] = rng.choice([0, 1, 4, 70]) if c["window"] else 0
    return c


# ------------------------------------------------------------------ inputs

def _type(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _lengths(case):
    """Positions after the append, new tokens and shared positions of each sequence (host)."""
    r = np.random.default_rng(case["mix"])
    n = case["n"]
    kv = r.integers(case["lo"], case["hi"] + 1, n)
    if case["kind"] == "read":
        return kv.astype(np.int32), kv.astype(np.int32), None
    q = np.minimum(r.integers(case["q_lo"], case["q_hi"] + 1, n), kv)
    if case["lo"] == case["q_lo"] and case["hi"] == case["q_hi"]:  # whole prompts
        q = kv
    shared = None
    if case["kind"] == "prefix":  # groups of about equal size, their prefixes whole pages
        at = np.arange(n) * case["groups"] // n
        each = r.integers(max(1, case["shared"] // 2), case["shared"] + 1, case["groups"])
        each[0] = case["shared"]
        each = each // case["page"] * case["page"]
        shared = each[at].astype(np.int32)
        kv = kv + shared
    return kv.astype(np.int32), q.astype(np.int32), shared


def _batch(case, seed):
    """The batch's device arrays: shuffled pages, as a cache in use has them."""
    kv, q, shared = _lengths(case)
    P, n = case["page"], case["n"]
    held = -(-kv // P)
    common = np.zeros(n, np.int64) if shared is None else shared // P
    group = np.zeros(n, np.int64) if shared is None else np.arange(n) * case["groups"] // n
    first = np.r_[True, group[1:] != group[:-1]] if shared is not None else np.ones(n, bool)
    fresh = held - np.where(first, 0, common)  # pages that nobody before it holds
    ld, total = int(held.max()), int(fresh.sum())
    n_pages = total + total // 8 + 1
    order = np.random.default_rng(seed).permutation(n_pages)[:total].astype(np.int32)
    table = np.full((n, ld), -1, np.int32)
    table[np.arange(ld)[None, :] < fresh[:, None]] = order
    if shared is not None:
        for s in range(n):
            if not first[s]:
                own_pages = table[s, :fresh[s]].copy()
                table[s, :common[s]] = table[s - 1, :common[s]]
                table[s, common[s]:held[s]] = own_pages
    start = np.concatenate([[0], np.cumsum(q)]).astype(np.int32)
    put = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    st = dict(case=case, n=n, rows=int(start[-1]), max_q=int(q.max()), max_kv=int(kv.max()),
              n_pages=n_pages, ld=ld, start=put(start), kv_len=put(kv), table=put(table))
    if shared is not None:
        at = np.flatnonzero(first)
        st["seq_start"] = put(np.r_[at, n].astype(np.int32))
        st["shared"] = put(np.ascontiguousarray(shared[at]))
        st["n_group"], st["max_shared"] = len(at), int(shared.max())
    return st


def _rope(n, hd):
    """(n, hd/2) fp32 tables, as an app builds them."""
    theta = 10000.0 ** (-2.0 * np.arange(hd // 2) / hd)
    ang = np.arange(n)[:, None] * theta[None, :]
    return [torch.from_numpy(f(ang).astype(np.float32)).cuda() for f in (np.cos, np.sin)]


def _codes(x, kv):
    """(codes as bytes, scales) of fp32 rows: scale max|x| / top, codes rounded to nearest even."""
    s = x.abs().amax(-1, keepdim=True) / TOP[kv]
    s = torch.where(s < TINY, 0.0, s)
    y = (x * torch.where(s > 0, 1.0 / s, 0.0)).clamp(-TOP[kv], TOP[kv])
    y = y.round().to(torch.int8) if kv == "i8" else y.to(torch.float8_e4m3fn)
    return y.view(torch.uint8), s[..., 0]


def _views(pool, P, hd):
    """Codes [pages, heads, P, hd] and scales [pages, heads, P] within a pool of bytes."""
    codes = pool[..., :P * hd].unflatten(-1, (P, hd))
    return codes, pool[..., P * hd:].view(torch.float32)


def _values(codes, kv, real=torch.float32):
    return (codes.view(torch.int8) if kv == "i8" else codes.view(torch.float8_e4m3fn)).to(real)


def _pool(st, normal):
    """A plane of pages in use, of the case's type."""
    case = st["case"]
    _, KH, hd = HEADS[case["heads"]]
    P, kv = case["page"], case["kv"]
    if kv not in TOP:
        return normal(st["n_pages"], KH, P, hd, dtype=_type(kv))
    pool = torch.empty(st["n_pages"], KH, P * (hd + 4), dtype=torch.uint8, device="cuda")
    codes, scales = _views(pool, P, hd)
    c, s = _codes(normal(st["n_pages"], KH, P, hd), kv)
    codes.copy_(c)
    scales.copy_(s)
    return pool


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * seed + 17)

    def normal(*shape, dtype=torch.float32, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(dtype)

    if case["kind"] == "adjust":
        return _prepare_adjust(case, seed, normal)
    H, KH, hd = HEADS[case["heads"]]
    st = _batch(case, seed)
    qt, k = _type(case["q"]), case["kind"]
    st["k"], st["v"] = _pool(st, normal), _pool(st, normal)
    if k in ("append", "read"):
        rt = torch.bfloat16 if k == "append" else qt
        st["k_rows"] = torch.empty(st["rows"], KH * hd, dtype=rt, device="cuda")
        st["v_rows"] = torch.empty_like(st["k_rows"])
    if k == "append":
        st["qkv"] = normal(st["rows"], (H + 2 * KH) * hd, dtype=qt, std=2.0)
        st["q"] = torch.empty(st["rows"], H * hd, dtype=qt, device="cuda")
        st["cos"], st["sin"] = _rope(st["max_kv"], hd)
        if case["weights"]:
            st["wq"], st["wk"] = 1 + normal(hd, std=0.1), 1 + normal(hd, std=0.1)
    elif k != "read":
        st["q"] = normal(st["rows"], H * hd, dtype=qt, std=1.5)
        st["out"] = torch.empty_like(st["q"])
    return st


def _prepare_adjust(case, seed, normal):
    """Logits, histories that repeat their ids, biases (some ids named twice), masks of a grammar."""
    rows, V = case["rows"], case["V"]
    r = np.random.default_rng(seed + 5)
    put = lambda a, t: torch.from_numpy(np.asarray(a, t)).cuda()  # noqa: E731
    start = lambda n: np.concatenate([[0], np.cumsum(n)])  # noqa: E731
    n_hist = r.integers(case["hist"] // 2, case["hist"] + 1, rows)
    n_bias = r.integers(case["bias"] // 2, case["bias"] + 1, rows)
    hist = np.minimum((r.pareto(0.7, int(n_hist.sum())) * 3).astype(np.int64), V - 1)
    hist = (hist * 7919 + r.integers(0, 3, hist.size)) % V
    ids = r.integers(0, V, int(n_bias.sum()))
    st = dict(case=case, x=normal(rows, V, std=2.5), out=torch.empty(rows, V, device="cuda"),
              hist_start=put(start(n_hist), np.int32), hist=put(hist, np.int32),
              count_from=put((n_hist * r.uniform(0, 1, rows)).astype(np.int64), np.int32),
              rep=put(r.uniform(1.0, 1.4, rows), np.float32), pres=put(r.uniform(0, 0.8, rows), np.float32),
              freq=put(r.uniform(0, 0.5, rows), np.float32), bias_start=put(start(n_bias), np.int32),
              bias_id=put(ids, np.int32), bias=put(r.normal(0, 3, ids.size), np.float32))
    if case["masks"]:
        words = (V + 31) // 32
        st["mask"] = put(r.integers(0, 1 << 32, (case["masks"], words)).astype(np.uint32).view(np.int32), np.int32)
        st["mask"] |= st["mask"].roll(1, 1)
        st["mask_row"] = put(r.integers(-1, case["masks"], rows), np.int32)
    return st


# ------------------------------------------------------------------ the framework's calls

def _own(st):
    from autoresearch_amd import engine
    case = st["case"]
    k, stream = case["kind"], torch.cuda.current_stream().cuda_stream
    at = lambda n: st[n].data_ptr() if n in st else 0  # noqa: E731
    if k == "adjust":
        rows, V = case["rows"], case["V"]
        cfg = engine.adjust_cfg(hist=at("hist"), hist_start=at("hist_start"), n_hist=st["hist"].numel(),
                                count_from=at("count_from"), rep=at("rep"), pres=at("pres"), freq=at("freq"),
                                bias=at("bias"), bias_id=at("bias_id"), bias_start=at("bias_start"),
                                n_bias=st["bias"].numel(), mask=at("mask"), mask_row=at("mask_row"),
                                n_mask=case["masks"])
        engine.adjust_rows(at("x"), rows, V, V, cfg, at("out"), V, stream)
        return st["out"]
    H, KH, hd = HEADS[case["heads"]]
    kind = {"f32": engine.FG_F32, "bf16": engine.FG_BF16, "i8": engine.FG_I8, "e4m3": engine.FG_E4M3}
    pages = engine.pages(at("k"), at("v"), st["n_pages"], case["page"], KH, hd, type=kind[case["kv"]])
    batch = engine.ragged(at("start"), at("kv_len"), at("table"), st["n"], st["rows"], st["max_q"],
                          st["max_kv"], st["ld"])
    if k == "read":
        engine.pages_read(pages, batch, at("k_rows"), at("v_rows"), bf16=case["q"] == "bf16", stream=stream)
        return st["k_rows"], st["v_rows"]
    if k == "append":
        cfg = engine.append_cfg(H, at("cos"), at("sin"), st["max_kv"], norm=case["norm"], eps=EPS, wq=at("wq"),
                                wk=at("wk"), bf16=case["q"] == "bf16")
        engine.qk_append(pages, batch, cfg, at("qkv"), at("q"), stream)
        engine.pages_read(pages, batch, at("k_rows"), at("v_rows"), bf16=True, stream=stream)
        return st["q"], st["k_rows"], st["v_rows"]
    cfg = engine.attn_cfg(H, window=case["window"], sinks=case["sinks"], bf16=case["q"] == "bf16")
    if k == "attn":
        if "work" not in st:
            st["work"] = torch.empty(engine.paged_attn_work(pages, batch, cfg), dtype=torch.uint8, device="cuda")
        engine.paged_attn(pages, batch, cfg, at("q"), at("out"), at("work"), st["work"].numel(), stream)
        return st["out"]
    pre = engine.prefix(at("seq_start"), at("shared"), st["n_group"], st["max_shared"])
    if "work" not in st:
        st["work"] = torch.empty(engine.prefix_attn_work(pages, batch, pre, cfg), dtype=torch.uint8, device="cuda")
    engine.prefix_attn(pages, batch, pre, cfg, at("q"), at("out"), at("work"), st["work"].numel(), stream)
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


def _plain_read(st, rt):
    """Keys and values of the rows' positions, in the type rt."""
    case = st["case"]
    hd, P = HEADS[case["heads"]][2], case["page"]
    seq, pos = _rows_of(st)
    page, slot = st["table"][seq, pos // P], pos % P
    out = []
    for pool in (st["k"], st["v"]):
        codes, scales = _views(pool, P, hd)
        x = _values(codes[page, :, slot], case["kv"]) * scales[page, :, slot][..., None]
        out.append(x.reshape(st["rows"], -1).to(rt))
    return out


def _plain_append(st):
    case = st["case"]
    H, KH, hd = HEADS[case["heads"]]
    P = case["page"]
    q, k, v = st["qkv"].float().view(st["rows"], -1, hd).split([H, KH, KH], 1)
    if case["norm"]:
        q = _head_norm(q, st["wq"] if case["weights"] else None)
        k = _head_norm(k, st["wk"] if case["weights"] else None)
    seq, pos = _rows_of(st)
    c, s = st["cos"][pos][:, None, :], st["sin"][pos][:, None, :]
    q, k = _rotate(q, c, s), _rotate(k, c, s)
    page, slot = st["table"][seq, pos // P], pos % P
    for pool, x in ((st["k"], k), (st["v"], v)):
        codes, scales = _views(pool, P, hd)
        codes[page, :, slot], scales[page, :, slot] = _codes(x, case["kv"])
    return [q.reshape(st["rows"], -1).to(st["q"].dtype)] + _plain_read(st, torch.bfloat16)


def _plain_attn(st):
    case = st["case"]
    H, KH, hd = HEADS[case["heads"]]
    n, Q, T, G, P = st["n"], st["max_q"], st["max_kv"], H // KH, case["page"]
    pages = st["table"].clamp(min=0)

    def rows(pool):
        if case["kv"] in TOP:
            codes, scales = _views(pool, P, hd)
            x = _values(codes[pages], case["kv"]) * scales[pages][..., None]
        else:
            x = pool[pages].float()
        return x.transpose(1, 2).reshape(n, KH, -1, hd)[:, :, :T]

    K, V = rows(st["k"]), rows(st["v"])
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


def _row_of_each(start, n):
    """The row that each entry of a list of lists belongs to."""
    return torch.bucketize(torch.arange(n, device="cuda", dtype=torch.int32), start[1:], right=True)


def _plain_adjust(st):
    rows, V = st["x"].shape
    x = st["x"].double()  # (differences of near values)
    n = st["hist"].numel()
    row = _row_of_each(st["hist_start"], n)
    at = row * V + st["hist"].long()
    late = torch.arange(n, device="cuda") - st["hist_start"][row] >= st["count_from"][row]
    count = torch.zeros(rows * V, device="cuda", dtype=torch.float64).index_add_(0, at, late.double()).view(rows, V)
    seen = torch.zeros(rows * V, device="cuda", dtype=torch.bool).index_fill_(0, at, True).view(rows, V)
    col = lambda k: st[k].double()[:, None]  # noqa: E731
    x = torch.where(count > 0, x - col("pres") - col("freq") * count, x)
    x = torch.where(seen, torch.where(x > 0, x / col("rep"), x * col("rep")), x)
    n = st["bias"].numel()
    at = _row_of_each(st["bias_start"], n) * V + st["bias_id"].long()
    x = x.view(-1).index_add(0, at, st["bias"].double()).view(rows, V)
    if "mask" in st:
        bits = (st["mask"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        allowed = bits.view(bits.shape[0], -1)[:, :V].bool()[st["mask_row"].clamp(min=0)]
        x = x.masked_fill(~allowed & (st["mask_row"] >= 0)[:, None], -math.inf)
    return x.float()


@torch.no_grad()
def run(st):
    if own:
        return _own(st)
    k = st["case"]["kind"]
    if k == "adjust":
        return _plain_adjust(st)
    if k == "read":
        return _plain_read(st, st["k_rows"].dtype)
    if k == "append":
        return _plain_append(st)
    return _plain_attn(st)


# ------------------------------------------------------------------ what a call cannot do without

def _seen(case, kv, q):
    """(query, key) pairs and the first visible key behind the sinks of a sequence."""
    w, s = case["window"], case["sinks"]
    if not w:
        return q * (kv - q) + q * (q + 1) / 2, 0
    pos = np.arange(int(kv - q), int(kv))
    first = np.maximum(0, pos - w + 1)
    pairs = (pos + 1 - first + np.minimum(first, s)).sum()
    return float(pairs), max(0, int(kv - q) - w + 1)


def work(case):
    k = case["kind"]
    if k == "adjust":
        rows, V = case["rows"], case["V"]
        lists = rows * 0.75 * (4.0 * case["hist"] + 8.0 * case["bias"])
        return {"bytes": rows * (8.0 * V + 40) + lists + case["masks"] * V / 8.0, "flops": 2.0 * rows * V}
    H, KH, hd = HEADS[case["heads"]]
    eq = 2 if case["q"] == "bf16" else 4
    row = {"f32": 4 * hd, "bf16": 2 * hd}.get(case["kv"], hd + 4)  # bytes of a key head's row
    kv, q, shared = _lengths(case)
    kv, q = kv.astype(np.float64), q.astype(np.float64)
    rows = q.sum()
    if k == "read":
        return {"bytes": float(2 * rows * KH * (row + hd * eq)), "flops": float(2 * rows * KH * hd)}
    if k == "append":
        by = rows * (hd * ((2 * H + 2 * KH) * eq + 2 * KH * 2) + 2 * KH * row) + kv.max() * hd * 4
        return {"bytes": float(by), "flops": float(rows * hd * (8 * (H + KH) + 6 * KH))}
    pairs = keys = 0.0
    groups = {}  # the first shared position that someone of the group sees, and the sinks
    for i, (a, b) in enumerate(zip(kv, q)):
        p, lo = _seen(case, a, b)
        pairs += p
        from_own = 0 if shared is None else int(shared[i])
        keys += a - max(lo, from_own) + max(0, min(lo, case["sinks"]) - from_own)
        if from_own:
            g = int(i * case["groups"] // case["n"])
            groups[g] = (from_own, min(lo, groups.get(g, (0, lo))[1]))
    for top, lo in groups.values():
        keys += max(0, top - lo) + min(lo, case["sinks"], top)
    return {"bytes": float(2 * rows * H * hd * eq + 2 * keys * KH * row), "flops": float(4.0 * hd * H * pairs)}


# ------------------------------------------------------------------ 64 bits

def _exact_values(st, name, page):
    """Float64 [positions, KH, hd] of the pages `page` in order."""
    case = st["case"]
    _, KH, hd = HEADS[case["heads"]]
    P, kv = case["page"], case["kv"]
    x = st[name][page]
    if kv in TOP:
        scale = x[:, :, P * hd:].contiguous().view(torch.float32).double()
        x = x[:, :, :P * hd].contiguous().view(torch.int8 if kv == "i8" else torch.float8_e4m3fn)
        x = x.to(torch.float32).double().reshape(-1, KH, P, hd) * scale[..., None]
    return x.double().permute(0, 2, 1, 3).reshape(-1, KH, hd)


def _exact_attn(st):
    case = st["case"]
    H, KH, hd = HEADS[case["heads"]]
    G, P = H // KH, case["page"]
    start, lens, table = (st[n].cpu().numpy() for n in ("start", "kv_len", "table"))
    out = torch.zeros(st["rows"], H, hd, device="cuda", dtype=torch.float64)
    for b in range(st["n"]):
        a, z, T = int(start[b]), int(start[b + 1]), int(lens[b])
        pages = torch.from_numpy(table[b, :-(-T // P)].astype(np.int64)).cuda()
        K, V = (_exact_values(st, n, pages)[:T] for n in ("k", "v"))
        p = torch.arange(T - (z - a), T, device="cuda")[:, None]
        j = torch.arange(T, device="cuda")[None, :]
        hidden = j > p
        if case["window"]:
            hidden = hidden | ((j <= p - case["window"]) & (j >= case["sinks"]))
        for h in range(H):
            key, val = K[:, h // G].contiguous(), V[:, h // G].contiguous()
            q = st["q"][a:z, h * hd:(h + 1) * hd].double()
            for r in range(0, z - a, 1024):
                s = (q[r:r + 1024] @ key.t().contiguous()) / math.sqrt(hd)
                s = s.masked_fill(hidden[r:r + 1024], -math.inf)
                out[a + r:a + r + s.shape[0], h] = torch.softmax(s, -1) @ val
    return out.reshape(st["rows"], H * hd)


def _exact_quantised(x, kv):
    """The values that float64 rows stand for in 8 bits."""
    top = TOP[kv]
    step = x.abs().amax(-1, keepdim=True) / top
    y = (x / step.clamp(min=1e-300)).clamp(-top, top)
    if kv == "i8":
        return torch.round(y) * step
    # e4m3: three bits behind the leading one, its exponent from -6 on
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    unit = torch.exp2(e - 3)
    return torch.round(y / unit) * unit * step


def _exact_append(st):
    case = st["case"]
    H, KH, hd = HEADS[case["heads"]]
    x = st["qkv"].double().reshape(st["rows"], H + 2 * KH, hd)
    start, lens = st["start"].cpu().numpy(), st["kv_len"].cpu().numpy()
    q = torch.empty(st["rows"], H * hd, device="cuda", dtype=torch.float64)
    k = torch.empty(st["rows"], KH, hd, device="cuda", dtype=torch.float64)
    h2 = hd // 2
    for b in range(st["n"]):
        a, z, T = int(start[b]), int(start[b + 1]), int(lens[b])
        pos = torch.arange(T - (z - a), T, device="cuda")
        c, s = st["cos"][pos].double()[:, None], st["sin"][pos].double()[:, None]
        y = x[a:z, :H + KH]
        if case["norm"]:
            y = y / ((y ** 2).sum(-1, keepdim=True) / hd + EPS).sqrt()
            if case["weights"]:
                y = torch.cat([y[:, :H] * st["wq"].double(), y[:, H:] * st["wk"].double()], 1)
        y = torch.cat([y[..., :h2] * c + y[..., h2:] * s, y[..., h2:] * c - y[..., :h2] * s], -1)
        q[a:z], k[a:z] = y[:, :H].reshape(z - a, -1), y[:, H:]
    v = x[:, H + KH:]
    return [q] + [_exact_quantised(t, case["kv"]).reshape(st["rows"], -1) for t in (k, v)]


def _exact_read(st):
    P = st["case"]["page"]
    lens, table = st["kv_len"].cpu().numpy(), st["table"].cpu().numpy()
    out = []
    for name in ("k", "v"):
        parts = []
        for b in range(st["n"]):
            T = int(lens[b])
            pages = torch.from_numpy(table[b, :-(-T // P)].astype(np.int64)).cuda()
            parts.append(_exact_values(st, name, pages)[:T].reshape(T, -1))
        out.append(torch.cat(parts))
    return out


def _exact_adjust(st):
    """Row by row on the host, from the definition."""
    x = st["x"].cpu().numpy().astype(np.float64)
    get = lambda n: st[n].cpu().numpy()  # noqa: E731
    hs, hist, start, bs, ids, bias = (get(n) for n in ("hist_start", "hist", "count_from", "bias_start", "bias_id",
                                                       "bias"))
    rep, pres, freq = (get(n).astype(np.float64) for n in ("rep", "pres", "freq"))
    for r in range(len(x)):
        h = hist[hs[r]:hs[r + 1]]
        which, times = np.unique(h[start[r]:], return_counts=True)
        x[r, which] -= pres[r] + freq[r] * times
        which = np.unique(h)
        y = x[r, which]
        x[r, which] = np.where(y > 0, y / rep[r], y * rep[r])
        np.add.at(x[r], ids[bs[r]:bs[r + 1]], bias[bs[r]:bs[r + 1]].astype(np.float64))
        if "mask" in st and get("mask_row")[r] >= 0:
            words = get("mask")[get("mask_row")[r]].view(np.uint32)
            bits = np.unpackbits(words.view(np.uint8), bitorder="little")[:x.shape[1]]
            x[r, bits == 0] = -np.inf
    return x


@torch.no_grad()
def exact(case, seed):
    st = prepare(case, seed)
    return {"adjust": _exact_adjust, "read": _exact_read, "append": _exact_append}.get(case["kind"], _exact_attn)(st)
