"""Refusals of the paged cache's operators, on the CPU: arguments are checked
before anything asks for a device, and nothing runs without one."""
import ctypes as C
import random
import resource

import pytest

from autoresearch_amd import engine

P = 1 << 20  # a 16-byte aligned address that nothing reads


def no_gpu():
    import torch
    return not torch.cuda.is_available()


def pages(**kw):
    a = dict(k=P, v=P, n_pages=8, page_size=16, n_kv_head=2, head_dim=64, bf16=False)
    a.update(kw)
    t = a.pop("type", None)
    s = engine.pages(**a)
    if t is not None:
        s.type = t
    return s


def batch(**kw):
    a = dict(q_start=P, kv_len=P, table=P, n_seq=2, n_rows=4, max_q=2, max_kv=32, table_ld=2)
    a.update(kw)
    return engine.ragged(**a)


def attn(pg=None, bt=None, q=P, out=P, work=0, work_bytes=0, n_head=4, **kw):
    t = kw.pop("type", None)
    cfg = engine.attn_cfg(n_head, **kw)
    if t is not None:
        cfg.type = t
    engine.paged_attn(pg or pages(), bt or batch(), cfg, q, out, work, work_bytes)


def append(pg=None, bt=None, qkv=P, q=P, n_head=4, **kw):
    engine.qk_append(pg or pages(), bt or batch(), engine.append_cfg(n_head, **kw), qkv, q)


def refused(match, f, *a, **kw):
    with pytest.raises(engine.FgptError, match=match) as e:
        f(*a, **kw)
    assert e.value.code == -1


BAD_PAGES = [("NULL", dict(k=0)), ("NULL", dict(v=0)), ("head_dim", dict(head_dim=96)),
             ("page_size", dict(page_size=8)), ("page_size", dict(page_size=48)),
             ("page_size", dict(page_size=512)), ("n_pages", dict(n_pages=0)),
             ("n_pages", dict(n_kv_head=0)), ("type", dict(type=5)), ("aligned", dict(k=P + 8)),
             ("n_kv_head", dict(n_kv_head=2000))]
BAD_BATCH = [("NULL", dict(q_start=0)), ("NULL", dict(kv_len=0)), ("NULL", dict(table=0)),
             ("n_seq", dict(n_seq=0)), ("n_rows", dict(n_rows=-1)), ("max_q", dict(max_q=-1)),
             ("max_kv", dict(max_kv=-1)), ("table_ld", dict(table_ld=0)), ("beyond", dict(max_kv=33)),
             ("above 2\\^23", dict(n_rows=(1 << 23) + 1)), ("above 2\\^26", dict(n_rows=(1 << 23))),
             ("above 2\\^22", dict(n_seq=(1 << 22)))]


@pytest.mark.parametrize("match,kw", BAD_PAGES)
def test_bad_pages(match, kw):
    refused(match, attn, pages(**kw))
    refused(match, append, pages(**kw))


@pytest.mark.parametrize("match,kw", BAD_BATCH)
def test_bad_batch(match, kw):
    refused(match, attn, bt=batch(**kw), n_head=16)
    refused(match, append, bt=batch(**kw), n_head=16)


@pytest.mark.parametrize("match,kw", [
    ("multiple of n_kv_head", dict(n_head=3)), ("multiple of n_kv_head", dict(n_head=0)),
    ("bf16 rows need bf16 pages", dict(bf16=True)), ("row type", dict(type=9)),
    ("window", dict(window=-1)), ("window", dict(sinks=-1)), ("scale", dict(scale=-1.0)),
    ("scale", dict(scale=float("nan"))), ("scale", dict(scale=float("inf"))),
    ("q_ld", dict(q_ld=255)), ("q_ld", dict(q_ld=258)), ("out_ld", dict(out_ld=128)),
    ("NULL", dict(q=0)), ("NULL", dict(out=0)), ("aligned", dict(q=P + 4)), ("aligned", dict(out=P + 8))])
def test_bad_attention(match, kw):
    refused(match, attn, **kw)


def test_attention_workspace():
    bt = batch(max_kv=4096, table_ld=256)
    need = engine.paged_attn_work(pages(), bt, engine.attn_cfg(4))
    assert need > 0
    refused("work", attn, bt=bt)
    refused("work", attn, bt=bt, work=P, work_bytes=need - 1)
    refused("aligned", attn, bt=bt, work=P + 4, work_bytes=need)
    assert engine.paged_attn_work(pages(), batch(n_rows=0, max_q=0), engine.attn_cfg(4)) == 0


@pytest.mark.parametrize("match,kw", [
    ("go together", dict(cos=P)), ("rope_n", dict(cos=P, sin=P, rope_n=31)),
    ("aligned", dict(cos=P + 4, sin=P, rope_n=32)), ("eps", dict(norm=True, eps=-1.0)),
    ("eps", dict(norm=True, eps=float("nan"))), ("qkv_ld", dict(qkv_ld=511)), ("q_ld", dict(q_ld=254)),
    ("NULL", dict(qkv=0)), ("NULL", dict(q=0)), ("aligned", dict(qkv=P + 8)),
    ("multiple of n_kv_head", dict(n_head=5))])
def test_bad_append(match, kw):
    refused(match, append, **kw)


def copy(src=(0,), dst=(1,), base=P, planes=2, plane_bytes=256, n_pages=4, page_bytes=64):
    engine.pages_copy(base, planes, plane_bytes, n_pages, page_bytes, list(src), list(dst))


@pytest.mark.parametrize("match,kw", [
    ("outside", dict(src=[4])), ("outside", dict(dst=[-1])), ("outside", dict(src=[-1])),
    ("named before", dict(src=[0, 2], dst=[1, 1])), ("also written", dict(src=[0, 1], dst=[1, 2])),
    ("named before", dict(src=[0, 2], dst=[1, 0])), ("also written", dict(src=[1], dst=[1])),
    ("n_planes", dict(planes=0)), ("n_planes", dict(planes=70000)), ("page_bytes", dict(page_bytes=24)),
    ("page_bytes", dict(page_bytes=0)), ("plane_bytes", dict(plane_bytes=192)),
    ("plane_bytes", dict(plane_bytes=264)), ("NULL", dict(base=0)), ("aligned", dict(base=P + 4))])
def test_bad_copy(match, kw):
    refused(match, copy, **kw)


def test_copy_lists_of_unlike_length():
    with pytest.raises(ValueError):
        copy(src=[0, 1], dst=[2])


def draw(logits=P, rows=2, V=100, ld=100, u=P, ids=P, **kw):
    engine.draw_rows(logits, rows, V, ld, u, ids, work=P, work_bytes=1 << 40, **kw)


@pytest.mark.parametrize("match,kw", [
    ("rows", dict(rows=-1)), ("above 2\\^21", dict(rows=(1 << 21) + 1)), ("V 0", dict(V=0)), ("V 262145", dict(V=262145, ld=262145)), ("ld", dict(ld=99)),
    ("NULL", dict(logits=0)), ("NULL", dict(u=0)), ("NULL", dict(ids=0))])
def test_bad_draw(match, kw):
    refused(match, draw, **kw)


def test_null_structs():
    lib = engine.load_library()
    n = C.c_int64()
    assert lib.fg_paged_attn(None, None, None, P, P, None, 0, None) == -1
    assert lib.fg_paged_attn(pages(), batch(), None, P, P, None, 0, None) == -1
    assert lib.fg_qk_append(pages(), None, None, P, P, None) == -1
    assert lib.fg_qk_append(pages(), batch(), None, P, P, None) == -1
    assert lib.fg_draw_rows(P, 1, 5, 5, None, P, None, None, 0, None) == -1
    assert lib.fg_paged_attn_work(pages(), batch(), engine.attn_cfg(4), None) == -1
    assert lib.fg_draw_rows_work(1, 5, None) == -1
    assert lib.fg_pages_copy(P, 1, 0, 4, 16, None, None, 1, None) == -1
    assert lib.fg_draw_rows_work(1, 5, C.byref(n)) == 0


@pytest.mark.skipif(not no_gpu(), reason="a GPU is visible")
def test_no_device_fails_loudly():
    for f in (lambda: attn(work=P, work_bytes=1 << 40), append, copy, draw):
        with pytest.raises(engine.FgptError) as e:
            f()
        assert e.value.code == -7


def test_nothing_to_do_needs_no_device():
    attn(bt=batch(n_rows=0))
    append(bt=batch(n_rows=0))
    copy(src=[], dst=[])
    draw(rows=0)


@pytest.mark.parametrize("max_q", [(1 << 31) - 1, 1 << 29, 1 << 20])
@pytest.mark.parametrize("n_head,n_rows,n_seq", [(8, 40, 1), (16, 4, 4), (16, 4, 3), (16, 32, 1)])
def test_a_loose_max_q_asks_for_no_more_than_the_rows(max_q, n_head, n_rows, n_seq):
    """No sequence has more new tokens than there are rows: any larger bound is
    that one (times the query heads of a key head it would pass 32 bits)."""
    kw = dict(n_seq=n_seq, n_rows=n_rows, max_kv=20000, table_ld=1250)
    cfg = engine.attn_cfg(n_head)
    want = engine.paged_attn_work(pages(), batch(max_q=n_rows, **kw), cfg)
    assert engine.paged_attn_work(pages(), batch(max_q=max_q, **kw), cfg) == want


@pytest.mark.parametrize("kw", [dict(), dict(window=8), dict(window=8, sinks=4)])
def test_a_cache_of_no_position(kw):
    """max_kv 0: no key to cut into parts."""
    for n_rows, n_seq in ((1, 1), (4, 2), (5000, 3)):
        bt = batch(max_kv=0, n_rows=n_rows, n_seq=n_seq, max_q=n_rows)
        assert engine.paged_attn_work(pages(), bt, engine.attn_cfg(16, **kw)) == 0


def copy_code(src, dst, **kw):
    with pytest.raises(engine.FgptError) as e:
        copy(src, dst, **kw)
    return e.value.code


@pytest.mark.skipif(not no_gpu(), reason="a GPU is visible")
@pytest.mark.parametrize("seed", range(30))
def test_copy_lists_against_their_definition(seed):
    """No page twice in dst, none in both; a source may serve several copies."""
    r = random.Random(seed)
    for _ in range(40):
        n = r.choice([1, 2, 15, 63, 64, 65, 300, 1000])
        n_pages = r.choice([2 * n, 2 * n + 7, 1 << 20, (1 << 31) - 1])
        pick = r.sample(range(n_pages), 2 * n)
        src, dst = pick[:n], pick[n:]
        i, j = r.randrange(n), r.randrange(n)
        what = r.choice(["good", "shared", "twice", "both"])
        if what == "shared":
            src[i] = src[j]
        elif what == "twice":
            dst[i] = dst[j]
        elif what == "both":
            src[i] = dst[j]
        good = len(set(dst)) == n and not set(src) & set(dst)
        assert copy_code(src, dst, planes=1, n_pages=n_pages, page_bytes=16) == (-7 if good else -1), what


@pytest.mark.skipif(not no_gpu(), reason="a GPU is visible")
def test_a_short_copy_list_costs_nothing_of_a_large_pool():
    """One page of a pool of 2^31 - 1: no memory for each page of it (the check
    comes to asking for a device under a limit of 256 MB more than now)."""
    with open("/proc/self/statm") as f:
        now = int(f.read().split()[0]) * resource.getpagesize()
    old = resource.getrlimit(resource.RLIMIT_AS)
    resource.setrlimit(resource.RLIMIT_AS, (now + (256 << 20), old[1]))
    try:
        code = copy_code([5], [(1 << 31) - 2], planes=1, n_pages=(1 << 31) - 1, page_bytes=16)
    finally:
        resource.setrlimit(resource.RLIMIT_AS, old)
    assert code == -7


@pytest.mark.parametrize("kw,good", [(dict(), True), (dict(q_ld=256), True), (dict(out_ld=256), True),
                                     (dict(q_ld=512, out_ld=512), True), (dict(q_ld=512), False),
                                     (dict(out_ld=260), False), (dict(q_ld=512, out_ld=516), False)])
@pytest.mark.skipif(not no_gpu(), reason="a GPU is visible")
def test_attention_in_place_keeps_the_row_distance(kw, good):
    """With another one, rows would be written over before they are read."""
    with pytest.raises(engine.FgptError, match="device" if good else "row distance"):
        attn(q=P, out=P, **kw)
    with pytest.raises(engine.FgptError, match="device"):  # (one row has no distance)
        attn(bt=batch(n_rows=1, max_q=1), q=P, out=P, **kw)
