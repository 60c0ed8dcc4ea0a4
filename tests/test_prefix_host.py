"""Refusals of fg_prefix_attn, on the CPU: arguments are checked before anything
asks for a device."""
import pytest

from autoresearch_amd import engine

from .test_paged_host import BAD_BATCH, BAD_PAGES, P, batch, no_gpu, pages, refused


def prefix(**kw):
    a = dict(seq_start=P, shared=P, n_group=1, max_shared=32)
    a.update(kw)
    return engine.prefix(**a)


def attn(pg=None, bt=None, pre=None, q=P, out=P, work=P, work_bytes=1 << 40, n_head=4, **kw):
    engine.prefix_attn(pg or pages(), bt or batch(), pre or prefix(), engine.attn_cfg(n_head, **kw), q, out, work,
                       work_bytes)


@pytest.mark.parametrize("match,kw", BAD_PAGES)
def test_bad_pages(match, kw):
    refused(match, attn, pages(**kw))


@pytest.mark.parametrize("match,kw", BAD_BATCH)
def test_bad_batch(match, kw):
    refused(match, attn, bt=batch(**kw), n_head=16)


@pytest.mark.parametrize("match,kw", [
    ("NULL", dict(seq_start=0)), ("NULL", dict(shared=0)), ("n_group", dict(n_group=0)),
    ("n_group", dict(n_group=3)), ("max_shared", dict(max_shared=-1)), ("max_shared", dict(max_shared=33))])
def test_bad_prefix(match, kw):
    refused(match, attn, pre=prefix(**kw))


@pytest.mark.parametrize("match,kw", [
    ("multiple of n_kv_head", dict(n_head=3)), ("bf16 rows need bf16 pages", dict(bf16=True)),
    ("window", dict(window=-1)), ("scale", dict(scale=-1.0)), ("q_ld", dict(q_ld=255)), ("NULL", dict(q=0)),
    ("NULL", dict(out=0)), ("aligned", dict(q=P + 4)), ("aligned", dict(work=P + 4)), ("work", dict(work=0)),
    ("another row distance", dict(q_ld=512))])
def test_bad_attention(match, kw):
    refused(match, attn, **kw)


def test_workspace():
    need = engine.prefix_attn_work(pages(), batch(), prefix(), engine.attn_cfg(4))
    assert need > 0
    refused("work", attn, work_bytes=need - 1)
    assert engine.prefix_attn_work(pages(), batch(n_rows=0, max_q=0), prefix(), engine.attn_cfg(4)) == 0
    attn(bt=batch(n_rows=0))  # nothing to do


@pytest.mark.skipif(not no_gpu(), reason="a GPU is visible")
def test_no_device():
    with pytest.raises(engine.FgptError) as e:
        attn()
    assert e.value.code in (-7, -4)
