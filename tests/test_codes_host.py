"""Refusals of the calls on 8-bit pages, on the CPU: arguments are checked before
anything asks for a device."""
import pytest

from autoresearch_amd import engine

from .test_paged_host import BAD_BATCH, BAD_PAGES, P, append, attn, batch, no_gpu, pages, refused


def read(pg=None, bt=None, k=P, v=P, **kw):
    engine.pages_read(pg or pages(type=engine.FG_I8), bt or batch(), k, v, **kw)


@pytest.mark.parametrize("match,kw", BAD_PAGES)
def test_bad_pages(match, kw):
    refused(match, read, pages(**kw))


@pytest.mark.parametrize("match,kw", BAD_BATCH)
def test_bad_batch(match, kw):
    refused(match, read, pages(n_kv_head=16), batch(**kw))


@pytest.mark.parametrize("match,kw", [
    ("ld", dict(ld=127)), ("ld", dict(ld=130)), ("ld", dict(ld=132, bf16=True)), ("ld", dict(ld=-128)),
    ("aligned", dict(k=P + 8)), ("aligned", dict(v=P + 4))])
def test_bad_read(match, kw):
    refused(match, read, **kw)


def test_bad_read_type():
    L = engine.load_library()
    for t in (-1, engine.FG_I8, engine.FG_E4M3, 7):
        assert L.fg_pages_read(pages(), batch(), t, 0, P, P, 0) == -1


def test_nothing_to_read():
    read(k=0, v=0)
    read(bt=batch(n_rows=0))


@pytest.mark.parametrize("kind", [engine.FG_I8, engine.FG_E4M3])
def test_rows_are_fp32_or_bf16(kind):
    """8-bit pages take both kinds of rows; rows are never of an 8-bit type."""
    for bf16 in (False, True):
        assert engine.paged_attn_work(pages(type=kind), batch(), engine.attn_cfg(4, bf16=bf16)) >= 0
    refused("row type", attn, pages(type=kind), type=kind)
    cfg = engine.append_cfg(4)
    cfg.type = kind
    refused("row type", engine.qk_append, pages(type=kind), batch(), cfg, P, P)
    refused("aligned", append, pages(type=kind), qkv=P + 8)


@pytest.mark.parametrize("kind,row", [(engine.FG_F32, 256), (engine.FG_BF16, 128), (engine.FG_I8, 68),
                                      (engine.FG_E4M3, 68)])
def test_page_bytes(kind, row):
    assert engine.page_bytes(32, 3, 64, kind) == 32 * 3 * row
    with pytest.raises(engine.FgptError, match="type"):
        engine.page_bytes(32, 3, 64, 4)
    with pytest.raises(engine.FgptError, match="head_dim"):
        engine.page_bytes(32, 3, 80, kind)
    assert engine.load_library().fg_page_bytes(None, None) == -1


@pytest.mark.skipif(not no_gpu(), reason="a GPU is visible")
def test_no_device():
    with pytest.raises(engine.FgptError) as e:
        read()
    assert e.value.code in (-7, -4)
