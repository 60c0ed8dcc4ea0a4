"""Refusals of fg_adjust_rows, on the CPU: arguments are checked before anything
asks for a device."""
import pytest

from autoresearch_amd import engine

from .test_paged_host import P, no_gpu, refused


def adjust(rows=2, V=100, ld=100, out_ld=100, x=P, out=P, **kw):
    engine.adjust_rows(x, rows, V, ld, engine.adjust_cfg(**kw), out, out_ld)


@pytest.mark.parametrize("match,kw", [
    ("rows", dict(rows=-1)), ("rows", dict(rows=(1 << 21) + 1)), ("V 0", dict(V=0)),
    ("V", dict(V=(1 << 18) + 1, ld=1 << 20, out_ld=1 << 20)), ("ld", dict(ld=99)), ("out_ld", dict(out_ld=99)),
    ("NULL", dict(x=0)), ("NULL", dict(out=0)), ("another row distance", dict(out_ld=104)),
    ("hist or hist_start", dict(n_hist=3, hist=P)), ("hist or hist_start", dict(n_hist=3, hist_start=P)),
    ("n_hist", dict(n_hist=-1)), ("n_hist", dict(n_hist=(1 << 30) + 1, hist=P, hist_start=P)),
    ("n_bias", dict(n_bias=-1)), ("bias", dict(n_bias=1, bias=P, bias_id=P)),
    ("bias", dict(n_bias=1, bias_start=P, bias_id=P)), ("mask is NULL", dict(n_mask=1)),
    ("n_mask", dict(n_mask=-1)), ("mask_ld", dict(mask=P, n_mask=2, mask_ld=3)),
    ("mask_ld", dict(mask_ld=-4)), ("2\\^40 words", dict(mask=P, n_mask=1 << 30, mask_ld=1 << 29)),
    ("1 masks for 2 rows", dict(mask=P, n_mask=1))])
def test_bad_adjust(match, kw):
    refused(match, adjust, **kw)


def test_more_than_a_launch_holds():
    """A row is taken in slices of 2048 ids; fewer than 2^24 of them."""
    V = 1 << 18
    refused("slices", adjust, rows=1 << 17, V=V, ld=V, out_ld=V)
    refused("slices", adjust, rows=1 << 21, V=2049 * 8, ld=V, out_ld=V)


def test_no_cfg():
    assert engine.load_library().fg_adjust_rows(P, 2, 100, 100, None, P, 100, None) == -1


def test_nothing_to_do():
    adjust(rows=0, x=0, out=0)


@pytest.mark.skipif(not no_gpu(), reason="a GPU is visible")
def test_no_device():
    with pytest.raises(engine.FgptError) as e:
        adjust()
    assert e.value.code in (-7, -4)


def step_cfg(**kw):
    """The lists of a Paged.step of two sequences as fg_adjust_cfg."""
    given = dict.fromkeys(("history", "count_from", "rep", "pres", "freq", "bias", "allowed")) | kw
    return engine.Paged._adjust(None, 2, [], *given.values())


@pytest.mark.parametrize("what", ["count_from", "rep", "pres", "freq"])
def test_penalties_need_a_history(what):
    assert step_cfg() is None
    for other in ({}, {"bias": [{}, {3: 1.0}]}):
        with pytest.raises(ValueError, match="without a history"):
            step_cfg(**{what: 1}, **other)


def test_lists_for_each_sequence():
    for kw in ({"history": [[1]]}, {"bias": [{}]}):
        with pytest.raises(ValueError, match="for each sequence"):
            step_cfg(**kw)


def test_unknown_page_type():
    with pytest.raises(ValueError, match="page type"):
        engine.Paged(None, 4, type=7)
