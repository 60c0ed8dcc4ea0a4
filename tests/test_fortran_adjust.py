"""Adjusted steps on an 8-bit paged cache through the Fortran binding
(tests/fortran/adjust_checks)."""
import os
import subprocess

import numpy as np
import pytest

from autoresearch_amd import engine
from autoresearch_amd.weights import Dims, rope_tables, seeded_weights, uniform_ids, write_npy_dir

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CHECKS = os.path.join(ROOT, "tests", "fortran", "adjust_checks")
DIMS = Dims(n_layer=2, d_model=128, n_head=2, n_kv_head=1, head_dim=64, vocab=512)


def run(args, timeout=120):
    return subprocess.run([CHECKS, *args], capture_output=True, text=True, timeout=timeout)


def test_refusals():
    r = run(["refusals"])
    assert r.returncode == 0 and "refusals: ok" in r.stdout, r.stdout + r.stderr


def test_usage_error():
    r = run(["nonsense"])
    assert r.returncode == 2 and "usage" in r.stderr


@pytest.mark.gpu
@pytest.mark.parametrize("n", [2, 33])
def test_banned_ids(tmp_path, n):
    """Odd ids, each at most once, and the same ones as through Python."""
    d, ngen = DIMS, 24
    w = seeded_weights(d, 71)
    write_npy_dir(str(tmp_path / "w"), d, w, ctx=n + ngen)
    prompt = uniform_ids(72, n, d.vocab)
    np.savetxt(tmp_path / "ids.txt", prompt[None, :], fmt="%d")
    r = run(["banned", str(tmp_path / "w"),
             *(str(x) for x in (d.n_layer, d.d_model, d.n_head, d.n_kv_head, d.head_dim, d.vocab)),
             str(tmp_path / "ids.txt"), str(ngen), str(tmp_path / "out.txt")])
    assert r.returncode == 0, r.stdout + r.stderr
    got = np.loadtxt(tmp_path / "out.txt", dtype=int)
    assert (got % 2 == 1).all() and np.unique(got).size == ngen
    m = engine.Model(d, stacks=w)
    c, s = rope_tables(n + ngen, d.head_dim)
    m.set_rope(c.reshape(-1), s.reshape(-1))
    pc = m.paged((n + ngen) // 16 + 2, 16, 1, type=engine.FG_I8)
    mine, ids = [], prompt
    for _ in range(ngen):
        _, nxt = pc.step({0: ids}, want_logits=False, bias=[[(i, -np.inf) for i in mine]],
                         allowed=[np.arange(d.vocab) % 2 == 1])
        mine.append(int(nxt[0]))
        ids = nxt
    pc.close()
    m.close()
    assert np.array_equal(got, mine)
