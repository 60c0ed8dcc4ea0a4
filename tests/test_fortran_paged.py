"""The paged cache through the Fortran binding (tests/fortran/paged_checks)."""
import os
import subprocess

import numpy as np
import pytest

from autoresearch_amd.weights import Dims, seeded_weights, uniform_ids, write_npy_dir
from oracle import oracle as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CHECKS = os.path.join(ROOT, "tests", "fortran", "paged_checks")
DIMS = Dims(n_layer=2, d_model=128, n_head=2, n_kv_head=1, head_dim=64, vocab=512)


def run(args, timeout=120):
    return subprocess.run([CHECKS, *args], capture_output=True, text=True, timeout=timeout)


def test_null_handles_refused():
    r = run(["refusals"])
    assert r.returncode == 0 and "refusals: ok" in r.stdout, r.stdout + r.stderr


def test_usage_error():
    r = run(["nonsense"])
    assert r.returncode == 2 and "usage" in r.stderr


@pytest.mark.gpu
@pytest.mark.parametrize("n", [2, 33, 80])
def test_greedy_sequences_equal_the_oracles(tmp_path, n):
    """A prompt and a fork of its first half, decoded side by side: each
    sequence's ids are the oracle's greedy ones for it alone."""
    d, ngen = DIMS, 7
    w = seeded_weights(d, 71)
    write_npy_dir(str(tmp_path / "w"), d, w, ctx=n + ngen)
    prompt = uniform_ids(72, n, d.vocab)
    np.savetxt(tmp_path / "ids.txt", prompt[None, :], fmt="%d")
    r = run(["greedy", str(tmp_path / "w"),
             *(str(x) for x in (d.n_layer, d.d_model, d.n_head, d.n_kv_head, d.head_dim, d.vocab)),
             str(tmp_path / "ids.txt"), str(ngen), str(tmp_path / "out.txt")])
    assert r.returncode == 0, r.stdout + r.stderr
    got = np.loadtxt(tmp_path / "out.txt", dtype=int)
    c, s = O.rope_tables(n + ngen, d.head_dim)
    for ids, mine in ((prompt, got[0]), (prompt[:n // 2], got[1])):
        want = O.greedy_decode(ids, w, d, ngen, c, s, maxT=n + ngen)[0]
        assert np.array_equal(mine, want)
