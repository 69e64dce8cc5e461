"""The split of an attention call over the paged KV cache, on the host: for
batches of every kind no two rows' partial results may share a place in the
workspace, and what the join reads of a row must be that row's pieces, each step
of its tiles once.  tests/c/paged_split.cpp follows the library's own functions."""
import os
import shutil
import subprocess

import numpy as np
import pytest

from paged_util import F16, Q4_0, Q8_0

HERE = os.path.dirname(__file__)
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")


@pytest.fixture(scope="session")
def split(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("split") / "paged_split")
    subprocess.run([HIPCC, "-O2", "-std=c++17", "--offload-host-only", "-x", "hip", os.path.join(HERE, "c", "paged_split.cpp"), "-o", exe],
                   check=True, capture_output=True, text=True)

    def run(batches):
        r = subprocess.run([exe], input="\n".join(batches) + "\n", capture_output=True, text=True, timeout=600)
        lines = r.stdout.splitlines()
        assert r.returncode == 0 and len(lines) == len(batches), (r.returncode, lines[-1:], r.stderr[-500:])
        return lines
    return run


def batch(t, n_head, n_kv, hd, lens, new=None, pad=0, n_prefix=0, window=0, page=16, max_len=None, offs=None):
    """One line of tests/c/paged_split.cpp; new None: one token each."""
    max_len = max(lens, default=0) if max_len is None else max_len
    if offs is None and new is not None:
        offs = [0] + [int(x) for x in np.cumsum(new)]
    n_tok = (offs[-1] if offs is not None else len(lens)) + pad
    head = [t, n_head, n_kv, hd, page, max_len, n_prefix, window, len(lens), n_tok, -(-max_len // page), int(offs is not None)]
    return " ".join(str(int(x)) for x in head + list(lens) + list(offs or []))


def _good(split, batches):
    bad = [(b[:150], line) for b, line in zip(batches, split(batches)) if not line.startswith("ok")]
    assert not bad, bad[:5]


def test_short_prefix_before_long_parts(split):
    # shares of several whole tiles of the prefix
    _good(split, [
        batch(F16, 8, 8, 128, [8192] * 8, n_prefix=100),
        batch(F16, 32, 8, 128, [32768], n_prefix=100),
        batch(Q8_0, 32, 8, 128, [8192] * 4, n_prefix=100),
        batch(F16, 8, 4, 256, [4096] * 8, n_prefix=60),
        batch(F16, 32, 8, 128, [512] * 4, new=[512] * 4, n_prefix=100),
        batch(F16, 32, 8, 128, [256] * 8, new=[256] * 8, n_prefix=500),
        batch(F16, 32, 8, 128, [64] * 64, new=[64] * 64, n_prefix=1000),
        batch(F16, 8, 4, 256, [1000] * 2, new=[1000] * 2, n_prefix=300),
        batch(F16, 8, 4, 256, [8192] * 4, n_prefix=50),
        batch(F16, 8, 4, 256, [2048], new=[2048], n_prefix=100),
        batch(F16, 8, 4, 256, [4300] * 4, new=[509] * 4, n_prefix=1000),
    ])


@pytest.mark.parametrize("seed", range(6))
def test_any_batch(split, seed):
    rng = np.random.default_rng(seed)
    log = lambda lo, hi: int(round(np.exp(rng.uniform(np.log(lo), np.log(hi)))))  # noqa: E731
    batches = []
    for _ in range(120):
        hd = int(rng.choice([64, 128, 256, 512]))
        n_kv = int(rng.choice([1, 2, 4, 8]))
        grp = int(rng.choice([1, 2, 3, 4, 6, 8, 12, 16, 20, 64, 128]))
        grp = min(grp, 64 if hd == 512 else 128)
        n_seq = log(1, 200)
        single = rng.random() < 0.4
        most = max(1, 20000 // (n_kv * grp * n_seq))
        new = None if single else [int(rng.integers(0, 1 + log(1, most))) if rng.random() < 0.8 else 1 for _ in range(n_seq)]
        longest = log(1, 20000)
        lens = [int(rng.integers(0, longest + 1)) + (0 if new is None else new[i]) for i in range(n_seq)]
        if rng.random() < 0.1:
            lens[0] = 0
        batches.append(batch(int(rng.choice([F16, Q8_0, Q4_0])), n_kv * grp, n_kv, hd, lens, new, pad=int(rng.integers(0, 4)) if new else 0,
                             n_prefix=int(rng.choice([0, log(1, 20000), log(1, 200)])), window=int(rng.choice([0, 0, 1, log(1, 30000)])),
                             max_len=max(lens) + int(rng.integers(0, 300))))
    _good(split, batches)
