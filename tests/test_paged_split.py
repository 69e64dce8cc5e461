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


def batch(t, n_head, n_kv, hd, lens, new=None, pad=0, n_prefix=0, window=0, page=16, max_len=None, offs=None, n_tok=None):
    """One line of tests/c/paged_split.cpp; new None: one token each."""
    max_len = max(lens, default=0) if max_len is None else max_len
    if offs is None and new is not None:
        offs = [0] + [int(x) for x in np.cumsum(new)]
    n_tok = (offs[-1] if offs is not None else len(lens)) + pad if n_tok is None else n_tok
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


def test_torn_offsets(split):
    # offsets that descend, leave the tokens or give them to several sequences: no
    # more steps than the host counted, and no row joined that was not noted
    many = [0, 4096] * 700
    _good(split, [
        batch(F16, 2, 1, 64, [60] * 4, n_prefix=20, offs=[0, 5, 2, 6, 3], n_tok=6),
        batch(F16, 2, 1, 64, [60, 40, 20], offs=[0, 2, 9, 6], n_tok=6),
        batch(F16, 2, 1, 64, [6000] * 4, n_prefix=20, offs=[0, 5, 2, 6, 3], n_tok=6),
        batch(F16, 2, 1, 64, [60] * 2, n_prefix=20, offs=[-3, 4, 6], n_tok=6),
        batch(F16, 2, 1, 64, [600] * 2, n_prefix=20, offs=[1 << 30, 4, 6], n_tok=6),
        batch(F16, 2, 1, 64, [600] * 2, n_prefix=20, offs=[0, 0, 7], n_tok=6),
        batch(F16, 2, 1, 64, [600] * 2, n_prefix=20, offs=[0, 6, -1 << 31], n_tok=6),
        batch(F16, 4, 4, 64, [1 << 20] * (len(many) - 1), n_prefix=20, offs=many, n_tok=4096),
        batch(F16, 4, 4, 64, [1 << 20] * (len(many) - 1), offs=many, n_tok=4096),
    ])


@pytest.mark.parametrize("seed", range(3))
def test_any_offsets(split, seed):
    rng = np.random.default_rng(100 + seed)
    batches = []
    for _ in range(150):
        n_seq, n_tok, n_kv, hd = int(rng.integers(1, 130)), int(rng.integers(1, 60)), int(rng.choice([1, 3])), int(rng.choice([64, 512]))
        offs = np.sort(rng.integers(0, n_tok + 1, n_seq + 1))
        for _ in range(int(rng.integers(0, 3))):
            offs[rng.integers(0, n_seq + 1)] = rng.integers(-5, n_tok + 6)
        lens = [int(n) for n in rng.integers(-2, 600, n_seq)]
        batches.append(batch(F16, n_kv * int(rng.choice([1, 4, 20])), n_kv, hd, lens, n_prefix=int(rng.choice([0, 30, 900])), max_len=560,
                             window=int(rng.choice([0, 50])), offs=[int(x) for x in offs], n_tok=n_tok))
    _good(split, batches)


def test_rows_before_and_behind_the_sequences(split):
    # a batch that is a part of a longer one's offsets
    _good(split, [batch(t, 8, 2, 128, [700, 600, 3], n_prefix=p, offs=[4, 5, 5 + n, 7 + n], n_tok=20 + n)
                  for t in (F16, Q8_0) for p in (0, 50, 3000) for n in (1, 2, 50)])


@pytest.mark.parametrize("t", [F16, Q8_0])
def test_windows_of_any_size(split, t):
    # padded slots hold tokens before position 0: a window as large as an int is no window
    for window in (1 << 26, (1 << 31) - 2, (1 << 31) - 1):
        _good(split, [batch(t, n_head, 2, 64, lens, new=new, n_prefix=p, window=window)
                      for n_head in (2, 40) for p in (0, 50) for lens, new in (([0, 5, 40], [3, 9, 40]), ([5, 700, 0], [200, 600, 200]), ([3] * 9, [4] * 9))])
