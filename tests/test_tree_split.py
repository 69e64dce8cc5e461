"""The split of an attention call over trees of new tokens, on the host, as
tests/test_paged_split.py looks at the other calls' (tests/c/tree_split.cpp)."""
import os
import subprocess

import numpy as np
import pytest

from paged_util import F16, Q4_0, Q8_0
from test_paged_split import HERE, HIPCC, batch

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")


@pytest.fixture(scope="session")
def split(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("split") / "tree_split")
    subprocess.run([HIPCC, "-O2", "-std=c++17", "--offload-host-only", "-x", "hip", os.path.join(HERE, "c", "tree_split.cpp"), "-o", exe],
                   check=True, capture_output=True, text=True)

    def run(batches):
        r = subprocess.run([exe], input="\n".join(batches) + "\n", capture_output=True, text=True, timeout=600)
        lines = r.stdout.splitlines()
        assert r.returncode == 0 and len(lines) == len(batches), (r.returncode, lines[-1:], r.stderr[-500:])
        bad = [(b[:150], line) for b, line in zip(batches, lines) if not line.startswith("ok")]
        assert not bad, bad[:5]
    return run


def test_light_and_heavy_tiles(split):
    batches = []
    for t in (F16, Q8_0, Q4_0):
        for hd, n_kv in ((64, 8), (128, 8), (256, 4), (512, 2)):
            for grp in (1, 2, 4, 20, 64):
                for new in ([1 + (7 * i) % 40 for i in range(32)], [1, 200] * 8, [64], [128, 1, 1, 1], [1] * 100 + [150]):
                    for n_prefix in (0, 77, 3000):
                        lens = [n + (997 * i) % 2500 for i, n in enumerate(new)]
                        batches.append(batch(t, grp * n_kv, n_kv, hd, lens, new, n_prefix=n_prefix, window=[0, 300][len(batches) % 2], max_len=5000))
    split(batches[::7])                                      # each kind of each


@pytest.mark.parametrize("seed", range(6))
def test_any_batch(split, seed):
    rng = np.random.default_rng(100 + seed)
    log = lambda lo, hi: int(round(np.exp(rng.uniform(np.log(lo), np.log(hi)))))  # noqa: E731
    batches = []
    for _ in range(60):
        hd = int(rng.choice([64, 128, 256, 512]))
        n_kv = int(rng.choice([1, 2, 4, 8]))
        grp = min(int(rng.choice([1, 2, 3, 4, 6, 8, 12, 16, 20, 64, 128])), 64 if hd == 512 else 128)
        n_seq = log(1, 200)
        most = max(1, 20000 // (n_kv * grp * n_seq))
        new = None if rng.random() < 0.2 else [int(rng.integers(0, 1 + log(1, most))) if rng.random() < 0.8 else 1 for _ in range(n_seq)]
        longest = log(1, 20000)
        lens = [int(rng.integers(0, longest + 1)) + (0 if new is None else new[i]) for i in range(n_seq)]
        if rng.random() < 0.1:
            lens[0] = 0
        batches.append(batch(int(rng.choice([F16, Q8_0, Q4_0])), n_kv * grp, n_kv, hd, lens, new, pad=int(rng.integers(0, 4)) if new else 0,
                             n_prefix=int(rng.choice([0, log(1, 20000), log(1, 200)])), window=int(rng.choice([0, 0, 1, log(1, 30000)])),
                             max_len=max(lens) + int(rng.integers(0, 300))))
    split(batches)
