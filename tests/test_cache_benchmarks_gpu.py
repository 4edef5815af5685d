"""The sweeps of the operators around the paged cache (``python -m flagattention_amd.benchmarks {paged_fp8,step}``)."""
import math

import pytest

from flagattention_amd import benchmarks


def test_codes_are_one_byte_each():
    assert benchmarks.kv_bytes(rows=64 * 4096, heads_kv=8, D=128, itemsize=1) * 2 == benchmarks.kv_bytes(64 * 4096, 8, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("which", benchmarks.CACHE_SWEEPS)
def test_every_sweep_runs_one_point(which):
    (r,) = benchmarks.run(which, quick=True, points=1)
    assert math.isfinite(r["ms"]) and r["ms"] > 0
    if which == "paged_fp8":
        assert (r["num_seqs"], r["group"], r["D"], r["ctx"], r["bytes"]) == (1, 1, 64, 512, 2 * 512 * 64 * 64)
    else:
        assert (r["bits"], r["num_seqs"], r["ctx"]) == (8, 1, 1024)
