"""The ranges in which the streaming attention for 8-bit caches hands out its line, on the CPU:
tests/prefix_shares.cu runs the library's own arithmetic."""
import os
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def shares(lq8_lib, tmp_path_factory):
    import build
    exe = str(tmp_path_factory.mktemp("shares") / "prefix_shares")
    r = subprocess.run([build._nvcc(), "-O2", "-std=c++17", "--expt-relaxed-constexpr", "-I", build.CSRC, "-I", build.INCLUDE,
                        "-o", exe, os.path.join(HERE, "prefix_shares.cu")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr

    def run(cases):
        r = subprocess.run([exe], input="\n".join(" ".join(map(str, c)) for c in cases), capture_output=True, text=True, timeout=600)
        assert r.returncode == 0
        out = r.stdout.split("\n")[:-1]
        assert len(out) == len(cases)
        return out

    return run


@pytest.mark.parametrize("workers", [1, 2, 3, 148, 264, 296, 444])
def test_ranges_cover_the_line(shares, workers):
    # (a plan has no fewer workers than a quarter of its steps, unless it has one for every CTA)
    rng = np.random.default_rng(workers)
    most = 1 << 26 if workers > 100 else 4 * workers
    totals = [0, 1, 2, workers - 1, workers, workers + 1, 4 * workers, *([16 * workers, 20 * workers - 1, 20 * workers, 20 * workers + 1, 37 * workers + 5, most]
              if workers > 100 else []), *np.exp(rng.uniform(0, np.log(most), 60)).astype(int)]
    cases = []
    for t in totals:
        t = int(min(max(t, 0), most))
        for sp in {0, t, int(rng.integers(0, t + 1))}:
            cases += [(workers, sp, t - sp, 0), (workers, sp, t - sp, 1)]
    out = shares(cases)
    assert all(o.startswith("ok") for o in out), [(c, o) for c, o in zip(cases, out) if not o.startswith("ok")][:5]
    for c, o in zip(cases, out):  # equal shares, or half of the line at most in the first ones
        total, (ranges, largest) = c[1] + c[2], map(int, o.split()[1:])
        if total:
            assert largest <= -(-total // workers) and (ranges == min(total, workers) or ranges == 5 * workers)


def test_the_model_sees_a_bad_cut(shares):
    """A multiplier of another number of workers is noticed (the largest line of few workers overflows it)."""
    assert shares([(1, 0, 1 << 26, 0)])[0].startswith("bad")
