"""The schedule of the bf16 shared-prefix attention, on the CPU: tests/prefix_schedule.cu runs the
library's own cut of the work and hand-out rule against a model of the kernel's scheduler and of the
warps that serve its two flows, and reports CTAs in which they would wait for each other."""
import os
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def schedule(lq8_lib, tmp_path_factory):
    import build
    exe = str(tmp_path_factory.mktemp("schedule") / "prefix_schedule")
    r = subprocess.run([build._nvcc(), "-O2", "-std=c++17", "--expt-relaxed-constexpr", "-I", build.CSRC, "-I", build.INCLUDE,
                        "-o", exe, os.path.join(HERE, "prefix_schedule.cu")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr

    def run(cases, rule=0):
        """cases: (kv lengths, heads, kv heads, prefix, rows a sequence); the output line of each."""
        text = "\n".join(" ".join(map(str, [rule, q, heads, kv_heads, prefix, q, max(kv), len(kv), *kv]))
                         for kv, heads, kv_heads, prefix, q in cases)
        r = subprocess.run([exe], input=text, capture_output=True, text=True, timeout=600)
        assert r.returncode == 0
        out = r.stdout.split("\n")[:-1]
        assert len(out) == len(cases)
        return out

    return run


def lengths(n, most, kind):
    i = np.arange(n)
    if kind == "random":
        return np.random.default_rng(n).integers(1, most + 1, n).tolist()
    if kind == "two sizes":
        return np.where(np.random.default_rng(n + 1).random(n) < 0.5, max(1, most // 8), most).tolist()
    if kind == "few long":
        return [most] * max(1, n // 3) + [min(most, 100)] * (n - max(1, n // 3))
    fall = (most * (n - i) // n).clip(1)
    return (fall if kind == "falling" else fall[::-1] if kind == "rising" else np.where(i % 2, fall[::-1], fall)).tolist()


KINDS = ["falling", "rising", "mixed", "random", "two sizes", "few long"]

# lengths whose flows have rounds so unequal that a scheduler which evens them out only at the
# end waits for the serving warps, and they for it
HARD = [
    ([4000 * (128 - i) // 128 + 1 for i in range(128)], 32, 32, 0, 1),
    *[([(4000 * (n - i) // n) or 1 for i in range(n)], 64, 8, prefix, 1) for n in (512, 640, 768, 1024) for prefix in (0, 2048, 32768)],
    ([32768] * 16 + [100] * 25, 8, 8, 0, 1),
    ([32768] * 16 + [100] * 11, 8, 8, 0, 1),
    ([8192] * 64 + [100] * 40, 8, 8, 0, 1),
]


def test_the_model_sees_a_schedule_that_waits_for_itself(schedule):
    """Rounds evened out only at the end: the first case stops in CTA 147."""
    out = schedule(HARD, rule=1)
    assert out[0] == "1 147" and all(int(o.split()[0]) > 0 for o in out), out


def test_hard_lengths_end(schedule):
    assert set(schedule(HARD)) == {"0 -1"}


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 2), (64, 8), (8, 8), (32, 32), (128, 1)])
@pytest.mark.parametrize("q", [1, 2, 40])
def test_every_schedule_ends(schedule, heads, kv_heads, q):
    cases = []
    for n in (1, 2, 3, 16, 17, 41, 128, 200, 513, 1024, 2048):
        if n * q > 4096:
            continue
        for kind in KINDS:
            cases += [(lengths(n, most, kind), heads, kv_heads, prefix, q) for most, prefix in
                      [(1, 0), (1, 2049), (300, 0), (300, 1), (4000, 0), (4000, 32768)]]
    rng = np.random.default_rng(heads * 100 + kv_heads + q)
    for _ in range(40):
        n = int(2 ** rng.uniform(0, 11 if q == 1 else 6))
        kv = (2 ** rng.uniform(0, 15 if n < 100 else 12, n)).astype(int).tolist()
        cases.append((kv, heads, kv_heads, int(rng.choice([0, 700, 131072])), q))
    out = schedule(cases)
    bad = [(c[1:], len(c[0]), o) for c, o in zip(cases, out) if o not in ("0 -1", "refused")]
    assert not bad, bad[:5]
    assert out.count("refused") < len(out) // 4
