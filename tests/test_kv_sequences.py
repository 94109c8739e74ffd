"""What the kernels make of a batch's arrays (csrc/spt_kv_seq.h), on the CPU:
compiled with checks of overflow and compared with the rule in Python's ints."""
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LOW, HIGH = -2 ** 31, 2 ** 31 - 1
MAIN = r"""
#include <cstdio>
#include "spt_kv_seq.h"
int main() {
    int lo, hi, len, n_rows, max_len, max_new;
    while (scanf("%d %d %d %d %d %d", &lo, &hi, &len, &n_rows, &max_len, &max_new) == 6) {
        const spt::KvSeq q = spt::kv_seq_of(lo, hi, len, n_rows, max_len, max_new);
        printf("%d %d %d %d %d\n", q.r0, q.n, q.first, q.end, (int)q.ok);
    }
}
"""


@pytest.fixture(scope="module")
def sequences(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv_seq")
    (d / "main.cpp").write_text(MAIN)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I",
                    os.path.join(ROOT, "stream-pt_amd", "csrc"), "-o", str(d / "main"), str(d / "main.cpp")], check=True)

    def run(cases):
        text = "\n".join(" ".join(map(str, c)) for c in cases)
        p = subprocess.run([str(d / "main")], input=text, capture_output=True, text=True)
        assert p.returncode == 0, p.stderr
        got = [tuple(map(int, line.split())) for line in p.stdout.splitlines()]
        assert len(got) == len(cases)
        return got

    return run


def _cases():
    ends = [LOW, LOW + 1, LOW + 5, LOW + 7, -100, -1, 0, 1, 4, 5, 6, 7, 8, 12, 2 ** 24, HIGH - 1, HIGH]
    out = [(lo, hi, n, rows, 64, new) for lo in ends for hi in ends for n in (LOW, -1, 0, 5, 64, 65, HIGH)
           for rows in (0, 1, 7, HIGH) for new in (1, 4, 2 ** 24)]
    rng = random.Random(0)
    for _ in range(2000):
        rows = rng.randint(0, 40)
        out.append((rng.randint(-10, 50), rng.randint(-10, 50), rng.randint(-3, 80), rows, 64, rng.randint(1, 30)))
    return out


def test_rows_stay_in_the_buffers(sequences):
    """Whatever the arrays hold, rows are inside the buffers and the sequence's."""
    for (lo, hi, n, rows, max_len, max_new), (r0, got, _, _, ok) in zip(_cases(), sequences(_cases())):
        what = (lo, hi, n, rows, max_len, max_new)
        assert 0 <= r0 <= rows and 0 <= got <= rows - r0, what
        assert got <= max(0, min(hi, rows) - max(0, lo)) and got <= max_new, what
        assert not ok or n <= max_len, what


def test_rows_are_the_last_positions(sequences):
    """Row hi - 1 is the last position, also where rows are cut at either end
    of the buffers; more rows than declared, cut or not, is a sequence too long."""
    for (lo, hi, n, rows, max_len, max_new), (r0, got, first, end, ok) in zip(_cases(), sequences(_cases())):
        what = (lo, hi, n, rows, max_len, max_new)
        assert ok == (n <= max_len and hi - lo <= max_new), what
        here = [r for r in (max(lo, 0), min(hi, rows) - 1) if 0 <= r < rows and lo <= r < hi]
        if ok and here:
            assert (r0, got) == (here[0], here[-1] - here[0] + 1), what
            assert [first, end - 1] == [max(0, n) - (hi - r) for r in here], what
