"""CPU: host-side rules of the decode-attention launches (kvmem_b200/csrc/attend_plan.cuh), compiled as plain C++."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run(tmp_path, body):
    src, exe = tmp_path / "x.cpp", tmp_path / "x"
    src.write_text('#include "attend_plan.cuh"\n#include <cstdio>\nusing namespace kvmb;\nint main() {\n' + body + "\n}\n")
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, "kvmem_b200", "csrc"), str(src), "-o", str(exe)], check=True)
    return subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()


@pytest.mark.parametrize("box", [16, 32, 64, 128])
def test_chunks_of_lists_and_tails(tmp_path, box):
    """As few as the table of 512 boxes allows: one for every list that fits it, and never a chunk that does not."""
    most = 512 * box // 128
    lists = [0, 1, most - 1, most, most + 1, 2 * most, 5 * most + 3, 254 * most, 300 * most]
    tails = [0, 1, 7, most, 1024, 40 * most]
    got = iter(run(tmp_path, "\n".join(f'printf("%u\\n", attend_least_chunks({a}ull, {b}ull, {most}ull));'
                                       for a in lists for b in tails)))
    for a in lists:
        for b in tails:
            n = int(next(got))
            if a <= most:
                assert n == 1
            elif n == 0:
                assert (a + b) // most >= 256
            else:
                assert n <= 256
                # chunk c takes tiles [all c / n, all (c + 1) / n), whatever the actual counts up to these are
                for x, y in ((a, b), (a, 0), (a - 1, b), (most + 1, b)):
                    t = x + y
                    assert max(min(t * (c + 1) // n, x) - min(t * c // n, x) for c in range(n)) <= most


def test_registers_that_the_split_needs(tmp_path):
    """640 x 96 = 128 x 64 + 256 x 136 + 256 x 72; 256 x 128 = 128 x 72 + 128 x 184. A kernel compiled to fewer cannot make
    the split (the launcher takes the other kernel then)."""
    quant = run(tmp_path, 'for (int r = 0; r <= 255; ++r) printf("%d\\n", ac_registers_fit(true, r));')
    narrow = run(tmp_path, 'for (int r = 0; r <= 255; ++r) printf("%d\\n", ac_registers_fit(false, r));')
    assert [r for r in range(256) if quant[r] == "1"] == list(range(96, 137))
    assert [r for r in range(256) if narrow[r] == "1"] == list(range(128, 185))
