"""The operators' argument checks (rosenna_b200/csrc/ops_checks.hpp), compiled as plain
host code and called on made-up addresses: nothing is read or run."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, SHAPE, ARG = 0, 4, 8

# expression -> status code
CASES = [
    # runs
    ("check_run(true, 8, 2, 4)", OK), ("check_run(true, 0, 0, 4)", OK), ("check_run(false, 8, 2, 4)", ARG),
    ("check_run(true, -1, 2, 4)", ARG), ("check_run(true, 8, -1, 4)", ARG), ("check_run(true, 8, (1LL << 28), 4)", SHAPE),
    ("check_run(true, (1LL << 38) + 1, 1, 1)", SHAPE), ("check_run(true, (1LL << 62), (1LL << 27), 1 << 20)", SHAPE),
    ("check_run(true, (1LL << 20), (1LL << 18), 2)", SHAPE), ("check_run(true, (1LL << 20), (1LL << 18), 1)", OK),
    # arrays
    ("check_array(A(0, 4, 8), 8, true)", ARG), ("check_array(A(0, 4, 8), 8, false)", OK), ("check_array(A(0, 4, 8), 0, true)", OK),
    ("check_array(A(0, 0, 8), 8, true)", OK), ("check_array(A(4098, 4, 8), 8, true)", ARG), ("check_array(A(4096, 4, 7), 8, true)", SHAPE),
    ("check_array(A(4096, 4, 1LL << 41), 8, true)", SHAPE), ("check_array(A(4096, 1LL << 30, 1LL << 40), 8, true)", SHAPE),
    # overlaps: apart, the same, the last element shared, columns of one array, the same with a column shared
    ("Status{overlap(A(4096, 4, 8), A(4096 + 128, 4, 8), 8)}", 0), ("Status{overlap(A(4096, 4, 8), A(4096, 4, 8), 8)}", 1),
    ("Status{overlap(A(4096, 4, 8), A(4096 + 124, 4, 8), 8)}", 1), ("Status{overlap(A(4096, 4, 16), A(4096 + 32, 4, 16), 8)}", 0),
    ("Status{overlap(A(4096, 4, 16), A(4096 + 28, 4, 16), 8)}", 1), ("Status{overlap(A(4096 + 32, 4, 16), A(4096, 4, 16), 8)}", 0),
    ("Status{overlap(A(4096, 4, 16), A(4096 + 32, 4, 17), 8)}", 1), ("Status{overlap(A(4096, 4, 16), A(0, 4, 16), 8)}", 0),
    # states: apart, in place, shifted, in place with another ld; an output on the state or on an input
    ("check_overlaps({A(4096, 4, 8)}, {A(8192, 4, 8), A(20480, 2, 8)}, A(16384, 2, 8), A(20480, 2, 8), 8)", OK),
    ("check_overlaps({A(4096, 4, 8)}, {A(8192, 4, 8), A(16384, 2, 8)}, A(16384, 2, 8), A(16384, 2, 8), 8)", OK),
    ("check_overlaps({A(4096, 4, 8)}, {A(8192, 4, 8), A(16388, 2, 8)}, A(16384, 2, 8), A(16388, 2, 8), 8)", ARG),
    ("check_overlaps({A(4096, 4, 8)}, {A(8192, 4, 8), A(16384, 2, 9)}, A(16384, 2, 8), A(16384, 2, 9), 8)", ARG),
    ("check_overlaps({A(4096, 4, 8)}, {A(16384, 4, 8), A(20480, 2, 8)}, A(16384, 2, 8), A(20480, 2, 8), 8)", ARG),
    ("check_overlaps({A(4096, 4, 8)}, {A(4096, 4, 8), A(0, 2, 8)}, A(0, 2, 8), A(0, 2, 8), 8)", ARG),
    ("check_overlaps({A(4096, 4, 8)}, {A(8192, 4, 8), A(8192, 2, 8)}, A(0, 2, 8), A(8192, 2, 8), 8)", ARG),
    # workspaces: none, none where one is needed, too small, not aligned, over an array
    ("check_workspace(nullptr, 0, 64, false, {}, 8)", OK), ("check_workspace(nullptr, 0, 64, true, {}, 8)", ARG),
    ("check_workspace(P(4096), 63, 64, false, {}, 8)", ARG), ("check_workspace(P(4104), 64, 64, false, {}, 8)", ARG),
    ("check_workspace(P(4096), 64, 64, true, {A(4160, 4, 8)}, 8)", OK), ("check_workspace(P(4096), 64, 64, true, {A(4156, 4, 8)}, 8)", ARG),
    ("check_workspace(P(4096), 64, 0, true, {A(4096, 4, 8)}, 8)", OK),
]


def test_checks(tmp_path):
    if not shutil.which("g++"):
        pytest.skip("no C++ compiler")
    src = tmp_path / "checks.cpp"
    body = "\n".join(f"    print({e});" for e, _ in CASES)
    src.write_text(f"""#include <cstdio>
#include "ops_checks.hpp"
namespace rosenna {{
static const void *P(intptr_t p) {{ return reinterpret_cast<const void *>(p); }}
static Array A(intptr_t p, int64_t rows, int64_t ld) {{ return Array{{"a", static_cast<const float *>(P(p)), rows, ld}}; }}
static void print(const Status &s) {{ std::printf("%d\\n", s.code); }}
static void run() {{
{body}
}}
}}
int main() {{ rosenna::run(); }}
""")
    exe = tmp_path / "checks"
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "rosenna_b200", "csrc"), "-o", str(exe), str(src)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    wrong = [(e, c, g) for (e, c), g in zip(CASES, got) if c != g]
    assert len(got) == len(CASES) and not wrong, wrong
