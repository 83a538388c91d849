"""Which operands share memory (genllm_amd/csrc/rows.hpp), against every byte written down."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r'''
#include <cstdio>
#include <random>
#include <set>
#include "rows.hpp"
using namespace genllm;

static std::set<long> bytes(const Rows& r, bool* twice = nullptr) {
    std::set<long> s;
    for (long i = 0; i < r.n[0]; ++i)
        for (long j = 0; j < r.n[1]; ++j)
            for (long k = 0; k < r.n[2]; ++k)
                for (long e = 0; e < r.bytes; ++e) {
                    const long at = reinterpret_cast<long>(r.p) + i * r.stride[0] + j * r.stride[1] + k * r.stride[2] + e;
                    if (!s.insert(at).second && twice) *twice = true;
                }
    return s;
}

int main() {
    std::mt19937 g(1);
    auto pick = [&](long lo, long hi) { return lo + long(g() % (hi - lo + 1)); };
    long seen[2] = {}, self[2] = {};
    for (int t = 0; t < 200000; ++t) {
        Rows r[2];
        const long row = pick(1, 6);
        for (Rows& x : r) {
            x.p = reinterpret_cast<const char*>(1000 + pick(-40, 40));
            x.bytes = pick(0, 12) ? pick(1, row) : 0;
            const int form = pick(0, 3);
            for (int d = 0; d < 3; ++d) x.n[d] = pick(0, 20) ? pick(1, 4) : 0;
            if (form == 0)  // any strides
                for (int d = 0; d < 3; ++d) x.stride[d] = pick(-12, 12);
            else if (form == 1)  // dense, some order
                x.stride[0] = row * 4 * 4, x.stride[1] = row * 4, x.stride[2] = row;
            else if (form == 2)
                x.stride[0] = row * 4 * 4, x.stride[1] = row, x.stride[2] = row * 4;
            else  // rows of a wider tensor
                x.stride[0] = 100, x.stride[1] = 25, x.stride[2] = pick(0, 1) ? row : 2 * row;
            if (t & 1 && &x == r + 1) for (int d = 0; d < 3; ++d) x.stride[d] = r[0].stride[d];
        }
        const std::set<long> a = bytes(r[0]), b = bytes(r[1]);
        bool want = false, twice = false;
        for (long x : a) want |= b.count(x) != 0;
        if (rows_shared(r[0], r[1]) != want || rows_shared(r[1], r[0]) != want) return printf("pair %d: %d\n", t, want), 1;
        const NamedRows one[] = {{"a", r[0]}}, two[] = {{"b", r[1]}};
        const char *x, *y;
        if (find_overlap(one, two, [](const Rows&, const Rows&) { return false; }, x, y) != want) return printf("named %d\n", t), 1;
        bytes(r[0], &twice);
        if (rows_shared_within(r[0]) != twice) return printf("rows %d: %d\n", t, twice), 1;
        ++seen[want], ++self[twice];
    }
    if (seen[0] < 1000 || seen[1] < 1000 || self[0] < 1000 || self[1] < 1000) return 2;
    // sizes in earnest: channels of one projection, 4 sequences of 8192 tokens, and a pair one row apart
    Rows q, o;
    q.p = reinterpret_cast<const char*>(1 << 20), q.bytes = 256;
    q.n[0] = 4, q.n[1] = 8192, q.n[2] = 16, q.stride[0] = 8192l * 16384, q.stride[1] = 16384, q.stride[2] = 256;
    o = q, o.p += 4096, o.n[2] = 32;
    if (rows_shared(q, o) || rows_shared_within(q)) return 3;
    o.p -= 1;
    if (!rows_shared(q, o)) return 4;
    o = q, o.p += 16384 - 256;
    if (!rows_shared(q, o)) return 5;
    // heads of one buffer in head order, every other head
    q.stride[0] = 32l * 8192 * 256, q.stride[1] = 256, q.stride[2] = 2l * 8192 * 256;
    o = q, o.p += 8192 * 256;
    if (rows_shared(q, o)) return 6;
    o.n[1] = 8193;
    if (!rows_shared(q, o)) return 7;
    // strides near the ends of 64 bits
    q.stride[0] = INT64_MAX / 2, q.stride[1] = -(INT64_MAX / 4), q.n[0] = q.n[1] = INT32_MAX;
    rows_shared(q, o), rows_shared_within(q);
    puts("as written down");
}
'''


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ builds the program")
def test_against_every_byte(tmp_path):
    src, exe = tmp_path / "rows.cpp", tmp_path / "rows"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-I" + os.path.join(ROOT, "genllm_amd", "csrc"), str(src),
                    "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "as written down" in r.stdout, (r.returncode, r.stdout)
