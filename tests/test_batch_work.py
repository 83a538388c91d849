"""How paged_attention_batch divides a batch among workgroups (genllm_amd/csrc/batch_work.hpp): the device code run on
the CPU, 64 lanes of a wave taking turns at each move between lanes, against units counted key by key."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r'''
#include <setjmp.h>
#include <ucontext.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <functional>
#include <map>
#include <random>
#include <vector>

// ---- a wave: a lane runs until it needs the others' values
static ucontext_t g_start[64], g_main;
static jmp_buf g_lane[64], g_all;
static std::vector<char> g_stack[64];
static int64_t g_box[2][64];
static int g_now, g_phase[64];
static bool g_begun[64], g_done[64];
static std::function<void()>* g_body;
struct Index { int x = 0; };
static Index threadIdx;

static const int64_t* exchange(int64_t x) {
    const int lane = g_now, at = g_phase[lane] & 1;
    g_box[at][lane] = x;
    ++g_phase[lane];
    if (!_setjmp(g_lane[lane])) _longjmp(g_all, 1);
    return g_box[at];
}
static void lane_main() {
    (*g_body)();
    g_done[g_now] = true;
    _longjmp(g_all, 1);
}
static void wave(std::function<void()> body) {
    g_body = &body;
    for (int i = 0; i < 64; ++i) g_begun[i] = g_done[i] = false, g_phase[i] = 0;
    for (;;) {
        for (g_now = 0; g_now < 64; ++g_now) {
            threadIdx.x = g_now;
            if (_setjmp(g_all)) continue;
            if (g_begun[g_now]) _longjmp(g_lane[g_now], 1);
            g_begun[g_now] = true;
            g_stack[g_now].resize(1 << 16);
            getcontext(&g_start[g_now]);
            g_start[g_now].uc_stack.ss_sp = g_stack[g_now].data();
            g_start[g_now].uc_stack.ss_size = g_stack[g_now].size();
            g_start[g_now].uc_link = nullptr;
            makecontext(&g_start[g_now], lane_main, 0);
            swapcontext(&g_main, &g_start[g_now]);
        }
        int done = 0;
        for (int i = 0; i < 64; ++i) {
            if (g_phase[i] != g_phase[0]) puts("lanes apart"), exit(9);
            done += g_done[i];
        }
        if (done == 64) return;
        if (done) puts("lanes end apart"), exit(9);
    }
}

// ---- what the device code uses
#define __device__
#define __forceinline__ inline
using std::max;
using std::min;
static int __builtin_amdgcn_readlane(int x, int lane) { return int(exchange(x)[lane]); }
static int __builtin_amdgcn_readfirstlane(int x) { return int(exchange(x)[0]); }
static unsigned long long __ballot(bool x) {
    const int64_t* all = exchange(x);
    unsigned long long r = 0;
    for (int i = 0; i < 64; ++i) r |= (unsigned long long)(all[i] != 0) << i;
    return r;
}
static float __builtin_amdgcn_rcpf(float x) { return std::nextafterf(1.0f / x, 2.0f); }  // off by a unit in the last place
// row_shr by 1 to 15, and a row's or two rows' last lane to the lanes behind; `old` where there is no source
static int __builtin_amdgcn_update_dpp(int old, int x, int ctrl, int rows, int, bool) {
    const int lane = g_now, row = lane >> 4;
    const int64_t* all = exchange(x);
    if (!(rows >> row & 1)) return old;
    if (ctrl >= 0x111 && ctrl <= 0x11f) return (lane & 15) >= ctrl - 0x110 ? int(all[lane - (ctrl - 0x110)]) : old;
    if (ctrl == 0x142) return row ? int(all[16 * row - 1]) : old;
    if (ctrl == 0x143) return row >= 2 ? int(all[31]) : old;
    puts("dpp"), exit(9);
}
namespace genllm {
constexpr int kPage = 16;
}
#include "batch_work.hpp"
using namespace genllm;

struct Batch {
    BatchSizes z;
    std::vector<int32_t> n, ql;
    int window = 0, sinks = 0;
    bool causal = true, huge = false;
};

// steps of each unit's tile: pages with a key that some row sees
static int64_t steps_of(const Batch& c, int b, int64_t tile, const BatchPlan& plan) {
    const int64_t G = c.z.n_q_heads / c.z.n_kv_heads, n = std::min<int64_t>(std::max(c.n[b], 0), int64_t(c.z.max_pages) * 16);
    const int64_t ql = std::min(std::max(c.ql[b], 0), c.z.seq_len), first = tile * plan.rows, last = std::min(first + plan.rows, ql * G) - 1;
    if (last < first) return -1;
    const int64_t p0 = n - ql + first / G, p1 = c.causal ? std::min(n - ql + last / G, n - 1) : n - 1;
    int64_t pages = 0;
    if (!c.window) {
        pages = (p1 + 16) / 16;
    } else {
        for (int64_t page = 0; 16 * page <= p1; ++page) {
            bool seen = false;
            for (int64_t t = 16 * page; t < 16 * page + 16 && t <= p1; ++t) seen |= t < c.sinks || t > p0 - c.window;
            pages += seen;
        }
    }
    return (std::max<int64_t>(pages, 0) + plan.step - 1) / plan.step;
}

template <int ROWS, int STEP>
static bool find(const BatchAttn& p, int w, Work& r) {
    bool found = false;
    Work of[64];
    bool is[64];
    wave([&] { const int lane = g_now; is[lane] = find_work<ROWS, STEP>(p, w, of[lane]); });
    for (int i = 0; i < 64; ++i)
        if (is[i] != is[0] || (is[0] && (of[i].b != of[0].b || of[i].tile != of[0].tile || of[i].sp != of[0].sp || of[i].h != of[0].h ||
                                         of[i].ns != of[0].ns || of[i].base != of[0].base || of[i].e.n != of[0].e.n || of[i].e.ql != of[0].e.ql)))
            puts("lanes differ"), exit(8);
    found = is[0], r = of[0];
    return found;
}

static int check(const char* name, const Batch& c) {
    if (c.z.refused() || c.z.empty()) return printf("%s: refused\n", name), 1;
    const BatchPlan plan = plan_of(c.z);
    if (plan.slots > kMostWorkgroups) return printf("%s: too many\n", name), 1;
    BatchAttn p;
    p.n_cached = c.n.data(), p.q_lens = c.ql.data(), p.B = c.z.batch, p.S = c.z.seq_len, p.Hq = c.z.n_q_heads, p.Hkv = c.z.n_kv_heads;
    p.G = p.Hq / p.Hkv, p.capacity = c.z.max_pages * 16, p.window = c.window ? std::min(c.window, kNoWindow) : kNoWindow, p.sinks = c.sinks;
    p.causal = c.causal, p.tiles_max = int(plan.tiles_max), p.target = plan.target, p.least = plan.least, p.can_split = plan.can_split;
    p.paired = plan.paired && c.causal, p.slots = int(plan.slots);
    // every unit with rows, its steps in ns pieces, each kv head: once
    std::map<std::pair<int, int>, int> splits;
    std::map<std::vector<int>, int> seen;
    int64_t found = 0, longest = 0, whole = 0;
    const int64_t upto = plan.slots + 3;  // none behind the last
    for (int64_t w = 0; w < upto; ++w) {
        Work r;
        const bool any = plan.decode ? find<16, kDecodeStep>(p, int(w), r)
                         : plan.rows == 64 ? find<64, kPrefillStep>(p, int(w), r) : find<128, kPrefillStep>(p, int(w), r);
        if (!any) continue;
        if (w >= plan.slots) return printf("%s: workgroup %ld has work\n", name, long(w)), 1;
        ++found;
        const int64_t steps = steps_of(c, r.b, r.tile, plan);
        if (steps < 0) return printf("%s: entry %d has no tile %d\n", name, r.b, r.tile), 1;
        if (r.e.n != std::min<int64_t>(std::max(c.n[r.b], 0), p.capacity) || r.e.ql != std::min(std::max(c.ql[r.b], 0), p.S)) return printf("%s: lengths\n", name), 1;
        if (r.sp < 0 || r.sp >= r.ns || r.h < 0 || r.h >= p.Hkv) return printf("%s: split %d of %d, head %d\n", name, r.sp, r.ns, r.h), 1;
        if (plan.can_split && (r.base + int64_t(r.sp) * p.Hkv + r.h != w || r.unit != r.b * p.tiles_max + r.tile)) return printf("%s: base\n", name), 1;
        if (!plan.can_split && r.ns != 1) return printf("%s: split\n", name), 1;
        // partials, and what the merge reads of them, lie in the workspace
        if (plan.can_split && (r.base < 0 || r.base + int64_t(r.ns) * p.Hkv > plan.slots)) return printf("%s: %d pieces from %d, %ld places\n", name, r.ns, r.base, long(plan.slots)), 1;
        const auto at = std::make_pair(r.b, r.tile);
        if (splits.count(at) && splits[at] != r.ns) return printf("%s: pieces differ\n", name), 1;
        splits[at] = r.ns;
        if (++seen[{r.b, r.tile, r.h, r.sp}] > 1) return printf("%s: work done twice\n", name), 1;
        longest = std::max(longest, (steps + r.ns - 1) / r.ns);
        whole = std::max(whole, steps);
    }
    int64_t want = 0, sum = 0;
    for (int b = 0; b < c.z.batch; ++b)
        for (int64_t t = 0; t < plan.tiles_max; ++t) {
            const int64_t steps = steps_of(c, b, t, plan);
            if (steps < 0) continue;
            if (!splits.count({b, int(t)})) return printf("%s: entry %d tile %ld left out\n", name, b, long(t)), 1;
            want += int64_t(splits[{b, int(t)}]) * p.Hkv, sum += steps * p.Hkv;
        }
    if (want != found) return printf("%s: %ld of %ld\n", name, long(found), long(want)), 1;
    // no piece is longer than twice an equal share, or than two of the least
    if (plan.can_split && longest > std::max<int64_t>(2 * plan.least, 2 * ((sum + plan.target - 1) / plan.target))) return printf("%s: a piece of %ld steps\n", name, long(longest)), 1;
    printf("%s: %ld workgroups, tiles of %d, split %d, longest %ld of %ld steps\n", name, long(found), plan.rows, plan.can_split, long(longest), long(whole));
    return 0;
}

static Batch batch(int B, int S, int Hq, int H, int D, int P, std::vector<int32_t> n, std::vector<int32_t> ql = {}) {
    Batch c;
    c.z = {B, S, Hq, H, D, P};
    c.n = n, c.ql = ql;
    while (int(c.n.size()) < B) c.n.push_back(c.n[c.n.size() - n.size()]);
    while (int(c.ql.size()) < B) c.ql.push_back(ql.empty() ? S : c.ql[c.ql.size() - ql.size()]);
    return c;
}

int main(int argc, char** argv) {
    const std::string what = argv[1];
    if (what == "batches") {
        Batch c = batch(8, 1, 32, 8, 128, 512, {1, 0, 8192, 17, 300, -5, 1 << 30, 16});
        if (check("tokens", c)) return 1;
        c.window = 700, c.sinks = 20;
        if (check("tokens in windows", c)) return 1;
        c = batch(3, 1, 4, 1, 64, 6, {96, 3, 0});
        if (check("short tables", c)) return 1;
        c = batch(150, 2, 8, 2, 64, 80, {1280, 3, 70, 0, 500}, {2, 0, 1});
        if (check("more entries than lanes", c)) return 1;
        c = batch(100, 2, 16, 1, 64, 200, {3200, 40, 17, 1000, 0, 2}, {2, 1, 0, 2});
        if (check("more units than lanes, tiles of 64", c)) return 1;
        c = batch(20, 130, 4, 1, 128, 100, {1600, 130, 600, 5}, {130, 130, 1, 5, 0});
        if (check("more units than lanes, tiles of 128", c)) return 1;
        c.window = 200, c.sinks = 30;
        if (check("windows, tiles of 128", c)) return 1;
        c = batch(2, 300, 6, 2, 256, 90, {1400, 310}, {300, 11});
        if (check("chunks", c)) return 1;
        c.causal = false;
        if (check("all keys", c)) return 1;
        c = batch(1, 2048, 16, 8, 128, 128, {2048});
        if (check("a prompt", c)) return 1;
        c = batch(64, 64, 8, 2, 128, 256, {64, 1, 1, 4096}, {64, 1, 1, 1});
        if (check("a chunk among tokens", c)) return 1;
        std::mt19937 g(1);
        auto pick = [&](int lo, int hi) { return lo + int(g() % unsigned(hi - lo + 1)); };
        for (int i = 0; i < 40; ++i) {
            const int G = pick(1, 8), H = pick(1, 4), B = pick(1, 90), S = pick(0, 2) ? pick(1, 16 / G + 2) : pick(1, 4000 / (B * G) + 1), D = 64 << pick(0, 2), P = pick(1, 300);
            c = batch(B, S, G * H, H, D, P, {0});
            for (int b = 0; b < B; ++b) c.n[b] = pick(0, 16 * P + 5), c.ql[b] = pick(0, S);
            if (pick(0, 1)) c.window = pick(1, 900), c.sinks = pick(0, 60);
            if (check("drawn", c)) return 1;
        }
    } else if (what == "long") {
        // the ends of what tables hold, for few rows (steps of two pages) and for more (of four)
        const int all = 1 << 26;
        if (check("one entry short of 2^24 steps", batch(1, 1, 1, 1, 64, all, {(1 << 29) - 32}))) return 1;
        if (check("one entry of 2^24 steps", batch(1, 1, 1, 1, 64, all, {1 << 29}))) return 1;
        if (check("one entry of the table", batch(1, 1, 1, 1, 64, all, {1 << 30}))) return 1;
        if (check("entries of the table", batch(5, 2, 6, 2, 256, all, {1 << 30, (1 << 29) + 40, 17, INT32_MAX, 5}))) return 1;
        if (check("a wave of entries", batch(64, 1, 4, 1, 128, all, {1 << 30}))) return 1;
        if (check("more than a wave of entries", batch(70, 1, 4, 1, 128, all, {1 << 30, 1 << 29, 300}))) return 1;
        if (check("tiles of 64", batch(2, 20, 1, 1, 64, all, {1 << 30, 90}))) return 1;
        if (check("tiles of 128", batch(1, 600, 1, 1, 128, all, {1 << 30}))) return 1;
    }
    if (what == "quotients") {
        // x up to 2^30 and a tile, by any divisor, the reciprocal off by a unit in the last place either way
        std::mt19937 g(2);
        const auto one = [](int64_t x, int64_t d) {
            if (x < 0 || x > (int64_t(1) << 30) + 128 || d < 1 || d > 1 << 30) return 0;
            for (float r : {1.0f / float(d), std::nextafterf(1.0f / float(d), 0.0f), std::nextafterf(1.0f / float(d), 2.0f)}) {
                Divisor by{int(d)};
                by.r = r;
                if (by(int(x)) != x / d) return printf("%ld / %ld is not %d\n", long(x), long(d), by(int(x))), 1;
            }
            return 0;
        };
        for (int i = 0; i < 3000000; ++i) {
            const int64_t d = 1 + (g() & ((1u << (1 + g() % 30)) - 1)), x = int64_t(g() & ((1u << (1 + g() % 31)) - 1));
            if (one(x, d) || one(x / d * d, d) || one(x / d * d - 1, d) || one(x / d * d + d - 1, d)) return 1;
        }
        for (int64_t d = 1; d < 5000; ++d)
            for (int64_t x : {int64_t(1) << 30, (int64_t(1) << 30) + 128, (int64_t(1) << 30) / d * d, (int64_t(1) << 30) / d * d - 1, d - 1, d, d + 1})
                if (one(x, d)) return 1;
    }
    puts("as counted");
}
'''


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    at = tmp_path_factory.mktemp("work")
    (at / "work.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-O2", "-std=c++20", "-Wall", "-Wno-parentheses", "-Wno-unused-function", "-Wno-unknown-pragmas", "-fno-strict-aliasing", "-U_FORTIFY_SOURCE",
                    "-I" + os.path.join(ROOT, "genllm_amd", "csrc"), str(at / "work.cpp"), "-o", str(at / "work")], check=True)
    return str(at / "work")


def workspace(*sizes):
    from genllm_amd import _lib

    return _lib.lib().genllm_paged_attention_batch_workspace_bytes(*sizes)


def run(program, what):
    r = subprocess.run([program, what], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.endswith("as counted\n"), (r.returncode, r.stdout[-2000:], r.stderr[-500:])


pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="g++ builds the program")


def test_batches(program):
    run(program, "batches")


def test_quotients(program):
    run(program, "quotients")


def test_tables_of_many_pages(program):
    """Contexts up to the 2^30 tokens that a table holds: the sum of the steps keeps all its bits, so that the pieces
    stay in the workspace."""
    run(program, "long")


@pytest.mark.parametrize("Hq,H", [(2 ** 31 - 1, 2 ** 31 - 1), (2 ** 30, 2 ** 30), (2 ** 31 - 2, 2 ** 30 - 1)])
@pytest.mark.parametrize("B,S", [(2 ** 31 - 1, 300), (2 ** 31 - 1, 5), (2 ** 31 - 1, 1), (2 ** 30, 33), (2 ** 24, 2 ** 20)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("P", [0, 100, 1 << 26])
def test_more_tiles_than_64_bits_count(B, S, Hq, H, D, P):
    """Sizes whose product leaves 64 bits are refused like others of more rows than a launch takes: no workspace."""
    assert workspace(B, S, Hq, H, D, P) == 0


def test_attention_refuses_more_tiles_than_64_bits_count():
    from test_batch_refusals import attend, refused, INV

    big = 2 ** 31 - 1
    for B, S in ((big, 300), (big, 1), (2 ** 30, 300)):
        refused(attend(B=B, S=S, Hq=big, H=big, qb=0, ob=0, kis=0, vis=0, kph=0, vph=0), INV, b"one launch")
