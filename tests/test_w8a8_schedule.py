"""The order in which the int8 products' kernels ask for, wait for, read and multiply their steps, run on the host from the
kernels' own lines: those of w8a8.hip between the marks below, compiled with calls in place of the DMAs, reads and products that
keep count of what is where.

A wave's DMAs return in the order in which it issued them; a wait leaves the last N of them on their way.  What has landed and
what has been read is the other waves' to use once this wave has passed a barrier, and one wave's order stands for every wave's."""
import re
import shutil
import subprocess

import pytest

from w8a8_rule import CALLS, CSRC, NAMES, shape

SOURCE = (CSRC / "w8a8.hip").read_text()


def lines(first, last, text=SOURCE):
    a = text.index(first)
    return text[a:text.index(last, a)]


SIZES = lines("    constexpr int NW = WM * WN, FM", "    // the wave's weight rows are permuted")
TILE = lines("    // asked for in the order in which they are waited for", "    // a lane's sums: NO neighbouring outputs")
RING = lines("    const int n = whole > wave ?", "    if (128 * whole < K && wave == whole % NW) {")
TILES = sorted(set(re.findall(r"launch_tiles<(\d+, \d+, \d+, \d+, \d+), GATED>", SOURCE)))
RINGS = sorted(set(re.findall(r"launch_ring<(\d+, \d+, \d+, \d+), \w+, \w+>", SOURCE)))

MODEL = r"""
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <set>
#include <tuple>
#include <vector>
static const char* what = "";
static int at_steps, at_whole;
static void no(const char* why, int s) { std::printf("%s, %d steps, %d whole: %s, step %d\n", what, at_steps, at_whole, why, s); std::exit(1); }

struct Dma { int kind, step, i; };
static std::vector<Dma> issued;
static size_t landed, shared_;                 // of `issued`: waited for by this wave; before its last barrier
static std::vector<std::pair<int, int>> reads; // (kind, step), in order
static size_t returned, passed;                // of `reads`: waited for; before the last barrier
template <int N>
static void vm_left() { if (issued.size() > N) landed = std::max(landed, issued.size() - N); }
static void lds_reads_done() { returned = reads.size(); }
static void barrier() { shared_ = landed; passed = returned; }
#define __builtin_amdgcn_s_barrier barrier
#define __builtin_amdgcn_sched_barrier(x) (void)0
#define BUFFERS(kind) ((kind) ? W_BUFFERS : X_BUFFERS)
static void restart() { issued.clear(), reads.clear(), landed = shared_ = returned = passed = 0; }

struct Frag { int step = -1, kk = -1, h = -1; bool kept = false; };
static Frag keep_bytes(Frag f, int, int) { f.kept = true; return f; }
"""

TILE_RUN = r"""
template <int BM, int BN, int WM, int WN, int S>
static void tile(int steps, int whole) {
%(sizes)s
    constexpr int X_BUFFERS = S, W_BUFFERS = S + 1;
    const int K = whole * BK + (whole < steps ? 5 : 0), quad = 0;
    at_steps = steps, at_whole = whole;
    restart();
    std::map<int, int> held[2];   // buffer -> step
    auto fetch = [&](int kind, int s, int i) {
        if (s >= steps) no("a step past the last is asked for", s);
        const int b = s %% BUFFERS(kind), old = held[kind].count(b) ? held[kind][b] : s;
        if (old != s) {
            for (size_t r = passed; r < reads.size(); ++r)
                if (reads[r] == std::make_pair(kind, old)) no("a buffer is filled while a wave may still read it", s);
            for (size_t d = shared_; d < issued.size(); ++d)
                if (issued[d].kind == kind && issued[d].step == old) no("a buffer is filled twice at once", s);
            int count = 0;
            for (auto& r : reads) count += r == std::make_pair(kind, old);
            if (!count) no("a buffer is filled before it was read", s);
        }
        held[kind][b] = s;
        issued.push_back({kind, s, i});
    };
    auto there = [&](int kind, int s) {   // every DMA of the step, for every wave
        const int b = s %% BUFFERS(kind);
        if (s >= steps || !held[kind].count(b) || held[kind][b] != s) return false;
        std::set<int> in;
        for (size_t d = 0; d < shared_; ++d)
            if (issued[d].kind == kind && issued[d].step == s) in.insert(issued[d].i);
        return (int)in.size() == (kind ? NB : NX);
    };
    auto fetch_x = [&](int s, int i) { fetch(0, s, i); };
    auto fetch_w = [&](int s, int i) { fetch(1, s, i); };
    Frag x[2][FM], w[2][JH];
    auto read_x = [&](int s, int kk) {
        for (int i = 0; i < FM; ++i) x[kk][i] = {there(0, s) ? s : -1, kk};
        reads.push_back({0, s});
    };
    auto read_w = [&](int s, int kk, int h, Frag (&to)[JH]) {
        for (int j = 0; j < JH; ++j) to[j] = {there(1, s) ? s : -1, kk, h};
        reads.push_back({1, s});
    };
    std::set<std::tuple<int, int, int, int>> done;
    auto multiply = [&](int kk, int h, int j, const Frag (&wj)[JH]) {
        const Frag f = wj[j];
        if (f.step < 0 || f.kk != kk || f.h != h) no("weights that are not there are multiplied", f.step);
        for (int i = 0; i < FM; ++i) {
            const Frag g = x[kk][i];
            if (g.step != f.step || g.kk != kk) no("tokens that are not there are multiplied", f.step);
            if (g.kept != (f.step >= whole)) no("a cut step's tokens are cleared, no other's", f.step);
        }
        if (!done.insert({f.step, kk, h, j}).second) no("a product is taken twice", f.step);
    };
%(tile)s
    if ((int)done.size() != steps * 2 * NH * JH) no("products are missing", steps);
    if ((int)issued.size() != steps * (NX + NB)) no("DMAs are missing", steps);
    if (landed != issued.size()) no("DMAs are on their way at the end", steps);
}
"""

RING_RUN = r"""
template <int TT, int WT, int U, int NW>
static void ring(int whole) {
    constexpr int NI = 2 * (TT + WT);
    at_steps = at_whole = whole;
    std::set<int> all;
    for (int wave = 0; wave < NW; ++wave) {
        restart();
        int held[U];
        std::fill(held, held + U, -1);
        std::vector<int> order;
        auto fetch = [&](int unit, int u) {
            if (unit >= whole) no("a unit past the last is asked for", unit);
            if (held[u] >= 0) {
                if (std::find(order.begin(), order.end(), held[u]) == order.end()) no("a slot is filled before it was read", unit);
                if (returned != reads.size()) no("a slot is filled while the wave still reads it", unit);
            }
            held[u] = unit;
            for (int i = 0; i < NI; ++i) issued.push_back({0, unit, i});
        };
        auto multiply = [&](int u) {
            int in = 0;
            for (size_t d = 0; d < landed; ++d) in += issued[d].step == held[u];
            if (held[u] < 0 || in != NI) no("a unit that is not there is multiplied", held[u]);
            reads.push_back({0, held[u]});
            order.push_back(held[u]);
            if (!all.insert(held[u]).second) no("a unit is taken twice", held[u]);
        };
%(ring)s
        if (landed != issued.size()) no("DMAs are on their way at the end", whole);
    }
    if ((int)all.size() != whole) no("units are missing", whole);
}
"""

# an order that is wrong, made from the kernels' lines: (what is changed, into what)
MISTAKES = [("vm_left<(S - 1) * (NX + NB) + NB>();", "vm_left<(S - 1) * (NX + NB) + NB + 1>();"),
            ("vm_left<(S - 2) * NX + (S - 1) * NB>();", "vm_left<(S - 2) * NX + (S - 1) * NB + 1>();"),
            ("        vm_left<0>();\n    arrive();", "        vm_left<1>();\n    arrive();"),
            ("                    vm_left<0>();", "                    vm_left<1>();"),
            ("        lds_reads_done();\n        __builtin", "        __builtin"),
            ("                arrive();\n", ""),
            ("if (q == 0 && s > 0 && s + S < steps)", "if (q == 0 && s > 0 && s + S + 1 < steps)"),
            ("fetch_w(s + S, i);", "fetch_w(s + S + 1, i);"),
            ("if (q == NQ - 1 && s + S < steps)", "if (q == 0 && s + S < steps)"),
            ("if (nh == 0) read_x(s, nk);", "if (nh == 1) read_x(s, nk);"),
            ("x[kk][i] = keep_bytes", "if (kk) x[kk][i] = keep_bytes"),
            ("if (i + U <= n)", "if (i + U <= n + 1)"),
            ("vm_left<(U - 1) * NI>();", "vm_left<U * NI>();"),
            ("        lds_reads_done();   // before", "        // before"),
            ("u = u + 1 == U ? 0 : u + 1;", "u = u + 1 == U ? 0 : u + 2;")]


def run(tmp_path, tile=TILE, ring=RING):
    """What the model finds in the kernels' lines ("" where all is well)."""
    sizes = re.sub(r"static_assert\(.*?\);\n", "", SIZES, flags=re.S)
    calls = "".join(f'    what = "tile {t}";\n    for (int s = 1; s <= 13; ++s) tile<{t}>(s, s), tile<{t}>(s, s - 1);\n' for t in TILES)
    calls += "".join(f'    what = "ring {r}";\n    for (int s = 0; s <= 70; ++s) ring<{r}>(s);\n' for r in RINGS)
    src, exe = tmp_path / "order.cpp", tmp_path / "order"
    src.write_text(MODEL + TILE_RUN % dict(sizes=sizes, tile=tile) + RING_RUN % dict(ring=ring) + "int main() {\n" + calls + "}\n")
    subprocess.run([shutil.which("g++") or "c++", "-std=c++17", "-O1", "-w", "-o", str(exe), str(src)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode in (0, 1), r
    return r.stdout.strip()


def test_every_step_is_there_when_it_is_read(tmp_path):
    assert len(TILES) == 5 and len(RINGS) >= 5
    assert run(tmp_path) == ""


@pytest.mark.parametrize("old,new", MISTAKES)
def test_the_model_sees_a_mistake(tmp_path, old, new):
    assert TILE.count(old) + RING.count(old) == 1
    assert run(tmp_path, TILE.replace(old, new), RING.replace(old, new)) != ""


def test_buffers_go_round_alike():
    """The model's buffers are the kernel's: steps modulo S for the tokens and S + 1 for the weights, where they are filled and
    where they are read."""
    for call in ("fetch_x", "read_x"):
        assert "(s % S) * (BM * BK)" in lines(f"auto {call} = ", "};"), call
    for call in ("fetch_w", "read_w"):
        assert "(s % (S + 1)) * (BN * BK)" in lines(f"auto {call} = ", "};"), call
    assert "(u * kSlot + i * 1024)" in lines("auto fetch = ", "};") and lines("auto multiply = ", "};").count("mine + u * kSlot") == 2


def test_every_shape_has_its_calls():
    """tests/test_gpu_w8a8_shapes.py runs each shape: the calls that it is given are those that the rule sends there."""
    for name, tokens, n_in, outputs, gated in CALLS:
        assert shape(tokens, n_in, outputs, gated) == name
    assert {(c[0], c[4]) for c in CALLS} == {(n, g) for n in NAMES for g in (False, True)}
