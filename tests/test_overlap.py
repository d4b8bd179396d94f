"""Whether strided rows share memory: overlap.hpp compiled for the host, against looking at every pair of rows."""
import os
import subprocess

from conftest import ROOT

CSRC = os.path.join(ROOT, "threedgaussiansplatting.jl_amd", "csrc")

SOURCE = r"""
#include <cstdio>
#include <random>
#include "overlap.hpp"
using namespace tdgs;
struct Raw { int64_t at, rows, step, width; };
static bool slow(const Raw& a, const Raw& b) {
    for (int64_t i = 0; i < a.rows; ++i)
        for (int64_t j = 0; j < b.rows; ++j) {
            const int64_t x = a.at + i * a.step, y = b.at + j * b.step;
            if (a.width > 0 && b.width > 0 && x < y + b.width && y < x + a.width) return true;
        }
    return false;
}
int main() {
    std::mt19937_64 rng(1);
    long wrong = 0, yes = 0, no = 0;
    for (int n = 0; n < 400000; ++n) {
        const int64_t most = n % 2 ? 12 : 60;
        auto raw = [&] {
            Raw r;
            r.rows = rng() % 12;
            r.width = n % 3 ? 1 + rng() % 4 : rng() % most;
            r.step = rng() % 8 == 0 ? 0 : n % 5 ? r.width + rng() % most : rng() % most;
            r.at = 1000 + rng() % (most * 6);
            return r;
        };
        const Raw a = raw();
        Raw b = raw();
        if (n % 4 == 0) b.step = a.step;
        const bool want = slow(a, b);
        const ByteRows x((void*)a.at, a.rows, a.step, a.width), y((void*)b.at, b.rows, b.step, b.width);
        wrong += rows_overlap(x, y) != want || rows_overlap(y, x) != want;
        (want ? yes : no) += 1;
    }
    // large numbers: two columns of rows 2^40 bytes apart, a run next to rows, far progressions that meet once
    const int64_t big = (int64_t)1 << 40;
    ByteRows p((void*)64, 1 << 20, big, 4096), q((void*)(64 + 4096), 1 << 20, big, 4096), r((void*)(64 + 4095), 1 << 20, big, 4096);
    wrong += rows_overlap(p, q) || !rows_overlap(p, r) || rows_overlap(q, ByteRows((void*)(64 + 8192), 1, 0, big - 8192));
    ByteRows u((void*)(1 << 20), 1000003, 1000003, 1), v((void*)(1 << 20), 1000033, 1000033, 1);   // meet at their starts
    ByteRows w((void*)((1 << 20) + 1000003), 1000003, 1000003, 1);
    wrong += !rows_overlap(u, v) || rows_overlap(w, v) || rows_overlap(v, w);                // (next at 1000003 * 1000033)
    ByteRows z((void*)((1 << 20) + 1000003), 1000034, 1000003, 1), v2((void*)(1 << 20), 1000040, 1000033, 1);
    wrong += !rows_overlap(z, v2) || !rows_overlap(v2, z);
    std::printf("%ld %ld %ld\n", wrong, yes, no);
}
"""


DIMS = r"""
#include <algorithm>
#include <cstdio>
#include <random>
#include <set>
#include <vector>
#include "overlap.hpp"
using namespace tdgs;
int main() {
    std::mt19937_64 rng(2);
    long wrong = 0, yes = 0, told = 0, twice = 0;
    for (int n = 0; n < 100000; ++n) {
        int64_t count[2][3], step[2][3], width[2], at[2];
        std::vector<int64_t> bytes[2];
        for (int t = 0; t < 2; ++t) {
            width[t] = 1 + rng() % 3;
            at[t] = 100 + rng() % 150;
            // dimensions in any order, each reaching past those before it, or (one in eight) not
            int order[3] = {0, 1, 2};
            std::shuffle(order, order + 3, rng);
            int64_t inside = width[t];
            for (int i : order) {
                count[t][i] = rng() % 4;
                if (rng() % 2) count[t][i] = std::max<int64_t>(count[t][i], 1);
                step[t][i] = rng() % 8 == 0 ? rng() % (inside + 1) : inside + (rng() % 2 ? 0 : rng() % 9);
                if (count[t][i] > 1) inside += (count[t][i] - 1) * step[t][i];
            }
            for (int64_t i = 0; i < count[t][0]; ++i)
                for (int64_t j = 0; j < count[t][1]; ++j)
                    for (int64_t k = 0; k < count[t][2]; ++k)
                        for (int64_t w = 0; w < width[t]; ++w)
                            bytes[t].push_back(at[t] + i * step[t][0] + j * step[t][1] + k * step[t][2] + w);
        }
        if (n % 8 == 0) at[1] = at[0];
        if (n % 8 == 0) {
            const int64_t move = bytes[1].empty() ? 0 : at[0] - *std::min_element(bytes[1].begin(), bytes[1].end());
            for (int64_t& b : bytes[1]) b += move;
        }
        const ByteDims a((void*)at[0], count[0], step[0], width[0]), b((void*)at[1], count[1], step[1], width[1]);
        const std::set<int64_t> x(bytes[0].begin(), bytes[0].end()), y(bytes[1].begin(), bytes[1].end());
        bool shared = false;
        for (int64_t v : x) shared |= y.count(v) > 0;
        const bool got = dims_overlap(a, b);
        wrong += got != dims_overlap(b, a) || (got && !shared);               // never refused without a reason
        wrong += shared && !got && a.dims <= 1 && b.dims <= 1;                // and always where it can be told
        wrong += !a.none && a.nested && x.size() != bytes[0].size();          // nested: no byte twice
        wrong += !a.same(a) || (a.same(b) && count[0][0] == count[1][0] && count[0][1] == count[1][1] && count[0][2] == count[1][2] &&
                                bytes[0] != bytes[1]);
        yes += shared, told += got, twice += !a.nested;
    }
    std::printf("%ld %ld %ld %ld\n", wrong, yes, told, twice);
}
"""


def run(tmp_path, source):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(source)
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    return [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]


def test_against_every_pair(tmp_path):
    wrong, yes, no = run(tmp_path, SOURCE)
    assert wrong == 0 and yes > 50000 and no > 50000


def test_three_dimensions(tmp_path):
    """Against the bytes one by one: what is refused shares memory; rows of one step are always told; nested tensors hold no
    byte twice; sameness is that of every element's place."""
    wrong, shared, told, twice = run(tmp_path, DIMS)
    assert wrong == 0 and shared > 10000 and told > shared / 2 and twice > 5000
