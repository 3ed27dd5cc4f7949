"""Whether two strided tensors share memory (csrc/extent.h), against marking the bytes that each covers: exact for tensors of the same strides that are nested
(packed caches among them), never missed for others."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton_amd", "csrc")
COUNT = r"""
#include <algorithm>
#include <cstdio>
#include <cstring>
#include <random>
#include "extent.h"
using namespace trn;
static char mem[1 << 14], mark[1 << 14];
template <class F> static void each(const Extent& e, F f) {
    for (int64_t i = 0; i < e.n[0]; ++i) for (int64_t j = 0; j < e.n[1]; ++j) for (int64_t k = 0; k < e.n[2]; ++k) for (int64_t w = 0; w < e.width; ++w)
        f((const char*)e.p + i * e.st[0] + j * e.st[1] + k * e.st[2] + w - mem);
}
int main() {
    std::mt19937 rng(3);
    auto draw = [&](int lo, int hi) { return (int64_t)(lo + (int)(rng() % (unsigned)(hi - lo + 1))); };
    long missed = 0, wrong = 0, shared = 0, packed = 0;
    for (int t = 0; t < 200000; ++t) {
        Extent x{}, y{};
        x.width = draw(1, 5); y.width = draw(0, 1) ? x.width : draw(1, 5);
        const bool nested = draw(0, 3) != 0;
        int order[3] = {0, 1, 2};
        for (int i = 2; i > 0; --i) std::swap(order[i], order[draw(0, i)]);
        int64_t all = 5;
        for (int a : order) {       // from the innermost axis out
            x.n[a] = draw(1, 4); y.n[a] = draw(0, 1) ? x.n[a] : draw(1, 4);
            x.st[a] = y.st[a] = nested ? all + draw(0, 6) + (draw(0, 3) ? 0 : all) : draw(0, 40);
            if (!nested && draw(0, 1)) y.st[a] = draw(0, 40);
            if (x.n[a] == 1 && draw(0, 1)) x.st[a] = draw(0, 40);           // (of one element any stride)
            if (y.n[a] == 1 && draw(0, 1)) y.st[a] = draw(0, 40);
            const int64_t st = x.n[a] == 1 ? y.st[a] : x.st[a];
            all += 4 * (st > 0 ? st : 0);
        }
        if (x.span() > 8000 || y.span() > 8000) continue;
        x.p = mem + draw(0, 8000); y.p = mem + (draw(0, 1) ? draw(0, 8000) : std::min<int64_t>(8000, (const char*)x.p - mem + draw(0, 60)));
        std::memset(mark, 0, sizeof mark);
        bool truth = false;
        each(x, [&](int64_t i) { mark[i] = 1; });
        each(y, [&](int64_t i) { truth = truth || mark[i]; });
        const bool said = meet(x, y);
        shared += truth;
        missed += truth && !said;
        if (nested) {
            wrong += said != truth;
            packed += !truth && !apart(x.p, x.span(), y.p, y.span());
        }
    }
    std::printf("%ld missed, %ld wrong, %ld shared, %ld packed\n", missed, wrong, shared, packed);
    return missed || wrong;
}
"""


def test_against_counting(tmp_path):
    src, exe = tmp_path / "count.cpp", tmp_path / "count"
    src.write_text(COUNT)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
    n = [int(w) for w in r.stdout.split() if w.isdigit()]
    assert n[2] > 10000 and n[3] > 5000, r.stdout
