"""How the work of an attention over an 8-bit cache is laid out (csrc/cache8_rules.h), walked over sizes on the CPU: the waves that have a row tile's keys
take each of its tiles once and none behind the last, every row tile has a workgroup, and shares are written by kernels that write them."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton_amd", "csrc")
WALK = r"""
#include <cstdio>
#include <initializer_list>
#include "cache8_rules.h"
using namespace trn;
static long bad = 0, plans = 0, fewer = 0;
static void look(int batch, int kv, int cap, int d, int hq, int sq, bool weights) {
    const Plan8 p = plan8(batch, kv, cap, d, hq, sq, weights);
    int nq = 0, ks = 0; bool past = false, fine = false;
    with_kernel8(p, [&](auto a, auto b, auto c, auto d) { nq = a; ks = b; past = c; fine = d; });
    ++plans;
    fewer += ks < 4;
    bool ok = nq == p.nq && ks == p.ks && past == (p.n_rt == 1) && fine == p.fine && (int64_t)p.n_rt * 16 * nq >= p.R && p.ns >= 1 && p.ns <= 64 && (p.n_rt - 1) * 16 * nq < p.R;
    ok = ok && (ks == 4 || nq == 2) && (ks > 1 || p.ns == 1) && (p.sp == 0 || (p.n_rt == 1 && p.R <= 16));
    // the tiles of 32 keys that a wave takes (those of all waves one after the other), of caches from none to all
    const int most = (cap + 31) / 32, waves = ks * p.ns;
    for (int T : {0, 1, 2, most / 3, most - 1, most}) {
        int64_t at = 0;
        for (int w = 0; w < waves; ++w) {
            const int64_t t0 = (int64_t)T * w / (p.ks * p.ns), t1 = (int64_t)T * (w + 1) / (p.ks * p.ns);
            ok = ok && t0 == at && t1 >= t0;
            at = t1;
        }
        ok = ok && at == T && (int64_t)T * waves <= 0x7fffffff;
    }
    // row tiles of the workgroups, 4 / ks each, from the last on
    const int per = 4 / ks, groups = (p.n_rt + per - 1) / per;
    ok = ok && (p.n_rt - 1) / per - (groups - 1) == 0;
    // the workspace's parts
    const int64_t heads = (int64_t)batch * kv, units = heads * p.n_rt;
    if (p.ns > 1) ok = ok && p.ml >= units * p.ns * 16 * nq * d * 4 && p.lse2 - p.ml >= units * p.ns * 16 * nq * 8;
    if (weights) {
        ok = ok && p.more - p.lse2 >= heads * p.R * 4;
        if (p.sp) ok = ok && p.sp >= cap && p.bytes - p.more >= heads * p.R * p.sp * 4;
        else ok = ok && (int64_t)p.n_chunks * p.chunk_tiles * 32 >= p.R && (p.n_chunks == 1 || p.bytes - p.more >= p.n_chunks * heads * cap * 4);
    }
    if (!ok && bad++ < 8)
        std::printf("batch %d, %d heads on %d of %d, %d queries, capacity %d: tiles of %d rows, %d of them, plan of %d waves, kernel of %d, %d shares\n", batch, hq, kv, d, sq, cap, 16 * nq,
                    p.n_rt, p.ks, ks, p.ns);
}
int main() {
    for (int d = 64; d <= 128; d += 64)
        for (int batch : {1, 2, 3, 7, 16, 32, 43, 48, 87, 88, 96, 160, 320, 350, 701, 2560, 3000})
            for (int kv : {1, 2, 3, 8, 16})
                for (int g : {1, 3, 4, 8, 71})
                    for (int sq : {1, 2, 3, 4, 5, 6, 8, 9, 16, 17, 20, 32, 33, 100, 512, 2047})
                        for (int cap : {1, 31, 33, 600, 1000, 1501, 4096, 13000, 131072, 1 << 26})
                            for (int w = 0; w < 2; ++w) look(batch, kv, cap, d, g * kv, sq, w);
    std::printf("%ld plans, %ld of fewer waves a row tile, %ld wrong\n", plans, fewer, bad);
    return bad != 0;
}
"""


def test_every_plan_covers_its_work_once(tmp_path):
    src, exe = tmp_path / "walk.cpp", tmp_path / "walk"
    src.write_text(WALK)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
    plans, fewer = int(r.stdout.split()[0]), int(r.stdout.split(", ")[1].split()[0])
    assert plans > 100000 and fewer > 1000, r.stdout
