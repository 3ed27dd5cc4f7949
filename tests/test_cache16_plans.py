"""How an attention behind a prefix is shared out where its caches have room: plain host arithmetic."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton_amd", "csrc")

ROOM = r"""
#include <cstdio>
#include <initializer_list>
#include "cache16_rules.h"
using namespace trn;
int main() {
    long bad = 0, plans = 0;
    auto check = [&](bool ok, int batch, int kv, int g, int sq, int d, int pre, int cap) {
        ++plans;
        if (!ok && bad++ < 5) printf("%d sequences, %d x %d heads of %d, %d queries, %d keys behind %d\n", batch, kv, g, d, sq, cap, pre);
    };
    for (int batch : {1, 4, 32, 128}) for (int kv : {1, 2, 8}) for (int g : {1, 4, 71}) for (int sq : {1, 3, 9}) for (int d : {64, 128}) for (int pre : {100, 1000, 8192, 16001}) {
        // from an eighth of the prefix on a larger cache leaves it its workgroups
        const PlanPrefix least = plan_prefix(batch, kv, pre / 8, d, pre, kv * g, sq);
        for (int cap : {pre / 4, pre, 4 * pre, 32 * pre, 1 << 26}) {
            const PlanPrefix p = plan_prefix(batch, kv, cap, d, pre, kv * g, sq);
            if (p.one || least.one) continue;
            check(p.ns_p == least.ns_p && p.first == least.first, batch, kv, g, sq, d, pre, cap);
        }
    }
    // 32 single tokens behind 8192 keys: sixteen shares, however large the cache
    for (int cap : {60, 701, 2048, 8192, 32768, 1 << 20}) check(plan_prefix(32, 8, cap, 128, 8192, 32, 1).ns_p == 16, 32, 8, 4, 1, 128, 8192, cap);
    printf("%ld plans, %ld bad\n", plans, bad);
    return bad != 0 || plans < 1000;
}
"""


def test_room_in_a_cache_leaves_the_prefix_its_workgroups(tmp_path):
    (tmp_path / "room.cpp").write_text(ROOM)
    subprocess.run(["g++", "-O1", "-std=c++17", f"-I{CSRC}", str(tmp_path / "room.cpp"), "-o", str(tmp_path / "room")], check=True)
    r = subprocess.run([str(tmp_path / "room")], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
