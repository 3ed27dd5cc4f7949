// How the work of an attention over fp16 caches is laid out (cache_prefix.hip, cache_sparse.hip): plain host arithmetic.
#pragma once
#include <cmath>
#include <cstdint>

namespace trn {

inline int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

// one: wide tiles of each sequence's rows walk over prefix and own keys.  Otherwise rows of all sequences walk over the prefix, in wide tiles or narrow ones, and those of each
// sequence, in narrow ones of 16 nq rows, over its own keys.  n_rt row tiles and ns shares of their keys (_p, _o; one: _p); slots: results of a row to be joined (one: none);
// first, second: workgroups of both parts; ml: offset of the statistics in the workspace, bytes: its size.
// short_rt: row tiles of eight waves each that have all keys, where pitches allow.
// fine: weights as two fp16 numbers in the first of these too (elsewhere always), where a sequence has up to 128 rows a KV head or 512 in all: by its own rows, so that how exact its outputs are does not depend on
// what else is in the batch.  The second number is half as much matrix work again, and the distance from 64 bits 1.0 in the place of 1.4 times that of a computation in 32 bits.  Steps, of a few tokens a
// sequence, are as exact as single tokens; of prompts the matrix pipe is the bound.  us with one number / with two: 32 heads of 128 on 8, 4 x 500 rows behind 4000 keys 136 / 184, 4 x 32 on 4096
// 32.2 / 33.8, 16 x 32 on 2048 40.6 / 43.6; 71 of 64 on 1, 16 x 5 behind 16001 45.7 / 56.4.
struct PlanPrefix { bool one, wide, fine; int short_rt; int G, R, nq, n_rt_p, ns_p, n_rt_o, ns_o, slots; int64_t first, second, ml, bytes; };

inline PlanPrefix plan_prefix(int batch, int n_kv_heads, int capacity, int head_dim, int prefix, int Hq, int Sq) {
    PlanPrefix p{};
    p.G = Hq / n_kv_heads;
    p.R = p.G * Sq;
    const int64_t heads = (int64_t)batch * n_kv_heads, rows_p = (int64_t)batch * p.R;
    // (rows of all sequences fill tiles better than those of each: up to one tile of these, where the prefix is what there is to read.  us by tiles of each / of all, 32 heads of 128 on 8: 16 x 20 rows, 200 keys behind
    // 8192 92.0 / 83.1, 48 x 20, 100 behind 4000 149 / 113, 4 x 20, 500 behind 4000 26.4 / 27.9, 16 x 32 (whole tiles), 200 behind 8192 111 / 123; 71 of 64 on 1, 16 x 1, 200 behind 16000 26.1 / 22.8.)
    p.one = p.R > 64 && !(p.R <= 128 && prefix > 4 * (int64_t)capacity && batch > 1);
    p.fine = p.R <= 128 || (int64_t)Hq * Sq <= 512;
    const int64_t tiles16 = (p.R + 15) / 16;
    // (as long as a wave's tiles, one after the other, take less than a second launch.  One query of 32 heads of 128 on 8, us by shares / by eight waves: one sequence, 60 keys behind 200 9.2 / 6.4, behind
    // 1000 9.7 / 10.4; 8 sequences 12.7 / 10.6, 500 behind 1000 13.3 / 13.5; 32 (wide tiles) 26.8 / 17.0, 60 behind 3000 24.4 / 20.9 before those had shares of 128 keys, 18.7 with them; 16 heads of
    // 64, 4 sequences, 60 behind 1000 8.9 / 7.6, 500 behind 1000 9.1 / 9.0, 60 behind 3000 9.8 / 11.4.)
    const bool shared = prefix > 0 && rows_p > 32;
    const int64_t rounds = (heads * tiles16 + 255) / 256, most = head_dim == 128 ? (shared ? 1800 : 1000) : (shared ? 2500 : 1500);
    if (rounds <= 2 && rounds * ((int64_t)prefix + capacity) <= most) p.short_rt = (int)tiles16;
    if (p.one) {
        p.wide = true; p.nq = 2;
        p.n_rt_p = (p.R + 127) / 128;
        const int64_t units = heads * p.n_rt_p, tiles = ((int64_t)prefix + 63) / 64 + (capacity + 63) / 64;
        int64_t ns = (head_dim == 128 ? 512 : 1024) / units;      // (two workgroups a compute unit, four of head_dim 64: 16 x 5 rows of 71 heads of 64 behind 16001 keys, 48 tiles, 46 to 48 us with 10 to 21 shares, 57 with 22; with weights as two numbers, of which three share one, 57.5 with 21 shares, 58.7 with 16, 60.0 with 10, 65.3 with 17)
        if (ns > tiles / 4) ns = tiles / 4;
        p.ns_p = (int)(ns < 1 ? 1 : ns > 32 ? 32 : ns);
        p.slots = p.ns_p;
        p.first = units * p.ns_p;
    } else {
        p.wide = rows_p > 32;
        p.nq = p.R > 16 || (!p.wide && rows_p > 16) ? 2 : 1;
        p.n_rt_p = (int)(p.wide ? (rows_p + 127) / 128 : (rows_p + 16 * p.nq - 1) / (16 * p.nq));
        p.n_rt_o = (p.R + 16 * p.nq - 1) / (16 * p.nq);
        const int64_t units_p = (int64_t)n_kv_heads * p.n_rt_p, units_o = heads * p.n_rt_o;
        // Workgroups of both parts run at once, two a compute unit: these are shared out by the parts' work (a wide tile's key counts twice), in shares of 256 keys at least, 128 of a wide
        // tile.  There a key takes some 0.012 us beside the other workgroups, and a share more is written and read again, 8 head_dim bytes a row at 4 TB/s: P / ns keys and ns shares take the least time at the root of the ratio.
        // 32 heads of 128 on 8, 32 sequences of 700 keys behind 8192, us with 8 / 16 / 32 shares of the prefix: 31.6 + 4.8 for the joining / 24.9 + 4.8 / 27.6 + 5.9.
        const int64_t cost_p = units_p * prefix * (p.wide ? 2 : 1), cost_o = units_o * capacity, cost = cost_p + cost_o;
        auto shares = [](int64_t groups, int64_t units, int64_t keys, int64_t least) {
            int64_t s = groups / units;
            if (s > (keys + least - 1) / least) s = (keys + least - 1) / least;
            return (int)(keys == 0 ? 0 : s < 1 ? 1 : s > 64 ? 64 : s);
        };
        // (the capacity is what a sequence's own keys may come to: a cache that is to be filled step by step has few at first.  So the prefix's shares are taken as if it held an eighth of the prefix's keys at most;
        // the own keys' divide the keys that are there.  One query of 32 heads of 128 on 8, us by the capacity itself / so: 32 sequences of 701 keys behind 8192, capacity 701 31.7 / 30.8, 2804 38.7 / 30.9, 22432
        // 193.6 / 31.1, full 8192 219 / 206; 4 of 61 behind 1000, 16384 14.8 / 11.5, full 47.4 / 47.1; 1 of 500 behind 8192, 131072 24.5 / 17.2; 128 of 701 behind 4096, 4096 126 / 85; 8 of 4096 behind 8192,
        // full, 34.0 / 35.2.)
        const int64_t cost_least = units_o * (capacity < prefix / 8 ? capacity : prefix / 8);
        p.ns_p = shares(cost_p ? 512 * cost_p / (cost_p + cost_least) : 0, units_p, prefix, p.wide ? 128 : 256);
        if (p.wide && p.ns_p > 1) {
            const int best = (int)std::sqrt(0.012 * prefix / (0.1 + (double)heads * p.R * head_dim * 2e-6));
            if (p.ns_p > best) p.ns_p = best < 1 ? 1 : best;
        }
        p.ns_o = shares(cost ? 512 * cost_o / cost : 0, units_o, capacity, 256);
        if (p.ns_p + p.ns_o == 0) p.ns_o = 1;      // (nothing to see: zeros)
        p.slots = p.ns_p + p.ns_o;
        p.first = units_p * p.ns_p; p.second = units_o * p.ns_o;
    }
    if (p.slots > 1) {
        p.ml = up256(heads * p.R * p.slots * head_dim * 4);
        p.bytes = p.ml + up256(heads * p.R * p.slots * 8);
    }
    return p;
}

// Up to so many blocks a workgroup holds a query's scores in registers.
constexpr int kMostBlocks = 8192;

// Selected blocks: a query's scores in rows of nbp floats, `step` queries of each head at a time; row tiles of 16 nq of a KV head's query heads, ns shares of a query's keys; offsets of
// the shares' parts behind the scores and the norms; rows: a wave a row tile rather than a workgroup.
// dense: all blocks are selected, and the attention is that over the cache, without a prefix.
struct PlanSparse { int G, nb, nq, n_rt, ns, step; bool rows, dense; int64_t nbp, norms, o, ml, bytes; };

inline PlanSparse plan_sparse(int batch, int n_kv_heads, int capacity, int head_dim, int block, int top, int Hq, int Sq) {
    PlanSparse p{};
    p.G = Hq / n_kv_heads;
    p.nb = (capacity + block - 1) / block;
    p.nbp = (p.nb + 63) / 64 * 64;
    const int64_t heads = (int64_t)batch * n_kv_heads, row = heads * p.nbp * 4;
    p.dense = p.nb <= top;
    if (p.dense) {
        p.step = (int)(0xffffff / heads < Sq ? 0xffffff / heads : Sq);
        p.ns = 1;
        p.bytes = plan_prefix(batch, n_kv_heads, capacity, head_dim, 0, Hq, Sq).bytes;
        return p;
    }
    int64_t step = row ? (64 << 20) / row : Sq;
    p.step = (int)(step < 1 ? 1 : step > Sq ? Sq : step);
    p.nq = p.G > 16 ? 2 : 1;
    p.n_rt = (p.G + 16 * p.nq - 1) / (16 * p.nq);
    const int64_t units = heads * Sq * p.n_rt, groups = 512, tiles = (int64_t)(top < p.nb ? top : p.nb) * (block / 32);
    int64_t ns = units ? groups / units : 1;
    if (ns > tiles / 8) ns = tiles / 8;
    p.ns = (int)(ns < 1 ? 1 : ns > 32 ? 32 : ns);
    // (us by workgroups a query / by waves: 1 x 96 queries of 32 heads of 128 on 8, 768 row tiles 65.5 / 71.3, 128 (1024) 71.8 / 72.6; 8 x 8 (512) 93.7 / 108, 8 x 16 (1024) 167 / 111; 400 of 8 on 2
    // (800) 91.3 / 89.0; 2 x 32 of 16 of 64 (1024) 59.0 / 58.7)
    p.rows = units >= 1024;
    p.norms = up256(row * p.step);
    p.o = p.norms + up256(row / 16);
    p.ml = p.o + (p.ns > 1 ? up256(heads * Sq * p.G * p.ns * head_dim * 4) : 0);
    p.bytes = p.ml + (p.ns > 1 ? up256(heads * Sq * p.G * p.ns * 8) : 0);
    return p;
}

}  // namespace trn
