// How the work of an attention over an 8-bit cache is laid out (cache8_attn.hip): plain host arithmetic, so that it can be walked over all sizes
// without a device.
#pragma once
#include <cstdint>
#include <type_traits>

namespace trn {

// G query heads a KV head, R rows; n_rt tiles of 16 nq rows; ks waves and ns workgroups (shares) have a tile's keys; the key weights of many rows in n_chunks of chunk_tiles
// row tiles, of few rows from sp scores a row; weights as two fp16 numbers or one (fine);
// offsets of the workspace's parts behind the shares' outputs, and its size.
struct Plan8 { int G, R, nq, ks, n_rt, ns, n_chunks, chunk_tiles, sp; bool fine; int64_t ml, lse2, more, bytes; };

// Rows of a tile: 32 where they make workgroups enough, otherwise 16, whose waves have half the work a key and need half the registers.  us, tiles of
// 16 / 32 rows, each with its best number of shares: 16 heads of 64, batch 4, 2000 keys, 64 queries (128 tiles of 32) 10.2 / 13.0, 300 (640) 23.6 / 21.6; 71
// heads on one, batch 8, 16 queries (288) 21.9 / 23.4, one sequence, 200 (444) 27.6 / 22.8; 32 heads of 128 on 8: batch 4, 8 queries, 2000 keys (32) 12.8 / 13.5, batch 16, 4000 keys (128) 31.7 / 28.9;
// one prompt of 1501 (1504) 49 / 37.  And where the keys are so many that shares make them (row tiles x tiles of 32 keys): 16 heads of 64, 311 queries on 8869 keys
// (160 x 278) 31.5 / 29.4; 32 of 128 on 8, 100 on 16000 (104 x 500) 56.8 / 46.3; 8 on 2, 2 x 102 on 36907 (52 x 1153) 64.6 / 52.5; but 71 of 64 on one, 8 x 16 on 3017 (288 x
// 95) 19.7 / 21.8.
// Shares of a row tile's keys: one workgroup a compute unit over the launch -- one share from 129 row tiles on where each head has one --, no more shares than tiles of 32 keys.  32 heads
// of 128 on 8, one query, us with 1 / 2 / 4 / 8 / 16 / 32 shares: 1025 keys 9.6 / 10.9 / 9.5 / 9.3 / 9.0 / 8.9; batch 8, 1500 keys 12.0 / 12.4 / 11.9 / 12.5 / 16.6; batch 12, 3000
// 23.7 / 19.5 / 20.8; batch 16, 4097 31.3 / 28.6 / 28.4; batch 24, 4000 33.9 / 41.6 / 39.9; batch 32, 8192 88.7 / 91.4 / 93.8; of two to one lengths 70.5 / 72.2 / 70.8.  A
// second launch is some 3 us: short caches have one share, but where few rows' weights need that launch anyway (512 keys 6.4, against 8.5; batch 8: 1025 keys 10.1 / 11.0; 16
// heads of 64: 1025 keys 7.6 / 8.1, 2000 10.7 / 8.3; batch 16, 32 heads of 128, 2000 17.5 / 18.6).
// Several row tiles are bound by their vector work rather than by memory: they rather fill two workgroups a compute unit (2.25 of head_dim 64 and 16 rows) with shares of
// 48 tiles of keys and more, if that is more than one and a half.  16 heads of 64, batch 4, 8000 keys, 20 queries 26.3 with two shares, 23.3 with four; 71 on
// one, batch 28, 11316 keys, one query, with 1 / 2 / 4 / 8 40.8 / 32.0 / 26.4 / 28.5; 32 on 8 of 128, 100 queries, 16000 keys (104 row tiles of 32), with 1 / 2 / 3 / 4 / 6
// 88.9 / 53.5 / 55.2 / 46.3 / 50.7; 4 x 40 queries, 8000 keys (160) 48.6 / 46.7 / 41.1 / 46.0; 8 on 2, 4 x 64 queries, 4000 keys (128 of 16) 19.6 / 17.1 / 18.8 / 17.1.
// Waves that share a row tile's keys: four where there are about as many row tiles of 32 as two workgroups a compute unit hold; with more the
// frame of a workgroup (queries, first keys, joining: a fifth to a half of a short prompt's time) is spent less often by two waves, or one that has all
// keys.  us with four / two / one, 32 heads of 128 on 8: 512 queries on 8448 keys (512 row tiles) 82.8 / 94.1 / 177; one prompt of 602 behind 64 keys (602) 17.6 / 16.1 /
// 20.4, behind 2500 47.4 / 52.9 / 69.7; 799 behind 64 (799) 20.8 / 18.6 / 24.8, behind 2500 59.4 / 56.6 / 73.7; 1600 behind 700 (1600) 62.0 / 55.3 / 62.7, 2400 (2400) 103 / 93.8 / 99.3; two of 1500
// (3008) 72.1 / 57.5 / 55.1; four of 512 (2048) 34.8 / 24.6 / 24.0, of 2047 (8192) 213 / 180 / 161; 71 heads of 64 on one, four of 700 (6216) 57.7 / 42.8 / 36.1.
// A cache that is read by one row tile goes past the caches (each byte once), us through / past: batch 32, 8192 keys 99.5 / 89.4, one sequence of 131072 56.7 /
// 51.2, of 4000 11.2 / 10.6; with two row tiles and more the others find it there: 64 rows, 16000 keys 18.7 / 20.6.
inline Plan8 plan8(int batch, int n_kv_heads, int capacity, int head_dim, int Hq, int Sq, bool weights) {
    Plan8 p;
    const bool d128 = head_dim == 128;
    p.G = Hq / n_kv_heads;
    p.R = p.G * Sq;
    const int64_t heads = (int64_t)batch * n_kv_heads, tiles = (capacity + 31) / 32;
    const int64_t tiles32 = (p.R + 31) / 32;
    p.nq = p.R > 16 && (heads * tiles32 >= (d128 ? 128 : 320) || heads * tiles32 * tiles >= 32768) ? 2 : 1;
    p.n_rt = (p.R + 16 * p.nq - 1) / (16 * p.nq);
    const int64_t units = heads * p.n_rt;
    int64_t ns = units ? 256 / units : 1;
    if (p.n_rt > 1) {
        const int64_t most = (d128 || p.nq == 2 ? 512 : 576) / units, worth = (tiles + 47) / 48, more = most < worth ? most : worth;
        if (units * more > 384) ns = more;
    }
    // (key weights: a score of 4 bytes goes out and comes back for each row and key, or K is read again)
    p.sp = weights && 8 * p.R <= head_dim ? (int)tiles * 32 : 0;
    if (!p.sp && tiles <= (d128 ? 26 : 34) + units / 2) ns = 1;
    if (ns > tiles) ns = tiles;
    p.ns = (int)(ns < 1 ? 1 : ns > 64 ? 64 : ns);
    // (there is one share above 288 row tiles, the most of which two fit; a wave that has all keys of its rows writes no share)
    p.ks = p.nq == 1 || p.n_rt == 1 || units <= 700 ? 4 : units < 2560 || p.ns > 1 ? 2 : 1;
    // (The errors of few rows' weights do not average out, and there the second product costs little.  us with one number / two: one row tile, 32 x 1 on 8193 81.8 / 82.5, 16 x 8
    // queries of 32 heads on 8 on 4000 29.4 / 30.5, 96 x 8 on 300 19.6 / 20.9; several of 512 rows at most, 32 on 8 of 128, 16 queries on 16000 keys 16.9 / 18.8, on 60000 47.6 /
    // 50.1, 71 on one of 64, 5 on 16000 12.4 / 13.5, on 60000 22.8 / 26.5; of more, 100 queries on 16000 46.2 / 57.2, the 512 on 8448 85 / 110, four prompts of 2047 169 / 209.)
    p.fine = p.n_rt == 1 || heads * p.R <= 512;
    auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
    p.ml = p.ns > 1 ? up(units * p.ns * 16 * p.nq * head_dim * 4) : 0;
    p.lse2 = p.ml + (p.ns > 1 ? up(units * p.ns * 32 * p.nq * 4) : 0);
    p.more = p.lse2 + (weights ? up(heads * p.R * 4) : 0);
    p.bytes = p.more;
    p.n_chunks = 1; p.chunk_tiles = (int)tiles32;
    if (p.sp) p.bytes += up(heads * p.R * p.sp * 4);
    else if (weights) {
        // (Two workgroups a compute unit, all that it holds; three for a prompt, half of whose queries and keys do not see each other; chunks of two row tiles
        // at least (a prompt of 128 with chunks of one / two / four / six 12.5 / 13.2 / 15.6 / 19.0, of 300 23.3 / 19.3 / 20.5 / 23.2).  32 heads of 128 on 8, us a call with one / two / three / four / six: prompts of 1501 82 / 65 / 61 / 66 / 63, of 4096 374 / 293 / 266 / 296 /
        // 269; 512 queries, 4096 keys 80 / 70 / 77 / 73 / 75.)
        // (By the capacity, as the host does not know the lengths: a prompt of 1501 on a cache of 1501 / 4096 / 8192 / 32768 keys 61 / 86 / 125 / 185 us.)
        const int64_t blocks = heads * ((capacity + 255) / 256);
        int64_t chunks = blocks ? (2 * Sq > capacity ? 768 : 512) / blocks : 1;
        if (chunks > tiles32 / 2) chunks = tiles32 / 2;
        if (chunks > 1) {
            p.chunk_tiles = (int)((tiles32 + chunks - 1) / chunks);
            p.n_chunks = (tiles32 + p.chunk_tiles - 1) / p.chunk_tiles;
            if (p.n_chunks > 1) p.bytes += up(p.n_chunks * heads * capacity * 4);
        }
    }
    return p;
}

// The kernel that such a plan is for: f(nq, ks, past, fine) of constants, past where a single row tile reads a cache.  What is launched, and by how much its
// waves divide a row tile's keys, are one choice: with ks of the plan and another one of the kernel, waves would walk behind the last key.
template <class F> inline void with_kernel8(const Plan8& p, F&& f) {
    const std::integral_constant<int, 1> one{};
    const std::integral_constant<int, 2> two{};
    const std::integral_constant<int, 4> four{};
    const std::true_type yes{};
    const std::false_type no{};
    if (p.n_rt == 1) p.nq == 1 ? f(one, four, yes, yes) : f(two, four, yes, yes);
    else if (p.nq == 1) p.fine ? f(one, four, no, yes) : f(one, four, no, no);
    else if (p.ks == 4) p.fine ? f(two, four, no, yes) : f(two, four, no, no);
    else if (p.ks == 2) f(two, two, no, no);
    else f(two, one, no, no);
}

}  // namespace trn
