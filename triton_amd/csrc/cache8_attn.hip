// Attention over an 8-bit key/value cache: o = softmax(scale * q (K8 ks)^T) (V8 vs), GQA / MQA, each sequence of a length of its own.
//
// The rows of a KV head are its query heads' queries, row r = (query r / G, head r % G): a tile of 16 NQ of them reads the head's keys
// once.  A wave has such a tile and keys of its own, 32 at a time: codes come from memory straight into LDS, 16 bytes a lane and whole
// rows, one tile ahead, and become fp16 on the way into the matrix pipe (every e4m3 number is one of fp16; queries enter as given).
// On the 16x16x32 MFMA, lane 16 g + n with the rows 16 qb + n:
//     S^T(kb, qb)[key][row] = K8[16 kb + key] . Q[16 qb + row]          16-byte reads, two contraction steps each; the lane receives the
//                                                                      keys 16 kb + 4 g ..+3
//     O^T(db, qb)[d][row]  += V8^T[16 db + d][slot] P^T[slot][row]      transposing 8-byte reads; slot 8 g + j is key 4 g + j, or
//                                                                      16 + 4 g + j - 4: the lane's own scores
// The scales cost no work by the element.  ks is part of the factor that the scores are multiplied by for the exponential anyway, and vs
// is added to the exponent: with t = s + log2 vs, p = 2^(t - m) is the weight of the CODES of V, and the sum of probabilities is
// that of p / vs, one multiplication a tile.  The reference m is a maximum of t: what counts for the output is near one in fp16, however
// much the blocks differ.  (A block whose vs is below 2^-64 adds nothing that fp16 could hold; it counts in the sum alone.)
// The product with V takes p as fp16.  Rounded once, it brings an error of 2^-12 of each key's part, about as much as the output's own rounding: the
// distance from 64 bits is then 1.0 to 1.45 times that of a computation in fp32 with more than 512 rows (400 drawn shapes), but up to 1.65 times with few, of which
// one may be off by 2^-11 throughout.  There p is two numbers of fp16 (1.00 times), at the price of the second product.
//
// A row tile's waves (four, two or one of a workgroup), and workgroups (shares), have consecutive runs of the keys that its rows see; their results
// are joined by (m, l, O) in LDS, and by a second launch.
//
// One query on a long cache is bound by memory: 32 sequences of up to 8193 keys, 8 heads of 128, 408 MB in 68 us, 6.0 TB/s; one of 131072, 269 MB, 47 us + 4
// for the joining of shares.  Chunks and prompts are bound by the conversion of K and V beside the products, which every row tile repeats: 512 queries of 32 heads on
// 8448 keys 80 us, 860 TFLOP/s (the attention on fp16 caches 93), four prompts of 2047 166 us, 830 (134), one of 4096 157, 870 (118).  So are a few hundred rows a head (71 heads of
// 64 on one, up to 16 queries on up to 3001 keys 19.2 us; all as long 22.3), with two or three workgroups a compute unit as they come.
// Sequences of very different lengths are not shared out evenly, as the host does not know them: one of 131072 keys among 31 of 1000, one query 600 us, as many keys
// in equal lengths 53.
#include "cache8.h"
#include "cache8_rules.h"

namespace trn {

// 32 keys of K and V a wave and stage
template <int D> constexpr int kTile = 32 * D;

// Where a 16-byte chunk of a stage row lies.  A K read is served 16 lanes at a time ({0-3, 12-15, 20-27} and the others): the rows {0-3, 12-15} at
// one chunk and {4-11} at its neighbour.  A V read is served in halves of the wave: the rows {0-7, 16-23} (or 8 further on) at one chunk.
template <int D> __device__ __forceinline__ int k_swz(int row) { return D == 128 ? (row >> 1) & 7 : -(row >> 2) & 3; }
template <int D> __device__ __forceinline__ int v_swz(int row) { return D == 128 ? ((row >> 1) & 3) | ((row >> 2) & 4) : ((row >> 2) & 1) | ((row >> 3) & 2); }

#if defined(__HIP_DEVICE_COMPILE__)
// One wave's 32 keys of K or V at `rows`: `bytes` of them, what lies past arrives as zeros.  lo, hi: the lane's offset in the first and the other
// half (V) or the even and odd ones (K) of the 1 KB loads, whose rows swizzle differently.  PAST: past the caches.
template <int D, bool V, bool PAST>
__device__ __forceinline__ void fetch32(const uint8_t* rows, int pitch, int bytes, uint8_t* dst, int lo, int hi) {
    constexpr int RPI = 1024 / D, N = 32 / RPI;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)rows, 0, bytes, 0x00020000);
#pragma unroll
    for (int n = 0; n < N; ++n)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(dst + n * 1024), 16, (V ? n >= N / 2 : n & 1) ? hi : lo, n * RPI * pitch, 0, PAST ? 2 : 0);
}
__device__ __forceinline__ uint2_t lds_read_tr8(const uint8_t* p) {
    typedef int int2_t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint2_t, __builtin_amdgcn_ds_read_tr8_b64_v2i32((int2_t __attribute__((address_space(3)))*)(p)));
}
// Which bytes of these are a NaN code (0x7f or 0xff), by their top bits.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
__device__ __forceinline__ float4_t mfma16(half8_t a, half8_t b, float4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
// Over the four lanes n, n + 16, n + 32, n + 48 of a row.
__device__ __forceinline__ void swap_rows16(float& a, float& b) { asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b)); }
__device__ __forceinline__ float quad_max(float x) { float a = x, b = x; swap_rows16(a, b); return half_max(fmaxf(a, b)); }
__device__ __forceinline__ float quad_sum(float x) { float a = x, b = x; swap_rows16(a, b); return half_sum(a + b); }
#endif

// KS waves of the four have a row tile's keys, one after the other; 4 / KS row tiles a workgroup.  PAST: a single row tile reads the cache, each byte
// once.  FINE: the weight enters the product with V as two fp16 numbers, what the first leaves over being the second, not rounded to one (see plan8).
template <int D, int NQ, int KS, bool PAST, bool FINE>
__global__ __launch_bounds__(256, 2) void cache8_attn_kernel(const Attn8Args a) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int NW = 4, NG = NW / KS, NJ = D / 64, NDB = D / 16, RT = 16 * NQ;      // 16-byte K reads a lane and key half, of two contraction steps each; output blocks
    __shared__ __attribute__((aligned(1024))) uint8_t Ks0[NW * kTile<D>];
    __shared__ __attribute__((aligned(1024))) uint8_t Ks1[NW * kTile<D>];
    __shared__ __attribute__((aligned(1024))) uint8_t Vs0[NW * kTile<D>];
    __shared__ __attribute__((aligned(1024))) uint8_t Vs1[NW * kTile<D>];
    __shared__ float ms[NW][RT], ls[NW][RT], m_all[NG][RT], l_all[NG][RT];

    const int lane = threadIdx.x & 63, n = lane & 15, g4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // (workgroups of one share of a head, the row tiles apart, follow each other at the distance of all shares: one XCD where that is a
    // multiple of eight; the last rows, which see the most keys, first)
    const int nth = a.by_units.of(blockIdx.x), unit = blockIdx.x - nth * a.by_units.d, grp = KS == NW ? 0 : wave / KS;
    const int rt0 = ((a.n_rt - 1) / NG - nth) * NG, rt = rt0 + grp;
    const int bh = a.by_ns.of(unit), share = unit - bh * a.ns;
    const int b = a.by_hkv.of(bh), kvh = bh - b * a.Hkv;

    const int L = keys_of(a.lengths, b, a.cap), C = tokens_of(a.counts, b, a.Sq);
    const int rows = min(a.R, C * a.G);
    if ((KS == 1 ? rt : rt0) * RT >= rows) return;             // no row of this tile, or of these, is there
    const int off = L - C;                                     // causal: query i sees keys <= i + off
    auto sees = [&](int row) { return a.causal ? min(L, max(0, a.by_g.of(row) + off + 1)) : L; };      // keys that a row sees: the first so many
    const int seen = sees(min(rt * RT + RT - 1, rows - 1)), all_see = sees(rt * RT);      // that some row sees, and all of them
    int last[NQ];                                              // the last key that the lane's rows see
    bool there[NQ];
    half8_t qB[NQ][2 * NJ];
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
        const int row = rt * RT + 16 * qb + n, qi = a.by_g.of(row), qg = row - qi * a.G;
        there[qb] = row < rows;
        last[qb] = there[qb] ? sees(row) - 1 : -1;
        const half_t* qp = a.q + (there[qb] ? b * a.qb + (int64_t)(kvh * a.G + qg) * a.qh + (int64_t)qi * a.qs : 0);
#pragma unroll
        for (int i = 0; i < 2 * NJ; ++i) qB[qb][i] = *reinterpret_cast<const half8_t*>(qp + 64 * (i >> 1) + 16 * g4 + 8 * (i & 1));
    }

    // This wave's tiles, and the first of them that not all rows see whole.
    const int T = rt * RT < rows ? (seen + 31) >> 5 : 0, w = share * KS + (KS == NW ? wave : wave % KS);
    const int t0 = a.by_w.of(T * w), t1 = a.by_w.of(T * (w + 1));       // (2^21 tiles and 512 waves at most)
    const int t_mask = min(t1, max(t0, all_see >> 5)), t_part = L >> 5;
    const int kpitch = (int)a.kst, vpitch = (int)a.vst, rest = L & 31;
    const int k_full = 31 * kpitch + D, v_full = 31 * vpitch + D, k_part = rest ? (rest - 1) * kpitch + D : 0, v_part = rest ? (rest - 1) * vpitch + D : 0;
    const uint8_t* kp = a.k + b * a.kb + kvh * a.kh + (int64_t)t0 * 32 * kpitch;      // of the tile that is requested next
    const uint8_t* vp = a.v + b * a.vb + kvh * a.vh + (int64_t)t0 * 32 * vpitch;
    const float* ksp = a.ks + b * a.ksb + kvh * a.ksh;
    const float* vsp = a.vs + b * a.vsb + kvh * a.vsh;

    // staging: load i of a wave covers rows RPI i + lane / CPR
    constexpr int CPR = D / 16, RPI = 64 / CPR;
    const int sr = lane / CPR, sc = lane % CPR;
    const int k_lo = sr * kpitch + ((sc ^ k_swz<D>(sr)) << 4), k_hi = sr * kpitch + ((sc ^ k_swz<D>(sr + RPI)) << 4);
    const int v_lo = sr * vpitch + ((sc ^ v_swz<D>(sr)) << 4), v_hi = sr * vpitch + ((sc ^ v_swz<D>(sr + 16)) << 4);
    uint8_t* const K0 = Ks0 + wave * kTile<D>;
    uint8_t* const K1 = Ks1 + wave * kTile<D>;
    uint8_t* const V0 = Vs0 + wave * kTile<D>;
    uint8_t* const V1 = Vs1 + wave * kTile<D>;
    // reads (the swizzles of rows 16 apart are the same for K)
    const int kr = n * D + ((g4 ^ k_swz<D>(n)) << 4);
    const int ar = n >> 1, vkey = 4 * g4 + (ar & 3) + 16 * (ar >> 2);
    const int vr = vkey * D + (v_swz<D>(vkey) << 4) + 8 * (n & 1);

    const float4_t zero = {0.f, 0.f, 0.f, 0.f};
    float4_t o[NDB][NQ];
    float m[NQ], l[NQ];
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
        m[qb] = -INFINITY; l[qb] = 0.f;
#pragma unroll
        for (int i = 0; i < NDB; ++i) o[i][qb] = zero;
    }

    float c8 = 0.f, lv8 = 0.f, inv8 = 0.f;        // lane i: factor of the scores, log2 vs and 1 / vs of the i-th tile of the 64 around this one
    float sk = 0.f, sv = 0.f;
    auto scales = [&](int t) {
        const int blk = min(t + lane, t1 - 1) >> (a.bshift - 5);
        sk = ksp[blk]; sv = vsp[blk];
    };
    auto settle = [&] {
        const float v = fmaxf(sv, 0x1p-64f);
        c8 = fmaxf(a.c * sk, 0x1p-100f);          // (a scale of zero: -inf stays -inf)
        lv8 = fast_log2(v); inv8 = __builtin_amdgcn_rcpf(v);
        asm volatile("" : "+v"(c8), "+v"(lv8), "+v"(inv8));       // (waited for here, not in every step)
    };
    auto of_lane = [](float x, int i) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), i)); };

    auto step = [&](auto mask_tag, int t, const uint8_t* Kt, const uint8_t* Vt) __attribute__((always_inline)) {
        constexpr bool MASK = decltype(mask_tag)::value;
        const int i64 = (t - t0) & 63, key0 = t * 32;
        const float c = of_lane(c8, i64), lv = of_lane(lv8, i64), inv = of_lane(inv8, i64);
        // (all codes of the tile are requested at once: left to the compiler each of V's reads came right before its products, and was waited for)
        uint4_t kw[2][NJ];
        uint2_t vw[NDB];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int j = 0; j < NJ; ++j) kw[kb][j] = *reinterpret_cast<const uint4_t*>(Kt + kb * 16 * D + (kr ^ (j << 6)));
#pragma unroll
        for (int i = 0; i < NDB; ++i) vw[i] = lds_read_tr8(Vt + (vr ^ (i << 4)));
        __builtin_amdgcn_sched_barrier(0);
        float4_t s[2][NQ];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const uint4_t w4 = kw[kb][j];
                const half8_t k0 = half_of_codes(w4.x, w4.y), k1 = half_of_codes(w4.z, w4.w);
#pragma unroll
                for (int qb = 0; qb < NQ; ++qb) {
                    s[kb][qb] = mfma16(k0, qB[qb][2 * j], j == 0 ? zero : s[kb][qb]);
                    s[kb][qb] = mfma16(k1, qB[qb][2 * j + 1], s[kb][qb]);
                }
            }
        if constexpr (MASK) {
#pragma unroll
            for (int qb = 0; qb < NQ; ++qb) {
                const int lim = last[qb] - key0 - 4 * g4;
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[kb][qb][e] = 16 * kb + e <= lim ? s[kb][qb][e] : -INFINITY;
            }
        }
        if (__builtin_expect(a.scores != nullptr, 0)) {
#pragma unroll
            for (int qb = 0; qb < NQ; ++qb)
                if (there[qb]) {
                    float* const to = a.scores + ((int64_t)bh * a.R + rt * RT + 16 * qb + n) * a.sp + key0 + 4 * g4;
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb) *reinterpret_cast<float4_t*>(to + 16 * kb) = s[kb][qb] * c;
                }
        }
        float tm[NQ];
        bool due = false;
#pragma unroll
        for (int qb = 0; qb < NQ; ++qb) {
            const float4_t &u = s[0][qb], &v = s[1][qb];
            tm[qb] = __builtin_fmaf(max3(max3(u[0], u[1], u[2]), max3(u[3], v[0], v[1]), fmaxf(v[2], v[3])), c, lv);
            due = due || tm[qb] > m[qb] + 8.f;
        }
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(due) != 0, 0)) {       // lazily: p stays below 2^8
#pragma unroll
            for (int qb = 0; qb < NQ; ++qb) {
                const float up = fmaxf(m[qb], quad_max(tm[qb])), alpha = up == -INFINITY ? 1.f : fast_exp2(m[qb] - up);
                m[qb] = up;
                l[qb] *= alpha;
#pragma unroll
                for (int i = 0; i < NDB; ++i) o[i][qb] = o[i][qb] * alpha;
            }
        }
        half8_t p[NQ], p_rest[NQ];
#pragma unroll
        for (int qb = 0; qb < NQ; ++qb) {
            const float d = (m[qb] == -INFINITY ? 0.f : -m[qb]) + lv;
            float sum[2];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[e] = fast_exp2(__builtin_fmaf(s[kb][qb][e], c, d));
                    p[qb][4 * kb + e] = (half_t)x[e];
                    if constexpr (FINE) p_rest[qb][4 * kb + e] = (half_t)(x[e] - (float)p[qb][4 * kb + e]);
                }
                sum[kb] = (x[0] + x[1]) + (x[2] + x[3]);
            }
            l[qb] = __builtin_fmaf(sum[0] + sum[1], inv, l[qb]);
        }
        uint32_t bad = 0;
        if constexpr (MASK) {
#pragma unroll
            for (int i = 0; i < NDB; ++i) bad |= nan_bytes(vw[i].x) | nan_bytes(vw[i].y);
        }
        // A NaN code of a key that not all rows see: a product would hand it to the rows that do not (0 * NaN).  It is taken out,
        // and the rows that see it get it in its columns.
        if constexpr (MASK) {
            if (__builtin_expect(__builtin_amdgcn_ballot_w64(bad != 0) != 0, 0)) {
                const half_t one = (half_t)1.f, nil = (half_t)0.f;
#pragma unroll
                for (int i = 0; i < NDB; ++i) {
                    const uint32_t nx = nan_bytes(vw[i].x), ny = nan_bytes(vw[i].y);
                    half8_t is;
#pragma unroll
                    for (int e = 0; e < 8; ++e) is[e] = ((e < 4 ? nx : ny) >> (8 * (e & 3)) & 0x80u) ? one : nil;
                    vw[i].x &= ~((nx >> 7) * 0xffu); vw[i].y &= ~((ny >> 7) * 0xffu);
#pragma unroll
                    for (int qb = 0; qb < NQ; ++qb) {
                        const int lim = last[qb] - key0 - 4 * g4;
                        half8_t see;
#pragma unroll
                        for (int e = 0; e < 8; ++e) see[e] = 16 * (e >> 2) + (e & 3) <= lim ? one : nil;
                        const float4_t hit = mfma16(is, see, zero);
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[i][qb][e] = hit[e] > 0.f ? NAN : o[i][qb][e];
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < NDB; ++i) {
            const half8_t v = half_of_codes(vw[i].x, vw[i].y);
#pragma unroll
            for (int qb = 0; qb < NQ; ++qb) {
                o[i][qb] = mfma16(v, p[qb], o[i][qb]);
                if constexpr (FINE) o[i][qb] = mfma16(v, p_rest[qb], o[i][qb]);
            }
        }
    };
    // Everything of the stage that the next load overwrites has been read: its values are in registers before the load goes out.
    auto ahead = [&](int t, uint8_t* Kt, uint8_t* Vt) __attribute__((always_inline)) {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        const bool full = t < t_part, any = t < t1;
        fetch32<D, false, PAST>(kp, kpitch, any ? (full ? k_full : k_part) : 0, Kt, k_lo, k_hi);      // (none: nothing is read, zeros arrive)
        fetch32<D, true, PAST>(vp, vpitch, any ? (full ? v_full : v_part) : 0, Vt, v_lo, v_hi);
        kp += 32 * (int64_t)kpitch; vp += 32 * (int64_t)vpitch;
        __builtin_amdgcn_sched_barrier(0);
    };
    auto arrived = [&] {       // the tile before the one that was requested last
        if constexpr (D == 128) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
    };
    const std::false_type whole{};
    const std::true_type partly{};
    if (t0 < t1) {
        scales(t0);
        ahead(t0, K0, V0);
        settle();
#pragma unroll
        for (int qb = 0; qb < NQ; ++qb)
#pragma unroll
            for (int i = 0; i < 2 * NJ; ++i) {
                const half8_t z = {};
                qB[qb][i] = there[qb] ? qB[qb][i] : z;
            }
        int t = t0;
        for (; t + 2 <= t_mask; t += 2) {
            if (__builtin_expect(t > t0 && ((t - t0) & 63) == 0, 0)) { scales(t); settle(); }
            ahead(t + 1, K1, V1);
            arrived();
            step(whole, t, K0, V0);
            ahead(t + 2, K0, V0);
            arrived();
            step(whole, t + 1, K1, V1);
        }
        for (; t < t1; t += 2) {
            if (t > t0 && ((t - t0) & 63) == 0) { scales(t); settle(); }
            ahead(t + 1, K1, V1);
            arrived();
            step(partly, t, K0, V0);
            ahead(t + 2, K0, V0);
            arrived();
            if (t + 1 < t1) step(partly, t + 1, K1, V1);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }

    // ---- a wave with rows of its own (never shared): out of its registers
    if constexpr (KS == 1) {
#pragma unroll
        for (int qb = 0; qb < NQ; ++qb) {
            const int r = rt * RT + 16 * qb + n, i0 = a.by_g.of(r), g0 = r - i0 * a.G;
            const float sum = quad_sum(l[qb]), inv = sum == 0.f ? 0.f : 1.f / sum;
            if (!there[qb]) continue;
            half_t* const to = a.o + b * a.ob + (int64_t)(kvh * a.G + g0) * a.oh + (int64_t)i0 * a.os + 4 * g4;
#pragma unroll
            for (int i = 0; i < NDB; ++i) {
                half4_t y;
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = (half_t)(o[i][qb][e] * inv);
                *reinterpret_cast<half4_t*>(to + 16 * i) = y;
            }
            if (g4 == 0) {
                const float x = m[qb] + fast_log2(sum);            // (-inf for a row that sees nothing)
                if (a.lse) a.lse[((int64_t)b * a.Hq + kvh * a.G + g0) * a.Sq + i0] = x * kLn2;
                if (a.lse2) a.lse2[(int64_t)bh * a.R + r] = x;
            }
        }
        return;
    }
    // ---- the results of a row tile's waves
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
        l[qb] = quad_sum(l[qb]);
        if (g4 == 0) { ms[wave][16 * qb + n] = m[qb]; ls[wave][16 * qb + n] = l[qb]; }
    }
    __syncthreads();
    // (a stage array holds RT rows of D floats of one wave; the 16-byte pieces of a row are swizzled by the row)
    auto area = [&](int i) __attribute__((always_inline)) {
        return reinterpret_cast<float4_t*>(i == 0 ? Ks0 : i == 1 ? Ks1 : i == 2 ? Vs0 : Vs1);
    };
    float4_t* const mem = area(wave);
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
        const int r = 16 * qb + n;
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int i = grp * KS; i < grp * KS + KS; ++i) top = fmaxf(top, ms[i][r]);
#pragma unroll
        for (int i = grp * KS; i < grp * KS + KS; ++i) sum = __builtin_fmaf(ls[i][r], ms[i][r] == -INFINITY ? 0.f : fast_exp2(ms[i][r] - top), sum);      // (a sum of NaN stays)
        const float mine = m[qb] == -INFINITY ? 0.f : fast_exp2(m[qb] - top);
#pragma unroll
        for (int i = 0; i < NDB; ++i) mem[r * (D / 4) + ((4 * i + g4) ^ n)] = o[i][qb] * mine;
        if (wave == grp * KS && g4 == 0) { m_all[grp][r] = top; l_all[grp][r] = sum; }
    }
    __syncthreads();
    constexpr int TPR = KS * 64 / RT, NP = D / 4 / TPR;                // threads a row, 16-byte pieces a thread
    static_assert(NP >= 1 && D / 4 >= 16, "a row's pieces for its threads, and for the swizzle");
    const int orow = threadIdx.x % (KS * 64) / TPR, sub = threadIdx.x % TPR;
    const int r = rt * RT + orow, i0 = a.by_g.of(r), g0 = r - i0 * a.G;
    if (r >= rows) return;
    const float rm = m_all[grp][orow], rl = l_all[grp][orow];
    const float inv = rl == 0.f ? 0.f : 1.f / rl;
    const int64_t at = (((int64_t)bh * a.n_rt + rt) * a.ns + share) * RT + orow;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int piece = sub + i * TPR;
        float4_t x = zero;
#pragma unroll
        for (int k2 = grp * KS; k2 < grp * KS + KS; ++k2) x = x + area(k2)[orow * (D / 4) + (piece ^ (orow & 15))];
        if (a.ns > 1) *reinterpret_cast<float4_t*>(a.part + at * D + 4 * piece) = x;
        else {
            half4_t y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = (half_t)(x[e] * inv);
            *reinterpret_cast<half4_t*>(a.o + b * a.ob + (int64_t)(kvh * a.G + g0) * a.oh + (int64_t)i0 * a.os + 4 * piece) = y;
        }
    }
    if (sub == 0) {
        if (a.ns > 1) { a.ml[at * 2] = rm; a.ml[at * 2 + 1] = rl; }
        else {
            const float x = rm + fast_log2(rl);            // (-inf for a row that sees nothing)
            if (a.lse) a.lse[((int64_t)b * a.Hq + kvh * a.G + g0) * a.Sq + i0] = x * kLn2;
            if (a.lse2) a.lse2[(int64_t)bh * a.R + r] = x;
        }
    }
#endif
}

// ------------------------------------------------------------------------------------------------ host
static Plan8 plan8(const trn_cache8* c, int Hq, int Sq, bool weights) { return plan8(c->batch, c->n_kv_heads, c->capacity, c->head_dim, Hq, Sq, weights); }

static int attn8_check(const trn_cache8* c, int32_t n_q_heads, int32_t seq_q) {
    const int st = cache8_check(c);
    if (st != TRN_OK) return st;
    if (n_q_heads <= 0 || n_q_heads % c->n_kv_heads || seq_q < 0) return TRN_E_SHAPE;
    if ((int64_t)n_q_heads / c->n_kv_heads * seq_q > (1 << 26) || (int64_t)c->batch * n_q_heads > (1 << 26)) return TRN_E_UNSUPPORTED;
    return TRN_OK;
}

// No queries: the keys' weights are what they were, and to be in weights_out all the same.
static int weights_of_nothing(const trn_cache8* c, const float* weights_in, float* weights_out, hipStream_t s) {
    if ((int64_t)c->batch * c->n_kv_heads * ((c->capacity + 255) / 256) > 0xffffff) return TRN_E_SHAPE;       // (threads in 32 bits)
    Attn8Args a{};
    a.lengths = c->lengths; a.B = c->batch; a.Hkv = c->n_kv_heads; a.cap = c->capacity; a.by_hkv = Div(c->n_kv_heads);
    a.w_in = weights_in; a.w_out = weights_out; a.n_chunks = 1;
    return launch_cache8_weights(a, c->head_dim, s) == hipSuccess ? TRN_OK : TRN_E_LAUNCH;
}

}  // namespace trn

extern "C" int64_t trn_cache8_attn_workspace_bytes(const trn_cache8* c, int32_t n_q_heads, int32_t seq_q, int32_t weights) {
    using namespace trn;
    if (!c || c->n_kv_heads <= 0 || n_q_heads <= 0 || n_q_heads % c->n_kv_heads || seq_q <= 0 || c->batch <= 0 || c->capacity <= 0) return 0;
    if ((int64_t)n_q_heads / c->n_kv_heads * seq_q > (1 << 26)) return 0;       // (refused by the call)
    return plan8(c, n_q_heads, seq_q, weights != 0).bytes;
}

extern "C" int trn_cache8_attn_f16(const trn_cache8* c, const void* q, void* o, int32_t n_q_heads, int32_t seq_q, int64_t q_stride_b,
                                   int64_t q_stride_h, int64_t q_stride_s, int64_t o_stride_b, int64_t o_stride_h, int64_t o_stride_s,
                                   float scale, int32_t causal, float* lse, const float* weights_in, float* weights_out, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
    using namespace trn;
    const int st = attn8_check(c, n_q_heads, seq_q);
    if (st != TRN_OK) return st;
    if (c->batch == 0) return TRN_OK;
    if (weights_in && !weights_out) return TRN_E_NULL;
    if (weights_in && weights_in != weights_out) {
        const int64_t size = (int64_t)c->batch * c->n_kv_heads * c->capacity * 4;
        if (!apart(weights_in, size, weights_out, size)) return TRN_E_UNSUPPORTED;
    }
    if (c->capacity == 0) weights_in = weights_out = nullptr;       // (no key has a weight)
    if (seq_q == 0) return weights_out && weights_in != weights_out ? weights_of_nothing(c, weights_in, weights_out, (hipStream_t)stream) : TRN_OK;
    if (!q || !o) return TRN_E_NULL;
    if (!(scale > 0.f)) return TRN_E_SHAPE;
    if ((c->batch > 1 && !o_stride_b) || (n_q_heads > 1 && !o_stride_h) || (seq_q > 1 && !o_stride_s)) return TRN_E_STRIDE;
    if (!aligned16(q) || (reinterpret_cast<uintptr_t>(o) & 7)) return TRN_E_ALIGN;
    for (int64_t s : {q_stride_b, q_stride_h, q_stride_s}) if (!pitch16(s, 2)) return TRN_E_ALIGN;
    for (int64_t s : {o_stride_b, o_stride_h, o_stride_s}) if (s & 3) return TRN_E_ALIGN;
    if (workspace && (reinterpret_cast<uintptr_t>(workspace) & 255)) return TRN_E_ALIGN;
    Plan8 p = plan8(c, n_q_heads, seq_q, weights_out != nullptr);
    if (!workspace || workspace_bytes < p.bytes) {
        if (weights_out) return TRN_E_SCRATCH;
        p.ns = 1;
    }
    Attn8Args a;
    a.k = (const uint8_t*)c->k; a.v = (const uint8_t*)c->v; a.ks = c->k_scale; a.vs = c->v_scale;
    a.lengths = c->lengths; a.counts = c->counts;
    a.q = (const half_t*)q; a.o = (half_t*)o; a.lse = lse;
    a.B = c->batch; a.Hq = n_q_heads; a.Hkv = c->n_kv_heads; a.Sq = seq_q; a.cap = c->capacity;
    a.G = p.G; a.R = p.R; a.n_rt = p.n_rt; a.rshift = p.nq == 1 ? 4 : 5; a.ns = p.ns; a.causal = causal != 0;
    a.bshift = c->block == 32 ? 5 : c->block == 64 ? 6 : 7;
    const int64_t heads = (int64_t)c->batch * c->n_kv_heads, units = heads * p.ns;
    if (heads * ((int64_t)p.R + 1) > 0x7fffffffLL) return TRN_E_SHAPE;
    // (workgroups of 256, and as many threads in all as 32 bits number: of every launch, before the first one)
    const int per = 4 / p.ks;
    const int64_t groups = units * ((p.n_rt + per - 1) / per), n_scores = p.sp ? heads * ((c->capacity + 1023) / 1024) : 0;
    const int64_t n_sums = weights_out && !p.sp ? heads * ((c->capacity + (p.n_chunks > 1 ? 63 : 255)) / (p.n_chunks > 1 ? 64 : 256)) : 0;
    if (groups > 0xffffff || (p.ns > 1 ? heads * p.R : 0) + n_scores > 0xffffff || n_sums > 0xffffff) return TRN_E_SHAPE;
    a.by_units = Div(units); a.by_g = Div(p.G); a.by_hkv = Div(c->n_kv_heads); a.by_ns = Div(p.ns);
    a.kb = c->k_stride_b; a.kh = c->k_stride_h; a.kst = c->k_stride_s;
    a.vb = c->v_stride_b; a.vh = c->v_stride_h; a.vst = c->v_stride_s;
    a.ksb = c->ks_stride_b; a.ksh = c->ks_stride_h; a.vsb = c->vs_stride_b; a.vsh = c->vs_stride_h;
    a.qb = q_stride_b; a.qh = q_stride_h; a.qs = q_stride_s; a.ob = o_stride_b; a.oh = o_stride_h; a.os = o_stride_s;
    a.c = scale * kLog2e;
    a.part = (float*)workspace; a.ml = (float*)((char*)workspace + p.ml);
    a.lse2 = weights_out ? (float*)((char*)workspace + p.lse2) : nullptr;
    a.w_in = weights_in; a.w_out = weights_out;
    a.sp = p.sp; a.scores = p.sp ? (float*)((char*)workspace + p.more) : nullptr;
    a.n_chunks = p.n_chunks; a.chunk_tiles = p.chunk_tiles; a.w_part = p.n_chunks > 1 ? (float*)((char*)workspace + p.more) : nullptr;
    const hipStream_t s = (hipStream_t)stream;
    const bool d128 = c->head_dim == 128;
    with_kernel8(p, [&](auto nq, auto ks, auto past, auto fine) {
        constexpr int NQ = decltype(nq)::value, KS = decltype(ks)::value;
        constexpr bool PAST = decltype(past)::value, FINE = decltype(fine)::value;
        a.by_w = Div(KS * p.ns);
        const dim3 grid((unsigned)groups), block(256);
        if (d128) hipLaunchKernelGGL((cache8_attn_kernel<128, NQ, KS, PAST, FINE>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((cache8_attn_kernel<64, NQ, KS, PAST, FINE>), grid, block, 0, s, a);
    });
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && (p.ns > 1 || p.sp)) e = launch_cache8_finish(a, c->head_dim, s);
    if (e == hipSuccess && weights_out && !p.sp) e = launch_cache8_weights(a, c->head_dim, s);
    return e == hipSuccess ? TRN_OK : TRN_E_LAUNCH;
}
