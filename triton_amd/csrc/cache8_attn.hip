// Attention over an 8-bit key/value cache: o = softmax(scale * q (K8 ks)^T) (V8 vs), GQA / MQA, each sequence of a length of its own.
//
// The rows of a KV head are its query heads' queries, row r = (query r / G, head r % G): a tile of 32 of them reads the head's keys
// once.  A wave has such a tile and keys of its own, 32 at a time: codes come from memory straight into LDS, 16 bytes a lane and whole
// rows, one tile ahead, and become fp16 on the way into the matrix pipe (every e4m3 number is one of fp16; queries enter as given):
//     S^T[key][row] = K8 . Q^T              contraction 16 ks + 8 e + ..: 16-byte reads, two steps each
//     O^T[d][row]  += V8^T[d][key] P^T      transposing 8-byte reads; the keys of a lane's scores are those of its operand
// The scales cost no work by the element.  ks is part of the factor that the scores are multiplied by for the exponential anyway, and vs
// is added to the exponent: with t = s + log2 vs, p = 2^(t - m) is the weight of the CODES of V, and the sum of probabilities is
// that of p / vs, one division a tile.  The reference m is a maximum of t: what counts for the output is near one in fp16, however
// much the blocks differ.  (A block whose vs is below 2^-64 adds nothing that fp16 could hold; it counts in the sum alone.)
//
// Waves of a workgroup, and workgroups (shares) of a row tile, have consecutive runs of the keys that its rows see; their results
// are joined by (m, l, O) in LDS, and by a second launch.
#include "cache8.h"

namespace trn {

// 32 keys of K and V a wave and stage
template <int D> constexpr int kTile = 32 * D;

// Where a 16-byte chunk of a stage row lies.  A K read has 32 rows at one chunk, served 16 lanes at a time ({0-3, 12-15, 20-27} and the
// others); a V read has the rows {0-3, 8-11} (or 4 further on) at two neighbouring chunks, served in halves of the wave.
template <int D> __device__ __forceinline__ int k_swz(int row) { return D == 128 ? (row >> 1) & 7 : (row >> 2) & 3; }
template <int D> __device__ __forceinline__ int v_swz(int row) { return D == 128 ? ((row & 2) | ((row >> 1) & 4)) : (row >> 2) & 2; }

#if defined(__HIP_DEVICE_COMPILE__)
// One wave's 32 keys of K or V from key0 on: rows past the sequence's end arrive as zeros.  vo: the lane's offset in an even and in
// an odd one of the 1 KB loads (whose rows swizzle differently).
template <int D>
__device__ __forceinline__ void fetch32(const uint8_t* head, int64_t pitch, int key0, int L, uint8_t* dst, int vo_even, int vo_odd) {
    constexpr int RPI = 1024 / D;
    const int rows = min(L - key0, 32);       // (none: nothing is read, zeros arrive)
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)(head + key0 * pitch), 0, rows > 0 ? (int)((rows - 1) * pitch) + D : 0, 0x00020000);
#pragma unroll
    for (int n = 0; n < 32 / RPI; ++n)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(dst + n * 1024), 16, n & 1 ? vo_odd : vo_even,
                                                 (int)(n * RPI * pitch), 0, 0);
}
__device__ __forceinline__ uint2_t lds_read_tr8(const uint8_t* p) {
    typedef int int2_t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint2_t, __builtin_amdgcn_ds_read_tr8_b64_v2i32((int2_t __attribute__((address_space(3)))*)(p)));
}
// Whether a byte of these is a NaN code (0x7f or 0xff).
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
#endif

template <int D, int NW>
__global__ __launch_bounds__(NW * 64, 2) void cache8_attn_kernel(const Attn8Args a) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int NJ = D / 32;       // 16-byte K reads a lane, two contraction steps each; tiles of 32 output columns
    __shared__ __attribute__((aligned(1024))) uint8_t Ks0[NW * kTile<D>];
    __shared__ __attribute__((aligned(1024))) uint8_t Ks1[NW * kTile<D>];
    __shared__ __attribute__((aligned(1024))) uint8_t Vs0[NW * kTile<D>];
    __shared__ __attribute__((aligned(1024))) uint8_t Vs1[NW * kTile<D>];
    __shared__ float ms[NW][32], ls[NW][32], m_all[32], l_all[32];

    const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // (workgroups of one share of a head, the row tiles apart, follow each other at the distance of all shares: one XCD where that is a
    // multiple of eight)
    const int rt = a.by_units.of(blockIdx.x), unit = blockIdx.x - rt * a.by_units.d;
    const int bh = a.by_ns.of(unit), share = unit - bh * a.ns;
    const int b = a.by_hkv.of(bh), kvh = bh - b * a.Hkv;

    const int L = keys_of(a.lengths, b, a.cap), C = tokens_of(a.counts, b, a.Sq);
    const int row = rt * 32 + n, qi = a.by_g.of(row), qg = row - qi * a.G;
    if (a.by_g.of(rt * 32) >= C) return;                       // no row of this tile is there
    const bool there = row < a.R && qi < C;
    const int off = L - C;                                     // causal: query i sees keys <= i + off
    const int last = there ? (a.causal ? min(L - 1, qi + off) : L - 1) : -1;
    const int last_q = min(a.by_g.of(min(rt * 32 + 31, a.R - 1)), C - 1);
    const int seen = a.causal ? min(L, max(0, last_q + off + 1)) : L;       // keys that some row sees
    const int all_see = a.causal ? min(L, a.by_g.of(rt * 32) + off + 1) : L;      // ... and that all rows there do

    // This wave's tiles.
    const int T = (seen + 31) >> 5, w = share * NW + wave;
    const int t0 = a.by_w.of(T * w), t1 = a.by_w.of(T * (w + 1));       // (2^21 tiles and 512 waves at most)

    const half_t* qp = a.q + (there ? b * a.qb + (int64_t)(kvh * a.G + qg) * a.qh + (int64_t)qi * a.qs : 0);
    half8_t qB[2 * NJ];
#pragma unroll
    for (int i = 0; i < 2 * NJ; ++i) qB[i] = *reinterpret_cast<const half8_t*>(qp + 16 * (2 * (i >> 1) + h) + 8 * (i & 1));

    const uint8_t* kp = a.k + b * a.kb + kvh * a.kh;
    const uint8_t* vp = a.v + b * a.vb + kvh * a.vh;
    const float* ksp = a.ks + b * a.ksb + kvh * a.ksh;
    const float* vsp = a.vs + b * a.vsb + kvh * a.vsh;

    // staging: load i of a wave covers rows RPI i + lane / CPR
    constexpr int CPR = D / 16, RPI = 64 / CPR;
    const int sr = lane / CPR, sc = lane % CPR;
    const int ko_e = (int)(sr * a.kst) + ((sc ^ k_swz<D>(sr)) << 4), ko_o = (int)(sr * a.kst) + ((sc ^ k_swz<D>(sr + RPI)) << 4);
    const int vo_e = (int)(sr * a.vst) + ((sc ^ v_swz<D>(sr)) << 4), vo_o = (int)(sr * a.vst) + ((sc ^ v_swz<D>(sr + RPI)) << 4);
    uint8_t* const K0 = Ks0 + wave * kTile<D>;
    uint8_t* const K1 = Ks1 + wave * kTile<D>;
    uint8_t* const V0 = Vs0 + wave * kTile<D>;
    uint8_t* const V1 = Vs1 + wave * kTile<D>;
    // reads
    const int kr = n * D + ((h ^ k_swz<D>(n)) << 4);
    const int g16 = lane >> 4, ar = (lane & 15) >> 1;
    const int vkey = 4 * h + (ar & 3) + 8 * (ar >> 2);
    const int vr = vkey * D + (((g16 & 1) ^ v_swz<D>(vkey)) << 4) + 8 * (lane & 1);

    float16_t o[NJ];
#pragma unroll
    for (int i = 0; i < NJ; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
    float m = -INFINITY, l = 0.f;

    float sk = 0.f, sv = 0.f;        // lane i: the scales of the i-th tile of the 64 around this one
    auto scales = [&](int t) {
        const int blk = min(t + lane, t1 - 1) >> (a.bshift - 5);
        sk = ksp[blk]; sv = vsp[blk];
    };
    auto settle = [&] { asm volatile("" : "+v"(sk), "+v"(sv)); };       // (waited for here, not in every step)

    auto step = [&](int t, const uint8_t* Kt, const uint8_t* Vt) __attribute__((always_inline)) {
        const int i64 = (t - t0) & 63;
        const float ksc = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sk), i64));
        const float vsc = fmaxf(__uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sv), i64)), 0x1p-64f);
        const float lv = fast_log2(vsc), c = a.c * ksc;
        float16_t s;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = 0.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const uint4_t w4 = *reinterpret_cast<const uint4_t*>(Kt + (kr ^ (j << 5)));
            s = mfma32(half_of_codes(w4.x, w4.y), qB[2 * j], s);
            s = mfma32(half_of_codes(w4.z, w4.w), qB[2 * j + 1], s);
        }
        const int key0 = t * 32;
        const bool masked = key0 + 32 > all_see;
        if (masked) {
            const int lim = last - key0 - 4 * h;
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = 8 * (e >> 2) + (e & 3) <= lim ? s[e] : -INFINITY;
        }
        if (a.scores && there) {
            float* const to = a.scores + ((int64_t)bh * a.R + row) * a.sp + key0 + 4 * h;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float4_t x;
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = s[4 * e + r] == -INFINITY ? -INFINITY : s[4 * e + r] * c;
                *reinterpret_cast<float4_t*>(to + 8 * e) = x;
            }
        }
        // (the largest score times a factor that is not negative; a score of -inf stays one beside a factor of zero)
        const float top = half_max(max16(s));
        const float tm = top == -INFINITY ? top : __builtin_fmaf(top, c, lv);
        if (__builtin_amdgcn_ballot_w64(tm > m + 8.f) != 0) {       // lazily: p stays below 2^8
            const float up = fmaxf(m, tm), alpha = up == -INFINITY ? 1.f : fast_exp2(m - up);
            m = up;
            l *= alpha;
#pragma unroll
            for (int i = 0; i < NJ; ++i) o[i] = o[i] * alpha;
        }
        const float d = (m == -INFINITY ? 0.f : -m) + lv;
        float p[16], sum = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            p[e] = fast_exp2(__builtin_fmaf(s[e], c, d));
            if (masked) p[e] = s[e] == -INFINITY ? 0.f : p[e];          // (-inf times a scale of zero)
        }
#pragma unroll
        for (int e = 0; e < 16; e += 4) sum += (p[e] + p[e + 1]) + (p[e + 2] + p[e + 3]);
        l = __builtin_fmaf(sum, __builtin_amdgcn_rcpf(vsc), l);
        half8_t pB[2];
#pragma unroll
        for (int e = 0; e < 16; ++e) pB[e >> 3][e & 7] = (half_t)p[e];
        // A NaN code of a key that not all rows see: a product would hand it to the rows that do not (0 * NaN).  It is taken out,
        // and the rows that see it get it in its columns.
        uint2_t vw[NJ][2];
        uint32_t bad = 0;
#pragma unroll
        for (int i = 0; i < NJ; ++i)
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2) {
                vw[i][k2] = lds_read_tr8(Vt + (vr ^ (i << 5)) + k2 * 16 * D);
                if (masked) bad |= nan_bytes(vw[i][k2].x) | nan_bytes(vw[i][k2].y);
            }
        if (masked && __builtin_amdgcn_ballot_w64(bad != 0) != 0) {
            const half_t one = (half_t)1.f, nil = (half_t)0.f;
            const int lim = last - key0 - 4 * h;
#pragma unroll
            for (int i = 0; i < NJ; ++i) {
                float16_t hit;
#pragma unroll
                for (int e = 0; e < 16; ++e) hit[e] = 0.f;
#pragma unroll
                for (int k2 = 0; k2 < 2; ++k2) {
                    const uint32_t nx = nan_bytes(vw[i][k2].x), ny = nan_bytes(vw[i][k2].y);
                    half8_t is, sees;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        is[e] = ((e < 4 ? nx : ny) >> (8 * (e & 3)) & 0x80u) ? one : nil;
                        const int key = 16 * k2 + 8 * (e >> 2) + (e & 3);
                        sees[e] = key <= lim ? one : nil;
                    }
                    hit = mfma32(is, sees, hit);
                    vw[i][k2].x &= ~((nx >> 7) * 0xffu); vw[i][k2].y &= ~((ny >> 7) * 0xffu);
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) o[i][e] = hit[e] > 0.f ? NAN : o[i][e];
            }
        }
#pragma unroll
        for (int i = 0; i < NJ; ++i)
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2) o[i] = mfma32(half_of_codes(vw[i][k2].x, vw[i][k2].y), pB[k2], o[i]);
    };
    // Everything of the stage that the next load overwrites has been read: its values are in registers before the load goes out.
    auto ahead = [&](int t, uint8_t* Kt, uint8_t* Vt) __attribute__((always_inline)) {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        const int end = t < t1 ? L : 0;
        fetch32<D>(kp, a.kst, t * 32, end, Kt, ko_e, ko_o);
        fetch32<D>(vp, a.vst, t * 32, end, Vt, vo_e, vo_o);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto arrived = [&] {       // the tile before the one that was requested last
        if constexpr (D == 128) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
    };
    if (t0 < t1) {
        scales(t0);
        ahead(t0, K0, V0);
        settle();
#pragma unroll
        for (int i = 0; i < 2 * NJ; ++i) {
            half8_t z = {};
            qB[i] = there ? qB[i] : z;
        }
        for (int t = t0; t < t1; t += 2) {
            if (t > t0 && ((t - t0) & 63) == 0) { scales(t); settle(); }
            ahead(t + 1, K1, V1);
            arrived();
            step(t, K0, V0);
            ahead(t + 2, K0, V0);
            arrived();
            if (t + 1 < t1) step(t + 1, K1, V1);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    l = half_sum(l);

    // ---- the waves' results
    if (h == 0) { ms[wave][n] = m; ls[wave][n] = l; }
    __syncthreads();
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) top = fmaxf(top, ms[i][n]);
#pragma unroll
    for (int i = 0; i < NW; ++i) sum = __builtin_fmaf(ls[i][n], ms[i][n] == -INFINITY ? 0.f : fast_exp2(ms[i][n] - top), sum);      // (a sum of NaN stays)
    const float mine = m == -INFINITY ? 0.f : fast_exp2(m - top);
    // (a stage array holds 32 rows of D floats of one wave in four; the 16-byte pieces of a row are swizzled by the row)
    auto area = [&](int i) __attribute__((always_inline)) {
        uint8_t* const base = i % 4 == 0 ? Ks0 : i % 4 == 1 ? Ks1 : i % 4 == 2 ? Vs0 : Vs1;
        return reinterpret_cast<float4_t*>(base + (i / 4) * 32 * D * 4);
    };
    {
        float4_t* const mem = area(wave);
#pragma unroll
        for (int i = 0; i < NJ; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int piece = 8 * i + 2 * e + h;               // columns 32 i + 8 e + 4 h ..
                float4_t x;
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = o[i][4 * e + r] * mine;
                mem[n * (D / 4) + (piece ^ (n & 15))] = x;
            }
    }
    if (wave == 0 && h == 0) { m_all[n] = top; l_all[n] = sum; }
    __syncthreads();
    constexpr int TPR = NW * 64 / 32, NP = D / 4 / TPR;                // threads a row, 16-byte pieces a thread
    static_assert(NP >= 1, "a row's pieces for its threads");
    const int orow = threadIdx.x / TPR, sub = threadIdx.x % TPR;
    const int r = rt * 32 + orow, i0 = a.by_g.of(r), g0 = r - i0 * a.G;
    if (r >= a.R || i0 >= C) return;
    const float rm = m_all[orow], rl = l_all[orow];
    const float inv = rl == 0.f ? 0.f : 1.f / rl;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int piece = sub + i * TPR;
        float4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k2 = 0; k2 < NW; ++k2) x = x + area(k2)[orow * (D / 4) + (piece ^ (orow & 15))];
        if (a.ns > 1) {
            const int64_t at = ((int64_t)bh * a.n_rt + rt) * a.ns + share;
            *reinterpret_cast<float4_t*>(a.part + (at * 32 + orow) * D + 4 * piece) = x;
        } else {
            half4_t y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = (half_t)(x[e] * inv);
            *reinterpret_cast<half4_t*>(a.o + b * a.ob + (int64_t)(kvh * a.G + g0) * a.oh + (int64_t)i0 * a.os + 4 * piece) = y;
        }
    }
    if (sub == 0) {
        if (a.ns > 1) {
            float* const to = a.ml + ((((int64_t)bh * a.n_rt + rt) * a.ns + share) * 32 + orow) * 2;
            to[0] = rm; to[1] = rl;
        } else {
            const float x = rm + fast_log2(rl);            // (-inf for a row that sees nothing)
            if (a.lse) a.lse[((int64_t)b * a.Hq + kvh * a.G + g0) * a.Sq + i0] = x * kLn2;
            if (a.lse2) a.lse2[(int64_t)bh * a.R + r] = x;
        }
    }
#endif
}

// ------------------------------------------------------------------------------------------------ host
struct Plan8 { int G, R, n_rt, ns, n_chunks, chunk_tiles, sp; int64_t ml, lse2, more, bytes; };

// How many workgroups share the keys of a row tile: two a compute unit over the launch, as long as a wave has two tiles.
static Plan8 plan8(const trn_cache8* c, int Hq, int Sq, bool weights) {
    Plan8 p;
    p.G = Hq / c->n_kv_heads;
    p.R = p.G * Sq;
    p.n_rt = (p.R + 31) / 32;
    const int64_t heads = (int64_t)c->batch * c->n_kv_heads, units = heads * p.n_rt, tiles = (c->capacity + 31) / 32;
    int64_t ns = units ? 512 / units : 1;
    if (ns > tiles / 8) ns = tiles / 8;
    p.ns = (int)(ns < 1 ? 1 : ns > 64 ? 64 : ns);
    auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
    p.ml = p.ns > 1 ? up(units * p.ns * 32 * c->head_dim * 4) : 0;
    p.lse2 = p.ml + (p.ns > 1 ? up(units * p.ns * 64 * 4) : 0);
    p.more = p.lse2 + (weights ? up(heads * p.R * 4) : 0);
    p.bytes = p.more;
    // Key weights: a score of 4 bytes goes out and comes back for each row and key, or K is read again.
    p.sp = weights && 8 * p.R <= c->head_dim ? (int)tiles * 32 : 0;
    p.n_chunks = 1; p.chunk_tiles = p.n_rt;
    if (p.sp) p.bytes += up(heads * p.R * p.sp * 4);
    else if (weights) {
        // (four workgroups a compute unit, a chunk of four row tiles at least)
        const int64_t blocks = heads * ((c->capacity + 255) / 256);
        int64_t chunks = blocks ? 1024 / blocks : 1;
        if (chunks > p.n_rt / 4) chunks = p.n_rt / 4;
        if (chunks > 1) {
            p.chunk_tiles = (int)((p.n_rt + chunks - 1) / chunks);
            p.n_chunks = (p.n_rt + p.chunk_tiles - 1) / p.chunk_tiles;
            if (p.n_chunks > 1) p.bytes += up(p.n_chunks * heads * c->capacity * 4);
        }
    }
    return p;
}

static int attn8_check(const trn_cache8* c, int32_t n_q_heads, int32_t seq_q) {
    const int st = cache8_check(c);
    if (st != TRN_OK) return st;
    if (n_q_heads <= 0 || n_q_heads % c->n_kv_heads || seq_q < 0) return TRN_E_SHAPE;
    if ((int64_t)n_q_heads / c->n_kv_heads * seq_q > (1 << 26) || (int64_t)c->batch * n_q_heads > (1 << 26)) return TRN_E_UNSUPPORTED;
    return TRN_OK;
}

}  // namespace trn

extern "C" int64_t trn_cache8_attn_workspace_bytes(const trn_cache8* c, int32_t n_q_heads, int32_t seq_q, int32_t weights) {
    using namespace trn;
    if (!c || c->n_kv_heads <= 0 || n_q_heads <= 0 || n_q_heads % c->n_kv_heads || seq_q <= 0 || c->batch <= 0 || c->capacity <= 0) return 0;
    return plan8(c, n_q_heads, seq_q, weights != 0).bytes;
}

extern "C" int trn_cache8_attn_f16(const trn_cache8* c, const void* q, void* o, int32_t n_q_heads, int32_t seq_q, int64_t q_stride_b,
                                   int64_t q_stride_h, int64_t q_stride_s, int64_t o_stride_b, int64_t o_stride_h, int64_t o_stride_s,
                                   float scale, int32_t causal, float* lse, const float* weights_in, float* weights_out, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
    using namespace trn;
    const int st = attn8_check(c, n_q_heads, seq_q);
    if (st != TRN_OK) return st;
    if (c->batch == 0 || seq_q == 0) return TRN_OK;
    if (!q || !o || (weights_in && !weights_out)) return TRN_E_NULL;
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
    a.G = p.G; a.R = p.R; a.n_rt = p.n_rt; a.ns = p.ns; a.causal = causal != 0;
    a.bshift = c->block == 32 ? 5 : c->block == 64 ? 6 : 7;
    const int64_t heads = (int64_t)c->batch * c->n_kv_heads, units = heads * p.ns;
    if (units * p.n_rt > 0x7fffffffLL || heads * ((int64_t)p.R + 1) > 0x7fffffffLL || heads * ((c->capacity + 255) / 256) * p.n_chunks > 0x3fffffffLL) return TRN_E_SHAPE;
    a.by_units = Div(units); a.by_g = Div(p.G); a.by_hkv = Div(c->n_kv_heads); a.by_ns = Div(p.ns); a.by_w = Div(4 * p.ns);
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
    if (d128) hipLaunchKernelGGL((cache8_attn_kernel<128, 4>), dim3((unsigned)(units * p.n_rt)), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((cache8_attn_kernel<64, 4>), dim3((unsigned)(units * p.n_rt)), dim3(256), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && (p.ns > 1 || p.sp)) e = launch_cache8_finish(a, c->head_dim, s);
    if (e == hipSuccess && weights_out && !p.sp && c->capacity > 0) e = launch_cache8_weights(a, c->head_dim, s);
    return e == hipSuccess ? TRN_OK : TRN_E_LAUNCH;
}
