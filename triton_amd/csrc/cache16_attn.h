// Attention over fp16 caches by tiles of rows: what the shared-prefix and the selected-blocks form have in common.
//
// The rows of a KV head are its query heads' queries, row r = (query r / G, head r % G): a tile of them reads a key once.  Two forms of a tile:
//   narrow   16 or 32 rows; each of a workgroup's four waves has 32 keys of its own at a time, so that four times as many bytes are on their way; the waves' results are
//            joined in LDS.  For few rows, which memory bounds.
//   wide     128 rows, 32 a wave; the waves share the keys in LDS, 32 at a time.  For many rows, which the matrix pipe bounds.
// In both K and V come from memory straight into LDS, ahead of their use, scores are formed transposed, S^T = K Q^T, so that a lane's scores are the
// operand P^T of O^T += V^T P^T as they are, and V is read transposing.  One pass with a running maximum m, taken anew only where a score exceeds it by 2^15 (wide: where a
// tile's weights come to more than 2^15 in all, so that no maximum is formed), and sum l.
// A workgroup may have a share of a tile's keys: (m, l, O) of the shares of a row are joined by a second launch (cache16_join).
#pragma once
#include "cache16.h"

namespace trn {

// Weights enter their product with V in fp16, 2^(score - m), and m lies 7 below the largest score when it is taken, so that they are 2^7 there and come to 2^15 at most.
// A key that has nearly all of the weight (what all queries look at first, its value often next to nothing) leaves little to each of the others: with the largest weight as 1, one is off by
// 2^-32 at most, or by its own rounding, where m at the largest score would make it 2^-25: keys of 2^-20 each are off by 0.03 % at most, and would be by 3 %.
constexpr float kBelow = 7.f;

// What became of a row's keys in one share: O unnormalised, and (m, l) with m in units of log2.  Row `row` of B Hkv M G has `slots` of them.
struct Parts { float* o; float* ml; int slots; };

// LDS of a workgroup: 32 keys of K and of V four times, a stage of a wide tile or of a wave's narrow one each.  They are arrays of their own: of one array the compiler takes each read to be of
// what the loads on their way write, and waits for all of them.
template <int D> struct Lds {
    half_t *k0, *k1, *k2, *k3, *v0, *v1, *v2, *v3;
    __device__ __forceinline__ half_t* k(int i) const { return i == 0 ? k0 : i == 1 ? k1 : i == 2 ? k2 : k3; }
    __device__ __forceinline__ half_t* v(int i) const { return i == 0 ? v0 : i == 1 ? v1 : i == 2 ? v2 : v3; }
};
#define TRN_LDS(D, name)                                                                                                                        \
    __shared__ __attribute__((aligned(1024))) half_t name##_k0[32 * D], name##_k1[32 * D], name##_k2[32 * D], name##_k3[32 * D], name##_v0[32 * D], \
        name##_v1[32 * D], name##_v2[32 * D], name##_v3[32 * D];                                                                              \
    const Lds<D> name{name##_k0, name##_k1, name##_k2, name##_k3, name##_v0, name##_v1, name##_v2, name##_v3}

#if defined(__HIP_DEVICE_COMPILE__)
__device__ __forceinline__ float4_t mfma16(half8_t a, half8_t b, float4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
// Over the four lanes n, n + 16, n + 32, n + 48 of a row.
__device__ __forceinline__ void swap_rows16(float& a, float& b) { asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b)); }
__device__ __forceinline__ float quad_max(float x) { float a = x, b = x; swap_rows16(a, b); return half_max(fmaxf(a, b)); }
__device__ __forceinline__ float quad_sum(float x) { float a = x, b = x; swap_rows16(a, b); return half_sum(a + b); }

// Where a 16-byte chunk of a narrow stage's row lies.  A K read is served 16 lanes at a time ({0-3, 12-15, 20-27} and the others): the rows {0-3, 12-15} at one
// chunk and {4-11} at its neighbour.  A transposing V read is served in halves of the wave: eight rows at two neighbouring chunks.
template <int D> __device__ __forceinline__ int kn_swz(int r) { return D == 128 ? ((r & 3) << 2) | ((r >> 3 & 1) * 3) : ((r >> 1 & 1) << 2) | ((r >> 3 & 1) * 3); }
template <int D> __device__ __forceinline__ int vn_swz(int r) { return D == 128 ? (r & 7) << 1 : (r >> 1 & 3) << 1; }

// Which of eight fp16 values are not finite.
__device__ __forceinline__ bool odd_values(half8_t v) {
    const uint4_t w = __builtin_bit_cast(uint4_t, v);
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) bad |= ((w[i] & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
    return bad != 0;
}
// ... as numbers: one where a value is +inf (kind 0), -inf (1), NaN (2), zero elsewhere.
__device__ __forceinline__ half8_t odd_kind(half8_t v, int kind) {
    half8_t r;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const half_t x = v[e];
        const bool is = kind == 0 ? x == (half_t)INFINITY : kind == 1 ? x == (half_t)-INFINITY : x != x;
        r[e] = is ? (half_t)1.f : (half_t)0.f;
    }
    return r;
}
__device__ __forceinline__ half8_t finite_only(half8_t v) {
    half8_t r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = fabsf((float)v[e]) < INFINITY ? v[e] : (half_t)0.f;
    return r;
}

// ------------------------------------------------------------------------------------------------ narrow
// One wave's tiles t0 <= t < t1, every STEP-th, of 32 keys for 16 NQ rows (queries in qB), into o, m, l.  `keys`: where the tile t begins and how many of its keys there are (0..32, wave-uniform; those
// from there on arrive as zeros and count for no row), as .k(t), .v(t), .n(t); and up to which key of a tile a row sees whose last one is `last`, .lim(t, last).
template <int D, int NQ, int STEP, class Keys>
__device__ __forceinline__ void narrow_walk(Keys& keys, int t0, int t1, int t_mask, int kpitch, int vpitch, float c, const half8_t (&qB)[NQ][D / 32], const int (&last)[NQ], half_t* Kt, half_t* Vt,
                                            float4_t (&o)[D / 16][NQ], float (&m)[NQ], float (&l)[NQ]) {
    constexpr int NI = D / 32, NDB = D / 16, RPI = 512 / D, NL = 32 / RPI, CPR = D / 8;
    const int lane = threadIdx.x & 63, n = lane & 15, g4 = lane >> 4;
    // staging: load i covers the rows RPI i + lane / CPR; swizzles repeat every other (or second other) load
    const int sr = lane / CPR, sc = lane % CPR;
    int k_off[2], v_off[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        k_off[i] = sr * kpitch * 2 + ((sc ^ kn_swz<D>(sr + 8 * i)) << 4);
        v_off[i] = sr * vpitch * 2 + ((sc ^ vn_swz<D>(sr + RPI * i)) << 4);
    }
    int kr[NI], vr[2];
#pragma unroll
    for (int i = 0; i < NI; ++i) kr[i] = n * D + (((4 * i + g4) ^ kn_swz<D>(n)) << 3);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int key = 16 * i + 4 * g4 + (n >> 2);
        vr[i] = key * D + ((vn_swz<D>(key) ^ ((n & 3) >> 1)) << 3) + 4 * (n & 1);
    }
    const float4_t zero = {0.f, 0.f, 0.f, 0.f};

    auto ahead = [&](int t) __attribute__((always_inline)) {
        const int there = keys.n(t);
        const __amdgpu_buffer_rsrc_t ks = __builtin_amdgcn_make_buffer_rsrc((void*)keys.k(t), 0, there ? ((there - 1) * kpitch + D) * 2 : 0, 0x00020000);
        const __amdgpu_buffer_rsrc_t vs = __builtin_amdgcn_make_buffer_rsrc((void*)keys.v(t), 0, there ? ((there - 1) * vpitch + D) * 2 : 0, 0x00020000);
#pragma unroll
        for (int i = 0; i < NL; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ks, (__attribute__((address_space(3))) void*)(Kt + i * 512), 16, k_off[(i * RPI >> 3) & 1], i * RPI * kpitch * 2, 0, 0);
#pragma unroll
        for (int i = 0; i < NL; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(vs, (__attribute__((address_space(3))) void*)(Vt + i * 512), 16, v_off[D == 128 ? i & 1 : 0], i * RPI * vpitch * 2, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    // A tile passes from LDS into registers whole, and the next one is requested into the same place before it is worked on: one stage a wave, so that two workgroups share a
    // compute unit, has as many bytes on their way as two stages of one.
    auto step = [&](auto mask_tag, int t) __attribute__((always_inline)) {
        constexpr bool MASK = decltype(mask_tag)::value;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        half8_t kw[2][NI], vw[NDB];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < NI; ++i) kw[kb][i] = *reinterpret_cast<const half8_t*>(Kt + kb * 16 * D + kr[i]);
#pragma unroll
        for (int i = 0; i < NDB; ++i) {
            const half4_t x = lds_read_tr16(Vt + (vr[0] ^ (i << 4))), y = lds_read_tr16(Vt + (vr[1] ^ (i << 4)));
            vw[i] = half8_t{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
        }
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (t + STEP < t1) ahead(t + STEP);
        __builtin_amdgcn_sched_barrier(0);
        float4_t s[2][NQ];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int qb = 0; qb < NQ; ++qb) s[kb][qb] = mfma16(kw[kb][i], qB[qb][i], i == 0 ? zero : s[kb][qb]);
        if constexpr (MASK) {
#pragma unroll
            for (int qb = 0; qb < NQ; ++qb) {
                const int lim = keys.lim(t, last[qb]) - 4 * g4;
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[kb][qb][e] = 16 * kb + e <= lim ? s[kb][qb][e] : -INFINITY;
            }
        }
        float tm[NQ];
        bool due = false;
#pragma unroll
        for (int qb = 0; qb < NQ; ++qb) {
            const float4_t &u = s[0][qb], &v = s[1][qb];
            tm[qb] = max3(max3(u[0], u[1], u[2]), max3(u[3], v[0], v[1]), fmaxf(v[2], v[3])) * c;
            due = due || tm[qb] > m[qb] + 15.f;
        }
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(due) != 0, 0)) {       // lazily: p stays below 2^15
#pragma unroll
            for (int qb = 0; qb < NQ; ++qb) {
                const float up = fmaxf(m[qb], quad_max(tm[qb]) - kBelow), alpha = up == -INFINITY ? 1.f : fast_exp2(m[qb] - up);
                m[qb] = up;
                l[qb] *= alpha;
#pragma unroll
                for (int i = 0; i < NDB; ++i) o[i][qb] = o[i][qb] * alpha;
            }
        }
        // (p enters the product with V as two fp16 numbers, what the first leaves over being the second: rounded once its error is up to 2^-11 of each key's part, as much as the output's own rounding)
        half8_t p[NQ], rest[NQ];
#pragma unroll
        for (int qb = 0; qb < NQ; ++qb) {
            const float d = m[qb] == -INFINITY ? 0.f : -m[qb];
            float sum[2];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[e] = fast_exp2(__builtin_fmaf(s[kb][qb][e], c, d));
                    p[qb][4 * kb + e] = (half_t)x[e];
                    rest[qb][4 * kb + e] = (half_t)(x[e] - (float)p[qb][4 * kb + e]);
                }
                sum[kb] = (x[0] + x[1]) + (x[2] + x[3]);
            }
            l[qb] += sum[0] + sum[1];
        }
        // An infinity or NaN of a key that not all rows see: a product would hand it to the rows that do not (0 * inf).  It is taken out, and the rows that see it get it by itself.
        if constexpr (MASK) {
            bool bad = false;
#pragma unroll
            for (int i = 0; i < NDB; ++i) bad = bad || odd_values(vw[i]);
            if (__builtin_expect(__builtin_amdgcn_ballot_w64(bad) != 0, 0)) {
#pragma unroll
                for (int qb = 0; qb < NQ; ++qb) {
                    const int lim = keys.lim(t, last[qb]) - 4 * g4;
                    half8_t see;
#pragma unroll
                    for (int e = 0; e < 8; ++e) see[e] = 16 * (e >> 2) + (e & 3) <= lim ? (half_t)1.f : (half_t)0.f;
#pragma unroll
                    for (int i = 0; i < NDB; ++i)
#pragma unroll 1
                        for (int kind = 0; kind < 3; ++kind) {
                            const float4_t hit = mfma16(odd_kind(vw[i], kind), see, zero);
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[i][qb][e] += hit[e] > 0.f ? (kind == 0 ? INFINITY : kind == 1 ? -INFINITY : NAN) : 0.f;
                        }
                }
#pragma unroll
                for (int i = 0; i < NDB; ++i) vw[i] = finite_only(vw[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < NDB; ++i)
#pragma unroll
            for (int qb = 0; qb < NQ; ++qb) {
                o[i][qb] = mfma16(vw[i], p[qb], o[i][qb]);
                o[i][qb] = mfma16(vw[i], rest[qb], o[i][qb]);
            }
    };
    if (t0 >= t1) return;
    ahead(t0);
    int t = t0;
    for (; t < t_mask; t += STEP) step(std::false_type{}, t);
    for (; t < t1; t += STEP) step(std::true_type{}, t);
}

// The results of a row tile's NW waves, joined and delivered: row i of the tile by put(i, first dimension, O, m, l, whether this is the row's first piece).  area(i, 0), area(i, 1): a wave's stage of K
// and of V, 16 rows of D floats each.
template <int NW> struct NarrowStats { float m[NW][32], l[NW][32], m_all[32], l_all[32]; };
template <int D, int NQ, int NW, class Area, class Put>
__device__ __forceinline__ void narrow_join(Area area, NarrowStats<NW>& st, float4_t (&o)[D / 16][NQ], float (&m)[NQ], float (&l)[NQ], Put put) {
    constexpr int NDB = D / 16, RT = 16 * NQ;
    const int lane = threadIdx.x & 63, n = lane & 15, g4 = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
        l[qb] = quad_sum(l[qb]);
        if (g4 == 0) { st.m[wave][16 * qb + n] = m[qb]; st.l[wave][16 * qb + n] = l[qb]; }
    }
    __syncthreads();
    // (the 16-byte pieces of a row are swizzled by the row)
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
        const int r = 16 * qb + n;
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) top = fmaxf(top, st.m[i][r]);
#pragma unroll
        for (int i = 0; i < NW; ++i) sum = __builtin_fmaf(st.l[i][r], st.m[i][r] == -INFINITY ? 0.f : fast_exp2(st.m[i][r] - top), sum);      // (a sum of NaN stays)
        const float mine = m[qb] == -INFINITY ? 0.f : fast_exp2(m[qb] - top);
#pragma unroll
        for (int i = 0; i < NDB; ++i) reinterpret_cast<float4_t*>(area(wave, qb))[n * (D / 4) + ((4 * i + g4) ^ n)] = o[i][qb] * mine;
        if (wave == 0 && g4 == 0) { st.m_all[r] = top; st.l_all[r] = sum; }
    }
    __syncthreads();
    constexpr int TPR = NW * 64 / RT, NP = (D / 4 + TPR - 1) / TPR;                // threads a row, 16-byte pieces a thread
    const int row = threadIdx.x / TPR, sub = threadIdx.x % TPR;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int piece = sub + i * TPR;
        if (D / 4 % TPR && piece >= D / 4) break;
        float4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NW; ++k) x = x + reinterpret_cast<const float4_t*>(area(k, row >> 4))[(row & 15) * (D / 4) + (piece ^ (row & 15))];
        put(row, 4 * piece, x, st.m_all[row], st.l_all[row], piece == 0);
    }
}

// ------------------------------------------------------------------------------------------------ wide
// A workgroup's tiles t0 <= t < t1 of 32 keys for 128 rows, of which this wave has 32 (none: idle).  keys: where a tile begins (.k, .v),
// the pitches there, how many keys lie from there on at these (.left), whether tiles are there as a whole (.whole), and up to which key of a tile a row sees (.lim).
// FINE: p enters the product with V as two numbers, as in the narrow form; as one its error is about the output's own, and averages out over many rows.
// Four stages: a tile is requested three tiles ahead, so that a workgroup alone on its compute unit has 48 KB on their way.
template <int D, bool FINE, class Keys>
__device__ __forceinline__ void wide_walk(const Keys keys, int t0, int t1, int t_mask, bool idle, float c, const half8_t (&qB)[D / 16], int last, const Lds<D>& lds, float16_t (&o)[D / 32], float& m, float& l) {
    constexpr int NS = D / 16, NDB = D / 32, CPR = D / 8, RPI = 64 / CPR, NL = 32 / (4 * RPI);
    const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (t0 >= t1) return;
    const int sr = wave * RPI + lane / CPR, sc = ((lane % CPR) ^ swz<D>(sr)) << 4;
    int kr[NS], vr[2];
#pragma unroll
    for (int i = 0; i < NS; ++i) kr[i] = 2 * n * D + (((2 * i + h) ^ swz<D>(n)) << 4);       // (in bytes)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int e = lane & 15, key = 8 * i + 4 * h + (e >> 2);
        vr[i] = 2 * key * D + (((2 * (lane >> 4 & 1) + ((e & 3) >> 1)) ^ swz<D>(key)) << 4) + 8 * (e & 1);
    }
    auto in = [](const half_t* p, int bytes) __attribute__((always_inline)) { return reinterpret_cast<const half_t*>(reinterpret_cast<const char*>(p) + bytes); };
    float16_t zero;
#pragma unroll
    for (int e = 0; e < 16; ++e) zero[e] = 0.f;
    float d = 0.f, most = -1.f;             // -m once there is one, and what the sum of a tile's weights may be without a look at its scores

    // Tiles are requested one after the other: pointers, pitches and how many keys there are move along (formed anew for each tile they were 30 scalar instructions a step).
    const half_t *kp = keys.k(t0), *vp = keys.v(t0);
    int kpitch = keys.kpitch(t0), vpitch = keys.vpitch(t0), keys_left = keys.left(t0), tiles_left = t1 - t0;
    int k_off = sr * kpitch * 2 + sc, v_off = sr * vpitch * 2 + sc;
    auto ahead = [&](half_t* Kt, half_t* Vt) __attribute__((always_inline)) {
        // (none: nothing is read, zeros arrive, and the loads on their way are as many as ever)
        const int last_row = min(32, keys_left) - 1;
        const __amdgpu_buffer_rsrc_t ks = __builtin_amdgcn_make_buffer_rsrc((void*)kp, 0, tiles_left > 0 ? (last_row * kpitch + D) * 2 : 0, 0x00020000);
        const __amdgpu_buffer_rsrc_t vs = __builtin_amdgcn_make_buffer_rsrc((void*)vp, 0, tiles_left > 0 ? (last_row * vpitch + D) * 2 : 0, 0x00020000);
        fetch_tile<NL, D, 4>(ks, Kt + wave * RPI * D, k_off, 0, RPI * kpitch * 2);
        fetch_tile<NL, D, 4>(vs, Vt + wave * RPI * D, v_off, 0, RPI * vpitch * 2);
        kp += (int64_t)32 * kpitch; vp += (int64_t)32 * vpitch;
        keys_left -= 32; --tiles_left;
        if (__builtin_expect(keys_left <= 0 && tiles_left > 0, 0)) {
            const int t = t1 - tiles_left;
            kp = keys.k(t); vp = keys.v(t); kpitch = keys.kpitch(t); vpitch = keys.vpitch(t); keys_left = keys.left(t);
            k_off = sr * kpitch * 2 + sc; v_off = sr * vpitch * 2 + sc;
        }
    };
    auto step = [&](auto mask_tag, int t, const half_t* Kt, const half_t* Vt) __attribute__((always_inline)) {
        constexpr bool MASK = decltype(mask_tag)::value;
        // (addresses are formed here, of these and a stage's constant: hoisted out of the loop those of all stages would take 64 registers)
#pragma unroll
        for (int i = 0; i < NS; ++i) asm volatile("" : "+v"(kr[i]));
        asm volatile("" : "+v"(vr[0]), "+v"(vr[1]));
        // (what is read is requested at once: left to the compiler each read came right before its product, and was waited for)
        half8_t kw[NS], vw[2][NDB];
        auto value = [&](int u, int i) __attribute__((always_inline)) {       // of the keys 16 u + (0..3, 8..11) + 4 h, for one dimension
            const half4_t x = lds_read_tr16(in(Vt + u * 16 * D, vr[0] ^ (i << 6))), y = lds_read_tr16(in(Vt + u * 16 * D, vr[1] ^ (i << 6)));
            return half8_t{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
        };
#pragma unroll
        for (int i = 0; i < NS; ++i) kw[i] = *reinterpret_cast<const half8_t*>(in(Kt, kr[i]));
        if constexpr (!MASK) {
#pragma unroll
            for (int i = 0; i < NDB; ++i) vw[0][i] = value(0, i);
        }
        __builtin_amdgcn_sched_barrier(0);
        float16_t s;
#pragma unroll
        for (int i = 0; i < NS; ++i) s = mfma32(kw[i], qB[i], i == 0 ? zero : s);
        if constexpr (!MASK) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < NDB; ++i) vw[1][i] = value(1, i);
            __builtin_amdgcn_sched_barrier(0);
        }
        auto masked = [&]() __attribute__((always_inline)) {
            if constexpr (MASK) {
                const int lim = keys.lim(t, last) - 4 * h;
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = 8 * (e >> 2) + (e & 3) <= lim ? s[e] : -INFINITY;
            }
        };
        // (s becomes the weights)
        auto weights = [&]() __attribute__((always_inline)) {
            float sum[4];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[e] = fast_exp2(__builtin_fmaf(s[e], c, d));
                sum[e & 3] = e < 4 ? s[e] : sum[e & 3] + s[e];
            }
            return (sum[0] + sum[1]) + (sum[2] + sum[3]);
        };
        masked();
        float sum = weights();
        // (their sum shows whether one exceeds 2^15, and `most` whether there was no maximum yet: only then scores are looked through, formed once more.  With a maximum of each tile 46.8 us in the place
        // of 45.4 at head_dim 64, 138.3 in the place of 132.8 at 128, calls with one number a weight back to back: the chunks that cache_prefix_rows_kernel names)
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(sum <= most)) != 0, 0)) {
            asm volatile("" ::: "memory");
#pragma unroll
            for (int i = 0; i < NS; ++i) s = mfma32(*reinterpret_cast<const half8_t*>(in(Kt, kr[i])), qB[i], i == 0 ? zero : s);
            masked();
            const float up = fmaxf(m, half_max(max16(s) * c) - kBelow), alpha = up == -INFINITY ? 1.f : fast_exp2(m - up);
            m = up;
            l *= alpha;
            if (m != -INFINITY) { d = -m; most = 32768.f; }
#pragma unroll
            for (int i = 0; i < NDB; ++i) o[i] = o[i] * alpha;
            sum = weights();
        }
        l += sum;
        half8_t p[2], rest[2];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            p[e >> 3][e & 7] = (half_t)s[e];
            if constexpr (FINE) rest[e >> 3][e & 7] = (half_t)(s[e] - (float)p[e >> 3][e & 7]);
        }
        bool odd = false;
        if constexpr (MASK) {               // (as in the narrow form)
            bool bad = false;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < NDB; ++i) { bad = bad || odd_values(value(u, i)); __builtin_amdgcn_sched_barrier(0); }
            odd = __builtin_amdgcn_ballot_w64(bad) != 0;
            if (__builtin_expect(odd, 0)) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int lim = keys.lim(t, last) - 16 * u - 4 * h;
                    half8_t see;
#pragma unroll
                    for (int e = 0; e < 8; ++e) see[e] = 8 * (e >> 2) + (e & 3) <= lim ? (half_t)1.f : (half_t)0.f;
#pragma unroll
                    for (int i = 0; i < NDB; ++i)
#pragma unroll 1
                        for (int kind = 0; kind < 3; ++kind) {
                            const float16_t hit = mfma32(odd_kind(value(u, i), kind), see, zero);
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[i][e] += hit[e] > 0.f ? (kind == 0 ? INFINITY : kind == 1 ? -INFINITY : NAN) : 0.f;
                        }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < NDB; ++i) {
                half8_t v;
                if constexpr (MASK) { v = value(u, i); if (__builtin_expect(odd, 0)) v = finite_only(v); }
                else v = vw[u][i];
                o[i] = mfma32(v, p[u], o[i]);
                if constexpr (FINE) o[i] = mfma32(v, rest[u], o[i]);
            }
    };
    ahead(lds.k0, lds.v0); ahead(lds.k1, lds.v1); ahead(lds.k2, lds.v2);
    // (the wave's pieces of tile t are there; behind the barrier everyone's are, and everyone is done with tile t - 1, whose stage is the next one's)
    auto arrived = [&] {
        if constexpr (D == 128) asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };
    for (int t = t0; t < t1; t += 4) {
        for (; t + 4 <= min(t1, t_mask) && keys.whole(t, t + 4); t += 4) {
            arrived(); ahead(lds.k3, lds.v3); if (!idle) step(std::false_type{}, t, lds.k0, lds.v0);
            arrived(); ahead(lds.k0, lds.v0); if (!idle) step(std::false_type{}, t + 1, lds.k1, lds.v1);
            arrived(); ahead(lds.k1, lds.v1); if (!idle) step(std::false_type{}, t + 2, lds.k2, lds.v2);
            arrived(); ahead(lds.k2, lds.v2); if (!idle) step(std::false_type{}, t + 3, lds.k3, lds.v3);
        }
#pragma unroll 1
        for (int i = 0; i < 4 && t + i < t1; ++i) {
            arrived();
            ahead(lds.k((i + 3) & 3), lds.v((i + 3) & 3));
            if (!idle) step(std::true_type{}, t + i, lds.k(i), lds.v(i));
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}
#endif

// ------------------------------------------------------------------------------------------------ joining
struct JoinArgs { Parts parts; half_t* o; const int32_t* counts; int B, Hkv, M, G, rows; int64_t os[3]; Div by_g, by_m, by_hkv; };
hipError_t launch_cache16_join(const JoinArgs& a, int head_dim, hipStream_t s);

}  // namespace trn
