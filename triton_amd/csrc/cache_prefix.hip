// Attention of a batch behind a prefix that all its sequences share: o = softmax(scale * q [Kp ; K]^T) [Vp ; V].
//
// The prefix is the same for all, so the rows of all sequences that look at one KV head are one tall matrix there and read it once; its own keys a sequence reads for
// itself.  The softmax over both is that of its parts: with (m, l, O) of each, m = max m_i, l = sum l_i 2^(m_i - m), O likewise.  Few rows a sequence: one launch whose first
// workgroups have shares of the prefix and the others shares of the sequences' own keys, and one that joins them.  Many rows (chunks, prompts): tiles of one sequence's rows
// walk over the prefix and go on with its own keys, and nothing needs joining where there are tiles enough.
#include "cache16_attn.h"
#include "cache16_rules.h"

namespace trn {

struct PrefixArgs {
    const half_t *k, *v, *kp, *vp, *q; half_t* o;
    const int32_t *lengths, *counts;
    int B, Hkv, M, cap, P, G, R, causal, n_rt_p, ns_p, n_rt_o, ns_o, first;
    int64_t ks[3], vs[3], kps[2], vps[2], qs[3], os[3];
    float c;               // scale * log2(e)
    Parts parts;
    Div by_g, by_r, by_hkv, by_b, by_nsp, by_nso, by_wp, by_wo;
};

#if defined(__HIP_DEVICE_COMPILE__)
// Keys one after the other.
struct Run {
    const half_t *kp, *vp; int kpitch, vpitch, L;
    __device__ __forceinline__ const half_t* k(int t) const { return kp + (int64_t)t * 32 * kpitch; }
    __device__ __forceinline__ const half_t* v(int t) const { return vp + (int64_t)t * 32 * vpitch; }
    __device__ __forceinline__ int n(int t) const { return min(32, L - 32 * t); }
    __device__ __forceinline__ int lim(int t, int last) const { return last - 32 * t; }
};
// ... of the prefix, `split` tiles, and of the sequence behind them.
struct TwoRuns {
    const half_t *kp, *vp, *ko, *vo; int kpp, vpp, kpo, vpo, P, L, split;
    __device__ __forceinline__ const half_t* k(int t) const { return t < split ? kp + (int64_t)t * 32 * kpp : ko + (int64_t)(t - split) * 32 * kpo; }
    __device__ __forceinline__ const half_t* v(int t) const { return t < split ? vp + (int64_t)t * 32 * vpp : vo + (int64_t)(t - split) * 32 * vpo; }
    __device__ __forceinline__ int kpitch(int t) const { return t < split ? kpp : kpo; }
    __device__ __forceinline__ int vpitch(int t) const { return t < split ? vpp : vpo; }
    __device__ __forceinline__ int n(int t) const { return min(32, left(t)); }
    __device__ __forceinline__ int left(int t) const { return t < split ? P - 32 * t : L - 32 * (t - split); }
    __device__ __forceinline__ bool whole(int t, int to) const { return !(P & 31) || to < split || t >= split; }      // but for those that do not all see it
    __device__ __forceinline__ int lim(int t, int last) const { return t < split ? P - 1 - 32 * t : last - 32 * (t - split); }
};
// A row's result, piece by piece: to the output, or to the row's slot.
template <int D> __device__ __forceinline__ void put(const PrefixArgs& a, int slot, int b, int kvh, int r, int d0, float4_t x, float m, float l, bool once) {
    if (a.parts.slots > 1) {
        const int64_t at = (((int64_t)b * a.Hkv + kvh) * a.R + r) * a.parts.slots + slot;
        *reinterpret_cast<float4_t*>(a.parts.o + at * D + d0) = x;
        if (once) *reinterpret_cast<float2_t*>(a.parts.ml + 2 * at) = float2_t{m, l};
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    half4_t y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (half_t)(x[e] * inv);
    const int i = a.by_g.of(r), g = r - i * a.G;
    *reinterpret_cast<half4_t*>(a.o + b * a.os[0] + (int64_t)(kvh * a.G + g) * a.os[1] + i * a.os[2] + d0) = y;
}
__device__ __forceinline__ const half_t* query(const PrefixArgs& a, int b, int kvh, int r) {
    const int i = a.by_g.of(r), g = r - i * a.G;
    return a.q + b * a.qs[0] + (int64_t)(kvh * a.G + g) * a.qs[1] + i * a.qs[2];
}
#endif

// Tiles of 128 rows of one sequence, over the prefix and its own keys.  32 heads of 128 on 8, 4 chunks of up to 500 behind 4000 keys: 132 to 136 us back to back,
// 830 to 850 TFLOP/s (151 under the profiler; a share of 1024 keys took 53 us with one array for all stages, 32 so); 71 heads of 64 on 1, 16 of up to 5 behind 16001: 53 us, 380 TFLOP/s, where the exponentials
// bound it and the weights' second numbers take a fifth.
template <int D, bool FINE>
__global__ __launch_bounds__(256, D == 128 ? 2 : FINE ? 3 : 4) void cache_prefix_rows_kernel(const PrefixArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    TRN_LDS(D, lds);
    const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // (a KV head's workgroups follow each other at the distance of all KV heads: one XCD where those are a multiple of eight; the last rows, which see the most keys, first)
    const int x = a.by_hkv.of(blockIdx.x), kvh = blockIdx.x - x * a.Hkv, y = a.by_b.of(x), b = x - y * a.B, z = a.by_nsp.of(y), share = y - z * a.ns_p, rt = a.n_rt_p - 1 - z;
    const int L = length_of(a.lengths, b, a.cap), C = count_of(a.counts, b, a.M), rows = C * a.G, off = L - C;
    if (rt * 128 >= rows) return;
    auto sees = [&](int r) { return a.causal ? min(L, max(0, a.by_g.of(r) + off + 1)) : L; };      // own keys that a row sees
    const int r0 = rt * 128 + wave * 32, row = r0 + n, split = (a.P + 31) >> 5;
    const int T = split + ((sees(min(rt * 128 + 127, rows - 1)) + 31) >> 5);
    const int t0 = a.by_wp.of(T * share), t1 = a.by_wp.of(T * (share + 1));
    half8_t qB[D / 16];
    const half_t* const qp = query(a, b, kvh, min(row, rows - 1));
#pragma unroll
    for (int i = 0; i < D / 16; ++i) qB[i] = *reinterpret_cast<const half8_t*>(qp + 16 * i + 8 * h);
    const TwoRuns keys{a.kp + kvh * a.kps[0], a.vp + kvh * a.vps[0], a.k + b * a.ks[0] + kvh * a.ks[1], a.v + b * a.vs[0] + kvh * a.vs[1],
                       (int)a.kps[1], (int)a.vps[1], (int)a.ks[2], (int)a.vs[2], a.P, L, split};
    float16_t o[D / 32];
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
    wide_walk<D, FINE>(keys, t0, t1, split + (sees(min(r0, rows - 1)) >> 5), r0 >= rows, a.c, qB, sees(min(row, rows - 1)) - 1, lds, o, m, l);
    if (row >= rows) return;
    l = half_sum(l);
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            put<D>(a, share, b, kvh, row, 32 * i + 8 * e + 4 * h, float4_t{o[i][4 * e], o[i][4 * e + 1], o[i][4 * e + 2], o[i][4 * e + 3]}, m, l, i == 0 && e == 0 && h == 0);
#endif
}

// Few keys: eight waves have 16 rows of one sequence, over the prefix (whose pitches are the cache's) and its own keys, and nothing is joined by a second launch.
template <int D>
__global__ __launch_bounds__(512, 1) void cache_prefix_short_kernel(const PrefixArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    __shared__ __attribute__((aligned(1024))) half_t lds[16][32 * D];
    __shared__ NarrowStats<8> stats;
    auto area = [&](int w, int v) __attribute__((always_inline)) { return lds[2 * w + v]; };
    const int lane = threadIdx.x & 63, n = lane & 15, g4 = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int x = a.by_hkv.of(blockIdx.x), kvh = blockIdx.x - x * a.Hkv, rt = a.by_b.of(x), b = x - rt * a.B;
    const int L = length_of(a.lengths, b, a.cap), C = count_of(a.counts, b, a.M), rows = C * a.G, off = L - C, split = (a.P + 31) >> 5;
    if (rt * 16 >= rows) return;
    auto sees = [&](int r) { return a.causal ? min(L, max(0, a.by_g.of(r) + off + 1)) : L; };
    const int row = rt * 16 + n, T = split + ((sees(min(rt * 16 + 15, rows - 1)) + 31) >> 5), t0 = T * wave >> 3, t1 = T * (wave + 1) >> 3;
    half8_t qB[1][D / 32];
    const half_t* const qp = query(a, b, kvh, min(row, rows - 1));
#pragma unroll
    for (int i = 0; i < D / 32; ++i) qB[0][i] = *reinterpret_cast<const half8_t*>(qp + 32 * i + 8 * g4);
    const int last[1] = {sees(min(row, rows - 1)) - 1};
    TwoRuns keys{a.kp + kvh * a.kps[0], a.vp + kvh * a.vps[0], a.k + b * a.ks[0] + kvh * a.ks[1], a.v + b * a.vs[0] + kvh * a.vs[1],
                 (int)a.ks[2], (int)a.vs[2], (int)a.ks[2], (int)a.vs[2], a.P, L, split};
    float4_t o[D / 16][1];
    float m[1] = {-INFINITY}, l[1] = {0.f};
#pragma unroll
    for (int i = 0; i < D / 16; ++i) o[i][0] = float4_t{0.f, 0.f, 0.f, 0.f};
    const int t_mask = a.P & 31 ? split - 1 : split + (sees(rt * 16) >> 5);
    narrow_walk<D, 1, 1>(keys, t0, t1, min(t1, max(t0, t_mask)), (int)a.ks[2], (int)a.vs[2], a.c, qB, last, area(wave, 0), area(wave, 1), o, m, l);
    narrow_join<D, 1, 8>(area, stats, o, m, l, [&](int i, int d0, float4_t v, float mm, float ll, bool once) __attribute__((always_inline)) {
        if (rt * 16 + i < rows) put<D>(a, 0, b, kvh, rt * 16 + i, d0, v, mm, ll, once);
    });
#endif
}

// The rows of all sequences over shares of the prefix (the first workgroups), each sequence's rows over shares of its own keys (the others).  32 heads of 128 on 8: 32 sequences of up to 701 keys behind
// 8192 (104 MB) 28.5 us, 3.7 TB/s; 4 of 61 behind 1000 7.2 us, of which memory's latency is most.
template <int D, int NQ, bool WIDE>
__global__ __launch_bounds__(256, 2) void cache_prefix_parts_kernel(const PrefixArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    TRN_LDS(D, lds);
    __shared__ NarrowStats<4> stats;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool prefix = (int)blockIdx.x < a.first;
    const int j = prefix ? blockIdx.x : blockIdx.x - a.first;
    const int x = a.by_hkv.of(j), kvh = j - x * a.Hkv;
    if (WIDE && prefix) {
        const int n = lane & 31, h = lane >> 5, rt = a.by_nsp.of(x), share = x - rt * a.ns_p;
        const int r0 = rt * 128 + wave * 32, row = min(r0 + n, a.B * a.R - 1), b = a.by_r.of(row), r = row - b * a.R;
        const bool there = r0 + n < a.B * a.R && r < count_of(a.counts, b, a.M) * a.G;
        if (!__syncthreads_or(there)) return;
        half8_t qB[D / 16] = {};
        if (there) {
            const half_t* const qp = query(a, b, kvh, r);
#pragma unroll
            for (int i = 0; i < D / 16; ++i) qB[i] = *reinterpret_cast<const half8_t*>(qp + 16 * i + 8 * h);
        }
        const half_t *const kp = a.kp + kvh * a.kps[0], *const vp = a.vp + kvh * a.vps[0];
        const int T = (a.P + 31) >> 5;
        const TwoRuns keys{kp, vp, kp, vp, (int)a.kps[1], (int)a.vps[1], (int)a.kps[1], (int)a.vps[1], a.P, 0, T};
        float16_t o[D / 32];
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
        wide_walk<D, true>(keys, a.by_nsp.of(T * share), a.by_nsp.of(T * (share + 1)), T, __builtin_amdgcn_ballot_w64(there) == 0, a.c, qB, a.P - 1, lds, o, m, l);
        if (!there) return;
        l = half_sum(l);
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                put<D>(a, share, b, kvh, r, 32 * i + 8 * e + 4 * h, float4_t{o[i][4 * e], o[i][4 * e + 1], o[i][4 * e + 2], o[i][4 * e + 3]}, m, l, i == 0 && e == 0 && h == 0);
        return;
    }
    constexpr int RT = 16 * NQ;
    const int n = lane & 15, g4 = lane >> 4;
    int rt, share, b0 = 0, L = a.P, all = a.B * a.R, off = 0;      // the tile's rows are those of `all` from rt * RT on
    if (prefix) { rt = a.by_nsp.of(x); share = x - rt * a.ns_p; }
    else {
        const int y = a.by_b.of(x);
        b0 = x - y * a.B;
        rt = a.by_nso.of(y); share = y - rt * a.ns_o;
        const int C = count_of(a.counts, b0, a.M);
        L = length_of(a.lengths, b0, a.cap);
        all = C * a.G; off = L - C;
        if (rt * RT >= all) return;
    }
    auto sees = [&](int r) { return !prefix && a.causal ? min(L, max(0, a.by_g.of(r) + off + 1)) : L; };
    half8_t qB[NQ][D / 32] = {};
    int last[NQ];
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
        const int row = min(rt * RT + 16 * qb + n, all - 1), b = prefix ? a.by_r.of(row) : b0, r = prefix ? row - b * a.R : row;
        const bool there = rt * RT + 16 * qb + n < all && (!prefix || r < count_of(a.counts, b, a.M) * a.G);
        last[qb] = there ? sees(r) - 1 : -1;
        if (there) {
            const half_t* const qp = query(a, b, kvh, r);
#pragma unroll
            for (int i = 0; i < D / 32; ++i) qB[qb][i] = *reinterpret_cast<const half8_t*>(qp + 32 * i + 8 * g4);
        }
    }
    const int T = (sees(min(rt * RT + RT - 1, all - 1)) + 31) >> 5, w = share * 4 + wave;
    const Div& by = prefix ? a.by_wp : a.by_wo;
    const int t0 = by.of(T * w), t1 = by.of(T * (w + 1));
    Run keys{prefix ? a.kp + kvh * a.kps[0] : a.k + b0 * a.ks[0] + kvh * a.ks[1], prefix ? a.vp + kvh * a.vps[0] : a.v + b0 * a.vs[0] + kvh * a.vs[1],
             (int)(prefix ? a.kps[1] : a.ks[2]), (int)(prefix ? a.vps[1] : a.vs[2]), L};
    float4_t o[D / 16][NQ];
    float m[NQ], l[NQ];
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
        m[qb] = -INFINITY; l[qb] = 0.f;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[i][qb] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
    narrow_walk<D, NQ, 1>(keys, t0, t1, min(t1, max(t0, sees(rt * RT) >> 5)), keys.kpitch, keys.vpitch, a.c, qB, last, lds.k(wave), lds.v(wave), o, m, l);
    narrow_join<D, NQ, 4>([&](int w, int v) { return v ? lds.v(w) : lds.k(w); }, stats, o, m, l, [&](int i, int d0, float4_t v, float mm, float ll, bool once) __attribute__((always_inline)) {
        const int row = rt * RT + i;
        if (row >= all) return;
        const int b = prefix ? a.by_r.of(row) : b0, r = prefix ? row - b * a.R : row;
        if (prefix && r >= count_of(a.counts, b, a.M) * a.G) return;
        put<D>(a, prefix ? share : a.ns_p + share, b, kvh, r, d0, v, mm, ll, once);
    });
#endif
}

// ------------------------------------------------------------------------------------------------ joining
// D / 4 threads a row and `sg` groups of them, each with every sg-th slot.  A launch's latency at few rows (3.4 us for 128 with four slots), 4 TB/s at many (8.7 us for 30 MB).
template <int D>
__global__ __launch_bounds__(256) void cache16_join_kernel(const JoinArgs a, int sg) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int TPR = D / 4, GROUPS = 256 / TPR, AHEAD = 4;
    __shared__ float4_t red[256];
    __shared__ float2_t stat[GROUPS];
    const int grp = threadIdx.x / TPR, piece = threadIdx.x % TPR, nth = grp & (sg - 1), at = blockIdx.x * (GROUPS / sg) + grp / sg, row = min(at, a.rows - 1), slots = a.parts.slots;
    const float2_t* const ml = reinterpret_cast<const float2_t*>(a.parts.ml) + (int64_t)row * slots;
    const float* const po = a.parts.o + (int64_t)row * slots * D + 4 * piece;
    float top = -INFINITY, sum = 0.f;
    float4_t x = {0.f, 0.f, 0.f, 0.f};
    // (a thread's next four slots are requested at once, with their statistics, and joined to what there is so far)
    for (int s0 = nth; s0 < slots; s0 += AHEAD * sg) {
        float2_t st[AHEAD];
        float4_t got[AHEAD];
#pragma unroll
        for (int e = 0; e < AHEAD; ++e) {
            const int s = min(s0 + e * sg, slots - 1);
            st[e] = ml[s];
            got[e] = *reinterpret_cast<const float4_t*>(po + (int64_t)s * D);
        }
        float up = top;
#pragma unroll
        for (int e = 0; e < AHEAD; ++e) up = fmaxf(up, st[e].x);
        const float alpha = top == -INFINITY ? 0.f : fast_exp2(top - up);
        sum *= alpha; x = x * alpha; top = up;
#pragma unroll
        for (int e = 0; e < AHEAD; ++e) {
            if (s0 + e * sg >= slots) break;
            const float f = st[e].x == -INFINITY ? 0.f : fast_exp2(st[e].x - top);
            sum = __builtin_fmaf(st[e].y, f, sum);                 // (a sum of NaN stays)
            x = x + got[e] * f;
        }
    }
    const int bm = a.by_g.of(row), g = row - bm * a.G, bh = a.by_m.of(bm), i = bm - bh * a.M, b = a.by_hkv.of(bh), kvh = bh - b * a.Hkv;
    const bool there = at < a.rows && i < count_of(a.counts, b, a.M);
    if (sg > 1) {
        red[threadIdx.x] = x;
        if (piece == 0) stat[grp] = float2_t{top, sum};
        __syncthreads();
        if (nth != 0) return;
        float up = top;
        for (int k = 1; k < sg; ++k) up = fmaxf(up, stat[grp + k].x);
        float f = top == -INFINITY ? 0.f : fast_exp2(top - up);
        sum *= f; x = x * f;
        for (int k = 1; k < sg; ++k) {
            f = stat[grp + k].x == -INFINITY ? 0.f : fast_exp2(stat[grp + k].x - up);
            sum = __builtin_fmaf(stat[grp + k].y, f, sum);
            x = x + red[threadIdx.x + k * TPR] * f;
        }
    }
    if (!there) return;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    half4_t y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (half_t)(x[e] * inv);
    *reinterpret_cast<half4_t*>(a.o + b * a.os[0] + (int64_t)(kvh * a.G + g) * a.os[1] + i * a.os[2] + 4 * piece) = y;
#endif
}

hipError_t launch_cache16_join(const JoinArgs& a, int head_dim, hipStream_t s) {
    const int groups = 1024 / head_dim, sg = a.parts.slots > 4 ? groups < 8 ? groups : 8 : 1;
    const unsigned per = groups / sg, grid = ((unsigned)a.rows + per - 1) / per;
    if (head_dim == 128) hipLaunchKernelGGL((cache16_join_kernel<128>), dim3(grid), dim3(256), 0, s, a, sg);
    else hipLaunchKernelGGL((cache16_join_kernel<64>), dim3(grid), dim3(256), 0, s, a, sg);
    return hipGetLastError();
}

// ------------------------------------------------------------------------------------------------ host
int attn16_check(const trn_cache16* c, const void* q, const void* o, int32_t n_q_heads, int32_t seq_q, const int64_t* q_stride, const int64_t* o_stride, float scale,
                 const void* workspace) {
    if (!(scale > 0.f) || !(scale < INFINITY)) return TRN_E_SHAPE;
    int st = rows16_check(q, q_stride, c->batch, n_q_heads, seq_q, 16, false);
    if (st != TRN_OK) return st;
    if ((st = rows16_check(o, o_stride, c->batch, n_q_heads, seq_q, 8, true)) != TRN_OK) return st;
    const Extent eo = rows_extent(o, o_stride, c->batch, n_q_heads, seq_q, c->head_dim);
    if (meet(eo, rows_extent(q, q_stride, c->batch, n_q_heads, seq_q, c->head_dim))) return TRN_E_UNSUPPORTED;
    if (c->capacity && (meet(eo, rows_extent(c->k, c->k_stride, c->batch, c->n_kv_heads, c->capacity, c->head_dim)) ||
                        meet(eo, rows_extent(c->v, c->v_stride, c->batch, c->n_kv_heads, c->capacity, c->head_dim)))) return TRN_E_UNSUPPORTED;
    return workspace && (reinterpret_cast<uintptr_t>(workspace) & 255) ? TRN_E_ALIGN : TRN_OK;
}
// Rows of queries that 32 bits number, also times the slots of the workspace's statistics and the tiles of a walk.
int attn16_rows(int32_t batch, int32_t n_kv_heads, int32_t n_q_heads, int32_t seq_q) {
    if (batch < 0 || n_kv_heads <= 0 || n_q_heads <= 0 || n_q_heads % n_kv_heads || n_q_heads > (1 << 16) || seq_q < 0) return TRN_E_SHAPE;
    return (int64_t)batch * n_q_heads * seq_q > (1 << 26) ? TRN_E_UNSUPPORTED : TRN_OK;
}

}  // namespace trn

extern "C" int64_t trn_cache_prefix_attn_workspace_bytes(const trn_cache16* c, int32_t prefix_keys, int32_t n_q_heads, int32_t seq_q) {
    using namespace trn;
    if (!c || attn16_rows(c->batch, c->n_kv_heads, n_q_heads, seq_q) != TRN_OK || c->batch == 0 || seq_q == 0) return 0;
    if (c->capacity < 0 || c->capacity > (1 << 26) || prefix_keys < 0 || prefix_keys > (1 << 26) || (c->head_dim != 64 && c->head_dim != 128)) return 0;
    return plan_prefix(c->batch, c->n_kv_heads, c->capacity, c->head_dim, prefix_keys, n_q_heads, seq_q).bytes;
}

extern "C" int trn_cache_prefix_attn_f16(const trn_cache16* c, const trn_prefix* prefix, const void* q, void* o, int32_t n_q_heads, int32_t seq_q,
                                         const int64_t* q_stride, const int64_t* o_stride, float scale, int32_t causal, void* workspace,
                                         int64_t workspace_bytes, void* stream) {
    using namespace trn;
    int st = cache16_check(c);
    if (st != TRN_OK) return st;
    if (!prefix) return TRN_E_NULL;
    if ((st = attn16_rows(c->batch, c->n_kv_heads, n_q_heads, seq_q)) != TRN_OK) return st;
    if (prefix->keys < 0) return TRN_E_SHAPE;
    if (prefix->keys > (1 << 26)) return TRN_E_UNSUPPORTED;
    if (c->batch == 0 || seq_q == 0) return TRN_OK;
    if ((st = attn16_check(c, q, o, n_q_heads, seq_q, q_stride, o_stride, scale, workspace)) != TRN_OK) return st;
    PrefixArgs a{};
    for (int i = 0; i < 2 && prefix->keys; ++i) {
        const int64_t* const s2 = i ? prefix->v_stride : prefix->k_stride;
        const void* const p = i ? prefix->v : prefix->k;
        const int64_t s3[3] = {0, s2[0], s2[1]};
        if ((st = rows16_check(p, s3, 1, c->n_kv_heads, prefix->keys, 16, false)) != TRN_OK) return st;
        if (s2[1] < c->head_dim && prefix->keys > 1) return TRN_E_STRIDE;
        if (s2[1] > (1 << 23) && prefix->keys > 1) return TRN_E_UNSUPPORTED;
        if (meet(rows_extent(o, o_stride, c->batch, n_q_heads, seq_q, c->head_dim), rows_extent(p, s3, 1, c->n_kv_heads, prefix->keys, c->head_dim))) return TRN_E_UNSUPPORTED;
        (i ? a.vps : a.kps)[0] = s2[0]; (i ? a.vps : a.kps)[1] = s2[1];
    }
    for (int i = 0; i < 3; ++i) { a.ks[i] = c->k_stride[i]; a.vs[i] = c->v_stride[i]; a.qs[i] = q_stride[i]; a.os[i] = o_stride[i]; }
    // (a stride between tokens of which there is one may be anything, but a tile's rows are all addressed by it: the other part's then, or that of contiguous rows)
    const bool many_p = prefix->keys > 1, many_o = c->capacity > 1;
    if (!many_o) { a.ks[2] = many_p ? a.kps[1] : c->head_dim; a.vs[2] = many_p ? a.vps[1] : c->head_dim; }
    if (!many_p) { a.kps[1] = a.ks[2]; a.vps[1] = a.vs[2]; }
    PlanPrefix p = plan_prefix(c->batch, c->n_kv_heads, c->capacity, c->head_dim, prefix->keys, n_q_heads, seq_q);
    const bool shrt = p.short_rt > 0 && a.kps[1] == a.ks[2] && a.vps[1] == a.vs[2];
    if (shrt) { p.slots = 1; p.bytes = 0; p.first = (int64_t)c->batch * c->n_kv_heads * p.short_rt; p.second = 0; }
    if (p.first + p.second > 0xffffff) return TRN_E_SHAPE;            // (threads in 32 bits)
    if (p.bytes && (!workspace || workspace_bytes < p.bytes)) return TRN_E_SCRATCH;
    a.k = (const half_t*)c->k; a.v = (const half_t*)c->v; a.kp = (const half_t*)prefix->k; a.vp = (const half_t*)prefix->v; a.q = (const half_t*)q; a.o = (half_t*)o;
    a.lengths = c->lengths; a.counts = c->counts;
    a.B = c->batch; a.Hkv = c->n_kv_heads; a.M = seq_q; a.cap = c->capacity; a.P = prefix->keys; a.G = p.G; a.R = p.R; a.causal = causal != 0;
    a.n_rt_p = p.n_rt_p; a.ns_p = p.ns_p; a.n_rt_o = p.n_rt_o; a.ns_o = p.ns_o; a.first = (int)p.first;
    a.c = scale * kLog2e;
    a.parts = Parts{(float*)workspace, (float*)((char*)workspace + p.ml), p.slots};
    auto div = [](int64_t n) { return Div(n > 0 ? n : 1); };
    a.by_g = Div(p.G); a.by_r = Div(p.R); a.by_hkv = Div(c->n_kv_heads); a.by_b = Div(c->batch); a.by_nsp = div(p.ns_p); a.by_nso = div(p.ns_o);
    a.by_wp = p.one ? Div(p.ns_p) : div(4 * p.ns_p); a.by_wo = div(4 * p.ns_o);
    const hipStream_t s = (hipStream_t)stream;
    const dim3 grid((unsigned)(p.first + p.second)), block(256);
    const bool d128 = c->head_dim == 128;
    if (shrt) {
        if (d128) hipLaunchKernelGGL((cache_prefix_short_kernel<128>), grid, dim3(512), 0, s, a);
        else hipLaunchKernelGGL((cache_prefix_short_kernel<64>), grid, dim3(512), 0, s, a);
    } else if (p.one) {
        if (p.fine) {
            if (d128) hipLaunchKernelGGL((cache_prefix_rows_kernel<128, true>), grid, block, 0, s, a);
            else hipLaunchKernelGGL((cache_prefix_rows_kernel<64, true>), grid, block, 0, s, a);
        } else {
            if (d128) hipLaunchKernelGGL((cache_prefix_rows_kernel<128, false>), grid, block, 0, s, a);
            else hipLaunchKernelGGL((cache_prefix_rows_kernel<64, false>), grid, block, 0, s, a);
        }
    } else {
        auto launch = [&](auto nq, auto wide) {
            constexpr int NQ = decltype(nq)::value;
            constexpr bool WIDE = decltype(wide)::value;
            if (d128) hipLaunchKernelGGL((cache_prefix_parts_kernel<128, NQ, WIDE>), grid, block, 0, s, a);
            else hipLaunchKernelGGL((cache_prefix_parts_kernel<64, NQ, WIDE>), grid, block, 0, s, a);
        };
        const std::integral_constant<int, 1> one{};
        const std::integral_constant<int, 2> two{};
        if (p.nq == 1) p.wide ? launch(one, std::true_type{}) : launch(one, std::false_type{});
        else p.wide ? launch(two, std::true_type{}) : launch(two, std::false_type{});
    }
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && p.slots > 1) {
        JoinArgs j{a.parts, a.o, a.counts, a.B, a.Hkv, a.M, a.G, (int)((int64_t)a.B * a.Hkv * a.R), {a.os[0], a.os[1], a.os[2]}, a.by_g, Div(a.M), a.by_hkv};
        e = launch_cache16_join(j, c->head_dim, s);
    }
    return e == hipSuccess ? TRN_OK : TRN_E_LAUNCH;
}
