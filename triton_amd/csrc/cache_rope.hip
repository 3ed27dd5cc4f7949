// New tokens of an fp16 cache in one pass: queries and keys normalised by head and rotated by their positions, keys and values to their
// places.  x' = x rsqrt(mean x^2 + eps) gamma; a pair (a, b) at the angle t = position * inv_freq becomes (a cos t - b sin t, b cos t + a sin t).
//
// Each element is read once and written once, so memory bounds it.  A lane has four pairs of a row as two pieces of 8 bytes, p..p+3 and p + pairs.. (interleaved: 16 bytes that
// follow each other), so that a rotation stays within a lane; what is not rotated follows, eight elements a lane.  A row has D / 8 lanes, a wave 512 / D rows of one token, and as many
// such steps as its share of the token's heads: all have the same four angles a lane.  Those are formed once, one a lane: in 64 bits as far as the
// fraction of a turn, whose sine and cosine are taken in 32 (the argument is then off by 2^-25 of a turn at most), and handed to the lanes that share them.
//
// 4 prompts of up to 2047 tokens, 32 heads of 128 on 8, norms (163 MB): 32.5 us, 5.0 TB/s (37.7 with loads and stores through the caches; 32.5 with eight pairs a lane); 48 single tokens: 5.2 us.
#include "cache16.h"

namespace trn {

struct RopeArgs {
    const half_t *q, *k, *v, *gq, *gk; half_t *qo, *kc, *vc;
    const double* inv; const int32_t *pos, *lengths, *counts;
    int B, Hq, Hkv, M, cap, pairs, inter, axes, norm, offset, end[3];      // end: of all sections but the last
    int n_parts, steps, n_units;                                   // a token's rows in n_parts shares of `steps` steps
    float eps;
    Div by_parts, by_m;
    int64_t qs[3], qos[3], ks[3], vs[3], kcs[3], vcs[3];
};

#if defined(__HIP_DEVICE_COMPILE__)
template <int CTRL> __device__ __forceinline__ float moved(float x) { return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true)); }
// Over the D / 8 lanes of a row: neighbours, pairs of them, quads (mirrored within eight), eights (mirrored within sixteen).
template <int D> __device__ __forceinline__ float row_sum(float x) {
    x += moved<0xb1>(x);
    x += moved<0x4e>(x);
    x += moved<0x141>(x);
    if constexpr (D == 128) x += moved<0x140>(x);
    return x;
}
#endif

template <int D, bool INTER>
__global__ __launch_bounds__(256) void cache_rope_kernel(const RopeArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int LPR = D / 8, RPW = 64 / LPR, AHEAD = 4;
    const int lane = threadIdx.x & 63, j = lane % LPR, rg = lane / LPR;
    const int unit = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (unit >= a.n_units) return;
    const int token = a.by_parts.of(unit), part = unit - token * a.n_parts;
    const int b = a.by_m.of(token), i = token - b * a.M;

    // a lane's pieces
    const bool turns = 4 * j < a.pairs;
    const int c0 = INTER || !turns ? 8 * j : 4 * j, c1 = INTER || !turns ? 8 * j + 4 : 4 * j + a.pairs;
    // (strides by value: of a choice between members of `a` the compiler makes a load from the chosen place)
    const int64_t q_h = a.qs[1], k_h = a.ks[1], v_h = a.vs[1], qo_h = a.qos[1], kc_h = a.kcs[1], vc_h = a.vcs[1];
    const half_t* const qp = a.q + b * a.qs[0] + i * a.qs[2];
    const half_t* const kp = a.k + b * a.ks[0] + i * a.ks[2];
    const half_t* const vp = a.v + b * a.vs[0] + i * a.vs[2];
    // (the pair 4 j + rg % 4 is this lane's to find the angle of; its frequency is requested before it is known whether and where the token is)
    const int p = 4 * j + (rg & 3);
    double freq = 0.;
    if (turns) freq = a.inv[p];
    const int L = length_of(a.lengths, b, a.cap), C = count_of(a.counts, b, a.M);
    if (i >= C) return;
    const int at = L - C + i;                        // (below zero: of more new tokens than keys)
    float cs = 1.f, sn = 0.f;
    if (turns) {
        double where = (double)at + (double)a.offset;
        if (a.pos) {
            const int axis = (p >= a.end[0]) + (p >= a.end[1]) + (p >= a.end[2]);
            where = a.pos[((int64_t)axis * a.B + b) * a.M + i];
        }
        const double turn = where * freq * 0.15915494309189535;
        const float frac = (float)(turn - __builtin_rint(turn));
        sincospif(2.f * frac, &sn, &cs);
    }
    float co[4], si[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        co[e] = __shfl(cs, (e & (RPW - 1)) * LPR + j, 64);
        si[e] = __shfl(sn, (e & (RPW - 1)) * LPR + j, 64);
    }
    float gq[8], gk[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) gq[e] = gk[e] = 1.f;
    if (a.gq) {
        const half4_t u = *reinterpret_cast<const half4_t*>(a.gq + c0), w = *reinterpret_cast<const half4_t*>(a.gq + c1);
#pragma unroll
        for (int e = 0; e < 4; ++e) { gq[e] = (float)u[e]; gq[4 + e] = (float)w[e]; }
    }
    if (a.gk) {
        const half4_t u = *reinterpret_cast<const half4_t*>(a.gk + c0), w = *reinterpret_cast<const half4_t*>(a.gk + c1);
#pragma unroll
        for (int e = 0; e < 4; ++e) { gk[e] = (float)u[e]; gk[4 + e] = (float)w[e]; }
    }
    half_t* const qo = a.qo + b * a.qos[0] + i * a.qos[2];
    half_t* const kc = a.kc + b * a.kcs[0] + at * a.kcs[2];
    half_t* const vc = a.vc + b * a.vcs[0] + at * a.vcs[2];
    const int rows = a.Hq + (at >= 0 ? 2 * a.Hkv : 0), r0 = part * a.steps * RPW + rg;
    half4_t x[AHEAD], y[AHEAD];
    auto load = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < AHEAD; ++e) {
            const int r = r0 + (s0 + e) * RPW;
            const half_t* const src = r < a.Hq ? qp + r * q_h : r < a.Hq + a.Hkv ? kp + (r - a.Hq) * k_h : vp + (r - a.Hq - a.Hkv) * v_h;
            if (s0 + e >= a.steps || r >= rows) continue;
            if constexpr (INTER) {
                const half8_t w = __builtin_nontemporal_load(reinterpret_cast<const half8_t*>(src + c0));
                x[e] = half4_t{w[0], w[1], w[2], w[3]}; y[e] = half4_t{w[4], w[5], w[6], w[7]};
            } else {
                x[e] = __builtin_nontemporal_load(reinterpret_cast<const half4_t*>(src + c0));
                y[e] = __builtin_nontemporal_load(reinterpret_cast<const half4_t*>(src + c1));
            }
        }
    };
    const float inv_d = 1.f / D;
    for (int s0 = 0; s0 < a.steps; s0 += AHEAD) {
        load(s0);
#pragma unroll
        for (int e = 0; e < AHEAD; ++e) {
            const int r = r0 + (s0 + e) * RPW;
            const bool is_q = r < a.Hq, is_v = r >= a.Hq + a.Hkv, there = s0 + e < a.steps && r < rows;
            float f[8];
#pragma unroll
            for (int c = 0; c < 4; ++c) { f[c] = (float)x[e][c]; f[4 + c] = (float)y[e][c]; }
            if (a.norm) {
                float sum = 0.f;
#pragma unroll
                for (int c = 0; c < 8; ++c) sum = __builtin_fmaf(f[c], f[c], sum);
                const float n = 1.f / sqrtf(__builtin_fmaf(row_sum<D>(sum), inv_d, a.eps));
#pragma unroll
                for (int c = 0; c < 8; ++c) f[c] = f[c] * n * (is_q ? gq[c] : gk[c]);
            }
            float t[8];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int u = INTER ? 2 * c : c, w = INTER ? 2 * c + 1 : 4 + c;
                t[u] = f[u] * co[c] - f[w] * si[c];
                t[w] = f[w] * co[c] + f[u] * si[c];
            }
            half4_t u, w;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                u[c] = is_v ? x[e][c] : (half_t)(turns ? t[c] : f[c]);
                w[c] = is_v ? y[e][c] : (half_t)(turns ? t[4 + c] : f[4 + c]);
            }
            if (there) {
                half_t* const to = is_q ? qo + r * qo_h : is_v ? vc + (r - a.Hq - a.Hkv) * vc_h : kc + (r - a.Hq) * kc_h;
                if constexpr (INTER) __builtin_nontemporal_store(half8_t{u[0], u[1], u[2], u[3], w[0], w[1], w[2], w[3]}, reinterpret_cast<half8_t*>(to + c0));
                else {
                    __builtin_nontemporal_store(u, reinterpret_cast<half4_t*>(to + c0));
                    __builtin_nontemporal_store(w, reinterpret_cast<half4_t*>(to + c1));
                }
            }
        }
    }
#endif
}

// ------------------------------------------------------------------------------------------------ host
int rows16_check(const void* p, const int64_t* st, int64_t b, int64_t h, int64_t s, int bytes, bool written) {
    if (!p || !st) return TRN_E_NULL;
    if (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) return TRN_E_ALIGN;
    const int64_t n[3] = {b, h, s};
    for (int i = 0; i < 3; ++i) {
        if (st[i] < 0 || (written && n[i] > 1 && !st[i])) return TRN_E_STRIDE;
        if (n[i] > 1 && (2 * st[i]) % bytes) return TRN_E_ALIGN;
    }
    return TRN_OK;
}

int cache16_check(const trn_cache16* c, bool values) {
    if (!c) return TRN_E_NULL;
    if (c->batch < 0 || c->n_kv_heads <= 0 || c->capacity < 0) return TRN_E_SHAPE;
    if (c->head_dim != 64 && c->head_dim != 128) return TRN_E_UNSUPPORTED;
    if (c->capacity > (1 << 26) || c->batch > (1 << 24) || c->n_kv_heads > (1 << 16)) return TRN_E_UNSUPPORTED;
    if (c->batch == 0 || c->capacity == 0) return TRN_OK;
    for (int i = 0; i < (values ? 2 : 1); ++i) {
        const int64_t* const st = i ? c->v_stride : c->k_stride;
        const int e = rows16_check(i ? c->v : c->k, st, c->batch, c->n_kv_heads, c->capacity, 16, false);
        if (e != TRN_OK) return e;
        if (st[2] < c->head_dim && c->capacity > 1) return TRN_E_STRIDE;
        if (st[2] > (1 << 23) && c->capacity > 1) return TRN_E_UNSUPPORTED;            // (64 rows in 32-bit offsets)
    }
    return TRN_OK;
}

}  // namespace trn

extern "C" int trn_cache_rope_append_f16(const trn_cache16* c, const trn_rope* rope, const void* q, void* q_out, const void* k, const void* v, int32_t n_q_heads,
                                         int32_t tokens, const int64_t* q_stride, const int64_t* q_out_stride, const int64_t* k_stride,
                                         const int64_t* v_stride, void* stream) {
    using namespace trn;
    int st = cache16_check(c);
    if (st != TRN_OK) return st;
    if (!rope) return TRN_E_NULL;
    if (tokens < 0 || n_q_heads <= 0 || n_q_heads > (1 << 16)) return TRN_E_SHAPE;
    if (rope->pairs < 0 || rope->pairs % 4 || 2 * rope->pairs > c->head_dim) return TRN_E_UNSUPPORTED;
    if (rope->axes < 1 || rope->axes > 4) return TRN_E_UNSUPPORTED;
    if (rope->norm && !(rope->eps >= 0.f)) return TRN_E_SHAPE;
    int64_t all = 0;
    for (int i = 0; i < rope->axes; ++i) {
        if (rope->sections[i] < 0) return TRN_E_SHAPE;
        all += rope->sections[i];
    }
    if (all != rope->pairs) return TRN_E_SHAPE;
    if (rope->offset && rope->positions) return TRN_E_UNSUPPORTED;
    if (c->batch == 0 || tokens == 0) return TRN_OK;
    if ((rope->pairs && !rope->inv_freq) || (rope->axes > 1 && !rope->positions)) return TRN_E_NULL;
    if ((reinterpret_cast<uintptr_t>(rope->inv_freq) | reinterpret_cast<uintptr_t>(rope->gamma_q) | reinterpret_cast<uintptr_t>(rope->gamma_k)) & 7) return TRN_E_ALIGN;
    if (!rope->norm && (rope->gamma_q || rope->gamma_k)) return TRN_E_UNSUPPORTED;
    const int64_t B = c->batch, Hq = n_q_heads, Hkv = c->n_kv_heads, M = tokens, D = c->head_dim;
    if ((st = rows16_check(q, q_stride, B, Hq, M, 16, false)) != TRN_OK) return st;
    if ((st = rows16_check(q_out, q_out_stride, B, Hq, M, 16, true)) != TRN_OK) return st;
    if ((st = rows16_check(k, k_stride, B, Hkv, M, 16, false)) != TRN_OK) return st;
    if ((st = rows16_check(v, v_stride, B, Hkv, M, 16, false)) != TRN_OK) return st;
    // (nothing is written twice, or read after another lane has written it)
    const Extent eq = rows_extent(q, q_stride, B, Hq, M, D), eo = rows_extent(q_out, q_out_stride, B, Hq, M, D), ek = rows_extent(k, k_stride, B, Hkv, M, D),
                 ev = rows_extent(v, v_stride, B, Hkv, M, D);
    bool same = q == q_out;
    for (int i = 0; i < 3; ++i) same = same && (eq.n[i] == 1 || q_stride[i] == q_out_stride[i]);
    if ((!same && meet(eq, eo)) || meet(eo, ek) || meet(eo, ev)) return TRN_E_UNSUPPORTED;
    if (c->capacity > 0) {
        const int64_t S = c->capacity;
        if (rows16_check(c->k, c->k_stride, B, Hkv, S, 16, true) != TRN_OK || rows16_check(c->v, c->v_stride, B, Hkv, S, 16, true) != TRN_OK) return TRN_E_STRIDE;
        const Extent kc = rows_extent(c->k, c->k_stride, B, Hkv, S, D), vc = rows_extent(c->v, c->v_stride, B, Hkv, S, D);
        if (meet(kc, vc)) return TRN_E_UNSUPPORTED;
        for (const Extent* x : {&eq, &eo, &ek, &ev}) if (meet(kc, *x) || meet(vc, *x)) return TRN_E_UNSUPPORTED;
    }
    RopeArgs a{};
    a.q = (const half_t*)q; a.k = (const half_t*)k; a.v = (const half_t*)v; a.qo = (half_t*)q_out; a.kc = (half_t*)c->k; a.vc = (half_t*)c->v;
    a.gq = (const half_t*)rope->gamma_q; a.gk = (const half_t*)rope->gamma_k;
    a.inv = rope->inv_freq; a.pos = rope->positions; a.lengths = c->lengths; a.counts = c->counts;
    a.B = c->batch; a.Hq = n_q_heads; a.Hkv = c->n_kv_heads; a.M = tokens; a.cap = c->capacity;
    a.pairs = rope->pairs; a.inter = rope->interleaved != 0; a.axes = rope->axes; a.norm = rope->norm != 0; a.eps = rope->eps; a.offset = rope->offset;
    for (int i = 0, sum = 0; i < 3; ++i) { sum += i < rope->axes ? rope->sections[i] : 0; a.end[i] = i + 1 < rope->axes ? sum : 0x7fffffff; }
    for (int i = 0; i < 3; ++i) {
        a.qs[i] = q_stride[i]; a.qos[i] = q_out_stride[i]; a.ks[i] = k_stride[i]; a.vs[i] = v_stride[i]; a.kcs[i] = c->k_stride[i]; a.vcs[i] = c->v_stride[i];
    }
    const int64_t rpw = 512 / D, all_steps = (Hq + 2 * Hkv + rpw - 1) / rpw;
    int64_t parts = B * M >= 8192 ? 1 : (8192 + B * M - 1) / (B * M);
    if (parts > all_steps) parts = all_steps;
    a.steps = (int)((all_steps + parts - 1) / parts);
    a.n_parts = (int)((all_steps + a.steps - 1) / a.steps);
    const int64_t units = B * M * a.n_parts, groups = (units + 3) / 4;
    if (groups > 0xffffff) return TRN_E_SHAPE;                       // (threads in 32 bits)
    a.n_units = (int)units;
    a.by_parts = Div(a.n_parts); a.by_m = Div(M);
    const dim3 grid((unsigned)groups), block(256);
    const hipStream_t s = (hipStream_t)stream;
    // (nothing to turn: pieces as the interleaved form has them, 16 bytes)
    if (a.inter || a.pairs == 0) {
        if (D == 128) hipLaunchKernelGGL((cache_rope_kernel<128, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((cache_rope_kernel<64, true>), grid, block, 0, s, a);
    } else {
        if (D == 128) hipLaunchKernelGGL((cache_rope_kernel<128, false>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((cache_rope_kernel<64, false>), grid, block, 0, s, a);
    }
    return hipGetLastError() == hipSuccess ? TRN_OK : TRN_E_LAUNCH;
}
