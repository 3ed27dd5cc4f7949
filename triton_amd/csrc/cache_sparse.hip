// Attention over those blocks of a long cache that a cheap score selects for each query: bounds of the blocks' keys by channel, a score from them, the selection,
// and the attention over what is selected.
//
// A key k within lo <= k <= hi scores q . k <= sum_d max(q_d lo_d, q_d hi_d) = sum_d (max(q_d, 0) hi_d + min(q_d, 0) lo_d): of a block of 64 keys that reads 2 rows in the place of
// 64, and is a product of matrices.  Selected is by that sum rounded from 64 bits, so that the order of additions does not show.  Up to 8192 blocks the matrix pipe computes it in 32 bits,
// with a bound of how far that is off, and 64 bits are spent where it matters: on blocks within twice the bound of the last score that is taken, if not all of them are.
#include "cache16_attn.h"
#include "cache16_rules.h"

namespace trn {

#if defined(__HIP_DEVICE_COMPILE__)
template <int CTRL> __device__ __forceinline__ float rotated(float x) { return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true)); }
#endif

// ------------------------------------------------------------------------------------------------ bounds
struct BoundsArgs { const half_t* k; half_t* bounds; const int32_t *lengths, *counts; int B, Hkv, M, cap, block, nb, per; int64_t ks[3]; Div by_per, by_hkv; };

// A workgroup has every per-th touched block of a head: all keys that it holds are read once.  One new token of 8 heads: 3.4 us, a launch and two loads one behind the other.
template <int D>
__global__ __launch_bounds__(256) void cache_bounds_kernel(const BoundsArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int LPR = D / 8, RPP = 256 / LPR, NP = 128 / RPP;
    __shared__ float lo_all[4][D], hi_all[4][D];
    const int bh = a.by_per.of(blockIdx.x), nth = blockIdx.x - bh * a.per, b = a.by_hkv.of(bh), h = bh - b * a.Hkv;
    const int L = length_of(a.lengths, b, a.cap), C = min(count_of(a.counts, b, a.M), L);
    if (C == 0) return;
    const int sub = threadIdx.x % LPR, r0 = threadIdx.x / LPR, wave = threadIdx.x >> 6, t = threadIdx.x;
    const half_t* const kh = a.k + b * a.ks[0] + h * a.ks[1] + sub * 8;
    for (int blk = (L - C) / a.block + nth; blk * a.block < L; blk += a.per) {
        const int base = blk * a.block, rows = min(a.block, L - base);
        half8_t x[NP];
#pragma unroll
        for (int p = 0; p < NP; ++p) x[p] = *reinterpret_cast<const half8_t*>(kh + (int64_t)(base + min(p * RPP + r0, rows - 1)) * a.ks[2]);      // (a row twice changes nothing)
        float lo[8], hi[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) { lo[e] = INFINITY; hi[e] = -INFINITY; }
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
            for (int e = 0; e < 8; ++e) { lo[e] = fminf(lo[e], (float)x[p][e]); hi[e] = fmaxf(hi[e], (float)x[p][e]); }
        // (over the lanes of one channel group, 8 and 16 apart and more, without LDS)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (D == 64) { lo[e] = fminf(lo[e], rotated<0x128>(lo[e])); hi[e] = fmaxf(hi[e], rotated<0x128>(hi[e])); }
            lo[e] = -quad_max(-lo[e]); hi[e] = quad_max(hi[e]);
        }
        if ((t & 63) < LPR) {
#pragma unroll
            for (int e = 0; e < 8; ++e) { lo_all[wave][sub * 8 + e] = lo[e]; hi_all[wave][sub * 8 + e] = hi[e]; }
        }
        __syncthreads();
        if (t < 2 * D) {
            const float (*all)[D] = t < D ? lo_all : hi_all;
            const int d = t < D ? t : t - D;
            const float w = all[0][d], x1 = all[1][d], y = all[2][d], z = all[3][d];
            a.bounds[((int64_t)bh * a.nb + blk) * 2 * D + t] = (half_t)(t < D ? fminf(fminf(w, x1), fminf(y, z)) : fmaxf(fmaxf(w, x1), fmaxf(y, z)));
        }
        __syncthreads();
    }
#endif
}

// ------------------------------------------------------------------------------------------------ scores
struct SelectArgs {
    const half_t *q, *bounds; const int32_t *lengths, *counts;
    float *scores, *norms; int32_t* selected;
    int B, Hkv, M, cap, G, block_shift, nb, top, sink, recent, i0, n, steps;      // queries i0 .. i0 + n
    int64_t nbp, qs[3];
    Div by_hkv, by_n;
};

#if defined(__HIP_DEVICE_COMPILE__)
template <int CTRL> __device__ __forceinline__ double moved64(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xf, 0xf, true), hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xf, 0xf, true);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int CTRL, int ROWS = 0xf> __device__ __forceinline__ uint32_t moved32(uint32_t x) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, true); }
// Over 16 lanes, by rotations.
__device__ __forceinline__ float row_max(float x) {
    x = fmaxf(x, rotated<0x121>(x));
    x = fmaxf(x, rotated<0x122>(x));
    x = fmaxf(x, rotated<0x124>(x));
    return fmaxf(x, rotated<0x128>(x));
}
// x of this lane and those below it, of an operation that zero leaves as it is; all of them in the last lane.
template <class F> __device__ __forceinline__ uint32_t scan64(uint32_t x, F f) {
    x = f(x, moved32<0x111>(x));       // row_shr:1, 2, 4, 8
    x = f(x, moved32<0x112>(x));
    x = f(x, moved32<0x114>(x));
    x = f(x, moved32<0x118>(x));
    x = f(x, moved32<0x142, 0xa>(x));  // the first and third row's last lane to the rows behind them
    return f(x, moved32<0x143, 0xc>(x));
}
template <class F> __device__ __forceinline__ uint32_t all64(uint32_t x, F f) { return (uint32_t)__builtin_amdgcn_readlane((int)scan64(x, f), 63); }
struct Or { __device__ __forceinline__ uint32_t operator()(uint32_t x, uint32_t y) const { return x | y; } };
struct Add { __device__ __forceinline__ uint32_t operator()(uint32_t x, uint32_t y) const { return x + y; } };
struct Max { __device__ __forceinline__ uint32_t operator()(uint32_t x, uint32_t y) const { return max(x, y); } };
// Scores as whole numbers of the same order; NaN is zero, the least.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x);
    return x != x ? 0u : u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float(u >> 31 ? u ^ 0x80000000u : ~u); }
#endif

// Scores by the matrix pipe.  A wave has 16 blocks or two times 16, whose bounds it holds as operands (lane 16 g + n: block n, channels 8 g..+7 of each 32).  HEADS: a query's heads are the other
// operand, 16 at a time, and their largest is taken over lanes; otherwise 16 queries are, their heads one after the other, and the largest stays in a lane: twice 16 blocks then, as rows in this shape are
// loaded at 16 bytes a clock and compute unit, which bounds it (256 queries on 512 blocks, 32 heads of 128 on 8: 11.4 us with 16 blocks, 10.0 with 32).
// norms: the largest |bound| vector (of each channel's larger end) of every 16 blocks, squared; infinite where a bound is not finite.
template <int D, bool HEADS>
__global__ __launch_bounds__(256) void cache_scores_kernel(const SelectArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int NI = D / 32, SETS = HEADS ? 1 : 2;
    const int lane = threadIdx.x & 63, n = lane & 15, g4 = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int bh = blockIdx.z, b = a.by_hkv.of(bh), kvh = bh - b * a.Hkv, set = (blockIdx.x * 4 + wave) * SETS;
    // (bounds are requested before it is known how many of them count; queries are read only where they are there)
    half8_t lo[SETS][NI], hi[SETS][NI], q[NI];
#pragma unroll
    for (int u = 0; u < SETS; ++u) {
        const half_t* const bp = a.bounds + ((int64_t)bh * a.nb + min((set + u) * 16 + n, a.nb - 1)) * 2 * D + 8 * g4;
#pragma unroll
        for (int i = 0; i < NI; ++i) { lo[u][i] = *reinterpret_cast<const half8_t*>(bp + 32 * i); hi[u][i] = *reinterpret_cast<const half8_t*>(bp + D + 32 * i); }
    }
    const half_t* const qh = a.q + b * a.qs[0] + (int64_t)kvh * a.G * a.qs[1] + 8 * g4;
    const int j_first = blockIdx.y * a.steps * (HEADS ? 1 : 16);
    auto load = [&](int i, int g) __attribute__((always_inline)) {
        const half_t* const p = qh + (int64_t)g * a.qs[1] + (int64_t)i * a.qs[2];
#pragma unroll
        for (int e = 0; e < NI; ++e) q[e] = *reinterpret_cast<const half8_t*>(p + 32 * e);
    };
    const int C = min(count_of(a.counts, b, a.M), a.i0 + a.n), L = length_of(a.lengths, b, a.cap), blocks = L > 0 ? ((L - 1) >> a.block_shift) + 1 : 0;
    if (a.i0 + j_first >= C) return;
    if constexpr (HEADS) load(a.i0 + j_first, min(n, a.G - 1));
    if (set * 16 >= blocks || blocks <= a.top) return;      // (where all blocks are taken no score is needed)
    if (blockIdx.y == 0) {
#pragma unroll
        for (int u = 0; u < SETS; ++u) {
            float sum = 0.f;
            bool bad = false;
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                bad = bad || odd_values(lo[u][i]) || odd_values(hi[u][i]);
#pragma unroll
                for (int e = 0; e < 8; ++e) { const float x = fmaxf(fabsf((float)lo[u][i][e]), fabsf((float)hi[u][i][e])); sum = __builtin_fmaf(x, x, sum); }
            }
            sum = quad_sum(bad ? INFINITY : sum);
            sum = row_max((set + u) * 16 + n < blocks ? sum : 0.f);
            if (lane == 0) a.norms[(int64_t)bh * (a.nbp >> 4) + set + u] = sum;
        }
    }
    const half8_t nil = {};
    float4_t best[SETS];
    auto add = [&](const half8_t (&q)[NI]) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < SETS; ++u) {
            float4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < NI; ++e) {
                x = mfma16(hi[u][e], __builtin_elementwise_max(q[e], nil), x);
                x = mfma16(lo[u][e], __builtin_elementwise_min(q[e], nil), x);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) best[u][e] = fmaxf(best[u][e], x[e]);
        }
    };
    float* const to = a.scores + (int64_t)bh * a.n * a.nbp + set * 16 + 4 * g4;
    for (int s = 0; s < a.steps; ++s) {
        const int j0 = j_first + s * (HEADS ? 1 : 16), i = a.i0 + j0 + (HEADS ? 0 : n);
        if (a.i0 + j0 >= C) return;
#pragma unroll
        for (int u = 0; u < SETS; ++u) best[u] = float4_t{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if constexpr (HEADS) {
            for (int g0 = 0; g0 < a.G; g0 += 16) {
                if (s > 0 || g0 > 0) load(i, min(g0 + n, a.G - 1));
                add(q);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) best[0][e] = row_max(best[0][e]);
            if (n == 0) *reinterpret_cast<float4_t*>(to + j0 * a.nbp) = best[0];
        } else {
            load(min(i, C - 1), 0);
            for (int g = 0; g < a.G; ++g) {
                half8_t now[NI];
#pragma unroll
                for (int e = 0; e < NI; ++e) now[e] = q[e];
                load(min(i, C - 1), min(g + 1, a.G - 1));
                add(now);
            }
#pragma unroll
            for (int u = 0; u < SETS; ++u)       // (a row has room for a multiple of 64 blocks)
                if (i < C) *reinterpret_cast<float4_t*>(to + (j0 + n) * a.nbp + 16 * u) = best[u];
        }
    }
#endif
}

// D / 8 lanes have a block, eight channels each; a wave 512 / D blocks at a time.
template <int D>
__global__ __launch_bounds__(256) void cache_scores64_kernel(const SelectArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int LPR = D / 8, PER = 64 / LPR;
    const int lane = threadIdx.x & 63, sub = lane % LPR, wave = threadIdx.x >> 6;
    const int bh = blockIdx.z, b = a.by_hkv.of(bh), kvh = bh - b * a.Hkv, i = a.i0 + blockIdx.y;
    const int L = length_of(a.lengths, b, a.cap), C = count_of(a.counts, b, a.M), last = L - C + i, n = last < 0 ? 0 : (last >> a.block_shift) + 1;
    // (no row of bounds is needed where all blocks are taken, or for those that are taken anyway)
    if (i >= C || n <= a.top) return;
    const half_t* const qp = a.q + b * a.qs[0] + (int64_t)kvh * a.G * a.qs[1] + i * a.qs[2] + sub * 8;
    float* const to = a.scores + ((int64_t)bh * a.n + blockIdx.y) * a.nbp;
    for (int s = 0; s < a.steps; ++s) {
        const int blk = ((blockIdx.x * a.steps + s) * 4 + wave) * PER + lane / LPR;
        if (((blockIdx.x * a.steps + s) * 4 + wave) * PER >= n) return;
        const half_t* const bp = a.bounds + ((int64_t)bh * a.nb + min(blk, n - 1)) * 2 * D + sub * 8;
        const half8_t lo8 = *reinterpret_cast<const half8_t*>(bp), hi8 = *reinterpret_cast<const half8_t*>(bp + D);
        float lo[8], hi[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) { lo[e] = (float)lo8[e]; hi[e] = (float)hi8[e]; }
        double best = -INFINITY;
        for (int g = 0; g < a.G; ++g) {
            const half8_t q8 = *reinterpret_cast<const half8_t*>(qp + g * a.qs[1]);
            double x = 0., y = 0.;
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float q0 = (float)q8[e], q1 = (float)q8[e + 1];
                x += (double)fmaxf(q0 * lo[e], q0 * hi[e]);
                y += (double)fmaxf(q1 * lo[e + 1], q1 * hi[e + 1]);
            }
            x += y;
            x += moved64<0xb1>(x);
            x += moved64<0x4e>(x);
            x += moved64<0x141>(x);
            if constexpr (D == 128) x += moved64<0x140>(x);
            best = fmax(best, x);
        }
        if (sub == 0 && blk < n) to[blk] = (float)best;
    }
#endif
}

// ------------------------------------------------------------------------------------------------ selection
#if defined(__HIP_DEVICE_COMPILE__)
// What the waves of a selection tell each other.
template <int T> struct SelectShared { int count[4][256]; uint32_t any[T / 64], none[T / 64], norm_q[T / 64], norm_b[T / 64], least[T / 64]; int sure[T / 64], maybe[T / 64], taken[T / 64]; };

// The want-th largest of a workgroup's open keys (bit r: key[r]; any, none: the bits that are set, and not set, in some of them), digit by digit of eight bits from the first one on that they differ
// in.  Returns the least number that the first `want` keys reach -- the want-th largest itself, or, where all keys of a digit are among them, that digit's first number --
// and in `left` how many of those that equal it belong to them (0: all that reach it).  `count` is zero before.
template <int T, int REGS>
__device__ __forceinline__ uint32_t kth(const uint32_t (&key)[REGS], uint32_t open, uint32_t any, uint32_t none, int want, int& left, int (&count)[4][256]) {
    const int lane = threadIdx.x & 63;
    const uint32_t differ = any & none;
    left = want;
    if (differ == 0) return any;
    int above = 32 - __builtin_clz(differ), pass = 0;
    uint32_t known = above == 32 ? 0u : any >> above << above;
    while (above > 0) {
        const int shift = max(above - 8, 0);
        const uint32_t width = (1u << (above - shift)) - 1;
        int (&bins)[256] = count[pass++];
#pragma unroll
        for (int r = 0; r < REGS; ++r)
            if ((open >> r & 1) && (above == 32 || (key[r] ^ known) >> above == 0)) atomicAdd(&bins[255 - (key[r] >> shift & width)], 1);      // (the largest first)
        __syncthreads();
        // (every wave looks for itself: four digits a lane)
        int c[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] = bins[4 * lane + e];
        const int mine = c[0] + c[1] + c[2] + c[3], upto = (int)scan64((uint32_t)mine, Add{});
        const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto >= left));
        int rest = left - (upto - mine), e = 0, in = c[0];
#pragma unroll
        for (int f = 1; f < 4; ++f)
            if (e == f - 1 && rest > in) { rest -= in; e = f; in = c[f]; }
        const int found = __builtin_amdgcn_readlane(4 * lane + e, at), done = __builtin_amdgcn_readlane(rest == in, at);
        left = __builtin_amdgcn_readlane(rest, at);
        known |= (uint32_t)(255 - found) << shift;
        if (done) { left = 0; break; }
        above = shift;
    }
    return known;
}
// The score of one block in 64 bits, by a wave: D / 8 lanes have eight channels each, and the others as many query heads at a time.
template <int D>
__device__ __forceinline__ float score64(const SelectArgs& a, const half_t* q, int bh, int blk) {
    constexpr int LPR = D / 8, PER = 64 / LPR;
    const int lane = threadIdx.x & 63, sub = lane % LPR;
    const half_t* const bp = a.bounds + ((int64_t)bh * a.nb + blk) * 2 * D + sub * 8;
    const half8_t lo = *reinterpret_cast<const half8_t*>(bp), hi = *reinterpret_cast<const half8_t*>(bp + D);
    double best = -INFINITY;
    for (int g0 = 0; g0 < a.G; g0 += PER) {
        const half8_t q8 = *reinterpret_cast<const half8_t*>(q + (int64_t)min(g0 + lane / LPR, a.G - 1) * a.qs[1] + sub * 8);
        double x = 0.;
#pragma unroll
        for (int e = 0; e < 8; ++e) x += (double)fmaxf((float)q8[e] * (float)lo[e], (float)q8[e] * (float)hi[e]);
#pragma unroll
        for (int d = 1; d < LPR; d *= 2) x += __shfl_xor(x, d, 64);
        best = fmax(best, x);
    }
#pragma unroll
    for (int d = LPR; d < 64; d *= 2) best = fmax(best, __shfl_xor(best, d, 64));
    return (float)best;
}

// A workgroup has one query of one KV head, and of its blocks' scores REGS a thread.  Scores s come with a bound e of how far they are off the definition's, r.  If t is the last of s that would be
// taken, the last of r is within e of t: s > t + 2 e belongs to what is taken, s < t - 2 e does not, and between them the definition decides, if that is needed.  e: matrix instructions add 128 products
// (of the two of a channel one is zero) and eight earlier sums, and may cut off 2^-23 of the largest sum at each: 136 2^-23 < 1.07 2^-16 of the sum of the products' magnitudes, which is |q| |b| at
// most; the rounding of r, and of t + 2 e, is 2^-24 each: e = 1.15 2^-16 |q| |b|.  (Products of fp16 numbers are normal in 32 bits; numbers below 2^-14 enter the pipe as they are.)
template <int REGS> struct SelectInputs { float s[REGS], bb; };
// What a selection needs, requested before it is known how many blocks there are: a thread's scores, neighbours; norms.
template <int D, int T, int REGS>
__device__ __forceinline__ void select_inputs(const SelectArgs& a, SelectInputs<REGS>& in, int bh, const float* from) {
    const int tid = threadIdx.x, x0 = tid * REGS;
#pragma unroll
    for (int r = 0; r < REGS; r += 4) {
        const float4_t v = x0 + r < a.nbp ? *reinterpret_cast<const float4_t*>(from + x0 + r) : float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 4; ++e) in.s[r + e] = v[e];
    }
    static_assert(T * REGS <= 16 * T, "a norm a thread");
    in.bb = tid < a.nbp >> 4 ? a.norms[(int64_t)bh * (a.nbp >> 4) + tid] : 0.f;
}
// Eight channels of one head a thread, of the query i, which is there.
template <int D>
__device__ __forceinline__ half8_t select_query(const SelectArgs& a, int b, int kvh, int i) {
    constexpr int LPR = D / 8;
    return *reinterpret_cast<const half8_t*>(a.q + b * a.qs[0] + (int64_t)(kvh * a.G + min((int)threadIdx.x / LPR, a.G - 1)) * a.qs[1] + (int64_t)i * a.qs[2] + (threadIdx.x & 63) % LPR * 8);
}

template <int D, int T, int REGS>
__device__ __forceinline__ void select_blocks(const SelectArgs& a, SelectShared<T>& sh, const SelectInputs<REGS>& in, half8_t q8, int bh, int b, int kvh, int i, int n, int32_t* to) {
    constexpr int W = T / 64, LPR = D / 8;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), x0 = tid * REGS;
    const float (&s)[REGS] = in.s;
    const half_t* const q = a.q + b * a.qs[0] + (int64_t)kvh * a.G * a.qs[1] + (int64_t)i * a.qs[2];
    float bb = tid < (n + 15) >> 4 ? in.bb : 0.f, qq = 0.f;
    for (int g0 = 0; g0 < a.G; g0 += T / LPR) {
        if (g0) q8 = *reinterpret_cast<const half8_t*>(q + (int64_t)min(g0 + tid / LPR, a.G - 1) * a.qs[1] + lane % LPR * 8);
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = __builtin_fmaf((float)q8[e], (float)q8[e], sum);
        if (odd_values(q8)) sum = INFINITY;
        sum += rotated<0xb1>(sum);
        sum += rotated<0x4e>(sum);
        sum += rotated<0x141>(sum);
        if constexpr (D == 128) sum += rotated<0x140>(sum);
        qq = fmaxf(qq, sum);
    }
    const int lo = a.sink, hi = n - a.recent;                     // what is chosen from (top > their number: not empty)
    int want = a.top - a.sink - a.recent;
#pragma unroll
    for (int e = 0; e < 4; ++e) for (int c = tid; c < 256; c += T) sh.count[e][c] = 0;
    uint32_t key[REGS], open = 0, any = 0, none = 0, sure = 0, maybe = 0, forced = 0;
#pragma unroll
    for (int r = 0; r < REGS; ++r) {
        const int x = x0 + r;
        key[r] = ordered(s[r]);
        if (x >= lo && x < hi) { open |= 1u << r; any |= key[r]; none |= ~key[r]; }
        else if (x < n) forced |= 1u << r;
    }
    if (want > 0) {
        // (magnitudes are ordered as their bits)
        any = all64(any, Or{}); none = all64(none, Or{});
        uint32_t nq = all64(__float_as_uint(qq), Max{}), nb = all64(__float_as_uint(bb), Max{});
        if (lane == 0) { sh.any[wave] = any; sh.none[wave] = none; sh.norm_q[wave] = nq; sh.norm_b[wave] = nb; }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) { any |= sh.any[w]; none |= sh.none[w]; nq = max(nq, sh.norm_q[w]); nb = max(nb, sh.norm_b[w]); }
        int left;
        const uint32_t reach = kth<T, REGS>(key, open, any, none, want, left, sh.count);
        // the last score that is taken: the least that reaches
        uint32_t least = 0;
#pragma unroll
        for (int r = 0; r < REGS; ++r) if ((open >> r & 1) && key[r] >= reach) least = max(least, ~key[r]);
        least = all64(least, Max{});
        if (lane == 0) sh.least[wave] = least;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) least = max(least, sh.least[w]);
        const float t = unordered(~least), e2 = 2.3f * 0x1p-16f * sqrtf(__uint_as_float(nq)) * sqrtf(__uint_as_float(nb));
        const bool bound = e2 < INFINITY;
        const float above = bound ? t + e2 : INFINITY, below = bound ? t - e2 : -INFINITY;
#pragma unroll
        for (int r = 0; r < REGS; ++r)
            if (open >> r & 1) {
                if (s[r] > above) sure |= 1u << r;
                else if (!(s[r] < below)) maybe |= 1u << r;
            }
        const uint32_t both = all64(__popc(sure) << 16 | __popc(maybe), Add{});
        if (lane == 0) { sh.sure[wave] = both >> 16; sh.maybe[wave] = both & 0xffff; }
        __syncthreads();
        int n_maybe = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) { want -= sh.sure[w]; n_maybe += sh.maybe[w]; }
        if (n_maybe == want) sure |= maybe;
        else {
            any = none = 0;
#pragma unroll
            for (int r = 0; r < REGS; ++r) {
                uint64_t todo = __builtin_amdgcn_ballot_w64(maybe >> r & 1);
                while (todo) {
                    const int bit = __builtin_ctzll(todo);
                    todo &= todo - 1;
                    const float x = score64<D>(a, q, bh, (wave * 64 + bit) * REGS + r);
                    if (lane == bit) key[r] = ordered(x);
                }
                if (maybe >> r & 1) { any |= key[r]; none |= ~key[r]; }
            }
            any = all64(any, Or{}); none = all64(none, Or{});
#pragma unroll
            for (int e = 0; e < 4; ++e) for (int c = tid; c < 256; c += T) sh.count[e][c] = 0;
            if (lane == 0) { sh.any[wave] = any; sh.none[wave] = none; }
            __syncthreads();
#pragma unroll
            for (int w = 0; w < W; ++w) { any |= sh.any[w]; none |= sh.none[w]; }
            const uint32_t from_here = kth<T, REGS>(key, maybe, any, none, want, left, sh.count);
            // those above; and of its equals the first `left` (none left: all of them)
            uint32_t equal = 0;
#pragma unroll
            for (int r = 0; r < REGS; ++r)
                if (maybe >> r & 1) {
                    if (key[r] > from_here || (left == 0 && key[r] == from_here)) sure |= 1u << r;
                    else if (key[r] == from_here) equal |= 1u << r;
                }
            if (left > 0) {
                const int mine = __popc(equal), upto = (int)scan64(mine, Add{});
                if (lane == 63) sh.taken[wave] = upto;
                __syncthreads();
                int rank = upto - mine;
                for (int w = 0; w < wave; ++w) rank += sh.taken[w];
#pragma unroll
                for (int r = 0; r < REGS; ++r)
                    if (equal >> r & 1) { if (rank < left) sure |= 1u << r; ++rank; }
                __syncthreads();
            }
        }
    }
    // what is taken, in order
    const uint32_t take = sure | forced;
    const int mine = __popc(take), upto = (int)scan64(mine, Add{});
    if (lane == 63) sh.taken[wave] = upto;
    __syncthreads();
    int at = upto - mine;
    for (int w = 0; w < wave; ++w) at += sh.taken[w];
#pragma unroll
    for (int r = 0; r < REGS; ++r)
        if (take >> r & 1) to[at++] = x0 + r;
}
#endif

template <int D, int T, int REGS>
__global__ __launch_bounds__(T) void cache_select_kernel(const SelectArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    __shared__ __attribute__((aligned(16))) SelectShared<T> sh;
    const int bh = a.by_n.of(blockIdx.x), j = blockIdx.x - bh * a.n, i = a.i0 + j, b = a.by_hkv.of(bh);
    SelectInputs<REGS> in;
    select_inputs<D, T, REGS>(a, in, bh, a.scores + ((int64_t)bh * a.n + j) * a.nbp);
    const int L = length_of(a.lengths, b, a.cap), C = count_of(a.counts, b, a.M), last = L - C + i, n = last < 0 ? 0 : (last >> a.block_shift) + 1;
    if (i >= C) return;
    const half8_t q8 = select_query<D>(a, b, bh - b * a.Hkv, i);
    int32_t* const to = a.selected + ((int64_t)bh * a.M + i) * a.top;
    if (n <= a.top) {
        for (int x = threadIdx.x; x < a.top; x += T) to[x] = x < n ? x : -1;
        return;
    }
    select_blocks<D, T, REGS>(a, sh, in, q8, bh, b, bh - b * a.Hkv, i, n, to);
#endif
}

// The same of any number of blocks, whose scores are the definition's.  The score of the last one that is taken is found digit by digit (eight bits of the ordered scores, a count of each of their 256
// values), then one walk over the blocks takes what is larger, and of its equals the first ones, in order.
__global__ __launch_bounds__(256) void cache_select_many_kernel(const SelectArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    __shared__ int count[256], waves[4], waves2[4], digit, left;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int bh = a.by_n.of(blockIdx.x), j = blockIdx.x - bh * a.n, i = a.i0 + j, b = a.by_hkv.of(bh);
    const int L = length_of(a.lengths, b, a.cap), C = count_of(a.counts, b, a.M), last = L - C + i, n = last < 0 ? 0 : (last >> a.block_shift) + 1;
    if (i >= C) return;
    int32_t* const to = a.selected + ((int64_t)bh * a.M + i) * a.top;
    if (n <= a.top) {
        for (int x = tid; x < a.top; x += 256) to[x] = x < n ? x : -1;
        return;
    }
    const float* const from = a.scores + ((int64_t)bh * a.n + j) * a.nbp;
    const int lo = a.sink, hi = n - a.recent;                     // what is chosen from (top > their number: not empty)
    int want = a.top - a.sink - a.recent;
    uint32_t known = 0;
    if (want > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            count[tid] = 0;
            __syncthreads();
            for (int x = lo + tid; x < hi; x += 256) {
                const uint32_t u = ordered(from[x]);
                if (shift == 24 || (u ^ known) >> (shift + 8) == 0) atomicAdd(&count[u >> shift & 255], 1);
            }
            __syncthreads();
            // from the largest digit down
            const int mine = count[255 - tid];
            int sum = mine;
#pragma unroll
            for (int d = 1; d < 64; d *= 2) { const int y = __shfl_up(sum, d, 64); if (lane >= d) sum += y; }
            if (lane == 63) waves[wave] = sum;
            __syncthreads();
            for (int w = 0; w < wave; ++w) sum += waves[w];
            if (sum >= want && sum - mine < want) { digit = 255 - tid; left = want - (sum - mine); }
            __syncthreads();
            known |= (uint32_t)digit << shift;
            want = left;
        }
    }
    // taken so far, and of the equals of `known`
    int done = 0, equals = 0;
    for (int x0 = 0; x0 < n; x0 += 256) {
        const int x = x0 + tid;
        const bool forced = x < n && (x < lo || x >= hi), open = x >= lo && x < hi && want > 0;
        const uint32_t u = open ? ordered(from[x]) : 0;
        const bool equal = open && u == known;
        const uint64_t eq = __builtin_amdgcn_ballot_w64(equal), below = (1ull << lane) - 1;
        if (lane == 0) waves[wave] = __popcll(eq);
        __syncthreads();
        int rank = equals + __popcll(eq & below);
        for (int w = 0; w < wave; ++w) rank += waves[w];
        const bool take = forced || (open && (u > known || (equal && rank < want)));
        const uint64_t tk = __builtin_amdgcn_ballot_w64(take);
        if (lane == 0) waves2[wave] = __popcll(tk);
        __syncthreads();
        int at = done + __popcll(tk & below);
        for (int w = 0; w < wave; ++w) at += waves2[w];
        if (take) to[at] = x;
        for (int w = 0; w < 4; ++w) { equals += waves[w]; done += waves2[w]; }
        __syncthreads();
    }
#endif
}

// ------------------------------------------------------------------------------------------------ attention
struct SparseArgs {
    const half_t *k, *v, *q; half_t* o; const int32_t *lengths, *counts, *selected;
    int B, Hkv, M, cap, G, block_shift, top, n_rt, ns;
    int64_t ks[3], vs[3], qs[3], os[3];
    float c;
    Parts parts;
    Div by_hkv, by_b, by_ns, by_rt, by_w;
};

#if defined(__HIP_DEVICE_COMPILE__)
// The keys of the selected blocks, tiles of 32 of each block one after the other.  A lane holds the block of its place from `from` on.
struct Chosen {
    const half_t *kp, *vp; const int32_t* list; int kpitch, vpitch, seen, shift, most, from, held;
    __device__ __forceinline__ void hold(int place) { from = place; held = list[min(place + (int)(threadIdx.x & 63), most - 1)]; }
    __device__ __forceinline__ int at(int t) {
        const int place = t >> (shift - 5);
        if (place < from || place - from > 63) hold(place);
        return (__builtin_amdgcn_readlane(held, place - from) << shift) + ((t & ((1 << (shift - 5)) - 1)) << 5);
    }
    __device__ __forceinline__ const half_t* k(int t) { return kp + (int64_t)at(t) * kpitch; }
    __device__ __forceinline__ const half_t* v(int t) { return vp + (int64_t)at(t) * vpitch; }
    __device__ __forceinline__ int n(int t) { return max(0, min(32, seen - at(t))); }
    __device__ __forceinline__ int lim(int t, int last) { return last - at(t); }
};
#endif

// SELECT: up to 1024 blocks the workgroup selects by itself, each of a query's shares the same, which is less than a launch (16 sequences of up to 30001 keys, 32 heads of 128 on 8, 40 of 469 blocks:
// 55 us in all against 60 with a launch for it; this kernel 37 us, 5.1 TB/s).
constexpr int kOwnBlocks = 1024;
template <int D, int NQ, bool SELECT>
__global__ __launch_bounds__(256, 2) void cache_sparse_attn_kernel(const SparseArgs a, const SelectArgs sel) {
#if defined(__HIP_DEVICE_COMPILE__)
    TRN_LDS(D, lds);
    __shared__ NarrowStats<4> stats;
    __shared__ __attribute__((aligned(16))) SelectShared<SELECT ? 256 : 64> sh;
    __shared__ int32_t list[SELECT ? kOwnBlocks : 1];
    constexpr int RT = 16 * NQ;
    const int lane = threadIdx.x & 63, n = lane & 15, g4 = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int x = a.by_hkv.of(blockIdx.x), kvh = blockIdx.x - x * a.Hkv, y = a.by_b.of(x), b = x - y * a.B, z = a.by_ns.of(y), share = y - z * a.ns, i = a.by_rt.of(z), rt = z - i * a.n_rt;
    [[maybe_unused]] SelectInputs<4> in;
    [[maybe_unused]] half8_t q8;
    if constexpr (SELECT) select_inputs<D, 256, 4>(sel, in, b * a.Hkv + kvh, sel.scores + (((int64_t)b * a.Hkv + kvh) * sel.n + i) * sel.nbp);
    const int L = length_of(a.lengths, b, a.cap), C = count_of(a.counts, b, a.M), seen = L - C + i + 1;       // the keys that the query sees
    if (i >= C) return;
    if constexpr (SELECT) q8 = select_query<D>(sel, b, kvh, i);
    const int ends = seen > 0 ? (seen - 1) >> a.block_shift : -1, most = min(a.top, ends + 1), per = 1 << (a.block_shift - 5);
    // (the last block is the query's own: the others are there as a whole)
    const int T = most > 0 ? (most - 1) * per + ((seen - (ends << a.block_shift) + 31) >> 5) : 0, whole = most > 0 ? (most - 1) * per + ((seen - (ends << a.block_shift)) >> 5) : 0;
    const int w = share * 4 + wave, t0 = a.by_w.of(T * w), t1 = a.by_w.of(T * (w + 1));
    half8_t qB[NQ][D / 32];
    int last[NQ];
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
        const int g = rt * RT + 16 * qb + n;
        const bool there = g < a.G;
        last[qb] = there ? seen - 1 : -1;
        const half_t* const qp = a.q + b * a.qs[0] + (int64_t)(kvh * a.G + (there ? g : 0)) * a.qs[1] + i * a.qs[2];
#pragma unroll
        for (int e = 0; e < D / 32; ++e) {
            const half8_t zero = {}, v = *reinterpret_cast<const half8_t*>(qp + 32 * e + 8 * g4);
            qB[qb][e] = there ? v : zero;
        }
    }
    if constexpr (SELECT) {
        if (ends + 1 > a.top) select_blocks<D, 256, 4>(sel, sh, in, q8, b * a.Hkv + kvh, b, kvh, i, ends + 1, list);
        else for (int x = threadIdx.x; x <= ends; x += 256) list[x] = x;
        __syncthreads();
        if (share == 0 && rt == 0)
            for (int x = threadIdx.x; x < a.top; x += 256) sel.selected[(((int64_t)b * a.Hkv + kvh) * a.M + i) * a.top + x] = x < most ? list[x] : -1;
    }
    Chosen keys{a.k + b * a.ks[0] + kvh * a.ks[1], a.v + b * a.vs[0] + kvh * a.vs[1], SELECT ? list : a.selected + (((int64_t)b * a.Hkv + kvh) * a.M + i) * a.top,
                (int)a.ks[2], (int)a.vs[2], seen, a.block_shift, max(most, 1), 0, 0};
    if (t0 < t1) keys.hold(t0 >> (a.block_shift - 5));
    float4_t o[D / 16][NQ];
    float m[NQ], l[NQ];
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
        m[qb] = -INFINITY; l[qb] = 0.f;
#pragma unroll
        for (int e = 0; e < D / 16; ++e) o[e][qb] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
    narrow_walk<D, NQ, 1>(keys, t0, t1, min(t1, max(t0, whole)), keys.kpitch, keys.vpitch, a.c, qB, last, lds.k(wave), lds.v(wave), o, m, l);
    narrow_join<D, NQ, 4>([&](int w, int v) { return v ? lds.v(w) : lds.k(w); }, stats, o, m, l, [&](int r, int d0, float4_t v, float mm, float ll, bool once) __attribute__((always_inline)) {
        const int g = rt * RT + r;
        if (g >= a.G) return;
        if (a.ns > 1) {
            const int64_t at = ((((int64_t)b * a.Hkv + kvh) * a.M + i) * a.G + g) * a.ns + share;
            *reinterpret_cast<float4_t*>(a.parts.o + at * D + d0) = v;
            if (once) *reinterpret_cast<float2_t*>(a.parts.ml + 2 * at) = float2_t{mm, ll};
            return;
        }
        const float inv = ll == 0.f ? 0.f : 1.f / ll;
        half4_t out;
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = (half_t)(v[e] * inv);
        *reinterpret_cast<half4_t*>(a.o + b * a.os[0] + (int64_t)(kvh * a.G + g) * a.os[1] + i * a.os[2] + d0) = out;
    });
#endif
}

// Many queries: a wave has one query's row tile, all its keys, and nothing is joined.  All walk up the cache at the same pace, so that blocks which several of them selected are found in
// the L2 of their XCD.  256 queries on 32756 keys, 32 heads of 128 on 8, 32 blocks each: 90 us, 24 TB/s from L2 (171 with a workgroup a query).
template <int D, int NQ>
__global__ __launch_bounds__(256, 2) void cache_sparse_rows_kernel(const SparseArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    TRN_LDS(D, lds);
    constexpr int RT = 16 * NQ;
    const int lane = threadIdx.x & 63, n = lane & 15, g4 = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int x = a.by_hkv.of(blockIdx.x), kvh = blockIdx.x - x * a.Hkv, y = a.by_b.of(x), b = x - y * a.B, z = y * 4 + wave, i = a.by_rt.of(z), rt = z - i * a.n_rt;
    const int L = length_of(a.lengths, b, a.cap), C = count_of(a.counts, b, a.M), seen = L - C + i + 1;
    if (i >= C) return;
    const int ends = seen > 0 ? (seen - 1) >> a.block_shift : -1, most = min(a.top, ends + 1), per = 1 << (a.block_shift - 5);
    const int T = most > 0 ? (most - 1) * per + ((seen - (ends << a.block_shift) + 31) >> 5) : 0, whole = most > 0 ? (most - 1) * per + ((seen - (ends << a.block_shift)) >> 5) : 0;
    half8_t qB[NQ][D / 32];
    int last[NQ];
    const half_t* const q0 = a.q + b * a.qs[0] + (int64_t)kvh * a.G * a.qs[1] + i * a.qs[2];
    half_t* const o0 = a.o + b * a.os[0] + (int64_t)kvh * a.G * a.os[1] + i * a.os[2];
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
        const int g = rt * RT + 16 * qb + n;
        const bool there = g < a.G;
        last[qb] = there ? seen - 1 : -1;
        const half_t* const qp = q0 + (there ? g : 0) * a.qs[1];
#pragma unroll
        for (int e = 0; e < D / 32; ++e) {
            const half8_t zero = {}, v = *reinterpret_cast<const half8_t*>(qp + 32 * e + 8 * g4);
            qB[qb][e] = there ? v : zero;
        }
    }
    Chosen keys{a.k + b * a.ks[0] + kvh * a.ks[1], a.v + b * a.vs[0] + kvh * a.vs[1], a.selected + (((int64_t)b * a.Hkv + kvh) * a.M + i) * a.top,
                (int)a.ks[2], (int)a.vs[2], seen, a.block_shift, max(most, 1), 0, 0};
    if (T > 0) keys.hold(0);
    float4_t o[D / 16][NQ];
    float m[NQ], l[NQ];
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
        m[qb] = -INFINITY; l[qb] = 0.f;
#pragma unroll
        for (int e = 0; e < D / 16; ++e) o[e][qb] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
    narrow_walk<D, NQ, 1>(keys, 0, T, whole, keys.kpitch, keys.vpitch, a.c, qB, last, lds.k(wave), lds.v(wave), o, m, l);
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
        const int g = rt * RT + 16 * qb + n;
        const float sum = quad_sum(l[qb]), inv = sum == 0.f ? 0.f : 1.f / sum;
        if (g >= a.G) continue;
#pragma unroll
        for (int e = 0; e < D / 16; ++e) {
            half4_t out;
#pragma unroll
            for (int c = 0; c < 4; ++c) out[c] = (half_t)(o[e][qb][c] * inv);
            *reinterpret_cast<half4_t*>(o0 + g * a.os[1] + 16 * e + 4 * g4) = out;
        }
    }
#endif
}

inline bool block16_ok(int block) { return block == 32 || block == 64 || block == 128; }
inline int shift_of(int block) { return block == 32 ? 5 : block == 64 ? 6 : 7; }

}  // namespace trn

extern "C" int trn_cache_bounds_f16(const trn_cache16* c, int32_t block, int32_t tokens, void* bounds, void* stream) {
    using namespace trn;
    const int st = cache16_check(c, false);
    if (st != TRN_OK) return st;
    if (!block16_ok(block)) return TRN_E_UNSUPPORTED;
    if (tokens < 0) return TRN_E_SHAPE;
    if (c->batch == 0 || c->capacity == 0 || tokens == 0) return TRN_OK;
    if (!bounds) return TRN_E_NULL;
    if (!aligned16(bounds)) return TRN_E_ALIGN;
    BoundsArgs a{};
    a.k = (const half_t*)c->k; a.bounds = (half_t*)bounds; a.lengths = c->lengths; a.counts = c->counts;
    a.B = c->batch; a.Hkv = c->n_kv_heads; a.M = tokens; a.cap = c->capacity; a.block = block; a.nb = (c->capacity + block - 1) / block;
    for (int i = 0; i < 3; ++i) a.ks[i] = c->k_stride[i];
    const int64_t heads = (int64_t)c->batch * c->n_kv_heads, size = heads * a.nb * 4 * c->head_dim;
    if (!apart(bounds, size, c->k, rows_extent(c->k, c->k_stride, c->batch, c->n_kv_heads, c->capacity, c->head_dim).span())) return TRN_E_UNSUPPORTED;
    const int most = tokens < c->capacity ? tokens : c->capacity;
    // (the blocks that the new tokens can touch -- the first of them may be the last of its block --, but no more workgroups than the card holds at once: the most new tokens
    // that a call allows are rarely there)
    const int64_t blocks = ((int64_t)most + 2 * block - 2) / block, at_once = (512 + heads - 1) / heads;
    a.per = (int)(blocks < at_once ? blocks : at_once);
    if (heads * a.per > 0xffffff) return TRN_E_SHAPE;                 // (threads in 32 bits)
    a.by_per = Div(a.per); a.by_hkv = Div(c->n_kv_heads);
    const dim3 grid((unsigned)(heads * a.per));
    if (c->head_dim == 128) hipLaunchKernelGGL((cache_bounds_kernel<128>), grid, dim3(256), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL((cache_bounds_kernel<64>), grid, dim3(256), 0, (hipStream_t)stream, a);
    return hipGetLastError() == hipSuccess ? TRN_OK : TRN_E_LAUNCH;
}

extern "C" int64_t trn_cache_sparse_attn_workspace_bytes(const trn_cache16* c, int32_t block, int32_t top, int32_t n_q_heads, int32_t seq_q) {
    using namespace trn;
    if (!c || attn16_rows(c->batch, c->n_kv_heads, n_q_heads, seq_q) != TRN_OK || c->batch == 0 || seq_q == 0 || !block16_ok(block) || top < 1 || top > (1 << 16)) return 0;
    if (c->capacity < 0 || c->capacity > (1 << 26) || (c->head_dim != 64 && c->head_dim != 128)) return 0;
    return plan_sparse(c->batch, c->n_kv_heads, c->capacity, c->head_dim, block, top, n_q_heads, seq_q).bytes;
}

extern "C" int trn_cache_sparse_attn_f16(const trn_cache16* c, const void* bounds, int32_t block, int32_t top, int32_t sink, int32_t recent, const void* q, void* o,
                                         int32_t* selected, int32_t n_q_heads, int32_t seq_q, const int64_t* q_stride, const int64_t* o_stride, float scale,
                                         void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace trn;
    int st = cache16_check(c);
    if (st != TRN_OK) return st;
    if (!block16_ok(block) || top > (1 << 16)) return TRN_E_UNSUPPORTED;
    if (sink < 0 || recent < 1 || top < 1 || (int64_t)sink + recent > top) return TRN_E_SHAPE;
    if ((st = attn16_rows(c->batch, c->n_kv_heads, n_q_heads, seq_q)) != TRN_OK) return st;
    if (c->batch == 0 || seq_q == 0) return TRN_OK;
    if ((st = attn16_check(c, q, o, n_q_heads, seq_q, q_stride, o_stride, scale, workspace)) != TRN_OK) return st;
    if (!selected || (c->capacity && !bounds)) return TRN_E_NULL;
    if ((reinterpret_cast<uintptr_t>(selected) & 3) || !aligned16(bounds)) return TRN_E_ALIGN;
    const int64_t heads = (int64_t)c->batch * c->n_kv_heads;
    // (what is written: apart from each other and from what the launches read)
    const Extent eo = rows_extent(o, o_stride, c->batch, n_q_heads, seq_q, c->head_dim), eq = rows_extent(q, q_stride, c->batch, n_q_heads, seq_q, c->head_dim);
    const int64_t n_bounds = c->capacity ? heads * ((c->capacity + block - 1) / block) * 4 * c->head_dim : 0, n_selected = heads * seq_q * top * 4;
    if (!apart(o, eo.span(), bounds, n_bounds) || !apart(o, eo.span(), selected, n_selected) || !apart(q, eq.span(), selected, n_selected) || !apart(bounds, n_bounds, selected, n_selected))
        return TRN_E_UNSUPPORTED;
    for (int i = 0; i < 2 && c->capacity; ++i)
        if (!apart(i ? c->v : c->k, rows_extent(i ? c->v : c->k, i ? c->v_stride : c->k_stride, c->batch, c->n_kv_heads, c->capacity, c->head_dim).span(), selected, n_selected))
            return TRN_E_UNSUPPORTED;
    const PlanSparse p = plan_sparse(c->batch, c->n_kv_heads, c->capacity, c->head_dim, block, top, n_q_heads, seq_q);
    if (p.bytes && (!workspace || workspace_bytes < p.bytes)) return TRN_E_SCRATCH;
    if (p.dense) {
        if (p.step < 1) return TRN_E_SHAPE;
        SelectArgs a{};
        a.lengths = c->lengths; a.counts = c->counts; a.selected = selected;
        a.B = c->batch; a.Hkv = c->n_kv_heads; a.M = seq_q; a.cap = c->capacity; a.G = p.G; a.block_shift = shift_of(block); a.nb = p.nb; a.top = top; a.sink = sink; a.recent = recent;
        a.by_hkv = Div(c->n_kv_heads);
        for (int64_t i0 = 0; i0 < seq_q; i0 += p.step) {
            a.i0 = (int)i0; a.n = (int)(seq_q - i0 < p.step ? seq_q - i0 : p.step);
            a.by_n = Div(a.n);
            hipLaunchKernelGGL(cache_select_many_kernel, dim3((unsigned)(heads * a.n)), dim3(256), 0, (hipStream_t)stream, a);
            if (hipGetLastError() != hipSuccess) return TRN_E_LAUNCH;
        }
        const trn_prefix none{};
        return trn_cache_prefix_attn_f16(c, &none, q, o, n_q_heads, seq_q, q_stride, o_stride, scale, 1, workspace, workspace_bytes, stream);
    }
    const int64_t groups = p.rows ? heads * (((int64_t)seq_q * p.n_rt + 3) / 4) : heads * seq_q * p.n_rt * p.ns;
    // (workgroups of 256, and as many threads in all as 32 bits number: of every launch, before the first one)
    const bool many = p.nb > kMostBlocks;
    // Scores by a query's heads (a tile of 16 heads a query) or by queries (a tile of 16 queries a head).  us of the whole call by queries / by heads, 16 blocks of 64 keys taken: 32 heads of 128 on 8, 32768 keys, 2
    // queries 19.5 / 17.8, 12 22.4 / 21.5, 32 25.4 / 25.8, 8 sequences of 16384 41.1 / 42.2 with 8 and 104 / 112 with 32; 16 heads of 64 on 16, 2 of 32768 18.4 / 18.7 with 4, 21.0 / 25.0 with 16; 8 heads of 128 on 1,
    // 65536 22.3 / 17.9 with 16, 27.4 / 25.7 with 128, 29.3 / 30.5 with 256; 64 on 2, 4 of 16384 57.8 / 46.5 with 64, 100 / 111 with 256; 71 of 64 on 1, 65536 34.5 / 19.5 with 16, 57.7 / 34.8 with 128.
    const bool by_heads = p.step < 12 || (p.G >= 8 && p.step <= 128);
    // Several tiles of queries a wave once there are 2048 waves: 32 heads of 128 on 8, 256 queries on 32768 keys 46.5 us from 512 waves on, 41.8 to 41.9 from 1024 on and without; others do not change.
    const int64_t q_tiles = by_heads ? p.step : (p.step + 15) / 16, waves = heads * (p.nbp / (by_heads || many ? 16 : 32)) * q_tiles;
    const int steps = many ? (waves > 4096 ? 4 : 1) : (int)(waves <= 2048 ? 1 : waves / 2048 < 8 ? waves / 2048 : 8);
    const int per64 = 4 * 512 / c->head_dim * steps;
    const dim3 score_grid((unsigned)(many ? (p.nb + (int64_t)per64 - 1) / per64 : by_heads ? p.nbp / 64 : (p.nbp + 127) / 128), (unsigned)(many ? p.step : (q_tiles + steps - 1) / steps), (unsigned)heads);
    const int threads = many ? 256 : p.nb > 6144 ? 1024 : p.nb > 1024 ? 512 : p.nb > 512 ? 256 : 128;
    const bool own = !p.rows && p.nb <= kOwnBlocks && p.step == seq_q;       // (the attention's workgroups select)
    if (groups > 0xffffff || heads > 65535 || heads * p.step * ((threads + 255) / 256) > 0xffffff || (int64_t)score_grid.x * score_grid.y * score_grid.z > 0xffffff) return TRN_E_SHAPE;
    const hipStream_t s = (hipStream_t)stream;
    const bool d128 = c->head_dim == 128;
    hipError_t e = hipSuccess;
    SelectArgs select{};
    for (int64_t i0 = 0; i0 < seq_q && e == hipSuccess; i0 += p.step) {
        SelectArgs a{};
        a.q = (const half_t*)q; a.bounds = (const half_t*)bounds; a.lengths = c->lengths; a.counts = c->counts; a.scores = (float*)workspace; a.selected = selected;
        a.B = c->batch; a.Hkv = c->n_kv_heads; a.M = seq_q; a.cap = c->capacity; a.G = p.G; a.block_shift = shift_of(block); a.nb = p.nb;
        a.top = top; a.sink = sink; a.recent = recent; a.i0 = (int)i0; a.n = (int)(seq_q - i0 < p.step ? seq_q - i0 : p.step); a.steps = steps; a.nbp = p.nbp;
        a.norms = (float*)((char*)workspace + p.norms);
        for (int i = 0; i < 3; ++i) a.qs[i] = q_stride[i];
        a.by_hkv = Div(c->n_kv_heads); a.by_n = Div(a.n);
        {      // (grid.y: 64 MB of scores, 64 of them at least, are 262144 queries, 16 a workgroup; 2048 where there are many blocks)
            dim3 grid = score_grid;
            grid.y = (unsigned)(many ? a.n : ((by_heads ? a.n : (a.n + 15) / 16) + steps - 1) / steps);
            if (many) {
                if (d128) hipLaunchKernelGGL((cache_scores64_kernel<128>), grid, dim3(256), 0, s, a);
                else hipLaunchKernelGGL((cache_scores64_kernel<64>), grid, dim3(256), 0, s, a);
            } else if (by_heads) {
                if (d128) hipLaunchKernelGGL((cache_scores_kernel<128, true>), grid, dim3(256), 0, s, a);
                else hipLaunchKernelGGL((cache_scores_kernel<64, true>), grid, dim3(256), 0, s, a);
            } else {
                if (d128) hipLaunchKernelGGL((cache_scores_kernel<128, false>), grid, dim3(256), 0, s, a);
                else hipLaunchKernelGGL((cache_scores_kernel<64, false>), grid, dim3(256), 0, s, a);
            }
            if ((e = hipGetLastError()) != hipSuccess) break;
        }
        select = a;
        if (own) break;
        const dim3 grid((unsigned)(heads * a.n));
        if (many) hipLaunchKernelGGL(cache_select_many_kernel, grid, dim3(256), 0, s, a);
        else if (d128) {
            if (threads == 128) hipLaunchKernelGGL((cache_select_kernel<128, 128, 4>), grid, dim3(128), 0, s, a);
            else if (threads == 256) hipLaunchKernelGGL((cache_select_kernel<128, 256, 4>), grid, dim3(256), 0, s, a);
            else if (threads == 512) hipLaunchKernelGGL((cache_select_kernel<128, 512, 12>), grid, dim3(512), 0, s, a);
            else hipLaunchKernelGGL((cache_select_kernel<128, 1024, 8>), grid, dim3(1024), 0, s, a);
        } else {
            if (threads == 128) hipLaunchKernelGGL((cache_select_kernel<64, 128, 4>), grid, dim3(128), 0, s, a);
            else if (threads == 256) hipLaunchKernelGGL((cache_select_kernel<64, 256, 4>), grid, dim3(256), 0, s, a);
            else if (threads == 512) hipLaunchKernelGGL((cache_select_kernel<64, 512, 12>), grid, dim3(512), 0, s, a);
            else hipLaunchKernelGGL((cache_select_kernel<64, 1024, 8>), grid, dim3(1024), 0, s, a);
        }
        e = hipGetLastError();
    }
    if (e != hipSuccess) return TRN_E_LAUNCH;
    SparseArgs a{};
    a.k = (const half_t*)c->k; a.v = (const half_t*)c->v; a.q = (const half_t*)q; a.o = (half_t*)o; a.lengths = c->lengths; a.counts = c->counts; a.selected = selected;
    a.B = c->batch; a.Hkv = c->n_kv_heads; a.M = seq_q; a.cap = c->capacity; a.G = p.G; a.block_shift = shift_of(block); a.top = top; a.n_rt = p.n_rt; a.ns = p.ns;
    for (int i = 0; i < 3; ++i) { a.ks[i] = c->k_stride[i]; a.vs[i] = c->v_stride[i]; a.qs[i] = q_stride[i]; a.os[i] = o_stride[i]; }
    a.c = scale * kLog2e;
    a.parts = Parts{(float*)((char*)workspace + p.o), (float*)((char*)workspace + p.ml), p.ns};
    a.by_hkv = Div(c->n_kv_heads); a.by_b = Div(c->batch); a.by_ns = Div(p.ns); a.by_rt = Div(p.n_rt); a.by_w = Div(4 * p.ns);
    const dim3 grid((unsigned)groups), block3(256);
    if (p.rows) {
        if (p.nq == 1) {
            if (d128) hipLaunchKernelGGL((cache_sparse_rows_kernel<128, 1>), grid, block3, 0, s, a);
            else hipLaunchKernelGGL((cache_sparse_rows_kernel<64, 1>), grid, block3, 0, s, a);
        } else {
            if (d128) hipLaunchKernelGGL((cache_sparse_rows_kernel<128, 2>), grid, block3, 0, s, a);
            else hipLaunchKernelGGL((cache_sparse_rows_kernel<64, 2>), grid, block3, 0, s, a);
        }
    } else {
        auto launch = [&](auto nq, auto selects) {
            constexpr int NQ = decltype(nq)::value;
            constexpr bool SELECT = decltype(selects)::value;
            if (d128) hipLaunchKernelGGL((cache_sparse_attn_kernel<128, NQ, SELECT>), grid, block3, 0, s, a, select);
            else hipLaunchKernelGGL((cache_sparse_attn_kernel<64, NQ, SELECT>), grid, block3, 0, s, a, select);
        };
        const std::integral_constant<int, 1> one{};
        const std::integral_constant<int, 2> two{};
        if (p.nq == 1) own ? launch(one, std::true_type{}) : launch(one, std::false_type{});
        else own ? launch(two, std::true_type{}) : launch(two, std::false_type{});
    }
    e = hipGetLastError();
    if (e == hipSuccess && p.ns > 1) {
        JoinArgs j{a.parts, a.o, a.counts, a.B, a.Hkv, a.M, a.G, (int)(heads * seq_q * p.G), {a.os[0], a.os[1], a.os[2]}, Div(p.G), Div(a.M), a.by_hkv};
        e = launch_cache16_join(j, c->head_dim, s);
    }
    return e == hipSuccess ? TRN_OK : TRN_E_LAUNCH;
}
