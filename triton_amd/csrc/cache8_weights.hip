// What follows an attention over an 8-bit cache: joining the shares of its keys, and the attention weight that each key gets, summed
// over the queries and the query heads of its KV head.  The weights need the rows' finished sums, so they are a second look at the scores.
// Few rows (8 R <= head_dim): the attention leaves its scores, 4 bytes a row and key, which cost less than K once more, and the launch that joins
// the shares turns them into weights.  Many rows: scores are formed again, with K in registers and the queries passing through LDS.
#include "cache8.h"

namespace trn {

#if defined(__HIP_DEVICE_COMPILE__)
// Over the 16 lanes of a row by rotations within it, over rows by exchanges.  (By __shfl_xor through LDS the sums of 32 rows a lane were 5 us of a prompt's 38.)
template <int CTRL> __device__ __forceinline__ float rotated(float x) { return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true)); }
__device__ __forceinline__ void swap_rows16(float& a, float& b) { asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b)); }
__device__ __forceinline__ float sum32(float x) {
    x += rotated<0x121>(x);       // row_ror:1, 2, 4, 8
    x += rotated<0x122>(x);
    x += rotated<0x124>(x);
    x += rotated<0x128>(x);
    float a = x, b = x;
    swap_rows16(a, b);
    return a + b;
}
__device__ __forceinline__ float max32(float x) {
    x = fmaxf(x, rotated<0x121>(x));
    x = fmaxf(x, rotated<0x122>(x));
    x = fmaxf(x, rotated<0x124>(x));
    x = fmaxf(x, rotated<0x128>(x));
    float a = x, b = x;
    swap_rows16(a, b);
    return fmaxf(a, b);
}

// The first 2 N of x as N: of number i and i + N a lane keeps the second if its index has bit N, and gets the same from the lane that DPP names.
template <int CTRL, int N> __device__ __forceinline__ void keep_half(float (&x)[16], int lane) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float keep = lane & N ? x[i + N] : x[i], give = lane & N ? x[i] : x[i + N];
        x[i] = keep + rotated<CTRL>(give);
    }
}

// (m, l) of a row's shares, a lane each; and out of them the factors by which they count, the row's sum, and log2 of it.
__device__ __forceinline__ float2_t shares_of(const Attn8Args& a, int bh, int r, int lane) {
    const int row = min(r, a.R - 1);
    return *reinterpret_cast<const float2_t*>(a.ml + (((((int64_t)bh * a.n_rt + (row >> a.rshift)) * a.ns + min(lane, a.ns - 1)) << a.rshift) + (row & ((1 << a.rshift) - 1))) * 2);
}
__device__ __forceinline__ void join_row(const Attn8Args& a, float2_t x, int lane, float& f, float& l, float& l2) {
    const float m = lane < a.ns ? x.x : -INFINITY, top = half_max(max32(m));
    f = m == -INFINITY ? 0.f : fast_exp2(m - top);
    l = half_sum(sum32(lane < a.ns ? x.y * f : 0.f));      // (a sum of NaN stays)
    l2 = top + fast_log2(l);
}
#endif

// Workgroups below n_merge: rows' shares, D / 4 threads a row and `sg` groups of them that have every sg-th share.  The others: 1024 keys'
// weights out of their scores.
template <int D>
__global__ __launch_bounds__(256) void cache8_finish_kernel(const Attn8Args a, int n_merge, int per_head, int sg) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int TPR = D / 4, GROUPS = 256 / TPR;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    __shared__ float fs[GROUPS][64], inv[32];
    if ((int)blockIdx.x < n_merge) {
        __shared__ float4_t red[256];
        const int rows = GROUPS / sg, bh = blockIdx.x / per_head, r0 = (blockIdx.x - bh * per_head) * rows;
        const int b = a.by_hkv.of(bh), kvh = bh - b * a.Hkv;
        const int grp = tid / TPR, piece = tid % TPR, i = grp / sg, nth = grp - i * sg, r = r0 + i;
        // (a thread's first four shares are requested at once with what their factors come from)
        const float2_t first = shares_of(a, bh, r0 + min(wave, rows - 1), lane);
        constexpr int PRE = 4;
        float4_t got[PRE];
        const int row = min(r, a.R - 1);
        const float* part = a.part + (((((int64_t)bh * a.n_rt + (row >> a.rshift)) * a.ns) << a.rshift) + (row & ((1 << a.rshift) - 1))) * D + 4 * piece;
#pragma unroll
        for (int e = 0; e < PRE; ++e) got[e] = *reinterpret_cast<const float4_t*>(part + ((int64_t)min(nth + e * sg, a.ns - 1) << a.rshift) * D);
        const int there = min(a.R, tokens_of(a.counts, b, a.Sq) * a.G);
        if (r0 >= there) return;
        for (int j = wave; j < rows; j += 4) {
            if (r0 + j >= there) break;
            float f, l, l2;
            join_row(a, j == wave ? first : shares_of(a, bh, r0 + j, lane), lane, f, l, l2);
            fs[j][lane] = f;
            if (lane == 0) {
                inv[j] = l == 0.f ? 0.f : 1.f / l;
                const int i0 = a.by_g.of(r0 + j), g0 = r0 + j - i0 * a.G;
                if (a.lse) a.lse[((int64_t)b * a.Hq + kvh * a.G + g0) * a.Sq + i0] = l2 * kLn2;
                if (a.lse2) a.lse2[(int64_t)bh * a.R + r0 + j] = l2;
            }
        }
        __syncthreads();
        const bool mine = r < there;
        float4_t x = {0.f, 0.f, 0.f, 0.f};
        if (mine) {
#pragma unroll
            for (int e = 0; e < PRE; ++e) x = x + (nth + e * sg < a.ns ? got[e] * fs[i][nth + e * sg] : float4_t{0.f, 0.f, 0.f, 0.f});
            for (int k = nth + PRE * sg; k < a.ns; k += sg) x = x + *reinterpret_cast<const float4_t*>(part + ((int64_t)k << a.rshift) * D) * fs[i][k];
        }
        if (sg > 1) {
            red[tid] = x;
            __syncthreads();
            if (nth != 0) return;
            for (int k = 1; k < sg; ++k) x = x + red[tid + k * TPR];
        }
        if (!mine) return;
        half4_t y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = (half_t)(x[e] * inv[i]);
        const int i0 = a.by_g.of(r), g0 = r - i0 * a.G;
        *reinterpret_cast<half4_t*>(a.o + b * a.ob + (int64_t)(kvh * a.G + g0) * a.oh + (int64_t)i0 * a.os + 4 * piece) = y;
        return;
    }
    const int n_kb = (a.cap + 1023) >> 10, u = blockIdx.x - n_merge, bh = u / n_kb, key0 = (u - bh * n_kb) << 10;
    const int b = a.by_hkv.of(bh);
    // (the scores of the first rows and the old weights are requested at once with what the rows' sums come from; what is past the sequence's keys counts nowhere)
    const bool shared = a.ns > 1;
    const float2_t first = shared ? shares_of(a, bh, wave, lane) : float2_t{0.f, a.lse2[(int64_t)bh * a.R + min(wave, a.R - 1)]};
    constexpr int PRE = 4;
    const float* s = a.scores + (int64_t)bh * a.R * a.sp;
    float got[PRE][4], old[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int key = key0 + 256 * i + tid;
#pragma unroll
        for (int r = 0; r < PRE; ++r) got[r][i] = s[(int64_t)min(r, a.R - 1) * a.sp + min(key, a.sp - 1)];
        old[i] = *((a.w_in ? a.w_in : a.w_out) + (int64_t)bh * a.cap + min(key, a.cap - 1));
    }
    const int L = keys_of(a.lengths, b, a.cap), rows = min(a.R, tokens_of(a.counts, b, a.Sq) * a.G);
    if (key0 >= L) return;
    for (int r = wave; r < rows; r += 4) {
        float f, l, l2;
        if (shared) join_row(a, r == wave ? first : shares_of(a, bh, r, lane), lane, f, l, l2);
        else l2 = r == wave ? first.y : a.lse2[(int64_t)bh * a.R + r];
        if (lane == 0) inv[r] = l2;
    }
    __syncthreads();
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    auto add = [&](int i, float x, float l2) { sum[i] += x == -INFINITY ? 0.f : fast_exp2(x - l2); };
#pragma unroll
    for (int r = 0; r < PRE; ++r)
        if (r < rows) {
#pragma unroll
            for (int i = 0; i < 4; ++i) add(i, got[r][i], inv[r]);
        }
#pragma unroll 4
    for (int r = PRE; r < rows; ++r) {
#pragma unroll
        for (int i = 0; i < 4; ++i) add(i, s[(int64_t)r * a.sp + min(key0 + 256 * i + tid, a.sp - 1)], inv[r]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int key = key0 + 256 * i + tid;
        const int64_t at = (int64_t)bh * a.cap + key;
        if (key < L) a.w_out[at] = (a.w_in ? old[i] : 0.f) + sum[i];
    }
#endif
}

hipError_t launch_cache8_finish(const Attn8Args& a, int head_dim, hipStream_t s) {
    const int groups = 1024 / head_dim, heads = a.B * a.Hkv;
    const int sg = a.ns >= 8 ? groups : 1;
    const int per_head = a.ns > 1 ? (a.R + groups / sg - 1) / (groups / sg) : 0, n_merge = heads * per_head;
    const unsigned grid = (unsigned)(n_merge + (a.scores ? heads * ((a.cap + 1023) / 1024) : 0));
    if (head_dim == 128) hipLaunchKernelGGL((cache8_finish_kernel<128>), dim3(grid), dim3(256), 0, s, a, n_merge, per_head, sg);
    else hipLaunchKernelGGL((cache8_finish_kernel<64>), dim3(grid), dim3(256), 0, s, a, n_merge, per_head, sg);
    return hipGetLastError();
}

// A prompt of 1501, 32 heads of 128 on 8: 23.4 us -- launch and the end of the chunks that see nothing 4.8, the first queries and keys and one tile 5, the
// sums over lanes 1, eleven tiles 12, near what their exponentials and products take.
// The weights that 256 keys get from a chunk of row tiles.  A wave has 64 keys, whose codes it holds as operands (A, two blocks of 32); the
// tile's queries (B) come through LDS, for all four waves, one tile ahead.  Per row and key: one exponential, one multiply-add and one addition.
template <int D>
__global__ __launch_bounds__(256, 2) void cache8_weights_kernel(const Attn8Args a) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int NS = D / 16, CPR = D / 8;          // contraction steps; 16-byte chunks a query
    __shared__ __attribute__((aligned(1024))) half_t Q0[32 * D];
    __shared__ __attribute__((aligned(1024))) half_t Q1[32 * D];
    const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // (a head's workgroups are as far apart as there are heads: where those are a multiple of eight, its queries are read by one XCD)
    const int heads = a.B * a.Hkv, kb = blockIdx.x / heads;
    const int chunk = blockIdx.y, bh = blockIdx.x - kb * heads, block0 = kb * 256, key0 = block0 + wave * 64;
    const int b = a.by_hkv.of(bh), kvh = bh - b * a.Hkv;
    const int L = keys_of(a.lengths, b, a.cap), C = tokens_of(a.counts, b, a.Sq), off = L - C;
    if (block0 >= L) return;
    const int rows = min(a.R, C * a.G);
    // (rows before the first that sees the block's first key add nothing)
    const int first = a.causal ? max(0, block0 - off) * a.G >> 5 : 0;
    const int t0 = max(first, chunk * a.chunk_tiles), t1 = min((rows + 31) >> 5, (chunk + 1) * a.chunk_tiles);
    float* const to = a.n_chunks > 1 ? a.w_part + ((int64_t)chunk * a.B * a.Hkv + bh) * a.cap : a.w_out + (int64_t)bh * a.cap;
    const float* from = a.n_chunks > 1 || !a.w_in ? nullptr : a.w_in + (int64_t)bh * a.cap;
    if (t0 >= t1) {
        const int key = block0 + threadIdx.x;
        if (key < L) to[key] = from ? from[key] : 0.f;
        return;
    }
    float sum[2][16];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 16; ++e) sum[k][e] = 0.f;
    {
        const half_t* qh = a.q + b * a.qb + (int64_t)kvh * a.G * a.qh;
        // staging: a wave-wide load has 64 / CPR rows, a wave every fourth of them
        constexpr int RPI = 64 / CPR, NL = 32 / RPI / 4;
        const int sr = lane / CPR, sc = lane % CPR;
        auto swz = [](int r) { return D == 128 ? r & 15 : (r >> 1) & 7; };
        auto fetch = [&](int t, half_t* dst) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const int r32 = (i * 4 + wave) * RPI + sr, r = min(t * 32 + r32, rows - 1), qi = a.by_g.of(r), qg = r - qi * a.G;
                const half_t* src = qh + (int64_t)qg * a.qh + (int64_t)qi * a.qs + ((sc ^ swz(r32)) << 3);
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)src,
                                                 (__attribute__((address_space(3))) uint32_t*)(dst + (i * 4 + wave) * RPI * D), 16, 0, 0);
            }
        };
        int qi = 0; float l2 = 0.f, l2_next;
        // (a row that is not there, or has no weight to give, adds zeros)
        auto row_sum = [&](int t) {
            const int r = t * 32 + n;
            const float x = r < rows ? a.lse2[(int64_t)bh * a.R + r] : INFINITY;
            return x == -INFINITY ? INFINITY : x;
        };
        fetch(t0, Q0);
        l2 = row_sum(t0);
        half8_t kA[2][NS];
        float c[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const uint8_t* kp = a.k + b * a.kb + kvh * a.kh + (int64_t)min(key0 + 32 * k + n, L - 1) * a.kst + h * 16;
#pragma unroll
            for (int j = 0; j < NS / 2; ++j) {
                const uint4_t w = *reinterpret_cast<const uint4_t*>(kp + 32 * j);
                kA[k][2 * j] = half_of_codes(w.x, w.y); kA[k][2 * j + 1] = half_of_codes(w.z, w.w);
            }
            c[k] = a.c * a.ks[b * a.ksb + kvh * a.ksh + (min(key0 + 32 * k, L - 1) >> a.bshift)];
        }
        auto tile = [&](int t, const half_t* Q) __attribute__((always_inline)) {
            const int row = t * 32 + n;
            qi = a.by_g.of(row);
            float16_t s[2];
#pragma unroll
            for (int e = 0; e < 16; ++e) s[0][e] = s[1][e] = 0.f;
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                const half8_t qB = *reinterpret_cast<const half8_t*>(Q + n * D + (((4 * (i >> 1) + 2 * h + (i & 1)) ^ swz(n)) << 3));
                s[0] = mfma32(kA[0][i], qB, s[0]);
                s[1] = mfma32(kA[1][i], qB, s[1]);
            }
            const int seen = a.causal ? min(L, a.by_g.of(t * 32) + off + 1) : L;         // by the tile's first row
            if (__builtin_expect(key0 + 64 > seen, 0)) {
                const int lim = (row < rows ? (a.causal ? min(L - 1, qi + off) : L - 1) : -1) - key0 - 4 * h;
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int e = 0; e < 16; ++e) sum[k][e] += 32 * k + 8 * (e >> 2) + (e & 3) <= lim ? fast_exp2(__builtin_fmaf(s[k][e], c[k], -l2)) : 0.f;
            } else {
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int e = 0; e < 16; ++e) sum[k][e] += fast_exp2(__builtin_fmaf(s[k][e], c[k], -l2));
            }
        };
        for (int t = t0; t < t1; t += 2) {
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();                       // this tile is there, and the one before it has been read
            if (t + 1 < t1) fetch(t + 1, Q1);
            l2_next = row_sum(t + 1);
            tile(t, Q0);
            l2 = l2_next;
            if (t + 1 >= t1) break;
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
            if (t + 2 < t1) fetch(t + 2, Q0);
            l2_next = row_sum(t + 2);
            tile(t + 1, Q1);
            l2 = l2_next;
        }
    }
    // Sums over the 32 lanes of a half, each lane left with one key's: a lane hands the half of its numbers that it does not keep to the one that does.
#pragma unroll
    for (int e = 0; e < 16; ++e) { swap_rows16(sum[0][e], sum[1][e]); sum[0][e] += sum[1][e]; }
    keep_half<0x128, 8>(sum[0], n);       // row_ror:8
    keep_half<0x141, 4>(sum[0], n);       // row_half_mirror: another four lanes, in reverse
    keep_half<0x4e, 2>(sum[0], n);        // quad_perm: the other two
    keep_half<0xb1, 1>(sum[0], n);        // ... and the other one
    const int key = key0 + 32 * (n >> 4) + 8 * ((n & 15) >> 2) + 4 * h + (n & 3);
    if (key < L) to[key] = (from ? from[key] : 0.f) + sum[0][0];
#endif
}

// The chunks' sums: 64 keys a workgroup, every fourth chunk a wave, in their order.  (One thread a key: 813 keys of one head in 192 chunks 10 us.)
__global__ __launch_bounds__(256) void cache8_weights_join_kernel(const Attn8Args a) {
    __shared__ float part[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n_kb = (a.cap + 63) >> 6, bh = blockIdx.x / n_kb, key = (blockIdx.x - bh * n_kb) * 64 + lane;
    const int b = a.by_hkv.of(bh);
    const int64_t at = (int64_t)bh * a.cap + min(key, a.cap - 1), step = (int64_t)a.B * a.Hkv * a.cap;
    float x = 0.f;
#pragma unroll 8
    for (int i = wave; i < a.n_chunks; i += 4) x += a.w_part[i * step + at];
    part[wave][lane] = x;
    __syncthreads();
    if (wave == 0 && key < keys_of(a.lengths, b, a.cap)) a.w_out[at] = (a.w_in ? a.w_in[at] : 0.f) + ((part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]));
}

hipError_t launch_cache8_weights(const Attn8Args& a, int head_dim, hipStream_t s) {
    const unsigned blocks = (unsigned)(a.B * a.Hkv * ((a.cap + 255) / 256));
    if (head_dim == 128) hipLaunchKernelGGL((cache8_weights_kernel<128>), dim3(blocks, (unsigned)a.n_chunks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((cache8_weights_kernel<64>), dim3(blocks, (unsigned)a.n_chunks), dim3(256), 0, s, a);
    if (a.n_chunks > 1) hipLaunchKernelGGL(cache8_weights_join_kernel, dim3((unsigned)(a.B * a.Hkv * ((a.cap + 63) / 64))), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace trn
