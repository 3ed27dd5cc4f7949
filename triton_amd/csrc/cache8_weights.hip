// What follows an attention over an 8-bit cache: joining the shares of its keys, and the attention weight that each key gets, summed
// over the queries and the query heads of its KV head.  The weights need the rows' finished sums, so they are a second look at the scores.
// Few rows (8 R <= head_dim): the attention leaves its scores, 4 bytes a row and key, which cost less than K once more, and the launch that joins
// the shares turns them into weights.  Many rows: scores are formed again, with K in registers and the queries passing through LDS.
#include "cache8.h"

namespace trn {

// (m, l) of a row's shares, a lane each: the factors by which they count, the row's sum, and log2 of it.
__device__ __forceinline__ void join_row(const Attn8Args& a, int bh, int r, int lane, float& f, float& l, float& l2) {
    const float2_t x = lane < a.ns ? *reinterpret_cast<const float2_t*>(a.ml + (((((int64_t)bh * a.n_rt + (r >> a.rshift)) * a.ns + lane) << a.rshift) + (r & ((1 << a.rshift) - 1))) * 2) : float2_t{-INFINITY, 0.f};
    float top = x.x;
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
    f = x.x == -INFINITY ? 0.f : fast_exp2(x.x - top);
    l = x.y * f;                                  // (a sum of NaN stays)
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) l += __shfl_xor(l, m, 64);
    l2 = top + fast_log2(l);
}

// Workgroups below n_merge: rows' shares, D / 4 threads a row and `sg` groups of them that have every sg-th share.  The others: 1024 keys'
// weights out of their scores.
template <int D>
__global__ __launch_bounds__(256) void cache8_finish_kernel(const Attn8Args a, int n_merge, int per_head, int sg) {
    constexpr int TPR = D / 4, GROUPS = 256 / TPR;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    __shared__ float fs[GROUPS][64], inv[32];
    if ((int)blockIdx.x < n_merge) {
        __shared__ float4_t red[256];
        const int rows = GROUPS / sg, bh = blockIdx.x / per_head, r0 = (blockIdx.x - bh * per_head) * rows;
        const int b = a.by_hkv.of(bh), kvh = bh - b * a.Hkv;
        const int there = min(a.R, tokens_of(a.counts, b, a.Sq) * a.G);
        if (r0 >= there) return;
        for (int i = wave; i < rows; i += 4) {
            const int r = r0 + i;
            if (r >= there) break;
            float f, l, l2;
            join_row(a, bh, r, lane, f, l, l2);
            fs[i][lane] = f;
            if (lane == 0) {
                inv[i] = l == 0.f ? 0.f : 1.f / l;
                const int i0 = a.by_g.of(r), g0 = r - i0 * a.G;
                if (a.lse) a.lse[((int64_t)b * a.Hq + kvh * a.G + g0) * a.Sq + i0] = l2 * kLn2;
                if (a.lse2) a.lse2[(int64_t)bh * a.R + r] = l2;
            }
        }
        __syncthreads();
        const int grp = tid / TPR, piece = tid % TPR, i = grp / sg, nth = grp - i * sg, r = r0 + i;
        const bool mine = r < there;
        float4_t x = {0.f, 0.f, 0.f, 0.f};
        if (mine) {
            const float* part = a.part + (((((int64_t)bh * a.n_rt + (r >> a.rshift)) * a.ns) << a.rshift) + (r & ((1 << a.rshift) - 1))) * D + 4 * piece;
#pragma unroll 4
            for (int k = nth; k < a.ns; k += sg) x = x + *reinterpret_cast<const float4_t*>(part + ((int64_t)k << a.rshift) * D) * fs[i][k];
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
    const int b = a.by_hkv.of(bh), L = keys_of(a.lengths, b, a.cap), rows = min(a.R, tokens_of(a.counts, b, a.Sq) * a.G);
    if (key0 >= L) return;
    for (int r = wave; r < rows; r += 4) {
        float f, l, l2;
        if (a.ns > 1) join_row(a, bh, r, lane, f, l, l2);
        else l2 = a.lse2[(int64_t)bh * a.R + r];
        if (lane == 0) inv[r] = l2;
    }
    __syncthreads();
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    const float* s = a.scores + (int64_t)bh * a.R * a.sp + key0 + tid;
#pragma unroll 4
    for (int r = 0; r < rows; ++r) {
        const float l2 = inv[r];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = key0 + 256 * i + tid < L ? s[(int64_t)r * a.sp + 256 * i] : -INFINITY;
            sum[i] += x == -INFINITY ? 0.f : fast_exp2(x - l2);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int key = key0 + 256 * i + tid;
        const int64_t at = (int64_t)bh * a.cap + key;
        if (key < L) a.w_out[at] = (a.w_in ? a.w_in[at] : 0.f) + sum[i];
    }
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

#if defined(__HIP_DEVICE_COMPILE__)
// The sum over the 32 lanes of a half, in all of them: rotations within 16 lanes, and the exchange of neighbouring sixteens.  (Through LDS, by __shfl_xor,
// a workgroup's 32 of them were 5 us of a prompt's 38.)
__device__ __forceinline__ float sum32(float x) {
    x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x121, 0xf, 0xf, true));      // row_ror:1, 2, 4, 8
    x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x122, 0xf, 0xf, true));
    x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x124, 0xf, 0xf, true));
    x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x128, 0xf, 0xf, true));
    float a = x, b = x;
    asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
    return a + b;
}
#endif

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
    const int n_kb = (a.cap + 255) >> 8;
    const int chunk = blockIdx.y, bh = blockIdx.x / n_kb, block0 = (blockIdx.x - bh * n_kb) * 256, key0 = block0 + wave * 64;
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
        fetch(t0, Q0);
        l2 = row_sum(t0);
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
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float x = sum32(sum[k][e]);
            const int key = key0 + 32 * k + 8 * (e >> 2) + 4 * h + (e & 3);
            if (n == e && key < L) to[key] = (from ? from[key] : 0.f) + x;
        }
#endif
}

// The chunks' sums, in their order.
__global__ __launch_bounds__(256) void cache8_weights_join_kernel(const Attn8Args a) {
    const int n_kb = (a.cap + 255) >> 8, bh = blockIdx.x / n_kb, key = (blockIdx.x - bh * n_kb) * 256 + threadIdx.x;
    const int b = a.by_hkv.of(bh);
    if (key >= keys_of(a.lengths, b, a.cap)) return;
    const int64_t at = (int64_t)bh * a.cap + key, step = (int64_t)a.B * a.Hkv * a.cap;
    float x = 0.f;
#pragma unroll 8
    for (int i = 0; i < a.n_chunks; ++i) x += a.w_part[i * step + at];
    a.w_out[at] = (a.w_in ? a.w_in[at] : 0.f) + x;
}

hipError_t launch_cache8_weights(const Attn8Args& a, int head_dim, hipStream_t s) {
    const unsigned blocks = (unsigned)(a.B * a.Hkv * ((a.cap + 255) / 256));
    if (head_dim == 128) hipLaunchKernelGGL((cache8_weights_kernel<128>), dim3(blocks, (unsigned)a.n_chunks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((cache8_weights_kernel<64>), dim3(blocks, (unsigned)a.n_chunks), dim3(256), 0, s, a);
    if (a.n_chunks > 1) hipLaunchKernelGGL(cache8_weights_join_kernel, dim3(blocks), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace trn
