// Eviction from a key/value cache by accumulated attention weight: of each sequence and KV head the `recent` last keys and those of the
// largest weight among the others, `keep` in all, gathered to the front in their order.
//
// Two launches, or three.  Selection: a workgroup has one head of a sequence.  The weights of its query heads are added up in 64 bits and rounded
// once to fp32, turned into integers that order as they do, and the smallest one kept is found by digits of 11, 11 and 10 bits, counted in
// LDS; ties are filled up from the front.  Up to 32768 keys stay in registers, and one scan over the counts of each 64 numbers what is
// kept.  Move: rows of K and V, 16 bytes a lane.  Into another cache, workgroups share the rows; within the same one, a workgroup has a column of
// all of a head's rows and moves them front to back: a row goes to its own place or one before it, so what a step overwrites has been read by
// this step or an earlier one, and columns never meet.
//
// Selection, 4 sequences of 4096 keys, 8 heads of 4 rows of weights: 7.4 us, of them launch and lengths 2.3, weights 1.8, the first digit 1.2, the others 0.3 and
// 0.7, places 1.0: latency of one workgroup, whose barriers are what is left.  Move, 1024 of each kept, 35 MB: 8.4 us; 8-bit, 16 sequences of 8193
// to 4096, 279 MB: 47.5 us, 5.9 TB/s; fp16 in place, 16 of 8192 to 4096, 537 MB: 92 us, 5.8 TB/s.  In place every row that stays is moved, onto itself too: 16
// sequences of 4096 within their budget of 4096 take 96 us, from codes 56.
//
// 8-bit caches: a block of the shortened cache takes the largest of the scales that its rows come with; codes of rows with a smaller
// one are multiplied by the ratio, which between powers of two only rounds what leaves e4m3's normal numbers.
#include "cache8.h"

namespace trn {

struct EvictArgs {
    const void* k; const void* v; void* k_out; void* v_out;
    const float *ks, *vs; float *ks_out, *vs_out;
    const void* w; void* w_out;
    const int32_t* lengths; int32_t *kept, *new_lengths;
    int B, Hkv, Hw, S, keep, recent, bshift, w_half, in_place[2];
    int64_t st[2][3], ot[2][3];        // strides of K and V in bytes, given and kept
    int64_t sst[2][2], sot[2][2];      // ... of their scales
    uint32_t* order; int summed;       // [B Hkv][S] if summed by a launch of its own, or too many keys for registers
    float* scales;                     // 8 bits: [2][B Hkv][n_blocks], the scales as they were
    int n_blocks;
    int32_t* now;                      // [2][B]: keys that stay, and that there were
    int chunks;                        // move: workgroups of a head's rows
    Div by_hkv, by_chunks, by_heads2;
};

// Larger numbers first, NaN last of all.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t u = __float_as_uint(x);
    if (x != x) return 0;
    return u & 0x80000000u ? ~u : u | 0x80000000u;       // (0xff800000's complement, of -inf, is 0x7fffff: above NaN's)
}

// The order of the NK keys first, first + 1024, .. (below `end`): their weights summed over the rows of their KV head, all keys of a row, and of four rows,
// on their way at once.  (A key after the other, each sum waited for its loads alone: 8 keys a thread took 8 us of a selection's 14.)
template <class T, int NK>
__device__ __forceinline__ void orders_of(const T* w, int64_t pitch, int rows, int first, int end, uint32_t (&u)[NK]) {
    constexpr int UR = NK == 1 ? 8 : NK <= 8 ? 4 : 1;
    double s[NK];
#pragma unroll
    for (int i = 0; i < NK; ++i) s[i] = 0.0;
    int g = 0;
    for (; g + UR <= rows; g += UR) {
        T x[UR][NK];
#pragma unroll
        for (int k = 0; k < UR; ++k)
#pragma unroll
            for (int i = 0; i < NK; ++i) x[k][i] = w[(g + k) * pitch + min(first + i * 1024, end - 1)];
#pragma unroll
        for (int k = 0; k < UR; ++k)
#pragma unroll
            for (int i = 0; i < NK; ++i) s[i] += (double)(float)x[k][i];
    }
    for (; g < rows; ++g) {
        T x[NK];
#pragma unroll
        for (int i = 0; i < NK; ++i) x[i] = w[g * pitch + min(first + i * 1024, end - 1)];
#pragma unroll
        for (int i = 0; i < NK; ++i) s[i] += (double)(float)x[i];
    }
#pragma unroll
    for (int i = 0; i < NK; ++i) u[i] = order_of((float)s[i]);
}
template <int NK>
__device__ __forceinline__ void orders_of(const EvictArgs& a, int64_t at, int rows, int first, int end, uint32_t (&u)[NK]) {
    if (a.w_half) orders_of(static_cast<const half_t*>(a.w) + at, a.S, rows, first, end, u);
    else orders_of(static_cast<const float*>(a.w) + at, a.S, rows, first, end, u);
}
#if defined(__HIP_DEVICE_COMPILE__)
// x summed over the lanes up to this one: within rows of 16 by shifts, over rows by handing on their last lanes.
template <int CTRL, int ROWS> __device__ __forceinline__ int moved(int x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false); }
__device__ __forceinline__ int scan64(int x) {
    x += moved<0x111, 0xf>(x);       // row_shr:1, 2, 4, 8
    x += moved<0x112, 0xf>(x);
    x += moved<0x114, 0xf>(x);
    x += moved<0x118, 0xf>(x);
    x += moved<0x142, 0xa>(x);       // row_bcast:15, 31
    return x + moved<0x143, 0xc>(x);
}
#endif

// The orders by a launch of their own, 256 keys a workgroup.
__global__ __launch_bounds__(256) void cache_evict_sums_kernel(const EvictArgs a) {
    const int n_kb = (a.S + 255) >> 8, bh = blockIdx.x / n_kb, j = (blockIdx.x - bh * n_kb) * 256 + threadIdx.x;
    const int b = a.by_hkv.of(bh), h = bh - b * a.Hkv, per = a.Hw / a.Hkv, n = keys_of(a.lengths, b, a.S);
    if (j >= n) return;
    uint32_t u[1];
    orders_of(a, ((int64_t)b * a.Hw + h * per) * a.S, per, j, n, u);
    a.order[(int64_t)bh * a.S + j] = u[0];
}

// NV: a thread has as many keys, 1024 apart, in registers (0: any number, whose orders lie in the workspace and are walked
// over 16384 at a time).
template <int NV>
__global__ __launch_bounds__(1024) void cache_evict_select_kernel(const EvictArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    __shared__ __attribute__((aligned(16))) int bins[3 * 2048];
    __shared__ __attribute__((aligned(16))) int waves[3][16];
    __shared__ int s_digit, s_above;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int bh = blockIdx.x, b = a.by_hkv.of(bh), h = bh - b * a.Hkv;
    const int n = keys_of(a.lengths, b, a.S), stay = min(n, a.keep);
    const int late = min(a.recent, stay), early = n - late;              // the last `late` keys stay in any case
    const int want = stay - late;                                        // ... and so many of the first `early`
    int32_t* kept = a.kept + (int64_t)bh * a.keep;
    uint32_t* order = a.order + (int64_t)bh * a.S;
    const int per = a.Hw / a.Hkv;
    const int64_t w0 = ((int64_t)b * a.Hw + h * per) * a.S;

    // (the scales as they were: the move writes where they lie)
    if (a.scales) {
        const int blocks = (n + (1 << a.bshift) - 1) >> a.bshift;
        for (int kv = 0; kv < 2; ++kv) {
            const float* s = (kv ? a.vs : a.ks) + b * a.sst[kv][0] + h * a.sst[kv][1];
            float* to = a.scales + ((int64_t)kv * a.B * a.Hkv + bh) * a.n_blocks;
            for (int i = tid; i < blocks; i += 1024) to[i] = s[i];
        }
    }
    if (h == 0 && tid == 0) { a.now[b] = stay; a.now[a.B + b] = n; }
    for (int i = tid; i < late; i += 1024) kept[want + i] = early + i;
    for (int i = stay + tid; i < a.keep; i += 1024) kept[i] = -1;
    if (want == 0) return;
    if (want == early) {
        for (int i = tid; i < early; i += 1024) kept[i] = i;
        return;
    }

    for (int i = tid; i < 3 * 2048; i += 1024) bins[i] = 0;
    constexpr int NU = NV ? NV : 16;
    uint32_t u[NU];
    auto stored = [&](int first) {
#pragma unroll
        for (int i = 0; i < NU; ++i) u[i] = order[min(first + i * 1024, early - 1)];
    };
    if (NV > 0 && a.summed) stored(tid);
    else if constexpr (NV == 32) {
        uint32_t half[16];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            orders_of(a, w0, per, tid + k * 16384, early, half);
#pragma unroll
            for (int i = 0; i < 16; ++i) u[16 * k + i] = half[i];
        }
    } else if constexpr (NV > 0) orders_of(a, w0, per, tid, early, u);
    // The smallest order kept: kept are those above it, and the first `rest` of its equals.
    uint32_t least = 0;
    int rest = want;
    __syncthreads();
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
        int* const bin = bins + pass * 2048;
        auto count = [&](uint32_t x) {
            if (pass == 0 || (x >> (shift + bits)) == (least >> (shift + bits))) atomicAdd(&bin[(x >> shift) & ((1 << bits) - 1)], 1);
        };
        for (int j0 = tid; NV ? j0 == tid : j0 < early; j0 += NU * 1024) {
            if constexpr (NV == 0) stored(j0);
#pragma unroll
            for (int i = 0; i < NU; ++i) if (j0 + i * 1024 < early) count(u[i]);
        }
        __syncthreads();
        // from the top: thread i has the bins 2047 - 2 i and one below
        const int hi = bin[2047 - 2 * tid], lo = bin[2046 - 2 * tid], upto = scan64(hi + lo);
        if (lane == 63) waves[pass][wave] = upto;
        __syncthreads();
        int before = upto - hi - lo;
#pragma unroll
        for (int i = 0; i < 16; ++i) before += i < wave ? waves[pass][i] : 0;
        if (before < rest && before + hi + lo >= rest) {
            const bool first = before + hi >= rest;
            s_digit = first ? 2047 - 2 * tid : 2046 - 2 * tid;
            s_above = first ? before : before + hi;
        }
        __syncthreads();
        least |= (uint32_t)s_digit << shift;
        rest -= s_above;
    }
    // Their places: by what is kept, and by how many equals of the least there are, before them -- counted for each wave's 64 consecutive keys, in
    // whose order the first wave adds them up.
    int2* const runs = reinterpret_cast<int2*>(bins);
    static_assert(sizeof(int2) * (NU * 16 + 1) <= sizeof(bins), "room for the runs and their sum");
    const uint64_t below = ((uint64_t)1 << lane) - 1;
    int2 base = {0, 0};
    for (int j0 = tid; NV ? j0 == tid : j0 - tid < early; j0 += NU * 1024) {
        if constexpr (NV == 0) { stored(j0); __syncthreads(); }
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const bool real = j0 + i * 1024 < early;
            const uint64_t up = __ballot(real && u[i] > least), eq = __ballot(real && u[i] == least);
            if (lane == 0) runs[i * 16 + wave] = int2{__popcll(up), __popcll(eq)};
        }
        __syncthreads();
        if (wave == 0) {
            constexpr int PER = NU / 4;
            int2 mine[PER], sum = {0, 0};
#pragma unroll
            for (int i = 0; i < PER; ++i) { mine[i] = runs[lane * PER + i]; sum.x += mine[i].x; sum.y += mine[i].y; }
            int2 at = {scan64(sum.x), scan64(sum.y)};
            if (lane == 63) runs[NU * 16] = at;
            at.x -= sum.x; at.y -= sum.y;
#pragma unroll
            for (int i = 0; i < PER; ++i) { runs[lane * PER + i] = at; at.x += mine[i].x; at.y += mine[i].y; }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int j = j0 + i * 1024;
            const bool up = j < early && u[i] > least, eq = j < early && u[i] == least;
            const uint64_t ub = __ballot(up), eb = __ballot(eq);
            const int2 run = runs[i * 16 + wave];
            const int tie = base.y + run.y + __popcll(eb & below);
            if (up || (eq && tie < rest)) kept[base.x + run.x + __popcll(ub & below) + min(tie, rest)] = j;
        }
        base.x += runs[NU * 16].x; base.y += runs[NU * 16].y;
    }
#endif
}

// Of a row of weights: those of the kept keys, to the front; and the new lengths.
template <int THREADS>
__device__ __forceinline__ void move_weights(const EvictArgs& a, int row) {
    const int tid = threadIdx.x, b = row / a.Hw, hw = row - b * a.Hw;
    const int stay = a.now[b];
    if (hw == 0 && tid == 0 && a.new_lengths) a.new_lengths[b] = stay;
    if (!a.w_out) return;
    const int32_t* kept = a.kept + ((int64_t)b * a.Hkv + hw / (a.Hw / a.Hkv)) * a.keep;
    const int64_t from = (int64_t)row * a.S;
    // (w_out may be w, whose rows are S apart, or a tensor of its own with rows of `keep`)
    const int64_t to = a.w_out == a.w ? from : (int64_t)row * a.keep;
    constexpr int NW = 4;
    for (int i0 = 0; i0 < stay; i0 += NW * THREADS) {
        float x[NW]; int j[NW];
#pragma unroll
        for (int e = 0; e < NW; ++e) j[e] = kept[min(i0 + e * THREADS + tid, stay - 1)];
        if (a.w_half) {
#pragma unroll
            for (int e = 0; e < NW; ++e) x[e] = (float)static_cast<const half_t*>(a.w)[from + j[e]];
        } else {
#pragma unroll
            for (int e = 0; e < NW; ++e) x[e] = static_cast<const float*>(a.w)[from + j[e]];
        }
        // (in place: what this step overwrites has been read; a barrier alone does not wait for loads whose values are used behind it)
#pragma unroll
        for (int e = 0; e < NW; ++e) asm volatile("" : "+v"(x[e]));
        __syncthreads();
#pragma unroll
        for (int e = 0; e < NW; ++e) {
            const int i = i0 + e * THREADS + tid;
            if (i < stay) {
                if (a.w_half) static_cast<half_t*>(a.w_out)[to + i] = (half_t)x[e];
                else static_cast<float*>(a.w_out)[to + i] = x[e];
            }
        }
    }
    // (the places that new keys will take have gathered nothing)
    if (a.w_out == a.w) {
        const int n = a.now[a.B + b];
        for (int i = stay + tid; i < n; i += THREADS) {
            if (a.w_half) static_cast<half_t*>(a.w_out)[to + i] = (half_t)0.f;
            else static_cast<float*>(a.w_out)[to + i] = 0.f;
        }
    }
}

// 8 bits: by what the codes of a step's rows, one a thread, are multiplied, and the scales of their blocks (whole ones) -- the largest of those that the rows
// come with.  s: the scale a row comes with, zero where there is none.  Holds two barriers.
__device__ __forceinline__ void block_scales(const EvictArgs& a, float s, float* top, float* ratio, float* scales_out, int row, int end) {
    const int tid = threadIdx.x;
    float t = s;
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) t = fmaxf(t, __shfl_xor(t, m, 64));
    if ((tid & 31) == 0) top[tid >> 5] = t;
    __syncthreads();
    const int groups = 1 << (a.bshift - 5), g0 = (tid >> 5) & ~(groups - 1);
    for (int i = 0; i < groups; ++i) t = fmaxf(t, top[g0 + i]);
    ratio[tid] = t > 0.f ? s / t : 1.f;
    if (scales_out && row < end && (tid & ((1 << a.bshift) - 1)) == 0) scales_out[row >> a.bshift] = t;
    __syncthreads();
}
__device__ __forceinline__ uint4_t recoded(uint4_t x, float f) {
    return f != 1.f ? uint4_t{recoded(x.x, f), recoded(x.y, f), recoded(x.z, f), recoded(x.w, f)} : x;
}

// Into another cache.  Workgroups from n_rows on: (head of a sequence, K or V, chunk of rows).  The first: a row of weights each.
// Past the caches, each byte once: 8-bit, 16 sequences of 8193 to 4096 47.6 us, through them 55.8; 4 of 4096 to 1024 in fp16 8.8 / 8.3.
template <bool BITS8>
__global__ __launch_bounds__(256) void cache_evict_move_kernel(const EvictArgs a, int piece_shift, int n_rows) {
    const int tid = threadIdx.x;
    if ((int)blockIdx.x < n_rows) { move_weights<256>(a, blockIdx.x); return; }
    constexpr int NB = 4;      // rows of a lane on their way at once
    const int u = a.by_chunks.of(blockIdx.x - n_rows), chunk = blockIdx.x - n_rows - u * a.chunks, kv = u & 1, bh = u >> 1;
    const int b = a.by_hkv.of(bh), h = bh - b * a.Hkv;
    const int stay = a.now[b], step = 256 >> piece_shift;
    const int from = chunk * NB * step, to = min(stay, from + NB * step);
    if (from >= to) return;
    const int32_t* kept = a.kept + (int64_t)bh * a.keep;
    const char* src = (const char*)(kv ? a.v : a.k) + b * a.st[kv][0] + h * a.st[kv][1];
    char* dst = (char*)(kv ? a.v_out : a.k_out) + b * a.ot[kv][0] + h * a.ot[kv][1];
    const int r0 = tid >> piece_shift, off = (tid & ((1 << piece_shift) - 1)) * 16;
    uint4_t x[NB]; int j[NB];
#pragma unroll
    for (int e = 0; e < NB; ++e) j[e] = kept[min(from + e * step + r0, to - 1)];
#pragma unroll
    for (int e = 0; e < NB; ++e) x[e] = __builtin_nontemporal_load(reinterpret_cast<const uint4_t*>(src + (int64_t)j[e] * a.st[kv][2] + off));
    __shared__ float ratio[256], top[8];
    if constexpr (BITS8) {
        const float* was = a.scales + ((int64_t)kv * a.B * a.Hkv + bh) * a.n_blocks;
        block_scales(a, from + tid < to ? was[kept[from + tid] >> a.bshift] : 0.f, top, ratio, (kv ? a.vs_out : a.ks_out) + b * a.sot[kv][0] + h * a.sot[kv][1], from + tid, to);
    }
#pragma unroll
    for (int e = 0; e < NB; ++e) {
        const int i = from + e * step + r0;
        if (i < to) {
            if constexpr (BITS8) x[e] = recoded(x[e], ratio[e * step + r0]);
            __builtin_nontemporal_store(x[e], reinterpret_cast<uint4_t*>(dst + (int64_t)i * a.ot[kv][2] + off));
        }
    }
}

// Within the same cache.  Workgroups from n_rows on: (column of 16 << SHIFT bytes, head of a sequence, K or V); the columns of a head as far apart as there are
// heads, on one XCD where those are a multiple of four.  A step's rows are requested before the last one's are stored: they lie behind all that
// those overwrite.  Columns of less than a line of 128 bytes go through the caches, where they meet: past them, 4 sequences of 8192 rows of 8 heads of 128
// to 4096 took 34 us, not 19; one of 65536 to 32768 145, not 114 (a compute unit's rate, of 64: with columns of 16 bytes 91, but 16384 rows
// of 16 heads of 64 to 4096 14 instead of 12).
template <bool BITS8, int SHIFT>
__global__ __launch_bounds__(1024) void cache_evict_shift_kernel(const EvictArgs a, int n_rows) {
    const int tid = threadIdx.x;
    if ((int)blockIdx.x < n_rows) { move_weights<1024>(a, blockIdx.x); return; }
    constexpr int NB = 4, ROWS = 1024 >> SHIFT, STEP = NB * ROWS;
    constexpr bool WHOLE = SHIFT >= 3;
    const int col = a.by_heads2.of(blockIdx.x - n_rows), u = blockIdx.x - n_rows - col * a.by_heads2.d, kv = u & 1, bh = u >> 1;
    const int b = a.by_hkv.of(bh), h = bh - b * a.Hkv;
    const int stay = a.now[b];
    if (stay == 0) return;
    const int32_t* kept = a.kept + (int64_t)bh * a.keep;
    const char* src = (const char*)(kv ? a.v : a.k) + b * a.st[kv][0] + h * a.st[kv][1];
    char* dst = (char*)(kv ? a.v_out : a.k_out) + b * a.ot[kv][0] + h * a.ot[kv][1];
    const int r0 = tid >> SHIFT, off = ((col << SHIFT) + (tid & ((1 << SHIFT) - 1))) * 16;
    const float* was = BITS8 ? a.scales + ((int64_t)kv * a.B * a.Hkv + bh) * a.n_blocks : nullptr;
    float* const scales_out = BITS8 && col == 0 ? (kv ? a.vs_out : a.ks_out) + b * a.sot[kv][0] + h * a.sot[kv][1] : nullptr;
    __shared__ float ratio[BITS8 ? 1024 : 1], top[BITS8 ? 32 : 1];
    // (past the last row that one again: a row that is there, and goes nowhere)
    auto places = [&](int i0, int (&j)[NB], int& own) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < NB; ++e) j[e] = kept[min(i0 + e * ROWS + r0, stay - 1)];
        if constexpr (BITS8) own = kept[min(i0 + tid, stay - 1)];
    };
    auto request = [&](const int (&j)[NB], int own, uint4_t (&x)[NB], float& s) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < NB; ++e) {
            const uint4_t* const from = reinterpret_cast<const uint4_t*>(src + (int64_t)j[e] * a.st[kv][2] + off);
            x[e] = WHOLE ? __builtin_nontemporal_load(from) : *from;
        }
        if constexpr (BITS8) s = was[own >> a.bshift];
    };
    uint4_t x[NB], x_next[NB]; int j[NB], own = 0; float s = 0.f, s_next = 0.f;
    places(0, j, own);
    request(j, own, x, s);
    places(STEP, j, own);
    for (int i0 = 0; i0 < stay; i0 += STEP) {
        request(j, own, x_next, s_next);
        places(i0 + 2 * STEP, j, own);
        // (what this step overwrites has been read by all waves: a barrier alone does not wait for loads whose values are used behind it)
#pragma unroll
        for (int e = 0; e < NB; ++e) asm volatile("" : "+v"(x[e]));
        const int end = min(stay, i0 + STEP);
        if constexpr (BITS8) block_scales(a, i0 + tid < end ? s : 0.f, top, ratio, scales_out, i0 + tid, end);
        else __syncthreads();
#pragma unroll
        for (int e = 0; e < NB; ++e) {
            const int i = i0 + e * ROWS + r0;
            if (i < stay) {
                if constexpr (BITS8) x[e] = recoded(x[e], ratio[e * ROWS + r0]);
                uint4_t* const to = reinterpret_cast<uint4_t*>(dst + (int64_t)i * a.ot[kv][2] + off);
                if constexpr (WHOLE) __builtin_nontemporal_store(x[e], to);
                else *to = x[e];
            }
            x[e] = x_next[e];
        }
        s = s_next;
        if constexpr (BITS8) __syncthreads();      // (`ratio` and `top` are written again)
    }
}

// Keys of which a thread of the selection has its own in registers; and from how many rows of weights a head on they are added up by a launch of their own
// (one KV head of 71 query heads, 4096 keys: 21 us by the selection's one workgroup).
constexpr int kMostKept = 32768, kManyRows = 9;
static bool orders_stored(const trn_cache_evict_desc* e) { return e->keys > kMostKept || e->n_weight_rows >= kManyRows * e->n_kv_heads; }

struct EvictSizes { int64_t scales, now, bytes; };
static EvictSizes evict_sizes(const trn_cache_evict_desc* e) {
    auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
    EvictSizes s;
    const int64_t heads = (int64_t)e->batch * e->n_kv_heads;
    s.scales = orders_stored(e) ? up(heads * e->keys * 4) : 0;
    s.now = s.scales + (e->code_bytes == 1 ? up(2 * heads * ((e->keys + 31) / 32) * 4) : 0);
    s.bytes = s.now + up((int64_t)e->batch * 8);
    return s;
}

}  // namespace trn

extern "C" int64_t trn_cache_evict_workspace_bytes(const trn_cache_evict_desc* e) {
    if (!e || e->batch <= 0 || e->n_kv_heads <= 0 || e->n_weight_rows <= 0 || e->keys <= 0 || e->keep <= 0) return 0;
    return trn::evict_sizes(e).bytes;
}

extern "C" int trn_cache_evict(const trn_cache_evict_desc* e, const void* k, const void* v, void* k_out, void* v_out, const float* k_scale,
                               const float* v_scale, float* k_scale_out, float* v_scale_out, const void* weights, void* weights_out,
                               const int32_t* lengths, int32_t* kept, int32_t* new_lengths, void* workspace, int64_t workspace_bytes,
                               void* stream) {
    using namespace trn;
    if (!e) return TRN_E_NULL;
    if (e->batch < 0 || e->n_kv_heads <= 0 || e->n_weight_rows <= 0 || e->n_weight_rows % e->n_kv_heads || e->keys <= 0 || e->keep <= 0 || e->recent < 0 || e->recent > e->keep) return TRN_E_SHAPE;
    // (a workgroup of 1024 threads a head, and as many threads in all as 32 bits number)
    if ((int64_t)e->batch * e->n_kv_heads > 0x3fffff || (int64_t)e->batch * e->n_weight_rows > 0x3fffff) return TRN_E_SHAPE;
    if (e->code_bytes != 1 && e->code_bytes != 2) return TRN_E_UNSUPPORTED;
    if (e->head_dim != 64 && e->head_dim != 128) return TRN_E_UNSUPPORTED;
    const bool bits8 = e->code_bytes == 1;
    if (bits8 && !block_ok(e->block)) return TRN_E_UNSUPPORTED;
    if (e->keys > (1 << 26) || e->keep > (1 << 26)) return TRN_E_UNSUPPORTED;
    if (e->batch == 0) return TRN_OK;
    if (!k || !v || !k_out || !v_out || !weights || !kept || !workspace) return TRN_E_NULL;
    if (bits8 && (!k_scale || !v_scale || !k_scale_out || !v_scale_out)) return TRN_E_NULL;
    for (const void* p : {k, v, (const void*)k_out, (const void*)v_out}) if (!aligned16(p)) return TRN_E_ALIGN;
    if ((uintptr_t)workspace & 255) return TRN_E_ALIGN;
    const EvictSizes sz = evict_sizes(e);
    if (workspace_bytes < sz.bytes) return TRN_E_SCRATCH;
    EvictArgs a;
    a.k = k; a.v = v; a.k_out = k_out; a.v_out = v_out; a.ks = k_scale; a.vs = v_scale; a.ks_out = k_scale_out; a.vs_out = v_scale_out;
    a.w = weights; a.w_out = weights_out; a.lengths = lengths; a.kept = kept; a.new_lengths = new_lengths;
    a.B = e->batch; a.Hkv = e->n_kv_heads; a.Hw = e->n_weight_rows; a.S = e->keys; a.keep = e->keep; a.recent = e->recent;
    a.w_half = e->weights_half != 0;
    a.bshift = e->block == 32 ? 5 : e->block == 64 ? 6 : 7;
    const int width = e->head_dim * e->code_bytes;
    const int64_t* in[2] = {e->k_stride, e->v_stride};
    const int64_t* out[2] = {e->k_out_stride, e->v_out_stride};
    const int rows_out = e->keep < e->keys ? e->keep : e->keys;
    Extent in_at[2], out_at[2];
    for (int i = 0; i < 2; ++i) {
        for (int j = 0; j < 3; ++j) {
            a.st[i][j] = in[i][j] * e->code_bytes; a.ot[i][j] = out[i][j] * e->code_bytes;
            if (in[i][j] < 0 || out[i][j] < 0) return TRN_E_STRIDE;
            if ((a.st[i][j] | a.ot[i][j]) & 15) return TRN_E_ALIGN;
        }
        if ((in[i][2] < e->head_dim && e->keys > 1) || (out[i][2] < e->head_dim && rows_out > 1)) return TRN_E_STRIDE;
        if ((e->batch > 1 && !out[i][0]) || (e->n_kv_heads > 1 && !out[i][1])) return TRN_E_STRIDE;
        in_at[i] = Extent{i ? v : k, {e->batch, e->n_kv_heads, e->keys}, {a.st[i][0], a.st[i][1], a.st[i][2]}, width};
        out_at[i] = Extent{i ? v_out : k_out, {e->batch, e->n_kv_heads, rows_out}, {a.ot[i][0], a.ot[i][1], a.ot[i][2]}, width};
        a.in_place[i] = in_at[i].p == out_at[i].p;
        if (a.in_place[i]) {       // the same cache, shortened
            for (int j = 0; j < 3; ++j)
                if (a.st[i][j] != a.ot[i][j]) return TRN_E_STRIDE;
        } else if (meet(in_at[i], out_at[i])) return TRN_E_UNSUPPORTED;
    }
    if (meet(in_at[0], out_at[1]) || meet(in_at[1], out_at[0]) || meet(out_at[0], out_at[1])) return TRN_E_UNSUPPORTED;
    if (weights_out && weights_out != weights) {
        const int64_t rows = (int64_t)e->batch * e->n_weight_rows, size = e->weights_half ? 2 : 4;
        if (!apart(weights, rows * e->keys * size, weights_out, rows * e->keep * size)) return TRN_E_UNSUPPORTED;
    }
    if (bits8) {
        for (const void* p : {k_scale, v_scale, (const float*)k_scale_out, (const float*)v_scale_out}) if ((uintptr_t)p & 3) return TRN_E_ALIGN;
        const int64_t *ks = e->k_scale_out_stride, *vs = e->v_scale_out_stride, blocks = (rows_out + e->block - 1) / e->block;
        for (const int64_t* st : {e->k_scale_stride, e->v_scale_stride, ks, vs}) if (st[0] < 0 || st[1] < 0) return TRN_E_STRIDE;
        // (a workgroup writes the scales of one head, of its keys or its values, and nothing else does)
        if ((e->batch > 1 && (!ks[0] || !vs[0])) || (e->n_kv_heads > 1 && (!ks[1] || !vs[1]))) return TRN_E_STRIDE;
        if (meet(Extent{k_scale_out, {e->batch, e->n_kv_heads, 1}, {4 * ks[0], 4 * ks[1], 0}, 4 * blocks},
                 Extent{v_scale_out, {e->batch, e->n_kv_heads, 1}, {4 * vs[0], 4 * vs[1], 0}, 4 * blocks})) return TRN_E_UNSUPPORTED;
    }
    a.sst[0][0] = e->k_scale_stride[0]; a.sst[0][1] = e->k_scale_stride[1]; a.sst[1][0] = e->v_scale_stride[0]; a.sst[1][1] = e->v_scale_stride[1];
    a.sot[0][0] = e->k_scale_out_stride[0]; a.sot[0][1] = e->k_scale_out_stride[1]; a.sot[1][0] = e->v_scale_out_stride[0]; a.sot[1][1] = e->v_scale_out_stride[1];
    a.order = (uint32_t*)workspace;
    a.scales = bits8 ? (float*)((char*)workspace + sz.scales) : nullptr;
    a.n_blocks = bits8 ? (e->keys + e->block - 1) / e->block : 0;
    a.now = (int32_t*)((char*)workspace + sz.now);
    const int64_t heads = (int64_t)e->batch * e->n_kv_heads;
    a.by_hkv = Div(e->n_kv_heads);
    // Rows are shared out; or within the same cache, columns: as wide as leaves a workgroup for each compute unit, 64 bytes at least.
    const bool within = a.in_place[0] || a.in_place[1];
    const int pieces = width / 16;
    int shift = 2;
    while ((1 << shift) < pieces && (!within || 2 * heads * (pieces >> (shift + 1)) >= 256)) ++shift;
    const int rows_per_chunk = 4 * (256 >> shift);
    a.chunks = (rows_out + rows_per_chunk - 1) / rows_per_chunk;
    const int64_t n_rows = weights_out || new_lengths ? (int64_t)e->batch * e->n_weight_rows : 0, grid = n_rows + 2 * heads * (within ? pieces >> shift : a.chunks);
    a.summed = orders_stored(e);
    const int64_t sums = heads * ((e->keys + 255) / 256);
    if (grid > (within ? 0x3fffff : 0xffffff) || (a.summed && sums > 0xffffff)) return TRN_E_SHAPE;
    a.by_chunks = Div(a.chunks); a.by_heads2 = Div(2 * heads);
    const hipStream_t s = (hipStream_t)stream;
    if (a.summed) hipLaunchKernelGGL(cache_evict_sums_kernel, dim3((unsigned)sums), dim3(256), 0, s, a);
    const dim3 sel((unsigned)heads);
    if (e->keys <= 4096) hipLaunchKernelGGL(cache_evict_select_kernel<4>, sel, dim3(1024), 0, s, a);
    else if (e->keys <= 8192) hipLaunchKernelGGL(cache_evict_select_kernel<8>, sel, dim3(1024), 0, s, a);
    else if (e->keys <= 16384) hipLaunchKernelGGL(cache_evict_select_kernel<16>, sel, dim3(1024), 0, s, a);
    else if (e->keys <= kMostKept) hipLaunchKernelGGL(cache_evict_select_kernel<32>, sel, dim3(1024), 0, s, a);
    else hipLaunchKernelGGL(cache_evict_select_kernel<0>, sel, dim3(1024), 0, s, a);
    if (hipGetLastError() != hipSuccess) return TRN_E_LAUNCH;       // (the move would go by places that nothing has set)
    const dim3 all((unsigned)grid);
#define TRN_SHIFT(S) do { if (bits8) hipLaunchKernelGGL((cache_evict_shift_kernel<true, S>), all, dim3(1024), 0, s, a, (int)n_rows); \
                          else hipLaunchKernelGGL((cache_evict_shift_kernel<false, S>), all, dim3(1024), 0, s, a, (int)n_rows); } while (0)
    if (within && shift == 2) TRN_SHIFT(2);
    else if (within && shift == 3) TRN_SHIFT(3);
    else if (within) hipLaunchKernelGGL((cache_evict_shift_kernel<false, 4>), all, dim3(1024), 0, s, a, (int)n_rows);      // (8-bit rows are 128 bytes at most)
#undef TRN_SHIFT
    else if (bits8) hipLaunchKernelGGL((cache_evict_move_kernel<true>), all, dim3(256), 0, s, a, shift, (int)n_rows);
    else hipLaunchKernelGGL((cache_evict_move_kernel<false>), all, dim3(256), 0, s, a, shift, (int)n_rows);
    return hipGetLastError() == hipSuccess ? TRN_OK : TRN_E_LAUNCH;
}
