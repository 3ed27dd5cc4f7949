// Shared by the kernels of the 8-bit key/value cache: e4m3 codes [batch, KV heads, capacity, head_dim] and a float32 scale for each
// head and block of 32, 64 or 128 tokens.
#pragma once
#include "common.h"
#include "extent.h"

namespace trn {

// The least scale, and that of a block without a number in it: fp16's smallest number is 2^-24, e4m3's largest 1.75 * 2^8.
constexpr float kScaleFloor = 0x1p-32f;

// The keys of a sequence (its new tokens among them) and its new tokens, as they stand on the device; nothing outside the cache or the
// launch is ever addressed by them.
__device__ __forceinline__ int keys_of(const int32_t* lengths, int b, int capacity) { return lengths ? min(max(lengths[b], 0), capacity) : capacity; }
__device__ __forceinline__ int tokens_of(const int32_t* counts, int b, int tokens) { return counts ? min(max(counts[b], 0), tokens) : tokens; }

// The smallest power of two by which a finite magnitude comes to no more than 448, at least the floor.
__device__ __forceinline__ float scale_for(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);       // (448 = 1.75 * 2^8)
    return fmaxf(__uint_as_float((uint32_t)max(e, 1) << 23), kScaleFloor);
}

// Four codes as four fp16 values: every e4m3 number is one of fp16.
__device__ __forceinline__ half4_t half_of_codes(uint32_t w) {
    const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false), hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true);
    return half4_t{(half_t)lo[0], (half_t)lo[1], (half_t)hi[0], (half_t)hi[1]};
}
__device__ __forceinline__ half8_t half_of_codes(uint32_t a, uint32_t b) {
    const half4_t x = half_of_codes(a), y = half_of_codes(b);
    return half8_t{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
}
// Four floats as codes, rounded to nearest even; anything past 464, and NaN, becomes NaN.
__device__ __forceinline__ uint32_t codes_of(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    return (uint32_t)w;
}
// ... of codes that are worth `ratio` times as much on another scale.
__device__ __forceinline__ uint32_t recoded(uint32_t w, float ratio) {
    const half4_t h = half_of_codes(w);
    return codes_of((float)h[0] * ratio, (float)h[1] * ratio, (float)h[2] * ratio, (float)h[3] * ratio);
}

// One attention over an 8-bit cache: the arguments of its launches.
struct Attn8Args {
    const uint8_t *k, *v; const float *ks, *vs;
    const int32_t *lengths, *counts;
    const half_t* q; half_t* o; float* lse;
    int B, Hq, Hkv, Sq, cap, G, R, rshift, n_rt, ns, bshift, causal;       // R = G * Sq rows in n_rt tiles of 2^rshift; ns shares
    Div by_units, by_g, by_hkv, by_ns, by_w;
    int64_t kb, kh, kst, vb, vh, vst, ksb, ksh, vsb, vsh, qb, qh, qs, ob, oh, os;
    float c;               // scale * log2(e)
    float *part, *ml;      // shares: [B Hkv][n_rt][ns][rows of a tile][D] and [..][rows][2] (m, l)
    float* lse2;           // [B Hkv][R]: log2 of the row sums, for the key weights (or null)
    const float* w_in; float* w_out;
    float* scores; int sp; // few rows: [B Hkv][R][sp] s = q k scale log2(e), what a row does not see -inf (or null)
    float* w_part; int n_chunks, chunk_tiles;      // many rows: [n_chunks][B Hkv][cap] sums over a chunk's row tiles
};

inline bool block_ok(int block) { return block == 32 || block == 64 || block == 128; }
// The checks of a cache that every entry point makes; base pointers, and strides of axes with more than one element.
int cache8_check(const trn_cache8* c);
// The second launch of an attention: shares joined, and the key weights of few rows out of their scores; the key weights of many rows.
hipError_t launch_cache8_finish(const Attn8Args& a, int head_dim, hipStream_t s);
hipError_t launch_cache8_weights(const Attn8Args& a, int head_dim, hipStream_t s);

}  // namespace trn
