// New keys and values of an 8-bit cache: quantised to e4m3 with a power of two for each head and block of tokens.
//
// A block's scale is the least power of two s with max |x| <= 448 s, so that x / s is exact and the code is x rounded once to four
// significant bits.  A block that already holds tokens keeps its scale unless a new one needs a larger: the codes that are there are
// then multiplied by (old / new), which a power of two makes exact but for those that leave e4m3's normal numbers.
//
// A workgroup has one block of one head, of the keys or of the values: it owns the scale, so nothing is shared and nothing atomic.
// The rows wait in registers between the maximum and the codes: each is read once, 16 bytes a lane, and written once, 8 bytes a lane.
// One token of 8 heads of 128: 3.6 us, a launch and two reads from memory, one behind the other.  Prompts of up to 2047 of four sequences, 41 MB: 10.5 us,
// 3.9 TB/s; all workgroups run at once, each through its one chain of lengths, rows, maximum and codes.
#include "cache8.h"

namespace trn {

struct AppendArgs {
    const half_t* x[2]; uint8_t* code[2]; float* scale[2];
    const int32_t *lengths, *counts;
    int B, Hkv, M, cap, block, n_blocks;      // n_blocks: that the new tokens of a sequence can touch
    Div by_blocks, by_heads;
    int64_t xb[2], xh[2], xs[2], cb[2], ch[2], cs[2], sb[2], sh[2];
};

template <int D>
__global__ __launch_bounds__(256) void cache8_append_kernel(const AppendArgs a) {
    constexpr int LPR = D / 8, RPP = 256 / LPR;      // lanes per row, rows per pass
    constexpr int NP = 128 / RPP;                    // passes over the largest block
    const int kv = blockIdx.y, unit = a.by_blocks.of(blockIdx.x), nth = blockIdx.x - unit * a.n_blocks;
    const int b = a.by_heads.of(unit), h = unit - b * a.Hkv;
    const int L = keys_of(a.lengths, b, a.cap), C = min(tokens_of(a.counts, b, a.M), L);
    // (of more new tokens than keys the last ones are the sequence's)
    const int skip = tokens_of(a.counts, b, a.M) - C;
    const int first = L - C, blk = first / a.block + nth, base = blk * a.block;
    if (base >= L || C == 0) return;

    const half_t* x = a.x[kv] + b * a.xb[kv] + h * a.xh[kv];
    uint8_t* code = a.code[kv] + b * a.cb[kv] + h * a.ch[kv];
    float* scale = a.scale[kv] + b * a.sb[kv] + h * a.sh[kv] + blk;
    const int sub = threadIdx.x % LPR, r0 = threadIdx.x / LPR;
    float was = base < first ? *scale : kScaleFloor;      // (a block that begins with a new token takes over nothing)

    half8_t v[NP];
    uint32_t top = 0;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        const int row = p * RPP + r0, pos = base + row;
        if (row < a.block && pos >= first && pos < L) v[p] = *reinterpret_cast<const half8_t*>(x + (int64_t)(pos - first + skip) * a.xs[kv] + sub * 8);
    }
    // (all are waited for here: where a row is there or not, the compiler waits at each use, for the stores before it as well)
#pragma unroll
    for (int p = 0; p < NP; ++p) asm volatile("" : "+v"(v[p]));
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        const int row = p * RPP + r0, pos = base + row;
        if (row < a.block && pos >= first && pos < L) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t u = __float_as_uint(fabsf((float)v[p][e]));
                if (u < 0x7f800000u) top = max(top, u);          // (magnitudes order as their bits; infinities and NaN do not count)
            }
        }
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m, 64));
    __shared__ uint32_t part[4];
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    asm volatile("" : "+v"(was));       // (read by every wave before the first thread writes it, behind the barrier)
    __syncthreads();
    top = max(max(part[0], part[1]), max(part[2], part[3]));
    const float s = fmaxf(was, scale_for(__uint_as_float(top))), inv = 1.f / s;

#pragma unroll
    for (int p = 0; p < NP; ++p) {
        const int row = p * RPP + r0, pos = base + row;
        if (row < a.block && pos >= first && pos < L) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = (float)v[p][e] * inv;
            *reinterpret_cast<uint2_t*>(code + (int64_t)pos * a.cs[kv] + sub * 8) = uint2_t{codes_of(f[0], f[1], f[2], f[3]), codes_of(f[4], f[5], f[6], f[7])};
        }
    }
    if (base < first && s != was) {
        const float ratio = was / s;
        for (int pos = base + r0; pos < first; pos += RPP) {
            uint2_t* to = reinterpret_cast<uint2_t*>(code + (int64_t)pos * a.cs[kv] + sub * 8);
            const uint2_t w = *to;
            *to = uint2_t{recoded(w.x, ratio), recoded(w.y, ratio)};
        }
    }
    if (threadIdx.x == 0 && s != was) *scale = s;
    if (threadIdx.x == 0 && base >= first) *scale = s;
}

int cache8_check(const trn_cache8* c) {
    if (!c) return TRN_E_NULL;
    if (c->batch < 0 || c->n_kv_heads <= 0 || c->capacity < 0) return TRN_E_SHAPE;
    if (c->head_dim != 64 && c->head_dim != 128) return TRN_E_UNSUPPORTED;
    if (!block_ok(c->block)) return TRN_E_UNSUPPORTED;
    if (c->capacity > (1 << 26)) return TRN_E_UNSUPPORTED;       // (products of tiles and workers in 32 bits)
    if (c->batch == 0 || c->capacity == 0) return TRN_OK;
    if (!c->k || !c->v || !c->k_scale || !c->v_scale) return TRN_E_NULL;
    if ((c->k_stride_s < c->head_dim || c->v_stride_s < c->head_dim) && c->capacity > 1) return TRN_E_STRIDE;
    if (c->k_stride_s > (1 << 24) || c->v_stride_s > (1 << 24)) return TRN_E_UNSUPPORTED;      // (32 rows in 32-bit offsets)
    if (!aligned16(c->k) || !aligned16(c->v)) return TRN_E_ALIGN;
    if ((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale)) & 3) return TRN_E_ALIGN;
    for (int64_t s : {c->k_stride_b, c->k_stride_h, c->k_stride_s, c->v_stride_b, c->v_stride_h, c->v_stride_s})
        if (s & 15) return TRN_E_ALIGN;
    return TRN_OK;
}

}  // namespace trn

extern "C" int trn_cache8_append_f16(const trn_cache8* c, const void* k, const void* v, int32_t tokens, int64_t k_stride_b,
                                     int64_t k_stride_h, int64_t k_stride_s, int64_t v_stride_b, int64_t v_stride_h,
                                     int64_t v_stride_s, void* stream) {
    using namespace trn;
    const int st = cache8_check(c);
    if (st != TRN_OK) return st;
    if (tokens < 0) return TRN_E_SHAPE;
    if (c->batch == 0 || c->capacity == 0 || tokens == 0) return TRN_OK;
    if (!k || !v) return TRN_E_NULL;
    // (what is written must not be written twice)
    if (c->batch > 1 && (!c->k_stride_b || !c->v_stride_b || !c->ks_stride_b || !c->vs_stride_b)) return TRN_E_STRIDE;
    if (c->n_kv_heads > 1 && (!c->k_stride_h || !c->v_stride_h || !c->ks_stride_h || !c->vs_stride_h)) return TRN_E_STRIDE;
    if (!aligned16(k) || !aligned16(v)) return TRN_E_ALIGN;
    for (int64_t s : {k_stride_b, k_stride_h, k_stride_s, v_stride_b, v_stride_h, v_stride_s})
        if (!pitch16(s, 2)) return TRN_E_ALIGN;
    AppendArgs a;
    a.x[0] = (const half_t*)k; a.x[1] = (const half_t*)v;
    a.code[0] = (uint8_t*)c->k; a.code[1] = (uint8_t*)c->v;
    a.scale[0] = c->k_scale; a.scale[1] = c->v_scale;
    a.lengths = c->lengths; a.counts = c->counts;
    a.B = c->batch; a.Hkv = c->n_kv_heads; a.M = tokens; a.cap = c->capacity; a.block = c->block;
    const int most = tokens < c->capacity ? tokens : c->capacity;
    a.n_blocks = (most + 2 * c->block - 2) / c->block;                  // (the first of them may be the last of its block)
    const int64_t units = (int64_t)c->batch * c->n_kv_heads;
    if (units * a.n_blocks > 0xffffff) return TRN_E_SHAPE;            // (threads in 32 bits)
    // (nor as keys by one workgroup and as values by another)
    auto same = [&](const void* x, const void* y, int64_t xb, int64_t xh, int64_t xs, int64_t yb, int64_t yh, int64_t ys, int64_t rows, int64_t width) {
        if (xb < 0 || xh < 0 || yb < 0 || yh < 0) return x == y;
        return meet(Extent{x, {c->batch, c->n_kv_heads, rows}, {xb, xh, xs}, width}, Extent{y, {c->batch, c->n_kv_heads, rows}, {yb, yh, ys}, width});
    };
    if (same(c->k, c->v, c->k_stride_b, c->k_stride_h, c->k_stride_s, c->v_stride_b, c->v_stride_h, c->v_stride_s, c->capacity, c->head_dim) ||
        same(c->k_scale, c->v_scale, 4 * c->ks_stride_b, 4 * c->ks_stride_h, 0, 4 * c->vs_stride_b, 4 * c->vs_stride_h, 0, 1, 4 * ((c->capacity + c->block - 1) / c->block)))
        return TRN_E_UNSUPPORTED;
    a.by_blocks = Div(a.n_blocks); a.by_heads = Div(c->n_kv_heads);
    a.xb[0] = k_stride_b; a.xh[0] = k_stride_h; a.xs[0] = k_stride_s;
    a.xb[1] = v_stride_b; a.xh[1] = v_stride_h; a.xs[1] = v_stride_s;
    a.cb[0] = c->k_stride_b; a.ch[0] = c->k_stride_h; a.cs[0] = c->k_stride_s;
    a.cb[1] = c->v_stride_b; a.ch[1] = c->v_stride_h; a.cs[1] = c->v_stride_s;
    a.sb[0] = c->ks_stride_b; a.sh[0] = c->ks_stride_h; a.sb[1] = c->vs_stride_b; a.sh[1] = c->vs_stride_h;
    const dim3 grid((unsigned)(units * a.n_blocks), 2);
    if (c->head_dim == 128) hipLaunchKernelGGL((cache8_append_kernel<128>), grid, dim3(256), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL((cache8_append_kernel<64>), grid, dim3(256), 0, (hipStream_t)stream, a);
    return hipGetLastError() == hipSuccess ? TRN_OK : TRN_E_LAUNCH;
}
