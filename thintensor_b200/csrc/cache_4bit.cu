// A block cache whose keys and values are held in 4 bits (see cache_4bit.cuh): writing it (with the rotation) and reading it back.  Head sizes 32,
// 64, 96 and 128, bfloat16 queries.
#include "cache_4bit.cuh"

namespace {

using cache4::block_bytes;
using cache4::code_bytes;

// ------------------------------------------------------------------------------------------------------------ appending
struct Group4 {
    float m, s, inverse;
    bool bad;
};

// m and s of a group from its least and greatest number (see above); all operations round to nearest except the two that do not.
__device__ __forceinline__ Group4 group_of(float least, float greatest, bool bad) {
    Group4 g;
    g.m = __bfloat162float(__float2bfloat16_rd(least));
    g.s = __bfloat162float(__float2bfloat16_ru(__fmul_rn(__fsub_rn(greatest, g.m), 1.0f / 15.0f)));
    g.bad = bad || !isfinite(g.m) || !isfinite(g.s);
    if (g.s < 1.17549435e-38f) g.s = 0.0f;
    g.inverse = g.s > 0.0f ? __frcp_rn(g.s) : 0.0f;
    return g;
}
__device__ __forceinline__ uint32_t code_of(const Group4& g, float x) {
    if (g.bad) return 0u;
    return (uint32_t)fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(x, g.m), g.inverse)), 0.0f), 15.0f);
}
__device__ __forceinline__ uint32_t bf16_bits(float x) { return __float_as_uint(x) >> 16; }      // of a number that is a bfloat16
__device__ __forceinline__ uint32_t scale_bits(const Group4& g) { return g.bad ? 0x7fc0u : bf16_bits(g.s); }
__device__ __forceinline__ uint32_t least_bits(const Group4& g) { return g.bad ? 0u : bf16_bits(g.m); }

// The group of the 32 numbers that 8 neighbouring lanes hold, four each (all 32 lanes call).
__device__ __forceinline__ Group4 group_of_lanes(const float (&x)[4]) {
    float least = fminf(fminf(x[0], x[1]), fminf(x[2], x[3])), greatest = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    bool bad = !(isfinite(x[0]) && isfinite(x[1]) && isfinite(x[2]) && isfinite(x[3]));
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
        greatest = fmaxf(greatest, __shfl_xor_sync(0xffffffffu, greatest, o));
    }
    bad = (__ballot_sync(0xffffffffu, bad) >> (threadIdx.x & 24)) & 0xffu;
    return group_of(least, greatest, bad);
}

// four neighbouring numbers, summed over the k-slices of the projection
template <bool VEC>
__device__ __forceinline__ void load_sums(const float* __restrict__ p, int splits, size_t stride, float (&x)[4]) {
    x[0] = x[1] = x[2] = x[3] = 0.0f;
    for (int s = 0; s < splits; ++s, p += stride) {
        if (VEC) {
            const float4 v = __ldg(reinterpret_cast<const float4*>(p));
            x[0] += v.x; x[1] += v.y; x[2] += v.z; x[3] += v.w;
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] += __ldg(p + k);
        }
    }
}

constexpr int APPEND_WARPS = 4;
constexpr int APPEND_MAX_HALF = 64;

// A warp takes rows (a head of a token) with four numbers a lane: queries and keys are rotated, queries narrowed, keys quantised;
// a row of values stands for up to four tokens of the sequence, those that share its code words with the token that owns them (the
// first of the step among them).  The angle position * frequency is formed in float64 and brought into one turn before the sine and
// cosine are taken in float32: a float32 product of a position in the hundred thousands is off by a hundredth of a radian, which moves
// codes.  grid = (tokens, parts).
template <int D, bool VEC>
__global__ void __launch_bounds__(APPEND_WARPS * 32)
rope_append_4bit_kernel(const float* __restrict__ qkv, int splits, size_t split_stride, const float* __restrict__ inv_freq, int rotary_dim,
                        int interleaved, float attention_scaling, __nv_bfloat16* __restrict__ q_out, uint8_t* __restrict__ k_pool,
                        uint8_t* __restrict__ v_pool, const int* __restrict__ table, int table_width, int pool_blocks,
                        const int* __restrict__ cu, const int* __restrict__ len_before, int sequences, int heads, int kv_heads,
                        int write_cache, unsigned* status) {
    constexpr int G = D / 32, LANES = D / 4, ROWS = 32 / LANES;        // lanes of a row, rows of a warp
    // Dependents start only behind this wait: a kernel that reads cache blocks ahead of its own wait then meets nothing older than this
    // launch still on its way.
    tt_pdl_wait();
    tt_pdl_launch_dependents();
    const int t = blockIdx.x;
    const int b = (sequences == (int)gridDim.x && cu[t] == t && cu[t + 1] == t + 1) ? t : tt_find_sequence(cu, sequences, t);
    const int seq_end = cu[b + 1];
    if (t >= seq_end) return;                                          // a row behind the last sequence
    const int pos = len_before[b] + (t - cu[b]);
    const int half = rotary_dim >> 1;
    __shared__ float cos_sh[APPEND_MAX_HALF], sin_sh[APPEND_MAX_HALF];
    for (int i = threadIdx.x; i < half; i += blockDim.x) {
        const double angle = (double)__ldg(inv_freq + i) * (double)pos;
        const double turned = fma(-rint(angle * 0.15915494309189535), 6.283185307179586, angle);
        float si, co;
        sincosf((float)turned, &si, &co);
        cos_sh[i] = co * attention_scaling;
        sin_sh[i] = si * attention_scaling;
    }
    int block = -1;
    if (write_cache) {
        const int entry = pos / TT_BLOCK_TOKENS;
        block = entry < table_width ? table[(size_t)b * table_width + entry] : -1;
        if (block >= pool_blocks) block = -1;
        if (block < 0 && threadIdx.x == 0) atomicOr(status, TT_STATUS_BAD_BLOCK);
    }
    const int slot = pos % TT_BLOCK_TOKENS;
    __syncthreads();
    const int cols = (heads + (write_cache ? 2 * kv_heads : 0)) * D;
    const float* row = qkv + (size_t)t * cols;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / LANES, l = lane % LANES;
    const int d0 = 4 * l, g = l >> 3, j = l & 7;
    const int rot_heads = heads + (write_cache ? kv_heads : 0);
    const int n_rot = (rot_heads + ROWS - 1) / ROWS;
    const bool owner = write_cache && block >= 0 && ((pos & 3) == 0 || t == cu[b]);
    const int n_val = owner ? (kv_heads + ROWS - 1) / ROWS : 0;
    for (int item = blockIdx.y * APPEND_WARPS + warp; item < n_rot + n_val; item += gridDim.y * APPEND_WARPS) {
        if (item < n_rot) {
            const int head = item * ROWS + sub;
            const bool active = sub < ROWS && head < rot_heads;
            float x[4] = {0.0f, 0.0f, 0.0f, 0.0f}, y[4];
            const float* p = row + (size_t)head * D;
            if (active) load_sums<VEC>(p + d0, splits, split_stride, x);
            if (interleaved) {
#pragma unroll
                for (int k = 0; k < 4; k += 2) {
                    const int i = (d0 + k) >> 1;
                    const bool turn = d0 + k < rotary_dim;
                    const float co = turn ? cos_sh[i] : 1.0f, si = turn ? sin_sh[i] : 0.0f;
                    y[k] = turn ? __fsub_rn(__fmul_rn(x[k], co), __fmul_rn(x[k + 1], si)) : x[k];
                    y[k + 1] = turn ? __fadd_rn(__fmul_rn(x[k + 1], co), __fmul_rn(x[k], si)) : x[k + 1];
                }
            } else {
                float other[4];                                        // the numbers that these are paired with
                if (VEC) {                                             // half a multiple of four: they are another lane's four
                    const int from = sub * LANES + (d0 < half ? l + (half >> 2) : (d0 < rotary_dim ? l - (half >> 2) : l));
#pragma unroll
                    for (int k = 0; k < 4; ++k) other[k] = __shfl_sync(0xffffffffu, x[k], from);
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int d = d0 + k;
                        other[k] = 0.0f;
                        if (active && d < rotary_dim)
                            for (int s = 0; s < splits; ++s) other[k] += __ldg(p + (d < half ? d + half : d - half) + s * split_stride);
                    }
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int d = d0 + k;
                    if (d < half) y[k] = __fsub_rn(__fmul_rn(x[k], cos_sh[d]), __fmul_rn(other[k], sin_sh[d]));
                    else if (d < rotary_dim) y[k] = __fadd_rn(__fmul_rn(x[k], cos_sh[d - half]), __fmul_rn(other[k], sin_sh[d - half]));
                    else y[k] = x[k];
                }
            }
            if (active && head < heads) {
                const __nv_bfloat162 lo = __floats2bfloat162_rn(y[0], y[1]), hi = __floats2bfloat162_rn(y[2], y[3]);
                uint2 v;
                v.x = *reinterpret_cast<const uint32_t*>(&lo);
                v.y = *reinterpret_cast<const uint32_t*>(&hi);
                *reinterpret_cast<uint2*>(q_out + ((size_t)t * heads + head) * D + d0) = v;
            }
            if (item * ROWS + ROWS <= heads) continue;                 // queries alone (the same for the whole warp)
            const Group4 grp = group_of_lanes(y);
            const int at = 8 * (j & 1);
            uint32_t word = code_of(grp, y[0]) << at | code_of(grp, y[1]) << (at + 16) | code_of(grp, y[2]) << (at + 4) | code_of(grp, y[3]) << (at + 20);
            word |= __shfl_xor_sync(0xffffffffu, word, 1);
            if (active && head >= heads && block >= 0) {
                uint8_t* dst = k_pool + ((size_t)block * kv_heads + (head - heads)) * block_bytes(D);
                if (!(j & 1)) reinterpret_cast<uint32_t*>(dst)[(slot * 4 + (j >> 1)) * G + g] = word;
                if (j == 0) reinterpret_cast<uint32_t*>(dst + code_bytes(D))[slot * G + g] = scale_bits(grp) | least_bits(grp) << 16;
            }
            continue;
        }
        const int kh = (item - n_rot) * ROWS + sub;
        const bool active = sub < ROWS && kh < kv_heads;
        uint8_t* dst = v_pool + ((size_t)block * kv_heads + (active ? kh : 0)) * block_bytes(D);
        uint16_t* scales = reinterpret_cast<uint16_t*>(dst + code_bytes(D));
        const int first = pos & 3, last = min(3, first + seq_end - 1 - t);   // the step's tokens among the word's four
        uint32_t words[4] = {0u, 0u, 0u, 0u}, fresh = 0u;
        for (int q = first; q <= last; ++q) {
            float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (active) load_sums<VEC>(row + (size_t)(q - first) * cols + (size_t)(rot_heads + kh) * D + d0, splits, split_stride, x);
            const Group4 grp = group_of_lanes(x);
            const int at = 8 * (q >> 1) + 16 * (q & 1);
            fresh |= 0xffu << at;
#pragma unroll
            for (int k = 0; k < 4; ++k) words[k] |= code_of(grp, x[k]) << (at + 4 * ((j >> 1) & 1));
            if (active && j == 0) {
                const int token = (slot & ~3) + q;
                scales[token * G + g] = (uint16_t)scale_bits(grp);
                scales[TT_BLOCK_TOKENS * G + g * TT_BLOCK_TOKENS + token] = (uint16_t)least_bits(grp);
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) words[k] |= __shfl_xor_sync(0xffffffffu, words[k], 2);      // numbers r and r + 8 share a word
        if (active) {
            const int a = slot >> 4, c = (slot >> 2) & 3, pick = j & 2;
            uint32_t* to = reinterpret_cast<uint32_t*>(dst) + ((((a * G + g) * 8 + 4 * (j & 1) + pick) * 4 + c) * 2 + (j >> 2));
            const uint32_t w0 = pick ? words[2] : words[0], w1 = pick ? words[3] : words[1];
            if (first == 0) {                                          // nothing older in these words
                to[0] = w0;
                to[8] = w1;
            } else {
                to[0] = (to[0] & ~fresh) | w0;
                to[8] = (to[8] & ~fresh) | w1;
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------------- reading back
// The blocks that a step sees, as bfloat16 blocks like the plain cache's (keys [token][D], values [D][token]), for kernels that read
// those: block w of sequence b goes to place b * span + w - (its first block that is seen), and table_tmp names the places (-1: not
// seen, or outside the pool).  Tokens behind the sequence's end become zeros.  Bound by the 16 bits a number that it writes.
// grid = (span, kv_heads, sequences).
template <int D>
__global__ void __launch_bounds__(128)
expand_4bit_kernel(const uint8_t* __restrict__ k_pool, const uint8_t* __restrict__ v_pool, const int* __restrict__ table, int table_width,
                   int pool_blocks, const int* __restrict__ cu, const int* __restrict__ len_before, int kv_heads, int window, int span,
                   __nv_bfloat16* __restrict__ keys, __nv_bfloat16* __restrict__ values, int* __restrict__ table_tmp, unsigned* status) {
    constexpr int G = D / 32;
    tt_pdl_wait();
    tt_pdl_launch_dependents();
    const int b = blockIdx.z, kh = blockIdx.y;
    const int before = len_before[b], length = before + cu[b + 1] - cu[b];
    const int first = tt_first_key(before, window) / TT_BLOCK_TOKENS, last = length > before ? (length - 1) / TT_BLOCK_TOKENS : first - 1;
    const int* table_row = table + (size_t)b * table_width;
    if (blockIdx.x == 0 && kh == 0) {
        for (int w = threadIdx.x; w < table_width; w += blockDim.x) {
            const bool there = w >= first && w <= last && w - first < span && table_row[w] >= 0 && table_row[w] < pool_blocks;
            table_tmp[(size_t)b * table_width + w] = there ? b * span + w - first : -1;
        }
        if (threadIdx.x == 0 && last - first >= span) atomicOr(status, TT_STATUS_BAD_SHAPE);
    }
    const int w = first + blockIdx.x;
    if (w > last) return;
    const int block = w < table_width ? table_row[w] : -1;
    if (block < 0 || block >= pool_blocks) {
        if (threadIdx.x == 0) atomicOr(status, TT_STATUS_BAD_BLOCK);
        return;
    }
    const int left = length - w * TT_BLOCK_TOKENS;                     // tokens of this block
    const size_t from = ((size_t)block * kv_heads + kh) * block_bytes(D), to = ((size_t)(b * span + blockIdx.x) * kv_heads + kh) * TT_BLOCK_TOKENS * D;
    const uint32_t* words = reinterpret_cast<const uint32_t*>(k_pool + from);
    const uint32_t* pairs = words + code_bytes(D) / 4;
    for (int i = threadIdx.x; i < TT_BLOCK_TOKENS * 4 * G; i += blockDim.x) {
        const int c = i & 3, g = (i >> 2) % G, token = (i >> 2) / G;   // eight neighbouring numbers
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (token < left) {
            const uint32_t word = __ldg(words + (token * 4 + c) * G + g), pair = __ldg(pairs + token * G + g);
            const float s = __uint_as_float(pair << 16), m = __uint_as_float(pair & 0xffff0000u);
            uint32_t out[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const __nv_bfloat162 two = __floats2bfloat162_rn(fmaf(s, (float)((word >> (4 * k)) & 15u), m), fmaf(s, (float)((word >> (4 * k + 16)) & 15u), m));
                out[k] = *reinterpret_cast<const uint32_t*>(&two);
            }
            v = make_uint4(out[0], out[1], out[2], out[3]);
        }
        *reinterpret_cast<uint4*>(keys + to + (size_t)token * D + 32 * g + 8 * c) = v;
    }
    words = reinterpret_cast<const uint32_t*>(v_pool + from);
    const __nv_bfloat16* scales = reinterpret_cast<const __nv_bfloat16*>(words + code_bytes(D) / 4);
    const __nv_bfloat16* least = scales + TT_BLOCK_TOKENS * G;
    for (int i = threadIdx.x; i < 16 * 16 * G; i += blockDim.x) {      // four tokens of two numbers
        const int c = i & 3, a = (i >> 2) & 3, r = (i >> 4) & 7, jj = (i >> 7) & 1, g = i >> 8;
        const uint32_t word = __ldg(words + (((a * G + g) * 8 + r) * 4 + c) * 2 + jj);
        const int token = 16 * a + 4 * c;
        float s[4], m[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            s[k] = __bfloat162float(scales[(token + k) * G + g]);
            m[k] = __bfloat162float(least[g * TT_BLOCK_TOKENS + token + k]);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                x[k] = token + k < left ? fmaf(s[k], (float)((word >> (4 * (2 * (k >> 1) + e) + 16 * (k & 1))) & 15u), m[k]) : 0.0f;
            const __nv_bfloat162 lo = __floats2bfloat162_rn(x[0], x[1]), hi = __floats2bfloat162_rn(x[2], x[3]);
            uint2 v;
            v.x = *reinterpret_cast<const uint32_t*>(&lo);
            v.y = *reinterpret_cast<const uint32_t*>(&hi);
            *reinterpret_cast<uint2*>(values + to + (size_t)(32 * g + 16 * jj + 8 * e + r) * TT_BLOCK_TOKENS + token) = v;
        }
    }
}

}  // namespace

extern "C" int tt_rope_append_4bit(const float* qkv, int splits, long long split_stride, const float* inv_freq, int rotary_dim, int interleaved,
                                   float attention_scaling, void* q_out, void* k_pool, void* v_pool, const int* table, int table_width,
                                   int pool_blocks, const int* cu, const int* len_before, int sequences, int n_tokens, int heads, int kv_heads,
                                   int head_dim, int write_cache, unsigned* status, cudaStream_t stream) {
    if (n_tokens <= 0) return 0;
    if (!cache4::takes(heads, kv_heads, head_dim) || rotary_dim < 0 || rotary_dim > head_dim || (rotary_dim & 1) || splits < 1 || sequences < 1 ||
        (((uintptr_t)q_out | (uintptr_t)k_pool | (uintptr_t)v_pool) & 15) != 0)
        return (int)cudaErrorInvalidValue;
    const bool vec = rotary_dim % 8 == 0 && split_stride % 4 == 0 && ((uintptr_t)qkv & 15) == 0;
    const int rows_per_warp = 32 / (head_dim / 4);
    const int items = (heads + (write_cache ? kv_heads : 0) + rows_per_warp - 1) / rows_per_warp + (write_cache ? (kv_heads + rows_per_warp - 1) / rows_per_warp : 0);
    // few tokens: a row a warp; prompts: a CTA a token, whose sines are taken once
    const int parts = n_tokens >= 512 ? 1 : (items + APPEND_WARPS - 1) / APPEND_WARPS;
#define TT_LAUNCH(D, V)                                                                                                                               \
    tt_launch_pdl(rope_append_4bit_kernel<D, V>, dim3(n_tokens, parts), dim3(APPEND_WARPS * 32), 0, stream, qkv, splits, (size_t)split_stride, inv_freq, \
                  rotary_dim, interleaved, attention_scaling, (__nv_bfloat16*)q_out, (uint8_t*)k_pool, (uint8_t*)v_pool, table, table_width, pool_blocks, \
                  cu, len_before, sequences, heads, kv_heads, write_cache, status)
#define TT_LAUNCH_D(D) (vec ? TT_LAUNCH(D, true) : TT_LAUNCH(D, false))
    switch (head_dim) {
        case 32: TT_LAUNCH_D(32); break;
        case 64: TT_LAUNCH_D(64); break;
        case 96: TT_LAUNCH_D(96); break;
        default: TT_LAUNCH_D(128); break;
    }
#undef TT_LAUNCH_D
#undef TT_LAUNCH
    TT_LAUNCH_CHECK();
}

extern "C" int tt_expand_4bit(const void* k_pool, const void* v_pool, const int* table, int table_width, int pool_blocks, const int* cu,
                              const int* len_before, int sequences, int kv_heads, int head_dim, int window, int span, void* keys, void* values,
                              int* table_tmp, unsigned* status, cudaStream_t stream) {
    if (sequences <= 0) return 0;
    if (!cache4::takes(kv_heads, kv_heads, head_dim) || span < 1 || sequences > 65535 || (((uintptr_t)keys | (uintptr_t)values) & 15) != 0) return (int)cudaErrorInvalidValue;
    const dim3 grid(span, kv_heads, sequences);
#define TT_LAUNCH(D)                                                                                                                             \
    tt_launch_pdl(expand_4bit_kernel<D>, grid, dim3(128), 0, stream, (const uint8_t*)k_pool, (const uint8_t*)v_pool, table, table_width, pool_blocks, \
                  cu, len_before, kv_heads, window, span, (__nv_bfloat16*)keys, (__nv_bfloat16*)values, table_tmp, status)
    switch (head_dim) {
        case 32: TT_LAUNCH(32); break;
        case 64: TT_LAUNCH(64); break;
        case 96: TT_LAUNCH(96); break;
        default: TT_LAUNCH(128); break;
    }
#undef TT_LAUNCH
    TT_LAUNCH_CHECK();
}
