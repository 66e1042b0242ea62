// A block cache whose keys and values are held in 4 bits (see cache_4bit.cuh): writing it (with the rotation) and reading it back.  Head sizes 32,
// 64, 96 and 128, bfloat16 queries.
#include <cuda_fp16.h>
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

// four neighbouring numbers of one k-slice of the projection
template <bool VEC>
__device__ __forceinline__ void load_four(const float* __restrict__ p, float (&x)[4]) {
    if (VEC) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(p));
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = __ldg(p + k);
    }
}

constexpr int APPEND_WARPS = 8;
constexpr int APPEND_MAX_HALF = 64;

// The values of a CTA's tokens: a warp takes a head of the (up to) four tokens that an owner among them stands for.
template <int D, bool VEC, int TOKENS>
__device__ __forceinline__ void values_of_tokens(const float* __restrict__ qkv, int splits, size_t split_stride, uint8_t* __restrict__ v_pool, int t0, int cols,
                                                 int rot_heads, int kv_heads, const int* pos_sh, const int* block_sh, const int* left_sh, const int* first_sh) {
    constexpr int G = D / 32, LANES = D / 4, ROWS = 32 / LANES;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / LANES, l = lane % LANES;
    const int d0 = 4 * l, g = l >> 3, j = l & 7, n_val = (kv_heads + ROWS - 1) / ROWS;
    // from the last warps on, which have the fewest rows of queries and keys
    for (int item = gridDim.y * APPEND_WARPS - 1 - (int)(blockIdx.y * APPEND_WARPS + warp); item < TOKENS * n_val; item += gridDim.y * APPEND_WARPS) {
        const int tok = item / n_val, t = t0 + tok, pos = pos_sh[tok], block = block_sh[tok], slot = pos % TT_BLOCK_TOKENS;
        if (block < 0 || left_sh[tok] <= 0 || ((pos & 3) != 0 && !first_sh[tok])) continue;    // another token owns the words (the same for the whole warp)
        const int kh = item % n_val * ROWS + sub;
        const bool active = sub < ROWS && kh < kv_heads;
        uint8_t* dst = v_pool + ((size_t)block * kv_heads + (active ? kh : 0)) * block_bytes(D);
        uint16_t* scales = reinterpret_cast<uint16_t*>(dst + code_bytes(D));
        const int first = pos & 3, last = min(3, first + left_sh[tok] - 1);    // the step's tokens among the words' four
        const float* row = qkv + (size_t)t * cols + (size_t)(rot_heads + (active ? kh : 0)) * D + d0;
        float v[4][4];
        for (int s = 0; s < splits; ++s) {
            float more[4][4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                more[q][0] = more[q][1] = more[q][2] = more[q][3] = 0.0f;
                if (active && q >= first && q <= last) load_four<VEC>(row + (ptrdiff_t)(q - first) * cols + s * split_stride, more[q]);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int k = 0; k < 4; ++k) v[q][k] = s ? v[q][k] + more[q][k] : more[q][k];
        }
        const int a = slot >> 4, c = (slot >> 2) & 3, pick = j & 2;
        uint32_t* to = reinterpret_cast<uint32_t*>(dst) + ((((a * G + g) * 8 + 4 * (j & 1) + pick) * 4 + c) * 2 + (j >> 2));
        uint32_t old0 = 0u, old1 = 0u;
        if (active && first != 0) { old0 = to[0]; old1 = to[8]; }      // older tokens' codes stay
        uint32_t words[4] = {0u, 0u, 0u, 0u}, fresh = 0u;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (q < first || q > last) continue;
            const Group4 grp = group_of_lanes(v[q]);
            const int at = 8 * (q >> 1) + 16 * (q & 1);
            fresh |= 0xffu << at;
#pragma unroll
            for (int k = 0; k < 4; ++k) words[k] |= code_of(grp, v[q][k]) << (at + 4 * ((j >> 1) & 1));
            if (active && j == 0) {
                const int token = (slot & ~3) + q;
                scales[token * G + g] = (uint16_t)scale_bits(grp);
                scales[TT_BLOCK_TOKENS * G + g * TT_BLOCK_TOKENS + token] = (uint16_t)least_bits(grp);
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) words[k] |= __shfl_xor_sync(0xffffffffu, words[k], 2);      // numbers r and r + 8 share a word
        if (active) {
            to[0] = (old0 & ~fresh) | (pick ? words[2] : words[0]);
            to[8] = (old1 & ~fresh) | (pick ? words[3] : words[1]);
        }
    }
}

// A warp takes rows (a head of a token) with four numbers a lane: queries and keys are rotated, queries narrowed, keys quantised;
// a row of values stands for up to four tokens of the sequence, those that share its code words with the token that owns them (the
// first of the step among them).  The angle position * frequency is formed in float64 and brought into one turn before the sine and
// cosine are taken in float32: a float32 product of a position in the hundred thousands is off by a hundredth of a radian, which moves
// codes.
//
// Prompts: a CTA takes TOKENS = 4 neighbouring tokens, whose places are looked up and whose 4 x 64 sines are taken by all its threads at
// once; a warp's rows are one token's, two at a time, and the next two are asked for before it works on them (2,048 tokens of 32/8 heads of 128: 21
// us, of which the bytes take 10; bound by the instructions of a row of keys or values, a hundred and more).  Few tokens: one a CTA, and as many
// CTAs a token as give every warp a row (8 tokens of 32/8 heads of 64 in four slices: 4 us).  grid = (tokens / TOKENS, parts).
template <int D, bool VEC, int TOKENS>
__global__ void __launch_bounds__(APPEND_WARPS * 32, TOKENS == 1 ? 2 : 4)
rope_append_4bit_kernel(const float* __restrict__ qkv, int splits, size_t split_stride, const float* __restrict__ inv_freq, int rotary_dim,
                        int interleaved, float attention_scaling, __nv_bfloat16* __restrict__ q_out, uint8_t* __restrict__ k_pool,
                        uint8_t* __restrict__ v_pool, const int* __restrict__ table, int table_width, int pool_blocks,
                        const int* __restrict__ cu, const int* __restrict__ len_before, int sequences, int n_tokens, int heads, int kv_heads,
                        int write_cache, unsigned* status) {
    constexpr int G = D / 32, LANES = D / 4, ROWS = 32 / LANES;        // lanes of a row, rows of a warp
    __shared__ float cos_sh[TOKENS][APPEND_MAX_HALF], sin_sh[TOKENS][APPEND_MAX_HALF];
    __shared__ int pos_sh[TOKENS], block_sh[TOKENS], left_sh[TOKENS], first_sh[TOKENS];        // left: tokens of the sequence from this one on, 0: none of any
    // Dependents start only behind this wait: a kernel that reads cache blocks ahead of its own wait then meets nothing older than this
    // launch still on its way.
    tt_pdl_wait();
    tt_pdl_launch_dependents();
    const int t0 = blockIdx.x * TOKENS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / LANES, l = lane % LANES;
    const int d0 = 4 * l, g = l >> 3, j = l & 7;
    const int rot_heads = heads + (write_cache ? kv_heads : 0);
    const int n_rot = (rot_heads + ROWS - 1) / ROWS;
    const int cols = (heads + (write_cache ? 2 * kv_heads : 0)) * D;
    // a warp's rows belong to one token: rows first_row, first_row + step, ... of its queries and keys, APPEND_ROWS at a time
    constexpr int PER_TOKEN = APPEND_WARPS / TOKENS, APPEND_ROWS = TOKENS == 1 ? 1 : 2, SLICES = TOKENS == 1 ? 3 : 1;
    const int tok = warp / PER_TOKEN, t = t0 + tok, step = gridDim.y * PER_TOKEN;
    int at_row = blockIdx.y * PER_TOKEN + warp % PER_TOKEN;
    const float* token_row = qkv + (size_t)t * cols + d0;
    auto mine = [&](int row) { return t < n_tokens && sub < ROWS && row * ROWS + sub < rot_heads; };
    // Slice s of the rows from `from` on, without touching what comes back: a thread waits for a number where it first computes with it.
    auto ask = [&](int from, int s, float (&x)[APPEND_ROWS][4]) {
#pragma unroll
        for (int i = 0; i < APPEND_ROWS; ++i) {
            x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.0f;
            if (mine(from + i * step)) load_four<VEC>(token_row + (size_t)((from + i * step) * ROWS + sub) * D + s * split_stride, x[i]);
        }
    };
    float x[APPEND_ROWS][4];
    ask(at_row, 0, x);                                                 // on their way while the places are looked up
    if (threadIdx.x < TOKENS) {
        const int u = t0 + threadIdx.x;
        int left = 0, pos = 0, block = -1, first = 0;
        if (u < n_tokens) {
            const int b = (TOKENS == 1 && sequences == (int)gridDim.x && cu[u] == u && cu[u + 1] == u + 1) ? u : tt_find_sequence(cu, sequences, u);
            left = max(0, cu[b + 1] - u);                              // a row behind the last sequence has none
            first = u == cu[b];
            pos = len_before[b] + (u - cu[b]);
            if (write_cache && left > 0) {
                const int entry = pos / TT_BLOCK_TOKENS;
                block = entry < table_width ? table[(size_t)b * table_width + entry] : -1;
                if (block >= pool_blocks) block = -1;
                if (block < 0) { block = -1; atomicOr(status, TT_STATUS_BAD_BLOCK); }
            }
        }
        pos_sh[threadIdx.x] = pos; block_sh[threadIdx.x] = block; left_sh[threadIdx.x] = left; first_sh[threadIdx.x] = first;
    }
    __syncthreads();
    const int half = rotary_dim >> 1;
    for (int i = threadIdx.x; i < TOKENS * half; i += APPEND_WARPS * 32) {
        const int of = i / half, f = i - of * half;
        const double angle = (double)__ldg(inv_freq + f) * (double)pos_sh[of];
        const double turned = fma(-rint(angle * 0.15915494309189535), 6.283185307179586, angle);
        float si, co;
        sincosf((float)turned, &si, &co);
        cos_sh[of][f] = co * attention_scaling;
        sin_sh[of][f] = si * attention_scaling;
    }
    __syncthreads();
    // the sines of this lane's four numbers: y = x * co + partner * si
    float co[4], si[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int d = d0 + k, f = interleaved ? d >> 1 : (d < half ? d : d - half);
        const bool turn = d < rotary_dim;
        co[k] = turn ? cos_sh[tok][f] : 1.0f;
        si[k] = turn ? sin_sh[tok][f] : 0.0f;
        if (interleaved ? !(d & 1) : d < half) si[k] = -si[k];
    }
    const int from_lane = sub * LANES + (d0 < half ? l + (half >> 2) : (d0 < rotary_dim ? l - (half >> 2) : l));
    const bool there = left_sh[tok] > 0;
    const int block = block_sh[tok], slot = pos_sh[tok] % TT_BLOCK_TOKENS;
    for (; at_row < n_rot; at_row += APPEND_ROWS * step) {
        for (int s = 1; s < splits; s += SLICES) {
            float more[SLICES][APPEND_ROWS][4];
#pragma unroll
            for (int e = 0; e < SLICES; ++e)
                if (s + e < splits) ask(at_row, s + e, more[e]);
#pragma unroll
            for (int e = 0; e < SLICES; ++e)
#pragma unroll
                for (int i = 0; i < APPEND_ROWS; ++i)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (s + e < splits) x[i][k] += more[e][i][k];
        }
        float ahead[APPEND_ROWS][4];
        ask(at_row + APPEND_ROWS * step, 0, ahead);
#pragma unroll
        for (int i = 0; i < APPEND_ROWS; ++i) {
            const int row = at_row + i * step;                         // the same for the whole warp
            if (row >= n_rot) break;
            const int head = row * ROWS + sub;
            const bool active = there && sub < ROWS && head < rot_heads;
            float y[4], other[4];                                      // the numbers that these are paired with
            if (interleaved) {
                other[0] = x[i][1]; other[1] = x[i][0]; other[2] = x[i][3]; other[3] = x[i][2];
            } else if (VEC) {                                          // half a multiple of four: they are another lane's four
#pragma unroll
                for (int k = 0; k < 4; ++k) other[k] = __shfl_sync(0xffffffffu, x[i][k], from_lane);
            } else {
                const float* p = token_row - d0 + (size_t)head * D;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int d = d0 + k;
                    other[k] = 0.0f;
                    if (active && d < rotary_dim)
                        for (int s = 0; s < splits; ++s) other[k] += __ldg(p + (d < half ? d + half : d - half) + s * split_stride);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] = d0 + k < rotary_dim ? __fadd_rn(__fmul_rn(x[i][k], co[k]), __fmul_rn(other[k], si[k])) : x[i][k];
            if (active && head < heads) {
                const __nv_bfloat162 lo = __floats2bfloat162_rn(y[0], y[1]), hi = __floats2bfloat162_rn(y[2], y[3]);
                uint2 v;
                v.x = *reinterpret_cast<const uint32_t*>(&lo);
                v.y = *reinterpret_cast<const uint32_t*>(&hi);
                *reinterpret_cast<uint2*>(q_out + ((size_t)t * heads + head) * D + d0) = v;
            }
            if (row * ROWS + ROWS <= heads) continue;                  // queries alone
            const Group4 grp = group_of_lanes(y);
            const int at = 8 * (j & 1);
            uint32_t word = code_of(grp, y[0]) << at | code_of(grp, y[1]) << (at + 16) | code_of(grp, y[2]) << (at + 4) | code_of(grp, y[3]) << (at + 20);
            word |= __shfl_xor_sync(0xffffffffu, word, 1);
            if (active && head >= heads && block >= 0) {
                uint8_t* dst = k_pool + ((size_t)block * kv_heads + (head - heads)) * block_bytes(D);
                if (!(j & 1)) reinterpret_cast<uint32_t*>(dst)[(slot * 4 + (j >> 1)) * G + g] = word;
                if (j == 0) reinterpret_cast<uint32_t*>(dst + code_bytes(D))[slot * G + g] = scale_bits(grp) | least_bits(grp) << 16;
            }
        }
#pragma unroll
        for (int i = 0; i < APPEND_ROWS; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) x[i][k] = ahead[i][k];
    }
    if (write_cache) values_of_tokens<D, VEC, TOKENS>(qkv, splits, split_stride, v_pool, t0, cols, rot_heads, kv_heads, pos_sh, block_sh, left_sh, first_sh);
}

// ---------------------------------------------------------------------------------------------------------- reading back
// The blocks that a step sees, as bfloat16 blocks like the plain cache's (keys [token][D], values [D][token]), for kernels that read
// those: block w of sequence b goes to place b * span + w - (its first block that is seen), and table_tmp names the places (-1: not
// seen, or outside the pool).  Tokens behind the sequence's end become zeros.  Bound by the 16 bits a number that it writes.
// grid = (2 * span, kv_heads, sequences): keys and values are CTAs of their own.
// HALF: float16 numbers instead, each times a power of two of its block and head, or of its token where a block's tokens are unlike, whose inverse goes to scales
// [keys or values][places][kv_heads] and marks [places][kv_heads][64] (a bfloat16 number would be m + s n rounded once more, to 8 bits; these have 11).  A
// group of values that is not a number becomes zeros, so that a product with a weight of zero is zero, and is marked.  See cache_4bit.cuh.
template <bool HALF>
__device__ __forceinline__ uint32_t two_numbers(float a, float b) {
    if constexpr (HALF) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}

template <int D, bool HALF>
__global__ void __launch_bounds__(256)
expand_4bit_kernel(const uint8_t* __restrict__ k_pool, const uint8_t* __restrict__ v_pool, const int* __restrict__ table, int table_width,
                   int pool_blocks, const int* __restrict__ cu, const int* __restrict__ len_before, int kv_heads, int window, int span,
                   uint16_t* __restrict__ keys, uint16_t* __restrict__ values, float* __restrict__ scales, uint8_t* __restrict__ marks, int* __restrict__ table_tmp, unsigned* status) {
    constexpr int G = D / 32;
    __shared__ float most[2][8], group_most[2][TT_BLOCK_TOKENS * G];
    __shared__ uint8_t steps_of[TT_BLOCK_TOKENS];
    __shared__ unsigned spread_sh;
    tt_pdl_wait();
    tt_pdl_launch_dependents();
    const int b = blockIdx.z, kh = blockIdx.y, place = blockIdx.x >> 1;
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
    const int w = first + place;
    if (w > last) return;
    const int block = w < table_width ? table_row[w] : -1;
    if (block < 0 || block >= pool_blocks) {
        if (threadIdx.x == 0) atomicOr(status, TT_STATUS_BAD_BLOCK);
        return;
    }
    const int left = length - w * TT_BLOCK_TOKENS;                     // tokens of this block
    const size_t from = ((size_t)block * kv_heads + kh) * block_bytes(D), to = ((size_t)(b * span + place) * kv_heads + kh) * TT_BLOCK_TOKENS * D;
    const bool of_keys = !(blockIdx.x & 1);
    const uint32_t* words = reinterpret_cast<const uint32_t*>((of_keys ? k_pool : v_pool) + from);
    const uint32_t* pairs = words + code_bytes(D) / 4;                 // of keys
    const __nv_bfloat16* tops = reinterpret_cast<const __nv_bfloat16*>(words + code_bytes(D) / 4);            // of values
    const __nv_bfloat16* least = tops + TT_BLOCK_TOKENS * G;
    float down = 1.0f;
    int exponent = 0, most_steps = 15;
    bool unlike = false;                                               // tokens have steps of their own
    auto down_of = [&](int token) { return HALF && unlike ? cache4::power_of_two(8 * min((int)steps_of[token], most_steps) - exponent) : down; };
    if constexpr (HALF) {
        // the largest number of the block and of each token: a thread a group of a token.  The marks need the keys' and the values'; the values' CTA writes them.
        const int sides = of_keys ? 1 : 2;
        float mine[2] = {0.0f, 0.0f};
        bool bad = false;
        if (threadIdx.x < TT_BLOCK_TOKENS * G && (int)threadIdx.x / G < left) {
            const uint32_t pair = __ldg(reinterpret_cast<const uint32_t*>(k_pool + from + code_bytes(D)) + threadIdx.x);
            const float s = __uint_as_float(pair << 16), m = __uint_as_float(pair & 0xffff0000u);
            if (s == s) mine[0] = fmaxf(fabsf(m), fabsf(fmaf(15.0f, s, m)));
            if (!of_keys) {
                const float vs = __bfloat162float(tops[threadIdx.x]), vm = __bfloat162float(least[threadIdx.x % G * TT_BLOCK_TOKENS + threadIdx.x / G]);
                bad = vs != vs;
                if (!bad) mine[1] = fmaxf(fabsf(vm), fabsf(fmaf(15.0f, vs, vm)));
            }
        }
        for (int k = 0; k < sides; ++k) {
            const uint32_t warp_most = __reduce_max_sync(0xffffffffu, __float_as_uint(mine[k]));
            if ((threadIdx.x & 31) == 0) most[k][threadIdx.x >> 5] = __uint_as_float(warp_most);
            if (threadIdx.x < TT_BLOCK_TOKENS * G) group_most[k][threadIdx.x] = mine[k];
        }
        if (threadIdx.x == 0) spread_sh = 0u;
        const bool any_bad = __syncthreads_or(bad);
        int steps[2] = {0, 0};
        for (int k = 0; k < sides; ++k) {
            float largest = most[k][0];
#pragma unroll
            for (int w = 1; w < 8; ++w) largest = fmaxf(largest, most[k][w]);
            exponent = cache4::half_exponent(largest);                 // its own kind's at last
            if (threadIdx.x < TT_BLOCK_TOKENS) {
                float token_most = 0.0f;
#pragma unroll
                for (int g = 0; g < G; ++g) token_most = fmaxf(token_most, group_most[k][threadIdx.x * G + g]);
                if (token_most > 0.0f) steps[k] = (exponent - cache4::half_exponent(token_most)) >> 3;
                steps_of[threadIdx.x] = (uint8_t)steps[k];
                if (steps[k] > 1) atomicOr(&spread_sh, 1u << k);       // more than a step between two tokens (a token of zeros goes with any)
            }
        }
        __syncthreads();
        const unsigned spread = spread_sh;
        steps[0] = spread & 1u ? min(steps[0], 15) : 0;
        most_steps = !of_keys && spread & 1u ? 14 : 15;
        steps[1] = spread & 2u ? min(steps[1], most_steps) : 0;
        unlike = spread >> (sides - 1) & 1u;
        down = cache4::power_of_two(-exponent);
        const size_t slot = ((size_t)b * span + place) * kv_heads + kh;
        const bool flagged = of_keys ? unlike : any_bad || unlike;
        if (threadIdx.x == 0) scales[(of_keys ? 0 : (size_t)gridDim.z * span * kv_heads) + slot] = flagged ? -cache4::power_of_two(exponent) : cache4::power_of_two(exponent);
        if (!of_keys && threadIdx.x < TT_BLOCK_TOKENS && (flagged || (spread & 1u))) {
            unsigned mask = 0;
            for (int k = 0; k < G; ++k) mask |= (unsigned)((int)threadIdx.x < left && tops[threadIdx.x * G + k] != tops[threadIdx.x * G + k]) << k;
            const unsigned mark = !(spread & 1u) ? (unsigned)steps[1] << 4 | mask
                                  : mask ? 0xf0u | (steps[0] || steps[1] ? 15u : mask) : (unsigned)(steps[1] << 4 | steps[0]);
            marks[slot * TT_BLOCK_TOKENS + threadIdx.x] = (uint8_t)mark;
        }
    }
    if (of_keys) {
#pragma unroll
        for (int k = 0; k < G; ++k) {
            const int i = k * 256 + threadIdx.x;
            const int c = i & 3, g = (i >> 2) % G, token = (i >> 2) / G;       // eight neighbouring numbers
            const uint32_t word = __ldg(words + (token * 4 + c) * G + g), pair = __ldg(pairs + token * G + g);
            const float times = down_of(token), s = __uint_as_float(pair << 16) * times, m = __uint_as_float(pair & 0xffff0000u) * times;
            uint32_t out[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t two = two_numbers<HALF>(fmaf(s, (float)((word >> (4 * e)) & 15u), m), fmaf(s, (float)((word >> (4 * e + 16)) & 15u), m));
                out[e] = token < left ? two : 0u;
            }
            *reinterpret_cast<uint4*>(keys + to + (size_t)token * D + 32 * g + 8 * c) = make_uint4(out[0], out[1], out[2], out[3]);
        }
        return;
    }
    const int c = threadIdx.x & 3, a = (threadIdx.x >> 2) & 3, r = (threadIdx.x >> 4) & 7, jj = threadIdx.x >> 7, token = 16 * a + 4 * c;
#pragma unroll
    for (int g = 0; g < G; ++g) {                                      // four tokens of two numbers
        const uint32_t word = __ldg(words + (((a * G + g) * 8 + r) * 4 + c) * 2 + jj);
        const uint2 low = __ldg(reinterpret_cast<const uint2*>(least + g * TT_BLOCK_TOKENS + token));
        const float m[4] = {__uint_as_float(low.x << 16), __uint_as_float(low.x & 0xffff0000u), __uint_as_float(low.y << 16), __uint_as_float(low.y & 0xffff0000u)};
        float s[4], times[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            times[k] = down_of(token + k);
            s[k] = __bfloat162float(tops[(token + k) * G + g]) * times[k];
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                x[k] = token + k < left && (!HALF || s[k] == s[k]) ? fmaf(s[k], (float)((word >> (4 * (2 * (k >> 1) + e) + 16 * (k & 1))) & 15u), m[k] * times[k]) : 0.0f;
            const uint2 v = make_uint2(two_numbers<HALF>(x[0], x[1]), two_numbers<HALF>(x[2], x[3]));
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
    const bool many = n_tokens >= 256;                                  // (598 tokens of 20/4 heads of 96: 18 us with a token a CTA, 10 with four)
    const dim3 grid(many ? (n_tokens + 3) / 4 : n_tokens, many ? 1 : (items + APPEND_WARPS - 1) / APPEND_WARPS);
#define TT_LAUNCH(D, V, T)                                                                                                                            \
    tt_launch_pdl(rope_append_4bit_kernel<D, V, T>, grid, dim3(APPEND_WARPS * 32), 0, stream, qkv, splits, (size_t)split_stride, inv_freq, rotary_dim, \
                  interleaved, attention_scaling, (__nv_bfloat16*)q_out, (uint8_t*)k_pool, (uint8_t*)v_pool, table, table_width, pool_blocks, cu,     \
                  len_before, sequences, n_tokens, heads, kv_heads, write_cache, status)
#define TT_LAUNCH_D(D) (vec ? (many ? TT_LAUNCH(D, true, 4) : TT_LAUNCH(D, true, 1)) : (many ? TT_LAUNCH(D, false, 4) : TT_LAUNCH(D, false, 1)))
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

// scales, marks: null for bfloat16 keys and values, else those of float16 ones.
extern "C" int tt_expand_4bit(const void* k_pool, const void* v_pool, const int* table, int table_width, int pool_blocks, const int* cu,
                              const int* len_before, int sequences, int kv_heads, int head_dim, int window, int span, void* keys, void* values,
                              float* scales, uint8_t* marks, int* table_tmp, unsigned* status, cudaStream_t stream) {
    if (sequences <= 0) return 0;
    if (!cache4::takes(kv_heads, kv_heads, head_dim) || span < 1 || sequences > 65535 || (scales != nullptr) != (marks != nullptr) || (((uintptr_t)keys | (uintptr_t)values) & 15) != 0) return (int)cudaErrorInvalidValue;
    if (span > (1 << 29)) return (int)cudaErrorInvalidValue;
    const dim3 grid(2 * span, kv_heads, sequences);
#define TT_LAUNCH_T(D, H)                                                                                                                           \
    tt_launch_pdl(expand_4bit_kernel<D, H>, grid, dim3(256), 0, stream, (const uint8_t*)k_pool, (const uint8_t*)v_pool, table, table_width, pool_blocks, \
                  cu, len_before, kv_heads, window, span, (uint16_t*)keys, (uint16_t*)values, scales, marks, table_tmp, status)
#define TT_LAUNCH(D) (scales ? TT_LAUNCH_T(D, true) : TT_LAUNCH_T(D, false))
    switch (head_dim) {
        case 32: TT_LAUNCH(32); break;
        case 64: TT_LAUNCH(64); break;
        case 96: TT_LAUNCH(96); break;
        default: TT_LAUNCH(128); break;
    }
#undef TT_LAUNCH
#undef TT_LAUNCH_T
    TT_LAUNCH_CHECK();
}
