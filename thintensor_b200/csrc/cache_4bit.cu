// A block cache whose keys and values are held in 4 bits: writing it (with the rotation), reading it back, and causal
// grouped-query attention over it.  Head sizes 32, 64, 96 and 128, bfloat16 queries, up to 16 query heads per key/value head.
//
// The numbers.  A head of D numbers is cut into G = D / 32 groups of 32 neighbouring ones.  A group of a token is held as 32
// codes n of 4 bits, a scale s and a least value m, both bfloat16, and stands for m + s n:
//   m = the least of the 32, rounded down to bfloat16;  s = (greatest - m) / 15, rounded up to bfloat16;
//   n = the nearest whole number to (x - m) / s, 0..15.
// Down and up, so that no number of the group lies outside what the codes reach and every one is met within s / 2.  A group that
// holds something not finite, or whose m or s would not be, has s = NaN, m = 0, n = 0: whoever sees it gets NaN, and a key that is
// masked adds 0 * m = 0.  A scale below 2^-126 (the inverse would overflow) is zero: the numbers then differ by less than 2^-122.
//
// Groups of 32 rather than whole heads: a key's few large channels cost precision only among their 31 neighbours.  5 bits a number
// against 16 of the bfloat16 cache.
//
// The bytes of one block (64 tokens) of one head, 20 * 64 * G each for keys and for values:
//   keys:   codes, 32-bit words [64 tokens][4][G]; then [64 tokens][G] pairs (s in the low half, m in the high half)
//           word [t][c][g]: numbers 32 g + 8 c + 2 i + h of token t at bits 4 i + 16 h (i = 0..3, h = 0, 1)
//   values: codes, 32-bit words [4][G][8][4][2]; then s [64 tokens][G]; then m [G][64 tokens]
//           word [a][g][r][c][j]: number 32 g + 16 j + 8 e + r of token 16 a + 4 c + 2 p + h at bits 4 (2 p + e) + 16 h
// Both are the order in which a lane of a tensor-core fragment (m16n8k16) wants them: (w >> 4 i) & 0x000f000f | 0x43004300 is a
// register of two bfloat16 numbers 128 + n, w & 0x000f000f | 0x64006400 one of two float16 numbers 1024 + n.  A value word holds four
// neighbouring tokens; whoever appends owns the word of its first token in it and keeps what earlier steps left in the others.
#include "attention_kernels.cuh"
#include "tcgen05.cuh"

#include <cuda_fp16.h>

#include <cooperative_groups.h>
namespace cg = cooperative_groups;

namespace {

constexpr int block_bytes(int d) { return 40 * d; }                 // of one head's keys, or values
constexpr int code_bytes(int d) { return 32 * d; }                  // the codes among them

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

// ------------------------------------------------------------------------------------------------------------- attention
// With codes n, scales s and least values m of key t and value t (primes for values), per group g:
//   score(q, t) = sum_g s_tg (q . n)_tg + m_tg (sum of q over g),     out_g = sum_t (p_t s'_tg) n'_t + p_t m'_tg.
// So the tensor cores multiply codes, not numbers.  As float16 the bits 0x000n are n 2^-24 and 0x00n0 are 16 n 2^-24 (numbers below the
// normal ones, which the tensor cores take as they are): an operand register of two codes is one mask away from the cache's word, and
// eight codes take one shift and four masks.  What the sixteens multiply is a sixteenth (queries) or is taken off the sums' rows
// (values), the 2^24 goes into the scale.  Group scales meet the 16 x 8 tile of a group's products (S^T: 16 keys, 8 queries) and the
// probabilities; the least values are one more product of each, in bfloat16.
//
// Queries are float16 after a power of two that brings a row's greatest number to 2^14: exact but for what lies 2^-28 below that.
// The weights p s' are rounded to float16 (11 bits): with weights in bfloat16 the two terms of out, which are of opposite sign and
// each several times their sum, were off by 0.4 % of it.  So that float16 holds them whatever the values' size, p is formed relative to
// the running maximum times 2^(E - 14), E the exponent of the largest scale that the warp has met (at least -40): the weights stay
// below 2^15, and what falls under 2^-14 is less than 2^-29 of the largest.  The second term takes p in two bfloat16 parts (16 bits)
// and m' as it is, the second term of S the queries' sums in three.  All sums are float32.
//
// Rows of up to four queries (DUP) stand twice in the tile's eight columns, which would otherwise be half empty: the weights of one
// group of numbers lie in the first four, those of the next group in the others, and the products of either group take the same
// operand.
//
// A warp owns up to 8 NQ query rows of one sequence and key/value head, (token, head of the group) pairs, and walks its share of the
// blocks; the copy engine brings a block's keys and values (5 KB each at D = 128) into its ring of shared-memory stages a block ahead.
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
    return d;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float bf16_low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
// 2^x on the special-function unit (relative error about 2^-22), 2^-inf = 0; what it gives is rounded to float16 or summed beside that.
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void bulk_copy(void* smem_dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(tc::smem_u32(smem_dst)), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
constexpr uint32_t ONES_MASK = 0x000f000fu, SIXTEENS_MASK = 0x00f000f0u;       // codes n and 16 n of a word
constexpr float CODE_UNIT = 5.9604644775390625e-08f;                            // 2^-24

template <int N> __device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
    if constexpr (N == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if constexpr (N == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x; w[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    }
}

template <int D, int NQ, bool DUP> struct Rows4 {
    static constexpr int G = D / 32;
    uint32_t q[NQ][G][4];               // query 8 nq + r: numbers 32 g + 8 c + 2 i and + 1 in register i, float16, those of odd i a sixteenth
    uint32_t q_sum[NQ][2];              // the sum of query 8 nq + r over group c, in three bfloat16 parts
    float o[2 * G][NQ][4];              // [0], [1]: number 16 dt + r, queries 8 nq + 2 c + e; [2], [3]: number + 8, sixteenfold
    float least[NQ][4];                 // row r = group r: the least values' share
    float scale[NQ][2];                 // of the scores of queries 8 nq + 2 c + e, in log2 units
    float m_run[NQ][2], l_run[NQ][2];   // l: this lane's share (its keys) until the end
    int e_run;                          // E: all weights and sums are relative to 2^(m_run + E - 14)
    int pos[NQ][2], first[NQ][2];       // queries 8 nq + 2 c + e see keys first .. pos
};

template <int D, int NQ, bool DUP>
__device__ __forceinline__ void block_of_keys(Rows4<D, NQ, DUP>& st, const uint8_t* __restrict__ kb, const uint8_t* __restrict__ vb, int key_base,
                                              bool all_visible, int first_seen, int last_pos, int r, int c) {
    constexpr int G = Rows4<D, NQ, DUP>::G;
    const int lane = 4 * r + c;
    const int token0 = 4 * (r >> 1) + (r & 1);                         // rows r and r + 8 of a tile of 16 keys: tokens token0 and + 2
    float s[4][NQ][4];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
        const int t0 = 16 * kt + token0;
        const uint8_t* pairs = kb + code_bytes(D) + t0 * 4 * G;
        uint32_t w0[G], w1[G], p0[G], p1[G];
        load_words<G>(kb + (t0 * 4 + c) * 4 * G, w0);
        load_words<G>(kb + ((t0 + 2) * 4 + c) * 4 * G, w1);
        load_words<G>(pairs, p0);
        load_words<G>(pairs + 8 * G, p1);
        // the least values of group c, twice in a register
        const uint32_t m0 = c < G ? __byte_perm(reinterpret_cast<const uint32_t*>(pairs)[c < G ? c : 0], 0u, 0x3232) : 0u;
        const uint32_t m1 = c < G ? __byte_perm(reinterpret_cast<const uint32_t*>(pairs + 8 * G)[c < G ? c : 0], 0u, 0x3232) : 0u;
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
            s[kt][nq][0] = s[kt][nq][1] = s[kt][nq][2] = s[kt][nq][3] = 0.0f;
            mma_bf16(s[kt][nq], m0, m1, m0, m1, st.q_sum[nq][0], st.q_sum[nq][1]);
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const uint32_t h0 = w0[g] >> 8, h1 = w1[g] >> 8;
            const float s0 = bf16_low(p0[g]), s1 = bf16_low(p1[g]);
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq) {
                float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                mma_f16(acc, w0[g] & ONES_MASK, w1[g] & ONES_MASK, w0[g] & SIXTEENS_MASK, w1[g] & SIXTEENS_MASK, st.q[nq][g][0], st.q[nq][g][1]);
                mma_f16(acc, h0 & ONES_MASK, h1 & ONES_MASK, h0 & SIXTEENS_MASK, h1 & SIXTEENS_MASK, st.q[nq][g][2], st.q[nq][g][3]);
                s[kt][nq][0] = fmaf(s0, acc[0], s[kt][nq][0]);
                s[kt][nq][1] = fmaf(s0, acc[1], s[kt][nq][1]);
                s[kt][nq][2] = fmaf(s1, acc[2], s[kt][nq][2]);
                s[kt][nq][3] = fmaf(s1, acc[3], s[kt][nq][3]);
            }
        }
    }
    const uint8_t* scales = vb + code_bytes(D);
    const uint8_t* mins = scales + 2 * TT_BLOCK_TOKENS * G;
    // the bits of the block's largest scale: a lane looks at two neighbouring tokens (positive bfloat16 numbers order like their bits; a scale
    // that is not a number counts for nothing here)
    uint32_t top = 0u;
    {
        uint32_t two[G];
        load_words<G>(scales + 2 * lane * 2 * G, two);
        if (all_visible) {
            __nv_bfloat162 most = *reinterpret_cast<const __nv_bfloat162*>(&two[0]);
#pragma unroll
            for (int i = 1; i < G; ++i) most = __hmax2(most, *reinterpret_cast<const __nv_bfloat162*>(&two[i]));
            const uint32_t bits = *reinterpret_cast<const uint32_t*>(&most), lo = bits & 0xffffu, hi = bits >> 16;
            top = max(lo <= 0x7f80u ? lo : 0u, hi <= 0x7f80u ? hi : 0u);
        } else {
#pragma unroll
            for (int i = 0; i < 2 * G; ++i) {
                const uint32_t bits = (two[i >> 1] >> (16 * (i & 1))) & 0xffffu;
                const int key = key_base + 2 * lane + i / G;
                if (bits <= 0x7f80u && key <= last_pos && key >= first_seen) top = max(top, bits);
            }
#pragma unroll
            for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                for (int hi = 0; hi < 2; ++hi) {
                    const int key = key_base + 16 * kt + token0 + 2 * hi;
#pragma unroll
                    for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            if (!(key <= st.pos[nq][e] && key >= st.first[nq][e])) s[kt][nq][2 * hi + e] = -INFINITY;
                }
        }
    }
    const int e_new = max(st.e_run, (int)(__reduce_max_sync(0xffffffffu, top) >> 7) - 127);
    const float e_old = (float)(st.e_run - 14), e_now = (float)(e_new - 14);
    st.e_run = e_new;
    float corr[NQ][2];
    bool grew = false;
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float mx = -INFINITY;
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) mx = fmaxf(mx, fmaxf(s[kt][nq][e], s[kt][nq][2 + e]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float m_new = fmaxf(st.m_run[nq][e], mx * st.scale[nq][e]);         // the scale is positive
            corr[nq][e] = m_new == -INFINITY ? 1.0f : fast_exp2((st.m_run[nq][e] - m_new) + (e_old - e_now));
            grew = grew || corr[nq][e] != 1.0f;
            const float base = m_new == -INFINITY ? 0.0f : -(m_new + e_now);
            float sum = 0.0f;
#pragma unroll
            for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                for (int hi = 0; hi < 2; ++hi) {
                    const float p = fast_exp2(fmaf(s[kt][nq][2 * hi + e], st.scale[nq][e], base));
                    s[kt][nq][2 * hi + e] = p;
                    sum += p;
                }
            st.l_run[nq][e] = st.l_run[nq][e] * corr[nq][e] + sum;
            // a key that is not a number has no part in the maximum; what this warp saw must count all the same where others' results join it
            st.m_run[nq][e] = (m_new == -INFINITY && sum != sum) ? 0.0f : m_new;
        }
    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
#pragma unroll
            for (int dt = 0; dt < 2 * G; ++dt) {
                st.o[dt][nq][0] *= corr[nq][0]; st.o[dt][nq][1] *= corr[nq][1];
                st.o[dt][nq][2] *= corr[nq][0]; st.o[dt][nq][3] *= corr[nq][1];
            }
            st.least[nq][0] *= corr[nq][0]; st.least[nq][1] *= corr[nq][1];
        }
    }
    constexpr int SETS = DUP ? (G + 1) / 2 : G;                        // operands of weights: with DUP one holds two groups'
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
        const int t0 = 16 * kt + token0;
        // least values: row g of the operand is group g, its columns are this lane's four tokens
        uint2 low = make_uint2(0u, 0u);
        if (r < G) low = *reinterpret_cast<const uint2*>(mins + (r * TT_BLOCK_TOKENS + 16 * kt + 4 * c) * 2);
        if (!all_visible) {                                            // what lies behind the sequence's end may be anything
            const int key = key_base + 16 * kt + 4 * c;
            if (key > last_pos) low.x &= 0xffff0000u;
            if (key + 1 > last_pos) low.x &= 0x0000ffffu;
            if (key + 2 > last_pos) low.y &= 0xffff0000u;
            if (key + 3 > last_pos) low.y &= 0x0000ffffu;
        }
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
            float rest[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) rest[i] = s[kt][nq][i] - bf16_high(__float_as_uint(s[kt][nq][i]));
            if constexpr (DUP) {                                       // the first part in the first four columns, the second in the others
#pragma unroll
                for (int i = 0; i < 4; ++i) rest[i] = c < 2 ? bf16_high(__float_as_uint(s[kt][nq][i])) : rest[i];
                mma_bf16(st.least[nq], low.x, 0u, low.y, 0u, transpose_8x8(pack_bf16(rest[0], rest[1])), transpose_8x8(pack_bf16(rest[2], rest[3])));
            } else {
                const uint32_t hi0 = __byte_perm(__float_as_uint(s[kt][nq][0]), __float_as_uint(s[kt][nq][1]), 0x7632);
                const uint32_t hi1 = __byte_perm(__float_as_uint(s[kt][nq][2]), __float_as_uint(s[kt][nq][3]), 0x7632);
                mma_bf16(st.least[nq], low.x, 0u, low.y, 0u, transpose_8x8(hi0), transpose_8x8(hi1));
                mma_bf16(st.least[nq], low.x, 0u, low.y, 0u, transpose_8x8(pack_bf16(rest[0], rest[1])), transpose_8x8(pack_bf16(rest[2], rest[3])));
            }
        }
        const __nv_bfloat16* scale0 = reinterpret_cast<const __nv_bfloat16*>(scales) + t0 * G;
#pragma unroll
        for (int set = 0; set < SETS; ++set) {
            const int mine = DUP ? min(2 * set + (c >> 1), G - 1) : set;       // the group whose weights this lane forms
            const float s0 = __bfloat162float(scale0[mine]), s1 = __bfloat162float(scale0[2 * G + mine]);
            uint32_t b0[NQ], b1[NQ];
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq) {
                float p0 = s[kt][nq][0] * s0, p1 = s[kt][nq][1] * s0, p2 = s[kt][nq][2] * s1, p3 = s[kt][nq][3] * s1;
                if (!all_visible) {                                    // a masked value adds nothing, whatever its scale
                    p0 = s[kt][nq][0] == 0.0f ? 0.0f : p0; p1 = s[kt][nq][1] == 0.0f ? 0.0f : p1;
                    p2 = s[kt][nq][2] == 0.0f ? 0.0f : p2; p3 = s[kt][nq][3] == 0.0f ? 0.0f : p3;
                }
                b0[nq] = transpose_8x8(pack_f16(p0, p1));
                b1[nq] = transpose_8x8(pack_f16(p2, p3));
            }
#pragma unroll
            for (int g = DUP ? 2 * set : set; g < (DUP ? min(2 * set + 2, G) : set + 1); ++g) {
                const uint2 w = *reinterpret_cast<const uint2*>(vb + ((kt * G + g) * 32 + lane) * 8);
                const uint32_t x8 = w.x >> 8, y8 = w.y >> 8;
#pragma unroll
                for (int nq = 0; nq < NQ; ++nq) {
                    mma_f16(st.o[2 * g][nq], w.x & ONES_MASK, w.x & SIXTEENS_MASK, x8 & ONES_MASK, x8 & SIXTEENS_MASK, b0[nq], b1[nq]);
                    mma_f16(st.o[2 * g + 1][nq], w.y & ONES_MASK, w.y & SIXTEENS_MASK, y8 & ONES_MASK, y8 & SIXTEENS_MASK, b0[nq], b1[nq]);
                }
            }
        }
    }
}

template <int D> struct Ring4 {
    static constexpr int WARPS = 8, STAGES = 2;
    static constexpr int STAGE = 2 * block_bytes(D);
    static constexpr int PITCH = D + 4;
    static constexpr int RING = WARPS * STAGES * STAGE;
    static constexpr int results(int rows) { return WARPS * rows * (PITCH + 2) * 4 + rows * (D + 2) * 4; }     // where the warps' results meet
    static constexpr int shared(int rows) { return RING > results(rows) ? RING : results(rows); }
};

// grid = (tiles, kv_heads, splits).  tokens_per_tile 1 with one token a sequence: tile = sequence.
template <int D, int NQ, bool DUP>
__global__ void __launch_bounds__(Ring4<D>::WARPS * 32)
attention_4bit_kernel(const __nv_bfloat16* __restrict__ q, const uint8_t* __restrict__ k_pool, const uint8_t* __restrict__ v_pool,
                      const int* __restrict__ table, int table_width, int pool_blocks, const int* __restrict__ cu,
                      const int* __restrict__ len_before, int sequences, int heads, int kv_heads, int tokens_per_tile, int one_token_each,
                      float scale_log2, int window, int splits, int cluster_merge, __nv_bfloat16* __restrict__ out,
                      float* __restrict__ part_acc, float* __restrict__ part_ml, unsigned* status, const float* __restrict__ sinks) {
    using R = Ring4<D>;
    constexpr int G = D / 32, WARPS = R::WARPS, STAGES = R::STAGES, COLS = 8 * NQ;
    extern __shared__ __align__(128) uint8_t shared[];
    __shared__ uint64_t landed[WARPS][STAGES];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const int kh = blockIdx.y, split = blockIdx.z, group = heads / kv_heads;
    if (lane == 0)
        for (int i = 0; i < STAGES; ++i) tc::mbar_init(tc::smem_u32(&landed[warp][i]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncwarp();
    tt_pdl_launch_dependents();
    tt_pdl_wait();

    // which sequence, and which of its tokens
    int b, tok0;
    if (one_token_each) {
        b = blockIdx.x;
        tok0 = 0;
    } else {
        int tile = blockIdx.x;
        b = -1;
        for (int base = 0; base < sequences && b < 0; base += 32) {
            const int mine = base + lane;
            const int count = mine < sequences ? (cu[mine + 1] - cu[mine] + tokens_per_tile - 1) / tokens_per_tile : 0;
            int prefix = count;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, prefix, o);
                if (lane >= o) prefix += up;
            }
            const unsigned owner = __ballot_sync(0xffffffffu, tile < prefix);
            if (owner) {
                const int at = __ffs(owner) - 1;
                b = base + at;
                tile -= __shfl_sync(0xffffffffu, prefix - count, at);
            } else {
                tile -= __shfl_sync(0xffffffffu, prefix, 31);
            }
        }
        if (b < 0) return;               // a spare CTA (the grid is an upper bound): all of its warps, and of its cluster, leave together
        tok0 = tile * tokens_per_tile;
    }
    const int seq_begin = cu[b], seq_new = cu[b + 1] - seq_begin;
    const int tokens = min(tokens_per_tile, seq_new - tok0);
    if (tokens <= 0) return;             // a sequence without a token: the same for the whole cluster
    const int pos0 = len_before[b] + tok0, last_pos = pos0 + tokens - 1;
    const int n_rows = tokens * group;
    const int first_key = tt_first_key(pos0, window), last_first = tt_first_key(last_pos, window);
    const int block0 = first_key / TT_BLOCK_TOKENS, n_blocks = last_pos / TT_BLOCK_TOKENS - block0 + 1;
    const int per = (n_blocks + splits - 1) / splits;
    const int begin = block0 + split * per, end = min(begin + per, block0 + n_blocks);
    const int n_mine = begin + warp < end ? (end - begin - warp + WARPS - 1) / WARPS : 0;
    const int* table_row = table + (size_t)b * table_width;
    uint8_t* ring = shared + (size_t)warp * STAGES * R::STAGE;

    int issued = 0;
    unsigned valid = 0;                  // bit i % 32: block i is in the pool
    auto issue_next = [&]() {
        const int i = issued++;
        const int kb = begin + warp + i * WARPS;
        const int block = kb < table_width ? __ldg(table_row + kb) : -1;
        const bool ok = block >= 0 && block < pool_blocks;
        valid = (valid & ~(1u << (i & 31))) | ((unsigned)ok << (i & 31));
        if (lane == 0) {
            const uint32_t bar = tc::smem_u32(&landed[warp][i % STAGES]);
            if (ok) {
                uint8_t* dst = ring + (size_t)(i % STAGES) * R::STAGE;
                const size_t from = ((size_t)block * kv_heads + kh) * block_bytes(D);
                tc::mbar_expect_tx(bar, R::STAGE);
                bulk_copy(dst, k_pool + from, block_bytes(D), bar);
                bulk_copy(dst + block_bytes(D), v_pool + from, block_bytes(D), bar);
            } else {
                tc::mbar_arrive(bar);
                atomicOr(status, TT_STATUS_BAD_BLOCK);
            }
        }
    };
    while (issued < min(n_mine, STAGES)) issue_next();

    Rows4<D, NQ, DUP> st;
    st.e_run = -40;
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
        const int row = DUP ? r & 3 : 8 * nq + r;
        const __nv_bfloat16* src = q + ((size_t)(seq_begin + tok0 + row / group) * heads + kh * group + row % group) * D + 8 * c;
        uint4 v[G];
        uint32_t most = 0u;                                            // bits of the row's greatest number without its sign
#pragma unroll
        for (int g = 0; g < G; ++g) {
            v[g] = row < n_rows ? *reinterpret_cast<const uint4*>(src + 32 * g) : make_uint4(0u, 0u, 0u, 0u);
            const uint32_t w[4] = {v[g].x, v[g].y, v[g].z, v[g].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) most = max(most, max((w[i] << 16) & 0x7fffffffu, w[i] & 0x7fff0000u));
        }
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // times 2^up: the greatest number's exponent becomes 14
        const int up = max(min(141 - (int)(most >> 23), 120), -100);
        const float factor = __uint_as_float((uint32_t)(127 + up) << 23);
        uint32_t parts[2] = {0u, 0u};
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const uint32_t w[4] = {v[g].x, v[g].y, v[g].z, v[g].w};
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = bf16_low(w[i]) * factor, b = bf16_high(w[i]) * factor, less = i & 1 ? 0.0625f : 1.0f;
                sum += a + b;
                st.q[nq][g][i] = pack_f16(a * less, b * less);
            }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if (c == g) {                                              // in units of the codes', in three parts
                sum *= CODE_UNIT;
                const float hi = __bfloat162float(__float2bfloat16_rn(sum)), mid = __bfloat162float(__float2bfloat16_rn(sum - hi));
                parts[0] = pack_bf16(hi, mid);
                parts[1] = pack_bf16(sum - hi - mid, 0.0f);
            }
        }
        st.q_sum[nq][0] = parts[0];
        st.q_sum[nq][1] = parts[1];
#pragma unroll
        for (int dt = 0; dt < 2 * G; ++dt) st.o[dt][nq][0] = st.o[dt][nq][1] = st.o[dt][nq][2] = st.o[dt][nq][3] = 0.0f;
        st.least[nq][0] = st.least[nq][1] = st.least[nq][2] = st.least[nq][3] = 0.0f;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int col = DUP ? (2 * c + e) & 3 : 8 * nq + 2 * c + e, local = col / group;
            const int back = __shfl_sync(0xffffffffu, up, 4 * (2 * c + e));
            st.scale[nq][e] = scale_log2 * __uint_as_float((uint32_t)(127 + 24 - back) << 23);
            st.m_run[nq][e] = -INFINITY;
            st.l_run[nq][e] = 0.0f;
            st.pos[nq][e] = col < n_rows ? pos0 + local : -1;
            st.first[nq][e] = tt_first_key(pos0 + local, window);
        }
    }

    bool in_time = true;
    int waited = 0;
    for (int i = 0; i < n_mine; ++i) {
        if (in_time && !tc::mbar_wait(tc::smem_u32(&landed[warp][i % STAGES]), (uint32_t)((i / STAGES) & 1))) {
            if (lane == 0) atomicOr(status, TT_STATUS_WAIT_EXPIRED);
            in_time = false;
        }
        in_time = __all_sync(0xffffffffu, in_time);
        waited = i + 1;
        if (!in_time) break;
        if ((valid >> (i & 31)) & 1u) {
            const uint8_t* src = ring + (size_t)(i % STAGES) * R::STAGE;
            const int key_base = (begin + warp + i * WARPS) * TT_BLOCK_TOKENS;
            const bool all_visible = key_base + TT_BLOCK_TOKENS - 1 <= pos0 && key_base >= last_first;
            block_of_keys<D, NQ, DUP>(st, src, src + block_bytes(D), key_base, all_visible, first_key, last_pos, r, c);
        }
        __syncwarp();                                                  // every lane has read the stage
        if (issued < n_mine) issue_next();
    }
    for (int i = waited; i < issued; ++i) tc::mbar_wait(tc::smem_u32(&landed[warp][i % STAGES]), (uint32_t)((i / STAGES) & 1));

    // the lanes' shares of the row sums together; the codes' unit out, the least values in
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float l = st.l_run[nq][e];
            l += __shfl_xor_sync(0xffffffffu, l, 4);
            l += __shfl_xor_sync(0xffffffffu, l, 8);
            l += __shfl_xor_sync(0xffffffffu, l, 16);
            st.l_run[nq][e] = l;
            if constexpr (DUP) st.least[nq][e] += __shfl_xor_sync(0xffffffffu, st.least[nq][e], 2);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const float add = __shfl_sync(0xffffffffu, st.least[nq][e], 4 * g + c);
#pragma unroll
                for (int dt = 2 * g; dt < 2 * g + 2; ++dt) {
                    st.o[dt][nq][e] = fmaf(st.o[dt][nq][e], 1.0f / CODE_UNIT, add);
                    st.o[dt][nq][2 + e] = fmaf(st.o[dt][nq][2 + e], 0.0625f / CODE_UNIT, add);
                }
            }
        }

    // the warps' results meet in shared memory (the stages are free now)
    __syncthreads();
    constexpr int PITCH = R::PITCH;
    float* sh_o = reinterpret_cast<float*>(shared);                    // [WARPS][COLS][PITCH]
    float* sh_m = sh_o + WARPS * COLS * PITCH;                         // [WARPS][COLS]
    float* sh_l = sh_m + WARPS * COLS;
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int col = DUP ? (2 * c + e) & 3 : 8 * nq + 2 * c + e;
            float* dst = sh_o + ((size_t)warp * COLS + col) * PITCH + r;
#pragma unroll
            for (int dt = 0; dt < 2 * G; ++dt)
                if (!DUP || ((dt >> 1) & 1) == (c >> 1)) { dst[16 * dt] = st.o[dt][nq][e]; dst[16 * dt + 8] = st.o[dt][nq][2 + e]; }
            if (r == 0 && (!DUP || c < 2)) {
                sh_m[warp * COLS + col] = st.m_run[nq][e] + (float)(st.e_run - 14);
                sh_l[warp * COLS + col] = st.l_run[nq][e];
            }
        }
    __syncthreads();
    float* cta_acc = sh_l + WARPS * COLS;                              // [COLS][D]
    float* cta_ml = cta_acc + COLS * D;                                // [COLS][2]
    for (int idx = threadIdx.x; idx < n_rows * (D / 2); idx += WARPS * 32) {
        const int row = idx / (D / 2), d = 2 * (idx - row * (D / 2));
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) m = fmaxf(m, sh_m[w * COLS + row]);
        float l = 0.0f, acc0 = 0.0f, acc1 = 0.0f;
        if (m != -INFINITY) {
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float weight = exp2f(sh_m[w * COLS + row] - m);  // 0 for a warp that saw no key
                const float2 o = *reinterpret_cast<const float2*>(sh_o + ((size_t)w * COLS + row) * PITCH + d);
                l = fmaf(sh_l[w * COLS + row], weight, l);
                acc0 = fmaf(o.x, weight, acc0);
                acc1 = fmaf(o.y, weight, acc1);
            }
        }
        const int head = kh * group + row % group;
        const size_t row_index = (size_t)(seq_begin + tok0 + row / group) * heads + head;
        if (sinks && split == 0) {                                     // one more term of the denominator, with no key and no value
            const float ms = __ldg(sinks + head) * 1.4426950408889634f;
            const float m2 = fmaxf(m, ms);
            const float keep = m == -INFINITY ? 0.0f : exp2f(m - m2);
            l = fmaf(l, keep, exp2f(ms - m2));
            acc0 *= keep;
            acc1 *= keep;
            m = m2;
        }
        if (splits == 1) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            *reinterpret_cast<__nv_bfloat162*>(out + row_index * D + d) = __floats2bfloat162_rn(acc0 * inv, acc1 * inv);
        } else if (cluster_merge) {
            *reinterpret_cast<float2*>(cta_acc + row * D + d) = make_float2(acc0, acc1);
            if (d == 0) { cta_ml[2 * row] = m; cta_ml[2 * row + 1] = l; }
        } else {
            const size_t slot = row_index * splits + split;
            *reinterpret_cast<float2*>(part_acc + slot * D + d) = make_float2(acc0, acc1);
            if (d == 0) {
                part_ml[slot * 2] = m * 0.6931471805599453f;           // the merge works with natural exponents
                part_ml[slot * 2 + 1] = l;
            }
        }
    }
    if (splits > 1 && cluster_merge) {                                 // the slices of a tile form a cluster: over distributed shared memory
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        const int rank = (int)cluster.block_rank();
        const int my_rows = rank < n_rows ? (n_rows - rank + splits - 1) / splits : 0;
        for (int idx = threadIdx.x; idx < my_rows * (D / 2); idx += WARPS * 32) {
            const int row = rank + (idx / (D / 2)) * splits, d = 2 * (idx % (D / 2));
            float m = -INFINITY;
            for (int s = 0; s < splits; ++s) m = fmaxf(m, cluster.map_shared_rank(cta_ml, s)[2 * row]);
            float l = 0.0f, acc0 = 0.0f, acc1 = 0.0f;
            if (m != -INFINITY) {
                for (int s = 0; s < splits; ++s) {
                    const float* ml = cluster.map_shared_rank(cta_ml, s);
                    const float weight = exp2f(ml[2 * row] - m);
                    const float2 o = *reinterpret_cast<const float2*>(cluster.map_shared_rank(cta_acc, s) + row * D + d);
                    l = fmaf(ml[2 * row + 1], weight, l);
                    acc0 = fmaf(o.x, weight, acc0);
                    acc1 = fmaf(o.y, weight, acc1);
                }
            }
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            const size_t row_index = (size_t)(seq_begin + tok0 + row / group) * heads + kh * group + row % group;
            *reinterpret_cast<__nv_bfloat162*>(out + row_index * D + d) = __floats2bfloat162_rn(acc0 * inv, acc1 * inv);
        }
        cluster.sync();                                                // no slice leaves while its shared memory is being read
    }
}

template <int D, int NQ, bool DUP>
cudaError_t launch_attention(const void* q, const uint8_t* k_pool, const uint8_t* v_pool, const int* table, int table_width, int pool_blocks,
                             const int* cu, const int* len_before, int sequences, int n_tokens, int heads, int kv_heads, float scale, int window,
                             int splits, int one_token_each, void* out, float* part_acc, float* part_ml, unsigned* status, const float* sinks,
                             cudaStream_t stream) {
    const int group = heads / kv_heads, tokens_per_tile = one_token_each ? 1 : (DUP ? 4 : 8 * NQ) / group;
    const int tiles = one_token_each ? sequences : n_tokens / tokens_per_tile + sequences;
    constexpr int shared = Ring4<D>::shared(8 * NQ);
    auto kernel = attention_4bit_kernel<D, NQ, DUP>;
    const cudaError_t err = tt_allow_shared(kernel, shared);
    if (err != cudaSuccess) return err;
    const bool cluster = splits > 1 && splits <= 8;
    const dim3 grid(tiles, kv_heads, splits), block(Ring4<D>::WARPS * 32);
    const float scale_log2 = scale * 1.4426950408889634f;
    cudaError_t code;
    if (cluster)
        code = tt_launch_pdl_cluster(kernel, grid, block, shared, stream, (unsigned)splits, (const __nv_bfloat16*)q, k_pool, v_pool, table, table_width,
                                     pool_blocks, cu, len_before, sequences, heads, kv_heads, tokens_per_tile, one_token_each, scale_log2, window, splits,
                                     1, (__nv_bfloat16*)out, part_acc, part_ml, status, sinks);
    else
        code = tt_launch_pdl(kernel, grid, block, shared, stream, (const __nv_bfloat16*)q, k_pool, v_pool, table, table_width, pool_blocks, cu,
                             len_before, sequences, heads, kv_heads, tokens_per_tile, one_token_each, scale_log2, window, splits, 0,
                             (__nv_bfloat16*)out, part_acc, part_ml, status, sinks);
    if (code != cudaSuccess) return code;
    if (splits > 8) {
        const long long rows = (long long)n_tokens * heads;
        return tt_launch_pdl(attention_merge_kernel<__nv_bfloat16>, dim3((unsigned)((rows + ATTN_WARPS - 1) / ATTN_WARPS)), dim3(ATTN_WARPS * 32), 0, stream,
                             (const float*)part_acc, (const float*)part_ml, splits, D, rows, (__nv_bfloat16*)out, AttnExtra{}, heads);
    }
    return cudaGetLastError();
}

bool takes(int heads, int kv_heads, int head_dim) {
    return kv_heads > 0 && kv_heads <= 65535 && heads % kv_heads == 0 && heads / kv_heads >= 1 && heads / kv_heads <= 16 &&
           (head_dim == 32 || head_dim == 64 || head_dim == 96 || head_dim == 128);
}

}  // namespace

extern "C" int tt_rope_append_4bit(const float* qkv, int splits, long long split_stride, const float* inv_freq, int rotary_dim, int interleaved,
                                   float attention_scaling, void* q_out, void* k_pool, void* v_pool, const int* table, int table_width,
                                   int pool_blocks, const int* cu, const int* len_before, int sequences, int n_tokens, int heads, int kv_heads,
                                   int head_dim, int write_cache, unsigned* status, cudaStream_t stream) {
    if (n_tokens <= 0) return 0;
    if (!takes(heads, kv_heads, head_dim) || rotary_dim < 0 || rotary_dim > head_dim || (rotary_dim & 1) || splits < 1 || sequences < 1 ||
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
    if (!takes(kv_heads, kv_heads, head_dim) || span < 1 || sequences > 65535 || (((uintptr_t)keys | (uintptr_t)values) & 15) != 0) return (int)cudaErrorInvalidValue;
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

// one_token_each: n_tokens == sequences and every sequence brings one.  splits > 1 cuts the keys into slices: up to 8 are combined by a
// thread-block cluster, more leave partial results in part_acc / part_ml for a second kernel.
extern "C" int tt_attention_4bit(const void* q, const void* k_pool, const void* v_pool, const int* table, int table_width, int pool_blocks,
                                 const int* cu, const int* len_before, int sequences, int n_tokens, int heads, int kv_heads, int head_dim,
                                 float scale, int window, int splits, int one_token_each, int wide, void* out, float* part_acc, float* part_ml,
                                 unsigned* status, const float* sinks, cudaStream_t stream) {
    if (n_tokens <= 0 || sequences <= 0) return 0;
    if (!takes(heads, kv_heads, head_dim) || splits < 1 || splits > 65535 || !(scale > 0.0f) || (((uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)q) & 15) != 0 ||
        (splits > 8 && (!part_acc || !part_ml)))
        return (int)cudaErrorInvalidValue;
    const int group = heads / kv_heads;
#define TT_LAUNCH(D, NQ, DUP)                                                                                                                    \
    return (int)launch_attention<D, NQ, DUP>(q, (const uint8_t*)k_pool, (const uint8_t*)v_pool, table, table_width, pool_blocks, cu, len_before, sequences, \
                                             n_tokens, heads, kv_heads, scale, window, splits, one_token_each, out, part_acc, part_ml, status, sinks, stream)
#define TT_LAUNCH_D(D)                              \
    if (group > 8 || wide) TT_LAUNCH(D, 2, false); \
    if (group > 4) TT_LAUNCH(D, 1, false);         \
    TT_LAUNCH(D, 1, true)
    switch (head_dim) {
        case 32: TT_LAUNCH_D(32);
        case 64: TT_LAUNCH_D(64);
        case 96: TT_LAUNCH_D(96);
        default: TT_LAUNCH_D(128);
    }
#undef TT_LAUNCH_D
#undef TT_LAUNCH
}
