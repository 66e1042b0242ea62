// Causal grouped-query attention over a block cache held in 4 bits (see cache_4bit.cuh): bfloat16 queries, head sizes 32, 64, 96 and 128, up to 16
// query heads per key/value head; decoding, and any number of tokens a sequence.
//
// With codes n, scales s and least values m of key t and value t (primes for values), per group g:
//   score(q, t) = sum_g s_tg (q . n)_tg + m_tg (sum of q over g),     out_g = sum_t (p_t s'_tg) n'_t + p_t m'_tg.
// So the tensor cores multiply codes, not numbers.  As float16 the bits 0x000n are n 2^-24 and 0x00n0 are 16 n 2^-24 (numbers below the
// normal ones, which the tensor cores take as they are): an operand register of two codes is one mask away from the cache's word, and
// eight codes take one shift and four masks.  What the sixteens multiply is a sixteenth (queries) or is taken off the sums' rows
// (values), the 2^24 goes into the scale.  Group scales meet the 16 x 8 tile of a group's products (S^T: 16 keys, 8 queries) and the
// probabilities; the least values are one more product of each, in bfloat16.  (Codes as e4m3 bytes take three instructions instead of
// five, but this architecture's mma.sync takes them apart again: 72 -> 97 us at 64 sequences of up to 4,096 tokens.)
//
// Queries are float16 after a power of two that brings a row's greatest number to 2^14: exact but for what lies 2^-28 below that.
// The weights p s' are rounded to float16 (11 bits): with weights in bfloat16 the two terms of out, which are of opposite sign and
// each several times their sum, were off by 0.4 % of it.  So that float16 holds them whatever the values' size, the running maximum is
// one of score + E - 14 in log2 units, E the exponent of the largest of the key's value scales and least values (at least -40), and p is relative to it:
// a row's weights stay below 2^15, and what falls under 2^-14, float16's last full number, is less than 2^-28 of the row's largest p times scale or least
// value.  A row's unit so depends on what it sees, and by how much it weighs it, alone (with the largest scale that the warp had met as the unit, a value
// of 2^34 that later tokens alone see, or of little weight, left the others no bits).  The second term takes p in two bfloat16 parts (16 bits)
// and m' as it is, the second term of S the queries' sums in three.  All sums are float32.
//
// Rows of up to four queries (DUP) stand twice in the tile's eight columns, which would otherwise be half empty: the weights of one
// group of numbers lie in the first four, those of the next group in the others, and the products of either group take the same
// operand.
//
// A warp owns up to 8 NQ query rows of one sequence and key/value head, (token, head of the group) pairs, and walks its share of the
// blocks; the copy engine brings a block's keys and values (5 KB each at D = 128) into its two places in shared memory.
#include "cache_4bit.cuh"
#include "tcgen05.cuh"

#include <cooperative_groups.h>
#include <cuda_fp16.h>
namespace cg = cooperative_groups;

namespace {

using cache4::block_bytes;
using cache4::code_bytes;

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
// the first product of a sum
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma_bf16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// two float32 numbers at a time
__device__ __forceinline__ void fma_two_up(float& a, float& b, float x0, float x1, float y0, float y1, float z) {
    asm("{\n\t.reg .b64 x, y, z, d;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %6};\n\t"
        "fma.rp.f32x2 d, x, y, z;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(a), "=f"(b) : "f"(x0), "f"(x1), "f"(y0), "f"(y1), "f"(z));
}
__device__ __forceinline__ void fma_two(float& a, float& b, float x0, float x1, float y0, float y1, float z0, float z1) {
    asm("{\n\t.reg .b64 x, y, z, d;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 d, x, y, z;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(a), "=f"(b) : "f"(x0), "f"(x1), "f"(y0), "f"(y1), "f"(z0), "f"(z1));
}
__device__ __forceinline__ void add_two(float& a, float& b, float x0, float x1) {
    asm("{\n\t.reg .b64 x, d;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 d, {%0, %1};\n\tadd.rn.f32x2 d, d, x;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "+f"(a), "+f"(b) : "f"(x0), "f"(x1));
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
    float m_run[NQ][2], l_run[NQ][2];   // the maximum of score + E - 14, to whose power of two all weights and sums are relative; l: this lane's share (its keys) until the end
    int pos[NQ][2], first[NQ][2];       // queries 8 nq + 2 c + e see keys first .. pos
};

// The scores of a block's 64 keys (before their scale): s[kt][nq] is a tile of 16 keys and 8 queries, rows r and r + 8 its tokens
// token0 and token0 + 2.
__device__ __forceinline__ int token_of_row(int r) { return 4 * (r >> 1) + (r & 1); }

template <int D, int NQ, bool DUP>
__device__ __forceinline__ void scores_of_block(const Rows4<D, NQ, DUP>& st, const uint8_t* __restrict__ kb, float (&s)[4][NQ][4], int r, int c) {
    constexpr int G = Rows4<D, NQ, DUP>::G;
    const int token0 = token_of_row(r);
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
            mma_bf16_first(s[kt][nq], m0, m1, m0, m1, st.q_sum[nq][0], st.q_sum[nq][1]);
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const uint32_t h0 = w0[g] >> 8, h1 = w1[g] >> 8;
            const float s0 = bf16_low(p0[g]), s1 = bf16_low(p1[g]);
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq) {
                float acc[4];
                mma_f16_first(acc, w0[g] & ONES_MASK, w1[g] & ONES_MASK, w0[g] & SIXTEENS_MASK, w1[g] & SIXTEENS_MASK, st.q[nq][g][0], st.q[nq][g][1]);
                mma_f16(acc, h0 & ONES_MASK, h1 & ONES_MASK, h0 & SIXTEENS_MASK, h1 & SIXTEENS_MASK, st.q[nq][g][2], st.q[nq][g][3]);
                s[kt][nq][0] = fmaf(s0, acc[0], s[kt][nq][0]);
                s[kt][nq][1] = fmaf(s0, acc[1], s[kt][nq][1]);
                s[kt][nq][2] = fmaf(s1, acc[2], s[kt][nq][2]);
                s[kt][nq][3] = fmaf(s1, acc[3], s[kt][nq][3]);
            }
        }
    }
}

// E - 14 of two neighbouring tokens as a pair of bfloat16 numbers: E the exponent of a token's largest scale or least value, at least -40 (a scale that is
// not a number counts for nothing here).
template <int G>
__device__ __forceinline__ uint32_t exponents_of(const uint8_t* __restrict__ two_tokens, const uint8_t* __restrict__ two_mins) {
    uint32_t w[G];                                                     // G scales of the first token, then those of the second
    load_words<G>(two_tokens, w);
    auto larger = [](uint32_t a, uint32_t b) {
        const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&m);
    };
    uint32_t most;                                                     // the first token's largest scale in the low half, the second's in the high one
    if constexpr (G == 1) most = w[0];
    else if constexpr (G == 2) most = larger(__byte_perm(w[0], w[1], 0x5410), __byte_perm(w[0], w[1], 0x7632));
    else if constexpr (G == 3) most = larger(larger(__byte_perm(w[0], w[1], 0x7610), __byte_perm(w[0], w[2], 0x5432)), __byte_perm(w[1], w[2], 0x7610));
    else {
        const uint32_t a = larger(w[0], w[1]), b = larger(w[2], w[3]);
        most = larger(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
    }
#pragma unroll
    for (int g = 0; g < G; ++g) most = larger(most, *reinterpret_cast<const uint32_t*>(two_mins + g * 2 * TT_BLOCK_TOKENS) & 0x7fff7fffu);
    const uint32_t lo = most & 0xffffu, hi = most >> 16;
    const int first = lo <= 0x7f80u ? (int)(lo >> 7) - 127 : -127, second = hi <= 0x7f80u ? (int)(hi >> 7) - 127 : -127;
    return pack_bf16((float)(max(first, -40) - 14), (float)(max(second, -40) - 14));       // whole numbers below 256: exact
}

// Their running softmax and what its weights make of the block's values.  MASKED: some query does not see some key of the block.
template <int D, int NQ, bool DUP, bool MASKED>
__device__ __forceinline__ void values_of_block(Rows4<D, NQ, DUP>& st, const uint8_t* __restrict__ vb, float (&s)[4][NQ][4], int key_base,
                                                int last_pos, int r, int c) {
    constexpr int G = Rows4<D, NQ, DUP>::G;
    const int lane = 4 * r + c, token0 = token_of_row(r);
    const uint8_t* scales = vb + code_bytes(D);
    const uint8_t* mins = scales + 2 * TT_BLOCK_TOKENS * G;
    if constexpr (MASKED) {
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
    const uint32_t exponents = exponents_of<G>(scales + 2 * lane * 2 * G, mins + 2 * lane * 2);        // of tokens 2 lane and 2 lane + 1
    float most[NQ][2];
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) most[nq][0] = most[nq][1] = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int hi = 0; hi < 2; ++hi) {
            const uint32_t two = __shfl_sync(0xffffffffu, exponents, 8 * kt + 2 * (r >> 1) + hi);
            const float unit = __uint_as_float(r & 1 ? two & 0xffff0000u : two << 16);
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq) {                          // the scale is positive; rounded up, so that no weight leaves float16's reach
                float x, y;
                fma_two_up(x, y, s[kt][nq][2 * hi], s[kt][nq][2 * hi + 1], st.scale[nq][0], st.scale[nq][1], unit);
                most[nq][0] = fmaxf(most[nq][0], x);
                most[nq][1] = fmaxf(most[nq][1], y);
            }
        }
    float corr[NQ][2];
    bool grew = false;
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
        float base[2], sum[2] = {0.0f, 0.0f}, m_new[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float mx = most[nq][e];
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            m_new[e] = fmaxf(st.m_run[nq][e], mx);
            corr[nq][e] = m_new[e] == -INFINITY ? 1.0f : fast_exp2(st.m_run[nq][e] - m_new[e]);
            grew = grew || corr[nq][e] != 1.0f;
            base[e] = m_new[e] == -INFINITY ? 0.0f : -m_new[e];
        }
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int hi = 0; hi < 4; hi += 2) {
                float& x = s[kt][nq][hi];
                float& y = s[kt][nq][hi + 1];
                fma_two(x, y, x, y, st.scale[nq][0], st.scale[nq][1], base[0], base[1]);
                if constexpr (MASKED) {                                // a masked key weighs minus zero: told from a weight too small for float32
                    x = x == -INFINITY ? -0.0f : fast_exp2(x);
                    y = y == -INFINITY ? -0.0f : fast_exp2(y);
                } else {
                    x = fast_exp2(x);
                    y = fast_exp2(y);
                }
                add_two(sum[0], sum[1], x, y);
            }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            // (the factor in two parts: keys whose values are zero may have gathered far more than float32's reach beside large values)
            const float part = fast_exp2(0.5f * (st.m_run[nq][e] - m_new[e]));
            st.l_run[nq][e] = m_new[e] == -INFINITY ? sum[e] : st.l_run[nq][e] * part * part + sum[e];
            // a key that is not a number has no part in the maximum; what this warp saw must count all the same where others' results join it
            st.m_run[nq][e] = (m_new[e] == -INFINITY && sum[e] != sum[e]) ? 0.0f : m_new[e];
        }
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
    auto masked = [](float p) { return __float_as_uint(p) == 0x80000000u; };
    constexpr int SETS = DUP ? (G + 1) / 2 : G;                        // operands of weights: with DUP one holds two groups'
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
        const int t0 = 16 * kt + token0;
        // least values: row g of the operand is group g, its columns are this lane's four tokens
        uint2 low = make_uint2(0u, 0u);
        if (r < G) low = *reinterpret_cast<const uint2*>(mins + (r * TT_BLOCK_TOKENS + 16 * kt + 4 * c) * 2);
        if constexpr (MASKED) {                                        // what lies behind the sequence's end may be anything
            const int key = key_base + 16 * kt + 4 * c;
            if (key > last_pos) low.x &= 0xffff0000u;
            if (key + 1 > last_pos) low.x &= 0x0000ffffu;
            if (key + 2 > last_pos) low.y &= 0xffff0000u;
            if (key + 3 > last_pos) low.y &= 0x0000ffffu;
        }
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
            uint32_t front[4];                                         // the first 16 bits' number
#pragma unroll
            for (int i = 0; i < 4; ++i) front[i] = __float_as_uint(s[kt][nq][i]) & 0xffff0000u;
            float part[4];
            if constexpr (DUP) {                                       // the first part in the first four columns, the second in the others
                const float whole = c < 2 ? 0.0f : 1.0f, less = c < 2 ? 1.0f : -1.0f;
#pragma unroll
                for (int i = 0; i < 4; i += 2)
                    fma_two(part[i], part[i + 1], __uint_as_float(front[i]), __uint_as_float(front[i + 1]), less, less, s[kt][nq][i] * whole, s[kt][nq][i + 1] * whole);
                mma_bf16(st.least[nq], low.x, 0u, low.y, 0u, transpose_8x8(pack_bf16(part[0], part[1])), transpose_8x8(pack_bf16(part[2], part[3])));
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) part[i] = s[kt][nq][i] - __uint_as_float(front[i]);
                mma_bf16(st.least[nq], low.x, 0u, low.y, 0u, transpose_8x8(__byte_perm(front[0], front[1], 0x7632)), transpose_8x8(__byte_perm(front[2], front[3], 0x7632)));
                mma_bf16(st.least[nq], low.x, 0u, low.y, 0u, transpose_8x8(pack_bf16(part[0], part[1])), transpose_8x8(pack_bf16(part[2], part[3])));
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
                if constexpr (MASKED) {                                // a masked value adds nothing, whatever its scale
                    p0 = masked(s[kt][nq][0]) ? 0.0f : p0; p1 = masked(s[kt][nq][1]) ? 0.0f : p1;
                    p2 = masked(s[kt][nq][2]) ? 0.0f : p2; p3 = masked(s[kt][nq][3]) ? 0.0f : p3;
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

// Sixteen warps an SM (eight with two column tiles), as many as registers hold at D = 128: a block is about 1,200 instructions of a warp, whose
// chains of loads, products and exponentials take it 3,200 cycles alone, so four warps keep a scheduler busy.  Each warp has one
// place for a block of keys and one for a block of values, asked for again as soon as it has read them: the keys arrive under the block's
// softmax and second product, the values under the next block's first.  (Two places each leave room for eight warps: 65 -> 77 us at
// 64 sequences of up to 4,096 tokens.)  Few CTAs have eight warps, so that a slice is done sooner, many have four.
template <int D, int NQ, int WARPS_> struct Ring4 {
    static constexpr int WARPS = WARPS_, CTAS = (NQ == 1 ? 16 : 8) / WARPS_;
    static constexpr int WARP_BYTES = 2 * block_bytes(D);
    static constexpr int PITCH = D + 4, COLS = 8 * NQ;
    static constexpr int RING = WARPS * WARP_BYTES;
    static constexpr int RESULTS = WARPS * COLS * (PITCH + 2) * 4 + COLS * (D + 2) * 4;        // where the warps' results meet
    static constexpr int SHARED = RING > RESULTS ? RING : RESULTS;
};

// How the work is cut.  A tile is a sequence's key/value head with up to 8 NQ query rows of neighbouring tokens.
// Slices: grid = (tiles, kv_heads, splits); a tile's blocks in equal slices, up to 8 of which a cluster joins over distributed shared
// memory, one launch: few tiles, where latency counts.
// Even runs (splits 0): the blocks of all tiles, tile after tile, in equal runs, one for each of the grid's CTAs, which all fit the
// device at once.  Sequences differ in length and tiles do not come in multiples of the SMs (64 sequences x 8 heads left 27 % of the
// SMs' time idle), runs are alike.  A run that begins or ends inside a tile leaves that part of the sums in scratch memory and draws a
// ticket; the CTA that draws a tile's last one joins its parts in their order (no CTA waits for another).
struct Runs {
    int total;                           // blocks of all tiles (the caller bounds them to 2^30)
    int per;                             // of a run: whole rounds of the CTA's warps
};
struct Sequence4 {
    int new_tokens, before, block0, blocks, tiles;     // tiles of all key/value heads, each over the same blocks
};

__device__ __forceinline__ Sequence4 sequence_of(int b, int sequences, const int* __restrict__ cu, const int* __restrict__ len_before, int window,
                                                 int tokens_per_tile, int kv_heads) {
    Sequence4 s = {0, 0, 0, 0, 0};
    if (b < sequences) {
        s.new_tokens = cu[b + 1] - cu[b];
        s.before = len_before[b];
        if (s.new_tokens > 0) {
            s.block0 = tt_first_key(s.before, window) / TT_BLOCK_TOKENS;
            s.blocks = (s.before + s.new_tokens - 1) / TT_BLOCK_TOKENS - s.block0 + 1;
            s.tiles = (s.new_tokens + tokens_per_tile - 1) / tokens_per_tile * kv_heads;
        }
    }
    return s;
}
__device__ __forceinline__ int warp_scan(int v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += up;
    }
    return v;
}
// What the blocks of all tiles come to, and where the run that starts at `cta` of `ctas` equal ones begins: its sequence (-1: behind the last) and
// the block within that.  Up to 128 sequences are looked at once, more a second time.
struct RunStart {
    Runs runs;
    int b, x;
    Sequence4 seq;
};
__device__ __forceinline__ RunStart start_of_run(int sequences, const int* __restrict__ cu, const int* __restrict__ len_before, int window, int tokens_per_tile,
                                                 int kv_heads, int cta, int ctas, int round) {
    constexpr int HELD = 4;
    const int lane = threadIdx.x & 31;
    Sequence4 held[HELD];
    int mine = 0;
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        held[i] = sequence_of(32 * i + lane, sequences, cu, len_before, window, tokens_per_tile, kv_heads);
        mine += held[i].blocks * held[i].tiles;
    }
    for (int b = 32 * HELD + lane; b < sequences; b += 32) {
        const Sequence4 s = sequence_of(b, sequences, cu, len_before, window, tokens_per_tile, kv_heads);
        mine += s.blocks * s.tiles;
    }
    RunStart start;
    start.runs.total = __reduce_add_sync(0xffffffffu, mine);
    start.runs.per = max((start.runs.total + ctas - 1) / ctas, 1);
    start.runs.per = (start.runs.per + round - 1) / round * round;
    start.x = (int)min((long long)start.runs.per * cta, (long long)start.runs.total);
    start.b = -1;
    auto look = [&](const Sequence4& s, int base) {
        const int blocks = s.blocks * s.tiles, upto = warp_scan(blocks, lane);
        const unsigned owner = __ballot_sync(0xffffffffu, start.x < upto);
        if (owner) {
            const int at = __ffs(owner) - 1;
            start.x -= __shfl_sync(0xffffffffu, upto - blocks, at);
            start.b = base + at;
            start.seq.new_tokens = __shfl_sync(0xffffffffu, s.new_tokens, at);
            start.seq.before = __shfl_sync(0xffffffffu, s.before, at);
            start.seq.block0 = __shfl_sync(0xffffffffu, s.block0, at);
            start.seq.blocks = __shfl_sync(0xffffffffu, s.blocks, at);
            start.seq.tiles = __shfl_sync(0xffffffffu, s.tiles, at);
        } else {
            start.x -= __shfl_sync(0xffffffffu, upto, 31);
        }
    };
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (start.b < 0 && 32 * i < sequences) look(held[i], 32 * i);
    for (int base = 32 * HELD; base < sequences && start.b < 0; base += 32)
        look(sequence_of(base + lane, sequences, cu, len_before, window, tokens_per_tile, kv_heads), base);
    return start;
}

template <int D, int NQ, bool DUP, int WARPS, bool EVEN>
__global__ void __launch_bounds__(WARPS * 32, Ring4<D, NQ, WARPS>::CTAS)
attention_4bit_kernel(const __nv_bfloat16* __restrict__ q, const uint8_t* __restrict__ k_pool, const uint8_t* __restrict__ v_pool,
                      const int* __restrict__ table, int table_width, int pool_blocks, const int* __restrict__ cu,
                      const int* __restrict__ len_before, int sequences, int heads, int kv_heads, int tokens_per_tile,
                      float scale_log2, int window, int splits, __nv_bfloat16* __restrict__ out,
                      float* __restrict__ part_acc, float* __restrict__ part_ml, unsigned* __restrict__ tickets, unsigned* status,
                      const float* __restrict__ sinks) {
    using R = Ring4<D, NQ, WARPS>;
    constexpr int G = D / 32, COLS = R::COLS, BYTES = block_bytes(D);
    extern __shared__ __align__(128) uint8_t shared[];
    __shared__ uint64_t keys_landed[WARPS], values_landed[WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const int group = heads / kv_heads;
    if (lane == 0) {
        tc::mbar_init(tc::smem_u32(&keys_landed[warp]), 1);
        tc::mbar_init(tc::smem_u32(&values_landed[warp]), 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncwarp();
    tt_pdl_launch_dependents();
    tt_pdl_wait();

    int b, tile;                         // tile: of the sequence's, with slices among one head's, with even runs among all heads'
    int left = 0;                        // blocks of the run that are still to do
    int block_in_tile = 0, per_run = 1, at_block = 0;                  // at_block: this run's place among the blocks of all tiles
    Sequence4 seq;
    if constexpr (EVEN) {
        const RunStart start = start_of_run(sequences, cu, len_before, window, tokens_per_tile, kv_heads, blockIdx.x, gridDim.x, WARPS);
        if (start.b < 0) return;
        per_run = start.runs.per;
        at_block = per_run * blockIdx.x;
        left = min(per_run, start.runs.total - at_block);
        b = start.b;
        seq = start.seq;
        tile = start.x / seq.blocks;
        block_in_tile = start.x % seq.blocks;
    } else if (tokens_per_tile == 1 && sequences == (int)gridDim.x) {  // one token a sequence
        b = blockIdx.x;
        tile = 0;
    } else {
        tile = blockIdx.x;
        b = -1;
        for (int base = 0; base < sequences && b < 0; base += 32) {
            const int mine = base + lane;
            const int count = mine < sequences ? (cu[mine + 1] - cu[mine] + tokens_per_tile - 1) / tokens_per_tile : 0;
            const int upto = warp_scan(count, lane);
            const unsigned owner = __ballot_sync(0xffffffffu, tile < upto);
            if (owner) {
                const int at = __ffs(owner) - 1;
                b = base + at;
                tile -= __shfl_sync(0xffffffffu, upto - count, at);
            } else {
                tile -= __shfl_sync(0xffffffffu, upto, 31);
            }
        }
        if (b < 0) return;               // a spare CTA (the grid is an upper bound): all of its warps, and of its cluster, leave together
    }

    uint8_t* key_ring = shared + (size_t)warp * R::WARP_BYTES;
    uint8_t* value_ring = key_ring + BYTES;
    unsigned done = 0;                   // blocks that this warp has fetched in earlier tiles: the barriers' phases go on
    bool in_time = true;
    // One tile, or the part of it that falls to this CTA; with even runs one after another.
    for (;;) {
    if constexpr (!EVEN) seq = sequence_of(b, sequences, cu, len_before, window, tokens_per_tile, kv_heads);
    const int seq_begin = cu[b], heads_tiles = EVEN ? seq.tiles / kv_heads : 1;
    const int kh = EVEN ? tile / heads_tiles : blockIdx.y, tok0 = (EVEN ? tile % heads_tiles : tile) * tokens_per_tile;
    const int tokens = min(tokens_per_tile, seq.new_tokens - tok0);
    if (tokens <= 0) return;             // a sequence without a token: the same for the whole cluster
    const int pos0 = seq.before + tok0, last_pos = pos0 + tokens - 1;
    const int n_rows = tokens * group;
    const int first_key = tt_first_key(pos0, window), last_first = tt_first_key(last_pos, window);
    int begin, end, part = -1;           // part: where in scratch memory the result goes (-1: it is the tile's whole)
    bool has_sink = true;
    if constexpr (EVEN) {
        const int take = min(left, seq.blocks - block_in_tile);
        begin = seq.block0 + block_in_tile;
        end = begin + take;
        if (take < seq.blocks) part = 2 * blockIdx.x + (block_in_tile > 0 ? 0 : 1);
        has_sink = block_in_tile == 0;
        left -= take;
    } else {
        const int block0 = first_key / TT_BLOCK_TOKENS, n_blocks = last_pos / TT_BLOCK_TOKENS - block0 + 1;
        const int per = (n_blocks + splits - 1) / splits;
        begin = block0 + (int)blockIdx.z * per;
        end = min(begin + per, block0 + n_blocks);
        has_sink = blockIdx.z == 0;
    }
    const int n_mine = begin + warp < end ? (end - begin - warp + WARPS - 1) / WARPS : 0;
    const int* table_row = table + (size_t)b * table_width;

    uint4 v[NQ][G];                      // the queries, asked for first
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
        const int row = DUP ? r & 3 : 8 * nq + r;
        const __nv_bfloat16* src = q + ((size_t)(seq_begin + tok0 + row / group) * heads + kh * group + row % group) * D + 8 * c;
#pragma unroll
        for (int g = 0; g < G; ++g) v[nq][g] = row < n_rows ? *reinterpret_cast<const uint4*>(src + 32 * g) : make_uint4(0u, 0u, 0u, 0u);
    }
    // Blocks of this warp, a lane each: lane i % 32 holds block i's place in the pool, for the 16 blocks at hand and the 16 behind them; -1
    // where the table entry lies outside the pool (nothing is copied then).
    auto look_up = [&](int i) {
        const int kb = begin + warp + i * WARPS;
        const int block = kb < end && kb < table_width ? __ldg(table_row + kb) : -1;
        return block < pool_blocks ? block : -1;
    };
    int ids = look_up(lane);
    auto block_at = [&](int i) { return __shfl_sync(0xffffffffu, ids, i & 31); };
    // lane 0 alone copies
    auto fetch = [&](const uint8_t* pool, uint8_t* dst, uint64_t* landed, int i) {
        const int block = block_at(i);
        if (lane == 0) {
            const uint32_t bar = tc::smem_u32(landed);
            if (block >= 0) {
                tc::mbar_expect_tx(bar, BYTES);
                bulk_copy(dst, pool + ((size_t)block * kv_heads + kh) * BYTES, BYTES, bar);
            } else {
                tc::mbar_arrive(bar);
                atomicOr(status, TT_STATUS_BAD_BLOCK);
            }
        }
    };
    if (in_time && n_mine > 0) {
        fetch(k_pool, key_ring, &keys_landed[warp], 0);
        fetch(v_pool, value_ring, &values_landed[warp], 0);
    }

    Rows4<D, NQ, DUP> st;
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
        uint32_t most = 0u;                                            // bits of the row's greatest number without its sign
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const uint32_t w[4] = {v[nq][g].x, v[nq][g].y, v[nq][g].z, v[nq][g].w};
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
            const uint32_t w[4] = {v[nq][g].x, v[nq][g].y, v[nq][g].z, v[nq][g].w};
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x0 = bf16_low(w[i]) * factor, x1 = bf16_high(w[i]) * factor, less = i & 1 ? 0.0625f : 1.0f;
                sum += x0 + x1;
                st.q[nq][g][i] = pack_f16(x0 * less, x1 * less);
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

    // A wait that runs out: nothing more is fetched, and what is on its way is waited for once more before shared memory is used again.
    auto landed_in_time = [&](uint64_t* landed, int i) {
        const bool there = tc::mbar_wait(tc::smem_u32(landed), (done + i) & 1);
        if (!there && lane == 0) atomicOr(status, TT_STATUS_WAIT_EXPIRED);
        return (bool)__all_sync(0xffffffffu, there);
    };
    for (int i = 0; i < n_mine && in_time; ++i) {
        const bool usable = block_at(i) >= 0;
        if (i > 0 && (i & 15) == 0 && (lane >> 4) == ((i >> 4) - 1 & 1)) ids = look_up(i + 16 + (lane & 15));
        float s[4][NQ][4];
        if (!landed_in_time(&keys_landed[warp], i)) {
            tc::mbar_wait(tc::smem_u32(&keys_landed[warp]), (done + i) & 1);
            tc::mbar_wait(tc::smem_u32(&values_landed[warp]), (done + i) & 1);
            in_time = false;
            break;
        }
        if (usable) scores_of_block<D, NQ, DUP>(st, key_ring, s, r, c);
        __syncwarp();                                                  // every lane has read the keys
        if (i + 1 < n_mine) fetch(k_pool, key_ring, &keys_landed[warp], i + 1);
        if (!landed_in_time(&values_landed[warp], i)) {
            tc::mbar_wait(tc::smem_u32(&values_landed[warp]), (done + i) & 1);
            if (i + 1 < n_mine) tc::mbar_wait(tc::smem_u32(&keys_landed[warp]), (done + i + 1) & 1);
            in_time = false;
            break;
        }
        if (usable) {
            const int key_base = (begin + warp + i * WARPS) * TT_BLOCK_TOKENS;
            const bool all_visible = key_base + TT_BLOCK_TOKENS - 1 <= pos0 && key_base >= last_first;
            if (all_visible) values_of_block<D, NQ, DUP, false>(st, value_ring, s, key_base, last_pos, r, c);
            else values_of_block<D, NQ, DUP, true>(st, value_ring, s, key_base, last_pos, r, c);
        }
        __syncwarp();
        if (i + 1 < n_mine) fetch(v_pool, value_ring, &values_landed[warp], i + 1);
    }
    done += n_mine;

    // the lanes' shares of the row sums together; the codes' unit out, the least values in; and relative to a power of two at which the weights' sum is 1/2 to 1:
    // what joins then compares by weight alone, not by the values' size as well
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float l = st.l_run[nq][e];
            l += __shfl_xor_sync(0xffffffffu, l, 4);
            l += __shfl_xor_sync(0xffffffffu, l, 8);
            l += __shfl_xor_sync(0xffffffffu, l, 16);
            const int up = l > 0.0f && l < INFINITY ? min((int)(__float_as_uint(l) >> 23) - 126, 120) : 0;
            const float down = __uint_as_float((uint32_t)(127 - up) << 23);
            st.l_run[nq][e] = l * down;
            st.m_run[nq][e] += (float)up;
            if constexpr (DUP) st.least[nq][e] += __shfl_xor_sync(0xffffffffu, st.least[nq][e], 2);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const float add = __shfl_sync(0xffffffffu, st.least[nq][e], 4 * g + c);
#pragma unroll
                for (int dt = 2 * g; dt < 2 * g + 2; ++dt) {
                    st.o[dt][nq][e] = fmaf(st.o[dt][nq][e], 1.0f / CODE_UNIT, add) * down;
                    st.o[dt][nq][2 + e] = fmaf(st.o[dt][nq][2 + e], 0.0625f / CODE_UNIT, add) * down;
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
                sh_m[warp * COLS + col] = st.m_run[nq][e];
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
        if (sinks && has_sink) {                                       // one more term of the denominator, with no key and no value
            const float ms = __ldg(sinks + head) * 1.4426950408889634f;
            const float m2 = fmaxf(m, ms);
            const float keep = m == -INFINITY ? 0.0f : exp2f(m - m2);
            l = fmaf(l, keep, ms == -INFINITY ? 0.0f : exp2f(ms - m2));      // (a slice in which the row sees no key has m = -inf, too)
            acc0 *= keep;
            acc1 *= keep;
            m = m2;
        }
        if (EVEN ? part < 0 : splits == 1) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            *reinterpret_cast<__nv_bfloat162*>(out + row_index * D + d) = __floats2bfloat162_rn(acc0 * inv, acc1 * inv);
        } else if constexpr (EVEN) {
            const size_t slot = (size_t)part * tokens_per_tile * group + row;
            *reinterpret_cast<float2*>(part_acc + slot * D + d) = make_float2(acc0, acc1);
            if (d == 0) *reinterpret_cast<float2*>(part_ml + 2 * slot) = make_float2(m, l);
        } else {
            *reinterpret_cast<float2*>(cta_acc + row * D + d) = make_float2(acc0, acc1);
            if (d == 0) { cta_ml[2 * row] = m; cta_ml[2 * row + 1] = l; }
        }
    }
    if constexpr (EVEN) {
        if (part >= 0) {                                               // the last of a tile's parts to get here joins them
            const int tile_at = at_block - block_in_tile, p0 = tile_at / per_run, p1 = (tile_at + seq.blocks - 1) / per_run;
            __threadfence();                                           // the part is there before its ticket
            __syncthreads();
            __shared__ unsigned drawn;
            if (threadIdx.x == 0) {
                drawn = atomicAdd(tickets + p0, 1u);                   // a tile that is cut begins in a run of its own
                if (drawn == (unsigned)(p1 - p0)) tickets[p0] = 0u;    // as it was found
            }
            __syncthreads();
            if (drawn == (unsigned)(p1 - p0)) {
                __threadfence();
                const int rows = tokens_per_tile * group;
                for (int idx = threadIdx.x; idx < n_rows * (D / 2); idx += WARPS * 32) {
                    const int row = idx / (D / 2), d = 2 * (idx - row * (D / 2));
                    float m = -INFINITY, l = 0.0f, acc0 = 0.0f, acc1 = 0.0f;
                    // eight parts' numbers asked for together; the sums go on relative to the largest maximum so far
                    for (int p = p0; p <= p1; p += 8) {
                        float2 ml[8], o[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const size_t slot = (size_t)(2 * (p + i) + (p + i == p0)) * rows + row;
                            ml[i] = p + i <= p1 ? __ldcg(reinterpret_cast<const float2*>(part_ml + 2 * slot)) : make_float2(-INFINITY, 0.0f);
                            o[i] = p + i <= p1 ? __ldcg(reinterpret_cast<const float2*>(part_acc + slot * D + d)) : make_float2(0.0f, 0.0f);
                        }
                        float most = m;
#pragma unroll
                        for (int i = 0; i < 8; ++i) most = fmaxf(most, ml[i].x);
                        if (most == -INFINITY) continue;
                        const float keep = exp2f(m - most);
                        l *= keep; acc0 *= keep; acc1 *= keep;
                        m = most;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float weight = exp2f(ml[i].x - m);   // 0 for a part that saw no key
                            l = fmaf(ml[i].y, weight, l);
                            acc0 = fmaf(o[i].x, weight, acc0);
                            acc1 = fmaf(o[i].y, weight, acc1);
                        }
                    }
                    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                    const size_t row_index = (size_t)(seq_begin + tok0 + row / group) * heads + kh * group + row % group;
                    *reinterpret_cast<__nv_bfloat162*>(out + row_index * D + d) = __floats2bfloat162_rn(acc0 * inv, acc1 * inv);
                }
            }
        }
        if (left <= 0) return;
        at_block += end - begin;
        block_in_tile = 0;
        if (++tile == seq.tiles) {
            tile = 0;
            do ++b; while (cu[b + 1] == cu[b]);                        // the run goes on, so there is one
            seq = sequence_of(b, sequences, cu, len_before, window, tokens_per_tile, kv_heads);
        }
        tc::fence_async_shared();                                      // the results' place is the rings' again
        __syncthreads();
        continue;
    }
    if (splits > 1) {                                                  // the slices of a tile form a cluster: over distributed shared memory
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
    return;
    }
}

struct Attention4 {
    const __nv_bfloat16* q;
    const uint8_t *k_pool, *v_pool;
    const int* table;
    int table_width, pool_blocks;
    const int *cu, *len_before;
    int sequences, n_tokens, heads, kv_heads;
    float scale_log2;
    int window, splits, one_token_each;
    __nv_bfloat16* out;
    float *part_acc, *part_ml;
    unsigned* tickets;
    long long part_rows;
    unsigned* status;
    const float* sinks;
};

template <int D, int NQ, bool DUP, int WARPS, bool EVEN>
cudaError_t launch_attention(const Attention4& a, int sms, cudaStream_t stream) {
    using R = Ring4<D, NQ, WARPS>;
    const int group = a.heads / a.kv_heads, tokens_per_tile = a.one_token_each ? 1 : (DUP ? 4 : 8 * NQ) / group;
    const int tiles = a.one_token_each ? a.sequences : a.n_tokens / tokens_per_tile + a.sequences;
    auto kernel = attention_4bit_kernel<D, NQ, DUP, WARPS, EVEN>;
    const cudaError_t code = tt_allow_shared(kernel, R::SHARED);
    if (code != cudaSuccess) return code;
    if (EVEN) {
        const int ctas = sms * R::CTAS;
        if ((long long)tiles * a.kv_heads * a.table_width >= 1LL << 30 || a.part_rows < 2LL * ctas * tokens_per_tile * group) return cudaErrorInvalidValue;
        // Not ahead of the kernel before it: whatever of that is still resident would leave an SM without room for one CTA of the grid, which
        // then starts when another one ends and takes as long again (measured with CTAs of four warps, where 6 of 592 were late: 55 -> 87 us).
        kernel<<<ctas, WARPS * 32, R::SHARED, stream>>>(a.q, a.k_pool, a.v_pool, a.table, a.table_width, a.pool_blocks, a.cu, a.len_before, a.sequences, a.heads,
                                                        a.kv_heads, tokens_per_tile, a.scale_log2, a.window, 0, a.out, a.part_acc, a.part_ml, a.tickets,
                                                        a.status, a.sinks);
        return cudaGetLastError();
    }
    return tt_launch_pdl_cluster(kernel, dim3(tiles, a.kv_heads, a.splits), dim3(WARPS * 32), R::SHARED, stream, (unsigned)a.splits, a.q, a.k_pool, a.v_pool, a.table,
                                 a.table_width, a.pool_blocks, a.cu, a.len_before, a.sequences, a.heads, a.kv_heads, tokens_per_tile, a.scale_log2, a.window,
                                 a.splits, a.out, a.part_acc, a.part_ml, a.tickets, a.status, a.sinks);
}

// Which form: even runs where the caller asks for them; slices with eight warps while all CTAs have an SM of their own (1 sequence of 2,048
// tokens, 8 heads of 64 in 8 slices: 6.7 us against 7.5 with four), with four otherwise (256 sequences of 1,024 tokens: 77 us against 87).
template <int D, int NQ, bool DUP>
cudaError_t launch_attention(const Attention4& a, cudaStream_t stream) {
    int sms = 0;
    const cudaError_t code = tt_sm_count(&sms);
    if (code != cudaSuccess) return code;
    if (a.splits == 0) return launch_attention<D, NQ, DUP, 8, true>(a, sms, stream);
    const long long tiles = a.one_token_each ? a.sequences : a.n_tokens * (a.heads / a.kv_heads) / (DUP ? 4 : 8 * NQ) + a.sequences;
    if (tiles * a.kv_heads * a.splits <= sms) return launch_attention<D, NQ, DUP, 8, false>(a, sms, stream);
    return launch_attention<D, NQ, DUP, 4, false>(a, sms, stream);
}

}  // namespace

// rows: query rows of a tile at most, 4, 8 or 16.  one_token_each: n_tokens == sequences and every sequence brings one.  splits 1..8: slices of the keys (see above); 0: even runs, whose
// parts need part_rows rows of head_dim numbers in part_acc and of 2 in part_ml, 2 for each row of a tile and each CTA that the device
// holds, and a ticket for each of those CTAs, zero before the call and after it.
extern "C" int tt_attention_4bit(const void* q, const void* k_pool, const void* v_pool, const int* table, int table_width, int pool_blocks,
                                 const int* cu, const int* len_before, int sequences, int n_tokens, int heads, int kv_heads, int head_dim,
                                 float scale, int window, int splits, int one_token_each, int rows, void* out, float* part_acc, float* part_ml,
                                 unsigned* tickets, long long part_rows, unsigned* status, const float* sinks, cudaStream_t stream) {
    if (n_tokens <= 0 || sequences <= 0) return 0;
    if (!cache4::takes(heads, kv_heads, head_dim) || splits < 0 || splits > 8 || !(scale > 0.0f) || (((uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)q) & 15) != 0 ||
        (splits == 0 && (!part_acc || !part_ml || !tickets)) || (rows != 4 && rows != 8 && rows != 16) || heads / kv_heads > rows)
        return (int)cudaErrorInvalidValue;
    const Attention4 a{(const __nv_bfloat16*)q, (const uint8_t*)k_pool, (const uint8_t*)v_pool, table, table_width, pool_blocks, cu, len_before, sequences, n_tokens,
                       heads, kv_heads, scale * 1.4426950408889634f, window, splits, one_token_each, (__nv_bfloat16*)out, part_acc, part_ml, tickets, part_rows,
                       status, sinks};
#define TT_LAUNCH_D(D)                                                                  \
    if (rows == 16) return (int)launch_attention<D, 2, false>(a, stream);              \
    if (rows == 8) return (int)launch_attention<D, 1, false>(a, stream);               \
    return (int)launch_attention<D, 1, true>(a, stream)
    switch (head_dim) {
        case 32: TT_LAUNCH_D(32);
        case 64: TT_LAUNCH_D(64);
        case 96: TT_LAUNCH_D(96);
        default: TT_LAUNCH_D(128);
    }
#undef TT_LAUNCH_D
}
