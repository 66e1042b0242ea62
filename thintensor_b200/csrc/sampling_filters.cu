// The next token of every row of float32 logits from a given random number, with the row's own temperature, top-k, top-p and min-p.
//
// With x the logits (NaN counts as minus infinity), M their maximum and w_j = exp((x_j - M) / T):
//   top-k  keeps the tokens whose logit is at least the k-th largest (ties with it stay);
//   top-p  keeps of these the tokens for which the weights of all strictly larger ones come to at most p times the weights of all;
//   min-p  keeps of these the tokens with w_j >= min_p;
//   the token is the first in order of its id at which the running sum of the kept weights exceeds u times their sum.
// T = 0: the largest logit, lowest id on ties.  k <= 0 or >= vocabulary, p >= 1 and min_p <= 0 switch a filter off.  A row without a finite logit or
// an infinite one: token 0.
//
// What must not depend on anything but the row: which token it is.  So the weights are formed in float64 (about 1e-14 relative) and
// summed as whole numbers of 2^-45: sums of those are exact, whatever their order.  Against exact real arithmetic a sum is off by the weights' rounding
// to whole numbers, 2^-46 of the largest weight each and so vocabulary * 2^-46 of it at most (2^-29 at 128,256; what lies below 2^-46 of the largest
// counts nothing), and only a random number, or a share, that close to a border could tell.  A float32 sum over 100,000 tokens is off by more than a rare
// token's whole weight.
//
// A row is read once, by a cluster of up to 8 CTAs that keep their slices of it in shared memory and talk over distributed shared
// memory.  One row of 128,256 takes 11 us for a nucleus of few tokens, 13 us with top-k and 25 us for a nucleus of tens of thousands, of which the
// float64 weights are 3 us a pass and the cluster's exchanges (10 for such a nucleus) and the passes' dependent steps most of the rest.
//
// With top-k, min-p or a nucleus near the largest logit, few tokens come into question, and they are found without a search: once a CTA's threads have seen their
// largest numbers, the k-th largest of those is reached by at least k of the slice's numbers and by few more, so a slice's k largest are
// among what reaches it.  The cluster sends such candidates to its first CTA, which compares them with each other and finishes the row alone.  A nucleus
// may hold half the vocabulary: it, a k beyond 256 and candidates beyond 512 go the general way, a search for the first key, from the largest
// down, at which a running sum (of ones, or of weights) exceeds a limit, by 2,048 bins and the members of the one in which it happens.
#include "common.cuh"

#include <cooperative_groups.h>
namespace cg = cooperative_groups;

namespace {

typedef unsigned long long u64;

constexpr int FILTER_THREADS = 512, FILTER_WARPS = FILTER_THREADS / 32;
constexpr int BINS = 2048;
constexpr int LISTED = 256;                          // members of a bin that are compared with each other
constexpr int CANDIDATES = 512;                      // of a row, at most, that the first CTA finishes alone
constexpr int MOST_K = 256;                          // largest top-k that is looked for among the threads' largest numbers
// How far a row's float32 sum of weights may be off: 2^-22 times the exponent, of which 40 counts (what is below 2^-40 of the largest weight comes to less
// than 2^-20), for each weight, and 2^-24 for each of a thread's 256 additions at most: less than 2^-14 together.
constexpr double SUM_ERROR = 1.0 / 1024.0;
constexpr int MAX_CLUSTER = 8;
constexpr int MAX_SLICE = 32768;                     // numbers of a row that a CTA keeps (128 KB)
constexpr int MOST_SLICE = 65536;                    // and that it may look at: 2^16 of a weight's 15-bit parts fit 32 bits
constexpr int CHUNK = 128;                           // neighbouring tokens whose weights are summed together

__device__ __forceinline__ unsigned order_key(float v) {
    const unsigned u = __float_as_uint(v);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);      // larger float <=> larger key
}

// What the phases keep in shared memory beside the row's slice.  The search and the candidates are never there together.
struct alignas(16) FilterShared {
    union {
        struct {
            unsigned part[3][BINS];                  // a bin's weights: sums of their bits 0..14, 15..29, 30..45 (64-bit additions are loops here)
            unsigned count[BINS];
            u64 list_mass[LISTED];
            unsigned list_key[LISTED];
        };
        struct {
            u64 candidate[CANDIDATES];               // key in the upper half, the id's complement in the lower
            u64 chosen[CANDIDATES];
            u64 chosen_mass[CANDIDATES];
        };
    };
    double powers[32];                               // 2^(j / 32)
    ulonglong2 exchange[2];                          // this CTA's words of the exchange under way, by its parity
    u64 warp_sums[FILTER_WARPS];
    u64 found_before;                                // results that one thread of the cluster hands to all
    unsigned found, found_count, listed, candidates, sent, chosen_count, unsure;
};

struct Filter {
    FilterShared* sh;
    cg::cluster_group cluster;
    int rank, ctas, parity;
    float top, far;                                  // M; M - 100 T, where weights have long been less than half a unit
    double inverse;                                  // 1 / T

    // exp((x - M) / T) in units of 2^-45: 2^(n / 32) from the table times the series of e^r, |r| <= ln 2 / 64 (its sixth power's term is
    // below 3e-15).  Without branches, so that several numbers' chains of float64 operations run together.
    __device__ __forceinline__ double weight(float x) const {
        const double z = ((double)fmaxf(x, far) - (double)top) * inverse;
        const double shifted = fma(z, 46.166241308446829, 6755399441055744.0);      // 32 / ln 2; 1.5 * 2^52: the nearest whole number in the low bits
        const int n = __double2loint(shifted);
        const double r = fma(shifted - 6755399441055744.0, -0.021660849392498290, z);
        double s = fma(r, 1.0 / 120.0, 1.0 / 24.0);
        s = fma(s, r, 1.0 / 6.0);
        s = fma(s, r, 0.5);
        s = fma(s, r, 1.0);
        const double base = sh->powers[n & 31];
        const double w = fma(base * r, s, base);
        const double scaled = __hiloint2double(__double2hiint(w) + (((n >> 5) + 45) << 20), __double2loint(w));
        return x == top ? 35184372088832.0 : x < far ? 0.0 : scaled;       // far is M itself where T is below its last bit
    }
    static __device__ __forceinline__ u64 units(double w) { return (u64)__double_as_longlong(w + 6755399441055744.0) - 0x4338000000000000ull; }
    __device__ __forceinline__ u64 mass(float x) const { return units(weight(x)); }

    // Two words of every CTA to every thread of the cluster: `join` folds them, from zeros, in order of rank.  What was written to shared memory
    // before is there for the whole cluster afterwards.
    template <typename Join> __device__ __forceinline__ void exchange(u64 (&word)[2], Join join) {
        ulonglong2* mine = &sh->exchange[parity];
        if (threadIdx.x == 0) *mine = make_ulonglong2(word[0], word[1]);
        cluster.sync();
        const int lane = threadIdx.x & 31;
        ulonglong2 other = make_ulonglong2(0ull, 0ull);
        if (lane < ctas) other = *cluster.map_shared_rank(mine, lane);
        u64 total[2] = {0ull, 0ull};
#pragma unroll
        for (int c = 0; c < MAX_CLUSTER; ++c) {
            const u64 a = __shfl_sync(0xffffffffu, other.x, c), b = __shfl_sync(0xffffffffu, other.y, c);      // zeros behind the last
            join(total, a, b, c);
        }
        word[0] = total[0];
        word[1] = total[1];
        parity ^= 1;                                 // written again two exchanges on: everybody has read it by then
    }
};

// A CTA's numbers of the row, four neighbouring ones at a time: from shared memory, cleaned and filled up with minus infinity, or, where
// the slice is too long for that, from the row itself.
struct Slice {
    const float* x;
    int n, quads;
    bool staged;
    __device__ __forceinline__ void four(int q, float (&v)[4]) const {
        if (staged) {
            const float4 u = reinterpret_cast<const float4*>(x)[q];
            v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float u = 4 * q + e < n ? __ldg(x + 4 * q + e) : -INFINITY;
                v[e] = u != u ? -INFINITY : u + 0.0f;
            }
        }
    }
};

template <typename T, typename Op> __device__ __forceinline__ T warp_fold(T v, Op op) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
// Over the CTA, from nothing being 0; all threads get it.
template <typename Op> __device__ __forceinline__ u64 block_fold(u64 v, u64* warps, Op op) {
    v = warp_fold(v, op);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_fold((threadIdx.x & 31) < FILTER_WARPS ? warps[threadIdx.x & 31] : 0ull, op);
}
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// A logit as the filters see it: what is no number weighs nothing, and there is one zero.
__device__ __forceinline__ float clean(float v) { return v != v ? -INFINITY : v + 0.0f; }
__device__ __forceinline__ u64 add64(u64 a, u64 b) { return a + b; }
__device__ __forceinline__ u64 max64(u64 a, u64 b) { return a > b ? a : b; }
// Sum of the values of the threads before this one, and of all.
__device__ __forceinline__ u64 block_before(u64 v, u64* warps, u64& all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u64 upto = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 up = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += up;
    }
    __syncthreads();
    if (lane == 31) warps[warp] = upto;
    __syncthreads();
    u64 before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < FILTER_WARPS; ++w) {
        const u64 sum = warps[w];
        if (w < warp) before += sum;
        all += sum;
    }
    return before + upto - v;
}

// The first key, from the largest down and not below `floor_key`, at which the running sum over the row (MASS: of the weights, else of ones)
// exceeds a limit: `limit`, or `share` of the whole sum.  x: this CTA's slice.
template <bool MASS>
__device__ unsigned search_key(Filter& f, const Slice& x, float lowest, unsigned floor_key, u64 limit, double share) {
    FilterShared* sh = f.sh;
    const float range = f.top - lowest;
    const float even = (range > 0.0f && range < INFINITY) ? (float)(BINS - 1) / range : 0.0f;
    unsigned from = floor_key, upto = 0xffffffffu;   // keys that are still in question
    bool by_bits = false, limited = !MASS;
    u64 before = 0;                                  // the sum of what lies above them
    u64 width = 0;
    __syncthreads();                                 // what an earlier search found has been read
    for (;;) {
        for (int i = threadIdx.x; i < BINS; i += FILTER_THREADS) {
            sh->count[i] = 0u;
            if (MASS) sh->part[0][i] = sh->part[1][i] = sh->part[2][i] = 0u;
        }
        if (threadIdx.x == 0) { sh->listed = 0u; sh->found = 0xffffffffu; }
        __syncthreads();
        // 0 for the largest.  Even in logit at first (subtraction, product and conversion keep the order), then by the bits.
        auto bin_of = [&](float v, unsigned key) {
            if (by_bits) return (int)((u64)(upto - key) * BINS / width);
            const float at = (f.top - v) * even;
            return v == f.top ? 0 : (at < (float)(BINS - 1) ? (int)at : BINS - 1);
        };
        // four numbers at a time: their weights' chains run together
#pragma unroll 2
        for (int q = threadIdx.x; q < x.quads; q += FILTER_THREADS) {
            float v[4];
            u64 m[4];
            x.four(q, v);
#pragma unroll
            for (int e = 0; e < 4; ++e) m[e] = MASS ? f.mass(v[e]) : 0ull;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const unsigned key = order_key(v[e]);
                if (key < from || key > upto) continue;                // minus infinity is below every floor
                const int bin = bin_of(v[e], key);
                atomicAdd(&sh->count[bin], 1u);
                if (MASS) {
                    const unsigned low = (unsigned)m[e] & 0x7fffu, middle = (unsigned)(m[e] >> 15) & 0x7fffu, high = (unsigned)(m[e] >> 30);
                    if (low) atomicAdd(&sh->part[0][bin], low);
                    if (middle) atomicAdd(&sh->part[1][bin], middle);
                    if (high) atomicAdd(&sh->part[2][bin], high);
                }
            }
        }
        f.cluster.sync();
        // every CTA adds up its share of the bins
        const int share_bins = BINS / f.ctas;
        u64 sums[BINS / FILTER_THREADS], mine = 0;
        unsigned counts[BINS / FILTER_THREADS];
        const int each = (share_bins + FILTER_THREADS - 1) / FILTER_THREADS;         // 4 bins a thread, or one
        const int first = f.rank * share_bins + threadIdx.x * each;
#pragma unroll
        for (int k = 0; k < BINS / FILTER_THREADS; ++k) {
            sums[k] = 0;
            counts[k] = 0;
            if (k < each && threadIdx.x * each + k < share_bins)
#pragma unroll
                for (int c = 0; c < MAX_CLUSTER; ++c) {               // the last CTA's again behind it, so that all loads go out together
                    const FilterShared* other = f.cluster.map_shared_rank(sh, min(c, f.ctas - 1));
                    const unsigned add = other->count[first + k];
                    const u64 sum = MASS ? (u64)other->part[0][first + k] + ((u64)other->part[1][first + k] << 15) + ((u64)other->part[2][first + k] << 30) : (u64)add;
                    if (c < f.ctas) { counts[k] += add; sums[k] += sum; }
                }
            mine += sums[k];
        }
        u64 word[2] = {0, 0};
        u64 running = block_before(mine, sh->warp_sums, word[0]);
        const int rank = f.rank;
        u64 lower = 0;
        f.exchange(word, [&](u64 (&total)[2], u64 a, u64, int c) {
            if (c == rank) lower = total[0];
            total[0] += a;
        });
        if (!limited) {
            const double most = share * (double)word[0];
            limit = most > 0.0 ? (u64)most : 0ull;
            limited = true;
        }
        running += before + lower;
#pragma unroll
        for (int k = 0; k < BINS / FILTER_THREADS; ++k) {
            if (sums[k] && running <= limit && running + sums[k] > limit)
                for (int c = 0; c < f.ctas; ++c) {
                    FilterShared* other = f.cluster.map_shared_rank(sh, c);
                    other->found = (unsigned)(first + k);
                    other->found_count = counts[k];
                    other->found_before = running;
                }
            running += sums[k];
        }
        f.cluster.sync();
        const unsigned bin = sh->found, members = sh->found_count;
        if (bin == 0xffffffffu) return from;         // the whole sum does not exceed the limit: nothing is dropped
        before = sh->found_before;
        if (members <= LISTED) {
            // to the first CTA's list, in any order
            FilterShared* head = f.cluster.map_shared_rank(sh, 0);
#pragma unroll 2
            for (int q = threadIdx.x; q < x.quads; q += FILTER_THREADS) {
                float v[4];
                x.four(q, v);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const unsigned key = order_key(v[e]);
                    if (key < from || key > upto || bin_of(v[e], key) != (int)bin) continue;
                    const unsigned at = atomicAdd(&head->listed, 1u);
                    head->list_key[at] = key;
                    head->list_mass[at] = MASS ? f.mass(v[e]) : 1ull;
                }
            }
            f.cluster.sync();
            if (f.rank == 0) {
                const int i = threadIdx.x;
                if (i < (int)members) {
                    const unsigned key = sh->list_key[i];
                    u64 above = before, with = 0;
                    for (int j = 0; j < (int)members; ++j) {
                        const unsigned other = sh->list_key[j];
                        const u64 m = sh->list_mass[j];
                        above += other > key ? m : 0ull;
                        with += other == key ? m : 0ull;
                    }
                    if (above <= limit && above + with > limit)        // equal keys find the same
                        for (int c = 0; c < f.ctas; ++c) f.cluster.map_shared_rank(sh, c)->found = key;
                }
            }
            f.cluster.sync();
            return sh->found;
        }
        // too many: their range of keys, and bins of it
        unsigned least = 0xffffffffu, greatest = 0u;
        for (int q = threadIdx.x; q < x.quads; q += FILTER_THREADS) {
            float v[4];
            x.four(q, v);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const unsigned key = order_key(v[e]);
                if (key < from || key > upto || bin_of(v[e], key) != (int)bin) continue;
                least = min(least, key);
                greatest = max(greatest, key);
            }
        }
        word[0] = block_fold((u64)~least, sh->warp_sums, max64);
        word[1] = block_fold((u64)greatest, sh->warp_sums, max64);
        f.exchange(word, [](u64 (&total)[2], u64 a, u64 b, int) { total[0] = max64(total[0], a); total[1] = max64(total[1], b); });
        from = ~(unsigned)word[0];
        upto = (unsigned)word[1];
        if (from == upto) return from;               // equal logits
        by_bits = true;
        width = (u64)(upto - from) + 1;
    }
}

// A key that at least k of the threads' keys reach and few more (0 where fewer than k are there); all threads call and get it.  Bit by bit from
// the first in which the keys differ, until it is reached by at most a quarter more than k.
__device__ __forceinline__ unsigned reached_by(unsigned key, int k, u64* warps) {
    const unsigned high = __reduce_max_sync(0xffffffffu, key), low = __reduce_max_sync(0xffffffffu, ~key);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __syncthreads();
    if (lane == 0) warps[warp] = (u64)high << 32 | low;
    __syncthreads();
    const u64 both = warps[lane & (FILTER_WARPS - 1)];
    const unsigned top = __reduce_max_sync(0xffffffffu, (unsigned)(both >> 32)), bottom = ~__reduce_max_sync(0xffffffffu, (unsigned)both);
    if (k > FILTER_THREADS) return 0u;
    if (top == bottom) return top;
    const int first = 31 - __clz(top ^ bottom);
    unsigned floor_key = first == 31 ? 0u : top >> (first + 1) << (first + 1);
    for (int bit = first; bit >= 0; --bit) {
        const unsigned candidate = floor_key | (1u << bit);
        const int count = __syncthreads_count(key >= candidate);
        if (count < k) continue;
        floor_key = candidate;
        if (count <= k + k / 4) break;
    }
    return floor_key;
}

// The row from its `count` candidates, by the first CTA: with top_k they are all that can be among the k largest, without all that min-p leaves, or
// (nucleus) all of one without top-k, whose border lies between low and high.  -1: a token's border does, too.
__device__ int choose_among(Filter& f, int count, int top_k, float top_p, bool nucleus, u64 low, u64 high, double least_units, float u) {
    FilterShared* sh = f.sh;
    constexpr int EACH = CANDIDATES / FILTER_THREADS;
    auto value_of = [](unsigned key) { return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key); };
    // the k-th largest key: bit by bit
    unsigned key[EACH], floor_key = 0u;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int i = e * FILTER_THREADS + threadIdx.x;
        key[e] = i < count ? (unsigned)(sh->candidate[i] >> 32) : 0u;
    }
    if (top_k > 0 && top_k < count) {
        // two bits a round, the counts of its three thresholds in fields of 10 bits (a warp's are at most 32 each)
        for (int bit = 30; bit >= 0; bit -= 2) {
            unsigned mine = 0u;
#pragma unroll
            for (int e = 0; e < EACH; ++e)
#pragma unroll
                for (int j = 1; j < 4; ++j) mine += (unsigned)(key[e] >= (floor_key | (unsigned)j << bit)) << (10 * (j - 1));
            const unsigned sum = __reduce_add_sync(0xffffffffu, mine);
            unsigned* counts = reinterpret_cast<unsigned*>(sh->warp_sums) + (bit & 2 ? FILTER_WARPS : 0);
            if ((threadIdx.x & 31) == 0) counts[threadIdx.x >> 5] = sum;
            __syncthreads();
            const unsigned w = (threadIdx.x & 31) < FILTER_WARPS ? counts[threadIdx.x & 31] : 0u;
            const int one = __reduce_add_sync(0xffffffffu, w & 1023u), two = __reduce_add_sync(0xffffffffu, w >> 10 & 1023u), three = __reduce_add_sync(0xffffffffu, w >> 20);
            floor_key |= (three >= top_k ? 3u : two >= top_k ? 2u : one >= top_k ? 1u : 0u) << bit;
        }
    }
    if (threadIdx.x == 0) sh->chosen_count = 0u;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int i = e * FILTER_THREADS + threadIdx.x;
        if (i < count && key[e] >= floor_key) {
            const unsigned at = atomicAdd(&sh->chosen_count, 1u);
            sh->chosen[at] = sh->candidate[i];
            sh->chosen_mass[at] = f.mass(value_of(key[e]));
        }
    }
    __syncthreads();
    const int n = (int)sh->chosen_count;
    // few: each number looks at all others
    u64 mass[EACH], sum = 0;
    unsigned id[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int i = e * FILTER_THREADS + threadIdx.x;
        const u64 both = i < n ? sh->chosen[i] : 0ull;
        key[e] = (unsigned)(both >> 32);
        id[e] = ~(unsigned)both;
        mass[e] = i < n ? sh->chosen_mass[i] : 0ull;
        sum += mass[e];
    }
    if (top_p < 1.0f) {
        if (!nucleus) {
            const double most = (double)top_p * (double)block_fold(sum, sh->warp_sums, add64);
            low = high = most > 0.0 ? (u64)most : 0ull;
        }
        u64 above[EACH] = {};
        if ((int)threadIdx.x < n)
#pragma unroll 4
            for (int j = 0; j < n; ++j) {
                const unsigned other = (unsigned)(sh->chosen[j] >> 32);
                const u64 m = sh->chosen_mass[j];
#pragma unroll
                for (int e = 0; e < EACH; ++e) above[e] += other > key[e] ? m : 0ull;
            }
        bool unsure = false;
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            unsure = unsure || (mass[e] && above[e] > low && above[e] <= high);
            if (above[e] > low) mass[e] = 0ull;
        }
        if (__syncthreads_or(unsure)) return -1;
    }
    sum = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int i = e * FILTER_THREADS + threadIdx.x;
        if (mass[e] && least_units > 0.0 && !(f.weight(value_of(key[e])) >= least_units)) mass[e] = 0ull;
        if (i < n) sh->chosen_mass[i] = mass[e];
        sum += mass[e];
    }
    const u64 total = block_fold(sum, sh->warp_sums, add64);
    const double wanted = (double)u * (double)total;
    const u64 target = min(wanted > 0.0 ? (u64)wanted : 0ull, total - 1);      // a random number of one or more: the last kept token
    u64 before[EACH] = {};
    if ((int)threadIdx.x < n)
#pragma unroll 4
        for (int j = 0; j < n; ++j) {
            const unsigned other = ~(unsigned)sh->chosen[j];
            const u64 m = sh->chosen_mass[j];
#pragma unroll
            for (int e = 0; e < EACH; ++e) before[e] += other < id[e] ? m : 0ull;
        }
#pragma unroll
    for (int e = 0; e < EACH; ++e)
        if (mass[e] && before[e] <= target && before[e] + mass[e] > target) sh->found = id[e];
    __syncthreads();
    return (int)sh->found;
}

// uniform in [0, 1) from (seed, request, step), 24 bits: the sampler's counter (sampling.cu)
__device__ __forceinline__ u64 mix64(u64 x) {
    x ^= x >> 30; x *= 0xBF58476D1CE4E5B9ull;
    x ^= x >> 27; x *= 0x94D049BB133111EBull;
    x ^= x >> 31;
    return x;
}
__device__ __forceinline__ float counter_uniform(u64 seed, u64 request, u64 step) {
    u64 x = mix64(seed + 0x9E3779B97F4A7C15ull);
    x = mix64(x ^ (request * 0xD1B54A32D192ED03ull));
    x = mix64(x ^ (step * 0x8CB92BA72F3D8DD7ull));
    return (float)(x >> 40) * (1.0f / 16777216.0f);
}

// grid = rows * cluster; a row's settings are arrays, or the same for all rows (pointers null).
__global__ void __launch_bounds__(FILTER_THREADS, 2)
sample_filtered_kernel(const float* __restrict__ logits, long long ld, int vocab, int slice, int staged, const float* __restrict__ temperatures, float temperature,
                       const int* __restrict__ top_ks, int top_k, const float* __restrict__ top_ps, float top_p, const float* __restrict__ min_ps, float min_p,
                       const float* __restrict__ uniforms, u64 seed, const int* __restrict__ requests, const int* __restrict__ steps, int* __restrict__ out) {
    extern __shared__ __align__(16) unsigned char filter_memory[];
    tt_pdl_launch_dependents();
    Filter f{reinterpret_cast<FilterShared*>(filter_memory), cg::this_cluster()};
    FilterShared* sh = f.sh;
    f.rank = (int)f.cluster.block_rank();
    f.ctas = (int)f.cluster.num_blocks();
    f.parity = 0;
    const int row = blockIdx.x / f.ctas, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x < 32) sh->powers[threadIdx.x] = exp2((double)threadIdx.x / 32.0);
    if (threadIdx.x == 0) sh->candidates = sh->sent = 0u;
    tt_pdl_wait();
    if (temperatures) temperature = __ldg(temperatures + row);
    if (top_ks) top_k = __ldg(top_ks + row);
    if (top_ps) top_p = __ldg(top_ps + row);
    if (min_ps) min_p = __ldg(min_ps + row);

    // this CTA's slice of the row, and the row's largest and smallest finite logits
    const int lo = f.rank * slice, n = max(0, min(slice, vocab - lo));
    const float* from = logits + (size_t)row * ld + lo;
    float* kept = reinterpret_cast<float*>(filter_memory + sizeof(FilterShared));
    u64* chunks = reinterpret_cast<u64*>(kept + (staged ? slice : 0));                     // slices are whole chunks
    float most = -INFINITY, least = INFINITY;
    auto look = [&](float v) {
        v = clean(v);
        most = fmaxf(most, v);
        if (v > -INFINITY) least = fminf(least, v);
        return v;
    };
    if ((((uintptr_t)from) & 15) == 0 && staged) {
        const float4* from4 = reinterpret_cast<const float4*>(from);
        float4* kept4 = reinterpret_cast<float4*>(kept);
#pragma unroll 4
        for (int i = threadIdx.x; i < n / 4; i += FILTER_THREADS) {
            float4 v = __ldg(from4 + i);
            v.x = look(v.x); v.y = look(v.y); v.z = look(v.z); v.w = look(v.w);
            kept4[i] = v;
        }
        for (int i = n / 4 * 4 + threadIdx.x; i < n; i += FILTER_THREADS) kept[i] = look(__ldg(from + i));
    } else {
#pragma unroll 8
        for (int i = threadIdx.x; i < n; i += FILTER_THREADS) {
            const float v = look(__ldg(from + i));
            if (staged) kept[i] = v;
        }
    }
    const Slice x{staged ? kept : from, n, (n + CHUNK - 1) / CHUNK * (CHUNK / 4), (bool)staged};
    if (staged)
        for (int i = n + threadIdx.x; i < 4 * x.quads; i += FILTER_THREADS) kept[i] = -INFINITY;
    u64 word[2];
    {
        const unsigned high = __reduce_max_sync(0xffffffffu, order_key(most)), low = __reduce_max_sync(0xffffffffu, ~order_key(least));
        if (lane == 0) sh->warp_sums[warp] = (u64)high << 32 | low;
        __syncthreads();
        const u64 both = sh->warp_sums[lane & (FILTER_WARPS - 1)];
        word[0] = __reduce_max_sync(0xffffffffu, (unsigned)(both >> 32));
        word[1] = __reduce_max_sync(0xffffffffu, (unsigned)both);
    }
    f.exchange(word, [](u64 (&total)[2], u64 a, u64 b, int) { total[0] = max64(total[0], a); total[1] = max64(total[1], b); });
    auto value_of = [](unsigned key) { return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key); };
    f.top = value_of((unsigned)word[0]);
    const float lowest = value_of(~(unsigned)word[1]);

    if (f.top == -INFINITY || !(temperature > 0.0f)) {                 // nothing to choose from, or the largest logit's lowest id
        u64 at = ~0ull;
        for (int q = threadIdx.x; q < x.quads && at == ~0ull; q += FILTER_THREADS) {       // a thread's first is its lowest
            float v[4];
            x.four(q, v);
#pragma unroll
            for (int e = 3; e >= 0; --e)
                if (v[e] == f.top && 4 * q + e < n) at = (u64)(lo + 4 * q + e);
        }
        word[0] = block_fold(~at, sh->warp_sums, max64);
        word[1] = 0;
        f.exchange(word, [](u64 (&total)[2], u64 a, u64, int) { total[0] = max64(total[0], a); });
        if (f.rank == 0 && threadIdx.x == 0) out[row] = f.top == -INFINITY ? 0 : (int)~word[0];
        f.cluster.sync();                                              // nobody leaves while its words are being read
        return;
    }
    f.inverse = 1.0 / (double)temperature;
    f.far = f.top - 100.0f * temperature;
    const float u = uniforms ? __ldg(uniforms + row)
                             : counter_uniform(seed, (u64)(unsigned)__ldg(requests + row), (u64)(unsigned)__ldg(steps + row));
    if (top_k >= vocab) top_k = 0;
    // what is minus infinity, or no number, weighs nothing, and beside an infinite logit nothing else does
    const unsigned lowest_key = f.top == INFINITY ? order_key(INFINITY) : order_key(-INFINITY) + 1;
    // min-p: weights well below it need not be formed
    const double least_weight = (double)fminf(min_p, 1.0f);
    unsigned min_p_key = lowest_key;
    if (least_weight > 0.0 && f.top < INFINITY && temperature < INFINITY) {
        const float below = f.top + temperature * logf(fminf(min_p, 1.0f)) * 1.0001f - 1e-3f * fabsf(f.top) - 1e-30f;
        min_p_key = max(min_p_key, order_key(below));
    }
    const double least_units = least_weight * 35184372088832.0;
    // A nucleus without top-k: the tokens within e^-7 of the likeliest, if they hold more than its share or min-p leaves no others.  A float32 sum
    // of all weights tells, unless a token's border lies within that sum's error.  (1 x 128,256 with
    // min-p: 28 -> 11 us; 64 rows of which a tenth gain and a tenth are looked at in vain: 53 -> 54.)
    const bool nucleus = top_k <= 0 && top_p < 1.0f && f.top < INFINITY && temperature < INFINITY;
    if (top_k > 0 ? top_k <= MOST_K : nucleus || min_p_key > lowest_key) {
        unsigned reach = lowest_key;
        if (top_k > 0) reach = max(reach, reached_by(order_key(most), top_k, sh->warp_sums));
        if (top_p >= 1.0f || nucleus) reach = max(reach, min_p_key);   // (of the k largest, a nucleus counts what min-p takes from it)
        if (nucleus) reach = max(reach, order_key(f.top - 7.0f * temperature));
        u64 low = 0, high = 0;                                         // top-p times all weights lies between
        bool enough = true;
        if (nucleus) {
            const float scale = (float)(f.inverse * 1.4426950408889634);
            float all = 0.0f, held = 0.0f;                             // weights of the slice, and of its candidates
#pragma unroll 2
            for (int q = threadIdx.x; q < x.quads; q += FILTER_THREADS) {
                float v[4];
                x.four(q, v);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float w = v[e] == f.top ? 1.0f : fast_exp2((v[e] - f.top) * scale);
                    all += w;
                    held += order_key(v[e]) >= reach ? w : 0.0f;
                }
            }
            word[0] = block_fold((u64)(all * 4294967296.0f), sh->warp_sums, add64);
            word[1] = block_fold((u64)(held * 4294967296.0f), sh->warp_sums, add64);
            f.exchange(word, [](u64 (&total)[2], u64 a, u64 b, int) { total[0] += a; total[1] += b; });
            const double share = (double)top_p * (double)word[0] * 8192.0;               // in units of 2^-45
            low = (u64)fmax(share * (1.0 - SUM_ERROR), 0.0);
            high = (u64)fmax(share * (1.0 + SUM_ERROR), 0.0) + 1;
            enough = reach <= min_p_key || (double)word[1] * 8192.0 * (1.0 - SUM_ERROR) > (double)high;
        }
        unsigned count = CANDIDATES + 1;
        if (enough) {
            FilterShared* head = f.cluster.map_shared_rank(sh, 0);
#pragma unroll 2
            for (int q = threadIdx.x; q < x.quads; q += FILTER_THREADS) {
                float v[4];
                x.four(q, v);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const unsigned key = order_key(v[e]);
                    if (key >= reach && (top_k > 0 || atomicAdd(&sh->sent, 1u) <= CANDIDATES)) {      // too many in one slice are too many in all
                        const unsigned at = atomicAdd(&head->candidates, 1u);
                        if (at < CANDIDATES) head->candidate[at] = (u64)key << 32 | (unsigned)~(lo + 4 * q + e);
                    }
                }
            }
            f.cluster.sync();
            count = head->candidates;
            f.cluster.sync();
        }
        if (count <= CANDIDATES) {
            if (f.rank == 0) {
                const int token = choose_among(f, (int)count, top_k, top_p, nucleus, low, high, least_units, u);
                if (threadIdx.x == 0) {
                    if (token >= 0) out[row] = token;
                    sh->unsure = token < 0;
                }
            }
            if (!nucleus) return;
            f.cluster.sync();
            const bool unsure = f.cluster.map_shared_rank(sh, 0)->unsure;
            f.cluster.sync();                                          // the first CTA's word has been read
            if (!unsure) return;
        }
    }

    unsigned floor_key = lowest_key;
    if (top_k > 0) floor_key = max(floor_key, search_key<false>(f, x, lowest, floor_key, (u64)(top_k - 1), 0.0));
    if (top_p < 1.0f) floor_key = max(floor_key, search_key<true>(f, x, lowest, floor_key, 0, (double)top_p));
    floor_key = max(floor_key, min_p_key);
    auto kept_mass = [&](float v) -> u64 {
        const double w = f.weight(v);
        return order_key(v) >= floor_key && w >= least_units ? Filter::units(w) : 0ull;
    };

    // the kept weights of a chunk of neighbouring tokens at a time, four a lane, and of the slice
    u64 mine = 0;
    const int n_chunks = x.quads / (CHUNK / 4);
#pragma unroll 2
    for (int c = warp; c < n_chunks; c += FILTER_WARPS) {
        float v[4];
        x.four(CHUNK / 4 * c + lane, v);
        u64 m = 0;
        if (__any_sync(0xffffffffu, order_key(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]))) >= floor_key)) {
            m = (kept_mass(v[0]) + kept_mass(v[1])) + (kept_mass(v[2]) + kept_mass(v[3]));
            m = warp_fold(m, add64);
        }
        if (lane == 0) { chunks[c] = m; mine += m; }
    }
    word[0] = block_fold(mine, sh->warp_sums, add64);
    word[1] = 0;
    u64 before = 0;
    const int rank = f.rank;
    const u64 own = word[0];
    f.exchange(word, [&](u64 (&total)[2], u64 a, u64, int c) {
        if (c == rank) before = total[0];
        total[0] += a;
    });
    const u64 total = word[0];
    const double wanted = (double)u * (double)total;
    u64 target = wanted > 0.0 ? (u64)wanted : 0ull;
    target = min(target, total - 1);                                   // a random number of one or more: the last kept token
    if (before <= target && before + own > target) {                   // it is in this slice
        const int each = (n_chunks + FILTER_THREADS - 1) / FILTER_THREADS, first = threadIdx.x * each;
        u64 sum = 0;
        for (int c = first; c < min(first + each, n_chunks); ++c) sum += chunks[c];
        u64 all;
        u64 running = before + block_before(sum, sh->warp_sums, all);
        for (int c = first; c < min(first + each, n_chunks); ++c) {
            if (running <= target && running + chunks[c] > target) { sh->found = (unsigned)c; sh->found_before = running; }
            running += chunks[c];
        }
        __syncthreads();
        if (warp == 0) {
            const int q = CHUNK / 4 * (int)sh->found + lane;
            float v[4];
            x.four(q, v);
            u64 m[4], upto = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) { m[e] = kept_mass(v[e]); upto += m[e]; }
            const u64 own_four = upto;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 up = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += up;
            }
            u64 at = sh->found_before + upto - own_four;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (at <= target && at + m[e] > target) out[row] = lo + 4 * q + e;
                at += m[e];
            }
        }
    }
    f.cluster.sync();                                                  // nobody leaves while its words are being read
}

}  // namespace

// Settings: a pointer each (one number a row), or null for the number beside it.  uniforms: one a row, or null: the counter's of (seed,
// requests[row], steps[row]).
extern "C" int tt_sample_filtered(const float* logits, long long ld, int rows, int vocab, const float* temperatures, float temperature, const int* top_ks, int top_k,
                                  const float* top_ps, float top_p, const float* min_ps, float min_p, const float* uniforms, unsigned long long seed,
                                  const int* requests, const int* steps, int* out, cudaStream_t stream) {
    if (rows <= 0) return 0;
    // one number short of what the slices could hold: 2^19 equal weights of 2^45 come to 2^64
    if (vocab <= 0 || vocab >= MAX_CLUSTER * MOST_SLICE || (!uniforms && (!requests || !steps))) return (int)cudaErrorInvalidValue;
    int sms = 0;
    cudaError_t code = tt_sm_count(&sms);
    if (code != cudaSuccess) return (int)code;
    // CTAs a row: slices of at most 16,384 numbers, so that two CTAs fit an SM (64 rows of 128,256: 53 us; 200 rows of 32,003 in slices of 8,192: 35 -> 44
    // us); more while SMs are free and slices are not below 2,048.
    int ctas = 1;
    while (ctas < MAX_CLUSTER && ((vocab + ctas - 1) / ctas > 16384 || ((long long)rows * ctas * 2 <= sms && vocab / (2 * ctas) >= 2048))) ctas *= 2;
    const int slice = ((vocab + ctas - 1) / ctas + CHUNK - 1) / CHUNK * CHUNK;
    const int staged = slice <= MAX_SLICE;
    if ((long long)rows * ctas > 0x7fffffff) return (int)cudaErrorInvalidValue;
    const size_t shared = sizeof(FilterShared) + (staged ? (size_t)slice * 4 : 0) + (size_t)(slice / CHUNK) * 8;
    if ((code = tt_allow_shared(sample_filtered_kernel, shared)) != cudaSuccess) return (int)code;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(rows * ctas));
    config.blockDim = dim3(FILTER_THREADS);
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    cudaLaunchAttribute attribute[2];
    attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[0].val.programmaticStreamSerializationAllowed = 1;
    attribute[1].id = cudaLaunchAttributeClusterDimension;
    attribute[1].val.clusterDim.x = (unsigned)ctas;
    attribute[1].val.clusterDim.y = 1;
    attribute[1].val.clusterDim.z = 1;
    config.attrs = attribute;
    config.numAttrs = 2;
    code = cudaLaunchKernelEx(&config, sample_filtered_kernel, logits, ld, vocab, slice, staged, temperatures, temperature, top_ks, top_k, top_ps, top_p, min_ps, min_p,
                              uniforms, (u64)seed, requests, steps, out);
    return (int)code;
}
