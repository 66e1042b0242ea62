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
// summed as whole numbers of 2^-45: sums of those are exact, whatever their order, and only a random number within 2^-27 / vocabulary or so of a
// border could tell them from exact real arithmetic.  A float32 sum over 100,000 tokens is off by more than a rare token's
// whole weight.
//
// A row is read once, by a cluster of up to 8 CTAs that keep their slices of it in shared memory and talk over distributed shared
// memory.  The k-th largest logit and the nucleus' edge are one search: the first key, from the largest down, at which a running
// sum (of ones, or of weights) exceeds a limit.  2,048 bins, even in logit, give the bin in which it happens; its few hundred
// members are compared with each other, or binned again by their bits where they are more.  Bound by the row's bytes where many
// rows are in flight, and by some ten exchanges across the cluster (half a microsecond to one each) for a single row.
#include "common.cuh"

#include <cooperative_groups.h>
namespace cg = cooperative_groups;

namespace {

typedef unsigned long long u64;

constexpr int FILTER_THREADS = 512, FILTER_WARPS = FILTER_THREADS / 32;
constexpr int BINS = 2048;
constexpr int LISTED = 256;                          // members of a bin that are compared with each other
constexpr int MAX_CLUSTER = 8;
constexpr int MAX_SLICE = 40960;                     // numbers of a row that a CTA keeps (160 KB)

__device__ __forceinline__ unsigned order_key(float v) {
    const unsigned u = __float_as_uint(v);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);      // larger float <=> larger key
}

// What the phases keep in shared memory beside the row's slice.
struct alignas(16) FilterShared {
    u64 mass[BINS];                                  // a bin's weights
    unsigned count[BINS];
    u64 list_mass[LISTED];
    unsigned list_key[LISTED];
    unsigned listed;
    double powers[32];                               // 2^(j / 32)
    u64 exchange[2][2];                              // this CTA's words of the exchange under way, by its parity
    u64 warp_sums[FILTER_WARPS];
    u64 found_before;                                // results that one thread of the cluster hands to all
    unsigned found, found_count;
};

struct Filter {
    FilterShared* sh;
    cg::cluster_group cluster;
    int rank, ctas, parity;
    float top;                                       // M
    double inverse, inverse32;                       // 1 / T, 32 log2(e) / T

    // exp((x - M) / T) in units of 2^-45, rounded to whole numbers: 2^(n / 32) from the table times the series of e^r, |r| <= ln 2 / 64
    // (its sixth power's term is below 3e-15).
    __device__ __forceinline__ double weight(float x) const {
        if (x == top) return 35184372088832.0;
        const double d = (double)x - (double)top;
        const double z = d * inverse;
        if (!(z > -33.0)) return 0.0;                // below half a unit
        const double shifted = d * inverse32 + 6755399441055744.0;            // 1.5 * 2^52: the nearest whole number in the low bits
        const int n = __double2loint(shifted);
        const double r = fma(shifted - 6755399441055744.0, -0.021660849392498290, z);
        double s = fma(r, 1.0 / 120.0, 1.0 / 24.0);
        s = fma(s, r, 1.0 / 6.0);
        s = fma(s, r, 0.5);
        s = fma(s, r, 1.0);
        const double base = sh->powers[n & 31];
        const double w = fma(base * r, s, base);
        return __hiloint2double(__double2hiint(w) + (((n >> 5) + 45) << 20), __double2loint(w));
    }
    static __device__ __forceinline__ u64 units(double w) { return (u64)__double_as_longlong(w + 6755399441055744.0) - 0x4338000000000000ull; }
    __device__ __forceinline__ u64 mass(float x) const { return units(weight(x)); }

    // Two words of every CTA to every thread of the cluster: `join` folds them, from zeros, in order of rank.  What was written to shared memory
    // before is there for the whole cluster afterwards.
    template <typename Join> __device__ __forceinline__ void exchange(u64 (&word)[2], Join join) {
        u64* mine = sh->exchange[parity];
        if (threadIdx.x == 0) { mine[0] = word[0]; mine[1] = word[1]; }
        cluster.sync();
        u64 total[2] = {0ull, 0ull}, others[MAX_CLUSTER][2];
#pragma unroll
        for (int c = 0; c < MAX_CLUSTER; ++c)
            if (c < ctas) {
                const u64* other = cluster.map_shared_rank(mine, c);
                others[c][0] = other[0];
                others[c][1] = other[1];
            }
#pragma unroll
        for (int c = 0; c < MAX_CLUSTER; ++c)
            if (c < ctas) join(total, others[c][0], others[c][1], c);
        word[0] = total[0];
        word[1] = total[1];
        parity ^= 1;                                 // written again two exchanges on: everybody has read it by then
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
// A logit as the filters see it: what is no number weighs nothing, and there is one zero.
__device__ __forceinline__ float clean(float v) { return v != v ? -INFINITY : v + 0.0f; }
__device__ __forceinline__ u64 add64(u64 a, u64 b) { return a + b; }
__device__ __forceinline__ u64 max64(u64 a, u64 b) { return a > b ? a : b; }
// Sum of the values of the threads before this one.
__device__ __forceinline__ u64 block_before(u64 v, u64* warps) {
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
    for (int w = 0; w < warp; ++w) before += warps[w];
    return before + upto - v;
}

// The first key, from the largest down and not below `floor_key`, at which the running sum over the row (MASS: of the weights, else of ones)
// exceeds a limit: count `limit`, or `share` of the whole sum.  x: this CTA's slice, n numbers.
template <bool MASS>
__device__ unsigned search_key(Filter& f, const float* x, int n, float lowest, unsigned floor_key, u64 limit, double share) {
    FilterShared* sh = f.sh;
    const float range = f.top - lowest;
    const float even = (range > 0.0f && range < INFINITY) ? (float)(BINS - 1) / range : 0.0f;
    unsigned from = floor_key, upto = 0xffffffffu;   // keys that are still in question
    bool by_bits = false, limited = !MASS;
    u64 before = 0;                                  // the sum of what lies above them
    u64 width = 0;
    __syncthreads();                                 // what an earlier search found has been read
    for (;;) {
        for (int i = threadIdx.x; i < BINS; i += FILTER_THREADS) { sh->count[i] = 0u; if (MASS) sh->mass[i] = 0ull; }
        if (threadIdx.x == 0) { sh->listed = 0u; sh->found = 0xffffffffu; }
        __syncthreads();
        // 0 for the largest.  Even in logit at first (subtraction, product and conversion keep the order), then by the bits.
        auto bin_of = [&](float v, unsigned key) {
            if (by_bits) return (int)((u64)(upto - key) * BINS / width);
            const float at = (f.top - v) * even;
            return v == f.top ? 0 : (at < (float)(BINS - 1) ? (int)at : BINS - 1);
        };
        for (int i = threadIdx.x; i < n; i += FILTER_THREADS) {
            const float v = clean(x[i]);
            const unsigned key = order_key(v);
            if (key < from || key > upto) continue;
            const int bin = bin_of(v, key);
            atomicAdd(&sh->count[bin], 1u);
            if (MASS) atomicAdd(&sh->mass[bin], f.mass(v));
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
#pragma unroll 8
                for (int c = 0; c < f.ctas; ++c) {
                    const unsigned add = f.cluster.map_shared_rank(sh->count, c)[first + k];
                    counts[k] += add;
                    sums[k] += MASS ? f.cluster.map_shared_rank(sh->mass, c)[first + k] : (u64)add;
                }
            mine += sums[k];
        }
        u64 running = block_before(mine, sh->warp_sums);
        u64 word[2] = {block_fold(mine, sh->warp_sums, add64), 0};
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
            for (int i = threadIdx.x; i < n; i += FILTER_THREADS) {
                const float v = clean(x[i]);
                const unsigned key = order_key(v);
                if (key < from || key > upto || bin_of(v, key) != (int)bin) continue;
                const unsigned at = atomicAdd(&head->listed, 1u);
                head->list_key[at] = key;
                head->list_mass[at] = MASS ? f.mass(v) : 1ull;
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
        for (int i = threadIdx.x; i < n; i += FILTER_THREADS) {
            const float v = clean(x[i]);
            const unsigned key = order_key(v);
            if (key < from || key > upto || bin_of(v, key) != (int)bin) continue;
            least = min(least, key);
            greatest = max(greatest, key);
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
__global__ void __launch_bounds__(FILTER_THREADS)
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
    tt_pdl_wait();
    if (temperatures) temperature = __ldg(temperatures + row);
    if (top_ks) top_k = __ldg(top_ks + row);
    if (top_ps) top_p = __ldg(top_ps + row);
    if (min_ps) min_p = __ldg(min_ps + row);

    // this CTA's slice of the row, and the row's largest and smallest finite logits
    const int lo = f.rank * slice, n = max(0, min(slice, vocab - lo));
    const float* from = logits + (size_t)row * ld + lo;
    float* kept = reinterpret_cast<float*>(filter_memory + sizeof(FilterShared));
    u64* chunks = reinterpret_cast<u64*>(kept + (staged ? (slice + 3) / 4 * 4 : 0));       // sums of 32 neighbouring tokens' weights
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
    u64 word[2] = {block_fold((u64)order_key(most), sh->warp_sums, max64), block_fold((u64)~order_key(least), sh->warp_sums, max64)};
    f.exchange(word, [](u64 (&total)[2], u64 a, u64 b, int) { total[0] = max64(total[0], a); total[1] = max64(total[1], b); });
    auto value_of = [](unsigned key) { return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key); };
    f.top = value_of((unsigned)word[0]);
    const float lowest = value_of(~(unsigned)word[1]);
    // a row that is too long for shared memory is read again by every pass
    const float* x = staged ? kept : from;

    if (f.top == -INFINITY || !(temperature > 0.0f)) {                 // nothing to choose from, or the largest logit's lowest id
        u64 at = ~0ull;
        for (int i = threadIdx.x; i < n; i += FILTER_THREADS)
            if (clean(x[i]) == f.top) { at = (u64)(lo + i); break; }          // a thread's first is its lowest
        word[0] = block_fold(~at, sh->warp_sums, max64);
        word[1] = 0;
        f.exchange(word, [](u64 (&total)[2], u64 a, u64, int) { total[0] = max64(total[0], a); });
        if (f.rank == 0 && threadIdx.x == 0) out[row] = f.top == -INFINITY ? 0 : (int)~word[0];
        f.cluster.sync();                                              // nobody leaves while its words are being read
        return;
    }
    f.inverse = 1.0 / (double)temperature;
    f.inverse32 = f.inverse * 46.166241308446829;                      // 32 / ln 2

    unsigned floor_key = order_key(-INFINITY) + 1;                     // what is minus infinity, or no number, weighs nothing
    if (top_k > 0 && top_k < vocab) floor_key = max(floor_key, search_key<false>(f, x, n, lowest, floor_key, (u64)(top_k - 1), 0.0));
    if (top_p < 1.0f) floor_key = max(floor_key, search_key<true>(f, x, n, lowest, floor_key, 0, (double)top_p));
    // min-p: weights well below it need not be formed
    const double least_weight = (double)fminf(min_p, 1.0f);
    if (least_weight > 0.0 && f.top < INFINITY && temperature < INFINITY) {
        const float below = (float)((double)f.top + (double)temperature * log(least_weight) * 1.0001 - 1e-3 * fabs((double)f.top) - 1e-30);
        floor_key = max(floor_key, order_key(below));
    }
    const double least_units = least_weight * 35184372088832.0;
    auto kept_mass = [&](float v) -> u64 {
        if (!(v > -INFINITY) || order_key(v) < floor_key) return 0ull;
        const double w = f.weight(v);
        return w >= least_units ? Filter::units(w) : 0ull;
    };

    // the kept weights of 32 neighbouring tokens at a time, and of the slice
    u64 mine = 0;
    const int n_chunks = (n + 31) / 32;
    for (int c = warp; c < n_chunks; c += FILTER_WARPS) {
        const int i = 32 * c + lane;
        const u64 m = i < n ? kept_mass(clean(x[i])) : 0ull;
        u64 sum = 0;
        if (__any_sync(0xffffffffu, m != 0ull)) sum = warp_fold(m, add64);
        if (lane == 0) { chunks[c] = sum; mine += sum; }
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
    const float u = uniforms ? __ldg(uniforms + row)
                             : counter_uniform(seed, (u64)(unsigned)__ldg(requests + row), (u64)(unsigned)__ldg(steps + row));
    const double wanted = (double)u * (double)total;
    u64 target = wanted > 0.0 ? (u64)wanted : 0ull;
    target = min(target, total - 1);                                   // a random number of one or more: the last kept token
    if (before <= target && before + own > target) {                   // it is in this slice
        const int each = (n_chunks + FILTER_THREADS - 1) / FILTER_THREADS, first = threadIdx.x * each;
        u64 sum = 0;
        for (int c = first; c < min(first + each, n_chunks); ++c) sum += chunks[c];
        u64 running = before + block_before(sum, sh->warp_sums);
        for (int c = first; c < min(first + each, n_chunks); ++c) {
            if (running <= target && running + chunks[c] > target) { sh->found = (unsigned)c; sh->found_before = running; }
            running += chunks[c];
        }
        __syncthreads();
        if (warp == 0) {
            const int i = 32 * (int)sh->found + lane;
            u64 upto = i < n ? kept_mass(clean(x[i])) : 0ull;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 up = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += up;
            }
            const unsigned past = __ballot_sync(0xffffffffu, sh->found_before + upto > target);
            if (lane == 0) out[row] = lo + 32 * (int)sh->found + __ffs(past) - 1;
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
    if (vocab <= 0 || (!uniforms && (!requests || !steps))) return (int)cudaErrorInvalidValue;
    int sms = 0;
    cudaError_t code = tt_sm_count(&sms);
    if (code != cudaSuccess) return (int)code;
    // CTAs a row: slices of at most 16,384 numbers, so that two CTAs fit an SM; more while SMs are free and slices are not below 2,048
    int ctas = 1;
    while (ctas < MAX_CLUSTER && ((vocab + ctas - 1) / ctas > 16384 || ((long long)rows * ctas * 2 <= sms && vocab / (2 * ctas) >= 2048))) ctas *= 2;
    const int slice = ((vocab + ctas - 1) / ctas + 31) / 32 * 32;
    const int staged = slice <= MAX_SLICE;
    if ((long long)rows * ctas > 0x7fffffff) return (int)cudaErrorInvalidValue;
    const size_t shared = sizeof(FilterShared) + (staged ? (size_t)slice * 4 : 0) + (size_t)(slice / 32) * 8;
    if (shared > 220 * 1024) return (int)cudaErrorInvalidValue;       // a vocabulary of millions
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
