// Sampling from logits (sdy_sample_dev): temperature, top-k, top-p and min-p, then the inverse of
// the running sum at a given uniform number.
//
// All filters keep a prefix of one order: the logits descending, equal ones by index. An entry of
// that order is one 64-bit number, order(i) = key(logit_i) << 32 | ~i, with key the usual
// order-preserving image of a float, so a filter is a lower bound on it ("cut"): top-k's is the k-th
// largest, top-p's the largest c with mass(order >= c) >= top_p * mass. Masses are integers:
// w = exp((l - max) / T) in 64 bits, rounded to 2^-44, so that 400000 of them fit 64 bits and their
// sum does not depend on the order of the additions. A 32-bit weight would be off by 2^-24 of
// itself, enough to move a choice whose uniform number lies next to a border once in some ten
// thousand rows; this leaves 10^-12.
//
// A cluster of up to eight CTAs holds a row in its shared memory, so the row is read once. Every
// thread knows its largest entry. A top-k of up to 512 takes from those a bound that the k-th
// largest is not below (bound_of: at least k / ranks threads of each CTA have an entry so large),
// gathers what is not below it, a little more than k entries, in the first CTA, and finishes there on
// the ranked list, filters, sums and choice. Otherwise a cut is found by a histogram of the row's
// distance from its largest logit (1024 buckets), of numbers for top-k and masses for top-p, merged
// over the cluster; the entries of the bucket where the sum crosses are gathered and ranked in the
// first CTA. A bucket of too many entries is split again by key, one of equal keys by index. Top-k
// comes first, so a top-p after it takes exponentials of the kept entries alone; the last pass forms
// the masses of what is kept in index order and finds the entry at the uniform number. Passes test
// entries against a range of values first, and where few are in it take those one after the other.
//
// Bound by latency for few rows (a cluster barrier, about 0.3 us, after each of three to a dozen
// passes) and by the issue of instructions for many: an exponential is about 25, an addition to a
// bucket 15. Measured: 1 row of 151936, top-k 40 and top-p, 11 us; 64 such rows with filters of
// all kinds 67-70 us (a top-p of the whole row, the longest kind, 25 us alone), 333 of 49152 80 us.
#include "draft.cuh"
#include "sample.cuh"
#include "sardyne_b200.h"

#include <cooperative_groups.h>
#include <float.h>
#include <limits.h>
#include <math.h>

namespace sdy {
namespace cg = cooperative_groups;
namespace {

constexpr int S_THREADS = 512, S_WARPS = S_THREADS / 32;
constexpr int S_MAX_VOCAB = SAMPLE_MAX_VOCAB;
constexpr int S_CLUSTER = 8;                   // CTAs to a row, at most
constexpr int S_BUCKETS = 1024, S_LIST = 1024;  // the list: entries ranked at once
constexpr int S_FEW = 512;                     // a top-k that the first CTA finishes alone, one entry to a thread (1000 so, two to a
                                               // thread: 41 us against 23 for 12 rows, the sums below quadratic)
constexpr double S_SCALE = 32.0;               // buckets per unit of (max - l) / T, for numbers of entries
constexpr int S_STEPS = 16;                    // steps of ln 2 / 256 to a bucket, for masses
constexpr double S_FAR = 31.3;                 // exp(-31.3) 2^44 < 1/2: no mass from here on
constexpr double MASS_ONE = 17592186044416.0;  // 2^44
typedef unsigned long long u64;

__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned key) {
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
__device__ __forceinline__ u64 order_of(float x, int i) { return (u64)key_of(x) << 32 | (unsigned)~i; }
__device__ __forceinline__ float value_of(u64 order) { return value_of((unsigned)(order >> 32)); }
__device__ __forceinline__ int index_of(u64 order) { return (int)~(unsigned)order; }

struct SampleShared {
    unsigned lo[S_BUCKETS], hi[S_BUCKETS];  // this CTA's entries: their number, or mass in two words
    u64 list[S_LIST], sorted[S_LIST];       // first CTA: gathered entries
    unsigned n_list, keep;
    u64 part[S_WARPS + 1];                  // sums per warp, then the CTA's
    u64 all[2][S_CLUSTER];                  // exchanged, by rank; two in turn
    u64 said[2][2];                         // what one CTA tells the others; two in turn
    double power[256];                      // 2^(44 + j/256)
};
__shared__ SampleShared sh;  // (by name, so that accesses are known to be to shared memory)
extern __shared__ __align__(16) uint8_t sample_row[];

// w = exp(x), x = (logit - max) / temperature <= 0, by the table method: y = x 256 / ln 2 = k + f with k
// whole and |f| <= 1/2, and w = 2^(k/256) 2^(f/256), the second factor by its series to f^4 (the rest is
// below 2^-53).
struct Weight {
    float top, far;  // the largest logit; no mass up to `far` (below top)
    double m, by;    // the largest (at most FLT_MAX); 256 / (temperature ln 2)
    static constexpr double MAGIC = 6755399441055744.0;  // 1.5 * 2^52: the sum's low word is the nearest integer
    __device__ __forceinline__ double distance(float v) const { return (double)fminf(v, FLT_MAX) - m; }
    __device__ __forceinline__ int steps(float v) const { return -__double2loint(fma(distance(v), by, MAGIC)); }
    // 2^44 w, and 0 for what rounds to no whole number; -k in `steps`
    __device__ __forceinline__ double scaled(float v, int &steps) const {
        constexpr double C = 0.0027076061740622863;  // ln 2 / 256
        const double d = distance(v), t = fma(d, by, MAGIC), f = fma(d, by, MAGIC - t);
        const int k = __double2loint(t);
        double e = fma(f, C * C * C * C / 24, C * C * C / 6);
        e = fma(e, f, C * C / 2);
        e = fma(e, f, C);
        e = fma(e, f, 1.0) * sh.power[k & 255];
        steps = -k;
        e = __hiloint2double(__double2hiint(e) + ((k & ~255) << 12), __double2loint(e));
        return v > far ? e : 0.0;  // (no branch: a thread's entries go abreast)
    }
    __device__ __forceinline__ double scaled(float v) const {
        int steps;
        return scaled(v, steps);
    }
    __device__ __forceinline__ static u64 whole(double m) {  // nearest integer, below 2^51
        return (u64)__double_as_longlong(m + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
    }
    __device__ __forceinline__ u64 mass(float v) const { return whole(scaled(v)); }
};

// The entries from one on, in their order.
struct Cut {
    float value;
    int index;
    __device__ __forceinline__ bool keeps(float v, int i) const { return v > value || (v == value && i <= index); }
};

template <class T>
struct Sampler {
    static constexpr int V = 16 / sizeof(T);  // entries read at once
    struct alignas(16) Vec {
        T v[V];
    };
    cg::cluster_group cl;
    int n, first;   // this CTA's entries (a multiple of V, the end filled up with -inf), the index of the first
    int rank, ranks, tid, warp, lane;
    Weight weight;
    bool near;      // distances can be taken in 32 bits
    float scale;    // buckets per unit of logit
    int turn = 0, told = 0;

    // Entries i V .. of this CTA, -inf behind its last.
    __device__ __forceinline__ void read(int i, int end, float (&v)[V]) const {
        Vec x;
        if (i < end) x = ((const Vec *)sample_row)[i];
#pragma unroll
        for (int j = 0; j < V; j++) v[j] = i < end ? to_f32(x.v[j]) : -INFINITY;
    }
    // at(values, index here of the first) for all entries, by whole warps, in any order
    template <class At> __device__ __forceinline__ void each(At at) const {
        for (int i = tid; i - lane < n / V; i += S_THREADS) {
            float v[V];
            read(i, n / V, v);
            at(v, i * V);
        }
    }
    // Which of V entries lie in [lo, hi], one bit each.
    __device__ __forceinline__ static unsigned within(const float (&v)[V], float lo, float hi) {
        unsigned mask = 0;
#pragma unroll
        for (int j = 0; j < V; j++) mask |= v[j] >= lo && v[j] <= hi ? 1u << j : 0u;
        return mask;
    }
    // Of `mask`, the entries from index i here on, what `cut` keeps (it holds none below the cut's value).
    __device__ __forceinline__ unsigned kept(const Cut &cut, const float (&v)[V], int i, unsigned mask) const {
        if (cut.index < INT_MAX)
#pragma unroll
            for (int j = 0; j < V; j++)
                if (v[j] == cut.value && first + i + j > cut.index) mask &= ~(1u << j);
        return mask;
    }
    // f(value) for the entries of `mask`, a lane's own of the V from index i on, by whole warps: few of them
    // one after the other, each lane at its next (f's second argument: whether it has one).
    template <class F> __device__ __forceinline__ void few_of(unsigned mask, int most, int i, F f) const {
        for (int k = 0; k < most; k++, mask &= mask - 1)
            f(mask ? to_f32(((const T *)sample_row)[i + __ffs(mask) - 1]) : weight.top, mask != 0);
    }
    // The values that can be in bucket b (and a few around): what is outside need not be placed.
    template <bool MASS> __device__ __forceinline__ void bucket_range(int b, float &lo, float &hi) const {
        if (MASS) {
            lo = __double2float_rd(weight.m - (S_STEPS * b + S_STEPS) / weight.by);
            hi = b ? __double2float_ru(weight.m - (S_STEPS * b - 1) / weight.by) : INFINITY;
            return;
        }
        const float slack = 1e-6f * (fabsf(weight.top) + (b + 1) / scale);
        lo = near && b < S_BUCKETS - 1 ? weight.top - (b + 0.51f) / scale - slack : -FLT_MAX;
        hi = near ? weight.top - (b - 0.51f) / scale + slack : INFINITY;
    }
    // Buckets by distance from the largest: for masses by the steps of the exponential, for numbers in 32
    // bits where the range allows it, the last one from 32 units on.
    template <bool MASS> __device__ __forceinline__ int bucket(float v) const {
        if (MASS) return (int)((unsigned)weight.steps(v) / S_STEPS);
        const float x = near ? (weight.top - v) * scale : (float)fmin(-weight.distance(v) * weight.by * (S_SCALE * 0.0027076061740622863), 1e6);
        const int b = (int)(__float_as_uint(fminf(x, S_BUCKETS - 1.0f) + 8388608.0f) & (S_BUCKETS - 1));
        return v == weight.top ? 0 : b;
    }

    // v summed over the threads of the CTA up to and with this one; the CTA's sum in sh.part[S_WARPS].
    __device__ u64 scan(u64 v) {
        u64 in = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 u = __shfl_up_sync(~0u, in, o);
            if (lane >= o) in = in + u;
        }
        __syncthreads();
        if (lane == 31) sh.part[warp] = in;
        __syncthreads();
        u64 below = 0, total = 0;
#pragma unroll
        for (int w = 0; w < S_WARPS; w++) {
            if (w < warp) below += sh.part[w];
            total += sh.part[w];
        }
        if (tid == 0) sh.part[S_WARPS] = total;
        return below + in;
    }
    // One number of every CTA, sh.part[S_WARPS], to all: in sh.all[the result].
    __device__ int gather_sums() {
        __syncthreads();
        if (tid < ranks) cl.map_shared_rank(&sh, tid)->all[turn][rank] = sh.part[S_WARPS];
        cl.sync();
        turn ^= 1;
        return turn ^ 1;
    }
    // The sums of the CTAs of lower rank and of all.
    __device__ void exchange(u64 &before, u64 &total) {
        const int at = gather_sums();
        before = total = 0;
        for (int r = 0; r < ranks; r++) {
            if (r < rank) before += sh.all[at][r];
            total += sh.all[at][r];
        }
    }
    // Two numbers from the one thread in the cluster whose `mine` is set, to all; its warp stores them.
    __device__ void tell(bool mine, u64 a, u64 b, u64 (&got)[2]) {
        const unsigned who = __ballot_sync(~0u, mine);
        if (who) {
            a = __shfl_sync(~0u, a, __ffs(who) - 1);
            b = __shfl_sync(~0u, b, __ffs(who) - 1);
            if (lane / 2 < ranks) cl.map_shared_rank(&sh, lane / 2)->said[told][lane % 2] = lane % 2 ? b : a;
        }
        cl.sync();
        got[0] = sh.said[told][0], got[1] = sh.said[told][1];
        told ^= 1;
    }
    // The entries in [lo, hi] that `cut` keeps and in(value) holds for, added to the first CTA's list: a
    // warp's together. Their number, in all CTAs; what is behind S_LIST is not in the list.
    template <class In> __device__ unsigned gather(float lo, float hi, const Cut &cut, In in) {
        SampleShared *lead = cl.map_shared_rank(&sh, 0);
        each([&](const float(&v)[V], int i) {
            unsigned mask = kept(cut, v, i, within(v, lo, hi));
            if (!__any_sync(~0u, mask)) return;
            for (unsigned m = mask; m; m &= m - 1)
                if (!in(to_f32(((const T *)sample_row)[i + __ffs(m) - 1]))) mask ^= m & -m;
            int at = __popc(mask);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(~0u, at, o);
                if (lane >= o) at += u;
            }
            unsigned from = lane == 31 && at ? atomicAdd(&lead->n_list, (unsigned)at) : 0;
            from = __shfl_sync(~0u, from, 31) + at - __popc(mask);
            for (; mask && from < S_LIST; mask &= mask - 1, from++) {
                const int j = i + __ffs(mask) - 1;
                lead->list[from] = order_of(to_f32(((const T *)sample_row)[j]), first + j);
            }
        });
        cl.sync();
        return lead->n_list;
    }
    // The first CTA's list of m entries in descending order: sorted bitonically, one entry to a thread,
    // or, where there are more, every one counts the ones before it.
    __device__ void rank_list(int m) {
        if (m <= S_THREADS) {
            u64 mine = tid < m ? sh.list[tid] : 0;
            int size = 2;
            for (; size / 2 < m; size *= 2)
                for (int j = size / 2; j; j /= 2) {
                    u64 other;
                    if (j < 32) {
                        other = __shfl_xor_sync(~0u, mine, j);
                    } else {
                        __syncthreads();
                        sh.sorted[tid] = mine;
                        __syncthreads();
                        other = sh.sorted[tid ^ j];
                    }
                    // descending where the run's bit is clear; the lower one of a pair keeps the larger
                    const bool larger = ((tid & size) == 0) == ((tid & j) == 0);
                    mine = larger == (mine > other) ? mine : other;
                }
            __syncthreads();
            sh.sorted[tid] = mine;
        } else {
            for (int i = tid; i < m; i += S_THREADS) {
                const u64 mine = sh.list[i];
                int at = 0;
#pragma unroll 8
                for (int j = 0; j < m; j++) at += sh.list[j] > mine;
                sh.sorted[at] = mine;
            }
        }
        __syncthreads();
    }

    // The index at which the running sum of of(value) over the entries in [lo, hi] that `cut` keeps, in
    // index order, passes want_of(total); the sum of all and the one there in `total` and `at`.
    template <class Of, class W>
    __device__ int locate(float lo, float hi, const Cut &cut, Of of, W want_of, u64 &total, u64 &at) {
        // a warp's entries are a run of indexes, in steps of 32 reads, whose sums it notes
        u64 *steps = sh.sorted + warp * 32;
        const int per = (n / V + S_WARPS - 1) / S_WARPS, i0 = min(warp * per, n / V), i1 = min(i0 + per, n / V);
        auto vec = [&](int i) -> u64 {  // by whole warps
            float v[V];
            read(i, i1, v);
            const unsigned mask = kept(cut, v, i * V, within(v, lo, hi));
            const int most = __reduce_max_sync(~0u, __popc(mask));
            u64 sum = 0;
            if (2 * most <= V) {
                few_of(mask, most, i * V, [&](float x, bool has) {
                    const u64 m = of(x);
                    sum += has ? m : 0;
                });
            } else {
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const u64 m = of(v[j]);
                    sum += mask >> j & 1 ? m : 0;
                }
            }
            return sum;
        };
        __syncthreads();  // (sh.sorted has been read)
        u64 mine = 0;
        for (int i = i0, k = 0; i < i1; i += 32, k++) {
            u64 m = vec(i + lane);
            if (__any_sync(~0u, m != 0))
#pragma unroll
                for (int o = 16; o; o >>= 1) m += __shfl_xor_sync(~0u, m, o);
            mine += m;
            if (lane == 0) steps[k] = m;
        }
        const u64 to = scan(lane == 31 ? mine : 0);
        u64 before;
        exchange(before, total);
        const u64 want = want_of(total), end = before + __shfl_sync(~0u, to, 31), begin = end - mine;
        bool here = false;
        u64 v[2] = {0, 0};
        if (want >= begin && want < end) {
            auto prefix = [&](u64 m) {
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const u64 u = __shfl_up_sync(~0u, m, o);
                    if (lane >= o) m += u;
                }
                return m;
            };
            // the step, the read, the entry
            const u64 step = lane * 32 < i1 - i0 ? steps[lane] : 0, upto = prefix(step);
            const int k = __ffs(__ballot_sync(~0u, want < begin + upto)) - 1;
            u64 c = begin + __shfl_sync(~0u, upto - step, k);
            const int i = i0 + 32 * k + lane;
            const u64 m = vec(i), to_here = prefix(m);
            here = lane == __ffs(__ballot_sync(~0u, want < c + to_here)) - 1;
            if (here) {
                c += to_here - m;
                for (int j = i * V;; j++) {
                    const float x = to_f32(((const T *)sample_row)[j]);
                    const u64 one = x >= lo && x <= hi && cut.keeps(x, first + j) ? of(x) : 0;
                    if (want < c + one) {
                        v[0] = first + j, v[1] = one;
                        break;
                    }
                    c += one;
                }
            }
            __syncwarp();
        }
        u64 got[2];
        tell(here, v[0], v[1], got);
        at = got[1];
        return (int)got[0];
    }

    // The shortest prefix of the entries that `cut` keeps whose number (MASS: mass) reaches
    // target_of(the sum of all of them).
    // bound: a value that the result is not below.
    template <bool MASS, class Target>
    __device__ Cut find_cut(Cut cut, float bound, Target target_of) {
        float v_hi = weight.top, v_lo = fmaxf(cut.value, bound);  // the values in question
        if (MASS) v_lo = fmaxf(v_lo, nextafterf(weight.far, INFINITY));
        unsigned k_hi = 0;                         // key of v_hi, and buckets by key >> shift from it
        int shift = -1;                            // (at first, buckets by distance)
        u64 done = 0, target = 0;                  // the sum before them; the one to reach
        while (true) {
            auto place = [&](float v) { return shift < 0 ? bucket<MASS>(v) : (int)((k_hi - key_of(v)) >> shift); };
            for (int b = tid; b < S_BUCKETS; b += S_THREADS) sh.lo[b] = sh.hi[b] = 0;
            if (tid == 0) sh.n_list = 0;
            __syncthreads();
            unsigned far = 0;  // by distance, the last bucket has most entries
            each([&](const float(&v)[V], int i) {
                const unsigned mask = kept(cut, v, i, within(v, v_lo, v_hi));
                const int most = __reduce_max_sync(~0u, __popc(mask));
                auto add = [&](bool has, int b, u64 m) {
                    if (MASS) {
                        if (!has) return;
                        const unsigned low = (unsigned)m, old = atomicAdd(&sh.lo[b], low);
                        const unsigned high = (unsigned)(m >> 32) + (old + low < low);
                        if (high) atomicAdd(&sh.hi[b], high);
                    } else {
                        const bool last = shift < 0 && b == S_BUCKETS - 1;
                        far += has && last;
                        if (has && !last) atomicAdd(&sh.lo[b], 1u);
                    }
                };
                auto both = [&](float x, int &b) -> u64 {
                    if (!MASS) return b = place(x), 1;
                    int steps;
                    const u64 m = Weight::whole(weight.scaled(x, steps));
                    b = shift < 0 ? (int)((unsigned)steps / S_STEPS) : place(x);
                    return m;
                };
                if (2 * most <= V) {
                    few_of(mask, most, i, [&](float x, bool has) {
                        int b;
                        const u64 m = both(x, b);
                        add(has, b, m);
                    });
                    return;
                }
                int b[V];
                u64 m[V];
#pragma unroll
                for (int j = 0; j < V; j++) m[j] = both(v[j], b[j]);
#pragma unroll
                for (int j = 0; j < V; j++) add(mask >> j & 1, b[j], m[j]);
            });
            if (!MASS) {
                for (int o = 16; o; o >>= 1) far += __shfl_xor_sync(~0u, far, o);
                if (lane == 0 && far) atomicAdd(&sh.lo[S_BUCKETS - 1], far);
            }
            cl.sync();
            // this CTA merges a run of buckets, two to a thread at most
            const int run = S_BUCKETS / ranks, per = (run + S_THREADS - 1) / S_THREADS, b0 = rank * run + tid * per;
            u64 own[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < 2; j++)
                if (j < per && tid * per + j < run)
                    for (int r = 0; r < ranks; r++) {
                        const SampleShared *o = cl.map_shared_rank(&sh, r);
                        own[j] += MASS ? (u64)o->hi[b0 + j] << 32 | o->lo[b0 + j] : o->lo[b0 + j];
                    }
            u64 c = scan(own[0] + own[1]), before, total;
            exchange(before, total);
            if (shift < 0) target = target_of(total);
            // the bucket in which the sum reaches the target
            c += done + before - own[0] - own[1];
            const bool one = c < target && target <= c + own[0], two = c + own[0] < target && target <= c + own[0] + own[1];
            u64 got[2];
            tell(one || two, b0 + two, two ? c + own[0] : c, got);
            const int crossing = (int)got[0];
            done = got[1];
            float lo_v = v_lo, hi_v = v_hi;
            if (shift < 0) bucket_range<MASS>(crossing, lo_v, hi_v);
            lo_v = fmaxf(lo_v, v_lo), hi_v = fminf(hi_v, v_hi);
            auto crosses = [&](float x) { return place(x) == crossing; };
            const unsigned m = gather(lo_v, hi_v, cut, crosses);
            if (m <= S_LIST) {  // ranked in the first CTA
                bool found = false;
                u64 w = 0;
                if (rank == 0) {
                    rank_list((int)m);
                    const unsigned i = 2 * tid;
                    const u64 e0 = i < m ? MASS ? weight.mass(value_of(sh.sorted[i])) : 1 : 0;
                    const u64 e1 = i + 1 < m ? MASS ? weight.mass(value_of(sh.sorted[i + 1])) : 1 : 0;
                    const u64 second = done + scan(e0 + e1), first_ = second - e1, none = first_ - e0;
                    found = none < target && target <= second;
                    if (found) w = sh.sorted[i + (first_ < target)];
                }
                tell(found, w, 0, got);
                return {value_of(got[0]), index_of(got[0])};
            }
            // too many for the list: the range of their keys into buckets again
            unsigned lo = ~0u, hi = 0;
            each([&](const float(&v)[V], int i) {
                for (unsigned mask = kept(cut, v, i, within(v, lo_v, hi_v)); mask; mask &= mask - 1) {
                    const float x = to_f32(((const T *)sample_row)[i + __ffs(mask) - 1]);
                    if (crosses(x)) lo = min(lo, key_of(x)), hi = max(hi, key_of(x));
                }
            });
            for (int o = 16; o; o >>= 1) {
                lo = min(lo, __shfl_xor_sync(~0u, lo, o));
                hi = max(hi, __shfl_xor_sync(~0u, hi, o));
            }
            __syncthreads();
            if (lane == 0) sh.part[warp] = (u64)lo << 32 | hi;
            __syncthreads();
            if (tid == 0) {
                for (int j = 1; j < S_WARPS; j++) lo = min(lo, (unsigned)(sh.part[j] >> 32)), hi = max(hi, (unsigned)sh.part[j]);
                sh.part[S_WARPS] = (u64)lo << 32 | hi;
            }
            const int at = gather_sums();
            lo = ~0u, hi = 0;
            for (int r = 0; r < ranks; r++) lo = min(lo, (unsigned)(sh.all[at][r] >> 32)), hi = max(hi, (unsigned)sh.all[at][r]);
            v_lo = value_of(lo), v_hi = value_of(hi);
            if (lo == hi) {  // equal ones: so many, by index
                const u64 size = MASS ? weight.mass(v_lo) : 1, need = (target - done + size - 1) / size;
                u64 total_, at_;
                const int i = locate(v_lo, v_lo, cut, [](float) -> u64 { return 1; }, [&](u64) { return need - 1; }, total_, at_);
                return {v_lo, i};
            }
            k_hi = hi;
            for (shift = 0; (hi - lo) >> shift >= S_BUCKETS;) shift++;
        }
    }

    // A value that the k-th largest entry of the row is not below, for k up to S_THREADS a CTA: with the
    // largest of every thread (`largest`) at hand, each CTA takes the bucket of its ceil(k / ranks)-th
    // largest of them, and the furthest of these buckets holds, with those before it, k entries at least.
    __device__ float bound_of(float largest, int k) {
        for (int b = tid; b < S_BUCKETS; b += S_THREADS) sh.lo[b] = 0;
        if (tid == 0) sh.n_list = 0, sh.keep = S_BUCKETS - 1;
        __syncthreads();
        if (largest > -INFINITY) atomicAdd(&sh.lo[bucket<false>(largest)], 1u);
        __syncthreads();
        const int a = sh.lo[2 * tid], b = sh.lo[2 * tid + 1], share = (k + ranks - 1) / ranks;
        const int to = (int)scan(a + b);
        if (to - (a + b) < share && to >= share) sh.keep = 2 * tid + (to - b < share);
        __syncthreads();
        if (tid == 0) sh.part[S_WARPS] = sh.keep;
        const int at = gather_sums();
        int bound = 0;
        for (int r = 0; r < ranks; r++) bound = max(bound, (int)sh.all[at][r]);
        float lo, hi;
        bucket_range<false>(bound, lo, hi);
        return lo;
    }

    // A top-k of at most S_FEW, finished in the first CTA: what is not below `bound` (bound_of) is
    // gathered, and the rest is work on a short list. False, in all CTAs, where the list would be too
    // long; true with the token in `id` (first CTA, one thread; else -1).
    __device__ bool few(float bound, int k, float top_p, double min_w, float u, int &id, float &prob) {
        const int m = (int)min(gather(bound, INFINITY, {-FLT_MAX, INT_MAX}, [](float) { return true; }), S_LIST + 1u);
        cl.sync();  // (read by all: the first CTA may write it again, or leave)
        if (m > S_LIST) return false;
        id = -1;
        if (rank) return true;
        rank_list(m);
        // number of entries kept, of the masses in descending order
        const int kept_k = min(k, m);
        const double w = tid < kept_k ? weight.scaled(value_of(sh.sorted[tid])) : 0.0;
        const u64 mass = Weight::whole(w);
        if (tid == 0) sh.keep = kept_k;
        const u64 upto = scan(mass);
        __syncthreads();
        const u64 all = sh.part[S_WARPS];
        if (top_p < 1.0f) {
            const u64 target = max((u64)ceil(max((double)top_p, 0.0) * (double)all), (u64)1);
            if (upto - mass < target && target <= upto) atomicMin(&sh.keep, (unsigned)tid + 1);
        }
        if (tid > 0 && tid < kept_k && w < min_w * MASS_ONE) atomicMin(&sh.keep, (unsigned)tid);
        __syncthreads();
        const int keep = (int)sh.keep;
        if (tid == keep - 1) sh.part[S_WARPS] = upto;
        u64 *masses = sh.list;
        if (tid < keep) masses[tid] = mass;
        __syncthreads();
        const u64 total = sh.part[S_WARPS];
        const double at_u = (u > 0.0f ? (double)u : 0.0) * (double)total;
        const u64 want = at_u >= (double)total ? total - 1 : (u64)at_u;
        if (tid < keep) {
            const u64 mine = sh.sorted[tid];
            u64 below = 0;
#pragma unroll 8
            for (int j = 0; j < keep; j++) below += (unsigned)sh.sorted[j] > (unsigned)mine ? masses[j] : 0;  // (~index)
            if (below <= want && want < below + mass) id = index_of(mine), prob = (float)((double)mass / (double)total);
        }
        return true;
    }
};

template <class T>
__global__ void __launch_bounds__(S_THREADS, 2) sample_kernel(const sdy_sample_args p, int per) {
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n" ::: "memory");  // (the CTAs of the row have begun)
    pdl_wait();
    using S = Sampler<T>;
    const cg::cluster_group cl = cg::this_cluster();
    const int ranks = cl.num_blocks(), rank = cl.block_rank(), tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const int64_t row = blockIdx.x / ranks;
    constexpr int V = S::V;
    const int first = min(rank * per, p.n_vocab), n = min(per, p.n_vocab - first), full = (n + V - 1) / V * V;
    const T *x = (const T *)p.logits + row * p.row_stride + first;
    if (tid < 256) sh.power[tid] = exp2(44 + tid / 256.0);

    // The row into shared memory (NaN as -inf, -0 as 0), and its largest entry: each thread meets its
    // own in rising order, so the first of equal ones stays.
    float largest = -INFINITY;
    int where = 0;
    auto take = [&](T t, int i) {
        const float v = to_f32(t) + 0.0f;
        if (v > largest) largest = v, where = i;
        return from_f32<T>(v != v ? -INFINITY : v);
    };
    const int vec = (uintptr_t)x % 16 == 0 ? n / V : 0;
#pragma unroll 4
    for (int i = tid; i < vec; i += S_THREADS) {
        typename S::Vec r = ((const typename S::Vec *)x)[i];
#pragma unroll
        for (int j = 0; j < V; j++) r.v[j] = take(r.v[j], i * V + j);
        ((typename S::Vec *)sample_row)[i] = r;
    }
#pragma unroll 4
    for (int i = vec * V + tid; i < full; i += S_THREADS) ((T *)sample_row)[i] = take(i < n ? x[i] : from_f32<T>(-INFINITY), i);
    u64 best = order_of(largest, first + where);
    for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(~0u, best, o));
    if (lane == 0) sh.part[warp] = best;
    __syncthreads();
    asm volatile("barrier.cluster.wait.aligned;\n" ::: "memory");
    if (tid < ranks) {
        for (int j = 0; j < S_WARPS; j++) best = max(best, sh.part[j]);
        cl.map_shared_rank(&sh, tid)->all[1][rank] = best;
    }
    cl.sync();
    best = 0;
    for (int r = 0; r < ranks; r++) best = max(best, sh.all[1][r]);

    const float top = value_of(best);
    const float temp = p.temperature ? p.temperature[row] : 1.0f;
    if (top == -INFINITY || !(temp > 0.0f)) {
        if (rank == 0 && tid == 0) {
            p.id[row] = top == -INFINITY ? -1 : index_of(best);
            if (p.prob) p.prob[row] = top == -INFINITY ? 0.0f : 1.0f;
        }
        return;  // (nobody reads this CTA's shared memory any more)
    }
    // (an infinite largest logit: the others are infinitely far whatever the temperature)
    const double t = isinf(top) ? 1.0 : (double)temp, m = (double)fminf(top, FLT_MAX);
    const Weight weight{top, fminf(__double2float_rd(m - S_FAR * t), nextafterf(top, -INFINITY)), m, 369.32993046757463 / t};  // 256 / ln 2
    // where no difference nor quotient that matters leaves the range of 32 bits
    const bool near = fabsf(top) < 1e37f && temp > 1e-30f && temp < 1e30f;
    S s{cl, full, first, rank, ranks, tid, warp, lane, weight, near, (float)(S_SCALE / t)};
    const int k = p.top_k ? p.top_k[row] : 0;
    const float top_p = p.top_p ? p.top_p[row] : 1.0f, u = p.u[row];
    double min_w = p.min_p ? (double)p.min_p[row] : 0.0;
    min_w = min_w != min_w ? 0.0 : min(min_w, 1.0);
    int id;
    Cut cut = {-FLT_MAX, INT_MAX};  // every finite entry and +inf
    if (k > 0 && k < p.n_vocab) {
        const float bound = k <= S_THREADS * ranks ? s.bound_of(largest, k) : -FLT_MAX;
        float prob;
        if (k <= S_FEW && s.few(bound, k, top_p, min_w, u, id, prob)) {
            if (id >= 0) {
                p.id[row] = id;
                if (p.prob) p.prob[row] = prob;
            }
            return;
        }
        cut = s.template find_cut<false>(cut, bound, [&](u64 all) { return min((u64)k, all); });
    }
    if (top_p < 1.0f)
        cut = s.template find_cut<true>(cut, -FLT_MAX, [&](u64 all) {
            return max((u64)ceil(max((double)top_p, 0.0) * (double)all), (u64)1);
        });
    // what is too far for min_p (or for any mass) needs no exponential
    float low = __double2float_rd(m - ((min_w > 0.0 ? fmin(S_FAR, -log(min_w)) : S_FAR) * 1.001 + 1e-9) * t);
    low = fmaxf(low, cut.value);
    u64 total, mass;
    id = s.locate(
        low, INFINITY, cut,
        [&](float v) -> u64 {
            const double w = weight.scaled(v);
            return w >= min_w * MASS_ONE ? Weight::whole(w) : 0;
        },
        [&](u64 all) {
            const double at = (u > 0.0f ? (double)u : 0.0) * (double)all;
            return at >= (double)all ? all - 1 : (u64)at;
        },
        total, mass);
    if (rank == 0 && tid == 0) {
        p.id[row] = id;
        if (p.prob) p.prob[row] = (float)((double)mass / (double)total);
    }
}

bool sample_check(const sdy_sample_args *a) {
    const char *fn = "sdy_sample_dev";
    const char *bad = nullptr;
    if (!a) bad = "no argument block";
    else if (a->type != T_F32 && a->type != T_F16 && a->type != T_BF16) bad = "type is not F32, F16 or BF16";
    else if (a->n_row < 0 || a->n_row > 1 << 24) bad = "bad counts";
    else if (a->n_vocab < 1 || a->n_vocab > S_MAX_VOCAB) bad = "n_vocab outside [1, 400000]";
    else if (!strides_fit({a->row_stride})) bad = "negative stride";
    else if (a->n_row && (!a->logits || !a->u || !a->id)) bad = "logits, u or id missing";
    else if ((uintptr_t)a->logits % value_bytes(a->type) ||
             ((uintptr_t)a->temperature | (uintptr_t)a->top_k | (uintptr_t)a->top_p | (uintptr_t)a->min_p |
              (uintptr_t)a->u | (uintptr_t)a->id | (uintptr_t)a->prob) % 4)
        bad = "a pointer is not aligned to its type";
    if (bad) {
        set_error("%s: %s", fn, bad);
        return false;
    }
    if (!a->n_row) return true;
    return device_pointers(fn, {{"logits", a->logits}, {"u", a->u}, {"id", a->id}, {"temperature", a->temperature}, {"top_k", a->top_k}, {"top_p", a->top_p}, {"min_p", a->min_p}, {"prob", a->prob}});
}

}  // namespace

// CTAs to a row: as few as hold it; more while all stay within one to an SM, and, where two would not
// share an SM, within eight. Measured with 1, 2, 4 and 8 to a row (us): 64 rows of 6000, top-k 40 and
// top-p, 9.4, 9.3, 11.6, 21.3; 128 rows 9.4, 11.9, 20.2, 35.8; 8 rows of 49152 with filters of all kinds
// 64, 44, 33, 28; 333 rows of 49152, bf16, 91, 80, 98, 155; 64 rows of 151936, bf16, 98 with 2, 72
// with 4, 63 with 8.
template <class T>
void sample_launch(const sdy_sample_args &a, cudaStream_t s) {
    constexpr int64_t ROOM = 196 * 1024, PAIR = 86 * 1024;  // beside the static shared memory: of one CTA in an SM, of two
    int ranks = 1;
    while (ranks < S_CLUSTER) {
        const int64_t part = (int64_t)(a.n_vocab * sizeof(T)) / ranks;
        if (part <= ROOM && (int64_t)a.n_row * ranks * 2 > (part > PAIR ? 8 * 148 : 148)) break;
        ranks *= 2;
    }
    const int per = ((a.n_vocab + ranks - 1) / ranks + 15) / 16 * 16;
    static std::atomic<uint64_t> done{0};
    smem_limit_once(sample_kernel<T>, (int)ROOM, done);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled();
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ranks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.n_row * ranks));
    cfg.blockDim = dim3(S_THREADS);
    cfg.dynamicSmemBytes = per * sizeof(T);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    SDY_CUDA(cudaLaunchKernelEx(&cfg, sample_kernel<T>, a, per));
    SDY_LAUNCHED();
}

void sample_rows(const sdy_sample_args &a, cudaStream_t s) {
    if (a.type == T_F32) sample_launch<float>(a, s);
    else if (a.type == T_F16) sample_launch<__half>(a, s);
    else sample_launch<__nv_bfloat16>(a, s);
}

}  // namespace sdy

using namespace sdy;

extern "C" int sdy_sample_dev(const sdy_sample_args *a, void *stream) {
    clear_error();
    if (!sample_check(a)) return -1;
    if (!a->n_row) return 0;
    sample_rows(*a, (cudaStream_t)stream);
    return last_error()[0] ? -1 : 0;
}
