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
// A cluster of up to eight CTAs holds a row in its shared memory, so the row is read once. A cut is
// found by a histogram of the row's distance from its largest logit (1024 buckets of 1/32, in units
// of the temperature), of numbers for top-k and masses for top-p, merged over the cluster; the
// entries of the bucket where the count crosses are gathered and ranked in the first CTA. A bucket of
// too many entries is split again by key, one of equal keys by index. Top-k comes first, so a top-p
// after it takes exponentials of the kept entries alone; the last pass forms the masses of what is
// kept in index order and finds the entry at the uniform number.
//
// Bound by latency for few rows (a dozen cluster barriers and passes over shared memory), for many by
// the exponentials (64 bits: about 20 operations at half the 32-bit rate) and the passes.
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
constexpr int S_FEW = 512;                     // a top-k that the first CTA finishes alone, one entry to a thread
constexpr double S_SCALE = 32.0;               // buckets per unit of (max - l) / T
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

struct Sum {
    u64 count, mass;
    __device__ Sum operator+(const Sum &o) const { return {count + o.count, mass + o.mass}; }
};
__device__ __forceinline__ Sum shfl_up(Sum v, int o) { return {__shfl_up_sync(~0u, v.count, o), __shfl_up_sync(~0u, v.mass, o)}; }

struct SampleShared {
    unsigned count[S_BUCKETS], lo[S_BUCKETS], hi[S_BUCKETS];  // of this CTA's entries (mass in two words)
    u64 list[S_LIST], sorted[S_LIST];                         // first CTA: gathered entries
    unsigned n_list, keep;
    Sum part[S_WARPS + 1];                                    // per warp, then the CTA
    Sum all[2][S_CLUSTER];                                    // exchanged, by rank; two in turn
    u64 said[2][4];                                           // what one CTA tells the others; two in turn
    double power[256];                                        // 2^(j/256)
};
__shared__ SampleShared sh;  // (by name, so that accesses are known to be to shared memory)
extern __shared__ __align__(16) uint8_t sample_row[];

// w = exp(x), x = (logit - max) / temperature <= 0, by the table method: y = x 256 / ln 2 = k + f with k
// whole and |f| <= 1/2, and w = 2^(k/256) 2^(f/256), the second factor by its series to f^4 (the rest is
// below 2^-53).
struct Weight {
    float top;          // the largest logit
    double m, inv, by;  // the same; 1 / temperature; 256 / (temperature ln 2)
    // 2^44 w, and 0 for what rounds to no whole number
    __device__ __forceinline__ double scaled(float v) const {
        constexpr double MAGIC = 6755399441055744.0;  // 1.5 * 2^52: the sum's low word is the nearest integer
        constexpr double C = 0.0027076061740622863;   // ln 2 / 256
        const double d = (double)v - m;
        const double t = fma(d, by, MAGIC), kd = t - MAGIC, f = fma(d, by, -kd);
        const int k = __double2loint(t);
        double e = fma(f, C * C * C * C / 24, C * C * C / 6);
        e = fma(e, f, C * C / 2);
        e = fma(e, f, C);
        e = fma(e, f, 1.0) * sh.power[k & 255];
        e = __longlong_as_double(__double_as_longlong(e) + ((long long)((k >> 8) + 44) << 52));
        return v == top ? MASS_ONE : d * inv > -S_FAR ? e : 0.0;  // (no branch: a thread's entries go abreast)
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
    __device__ __forceinline__ void bucket_range(int b, float &lo, float &hi) const {
        const float slack = 1e-6f * (fabsf(weight.top) + (b + 1) / scale);
        lo = near && b < S_BUCKETS - 1 ? weight.top - (b + 0.51f) / scale - slack : -FLT_MAX;
        hi = near ? weight.top - (b - 0.51f) / scale + slack : INFINITY;
    }
    // Buckets by distance from the largest; the last one's entries have no mass.
    __device__ __forceinline__ int bucket(float v) const {
        const float x = near ? (weight.top - v) * scale : (float)fmin((weight.m - (double)v) * weight.inv * S_SCALE, 1e6);
        const int b = (int)(__float_as_uint(fminf(x, S_BUCKETS - 1.0f) + 8388608.0f) & (S_BUCKETS - 1));
        return v == weight.top ? 0 : b;
    }

    // v summed over the threads of the CTA up to and with this one; the CTA's sum in sh.part[S_WARPS].
    __device__ Sum scan(Sum v) {
        Sum in = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const Sum u = shfl_up(in, o);
            if (lane >= o) in = in + u;
        }
        __syncthreads();
        if (lane == 31) sh.part[warp] = in;
        __syncthreads();
        Sum below = {0, 0}, total = {0, 0};
#pragma unroll
        for (int w = 0; w < S_WARPS; w++) {
            if (w < warp) below = below + sh.part[w];
            total = total + sh.part[w];
        }
        if (tid == 0) sh.part[S_WARPS] = total;
        return below + in;
    }
    // One Sum of every CTA, sh.part[S_WARPS], to all: in sh.all[the result].
    __device__ int gather_sums() {
        __syncthreads();
        if (tid < ranks) cl.map_shared_rank(&sh, tid)->all[turn][rank] = sh.part[S_WARPS];
        cl.sync();
        turn ^= 1;
        return turn ^ 1;
    }
    // The sums of the CTAs of lower rank and of all.
    __device__ void exchange(Sum &before, Sum &total) {
        const int at = gather_sums();
        before = total = {0, 0};
        for (int r = 0; r < ranks; r++) {
            if (r < rank) before = before + sh.all[at][r];
            total = total + sh.all[at][r];
        }
    }
    // Four numbers from the one thread in the cluster whose `mine` is set, to all; its warp stores them.
    __device__ void tell(bool mine, const u64 (&v)[4], u64 (&got)[4]) {
        const unsigned who = __ballot_sync(~0u, mine);
        if (who) {
            u64 word = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const u64 x = __shfl_sync(~0u, v[i], __ffs(who) - 1);
                if (lane % 4 == i) word = x;
            }
            if (lane / 4 < ranks) cl.map_shared_rank(&sh, lane / 4)->said[told][lane % 4] = word;
        }
        cl.sync();
#pragma unroll
        for (int i = 0; i < 4; i++) got[i] = sh.said[told][i];
        told ^= 1;
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
        const Sum to = scan({0, lane == 31 ? mine : 0});
        Sum before, sum;
        exchange(before, sum);
        total = sum.mass;
        const u64 want = want_of(total), end = before.mass + __shfl_sync(~0u, to.mass, 31), begin = end - mine;
        bool here = false;
        u64 v[4] = {0, 0, 0, 0};
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
        u64 got[4];
        tell(here, v, got);
        at = got[1];
        return (int)got[0];
    }

    // The shortest prefix of the entries that `cut` keeps whose number (MASS: mass) reaches
    // target_of(the sum of all of them).
    // bound: a value that the result is not below.
    template <bool MASS, class Target>
    __device__ Cut find_cut(Cut cut, float bound, Target target_of) {
        float v_hi = weight.top, v_lo = fmaxf(cut.value, bound);  // the values in question
        unsigned k_hi = 0;                         // key of v_hi, and buckets by key >> shift from it
        int shift = -1;                            // (at first, buckets by distance)
        Sum done = {0, 0};                         // before them
        u64 target = 0;
        while (true) {
            auto place = [&](float v) { return shift < 0 ? bucket(v) : (int)((k_hi - key_of(v)) >> shift); };
            for (int b = tid; b < S_BUCKETS; b += S_THREADS) sh.count[b] = sh.lo[b] = sh.hi[b] = 0;
            if (tid == 0) sh.n_list = 0;
            __syncthreads();
            unsigned far = 0;  // by distance, the last bucket has most entries (and none of them mass)
            each([&](const float(&v)[V], int i) {
                const unsigned mask = kept(cut, v, i, within(v, v_lo, v_hi));
                const int most = __reduce_max_sync(~0u, __popc(mask));
                auto count = [&](bool has, int b, u64 m) {
                    const bool last = shift < 0 && b == S_BUCKETS - 1;
                    far += has && last;
                    if (!has || last) return;
                    atomicAdd(&sh.count[b], 1u);
                    if (MASS) {
                        const unsigned low = (unsigned)m, old = atomicAdd(&sh.lo[b], low);
                        const unsigned high = (unsigned)(m >> 32) + (old + low < low);
                        if (high) atomicAdd(&sh.hi[b], high);
                    }
                };
                if (2 * most <= V) {
                    few_of(mask, most, i, [&](float x, bool has) { count(has, place(x), MASS ? weight.mass(x) : 0); });
                    return;
                }
                int b[V];
                u64 m[V];
#pragma unroll
                for (int j = 0; j < V; j++) b[j] = place(v[j]), m[j] = MASS ? weight.mass(v[j]) : 0;
#pragma unroll
                for (int j = 0; j < V; j++) count(mask >> j & 1, b[j], m[j]);
            });
            for (int o = 16; o; o >>= 1) far += __shfl_xor_sync(~0u, far, o);
            if (lane == 0 && far) atomicAdd(&sh.count[S_BUCKETS - 1], far);
            cl.sync();
            // this CTA merges a run of buckets, two to a thread at most
            const int run = S_BUCKETS / ranks, per = (run + S_THREADS - 1) / S_THREADS, b0 = rank * run + tid * per;
            Sum own[2] = {{0, 0}, {0, 0}};
#pragma unroll
            for (int j = 0; j < 2; j++)
                if (j < per && tid * per + j < run)
                    for (int r = 0; r < ranks; r++) {
                        const SampleShared *o = cl.map_shared_rank(&sh, r);
                        own[j].count += o->count[b0 + j];
                        if (MASS) own[j].mass += (u64)o->hi[b0 + j] << 32 | o->lo[b0 + j];
                    }
            const Sum to = scan(own[0] + own[1]);
            Sum before, total;
            exchange(before, total);
            if (shift < 0) target = target_of(total);
            // the bucket in which the sum reaches the target
            bool here = false;
            u64 v[4] = {0, 0, 0, 0};
            Sum c = done + before + to;
            c = {c.count - own[0].count - own[1].count, c.mass - own[0].mass - own[1].mass};
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const u64 from = MASS ? c.mass : c.count;
                const Sum next = c + own[j];
                if (!here && from < target && target <= (MASS ? next.mass : next.count)) {
                    here = true;
                    v[0] = b0 + j, v[1] = c.count, v[2] = c.mass, v[3] = own[j].count;
                }
                c = next;
            }
            u64 got[4];
            tell(here, v, got);
            const int crossing = (int)got[0];
            done = {got[1], got[2]};
            float lo_v = v_lo, hi_v = v_hi;
            if (shift < 0) bucket_range(crossing, lo_v, hi_v);
            lo_v = fmaxf(lo_v, v_lo), hi_v = fminf(hi_v, v_hi);
            auto crossing_ones = [&](auto f) {
                each([&](const float(&v)[V], int i) {
                    for (unsigned mask = kept(cut, v, i, within(v, lo_v, hi_v)); mask; mask &= mask - 1) {
                        const int j = i + __ffs(mask) - 1;
                        const float x = to_f32(((const T *)sample_row)[j]);
                        if (place(x) == crossing) f(x, j);
                    }
                });
            };
            if (got[3] <= S_LIST) {  // gathered and ranked in the first CTA
                SampleShared *lead = cl.map_shared_rank(&sh, 0);
                crossing_ones([&](float x, int i) { lead->list[atomicAdd(&lead->n_list, 1u)] = order_of(x, first + i); });
                cl.sync();
                bool found = false;
                u64 w[4] = {0, 0, 0, 0};
                if (rank == 0) {
                    const int m = (int)got[3];
                    rank_list(m);
                    Sum e[2];
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const int i = 2 * tid + j;
                        e[j] = i < m ? Sum{1, MASS ? weight.mass(value_of(sh.sorted[i])) : 0} : Sum{0, 0};
                    }
                    const Sum upto = done + scan(e[0] + e[1]);
                    const u64 second = MASS ? upto.mass : upto.count, one = second - (MASS ? e[1].mass : e[1].count);
                    const u64 none = one - (MASS ? e[0].mass : e[0].count);
                    if (none < target && target <= one) found = true, w[0] = sh.sorted[2 * tid];
                    else if (one < target && target <= second) found = true, w[0] = sh.sorted[2 * tid + 1];
                }
                tell(found, w, got);
                return {value_of(got[0]), index_of(got[0])};
            }
            // too many for the list: the range of their keys into buckets again
            unsigned lo = ~0u, hi = 0;
            crossing_ones([&](float x, int) { lo = min(lo, key_of(x)), hi = max(hi, key_of(x)); });
            for (int o = 16; o; o >>= 1) {
                lo = min(lo, __shfl_xor_sync(~0u, lo, o));
                hi = max(hi, __shfl_xor_sync(~0u, hi, o));
            }
            __syncthreads();
            if (lane == 0) sh.part[warp] = {lo, hi};
            __syncthreads();
            if (tid == 0) {
                for (int j = 1; j < S_WARPS; j++) lo = min(lo, (unsigned)sh.part[j].count), hi = max(hi, (unsigned)sh.part[j].mass);
                sh.part[S_WARPS] = {lo, hi};
            }
            const int at = gather_sums();
            lo = ~0u, hi = 0;
            for (int r = 0; r < ranks; r++) lo = min(lo, (unsigned)sh.all[at][r].count), hi = max(hi, (unsigned)sh.all[at][r].mass);
            v_lo = value_of(lo), v_hi = value_of(hi);
            if (lo == hi) {  // equal ones: so many, by index
                const u64 size = MASS ? weight.mass(v_lo) : 1, need = (target - (MASS ? done.mass : done.count) + size - 1) / size;
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
        for (int b = tid; b < S_BUCKETS; b += S_THREADS) sh.count[b] = 0;
        if (tid == 0) sh.n_list = 0, sh.keep = S_BUCKETS - 1;
        __syncthreads();
        if (largest > -INFINITY) atomicAdd(&sh.count[bucket(largest)], 1u);
        __syncthreads();
        const int a = sh.count[2 * tid], b = sh.count[2 * tid + 1], share = (k + ranks - 1) / ranks;
        const int to = (int)scan({(u64)(a + b), 0}).count;
        if (to - (a + b) < share && to >= share) sh.keep = 2 * tid + (to - b < share);
        __syncthreads();
        if (tid == 0) sh.part[S_WARPS].count = sh.keep;
        const int at = gather_sums();
        int bound = 0;
        for (int r = 0; r < ranks; r++) bound = max(bound, (int)sh.all[at][r].count);
        float lo, hi;
        bucket_range(bound, lo, hi);
        return lo;
    }

    // A top-k of at most S_FEW, finished in the first CTA: what is not below `bound` (bound_of) is
    // gathered, and the rest is work on a short list. False, in all CTAs, where the list would be too
    // long; true with the token in `id` (first CTA, one thread; else -1).
    __device__ bool few(float bound, int k, float top_p, double min_w, float u, int &id, float &prob) {
        SampleShared *lead = cl.map_shared_rank(&sh, 0);
        each([&](const float(&v)[V], int i) {
            for (unsigned mask = within(v, bound, INFINITY); mask; mask &= mask - 1) {
                const int j = i + __ffs(mask) - 1;
                const unsigned at = atomicAdd(&lead->n_list, 1u);
                if (at < S_LIST) lead->list[at] = order_of(to_f32(((const T *)sample_row)[j]), first + j);
            }
        });
        cl.sync();
        const int m = (int)lead->n_list;
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
        const u64 upto = scan({0, mass}).mass;
        __syncthreads();
        const u64 all = sh.part[S_WARPS].mass;
        if (top_p < 1.0f) {
            const u64 target = max((u64)ceil(max((double)top_p, 0.0) * (double)all), (u64)1);
            if (upto - mass < target && target <= upto) atomicMin(&sh.keep, (unsigned)tid + 1);
        }
        if (tid > 0 && tid < kept_k && w < min_w * MASS_ONE) atomicMin(&sh.keep, (unsigned)tid);
        __syncthreads();
        const int keep = (int)sh.keep;
        if (tid == keep - 1) sh.part[S_WARPS].mass = upto;
        u64 *masses = sh.list;
        if (tid < keep) masses[tid] = mass;
        __syncthreads();
        const u64 total = sh.part[S_WARPS].mass;
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
    if (tid < 256) sh.power[tid] = exp2(tid / 256.0);

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
    if (lane == 0) sh.part[warp].mass = best;
    __syncthreads();
    asm volatile("barrier.cluster.wait.aligned;\n" ::: "memory");
    if (tid < ranks) {
        for (int j = 0; j < S_WARPS; j++) best = max(best, sh.part[j].mass);
        cl.map_shared_rank(&sh, tid)->all[1][rank].mass = best;
    }
    cl.sync();
    best = 0;
    for (int r = 0; r < ranks; r++) best = max(best, sh.all[1][r].mass);

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
    const double inv = isinf(top) ? 1.0 : 1.0 / (double)temp;
    const Weight weight{top, (double)top, inv, inv * 369.32993046757463};  // 256 / ln 2
    // where no difference nor quotient that matters leaves the range of 32 bits
    const bool near = fabsf(top) < 1e37f && temp > 1e-30f && temp < 1e30f;
    S s{cl, full, first, rank, ranks, tid, warp, lane, weight, near, (float)(inv * S_SCALE)};
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
        cut = s.template find_cut<false>(cut, bound, [&](Sum all) { return min((u64)k, all.count); });
    }
    if (top_p < 1.0f)
        cut = s.template find_cut<true>(cut, -FLT_MAX, [&](Sum all) {
            return max((u64)ceil(max((double)top_p, 0.0) * (double)all.mass), (u64)1);
        });
    // what is too far for min_p (or for any mass) needs no exponential
    float low = near ? (float)((double)top - (min_w > 0.0 ? fmin(S_FAR, -log(min_w)) : S_FAR) * 1.001 * (double)temp) : -FLT_MAX;
    low = fmaxf(low - 1e-5f * fabsf(low), cut.value);
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

// CTAs to a row: as few as hold it, more while that leaves eight to an SM.
template <class T>
void sample_launch(const sdy_sample_args &a, cudaStream_t s) {
    constexpr int64_t ROOM = 196 * 1024;  // beside the static shared memory
    int ranks = 1;
    while (ranks < S_CLUSTER && ((int64_t)(a.n_vocab * sizeof(T)) > ranks * ROOM || (int64_t)a.n_row * ranks * 2 <= 8 * 148)) ranks *= 2;
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
