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
#include <math.h>

namespace sdy {
namespace cg = cooperative_groups;
namespace {

constexpr int S_THREADS = 512, S_WARPS = S_THREADS / 32;
constexpr int S_MAX_VOCAB = SAMPLE_MAX_VOCAB;
constexpr int S_CLUSTER = 8;                   // CTAs to a row, at most
constexpr int S_BUCKETS = 1024, S_LIST = 1024;  // the list: entries ranked at once
constexpr double S_SCALE = 32.0;               // buckets per unit of (max - l) / T
constexpr unsigned KEY_NEG_INF = 0x007FFFFFu;  // key(-inf); NaN takes key 0
constexpr double MASS_ONE = 17592186044416.0;  // 2^44
typedef unsigned long long u64;

__device__ __forceinline__ unsigned key_of(float x) {
    if (x != x) return 0;
    const unsigned b = __float_as_uint(x + 0.0f);  // (-0 is the same logit as 0)
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned key) {
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
__device__ __forceinline__ u64 order_of(unsigned key, int i) { return (u64)key << 32 | (unsigned)~i; }

struct Sum {
    u64 count, mass;
    __device__ Sum operator+(const Sum &o) const { return {count + o.count, mass + o.mass}; }
};
__device__ __forceinline__ Sum shfl_up(Sum v, int o) { return {__shfl_up_sync(~0u, v.count, o), __shfl_up_sync(~0u, v.mass, o)}; }

struct SampleShared {
    unsigned count[S_BUCKETS], lo[S_BUCKETS], hi[S_BUCKETS];  // of this CTA's entries (mass in two words)
    u64 list[S_LIST], sorted[S_LIST];                         // first CTA: gathered entries
    unsigned n_list;
    Sum part[S_WARPS + 1];                                    // per warp, then the CTA
    Sum all[2][S_CLUSTER];                                    // exchanged, by rank; two in turn
    u64 said[2][4];                                           // what one CTA tells the others; two in turn
    double power[64];                                         // 2^(j/64)
};
__shared__ SampleShared sh;  // (by name, so that accesses are known to be to shared memory)
extern __shared__ __align__(16) uint8_t sample_row[];

// w = exp(x), x = (logit - max) / temperature <= 0, by the table method: x = (64 n + j) ln 2 / 64 + r, 2^n
// 2^(j/64) exp(r), |r| <= ln 2 / 128, with the series of exp(r) to r^5 (the rest is below 2^-54).
struct Weight {
    unsigned top;   // key of the largest logit
    double m, inv;  // its value, 1 / temperature
    // 2^scale w, and 0 for what rounds to no multiple of 2^-44
    __device__ __forceinline__ double scaled(unsigned key, int scale) const {
        const double x = ((double)value_of(key) - m) * inv;
        if (key == top) return __longlong_as_double((u64)(1023 + scale) << 52);
        if (!(x > -31.2)) return 0.0;
        constexpr double MAGIC = 6755399441055744.0;  // 1.5 * 2^52: the sum's low word is the nearest integer
        const double t = fma(x, 92.332482616893656877, MAGIC);
        const int k = __double2loint(t);
        const double kd = t - MAGIC;
        double r = fma(-kd, 0.010830424696249145, x);  // ln 2 / 64 in two parts
        r = fma(-kd, 3.6235106466348430e-19, r);
        double e = fma(r, 1.0 / 120, 1.0 / 24);
        e = fma(e, r, 1.0 / 6);
        e = fma(e, r, 0.5);
        e = fma(e, r, 1.0);
        e = fma(e, r, 1.0) * sh.power[k & 63];
        return __longlong_as_double(__double_as_longlong(e) + ((long long)((k >> 6) + scale) << 52));
    }
    __device__ __forceinline__ static u64 whole(double m) {  // nearest integer, below 2^51
        return (u64)__double_as_longlong(m + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
    }
    __device__ __forceinline__ u64 mass(unsigned key) const { return whole(scaled(key, 44)); }
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
    int turn = 0, told = 0;

    __device__ __forceinline__ unsigned key(int i) const { return key_of(to_f32(((const T *)sample_row)[i])); }
    // at(key, index here) for all entries, in any order
    template <class At> __device__ __forceinline__ void each(At at) const {
        for (int i = tid; i < n / V; i += S_THREADS) {
            const Vec x = ((const Vec *)sample_row)[i];
#pragma unroll
            for (int j = 0; j < V; j++) at(key_of(to_f32(x.v[j])), i * V + j);
        }
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
    // The sums of the CTAs of lower rank and of all, from every CTA's sum in sh.part[S_WARPS].
    __device__ void exchange(Sum &before, Sum &total) {
        __syncthreads();
        if (tid < ranks) cl.map_shared_rank(&sh, tid)->all[turn][rank] = sh.part[S_WARPS];
        cl.sync();
        before = total = {0, 0};
        for (int r = 0; r < ranks; r++) {
            if (r < rank) before = before + sh.all[turn][r];
            total = total + sh.all[turn][r];
        }
        turn ^= 1;
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

    // The index at which the running sum of f(key, index), in index order, passes want_of(total); the
    // sum of all and the f there in `total` and `at`.
    template <class F, class W>
    __device__ int locate(F f, W want_of, u64 &total, u64 &at) {
        // a warp's entries are a run of indexes
        const int per = (n / V + S_WARPS - 1) / S_WARPS, i0 = min(warp * per, n / V), i1 = min(i0 + per, n / V);
        auto vec = [&](int i) -> u64 {
            u64 sum = 0;
            if (i < i1) {
                const Vec x = ((const Vec *)sample_row)[i];
#pragma unroll
                for (int j = 0; j < V; j++) sum += f(key_of(to_f32(x.v[j])), i * V + j);
            }
            return sum;
        };
        u64 mine = 0;
        for (int i = i0 + lane; i < i1; i += 32) mine += vec(i);
        for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(~0u, mine, o);
        const Sum to = scan({0, lane == 31 ? mine : 0});
        Sum before, sum;
        exchange(before, sum);
        total = sum.mass;
        const u64 want = want_of(total), end = before.mass + __shfl_sync(~0u, to.mass, 31), begin = end - mine;
        bool here = false;
        u64 v[4] = {0, 0, 0, 0};
        if (want >= begin && want < end) {
            u64 c = begin;
            for (int i = i0;; i += 32) {
                const u64 m = vec(i + lane);
                u64 in = m;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const u64 u = __shfl_up_sync(~0u, in, o);
                    if (lane >= o) in += u;
                }
                const unsigned past = __ballot_sync(~0u, want < c + in);
                if (past) {
                    here = lane == __ffs(past) - 1;
                    if (here) {
                        c += in - m;
                        for (int j = (i + lane) * V;; j++) {
                            const u64 one = f(key(j), j);
                            if (want < c + one) {
                                v[0] = first + j, v[1] = one;
                                break;
                            }
                            c += one;
                        }
                    }
                    break;
                }
                c += __shfl_sync(~0u, in, 31);
            }
            __syncwarp();
        }
        u64 got[4];
        tell(here, v, got);
        at = got[1];
        return (int)got[0];
    }

    // The lowest order of the shortest prefix whose number (MASS: mass) reaches target_of(the sum of
    // all entries from `cut` on). near: distances can be taken in 32 bits.
    template <bool MASS, class Target>
    __device__ u64 find_cut(const Weight &weight, bool near, u64 cut, Target target_of) {
        const float top = value_of(weight.top), scale = (float)(weight.inv * S_SCALE);
        unsigned k_hi = weight.top, k_lo = KEY_NEG_INF + 1;  // the keys in question
        int shift = -1;                                      // buckets by distance, then by key >> shift
        Sum done = {0, 0};                                   // before them
        u64 target = 0;
        while (true) {
            auto in_question = [&](unsigned key, int i) { return key >= k_lo && key <= k_hi && order_of(key, first + i) >= cut; };
            auto bucket = [&](unsigned key) -> int {
                if (shift >= 0) return (int)((k_hi - key) >> shift);
                if (key == weight.top) return 0;
                if (near) return (int)fminf((top - value_of(key)) * scale, S_BUCKETS - 1.0f);
                return (int)fmin((weight.m - (double)value_of(key)) * weight.inv * S_SCALE, S_BUCKETS - 1.0);
            };
            for (int b = tid; b < S_BUCKETS; b += S_THREADS) sh.count[b] = sh.lo[b] = sh.hi[b] = 0;
            if (tid == 0) sh.n_list = 0;
            __syncthreads();
            unsigned far = 0;  // by distance, the last bucket has most entries (and none of them mass)
            each([&](unsigned k, int i) {
                if (!in_question(k, i)) return;
                const int b = bucket(k);
                if (b == S_BUCKETS - 1 && shift < 0) {
                    far++;
                    return;
                }
                atomicAdd(&sh.count[b], 1u);
                if (MASS) {
                    const u64 m = weight.mass(k);
                    const unsigned low = (unsigned)m, old = atomicAdd(&sh.lo[b], low);
                    const unsigned high = (unsigned)(m >> 32) + (old + low < low);
                    if (high) atomicAdd(&sh.hi[b], high);
                }
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
            if (got[3] <= S_LIST) {
                // gathered and ranked in the first CTA: every entry counts the ones before it
                SampleShared *lead = cl.map_shared_rank(&sh, 0);
                each([&](unsigned k, int i) {
                    if (in_question(k, i) && bucket(k) == crossing) lead->list[atomicAdd(&lead->n_list, 1u)] = order_of(k, first + i);
                });
                cl.sync();
                bool found = false;
                u64 w[4] = {0, 0, 0, 0};
                if (rank == 0) {
                    const int m = (int)got[3];
                    for (int i = tid; i < m; i += S_THREADS) {
                        const u64 mine = sh.list[i];
                        int at = 0;
#pragma unroll 8
                        for (int j = 0; j < m; j++) at += sh.list[j] > mine;
                        sh.sorted[at] = mine;
                    }
                    __syncthreads();
                    Sum e[2];
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const int i = 2 * tid + j;
                        e[j] = i < m ? Sum{1, MASS ? weight.mass((unsigned)(sh.sorted[i] >> 32)) : 0} : Sum{0, 0};
                    }
                    const Sum upto = done + scan(e[0] + e[1]);
                    const u64 second = MASS ? upto.mass : upto.count, one = second - (MASS ? e[1].mass : e[1].count);
                    const u64 none = one - (MASS ? e[0].mass : e[0].count);
                    if (none < target && target <= one) found = true, w[0] = sh.sorted[2 * tid];
                    else if (one < target && target <= second) found = true, w[0] = sh.sorted[2 * tid + 1];
                }
                tell(found, w, got);
                return max(cut, got[0]);
            }
            // too many for the list: the range of their keys into buckets again
            unsigned lo = ~0u, hi = 0;
            each([&](unsigned k, int i) {
                if (in_question(k, i) && bucket(k) == crossing) lo = min(lo, k), hi = max(hi, k);
            });
            for (int o = 16; o; o >>= 1) {
                lo = min(lo, __shfl_xor_sync(~0u, lo, o));
                hi = max(hi, __shfl_xor_sync(~0u, hi, o));
            }
            __syncthreads();
            if (lane == 0) sh.part[warp] = {lo, hi};
            __syncthreads();
            if (tid < ranks) {
                for (int j = 0; j < S_WARPS; j++) lo = min(lo, (unsigned)sh.part[j].count), hi = max(hi, (unsigned)sh.part[j].mass);
                cl.map_shared_rank(&sh, tid)->all[turn][rank] = {lo, hi};
            }
            cl.sync();
            lo = ~0u, hi = 0;
            for (int r = 0; r < ranks; r++) lo = min(lo, (unsigned)sh.all[turn][r].count), hi = max(hi, (unsigned)sh.all[turn][r].mass);
            turn ^= 1;
            if (lo == hi) {  // equal ones: so many, by index
                const u64 size = MASS ? weight.mass(lo) : 1, need = (target - (MASS ? done.mass : done.count) + size - 1) / size;
                u64 total_, at_;
                const int i = locate([&](unsigned k, int j) -> u64 { return k == lo && order_of(lo, first + j) >= cut; },
                                     [&](u64) { return need - 1; }, total_, at_);
                return max(cut, order_of(lo, i));
            }
            k_lo = lo, k_hi = hi;
            for (shift = 0; (k_hi - k_lo) >> shift >= S_BUCKETS;) shift++;
        }
    }
};

template <class T>
__global__ void __launch_bounds__(S_THREADS) sample_kernel(const sdy_sample_args p, int per) {
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n" ::: "memory");  // (the CTAs of the row have begun)
    pdl_wait();
    const cg::cluster_group cl = cg::this_cluster();
    const int ranks = cl.num_blocks(), rank = cl.block_rank(), tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const int64_t row = blockIdx.x / ranks;
    constexpr int V = Sampler<T>::V;
    const int first = min(rank * per, p.n_vocab), n = min(per, p.n_vocab - first), full = (n + V - 1) / V * V;
    const T *x = (const T *)p.logits + row * p.row_stride + first;
    Sampler<T> s{cl, full, first, rank, ranks, tid, warp, lane};
    if (tid >= S_THREADS - 64) sh.power[tid - (S_THREADS - 64)] = exp2((tid - (S_THREADS - 64)) / 64.0);

    // the row into shared memory, and its largest entry
    u64 best = 0;
    auto take = [&](T v, int i) { best = max(best, order_of(key_of(to_f32(v)), first + i)); };
    const int vec = (uintptr_t)x % 16 == 0 ? n / V : 0;
#pragma unroll 4
    for (int i = tid; i < vec; i += S_THREADS) {
        const typename Sampler<T>::Vec r = ((const typename Sampler<T>::Vec *)x)[i];
        ((typename Sampler<T>::Vec *)sample_row)[i] = r;
#pragma unroll
        for (int j = 0; j < V; j++) take(r.v[j], i * V + j);
    }
#pragma unroll 4
    for (int i = vec * V + tid; i < full; i += S_THREADS) {
        const T v = i < n ? x[i] : from_f32<T>(-INFINITY);
        ((T *)sample_row)[i] = v;
        take(v, i);
    }
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

    const unsigned top = (unsigned)(best >> 32);
    const float temp = p.temperature ? p.temperature[row] : 1.0f;
    if (top <= KEY_NEG_INF || !(temp > 0.0f)) {
        if (rank == 0 && tid == 0) {
            p.id[row] = top <= KEY_NEG_INF ? -1 : (int)~(unsigned)best;
            if (p.prob) p.prob[row] = top <= KEY_NEG_INF ? 0.0f : 1.0f;
        }
        return;  // (nobody reads this CTA's shared memory any more)
    }
    // (an infinite largest logit: the others are infinitely far whatever the temperature)
    const float top_value = value_of(top);
    const Weight weight{top, (double)top_value, isinf(top_value) ? 1.0 : 1.0 / (double)temp};
    // where no difference nor quotient that matters leaves the range of 32 bits
    const bool near = fabsf(top_value) < 1e37f && temp > 1e-30f && temp < 1e30f;
    const int k = p.top_k ? p.top_k[row] : 0;
    const float top_p = p.top_p ? p.top_p[row] : 1.0f;
    double min_w = p.min_p ? (double)p.min_p[row] : 0.0;
    min_w = min_w != min_w ? 0.0 : min(min_w, 1.0);
    u64 cut = 0;
    if (k > 0 && k < p.n_vocab) cut = s.template find_cut<false>(weight, near, cut, [&](Sum all) { return min((u64)k, all.count); });
    if (top_p < 1.0f)
        cut = s.template find_cut<true>(weight, near, cut, [&](Sum all) {
            return max((u64)ceil(max((double)top_p, 0.0) * (double)all.mass), (u64)1);
        });
    // keys that are too far for min_p (or for any mass) need no exponential
    float bound = near ? (float)((double)top_value - (min_w > 0.0 ? fmin(31.3, -log(min_w)) : 31.3) * 1.001 * (double)temp) : -INFINITY;
    bound -= 1e-5f * fabsf(bound);
    const unsigned low = max(max(key_of(bound), KEY_NEG_INF + 1), (unsigned)(cut >> 32));
    const float u = p.u[row];
    u64 total, mass;
    const int id = s.locate(
        [&](unsigned key, int i) -> u64 {
            if (key < low || order_of(key, first + i) < cut) return 0;
            const double w = weight.scaled(key, 44);
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
    const struct { const char *name; const void *p; } all[] = {
        {"logits", a->logits}, {"u", a->u}, {"id", a->id}, {"temperature", a->temperature}, {"top_k", a->top_k},
        {"top_p", a->top_p}, {"min_p", a->min_p}, {"prob", a->prob}};
    for (const auto &x : all)
        if (x.p && !device_pointer(fn, x.name, x.p)) return false;
    return true;
}

}  // namespace

// CTAs to a row: as few as hold it (so that no barrier is needed where one does), more while the SMs
// are not all taken.
template <class T>
void sample_launch(const sdy_sample_args &a, cudaStream_t s) {
    constexpr int64_t ROOM = 197 * 1024;  // beside the static shared memory
    int ranks = 1;
    while (ranks < S_CLUSTER && ((int64_t)(a.n_vocab * sizeof(T)) > ranks * ROOM || (int64_t)a.n_row * ranks * 2 <= 148)) ranks *= 2;
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
