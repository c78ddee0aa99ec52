// Sampling from logits (sdy_sample_dev): temperature, top-k, top-p and min-p, then the inverse of
// the running sum at a given uniform number.
//
// All filters keep a prefix of one order: the logits descending, equal ones by index. An entry of
// that order is one 64-bit number, order(i) = key(logit_i) << 32 | ~i, with key the usual
// order-preserving image of a float, so a filter is a lower bound on it: top-k's is the k-th
// largest, top-p's the largest c with mass(order >= c) >= top_p * mass. Masses are integers:
// w = exp((l - max) / T) in 64 bits, rounded to 2^-44, so that 400000 of them fit 64 bits and their
// sum does not depend on the order of the additions. A 32-bit weight would be off by 2^-24 of
// itself, enough to move a choice whose uniform number lies next to a border once in some ten
// thousand rows; this leaves 10^-12.
#include "draft.cuh"
#include "sample.cuh"
#include "sardyne_b200.h"

#include <math.h>

namespace sdy {
namespace {

constexpr int S_THREADS = 1024;
constexpr int S_MAX_VOCAB = SAMPLE_MAX_VOCAB;
constexpr unsigned KEY_NEG_INF = 0x007FFFFFu;  // key(-inf); NaN takes key 0
constexpr double MASS_ONE = 17592186044416.0;  // 2^44
typedef unsigned long long u64;

__device__ __forceinline__ unsigned key_of(float x) {
    if (x != x) return 0;
    const unsigned b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned key) {
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
__device__ __forceinline__ u64 order_of(unsigned key, int i) { return (u64)key << 32 | (unsigned)~i; }

struct Weight {
    unsigned top;   // key of the largest logit
    double m, inv;  // its value, 1 / temperature
    __device__ double operator()(unsigned key) const {
        return key == top ? 1.0 : exp(((double)value_of(key) - m) * inv);
    }
    __device__ u64 mass(unsigned key) const { return (u64)__double2ll_rn((*this)(key) * MASS_ONE); }
};

__device__ u64 block_sum(u64 v, u64 *part) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    __syncthreads();
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = v;
    __syncthreads();
    v = part[threadIdx.x % 32];
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    return v;
}
__device__ u64 block_max(u64 v, u64 *part) {
    for (int o = 16; o; o >>= 1) v = max(v, __shfl_xor_sync(~0u, v, o));
    __syncthreads();
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = v;
    __syncthreads();
    v = part[threadIdx.x % 32];
    for (int o = 16; o; o >>= 1) v = max(v, __shfl_xor_sync(~0u, v, o));
    return v;
}

template <class T>
__global__ void __launch_bounds__(S_THREADS) sample_kernel(const sdy_sample_args p) {
    __shared__ u64 part[32];
    __shared__ u64 before[S_THREADS];
    pdl_wait();
    const int64_t row = blockIdx.x;
    const T *x = (const T *)p.logits + row * p.row_stride;
    const int n = p.n_vocab;
    auto key_at = [&](int i) { return key_of(to_f32(x[i])); };

    u64 best = 0;
    for (int i = threadIdx.x; i < n; i += S_THREADS) best = max(best, order_of(key_at(i), i));
    best = block_max(best, part);
    const unsigned top = (unsigned)(best >> 32);
    const float temp = p.temperature ? p.temperature[row] : 1.0f;
    if (top <= KEY_NEG_INF || !(temp > 0.0f)) {
        if (threadIdx.x == 0) {
            p.id[row] = top <= KEY_NEG_INF ? -1 : (int)~(unsigned)best;
            if (p.prob) p.prob[row] = top <= KEY_NEG_INF ? 0.0f : 1.0f;
        }
        return;
    }
    const Weight weight{top, (double)value_of(top), 1.0 / (double)temp};
    const int k = p.top_k ? p.top_k[row] : 0;
    const float top_p = p.top_p ? p.top_p[row] : 1.0f;
    double min_w = p.min_p ? (double)p.min_p[row] : 0.0;
    min_w = min_w != min_w ? 0.0 : min(min_w, 1.0);

    // sum over the entries from `bound` on: their number, or their mass
    auto sum_from = [&](u64 bound, bool masses) {
        u64 s = 0;
        for (int i = threadIdx.x; i < n; i += S_THREADS) {
            const unsigned key = key_at(i);
            if (key > KEY_NEG_INF && order_of(key, i) >= bound) s += masses ? weight.mass(key) : 1;
        }
        return block_sum(s, part);
    };
    // the largest bound from which on there is still `want`
    auto search = [&](u64 want, bool masses) {
        u64 c = 0;
        for (int b = 63; b >= 0; b--)
            if (sum_from(c | 1ull << b, masses) >= want) c |= 1ull << b;
        return c;
    };
    u64 cut = 0;
    if (k > 0 && k < n) cut = search(k, false);
    if (top_p < 1.0f) {
        const double want = ceil(max((double)top_p, 0.0) * (double)sum_from(cut, true));
        cut = max(cut, search(max((u64)want, 1ull), true));
    }
    // each thread sums its own run of indexes, so that the running sum goes in index order
    const int run = (n + S_THREADS - 1) / S_THREADS;
    const int i0 = min((int)threadIdx.x * run, n), i1 = min(i0 + run, n);
    auto kept_mass = [&](int i) -> u64 {
        const unsigned key = key_at(i);
        if (key <= KEY_NEG_INF || order_of(key, i) < cut) return 0;
        const double w = weight(key);
        return w >= min_w ? (u64)__double2ll_rn(w * MASS_ONE) : 0;
    };
    u64 mine = 0;
    for (int i = i0; i < i1; i++) mine += kept_mass(i);
    const u64 total = block_sum(mine, part);
    before[threadIdx.x] = mine;
    __syncthreads();
    u64 c = 0;
    for (int t = 0; t < (int)threadIdx.x; t++) c += before[t];
    const float u = p.u[row];
    const double at = (u > 0.0f ? (double)u : 0.0) * (double)total;
    const u64 want = at >= (double)total ? total - 1 : (u64)at;
    if (want >= c && want < c + mine) {
        for (int i = i0;; i++) {
            const u64 m = kept_mass(i);
            if (want < c + m) {
                p.id[row] = i;
                if (p.prob) p.prob[row] = (float)((double)m / (double)total);
                break;
            }
            c += m;
        }
    }
}

bool sample_check(const sdy_sample_args *a) {
    const char *fn = "sdy_sample_dev";
    const char *bad = nullptr;
    if (!a) bad = "no argument block";
    else if (a->type != T_F32 && a->type != T_F16 && a->type != T_BF16) bad = "type is not F32, F16 or BF16";
    else if (a->n_row < 0) bad = "bad counts";
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

void sample_rows(const sdy_sample_args &a, cudaStream_t s) {
    if (a.type == T_F32) launch(sample_kernel<float>, a.n_row, S_THREADS, 0, s, a);
    else if (a.type == T_F16) launch(sample_kernel<__half>, a.n_row, S_THREADS, 0, s, a);
    else launch(sample_kernel<__nv_bfloat16>, a.n_row, S_THREADS, 0, s, a);
    SDY_LAUNCHED();
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
