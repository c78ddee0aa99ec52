// Rotary positions of a batch of tokens with the KV store (sdy_rope_dev), and the frequencies of
// the scaled forms (sdy_rope_freqs).
//
// Pair i of a head, (a, b), becomes m * (a cos - b sin, a sin + b cos) with the angle pos * freq[i].
// The angle grows to 10^6 radians in long contexts, where 32 bits leave an error of 0.06, so it is
// formed and reduced in 64: t = pos * freq / 2 pi turns, the nearest quarter turn taken off exactly,
// and only the remainder of at most an eighth of a turn (error 2^-28 turns) goes through the 32-bit
// sine and cosine.
//
// Bound by memory: every element is read once and written once. One CTA per token: its n_rot/2
// angles are computed once into shared memory and serve all heads; a thread moves 16 bytes of each
// half of a pair run at a time (rope_kernel<T, true>), or one pair at a time where an alignment, a
// stride or an odd count forbids that (rope_kernel<T, false>).
// Measured: 8192 tokens of 32 + 4 heads of 128, bf16, 32 us (5.3 TB/s, 81% of a copy); one token 3.3 us
// on the device, 7.8 with the host's call.
#include "draft.cuh"
#include "sardyne_b200.h"

#include <cuda.h>
#include <math.h>

namespace sdy {
namespace {

constexpr int ROPE_THREADS = 256;
constexpr int ROPE_MAX_DIM = 1024;

// One token's cosines and sines (times m) into shared memory.
__device__ __forceinline__ void fill_angles(float2 *cs, const double *freq, double pos, int pairs, float m) {
    for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
        const double t = pos * freq[i] * 0.15915494309189533577;  // turns
        const double k = rint(4.0 * t);
        float s, c;
        sincospif((float)(2.0 * (t - 0.25 * k)), &s, &c);  // at most a quarter of pi
        const int q = (int)((long long)k & 3);
        const float cc = q & 1 ? s : c, ss = q & 1 ? c : s;
        cs[i] = make_float2((q == 1 || q == 2 ? -cc : cc) * m, (q >= 2 ? -ss : ss) * m);
    }
}

template <class T, int V>
struct alignas(sizeof(T) * V) Run {
    T v[V];
};

template <class T>
__device__ __forceinline__ void rotate(T &a, T &b, float2 cs) {
    const float x = to_f32(a), y = to_f32(b);
    a = from_f32<T>(x * cs.x - y * cs.y);
    b = from_f32<T>(x * cs.y + y * cs.x);
}

// Work item `it` of one head: the pairs first, then the elements that are copied. V elements at a
// time; in scalar form an interleaved item is one pair.
template <class T, bool VEC>
__device__ __forceinline__ void head_item(const T *src, T *dst, int it, int hd, int n_rot, bool interleaved,
                                          const float2 *cs) {
    constexpr int V = VEC ? 16 / sizeof(T) : 1;
    using R = Run<T, V>;
    const int half = n_rot / 2;
    const int pair_items = VEC ? (interleaved ? n_rot : half) / V : half;
    if (it >= pair_items) {
        const int e = n_rot + (it - pair_items) * V;
        *(R *)(dst + e) = *(const R *)(src + e);
    } else if (!interleaved) {
        const int e = it * V;
        R a = *(const R *)(src + e), b = *(const R *)(src + e + half);
#pragma unroll
        for (int j = 0; j < V; j++) rotate(a.v[j], b.v[j], cs[e + j]);
        *(R *)(dst + e) = a;
        *(R *)(dst + e + half) = b;
    } else if (VEC) {
        const int e = it * V;
        R a = *(const R *)(src + e);
#pragma unroll
        for (int j = 0; j + 1 < V; j += 2) rotate(a.v[j], a.v[j + 1], cs[(e + j) / 2]);
        *(R *)(dst + e) = a;
    } else {
        T a = src[2 * it], b = src[2 * it + 1];
        rotate(a, b, cs[it]);
        dst[2 * it] = a;
        dst[2 * it + 1] = b;
    }
}

template <class T, bool VEC>
__global__ void __launch_bounds__(ROPE_THREADS) rope_kernel(const sdy_rope_args p) {
    __shared__ float2 cs[ROPE_MAX_DIM / 2];
    constexpr int V = VEC ? 16 / sizeof(T) : 1;
    pdl_wait();
    const int64_t t = blockIdx.x;
    const int half = p.n_rot / 2;
    if (half) fill_angles(cs, p.freq, (double)p.pos[t], half, p.mscale);
    __syncthreads();
    int64_t at = -1;  // the token's row in the cache
    if (p.n_kv_head) {
        const int64_t slot = p.slot ? p.slot[t] : t;
        if (slot >= 0 && slot < p.n_seq * p.max_seq)
            at = slot / p.max_seq * p.cache_seq + slot % p.max_seq * p.cache_row;
    }
    const int pair_items = VEC ? (p.interleaved ? p.n_rot : half) / V : half;
    const int items = pair_items + (p.head_dim - p.n_rot) / V;  // per rotated head
    const int v_items = p.head_dim / V;
    const int n_q = p.n_head * items, n_k = at >= 0 ? p.n_kv_head * items : 0;
    const int n_v = at >= 0 && p.v ? p.n_kv_head * v_items : 0;
    for (int w = threadIdx.x; w < n_q + n_k + n_v; w += blockDim.x) {
        if (w < n_q) {
            const int h = w / items;
            head_item<T, VEC>((const T *)p.q + t * p.q_tok + h * p.q_head,
                              (T *)p.q_out + t * p.q_out_tok + h * p.q_out_head, w - h * items, p.head_dim, p.n_rot,
                              p.interleaved, cs);
        } else if (w < n_q + n_k) {
            const int h = (w - n_q) / items;
            head_item<T, VEC>((const T *)p.k + t * p.k_tok + h * p.k_head, (T *)p.k_cache + at + h * p.cache_head,
                              w - n_q - h * items, p.head_dim, p.n_rot, p.interleaved, cs);
        } else {
            const int h = (w - n_q - n_k) / v_items, e = (w - n_q - n_k - h * v_items) * V;
            *(Run<T, V> *)((T *)p.v_cache + at + h * p.cache_head + e) =
                *(const Run<T, V> *)((const T *)p.v + t * p.v_tok + h * p.v_head + e);
        }
    }
}

bool rope_check(const sdy_rope_args *a) {
    const char *fn = "sdy_rope_dev";
    const char *bad = nullptr;
    if (!a) bad = "no argument block";
    else if (a->type != T_F32 && a->type != T_F16 && a->type != T_BF16) bad = "type is not F32, F16 or BF16";
    else if (a->n_tok < 0 || a->n_head < 0 || a->n_kv_head < 0 || a->n_head > 65536 || a->n_kv_head > 65536)
        bad = "bad counts";
    else if (a->head_dim < 1 || a->head_dim > ROPE_MAX_DIM) bad = "head_dim outside [1, 1024]";
    else if (a->n_rot < 0 || a->n_rot > a->head_dim || a->n_rot % 2) bad = "n_rot is not even or not in [0, head_dim]";
    else if (!isfinite(a->mscale)) bad = "mscale is not finite";
    else if (a->n_tok && a->n_rot && (!a->freq || !a->pos)) bad = "freq or pos missing";
    else if (a->n_tok && a->n_head && (!a->q || !a->q_out)) bad = "q or q_out missing";
    else if (a->n_tok && a->n_kv_head && (!a->k || !a->k_cache || (a->v && !a->v_cache))) bad = "k or a cache missing";
    else if (a->n_kv_head && (a->n_seq < 1 || a->max_seq < 1 || a->n_seq > INT32_MAX || a->max_seq > INT32_MAX))
        bad = "cache of no rows";
    else if (!strides_fit({a->q_tok, a->q_head, a->k_tok, a->k_head, a->v_tok, a->v_head})) bad = "negative stride";
    else if (a->n_head && !disjoint({{a->q_out_tok, a->n_tok}, {a->q_out_head, a->n_head}}, a->head_dim))
        bad = "rows of q_out overlap";
    else if (a->n_kv_head && !disjoint({{a->cache_seq, a->n_seq}, {a->cache_head, a->n_kv_head},
                                        {a->cache_row, a->max_seq}}, a->head_dim))
        bad = "rows of the cache overlap";
    else if (a->n_head && a->q == a->q_out && (a->q_tok != a->q_out_tok || a->q_head != a->q_out_head))
        bad = "in place with other strides";
    const int sz = !bad ? value_bytes(a->type) : 1;
    if (!bad) {
        for (const void *p : {a->q, (const void *)a->q_out, a->k, a->v, (const void *)a->k_cache, (const void *)a->v_cache})
            if ((uintptr_t)p % sz) bad = "a pointer is not aligned to its type";
        if ((uintptr_t)a->freq % 8 || (uintptr_t)a->slot % 8 || (uintptr_t)a->pos % 4)
            bad = "a pointer is not aligned to its type";
    }
    if (bad) {
        set_error("%s: %s", fn, bad);
        return false;
    }
    if (!a->n_tok || (!a->n_head && !a->n_kv_head)) return true;
    if (a->n_rot && !device_pointers(fn, {{"freq", a->freq}, {"pos", a->pos}})) return false;
    if (a->n_head && !device_pointers(fn, {{"q", a->q}, {"q_out", a->q_out}})) return false;
    return !a->n_kv_head || device_pointers(fn, {{"k", a->k}, {"k_cache", a->k_cache}, {"v", a->v},
                                                 {"v_cache", a->v ? a->v_cache : nullptr}, {"slot", a->slot}});
}

// Whole 16-byte runs everywhere?
bool rope_vec(const sdy_rope_args &a) {
    const int v = 16 / value_bytes(a.type);
    bool ok = a.head_dim % v == 0 && (a.interleaved ? a.n_rot : a.n_rot / 2) % v == 0;
    if (a.n_head)
        ok = ok && ((uintptr_t)a.q | (uintptr_t)a.q_out) % 16 == 0 &&
             (a.q_tok | a.q_head | a.q_out_tok | a.q_out_head) % v == 0;
    if (a.n_kv_head) {
        ok = ok && ((uintptr_t)a.k | (uintptr_t)a.k_cache) % 16 == 0 &&
             (a.k_tok | a.k_head | a.cache_seq | a.cache_head | a.cache_row) % v == 0;
        if (a.v) ok = ok && ((uintptr_t)a.v | (uintptr_t)a.v_cache) % 16 == 0 && (a.v_tok | a.v_head) % v == 0;
    }
    return ok;
}

template <class T>
void rope_launch(const sdy_rope_args &a, cudaStream_t s) {
    // Small CTAs where there are many: their waits for positions, angles and data overlap (8192 tokens of
    // 40 heads of 128 in bf16: 31.8 us with 128 threads, 36.4 with 256, 41 with 384); where a token has an SM
    // for itself, twice the threads take 0.3 us less.
    const int threads = a.n_tok >= 8 * 148 ? ROPE_THREADS / 2 : ROPE_THREADS;
    if (rope_vec(a)) launch(rope_kernel<T, true>, a.n_tok, threads, 0, s, a);
    else launch(rope_kernel<T, false>, a.n_tok, threads, 0, s, a);
    SDY_LAUNCHED();
}

}  // namespace

bool pointer_device(const void *p, int *device) {
    typedef CUresult (*Query)(void *, CUpointer_attribute, CUdeviceptr);
    static const Query query = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPointByVersion("cuPointerGetAttribute", &f, 12000, cudaEnableDefault, &r) != cudaSuccess ||
            r != cudaDriverEntryPointSuccess)
            f = nullptr;
        return (Query)f;
    }();
    return query && query(device, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL, (CUdeviceptr)p) == CUDA_SUCCESS;
}

}  // namespace sdy

using namespace sdy;

extern "C" int sdy_rope_freqs(const sdy_rope_spec *p, double *freq) {
    clear_error();
    const char *bad = nullptr;
    const bool scaled = p && p->scaling != 0;
    if (!p || !freq) bad = "no argument block or no result";
    else if (p->n_rot < 2 || p->n_rot > ROPE_MAX_DIM || p->n_rot % 2) bad = "n_rot is not even or not in [2, 1024]";
    else if (p->scaling < 0 || p->scaling > 3) bad = "unknown scaling";
    else if (!(p->theta > 0) || !isfinite(p->theta)) bad = "theta is not positive";
    else if (scaled && (!(p->factor > 0) || !isfinite(p->factor))) bad = "factor is not positive";
    else if (p->scaling >= 2 && (p->orig_ctx < 1 || !(p->low > 0) || !(p->high > p->low) || !isfinite(p->high)))
        bad = "needs orig_ctx >= 1 and 0 < low < high";
    else if (p->scaling == 3 && !(p->theta > 1)) bad = "scaling by dimension needs theta > 1";
    if (!bad && p->factors)
        for (int i = 0; i < p->n_rot / 2; i++)
            if (!(p->factors[i] > 0) || !isfinite(p->factors[i])) bad = "factors are not positive";
    if (bad) {
        set_error("sdy_rope_freqs: %s", bad);
        return -1;
    }
    constexpr double TWO_PI = 6.283185307179586477;
    const int pairs = p->n_rot / 2;
    double lo = 0, hi = 0;
    if (p->scaling == 3) {  // the pairs that turn high and low times over orig_ctx positions
        auto pair_of = [&](double turns) {
            return p->n_rot * log(p->orig_ctx / (turns * TWO_PI)) / (2 * log(p->theta));
        };
        lo = std::max(floor(pair_of(p->high)), 0.0);
        hi = std::min(ceil(pair_of(p->low)), p->n_rot - 1.0);
    }
    for (int i = 0; i < pairs; i++) {
        double f = pow(p->theta, -2.0 * i / p->n_rot);
        if (p->factors) f /= p->factors[i];
        double keep = 1.0;  // the share of the unscaled frequency
        if (p->scaling == 1) keep = 0.0;
        if (p->scaling == 2) keep = (p->orig_ctx * f / TWO_PI - p->low) / (p->high - p->low);
        if (p->scaling == 3) keep = 1.0 - (i - lo) / std::max(hi - lo, 0.001);
        keep = std::min(std::max(keep, 0.0), 1.0);
        freq[i] = scaled ? keep * f + (1.0 - keep) * f / p->factor : f;
    }
    return 0;
}

extern "C" int sdy_rope_dev(const sdy_rope_args *a, void *stream) {
    clear_error();
    if (!rope_check(a)) return -1;
    if (!a->n_tok || (!a->n_head && !a->n_kv_head)) return 0;
    if (a->type == T_F32) rope_launch<float>(*a, (cudaStream_t)stream);
    else if (a->type == T_F16) rope_launch<__half>(*a, (cudaStream_t)stream);
    else rope_launch<__nv_bfloat16>(*a, (cudaStream_t)stream);
    return last_error()[0] ? -1 : 0;
}
