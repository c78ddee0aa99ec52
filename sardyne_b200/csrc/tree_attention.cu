// Attention of drafted tokens over a KV cache (sdy_tree_attention_dev).
//
// Sequence s has n_past cached keys, which every live node sees, and n_node drafted ones behind
// them, of which node i sees its own path to the root. Which those are is one bit per node:
// the path of i is the path of parent[i] and i itself.
#include "draft.cuh"
#include "sardyne_b200.h"

#include <math.h>

namespace sdy {
namespace {

constexpr int TA_MAX_NODES = 256;
constexpr int TA_MAX_DIM = 256;
constexpr int TA_WORDS = TA_MAX_NODES / 32;

// Bits of the nodes on node i's path (itself included) into path[0..n_words); none for a padding
// node. Every step goes to an earlier node, so the walk ends after at most i + 1.
__device__ __forceinline__ void node_path(const int32_t *parent, int i, int n_words, uint32_t *path) {
    for (int w = 0; w < n_words; w++) path[w] = 0;
    int j = i;
    while (j >= 0) {
        path[j >> 5] |= 1u << (j & 31);
        const int up = parent ? parent[j] : j - 1;
        j = up == -1 ? -1 : up >= 0 && up < j ? up : -2;
    }
    if (j == -2)
        for (int w = 0; w < n_words; w++) path[w] = 0;
}

// One CTA per (head, node, sequence): each warp takes every fourth key it sees, lane l holding
// elements l, l+32, ..; the warps' running maxima and sums are joined at the end.
constexpr int SIMPLE_WARPS = 4;
template <class T>
__global__ void __launch_bounds__(32 * SIMPLE_WARPS) tree_simple_kernel(const sdy_tree_attention_args p) {
    __shared__ uint32_t path[TA_WORDS];
    __shared__ float m_w[SIMPLE_WARPS], l_w[SIMPLE_WARPS], o_w[SIMPLE_WARPS][TA_MAX_DIM];
    pdl_wait();
    const int h = blockIdx.x, node = blockIdx.y, s = blockIdx.z, hd = p.head_dim;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int words = (p.n_node + 31) / 32;
    if (threadIdx.x == 0) node_path(p.parent ? p.parent + (int64_t)s * p.n_node : nullptr, node, words, path);
    __syncthreads();
    const int past = max(p.n_past[s], 0);
    const int keys = (int)min((int64_t)past + node + 1, (int64_t)p.max_seq);
    const bool live = path[node >> 5] >> (node & 31) & 1;
    const T *q = (const T *)p.q + s * p.q_seq + node * p.q_node + h * p.q_head;
    const int64_t base = s * p.cache_seq + h / (p.n_head / p.n_kv_head) * p.cache_head;
    const T *K = (const T *)p.k_cache + base, *V = (const T *)p.v_cache + base;
    constexpr int E = TA_MAX_DIM / 32;
    float qv[E], o[E], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++) {
        qv[e] = lane + 32 * e < hd ? to_f32(q[lane + 32 * e]) * p.scale : 0.0f;
        o[e] = 0.0f;
    }
    for (int j = warp; live && j < keys; j += SIMPLE_WARPS) {
        const int d = j - past;
        if (d >= 0 && !(path[d >> 5] >> (d & 31) & 1)) continue;
        float x = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++)
            if (lane + 32 * e < hd) x += qv[e] * to_f32(K[j * p.cache_row + lane + 32 * e]);
        for (int b = 16; b; b >>= 1) x += __shfl_xor_sync(~0u, x, b);
        const float up = fmaxf(m, x);
        if (up == -INFINITY) continue;
        const float keep = expf(m - up), w = expf(x - up);
        m = up;
        l = l * keep + w;
#pragma unroll
        for (int e = 0; e < E; e++)
            if (lane + 32 * e < hd) o[e] = o[e] * keep + w * to_f32(V[j * p.cache_row + lane + 32 * e]);
    }
    if (lane == 0) m_w[warp] = m, l_w[warp] = l;
#pragma unroll
    for (int e = 0; e < E; e++)
        if (lane + 32 * e < hd) o_w[warp][lane + 32 * e] = o[e];
    __syncthreads();
    float top = -INFINITY;
    for (int w = 0; w < SIMPLE_WARPS; w++) top = fmaxf(top, m_w[w]);
    for (int e = threadIdx.x; e < hd; e += blockDim.x) {
        float sum = 0.0f, out = 0.0f;
        for (int w = 0; w < SIMPLE_WARPS; w++) {
            if (l_w[w] == 0.0f) continue;
            const float f = expf(m_w[w] - top);
            sum += f * l_w[w];
            out += f * o_w[w][e];
        }
        ((T *)p.out)[s * p.out_seq + node * p.out_node + h * p.out_head + e] = from_f32<T>(sum > 0.0f ? out / sum : 0.0f);
    }
}

const char *counts_bad(const sdy_tree_attention_args *a) {
    if (!a) return "no argument block";
    if (a->type != T_F32 && a->type != T_F16 && a->type != T_BF16) return "type is not F32, F16 or BF16";
    if (a->n_seq < 0 || a->n_seq > 65535) return "n_seq outside [0, 65535]";
    if (a->n_node < 1 || a->n_node > TA_MAX_NODES) return "n_node outside [1, 256]";
    if (a->n_kv_head < 1 || a->n_head < a->n_kv_head || a->n_head % a->n_kv_head || a->n_head > 4096)
        return "n_head is not a multiple of n_kv_head, up to 4096";
    if (a->head_dim < 8 || a->head_dim > TA_MAX_DIM || a->head_dim % 8) return "head_dim is not a multiple of 8 in [8, 256]";
    if (a->max_seq < 1) return "cache of no rows";
    return nullptr;
}

bool tree_check(const sdy_tree_attention_args *a) {
    const char *fn = "sdy_tree_attention_dev";
    const char *bad = counts_bad(a);
    if (!bad) {
        const int v = 16 / value_bytes(a->type);
        if (!isfinite(a->scale)) bad = "scale is not finite";
        else if (a->n_seq && (!a->q || !a->k_cache || !a->v_cache || !a->n_past || !a->out)) bad = "q, a cache, n_past or out missing";
        else if (((uintptr_t)a->q | (uintptr_t)a->k_cache | (uintptr_t)a->v_cache | (uintptr_t)a->out | (uintptr_t)a->ws) % 16 ||
                 ((uintptr_t)a->n_past | (uintptr_t)a->parent) % 4)
            bad = "a pointer is not aligned to 16 bytes";
        else if (!strides_fit({a->q_seq, a->q_node, a->q_head, a->cache_seq, a->cache_head, a->cache_row})) bad = "negative stride";
        else if ((a->q_seq | a->q_node | a->q_head | a->cache_seq | a->cache_head | a->cache_row | a->out_seq |
                  a->out_node | a->out_head) % v)
            bad = "a stride is not a multiple of 16 bytes";
        else if (!disjoint({{a->out_seq, a->n_seq}, {a->out_node, a->n_node}, {a->out_head, a->n_head}}, a->head_dim))
            bad = "rows of out overlap";
        else if (a->n_seq && a->out == a->q) bad = "out is q";
        else if (a->n_seq && (a->ws_bytes < sdy_tree_attention_bytes(a) || (!a->ws && sdy_tree_attention_bytes(a))))
            bad = "ws missing or smaller than sdy_tree_attention_bytes";
    }
    if (bad) {
        set_error("%s: %s", fn, bad);
        return false;
    }
    if (!a->n_seq) return true;
    const struct { const char *name; const void *p; } all[] = {
        {"q", a->q}, {"k_cache", a->k_cache}, {"v_cache", a->v_cache}, {"n_past", a->n_past}, {"parent", a->parent},
        {"out", a->out}, {"ws", a->ws}};
    for (const auto &x : all)
        if (x.p && !device_pointer(fn, x.name, x.p)) return false;
    return true;
}

template <class T>
void tree_launch(const sdy_tree_attention_args &a, cudaStream_t s) {
    launch(tree_simple_kernel<T>, dim3(a.n_head, a.n_node, a.n_seq), 32 * SIMPLE_WARPS, 0, s, a);
    SDY_LAUNCHED();
}

}  // namespace
}  // namespace sdy

using namespace sdy;

extern "C" size_t sdy_tree_attention_bytes(const sdy_tree_attention_args *a) {
    clear_error();
    if (const char *bad = counts_bad(a)) {
        set_error("sdy_tree_attention_bytes: %s", bad);
        return 0;
    }
    return 256;
}

extern "C" int sdy_tree_attention_dev(const sdy_tree_attention_args *a, void *stream) {
    clear_error();
    if (!tree_check(a)) return -1;
    if (!a->n_seq) return 0;
    if (a->type == T_F32) tree_launch<float>(*a, (cudaStream_t)stream);
    else if (a->type == T_F16) tree_launch<__half>(*a, (cudaStream_t)stream);
    else tree_launch<__nv_bfloat16>(*a, (cudaStream_t)stream);
    return last_error()[0] ? -1 : 0;
}
