// Attention of drafted tokens over a KV cache (sdy_tree_attention_dev).
//
// Sequence s has n_past cached keys, which every live node sees, and n_node drafted ones behind
// them, of which node i sees its own path to the root. Which those are is one bit per node:
// the path of i is the path of parent[i] and i itself.
#include "tree_attention.cuh"

#include <math.h>

namespace sdy {
namespace {

constexpr int TA_WORDS = TA_MAX_NODES / 32;

// Bits of the nodes on node i's path (itself included) into path[0..n_words); none for a padding
// node.
__device__ __forceinline__ void node_path(const int32_t *parent, int i, int n_words, uint32_t *path) {
    for (int w = 0; w < n_words; w++) path[w] = 0;
    int j = i;
    for (; j >= 0; j = node_up(parent, j)) path[j >> 5] |= 1u << (j & 31);
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

// The results of the row groups that the shares cut: out = sum_c f_c o_c / sum_c f_c l_c over the
// CTAs that hold tiles of the group, in their order, with f_c = 2^(m_c - max m). One block per row
// group and eight rows; a thread holds four elements of a row.
constexpr int JOIN_ROWS = 8, JOIN_THREADS = 256;
template <class T>
__global__ void __launch_bounds__(JOIN_THREADS)
    join_kernel(const sdy_tree_attention_args p, const int64_t *base, const float4 *o, const float2 *ml, int rows_per_group,
                int max_ctas) {
    pdl_wait();
    const int rep = p.n_head / p.n_kv_head, rows = p.n_node * rep;
    const int groups = (rows + rows_per_group - 1) / rows_per_group, per_tile = p.n_kv_head * groups;
    const int s = blockIdx.x / per_tile, kv = blockIdx.x % per_tile / groups, group = blockIdx.x % groups;
    const int64_t units = base[p.n_seq] * per_tile, tiles = base[s + 1] - base[s], ctas = min((int64_t)max_ctas, units);
    const int64_t u0 = base[s] * per_tile + (kv * groups + group) * tiles, u1 = u0 + tiles;
    const int c0 = (int)(((u0 + 1) * ctas - 1) / units), c1 = (int)((u1 * ctas - 1) / units);
    if (c0 == c1) return;  // written by the CTA that holds it
    // the slot of CTA c's part: its share's first run, except where the group starts inside the share
    const int first = units * c0 / ctas == u0 ? 0 : 1;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int in_group = blockIdx.y * JOIN_ROWS + lane / 4, row = group * rows_per_group + in_group;
    if (in_group >= rows_per_group || row >= rows) return;
    auto slot_of = [&](int c) { return (int64_t)2 * c + (c == c0 ? first : 0); };
    float top = -INFINITY, sum = 0.0f;
    bool dead = false;
#pragma unroll 8
    for (int c = c0; c <= c1; c++) {
        const float2 x = ml[slot_of(c) * rows_per_group + in_group];
        dead = dead || x.y < 0.0f;
        top = fmaxf(top, x.x);
    }
    if (top == -INFINITY) top = 0.0f;
    const int quads = p.head_dim / 4, node = row / rep, head = kv * rep + row - node * rep;
    for (int d = 4 * warp + lane % 4; d < quads; d += JOIN_THREADS / JOIN_ROWS) {
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        sum = 0.0f;
#pragma unroll 8
        for (int c = c0; c <= c1; c++) {
            const int64_t slot = slot_of(c);
            const float2 x = ml[slot * rows_per_group + in_group];
            const float4 v = o[(slot * quads + d) * rows_per_group + in_group];
            if (x.x == -INFINITY) continue;
            const float f = exp2f(x.x - top);
            sum += f * x.y;
            acc.x += f * v.x, acc.y += f * v.y, acc.z += f * v.z, acc.w += f * v.w;
        }
        const bool none = dead || sum == 0.0f;
        const float inv = none ? 0.0f : 1.0f / sum;
        T *out = (T *)p.out + s * p.out_seq + node * p.out_node + head * p.out_head + 4 * d;
        struct alignas(4 * sizeof(T)) Quad { T v[4]; } q;
        q.v[0] = from_f32<T>(none ? 0.0f : acc.x * inv), q.v[1] = from_f32<T>(none ? 0.0f : acc.y * inv);
        q.v[2] = from_f32<T>(none ? 0.0f : acc.z * inv), q.v[3] = from_f32<T>(none ? 0.0f : acc.w * inv);
        *(Quad *)out = q;
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

size_t tree_bytes(const sdy_tree_attention_args &a) {
    return tree_tc_takes(a) ? tree_space(a, tree_tc_rows(a)).bytes : 256;
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
        else if (a->n_seq && (!a->ws || a->ws_bytes < tree_bytes(*a)))
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
    if (tree_tc_takes(a)) return tree_tc(a, s);
    launch(tree_simple_kernel<T>, dim3(a.n_head, a.n_node, a.n_seq), 32 * SIMPLE_WARPS, 0, s, a);
    SDY_LAUNCHED();
}

}  // namespace

void tree_join(const sdy_tree_attention_args &a, const TreeSpace &sp, int rows, int ctas, cudaStream_t s) {
    const int total = a.n_node * (a.n_head / a.n_kv_head), groups = (total + rows - 1) / rows;
    const dim3 grid((unsigned)(a.n_seq * a.n_kv_head * groups), (std::min(total, rows) + JOIN_ROWS - 1) / JOIN_ROWS);
    const auto kernel = a.type == T_F32 ? join_kernel<float> : a.type == T_F16 ? join_kernel<__half> : join_kernel<__nv_bfloat16>;
    launch(kernel, grid, JOIN_THREADS, 0, s, a, (const int64_t *)sp.base, (const float4 *)sp.o, (const float2 *)sp.ml, rows, ctas);
    SDY_LAUNCHED();
}

}  // namespace sdy

using namespace sdy;

extern "C" size_t sdy_tree_attention_bytes(const sdy_tree_attention_args *a) {
    clear_error();
    if (const char *bad = counts_bad(a)) {
        set_error("sdy_tree_attention_bytes: %s", bad);
        return 0;
    }
    return tree_bytes(*a);
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
