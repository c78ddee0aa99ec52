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
// CTAs that hold tiles of the group, in their order, with f_c = 2^(m_c - max m). A warp takes one row
// of a cut group (two or four where rows are narrow), the warps of all SMs in turn: its lanes start the
// copies of the first sixteen parts into shared memory (as many loads into registers the compiler
// would not keep in flight), form the factors meanwhile, and add up four elements of a row each.
// Bound by the latencies of the cuts, the maxima and the parts, one after the other (about 1 us each
// on B200), and for many wide parts by what an SM reads from L2, 64 bytes a cycle.
constexpr int JOIN_WARPS = 4, JOIN_AHEAD = 16, JOIN_BLOCKS = 5 * TA_CTAS;
constexpr int JOIN_FEW = 4;  // so many parts at most are loaded straight into registers
constexpr int JOIN_RUNS = (TA_CTAS + 31) / 32;  // cuts, or parts, a lane looks at
template <class T> __device__ __forceinline__ void store_quad(T *out, float4 v, float f) {
    struct alignas(4 * sizeof(T)) Quad { T v[4]; } q;
    q.v[0] = from_f32<T>(f == 0.0f ? 0.0f : v.x * f), q.v[1] = from_f32<T>(f == 0.0f ? 0.0f : v.y * f);
    q.v[2] = from_f32<T>(f == 0.0f ? 0.0f : v.z * f), q.v[3] = from_f32<T>(f == 0.0f ? 0.0f : v.w * f);
    *(Quad *)out = q;
}
template <class T>
__global__ void __launch_bounds__(32 * JOIN_WARPS)
    join_kernel(const sdy_tree_attention_args p, const Cut *__restrict__ cuts, const float *__restrict__ o,
                const float2 *__restrict__ ml, int rows_per_group) {
    __shared__ float factor[JOIN_WARPS][4][TA_CTAS];
    __shared__ int16_t active[JOIN_WARPS][TA_CTAS];
    extern __shared__ float4 ahead[];  // [warps][JOIN_AHEAD][32]
    pdl_wait();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    int n_active = 0;
#pragma unroll
    for (int i = 0; i < JOIN_RUNS; i++) {
        const int c = 32 * i + lane;
        const bool cut = c < TA_CTAS && cuts[c].parts > 0;
        const uint32_t all = __ballot_sync(~0u, cut);
        if (cut) active[warp][n_active + __popc(all & ((1u << lane) - 1))] = (int16_t)c;
        n_active += __popc(all);
    }
    __syncwarp();
    const int rep = p.n_head / p.n_kv_head, rows = p.n_node * rep, hd = p.head_dim;
    const int groups = (rows + rows_per_group - 1) / rows_per_group;
    const int per_warp = hd > 64 ? 1 : hd > 32 ? 2 : 4, wide = 32 / per_warp;  // rows to a warp, lanes to a row
    const int runs = (min(rows, rows_per_group) + per_warp - 1) / per_warp;
    const int64_t stride = part_stride(rows_per_group, hd);
    float4 *mine = ahead + warp * JOIN_AHEAD * 32 + lane;
    for (int w = blockIdx.x + gridDim.x * warp; w < n_active * runs; w += gridDim.x * JOIN_WARPS) {
        const int who = active[warp][w / runs], first = w % runs * per_warp, c0 = who - 1;
        const Cut cut = cuts[who];
        const int parts = cut.parts, s = cut.s, kv = cut.item / groups, group = cut.item - kv * groups;
        const int here = min(rows_per_group, rows - group * rows_per_group);  // rows of the group
        auto slot_of = [&](int c) { return c ? 2 * (c0 + c) : cut.first_slot; };
        const int r = lane / wide, in_group = first + r;
        const bool real = in_group < here;
        auto fetch = [&](int c, int d) {
            if (c < parts && real && d < hd)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"((uint32_t)__cvta_generic_to_shared(mine + c % JOIN_AHEAD * 32)),
                             "l"(o + slot_of(c) * stride + (int64_t)in_group * hd + d)
                             : "memory");
            asm volatile("cp.async.commit_group;\n" ::: "memory");
        };
        const int row = group * rows_per_group + in_group, node = row / rep, head = kv * rep + row - node * rep;
        T *out = (T *)p.out + s * p.out_seq + node * p.out_node + head * p.out_head;
        if (parts <= JOIN_FEW) {
            for (int d = 4 * (lane % wide); real && d < hd; d += 4 * wide) {
                float2 x[JOIN_FEW];
                float4 v[JOIN_FEW];
                float top = -INFINITY, sum = 0.0f;
                bool dead = false;
#pragma unroll
                for (int c = 0; c < JOIN_FEW; c++) {
                    const int slot = slot_of(min(c, parts - 1));
                    x[c] = ml[(int64_t)slot * rows_per_group + in_group];
                    v[c] = *(const float4 *)(o + slot * stride + (int64_t)in_group * hd + d);
                    if (c >= parts) x[c] = make_float2(-INFINITY, 0.0f);
                }
#pragma unroll
                for (int c = 0; c < JOIN_FEW; c++) {
                    dead = dead || x[c].y < 0.0f;
                    top = fmaxf(top, x[c].x);
                }
                float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int c = 0; c < JOIN_FEW; c++) {
                    const float f = x[c].x == -INFINITY ? 0.0f : exp2f(x[c].x - top);
                    sum += f * x[c].y;
                    if (f == 0.0f) v[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    acc.x += f * v[c].x, acc.y += f * v[c].y, acc.z += f * v[c].z, acc.w += f * v[c].w;
                }
                store_quad(out + d, acc, dead || sum == 0.0f ? 0.0f : 1.0f / sum);
            }
            continue;
        }
        for (int c = 0; c < JOIN_AHEAD; c++) fetch(c, 4 * (lane % wide));
        __syncwarp();  // the factors of the row before have been read
        for (int k = 0; k < per_warp && first + k < here; k++) {
            float2 x[JOIN_RUNS];
            float top = -INFINITY, sum = 0.0f;
            bool dead = false;
#pragma unroll
            for (int i = 0; i < JOIN_RUNS; i++) {
                const int c = 32 * i + lane;
                if (32 * i >= parts) break;
                x[i] = c < parts ? ml[(int64_t)slot_of(c) * rows_per_group + first + k] : make_float2(-INFINITY, 0.0f);
            }
#pragma unroll
            for (int i = 0; i < JOIN_RUNS; i++) {
                if (32 * i >= parts) break;
                dead = dead || x[i].y < 0.0f;
                top = fmaxf(top, x[i].x);
            }
            for (int b = 16; b; b >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, b));
            dead = __any_sync(~0u, dead);
#pragma unroll
            for (int i = 0; i < JOIN_RUNS; i++) {
                if (32 * i >= parts) break;
                x[i].x = x[i].x == -INFINITY ? 0.0f : exp2f(x[i].x - top);
                sum += x[i].x * x[i].y;
            }
            for (int b = 16; b; b >>= 1) sum += __shfl_xor_sync(~0u, sum, b);
            const float inv = dead || sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
            for (int i = 0; i < JOIN_RUNS; i++)
                if (32 * i + lane < parts) factor[warp][k][32 * i + lane] = inv == 0.0f ? 0.0f : x[i].x * inv;
        }
        __syncwarp();
        for (int d = 4 * (lane % wide); d < hd; d += 4 * wide) {
            if (d >= 4 * wide)
                for (int c = 0; c < JOIN_AHEAD; c++) fetch(c, d);
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (int c = 0; c < parts; c++) {
                asm volatile("cp.async.wait_group %0;\n" ::"n"(JOIN_AHEAD - 1) : "memory");
                const float4 v = mine[c % JOIN_AHEAD * 32];  // (which this lane copied itself)
                const float f = factor[warp][r][c];
                fetch(c + JOIN_AHEAD, d);
                if (f == 0.0f) continue;  // nothing seen there
                acc.x += f * v.x, acc.y += f * v.y, acc.z += f * v.z, acc.w += f * v.w;
            }
            if (real) store_quad(out + d, acc, 1.0f);
        }
        asm volatile("cp.async.wait_group 0;\n" ::: "memory");
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

void tree_join(const sdy_tree_attention_args &a, const TreeSpace &sp, int rows, cudaStream_t s) {
    const auto kernel = a.type == T_F32 ? join_kernel<float> : a.type == T_F16 ? join_kernel<__half> : join_kernel<__nv_bfloat16>;
    launch(kernel, JOIN_BLOCKS, 32 * JOIN_WARPS, JOIN_WARPS * JOIN_AHEAD * 32 * sizeof(float4), s, a, (const Cut *)sp.cuts,
           (const float *)sp.o, (const float2 *)sp.ml, rows);
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
