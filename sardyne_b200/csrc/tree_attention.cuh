// What the kernels of tree_attention.cu and tree_attention_tc.cu share: the drafted nodes' paths and
// the split of a call over the CTAs.
#pragma once
#include "draft.cuh"
#include "sardyne_b200.h"

namespace sdy {

constexpr int TA_MAX_NODES = 256;
constexpr int TA_MAX_DIM = 256;

// The split. A row group is the rows (node, query head) of one KV head of one sequence that a CTA
// holds at once; a unit is one row group over one tile of keys. The units of a call, sequence by
// sequence, KV head by KV head, row group by row group, tile by tile, are dealt to TA_CTAS CTAs in
// equal contiguous shares (to as many CTAs as there are units, if fewer), whatever the lengths of the sequences, which only the device knows. A
// CTA writes the result of a row group whose tiles it holds all; of one that its share cuts it
// leaves the unnormalised sum, the maximum and the sum of weights in one of its two slots of the
// workspace (first and last of its share), and join_kernel adds them up in the order of the CTAs.
constexpr int TA_CTAS = 148;  // one per SM

// Where things are in the workspace.
struct TreeSpace {
    int64_t *base;  // [n_seq + 1]: tiles of the sequences before
    float *o;       // [TA_CTAS * 2][head_dim / 4][rows][4]
    float2 *ml;     // [TA_CTAS * 2][rows]: maximum (in log2 units), sum; sum < 0: padding
    size_t bytes;
};
inline TreeSpace tree_space(const sdy_tree_attention_args &a, int rows) {
    TreeSpace t;
    size_t at = align_up(((size_t)a.n_seq + 1) * 8, 256);
    t.base = (int64_t *)a.ws;
    t.o = (float *)((uint8_t *)a.ws + at);
    at += align_up((size_t)TA_CTAS * 2 * rows * a.head_dim * 4, 256);
    t.ml = (float2 *)((uint8_t *)a.ws + at);
    t.bytes = at + align_up((size_t)TA_CTAS * 2 * rows * 8, 256);
    return t;
}

#ifdef __CUDACC__
// Rows of the cache that sequence s may look at: [0, cached) and its drafted ones up to `keys`.
struct Lengths {
    int past;    // n_past, at least 0
    int cached;  // of those, the ones that exist
    int keys;    // existing rows, drafted ones included (at least 1)
};
__device__ __forceinline__ Lengths lengths_of(const sdy_tree_attention_args &p, int s) {
    Lengths l;
    l.past = max(p.n_past[s], 0);
    l.cached = min(l.past, p.max_seq);
    l.keys = (int)min((int64_t)l.past + p.n_node, (int64_t)p.max_seq);
    return l;
}

// Node above j: -1 for none, -2 when j is a padding node.
__device__ __forceinline__ int node_up(const int32_t *parent, int j) {
    const int up = parent ? parent[j] : j - 1;
    return up == -1 || (up >= 0 && up < j) ? up : -2;
}
// Does node j's path end in a root? Every step goes to an earlier node, so the walk ends.
__device__ __forceinline__ bool node_live(const int32_t *parent, int j) {
    while (j >= 0) j = node_up(parent, j);
    return j == -1;
}

// One CTA's share of the units, one run of tiles of one row group after the other.
struct Segment {
    int s, head, group, t0, t1, tiles;  // tiles [t0, t1) of the group's `tiles`
};
template <int KEYS>
struct Share {
    const sdy_tree_attention_args &p;
    int64_t u, end, base;
    int s, tiles, per_tile;  // per_tile: units per tile of a sequence
    __device__ Share(const sdy_tree_attention_args &p_, int64_t u_, int64_t end_, int s_, int64_t base_, int per_tile_)
        : p(p_), u(u_), end(end_), base(base_), s(s_), per_tile(per_tile_) {
        tiles = u < end ? (lengths_of(p, s).keys + KEYS - 1) / KEYS : 0;
    }
    __device__ bool next(Segment &g, int groups) {
        if (u >= end) return false;
        while (u >= (base + tiles) * per_tile) {
            base += tiles;
            tiles = (lengths_of(p, ++s).keys + KEYS - 1) / KEYS;
        }
        const int64_t r = u - base * per_tile;
        const int item = (int)(r / tiles);
        g.s = s;
        g.head = item / groups;
        g.group = item - g.head * groups;
        g.tiles = tiles;
        g.t0 = (int)(r - (int64_t)item * tiles);
        g.t1 = (int)min((int64_t)tiles, g.t0 + end - u);
        u += g.t1 - g.t0;
        return true;
    }
};

// Where CTA `cta`'s share begins, found by the whole block (THREADS threads, all of them): the
// tiles before each run of sequences by a scan over the threads, the rest by walking that run.
// out[0..3] = first unit, end, first sequence, tiles before it. CTA 0 also leaves the table of
// tiles before every sequence for join_kernel.
template <int KEYS, int THREADS>
__device__ __forceinline__ void find_share(const sdy_tree_attention_args &p, int per_tile, int cta, int ctas,
                                           int64_t *base_table, int64_t *scan /* THREADS + 1 */, int64_t *out) {
    const int t = threadIdx.x, run = (p.n_seq + THREADS - 1) / THREADS;
    const int s0 = min(t * run, p.n_seq), s1 = min(s0 + run, p.n_seq);
    int64_t mine = 0;
    for (int s = s0; s < s1; s++) mine += (lengths_of(p, s).keys + KEYS - 1) / KEYS;
    int64_t sum = mine;  // inclusive over the warp
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(~0u, sum, o);
        if (t % 32 >= o) sum += v;
    }
    if (t % 32 == 31) scan[t / 32] = sum;
    __syncthreads();
    int64_t before = 0, total = 0;
    for (int w = 0; w < THREADS / 32; w++) {
        if (w < t / 32) before += scan[w];
        total += scan[w];
    }
    before += sum - mine;
    const int64_t units = total * per_tile, n = min((int64_t)ctas, units);
    const int64_t u0 = cta < n ? units * cta / n : 0, u1 = cta < n ? units * (cta + 1) / n : 0;
    if (t == 0) out[0] = u0, out[1] = u1, out[2] = 0, out[3] = 0;
    __syncthreads();
    if (u0 < u1 && u0 >= before * per_tile && u0 < (before + mine) * per_tile) {
        int s = s0;
        for (int64_t b = before;; s++) {
            const int64_t n = (lengths_of(p, s).keys + KEYS - 1) / KEYS;
            if (u0 < (b + n) * per_tile) {
                out[2] = s, out[3] = b;
                break;
            }
            b += n;
        }
    }
    if (cta == 0) {
        for (int s = s0; s < s1; s++) {
            base_table[s] = before;
            before += (lengths_of(p, s).keys + KEYS - 1) / KEYS;
        }
        if (t == 0) base_table[p.n_seq] = total;
    }
    __syncthreads();
}
#endif

// out of the partial results (tree_attention.cu). rows: rows per group.
void tree_join(const sdy_tree_attention_args &a, const TreeSpace &sp, int rows, int ctas, cudaStream_t s);

// 16-bit caches of up to 128 elements a head on the tensor cores (tree_attention_tc.cu).
bool tree_tc_takes(const sdy_tree_attention_args &a);
int tree_tc_rows(const sdy_tree_attention_args &a);  // rows per group
void tree_tc(const sdy_tree_attention_args &a, cudaStream_t s);
unsigned tree_tc_status();  // nonzero: a bounded wait ran out
void tree_tc_clear_status();

}  // namespace sdy
