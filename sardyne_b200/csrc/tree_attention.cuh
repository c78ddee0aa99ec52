// What the kernels of tree_attention.cu and tree_attention_tc.cu share: the drafted nodes' paths and
// the split of a call over the CTAs.
#pragma once
#include "draft.cuh"
#include "sardyne_b200.h"

namespace sdy {

constexpr int TA_MAX_NODES = 256;
constexpr int TA_MAX_DIM = 256;
constexpr int TC_MAX_DIM = 128;  // of the tensor-core kernel

// The split. A row group is the rows (node, query head) of one KV head of one sequence that a CTA
// holds at once. Its work is its tiles of keys and, unless every tile finds a CTA of its own,
// SETUP more units for loading the queries and storing the result (about as long as that many
// tiles, most of the time of a short sequence). The units of a call, sequence
// by sequence, KV head by KV head, row group by row group, are dealt to TA_CTAS CTAs in equal
// contiguous shares, whatever the lengths of the sequences, which only the device knows. A CTA
// writes the result of a row group whose tiles it holds all; of one that its share cuts it leaves
// the unnormalised sum, the maximum and the sum of weights in one of its two slots of the workspace
// (first and last row group of its share), and join_kernel adds them up in the order of the CTAs.
constexpr int TA_CTAS = 148;  // one per SM

// A row group to join, noted by the second CTA that holds tiles of it: the parts are the slot of
// that CTA's predecessor and the first slots of the CTAs from it on.
struct Cut {
    int s, item, parts, first_slot;  // item: KV head x row groups + row group; parts 0: nothing to join
};

// Where things are in the workspace.
struct TreeSpace {
    Cut *cuts;      // [TA_CTAS]
    float *o;       // [TA_CTAS * 2] of part_stride floats: [rows][head_dim]
    float2 *ml;     // [TA_CTAS * 2][rows]: maximum (in log2 units), sum; sum < 0: padding
    size_t bytes;
};
// Floats from one slot to the next: off a power of two, so that a row's parts lie in all L2 slices.
__host__ __device__ inline int64_t part_stride(int rows, int head_dim) { return (int64_t)rows * head_dim + 1088; }
inline TreeSpace tree_space(const sdy_tree_attention_args &a, int rows) {
    TreeSpace t;
    size_t at = align_up(TA_CTAS * sizeof(Cut), 256);
    t.cuts = (Cut *)a.ws;
    t.o = (float *)((uint8_t *)a.ws + at);
    at += align_up((size_t)TA_CTAS * 2 * part_stride(rows, a.head_dim) * 4, 256);
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
__device__ __forceinline__ Lengths lengths_of(const sdy_tree_attention_args &p, int s, int past) {
    Lengths l;
    l.past = past;
    l.cached = min(l.past, p.max_seq);
    l.keys = (int)min((int64_t)l.past + p.n_node, (int64_t)p.max_seq);
    return l;
}
__device__ __forceinline__ Lengths lengths_of(const sdy_tree_attention_args &p, int s) {
    return lengths_of(p, s, max(p.n_past[s], 0));
}

// Node above j: -1 for none, -2 when j is a padding node.
__device__ __forceinline__ int node_up(const int32_t *parent, int j) {
    const int up = parent ? parent[j] : j - 1;
    return up == -1 || (up >= 0 && up < j) ? up : -2;
}
// The nodes above, checked, into shared memory by one warp; a walk along it calls at(node) from node
// j on (negative: no walk) and is true for a path that ends in a root. Every step goes to an earlier
// node, so walks end.
__device__ __forceinline__ void load_tree(int16_t *up, const int32_t *parent, int n_node) {
    for (int j = threadIdx.x % 32; j < n_node; j += 32) up[j] = (int16_t)node_up(parent, j);
    __syncwarp();
}
template <class At> __device__ __forceinline__ bool walk_tree(const int16_t *up, int j, At at) {
    while (j >= 0) {
        at(j);
        j = up[j];
    }
    return j == -1;
}

// First unit of CTA c's share, and the CTA whose share holds unit u. (Division by the constant.)
__device__ __forceinline__ int64_t share_begin(int64_t units, int c) {
    return units >= TA_CTAS ? units * c / TA_CTAS : min((int64_t)c, units);
}
__device__ __forceinline__ int share_of(int64_t units, int64_t u) {
    return units >= TA_CTAS ? (int)(((u + 1) * TA_CTAS - 1) / units) : (int)u;
}

// One CTA's share, one run of tiles [t0, t1) of a row group after the other.
struct Segment {
    int s, head, group, t0, t1, tiles, past;
};
template <int KEYS>
struct Share {
    const sdy_tree_attention_args &p;
    int64_t u, end, base;   // next unit, end, units of the sequences before s
    int s, tiles, past, items, setup;  // items: row groups per sequence; setup: units before a group's tiles
    __device__ Share(const sdy_tree_attention_args &p_, const int64_t (&found)[8], int items_)
        : p(p_), u(found[0]), end(found[1]), base(found[3]), s((int)found[2]), tiles((int)found[4]),
          past((int)found[6]), items(items_), setup((int)found[7]) {}
    // The next run; runs that hold no tile (only the end of a row group's setup) are passed over.
    __device__ bool next(Segment &g, int groups) {
        while (u < end) {
            while (u >= base + (int64_t)(tiles + setup) * items) {
                base += (int64_t)(tiles + setup) * items;
                s++;
                past = max(p.n_past[s], 0);
                tiles = (lengths_of(p, s, past).keys + KEYS - 1) / KEYS;
            }
            const int64_t r = u - base;
            const int per = tiles + setup, item = r >> 31 ? (int)(r / per) : (int)((unsigned)r / (unsigned)per);
            const int at = (int)(r - (int64_t)item * per);
            const int to = (int)min((int64_t)per, at + end - u);
            u += to - at;
            if (to <= setup) continue;
            g.s = s;
            g.head = item / groups;
            g.group = item - g.head * groups;
            g.tiles = tiles;
            g.past = past;
            g.t0 = max(at - setup, 0);
            g.t1 = to - setup;
            return true;
        }
        return false;
    }
};

// Where CTA `cta`'s share begins, for all threads of the block: out[0..7] = first unit, end, first
// sequence, units before it, its tiles, all units, its length, the setup. Up to 32 sequences are
// found by every warp for itself; more by a scan over the block's threads, each with a run of sequences.
template <int KEYS, int THREADS, int SETUP>
__device__ __forceinline__ void find_share(const sdy_tree_attention_args &p, int items, int cta,
                                           int64_t *scan /* shared, THREADS / 32 + 8 */, int64_t (&out)[8]) {
    const int t = threadIdx.x, lane = t % 32;
    auto tiles_at = [&](int past) { return (lengths_of(p, 0, past).keys + KEYS - 1) / KEYS; };
    auto past_of = [&](int s) { return max(p.n_past[s], 0); };
    if (p.n_seq <= 32) {
        const int past = lane < p.n_seq ? past_of(lane) : 0, mine = lane < p.n_seq ? tiles_at(past) : 0;
        int sum = mine;  // inclusive (fewer than 2^25 tiles to a sequence)
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(~0u, sum, o);
            if (lane >= o) sum += v;
        }
        const int total = __shfl_sync(~0u, sum, 31), setup = (int64_t)total * items <= TA_CTAS ? 0 : SETUP;
        const int64_t units = ((int64_t)total + p.n_seq * setup) * items;
        const int64_t u0 = share_begin(units, cta), u1 = share_begin(units, cta + 1);
        const int before = sum - mine + lane * setup;
        const unsigned here = __ballot_sync(~0u, lane < p.n_seq && (int64_t)before * items <= u0);
        const int s = 31 - __clz(here);  // the last sequence that begins by u0
        out[0] = u0, out[1] = u1, out[2] = s, out[3] = (int64_t)__shfl_sync(~0u, before, s) * items;
        out[4] = __shfl_sync(~0u, mine, s), out[5] = units, out[6] = __shfl_sync(~0u, past, s), out[7] = setup;
        return;
    }
    const int run = (p.n_seq + THREADS - 1) / THREADS;
    const int s0 = min(t * run, p.n_seq), s1 = min(s0 + run, p.n_seq);
    int64_t mine = 0;
    for (int s = s0; s < s1; s++) mine += tiles_at(past_of(s));
    int64_t sum = mine, *said = scan + THREADS / 32;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(~0u, sum, o);
        if (lane >= o) sum += v;
    }
    if (lane == 31) scan[t / 32] = sum;
    if (t < 8) said[t] = 0;
    __syncthreads();
    int64_t before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; w++) {
        if (w < t / 32) before += scan[w];
        total += scan[w];
    }
    const int setup = total * items <= TA_CTAS ? 0 : SETUP;
    before += sum - mine + (int64_t)s0 * setup;
    mine += (int64_t)(s1 - s0) * setup;
    const int64_t units = (total + (int64_t)p.n_seq * setup) * items;
    const int64_t u0 = share_begin(units, cta), u1 = share_begin(units, cta + 1);
    if (u0 < u1 && u0 >= before * items && u0 < (before + mine) * items) {
        int s = s0, past = past_of(s0), n = tiles_at(past);
        int64_t b = before * items;
        while (u0 >= b + (int64_t)(n + setup) * items) {
            b += (int64_t)(n + setup) * items;
            s++;
            past = past_of(s);
            n = tiles_at(past);
        }
        said[2] = s, said[3] = b, said[4] = n, said[6] = past;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i++) out[i] = said[i];
    out[0] = u0, out[1] = u1, out[5] = units, out[7] = setup;
}
// What CTA `cta` notes for join_kernel (one thread, after find_share).
template <int KEYS>
__device__ __forceinline__ void note_cut(const sdy_tree_attention_args &p, int items, int groups, int cta,
                                         const int64_t (&found)[8], Cut *cuts) {
    Cut cut = {0, 0, 0, 0};
    Share<KEYS> share(p, found, items);
    Segment g;
    if (share.next(g, groups) && g.t0 > 0) {
        const int64_t units = found[5], item = g.head * groups + g.group;
        const int64_t u0 = share.base + item * (g.tiles + share.setup);
        const int first = share_of(units, u0 + share.setup);  // the CTA that holds the first tile
        if (first == cta - 1) {
            cut.s = g.s, cut.item = (int)item;
            cut.parts = share_of(units, u0 + share.setup + g.tiles - 1) - first + 1;
            cut.first_slot = 2 * first + (share_begin(units, first) < u0);
        }
    }
    cuts[cta] = cut;
}
#endif

// out of the partial results (tree_attention.cu). rows: rows per group.
void tree_join(const sdy_tree_attention_args &a, const TreeSpace &sp, int rows, cudaStream_t s);

// 16-bit caches of up to 128 elements a head on the tensor cores (tree_attention_tc.cu).
bool tree_tc_takes(const sdy_tree_attention_args &a);
int tree_tc_rows(const sdy_tree_attention_args &a);  // rows per group
void tree_tc(const sdy_tree_attention_args &a, cudaStream_t s);
unsigned tree_tc_status();  // nonzero: a bounded wait ran out
void tree_tc_clear_status();

}  // namespace sdy
