// Attention of drafted tokens over a KV cache (sdy_tree_attention_dev): the checks, the kernel in 32
// bits, and the one that joins partial results.
//
// Sequence s has n_past cached keys, which every live node sees, and n_node drafted ones behind
// them, of which node i sees its own path to the root.
#include "tree_attention.cuh"

#include <math.h>

#include <type_traits>

namespace sdy {
namespace {

// In 32 bits on the CUDA cores: f32 caches, and 16-bit ones that tree_attention_tc.cu does not take. A
// warp holds RW rows of one KV head and takes the 64 keys of a tile, or with WK 2 half of them, the
// other half by a second warp and joined at the end. For the scores its halves take every other four
// elements, their 16 lanes two or four keys each; for the result they take every other four keys,
// their lanes hd / 16 elements each. A 16-byte read of shared memory takes four cycles for a warp, or
// little less where lanes read the same, so what counts is how many there are: per 8 elements 2 or 4 for
// K and one for a row's Q, per 8 keys hd / 16 for V and one for a row's probabilities. K and V tiles
// come by cp.async, the next ones under this one's products.
//
// Bound by HBM and latency for few rows; for many by those reads (a tile of 64 rows of 128: 10200 cycles),
// then the 32-bit multiply-adds (2 x 64 x head_dim per row and tile: 8200); the softmax takes 1000 and to send
// for the next tile and wait 2000. Measured: 1 token, 32 over 8 heads of 128, 30000 keys 89 us (2.8
// TB/s; 115 with 16 rows to a group instead of 8), 16 sequences x 4 nodes over 2000 keys 55 us, 3 x 5 over
// 45953, 40 rows, 214 us (232 with whole warps at the same four elements, 286 in groups of 64), 7 x 52 over
// 4367 428 us (31 TFLOP/s; 461), 1 token over 701 keys of 3 heads of 64 9.4 us, most of it the launches
// and the latencies of one tile and of the join. F_SETUP, the tiles that the rest of a row group
// takes the time of: with 0, 1, 2 and 6 the second took 93, 72, 75 and 93 us in groups of 16.
constexpr int FK = 64, F_WARPS = 8, F_THREADS = 32 * F_WARPS, F_SETUP = 1;
struct Fp32Layout {
    int rows, ld, stages;  // row stride of Q, K and V in floats
    __host__ __device__ int q() const { return 0; }
    __host__ __device__ int k(int stage) const { return rows * ld + stage * 2 * FK * ld; }
    __host__ __device__ int v(int stage) const { return k(stage) + FK * ld; }
    __host__ __device__ int p() const { return rows * ld + stages * 2 * FK * ld; }
    __host__ __device__ int bytes() const { return (p() + rows * (FK + 4)) * 4; }
};
constexpr int F_SMEM = 217 * 1024;  // beside the static shared memory
// Rows to a group: those whose groups take the least time for a tile in all (about so many cycles of
// shared memory for heads of 128).
inline int fp32_rows(const sdy_tree_attention_args &a) {
    static const int size[5] = {64, 48, 32, 16, 8}, cost[5] = {10200, 8700, 7200, 4600, 3300};
    const int rows = a.n_node * (a.n_head / a.n_kv_head);
    auto all = [&](int i) { return cost[i] * ((rows + size[i] - 1) / size[i]); };
    int best = a.head_dim > 128 ? 2 : 0;  // (wider heads: 32 at most, for the registers)
    for (int i = best + 1; i < 5; i++)
        if (all(i) < all(best)) best = i;
    return size[best];
}
inline Fp32Layout fp32_layout(const sdy_tree_attention_args &a) {
    Fp32Layout l = {fp32_rows(a), a.head_dim + 4, 2};
    if (l.bytes() > F_SMEM) l.stages = 1;
    return l;
}

template <class T> __device__ __forceinline__ float4 load4(const T *p) {
    return make_float4(to_f32(p[0]), to_f32(p[1]), to_f32(p[2]), to_f32(p[3]));
}
template <> __device__ __forceinline__ float4 load4(const float *p) { return *(const float4 *)p; }
template <class T, int N> __device__ __forceinline__ void store_elements(T *out, const float *v, float f) {
    struct alignas(N * sizeof(T)) Pack { T v[N]; } q;
#pragma unroll
    for (int j = 0; j < N; j++) q.v[j] = from_f32<T>(f == 0.0f ? 0.0f : v[j] * f);
    *(Pack *)out = q;
}

template <int N> struct Elements { float v[N]; };  // of one of 16 lanes: 4 x .. + 3, 64 + 4 x .. + 3, ..
template <int N> __device__ __forceinline__ Elements<N> load_elements(const float *p, int x) {
    Elements<N> r;
#pragma unroll
    for (int j = 0; j < N; j += 4) {
        const float4 a = *(const float4 *)(p + 16 * j + 4 * x);
        r.v[j] = a.x, r.v[j + 1] = a.y, r.v[j + 2] = a.z, r.v[j + 3] = a.w;
    }
    return r;
}

template <class T, int RW, int WK, int NE>
__global__ void __launch_bounds__(F_THREADS, 1)
    tree_fp32_kernel(const sdy_tree_attention_args p, const Fp32Layout lay, Cut *cuts, float *part_o, float2 *part_ml) {
    constexpr int KL = 2 / WK, WR = F_WARPS / WK, R = RW * WR;  // keys to a lane, warps along the rows
    constexpr int EW = NE < 4 ? NE : 4, NL = 2 * NE;            // elements side by side; a lane's while halves differ
    __shared__ int64_t scan[F_THREADS / 32 + 8];
    int64_t found[8];
    __shared__ int16_t up[TA_MAX_NODES];
    __shared__ uint32_t path[TA_MAX_NODES][TA_MAX_NODES / 32 + 1];  // the nodes each node sees; 0: padding
    extern __shared__ __align__(16) float mem[];
    pdl_wait();
    const int tid = threadIdx.x, lane = tid % 32, x = lane % 16, half = lane / 16, wr = tid / 32 % WR, wk = tid / 32 / WR, hd = p.head_dim, ld = lay.ld;
    const int rep = p.n_head / p.n_kv_head, rows = p.n_node * rep, groups = (rows + R - 1) / R, items = p.n_kv_head * groups;
    find_share<FK, F_THREADS, F_SETUP>(p, items, blockIdx.x, scan, found);
    if (tid == 0) note_cut<FK>(p, items, groups, blockIdx.x, found, cuts);
    Share<FK> share(p, found, items);
    Segment g;
    float *Q = mem + lay.q(), *P = mem + lay.p();
    const float c = p.scale * 1.4426950408889634f;
    for (int seg = 0; share.next(g, groups); seg++) {
        const Lengths len = lengths_of(p, g.s, g.past);
        const int32_t *parent = p.parent ? p.parent + (int64_t)g.s * p.n_node : nullptr;
        const T *kc = (const T *)p.k_cache + g.s * p.cache_seq + g.head * p.cache_head;
        const T *vc = (const T *)p.v_cache + g.s * p.cache_seq + g.head * p.cache_head;
        const int quads = hd / 4, r0 = tid / quads, c0 = tid % quads, dr = F_THREADS / quads, dc = F_THREADS % quads;
        // a tile into stage `st`; rows that do not exist are zero
        auto fetch = [&](int tile, int st) {
            for (int r = r0, c = c0; r < FK; r += dr, c += dc) {
                if (c >= quads) {
                    c -= quads;
                    if (++r >= FK) break;
                }
                const int e = 4 * c, j = tile * FK + r;
                float *k = mem + lay.k(st) + r * ld + e, *v = mem + lay.v(st) + r * ld + e;
                if (j >= len.keys) {
                    *(float4 *)k = *(float4 *)v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                } else if (std::is_same<T, float>::value) {
                    const uint32_t kd = (uint32_t)__cvta_generic_to_shared(k), vd = (uint32_t)__cvta_generic_to_shared(v);
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(kd), "l"(kc + j * p.cache_row + e) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(vd), "l"(vc + j * p.cache_row + e) : "memory");
                } else {
                    *(float4 *)k = load4(kc + j * p.cache_row + e);
                    *(float4 *)v = load4(vc + j * p.cache_row + e);
                }
            }
            asm volatile("cp.async.commit_group;\n" ::: "memory");
        };
        __syncthreads();  // the segment before has been read
        const bool edges = g.t1 * FK > len.cached;
        if (lay.stages == 2) fetch(g.t0, 0);
        for (int w = tid; w < R * quads; w += F_THREADS) {
            const int r = w / quads, e = 4 * (w - r * quads), row = g.group * R + r, node = row / rep;
            const T *q = (const T *)p.q + g.s * p.q_seq + node * p.q_node + (g.head * rep + row - node * rep) * p.q_head + e;
            float *to = Q + r * ld + e;
            if (row >= rows) *(float4 *)to = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            else if (std::is_same<T, float>::value)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(q) : "memory");
            else *(float4 *)to = load4(q);
        }
        if (lay.stages == 2) asm volatile("cp.async.commit_group;\n" ::: "memory");
        if (edges) {
            if (tid < 32) load_tree(up, parent, p.n_node);
            __syncthreads();
            for (int i = tid; i < p.n_node; i += F_THREADS) {
#pragma unroll
                for (int w = 0; w <= TA_MAX_NODES / 32; w++) path[i][w] = 0;
                const bool live = walk_tree(up, i, [&](int j) { path[i][j >> 5] |= 1u << (j & 31); });
                if (!live)
#pragma unroll
                    for (int w = 0; w <= TA_MAX_NODES / 32; w++) path[i][w] = 0;
            }
        }
        float m[RW], l[RW];
        Elements<NL> o[RW];  // of the half's keys
        unsigned live = ~0u;  // rows of live nodes, as far as this segment knows
        auto row_of = [&](int i) { return g.group * R + wr * RW + i; };
#pragma unroll
        for (int i = 0; i < RW; i++) {
            m[i] = -INFINITY, l[i] = 0.0f;
#pragma unroll
            for (int j = 0; j < NL; j++) o[i].v[j] = 0.0f;
        }
        for (int t = g.t0; t < g.t1; t++) {
            const int st = lay.stages == 2 ? (t - g.t0) & 1 : 0, j0 = t * FK;
            if (lay.stages == 2) {
                if (t + 1 < g.t1) {
                    fetch(t + 1, st ^ 1);  // (its group is the last: what came before, the queries too, is waited for)
                    asm volatile("cp.async.wait_group 1;\n" ::: "memory");
                } else {
                    asm volatile("cp.async.wait_group 0;\n" ::: "memory");
                }
            } else {
                fetch(t, 0);
                asm volatile("cp.async.wait_group 0;\n" ::: "memory");
            }
            __syncthreads();
            const float *K = mem + lay.k(st);
            float *V = mem + lay.v(st);
            // drafted rows: which keys a row sees; V of padding nodes is zero, and NaN or infinities of
            // others meet only the rows that see them
            uint64_t sees[RW];
            bool odd = false;
#pragma unroll
            for (int i = 0; i < RW; i++) sees[i] = ~0ull;
            if (j0 + FK > len.cached) {
                const int from = min(max(len.cached - j0, 0), FK), d0 = j0 + from - len.past;  // first drafted row of the tile
                const int drafted = min(len.keys - j0, FK) - from;
                const int row = row_of(lane % RW), node = row < rows ? row / rep : 0;  // a lane finds one row's
                const bool lives = row < rows && (path[node][node >> 5] >> (node & 31) & 1);
                uint64_t bits = 0;
                if (lives && drafted > 0) {  // bits d0 .. of the path
                    const uint32_t *w = path[node] + (d0 >> 5);
                    const int words = TA_MAX_NODES / 32 - (d0 >> 5);  // (the last word is zero)
                    const uint64_t lo = w[0] | (uint64_t)(words > 1 ? w[1] : 0) << 32, hi = words > 2 ? w[2] : 0;
                    bits = lo >> (d0 & 31) | ((d0 & 31) ? hi << (64 - (d0 & 31)) : 0);
                    if (drafted < 64) bits &= (1ull << drafted) - 1;
                }
                bits = !lives ? 0 : from == 64 ? ~0ull : ((1ull << from) - 1) | bits << from;
                live = __ballot_sync(~0u, lives);
#pragma unroll
                for (int i = 0; i < RW; i++) sees[i] = __shfl_sync(~0u, bits, i);
                for (int w = tid; w < max(drafted, 0) * quads; w += F_THREADS) {
                    const int r = w / quads, d = d0 + r;
                    float4 *v = (float4 *)(V + (from + r) * ld + 4 * (w - r * quads));
                    if (!(path[d][d >> 5] >> (d & 31) & 1)) *v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    else odd = odd || !isfinite(v->x) || !isfinite(v->y) || !isfinite(v->z) || !isfinite(v->w);
                }
                odd = __syncthreads_or(odd);
            }
            // each half of the warp takes every other four elements of all the warp's keys, then half the keys
            const int k0 = wk * 32 * KL, key = k0 + x + half * 16 * KL;  // (and 16 behind it)
            float part[RW][2 * KL], s[RW][KL];
#pragma unroll
            for (int i = 0; i < RW; i++)
#pragma unroll
                for (int j = 0; j < 2 * KL; j++) part[i][j] = 0.0f;
#pragma unroll 2
            for (int e = 4 * half; e < hd; e += 8) {
                float4 k[2 * KL];
#pragma unroll
                for (int j = 0; j < 2 * KL; j++) k[j] = *(const float4 *)(K + (k0 + x + 16 * j) * ld + e);
#pragma unroll
                for (int i = 0; i < RW; i++) {
                    const float4 q = *(const float4 *)(Q + (wr * RW + i) * ld + e);
#pragma unroll
                    for (int j = 0; j < 2 * KL; j++) part[i][j] += q.x * k[j].x + q.y * k[j].y + q.z * k[j].z + q.w * k[j].w;
                }
            }
#pragma unroll
            for (int i = 0; i < RW; i++)
#pragma unroll
                for (int j = 0; j < KL; j++)
                    s[i][j] = (half ? part[i][KL + j] : part[i][j]) + __shfl_xor_sync(~0u, half ? part[i][j] : part[i][KL + j], 16);
            float f[RW], *own = P + wr * RW * (FK + 4);
#pragma unroll
            for (int i = 0; i < RW; i++) {
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < KL; j++) {
                    s[i][j] = sees[i] >> (key + 16 * j) & 1 ? s[i][j] * c : -INFINITY;
                    top = fmaxf(top, s[i][j]);
                }
#pragma unroll
                for (int b = 16; b; b >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, b));
                const float now = fmaxf(m[i], top), off = now == -INFINITY ? 0.0f : now;
                f[i] = exp2f(m[i] - off);  // (0 at first)
                m[i] = now;
                l[i] *= f[i];
#pragma unroll
                for (int j = 0; j < KL; j++) {
                    const float w = exp2f(s[i][j] - off);
                    own[i * (FK + 4) + key + 16 * j] = w;
                    l[i] += w;
                }
            }
            __syncwarp();
            // (a tile's sum on its own, then to the others': a long cache's sums err by its tiles, not its keys)
            Elements<NL> sum[RW];
#pragma unroll
            for (int i = 0; i < RW; i++)
#pragma unroll
                for (int j = 0; j < NL; j++) sum[i].v[j] = 0.0f;
            auto products = [&](auto skip_zero) {
#pragma unroll 2
                for (int k = k0 + 4 * half; k < k0 + 32 * KL; k += 8) {
                    Elements<NL> v[4];
#pragma unroll
                    for (int b = 0; b < 4; b++) v[b] = load_elements<NL>(V + (k + b) * ld, x);
#pragma unroll
                    for (int i = 0; i < RW; i++) {
                        const float4 w4 = *(const float4 *)(own + i * (FK + 4) + k);
                        const float w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                        for (int b = 0; b < 4; b++) {
                            if (skip_zero() && w[b] == 0.0f) continue;
#pragma unroll
                            for (int j = 0; j < NL; j++) sum[i].v[j] += w[b] * v[b].v[j];
                        }
                    }
                }
            };
            if (odd) products(std::true_type());
            else products(std::false_type());
#pragma unroll
            for (int i = 0; i < RW; i++)
#pragma unroll
                for (int j = 0; j < NL; j++) o[i].v[j] = o[i].v[j] * f[i] + sum[i].v[j];
            __syncthreads();  // the tile has been read
        }
        const bool whole = g.t0 == 0 && g.t1 == g.tiles;
        const int64_t slot = 2 * blockIdx.x + (seg > 0);
        Elements<NE> sum[RW];
#pragma unroll
        for (int i = 0; i < RW; i++) {
#pragma unroll
            for (int b = 16; b; b >>= 1) l[i] += __shfl_xor_sync(~0u, l[i], b);
            // both halves' keys, of half the elements each
#pragma unroll
            for (int j = 0; j < NE; j++) {
                const int a = j / EW * 2 * EW + j % EW;
                sum[i].v[j] = (half ? o[i].v[a + EW] : o[i].v[a]) + __shfl_xor_sync(~0u, half ? o[i].v[a] : o[i].v[a + EW], 16);
            }
        }
        if (WK == 2) {  // the second warp's through shared memory (the first stage's, which has been read)
            float *shared_o = mem + lay.k(0) + wr * RW * 32 * NE, *shared_ml = P + wr * RW * 2;
            if (wk == 1) {
#pragma unroll
                for (int i = 0; i < RW; i++) {
#pragma unroll
                    for (int j = 0; j < NE; j++) shared_o[(i * NE + j) * 32 + lane] = sum[i].v[j];
                    if (lane == 0) shared_ml[2 * i] = m[i], shared_ml[2 * i + 1] = l[i];
                }
            }
            __syncthreads();
            if (wk == 1) continue;
#pragma unroll
            for (int i = 0; i < RW; i++) {
                const float m1 = shared_ml[2 * i], now = fmaxf(m[i], m1), off = now == -INFINITY ? 0.0f : now;
                const float f0 = exp2f(m[i] - off), f1 = exp2f(m1 - off);
                m[i] = now, l[i] = l[i] * f0 + shared_ml[2 * i + 1] * f1;
#pragma unroll
                for (int j = 0; j < NE; j++) sum[i].v[j] = sum[i].v[j] * f0 + shared_o[(i * NE + j) * 32 + lane] * f1;
            }
        }
#pragma unroll
        for (int i = 0; i < RW; i++) {
            const int r = wr * RW + i, row = row_of(i), node = row / rep;
            if (row >= rows) continue;
            const bool lives = live >> i & 1;
            if (!whole && lane == 0) part_ml[slot * R + r] = make_float2(m[i], lives ? l[i] : -1.0f);
            T *out = (T *)p.out + g.s * p.out_seq + node * p.out_node + (g.head * rep + row - node * rep) * p.out_head;
            float *part = part_o + slot * part_stride(R, hd) + (int64_t)r * hd;
            const float by = lives && l[i] != 0.0f ? 1.0f / l[i] : 0.0f;
#pragma unroll
            for (int j = 0; j < NE; j += EW) {
                const int e = NE < 4 ? 4 * x + 2 * half : 32 * j + 4 * lane;
                if (e >= hd) continue;
                if (whole) store_elements<T, EW>(out + e, sum[i].v + j, by);
                else store_elements<float, EW>(part + e, sum[i].v + j, 1.0f);
            }
        }
    }
}

// The results of the row groups that the shares cut: out = sum_c f_c o_c / sum_c f_c l_c over the
// CTAs that hold tiles of the group, in their order, with f_c = 2^(m_c - max m). A warp takes one row
// of a cut group (two or four where rows are narrow), the warps of all SMs in turn: its lanes start the
// copies of the first eight parts into shared memory (as many loads into registers the compiler
// would not keep in flight), form the factors meanwhile, and add up four elements of a row each.
// Bound by the latencies of the cuts, the maxima and the parts, one after the other (about 1 us each
// on B200), and for many wide parts by what an SM reads from L2, 64 bytes a cycle.
// Both kernels of 16 sequences of 24 nodes, up to 8192 keys: 57.6 us with eight parts ahead and six CTAs
// to an SM, 59 with eight and four, 58.9 with sixteen and four, 62.4 with sixteen and five (of which one
// waits for room).
constexpr int JOIN_WARPS = 4, JOIN_AHEAD = 8, JOIN_BLOCKS = 6 * TA_CTAS;
constexpr int JOIN_FEW = 4;  // so many parts at most are loaded straight into registers
constexpr int JOIN_RUNS = (TA_CTAS + 31) / 32;  // cuts, or parts, a lane looks at
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
                store_elements<T, 4>(out + d, &acc.x, dead || sum == 0.0f ? 0.0f : 1.0f / sum);
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
            if (real) store_elements<T, 4>(out + d, &acc.x, 1.0f);
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

// The workspace of the shape, whichever kernel its strides choose (the tensor cores' groups are larger).
size_t tree_bytes(const sdy_tree_attention_args &a) {
    return tree_space(a, a.type != T_F32 && a.head_dim <= TC_MAX_DIM ? tree_tc_rows(a) : fp32_rows(a)).bytes;
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
    return device_pointers(fn, {{"q", a->q}, {"k_cache", a->k_cache}, {"v_cache", a->v_cache}, {"n_past", a->n_past}, {"parent", a->parent}, {"out", a->out}, {"ws", a->ws}});
}

template <class T, int RW, int WK, int NE>
void fp32_launch(const sdy_tree_attention_args &a, const TreeSpace &sp, cudaStream_t s) {
    const Fp32Layout lay = fp32_layout(a);
    static std::atomic<uint64_t> done{0};
    smem_limit_once(tree_fp32_kernel<T, RW, WK, NE>, F_SMEM, done);
    launch(tree_fp32_kernel<T, RW, WK, NE>, TA_CTAS, F_THREADS, lay.bytes(), s, a, lay, sp.cuts, sp.o, sp.ml);
    SDY_LAUNCHED();
}
template <class T, int RW, int WK>
void fp32_pick(const sdy_tree_attention_args &a, const TreeSpace &sp, cudaStream_t s) {
    if (a.head_dim <= 64) fp32_launch<T, RW, WK, 2>(a, sp, s);
    else fp32_launch<T, RW, WK, 4>(a, sp, s);
}
template <class T>
void tree_launch(const sdy_tree_attention_args &a, cudaStream_t s) {
    if (tree_tc_takes(a)) return tree_tc(a, s);
    const int rows = fp32_rows(a);
    const TreeSpace sp = tree_space(a, rows);
    if (a.head_dim > 128) {
        if (rows == 8) fp32_launch<T, 2, 2, 8>(a, sp, s);
        else if (rows == 16) fp32_launch<T, 4, 2, 8>(a, sp, s);
        else fp32_launch<T, 4, 1, 8>(a, sp, s);
    } else if (rows == 8) fp32_pick<T, 2, 2>(a, sp, s);
    else if (rows == 16) fp32_pick<T, 4, 2>(a, sp, s);
    else if (rows == 32) fp32_pick<T, 8, 2>(a, sp, s);
    else if (rows == 48) fp32_pick<T, 6, 1>(a, sp, s);
    else fp32_pick<T, 8, 1>(a, sp, s);
    tree_join(a, sp, rows, s);
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
