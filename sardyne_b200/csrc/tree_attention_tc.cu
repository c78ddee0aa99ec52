// Tree attention over 16-bit caches on the tensor cores (tcgen05, accumulators in TMEM).
//
// For one KV head of one sequence the rows are its (node, query head) pairs, 128 to an MMA tile;
// per tile of 128 keys, S = Q K^T (128 x 128, f32 in TMEM), P = 2^(c S - m) as 16-bit values over
// S's own columns, O += P V with P read from TMEM. m is a row's running maximum; O and the sum are
// rescaled only when it has grown by more than 2^8 since it was last set (the division by the sum
// takes out any common factor; 2^8 keeps P inside the range of f16), which after the first tiles
// hardly ever happens, so O stays in TMEM.
//
// One CTA per SM, twelve warps: a TMA producer (K and V tiles of 128 keys through a ring of shared
// memory slots), an MMA issuer, and two streams of four warps that turn S into P, one row to a
// thread, so that one stream's exponentials run under the other's MMAs. With more than 128 rows the
// streams hold two row tiles and share every K and V tile (DUAL); with fewer they share the rows
// and take the tiles in turn, and the first stream joins the two results at the end.
//
// Bound by the tensor pipe and the exponentials alike from about 256 rows (128 x 128 scores take
// 1024 cycles of MMA and 1024 of the exponential unit), by HBM below about 64.
#include "tree_attention.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>

#include <math.h>

#include <type_traits>

namespace sdy {
namespace {

constexpr int TK = 128;       // keys per tile
constexpr int TR = 128;       // rows per MMA tile
constexpr int TT = 384;       // threads
constexpr int CHUNK = TK * 128;  // bytes of 64 elements of 128 rows, 128-byte swizzled
constexpr long long WAIT_LIMIT = 1ll << 22;  // mbarrier polls before giving up (about a second)
constexpr uint32_t TM_S = 0, TM_O = 256;     // TMEM columns of the streams' S and O, 128 each
constexpr float GROWTH = 8.0f;

__device__ unsigned g_tree_status;  // nonzero: a wait ran out

constexpr int tc_slots(bool dual, int hc) { return hc == 1 ? 10 : dual ? 5 : 6; }
constexpr int tc_smem(bool dual, int hc) { return ((dual ? 2 : 1) + tc_slots(dual, hc)) * hc * CHUNK + 1024; }

struct Shared {
    uint64_t full[10], empty[10];
    uint64_t q_ready[2], s_full[2], p_ready[2], o_done[2];
    uint64_t merge_full, merge_done, drain;
    uint32_t tmem, abort;
    int odd;  // the last segment (from 1) whose drafted V rows hold NaN or infinities
    int64_t scan[TT / 32], share[4];
    float2 ml[TR];
};

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint64_t *b, int n) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(smem_u32(b)), "r"(n) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t *b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(smem_u32(b)) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint64_t *b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(smem_u32(b)), "r"(bytes) : "memory");
}
// Bounded: false, with the abort flag set, when the limit ran out here or in another role.
__device__ __forceinline__ bool mbar_wait(uint64_t *b, uint32_t parity, Shared *sh) {
    const uint32_t bar = smem_u32(b);
    for (long long it = 0; it < WAIT_LIMIT; it++) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}\n"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (done) return true;
        if ((it & 255) == 255 && *(volatile uint32_t *)&sh->abort) return false;
    }
    *(volatile uint32_t *)&sh->abort = 1;
    return false;
}
__device__ __forceinline__ bool warp_wait(uint64_t *b, uint32_t parity, Shared *sh) {
    return __all_sync(~0u, mbar_wait(b, parity, sh));
}

__device__ __forceinline__ void tma_tile(const CUtensorMap *map, uint64_t *bar, uint32_t dst, int x, int row, int head, int s) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];\n" ::"r"(dst),
        "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(row), "r"(head), "r"(s)
        : "memory");
}

// Shared memory descriptors of tiles in the 128-byte swizzle: K-major (Q and K: 8-row groups of
// 1024 bytes) and N-major (V: 64-element chunks at CHUNK, 8-key groups of 1024 bytes).
__device__ __forceinline__ uint64_t desc_of(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)(lbo >> 4) << 16 | (uint64_t)(sbo >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// kind::f16: f32 accumulator, A and B of one 16-bit type, M = 128; b_mn: B is N-major.
__device__ __forceinline__ uint32_t idesc_f16(bool bf16, int n, bool b_mn) {
    return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (b_mn ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(TR >> 4) << 24;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t *b) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(smem_u32(b)) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }

#define R32(v, o)                                                                                                       \
    v[o], v[o + 1], v[o + 2], v[o + 3], v[o + 4], v[o + 5], v[o + 6], v[o + 7], v[o + 8], v[o + 9], v[o + 10], v[o + 11], \
        v[o + 12], v[o + 13], v[o + 14], v[o + 15], v[o + 16], v[o + 17], v[o + 18], v[o + 19], v[o + 20], v[o + 21],     \
        v[o + 22], v[o + 23], v[o + 24], v[o + 25], v[o + 26], v[o + 27], v[o + 28], v[o + 29], v[o + 30], v[o + 31]
#define OUT4(v, o) "=f"(v[o]), "=f"(v[o + 1]), "=f"(v[o + 2]), "=f"(v[o + 3])
#define IN4(v, o) "r"(v[o]), "r"(v[o + 1]), "r"(v[o + 2]), "r"(v[o + 3])
#define LIST32                                                                                                        \
    "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, " \
    "%24, %25, %26, %27, %28, %29, %30, %31}"
// 32 columns of this thread's lane (the warp's four-lane quarter in the address).
__device__ __forceinline__ void tmem_ld(uint32_t addr, float *v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 " LIST32 ", [%32];\n"
                 : OUT4(v, 0), OUT4(v, 4), OUT4(v, 8), OUT4(v, 12), OUT4(v, 16), OUT4(v, 20), OUT4(v, 24), OUT4(v, 28)
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_st(uint32_t addr, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], " LIST32 ";\n" ::IN4(v, 0), IN4(v, 4), IN4(v, 8), IN4(v, 12),
                 IN4(v, 16), IN4(v, 20), IN4(v, 24), IN4(v, 28), "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
template <class T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    __half2 h = __floats2half2_rn(lo, hi);
    return *(uint32_t *)&h;
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *(uint32_t *)&h;
}
// Of two packed 16-bit values, the ones that are NaN or infinite replaced by zero.
template <class T> __device__ __forceinline__ uint32_t finite2(uint32_t w) {
    constexpr uint32_t E = sizeof(T) == 2 && std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
    if ((w & E) == E) w &= 0xFFFF0000u;
    if (((w >> 16) & E) == E) w &= 0x0000FFFFu;
    return w;
}

// Position in the ring's load order, counted from the segment's first load, of tile i's K and V:
// the order in which the MMAs take them.
template <bool DUAL> __device__ __forceinline__ int k_pos(int i) { return DUAL ? 2 * i : i < 2 ? i : 2 * i - 1; }
template <bool DUAL> __device__ __forceinline__ int v_pos(int i, int n) {
    return DUAL || i == n - 1 ? 2 * i + 1 : 2 * i + 2;
}

template <class T, bool DUAL, int HC>
__global__ void __launch_bounds__(TT, 1)
    tree_tc_kernel(const sdy_tree_attention_args p, const __grid_constant__ CUtensorMap kmap,
                   const __grid_constant__ CUtensorMap vmap, int64_t *base_table, float *part_o, float2 *part_ml) {
    constexpr int NS = tc_slots(DUAL, HC), NQ = DUAL ? 2 : 1, LEAD = DUAL ? 1 : 2;
    constexpr int TILE = HC * CHUNK, ROWS = NQ * TR;
    constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
    __shared__ Shared sh;
    extern __shared__ uint8_t dyn[];
    uint8_t *qbuf = (uint8_t *)(((uintptr_t)dyn + 1023) & ~(uintptr_t)1023), *ring = qbuf + NQ * TILE;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int rep = p.n_head / p.n_kv_head, rows = p.n_node * rep, groups = (rows + ROWS - 1) / ROWS;
    const int n_pv = (p.head_dim + 15) & ~15, k_steps = (p.head_dim + 15) / 16;

    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(smem_u32(&sh.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < NS; i++) mbar_init(&sh.full[i], 1), mbar_init(&sh.empty[i], 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(&sh.q_ready[i], TR), mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.p_ready[i], TR), mbar_init(&sh.o_done[i], 1);
        }
        mbar_init(&sh.merge_full, TR), mbar_init(&sh.merge_done, TR), mbar_init(&sh.drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        sh.abort = 0, sh.odd = 0;
    }
    pdl_wait();
    find_share<TK, TT>(p, p.n_kv_head * groups, blockIdx.x, gridDim.x, base_table, sh.scan, sh.share);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = sh.tmem;
    Share<TK> share(p, sh.share[0], sh.share[1], (int)sh.share[2], sh.share[3], p.n_kv_head * groups);
    Segment g;

    if (warp == 0) {
        if (lane == 0) {
            int pos = 0;  // loads so far
            bool ok = true;
            auto load = [&](const CUtensorMap *map, int tile) {
                const int slot = pos % NS, turn = pos / NS;
                if (turn && !mbar_wait(&sh.empty[slot], (turn - 1) & 1, &sh)) return false;
                mbar_expect(&sh.full[slot], TILE);
                for (int c = 0; c < HC; c++)
                    tma_tile(map, &sh.full[slot], smem_u32(ring + slot * TILE + c * CHUNK), 64 * c, tile * TK, g.head, g.s);
                pos++;
                return true;
            };
            while (ok && share.next(g, groups)) {
                const int n = g.t1 - g.t0;
                for (int i = 0; ok && i < min(LEAD, n); i++) ok = load(&kmap, g.t0 + i);
                for (int i = 0; ok && i < n; i++) {
                    ok = load(&vmap, g.t0 + i);
                    if (ok && i + LEAD < n) ok = load(&kmap, g.t0 + i + LEAD);
                }
            }
            if (!ok) {  // let the copies in flight land before the memory is given up
                sh.abort = 1;
                atomicOr(&g_tree_status, 1u);
                for (int q = max(0, pos - NS); q < pos; q++)
                    for (long long it = 0; it < WAIT_LIMIT; it++) {
                        uint32_t done;
                        asm volatile(
                            "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
                            : "=r"(done)
                            : "r"(smem_u32(&sh.full[q % NS])), "r"(q / NS & 1)
                            : "memory");
                        if (done) break;
                    }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t id_qk = idesc_f16(BF, TK, false), id_pv = idesc_f16(BF, n_pv, true);
            int base = 0, seg = 0;        // ring position of the segment's first load, segments so far
            uint32_t p_parity[2] = {0, 0};
            bool ok = true;
            auto wait_full = [&](int pos) { return mbar_wait(&sh.full[pos % NS], pos / NS & 1, &sh); };
            auto qk = [&](int st, int pos) {
                const uint32_t qa = smem_u32(qbuf + (DUAL ? st : 0) * TILE), ka = smem_u32(ring + pos % NS * TILE);
                for (int k = 0; k < k_steps; k++) {
                    const uint32_t off = (k / 4) * CHUNK + (k % 4) * 32;
                    mma_ss(tmem + TM_S + st * 128, desc_of(qa + off, 16, 1024), desc_of(ka + off, 16, 1024), id_qk, k > 0);
                }
                mma_commit(&sh.s_full[st]);
            };
            auto pv = [&](int st, int pos, bool first) {
                const uint32_t va = smem_u32(ring + pos % NS * TILE);
                for (int k = 0; k < TK / 16; k++)
                    mma_ts(tmem + TM_O + st * 128, tmem + TM_S + st * 128 + 8 * k, desc_of(va + 2048 * k, CHUNK, 1024), id_pv,
                           k > 0 || !first);
            };
            while (ok && share.next(g, groups)) {
                const int n = g.t1 - g.t0;
                for (int st = 0; ok && st < NQ; st++) ok = mbar_wait(&sh.q_ready[st], seg & 1, &sh);
                for (int i = 0; ok && i < min(LEAD, n); i++) {
                    const int pos = base + k_pos<DUAL>(i);
                    if (!(ok = wait_full(pos))) break;
                    fence_after();
                    for (int st = DUAL ? 0 : i; st < (DUAL ? 2 : i + 1); st++) qk(st, pos);
                    mma_commit(&sh.empty[pos % NS]);
                }
                for (int i = 0; ok && i < n; i++) {
                    const int vp = base + v_pos<DUAL>(i, n), kp = base + k_pos<DUAL>(i + LEAD);
                    const bool more = i + LEAD < n;
                    for (int st = DUAL ? 0 : i & 1; ok && st < (DUAL ? 2 : (i & 1) + 1); st++) {
                        if (!(ok = mbar_wait(&sh.p_ready[st], p_parity[st], &sh))) break;
                        p_parity[st] ^= 1;
                        if (!(ok = wait_full(vp))) break;
                        fence_after();
                        pv(st, vp, DUAL ? i == 0 : i < 2);
                        if (!DUAL || st == 1) mma_commit(&sh.empty[vp % NS]);
                        if (more) {
                            if (!(ok = wait_full(kp))) break;
                            qk(st, kp);
                            if (!DUAL || st == 1) mma_commit(&sh.empty[kp % NS]);
                        } else {
                            mma_commit(&sh.o_done[st]);
                        }
                    }
                }
                base += 2 * n;
                seg++;
            }
            if (!ok) {  // the MMAs in flight end before the tensor memory is freed
                atomicOr(&g_tree_status, 1u);
                sh.abort = 1;
                mma_commit(&sh.drain);
                for (long long it = 0; it < WAIT_LIMIT; it++) {
                    uint32_t done;
                    asm volatile(
                        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], 0;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
                        : "=r"(done)
                        : "r"(smem_u32(&sh.drain))
                        : "memory");
                    if (done) break;
                }
            }
        }
        __syncwarp();
    } else if (warp >= 4) {
        const int st = (warp - 4) / 4, tid = threadIdx.x - 128 - 128 * st;  // stream, row of its tile
        const uint32_t lanes = (uint32_t)(warp % 4) << 21;                  // 32 lanes to a warp
        const uint32_t tm_s = tmem + TM_S + st * 128 + lanes, tm_o = tmem + TM_O + st * 128 + lanes;
        const float c = fabsf(p.scale) * 1.4426950408889634f;
        const uint32_t flip = p.scale < 0.0f ? 0x80008000u : 0u;
        const int chunks = p.head_dim / 8;  // 16-byte pieces of a row
        int base = 0, seg = 0;
        uint32_t s_parity = 0, o_parity = 0;
        bool ok = true;
        while (ok && share.next(g, groups)) {
            const int n = g.t1 - g.t0;
            const Lengths len = lengths_of(p, g.s);
            const int32_t *parent = p.parent ? p.parent + (int64_t)g.s * p.n_node : nullptr;
            const int row = g.group * ROWS + (DUAL ? st * TR : 0) + tid;
            const bool real = row < rows;
            const int node = real ? row / rep : 0, head = g.head * rep + (real ? row - node * rep : 0);
            const bool busy = __any_sync(~0u, real);  // a warp without rows does no arithmetic
            if (DUAL || st == 0) {  // this row of Q into the swizzled tile
                const T *q = (const T *)p.q + g.s * p.q_seq + node * p.q_node + head * p.q_head;
                uint8_t *dst = qbuf + (DUAL ? st : 0) * TILE + tid * 128;
#pragma unroll
                for (int j = 0; j < HC * 8; j++) {
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (real && j < chunks) v = *(const uint4 *)(q + 8 * j);
                    v.x ^= flip, v.y ^= flip, v.z ^= flip, v.w ^= flip;
                    *(uint4 *)(dst + (j / 8) * CHUNK + (((j & 7) ^ (tid & 7)) << 4)) = v;
                }
                fence_async_smem();
                mbar_arrive(&sh.q_ready[st]);
            }
            float m = -INFINITY, l = 0.0f;
            const bool live = g.t1 * TK <= len.cached || (real && node_live(parent, node));
            for (int i = DUAL ? 0 : st; i < n; i += DUAL ? 1 : 2) {
                const int j0 = (g.t0 + i) * TK;
                const bool edge = j0 + TK > len.cached;  // not all of its keys are cached ones
                uint32_t sees[4] = {~0u, ~0u, ~0u, ~0u};
                if (edge) {
#pragma unroll
                    for (int w = 0; w < 4; w++) {
                        const int k = len.cached - j0 - 32 * w;
                        sees[w] = !live ? 0u : k >= 32 ? ~0u : k <= 0 ? 0u : (1u << k) - 1u;
                    }
                    for (int j = live ? node : -1; j >= 0; j = node_up(parent, j)) {
                        const int64_t at = (int64_t)len.past + j - j0;
                        if (at < 0 || at >= TK || len.past + (int64_t)j >= p.max_seq) continue;
#pragma unroll
                        for (int w = 0; w < 4; w++)
                            if (at >> 5 == w) sees[w] |= 1u << (at & 31);
                    }
                    // this thread's V row: nothing of it may meet a weight of zero unless it is finite
                    const int vp = base + v_pos<DUAL>(i, n);
                    if (!(ok = warp_wait(&sh.full[vp % NS], vp / NS & 1, &sh))) break;
                    const int j = j0 + tid;
                    if (j >= len.cached) {
                        uint4 *v = (uint4 *)(ring + vp % NS * TILE + tid * 128);
                        const bool gone = j >= len.keys || !node_live(parent, j - len.past);
#pragma unroll
                        for (int e = 0; e < HC * 8; e++) {
                            uint4 *at = v + (e / 8) * (CHUNK / 16) + (e & 7);
                            const uint4 x = *at;
                            const uint4 y = gone ? make_uint4(0, 0, 0, 0)
                                                 : make_uint4(finite2<T>(x.x), finite2<T>(x.y), finite2<T>(x.z), finite2<T>(x.w));
                            if (x.x != y.x || x.y != y.y || x.z != y.z || x.w != y.w) {
                                *at = y;
                                if (!gone) *(volatile int *)&sh.odd = seg + 1;
                            }
                        }
                    }
                    fence_async_smem();
                }
                if (!(ok = warp_wait(&sh.s_full[st], s_parity, &sh))) break;
                s_parity ^= 1;
                fence_after();
                if (busy) {
                    float s[TK];
#pragma unroll
                    for (int w = 0; w < 4; w++) tmem_ld(tm_s + 32 * w, s + 32 * w);
                    tmem_ld_wait();
                    if (edge) {
#pragma unroll
                        for (int k = 0; k < TK; k++)
                            if (!(sees[k >> 5] >> (k & 31) & 1)) s[k] = -INFINITY;
                    }
                    float x0 = s[0], x1 = s[1], x2 = s[2], x3 = s[3];
#pragma unroll
                    for (int k = 4; k < TK; k += 4) {
                        x0 = fmaxf(x0, s[k]), x1 = fmaxf(x1, s[k + 1]);
                        x2 = fmaxf(x2, s[k + 2]), x3 = fmaxf(x3, s[k + 3]);
                    }
                    const float top = fmaxf(m, fmaxf(fmaxf(x0, x1), fmaxf(x2, x3)) * c);
                    if (__any_sync(~0u, top > m + GROWTH)) {
                        const float f = m == -INFINITY ? 0.0f : exp2_fast(m - top);
                        l *= f;
                        m = top;
                        if (i >= (DUAL ? 1 : 2)) {  // O holds something (the S that has arrived came after the last P V)
                            for (int d = 0; d < n_pv; d += 32) {
                                float o[32];
                                tmem_ld(tm_o + d, o);
                                tmem_ld_wait();
#pragma unroll
                                for (int e = 0; e < 32; e++) o[e] *= f;
                                tmem_st(tm_o + d, (const uint32_t *)o);
                            }
                        }
                    }
                    const float off = m == -INFINITY ? 0.0f : m;
                    float l0 = 0.0f, l1 = 0.0f, l2 = 0.0f, l3 = 0.0f;
                    uint32_t w[TK / 2];
#pragma unroll
                    for (int k = 0; k < TK; k += 4) {
                        const float e0 = exp2_fast(fmaf(s[k], c, -off)), e1 = exp2_fast(fmaf(s[k + 1], c, -off));
                        const float e2 = exp2_fast(fmaf(s[k + 2], c, -off)), e3 = exp2_fast(fmaf(s[k + 3], c, -off));
                        l0 += e0, l1 += e1, l2 += e2, l3 += e3;
                        w[k / 2] = pack2<T>(e0, e1);
                        w[k / 2 + 1] = pack2<T>(e2, e3);
                    }
                    l += (l0 + l1) + (l2 + l3);
                    tmem_st(tm_s, w);
                    tmem_st(tm_s + 32, w + 32);
                    tmem_st_wait();
                }
                fence_before();
                mbar_arrive(&sh.p_ready[st]);
            }
            if (!ok) break;
            // the segment's end: O of this stream, or of both, is complete
            if (DUAL || st < n) {
                if (!(ok = warp_wait(&sh.o_done[st], o_parity, &sh))) break;
                o_parity ^= 1;
            }
            fence_after();
            float f = 1.0f, f1 = 0.0f;  // factors of this stream's O and the other's
            if (!DUAL) {
                if (st == 1) {
                    sh.ml[tid] = make_float2(m, l);
                    fence_before();
                    mbar_arrive(&sh.merge_full);
                    if (!(ok = warp_wait(&sh.merge_done, seg & 1, &sh))) break;
                    seg++;
                    base += 2 * n;
                    continue;
                }
                if (!(ok = warp_wait(&sh.merge_full, seg & 1, &sh))) break;
                fence_after();
                const float2 other = sh.ml[tid];
                const float top = fmaxf(m, other.x);
                f = m == -INFINITY ? 0.0f : exp2_fast(m - top);
                f1 = other.x == -INFINITY ? 0.0f : exp2_fast(other.x - top);
                l = l * f + other.y * f1;
                m = top;
            }
            if (busy) {
                const bool whole = g.t0 == 0 && g.t1 == g.tiles;
                const int in_group = (DUAL ? st * TR : 0) + tid;
                const int64_t slot = 2 * blockIdx.x + (seg > 0);
                const bool odd = *(volatile int *)&sh.odd == seg + 1;
                const float inv = whole ? (live && l != 0.0f ? 1.0f / l : 0.0f) : 1.0f;
                if (real && !whole) part_ml[slot * ROWS + in_group] = make_float2(m, live ? l : -1.0f);
                T *out = (T *)p.out + g.s * p.out_seq + node * p.out_node + head * p.out_head;
                for (int d = 0; d < p.head_dim; d += 32) {
                    float o[32], o1[32];
                    __syncwarp();
                    tmem_ld(tm_o + d, o);
                    if (!DUAL) tmem_ld(tm_o + 128 + d, o1);
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 32; e++) {
                        o[e] = f == 0.0f ? 0.0f : o[e] * f;
                        if (!DUAL && f1 != 0.0f) o[e] += o1[e] * f1;
                    }
                    if (odd && live) {  // what this row sees of the values that were left out
                        const T *v = (const T *)p.v_cache + g.s * p.cache_seq + g.head * p.cache_head + d;
                        for (int j = node; j >= 0; j = node_up(parent, j)) {
                            const int64_t r = (int64_t)len.past + j;
                            if (r < (int64_t)g.t0 * TK || r >= (int64_t)g.t1 * TK || r >= p.max_seq) continue;
#pragma unroll
                            for (int e = 0; e < 32; e++) {
                                const float x = d + e < p.head_dim ? to_f32(v[r * p.cache_row + e]) : 0.0f;
                                if (!isfinite(x)) o[e] += x;
                            }
                        }
                    }
                    if (real && whole) {
#pragma unroll
                        for (int e = 0; e < 32; e += 8)
                            if (d + e < p.head_dim) {
                                // a padding node's zero, whatever its sums hold
#pragma unroll
                                for (int b = 0; b < 8; b++) o[e + b] = inv == 0.0f ? 0.0f : o[e + b] * inv;
                                *(uint4 *)(out + d + e) = make_uint4(pack2<T>(o[e], o[e + 1]), pack2<T>(o[e + 2], o[e + 3]),
                                                                     pack2<T>(o[e + 4], o[e + 5]), pack2<T>(o[e + 6], o[e + 7]));
                            }
                    } else if (real) {
                        float4 *dst = (float4 *)part_o + (slot * (p.head_dim / 4) + d / 4) * ROWS + in_group;
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            if (d + e < p.head_dim) dst[(e / 4) * ROWS] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                    }
                }
            }
            __syncwarp();
            fence_before();
            if (!DUAL) mbar_arrive(&sh.merge_done);
            seg++;
            base += 2 * n;
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem));
}

// cuTensorMapEncodeTiled, looked up in the driver so that the library loads without one.
PFN_cuTensorMapEncodeTiled_v12000 encoder() {
    static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &r) != cudaSuccess ||
            r != cudaDriverEntryPointSuccess)
            f = nullptr;
        return (PFN_cuTensorMapEncodeTiled_v12000)f;
    }();
    return fn;
}

// Strides of axes of one element may be anything; the map wants sensible ones.
cuuint64_t map_stride(int64_t stride, int64_t count, int64_t head_dim) { return 2 * (cuuint64_t)(count > 1 ? stride : (head_dim + 7) / 8 * 8); }

bool cache_map(CUtensorMap *m, const sdy_tree_attention_args &a, const void *base) {
    const cuuint64_t dims[4] = {(cuuint64_t)a.head_dim, (cuuint64_t)a.max_seq, (cuuint64_t)a.n_kv_head, (cuuint64_t)a.n_seq};
    const cuuint64_t strides[3] = {map_stride(a.cache_row, a.max_seq, a.head_dim), map_stride(a.cache_head, a.n_kv_head, a.head_dim),
                                   map_stride(a.cache_seq, a.n_seq, a.head_dim)};
    const cuuint32_t box[4] = {64, TK, 1, 1}, step[4] = {1, 1, 1, 1};
    const auto encode = encoder();
    if (!encode) {
        set_error("sdy_tree_attention_dev: cuTensorMapEncodeTiled is missing from the driver");
        return false;
    }
    const CUresult r = encode(m, a.type == T_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                              const_cast<void *>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) set_error("sdy_tree_attention_dev: cuTensorMapEncodeTiled failed (%d)", (int)r);
    return r == CUDA_SUCCESS;
}

template <class T, bool DUAL, int HC>
void tc_launch(const sdy_tree_attention_args &a, const TreeSpace &sp, const CUtensorMap &k, const CUtensorMap &v, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    smem_limit_once(tree_tc_kernel<T, DUAL, HC>, tc_smem(DUAL, HC), done);
    launch(tree_tc_kernel<T, DUAL, HC>, TA_CTAS, TT, tc_smem(DUAL, HC), s, a, k, v, sp.base, sp.o, sp.ml);
    SDY_LAUNCHED();
}
template <class T>
void tc_pick(const sdy_tree_attention_args &a, const TreeSpace &sp, const CUtensorMap &k, const CUtensorMap &v, cudaStream_t s) {
    const bool dual = tree_tc_rows(a) > TR;
    if (a.head_dim <= 64) dual ? tc_launch<T, true, 1>(a, sp, k, v, s) : tc_launch<T, false, 1>(a, sp, k, v, s);
    else dual ? tc_launch<T, true, 2>(a, sp, k, v, s) : tc_launch<T, false, 2>(a, sp, k, v, s);
}

}  // namespace

bool tree_tc_takes(const sdy_tree_attention_args &a) {
    auto mappable = [](int64_t stride, int64_t count) { return count == 1 || (stride > 0 && stride < (int64_t)1 << 39); };
    return a.type != T_F32 && a.head_dim <= 128 && mappable(a.cache_row, a.max_seq) && mappable(a.cache_head, a.n_kv_head) &&
           mappable(a.cache_seq, a.n_seq);
}

int tree_tc_rows(const sdy_tree_attention_args &a) { return a.n_node * (a.n_head / a.n_kv_head) > TR ? 2 * TR : TR; }

void tree_tc(const sdy_tree_attention_args &a, cudaStream_t s) {
    CUtensorMap k, v;
    if (!cache_map(&k, a, a.k_cache) || !cache_map(&v, a, a.v_cache)) return;
    const TreeSpace sp = tree_space(a, tree_tc_rows(a));
    if (a.type == T_F16) tc_pick<__half>(a, sp, k, v, s);
    else tc_pick<__nv_bfloat16>(a, sp, k, v, s);
    tree_join(a, sp, tree_tc_rows(a), TA_CTAS, s);
}

unsigned tree_tc_status() {
    unsigned v = 0;
    if (cudaMemcpyFromSymbol(&v, g_tree_status, sizeof v) != cudaSuccess) return ~0u;
    return v;
}
void tree_tc_clear_status() {
    const unsigned z = 0;
    SDY_CUDA(cudaMemcpyToSymbol(g_tree_status, &z, sizeof z));
}

}  // namespace sdy
