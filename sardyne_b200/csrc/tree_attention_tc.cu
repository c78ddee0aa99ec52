// Tree attention over 16-bit caches on the tensor cores (tcgen05, accumulators in TMEM).
//
// For one KV head of one sequence the rows are its (node, query head) pairs, 128 to an MMA tile;
// per tile of 128 keys, S = Q K^T (128 x 128, f32 in TMEM), P = 2^(c S - m) as 16-bit values over S's
// own columns, O += P V with P as the A operand. P takes the type of V because one tcgen05.mma has one
// type for both; its rounding (2^-9 of a probability in bf16, 2^-12 in f16) is of the size of the
// output's own and adds to it as independent errors do: 1.4 times the output's rounding in all. m is a
// row's running maximum; O and the sum are rescaled only when it has grown by more than 2^8 since it
// was last set (the division by the sum takes out any common factor; 2^8 keeps P inside the range of
// f16), which after the first tiles hardly ever happens, so O stays in TMEM.
//
// One CTA per SM, twelve warps: a TMA producer (K and V tiles through rings of shared memory slots),
// an MMA issuer, one that notes the cuts and fetches queries ahead, and two streams of four warps that
// turn S into P, one row to a thread. With more than 128 rows the streams hold two row tiles and share
// every K and V tile (DUAL); with fewer they share the rows and take the tiles in turn, and the first
// stream joins the two results at the end.
//
// What bounds it, for many rows, is a stream's cycle: the exponentials (128 x 128 at 16 a cycle are 1024
// cycles; with the reads of S, the maxima and the stores of P 2000), then P V and the next Q K^T (512
// cycles each alone; Q K^T reads 128 bytes of shared memory a cycle, all there is, and loses some to the
// arriving tiles), the other stream's MMAs under this one's exponentials: 3360 cycles per 2 x 128 rows
// and 128 keys, 0.61 of the tensor pipe's rate, and the power limit then holds the clock near 1.66 GHz (2
// sequences of 64 nodes and 32 heads over 65537 keys: 165 us, 830 TFLOP/s). Tried and slower: S of 80
// keys beside P, with the next Q K^T under the exponentials (four waits more per key, and a wait on a
// barrier that is complete takes 100 to 200 cycles of an issuer that cannot run ahead: 4100 cycles per
// 128 keys); the scores in four parts, each part's maximum under the one before's exponentials (a
// vote per part: 3900). For few rows it is bound by latency: about 12 us from the launch to the last store,
// of which loading the queries, the first tile and storing the result take 2 us each.
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
// Tiles that the rest of a row group takes the time of: 16 sequences of 24 nodes, up to 8192 keys, and 21 of
// 13 over up to 5285 take 68.2 and 55.8 us with 3, 62.4 and 48.3 with 6, 63.6 and 47.5 with 9.
constexpr int T_SETUP = 6;
constexpr int CHUNK = TK * 128, QCHUNK = TR * 128;  // bytes of 64 elements of a tile's rows, 128-byte swizzled
constexpr int WAIT_LIMIT = 1 << 22;  // mbarrier polls before giving up (about a second)
// TMEM columns of stream 0's S (and P over it) and O; stream 1's are 128 on.
constexpr uint32_t TM_S = 0, TM_O = 256;
constexpr float GROWTH = 8.0f;

__device__ unsigned g_tree_status;  // nonzero: a wait ran out

constexpr int SLOTS = 12;  // ring slots, at most
// Slots of a ring: one ring for both streams (DUAL), or one for each.
constexpr int tc_slots(bool dual, int hc) { return dual ? 10 / hc : 6 / hc; }
constexpr int tc_smem(bool dual, int hc) { return (dual ? 2 : 1) * hc * QCHUNK + (dual ? 1 : 2) * tc_slots(dual, hc) * hc * CHUNK; }

struct Shared {
    uint64_t full[SLOTS], empty[SLOTS];
    uint64_t q_ready[2], s_full[2], p_ready[2], o_done[2];
    uint64_t merge_full, merge_done, drain;
    uint32_t tmem;
    int odd;  // the last segment (from 1) whose drafted V rows hold NaN or infinities
    int64_t scan[TT / 32 + 8];
    int16_t up[2][TA_MAX_NODES];  // per stream (its warps are in one segment while they walk)
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
// Bounded: false when the limit ran out. A few instructions only: the code of the roles shares the
// instruction caches, and the MMA issuer's waits are on the critical path.
__device__ __forceinline__ bool mbar_wait(uint64_t *b, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .u32 n;\n\tmov.u32 n, %3;\n"
        "again:\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "@p bra done;\n\t"
        "sub.u32 n, n, 1;\n\t"
        "setp.ne.u32 p, n, 0;\n\t"
        "@p bra again;\n"
        "done:\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(ok)
        : "r"(smem_u32(b)), "r"(parity), "n"(WAIT_LIMIT)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool warp_wait(uint64_t *b, uint32_t parity) { return __all_sync(~0u, mbar_wait(b, parity)); }

__device__ __forceinline__ void tma_tile(const CUtensorMap *map, uint64_t *bar, uint32_t dst, int x, int row, int head, int s) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];\n" ::"r"(dst),
        "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(row), "r"(head), "r"(s)
        : "memory");
}

// Shared memory descriptors of tiles in the 128-byte swizzle: K-major (Q and K: 8-row groups of
// 1024 bytes) and N-major (V: 64-element chunks at CHUNK, 8-key groups of 1024 bytes).
// The low word holds the address and LBO, the high word SBO, the version and the swizzle.
constexpr uint32_t DESC_HI = 1024 >> 4 | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) { return (addr >> 4) | (lbo >> 4) << 16; }
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(one));
    return one != 0;
}
// kind::f16: f32 accumulator, A and B of one 16-bit type, M = 128; b_mn: B is N-major.
__device__ __forceinline__ uint32_t idesc_f16(bool bf16, int n, bool b_mn) {
    return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (b_mn ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(TR >> 4) << 24;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(DESC_HI)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 y, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(DESC_HI)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t *b) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(smem_u32(b)) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }

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
__device__ __forceinline__ void tmem_ld16(uint32_t addr, float *v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
                 "[%16];\n"
                 : OUT4(v, 0), OUT4(v, 4), OUT4(v, 8), OUT4(v, 12)
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
                 "%14, %15};\n" ::IN4(v, 0), IN4(v, 4), IN4(v, 8), IN4(v, 12), "r"(addr)
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
// Nonzero when one of two packed 16-bit values is NaN or infinite (an exponent of ones: adding one
// to it carries into the sign's place), and the pair with such values replaced by zero.
template <class T> __device__ __forceinline__ uint32_t infinite2(uint32_t w) {
    constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7C007C00u : 0x7F807F80u, ONE = E & ~(E << 1);
    return ((w & E) + ONE) & 0x80008000u;
}
template <class T> __device__ __forceinline__ uint32_t finite2(uint32_t w) {
    const uint32_t bad = infinite2<T>(w);
    return w & ~((bad & 0x8000u ? 0xFFFFu : 0u) | (bad & 0x80000000u ? 0xFFFF0000u : 0u));
}

// The paths of up to 64 nodes by pointer doubling over the warp, which holds the nodes above lane and
// lane + 32 in up[]: after k rounds a node knows 2^k nodes of its way. `path` is that of `node`,
// `alive` has the nodes whose way ends in a root.
__device__ __forceinline__ void warp_paths(const int (&above)[2], int n_node, int node, uint64_t &path, uint64_t &alive) {
    const int lane = threadIdx.x % 32;
    int up[2] = {above[0], above[1]};
    uint64_t bits[2] = {1ull << lane, 1ull << (lane + 32)};
    const bool wide = n_node > 32;
    for (int hop = 1; hop < n_node; hop *= 2) {
        int to[2];
        uint64_t more[2];
#pragma unroll
        for (int w = 0; w < 2; w++) {
            to[w] = -2, more[w] = 0;
            if (w && !wide) continue;
            const int from = up[w] & 31;
            const int t0 = __shfl_sync(~0u, up[0], from);
            const uint64_t b0 = __shfl_sync(~0u, bits[0], from);
            to[w] = t0, more[w] = b0;
            if (wide) {
                const int t1 = __shfl_sync(~0u, up[1], from);
                const uint64_t b1 = __shfl_sync(~0u, bits[1], from);
                if (up[w] >= 32) to[w] = t1, more[w] = b1;
            }
        }
#pragma unroll
        for (int w = 0; w < 2; w++)
            if (up[w] >= 0) {
                bits[w] |= more[w];
                up[w] = to[w];
            }
    }
    const uint64_t p0 = __shfl_sync(~0u, bits[0], node & 31), p1 = __shfl_sync(~0u, bits[1], node & 31);
    path = node < 32 ? p0 : p1;
    alive = __ballot_sync(~0u, up[0] == -1) | (uint64_t)__ballot_sync(~0u, wide && up[1] == -1) << 32;
}

template <class T, bool DUAL, int HC>
__global__ void __launch_bounds__(TT, 1)
    tree_tc_kernel(const sdy_tree_attention_args p, const __grid_constant__ CUtensorMap kmap,
                   const __grid_constant__ CUtensorMap vmap, Cut *cuts, float *part_o, float2 *part_ml) {
    constexpr int NQ = DUAL ? 2 : 1, STEP = DUAL ? 1 : 2;  // a stream takes every STEP-th tile
    constexpr int NS = tc_slots(DUAL, HC);                  // slots of a ring: K, V, K, V, .. of its tiles
    constexpr int TILE = HC * CHUNK, QTILE = HC * QCHUNK, ROWS = NQ * TR;
    constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
    __shared__ Shared sh;
    extern __shared__ __align__(1024) uint8_t qbuf[];
    uint8_t *ring = qbuf + NQ * QTILE;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int rep = p.n_head / p.n_kv_head, rows = p.n_node * rep, groups = (rows + ROWS - 1) / ROWS;
    const int n_pv = (p.head_dim + 15) & ~15, k_steps = (p.head_dim + 15) / 16;

    if (warp == 3 && lane == 0) {
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(&kmap) : "memory");
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(&vmap) : "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(smem_u32(&sh.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < NS * STEP; i++) mbar_init(&sh.full[i], 1), mbar_init(&sh.empty[i], 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(&sh.q_ready[i], TR), mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.p_ready[i], TR), mbar_init(&sh.o_done[i], 1);
        }
        mbar_init(&sh.merge_full, TR), mbar_init(&sh.merge_done, TR), mbar_init(&sh.drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        sh.odd = 0;
    }
    pdl_wait();
    int64_t found[8];
    find_share<TK, TT, T_SETUP>(p, p.n_kv_head * groups, blockIdx.x, sh.scan, found);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = sh.tmem;
    Share<TK> share(p, found, p.n_kv_head * groups);
    Segment g;
    bool more = share.next(g, groups);  // (the first run here, by the same instructions in all roles)

    // registers go to the two warpgroups that hold rows: 72 x 128 + 216 x 256 <= 168 x 384
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;\n" ::);
        if (warp == 0 && lane == 0) {
            int pos[STEP] = {}, event[STEP] = {};  // loads and arrivals so far, per ring
            bool ok = true, begun = false;
            // the stream's tile i into the next slot of ring r, with `bytes` more to come on the arrival
            auto load = [&](const CUtensorMap *map, int r, int i, int bytes) {
                const int slot = r * NS + pos[r] % NS, turn = pos[r] / NS;
                uint64_t *full = &sh.full[r * NS + event[r] % NS];
                if (turn && !mbar_wait(&sh.empty[slot], (turn - 1) & 1)) return false;
                if (bytes) mbar_expect(full, bytes);
                for (int c = 0; c < HC; c++)
                    tma_tile(map, full, smem_u32(ring + slot * TILE + c * CHUNK), 64 * c, (g.t0 + i * STEP + r) * TK, g.head, g.s);
                pos[r]++;
                return true;
            };
            for (; ok && more; more = share.next(g, groups)) {
                const int n = g.t1 - g.t0;
#pragma unroll
                for (int r = 0; r < STEP; r++)
                    if (r < n) ok = ok && load(&kmap, r, 0, TILE), event[r]++;
                // the first queries do not queue behind rings full of tiles
                if (!begun) ok = ok && mbar_wait(&sh.q_ready[0], 0) && (!DUAL || mbar_wait(&sh.q_ready[1], 0));
                begun = true;
                for (int i = 0; ok && i * STEP < n; i++) {
#pragma unroll
                    for (int r = 0; r < STEP; r++) {  // V, and the K that follows it, arrive together
                        if (i * STEP + r >= n) continue;
                        const bool last = (i + 1) * STEP + r >= n;
                        ok = ok && load(&vmap, r, i, last ? TILE : 2 * TILE);
                        if (!last) ok = ok && load(&kmap, r, i + 1, 0);
                        event[r]++;
                    }
                }
            }
            if (!ok) {  // let the copies in flight land before the memory is given up
                atomicOr(&g_tree_status, 1u);
                for (int r = 0; r < STEP; r++)
                    for (int q = max(0, event[r] - NS); q < event[r]; q++) mbar_wait(&sh.full[r * NS + q % NS], q / NS & 1);
            }
        }
        if (warp == 3 && lane == 0) note_cut<TK>(p, p.n_kv_head * groups, groups, blockIdx.x, found, cuts);
        if (warp == 3) {  // the queries of the share into L2, ahead of the loads that keep HBM busy
            for (; more; more = share.next(g, groups)) {
                const int first = g.group * ROWS, last = min(rows, first + ROWS);
                for (int r = first + lane; r < last; r += 32) {
                    const int node = r / rep;
                    const T *q = (const T *)p.q + g.s * p.q_seq + node * p.q_node + (g.head * rep + r - node * rep) * p.q_head;
                    for (int e = 0; e < p.head_dim; e += 64) asm volatile("prefetch.global.L2 [%0];\n" ::"l"(q + e));
                }
            }
        }
        if (warp == 1) {
            // One warp issues for both streams in turn, which keeps them out of step: the one's MMAs run
            // under the other's exponentials (with a warp for each they fall into step and share both
            // pipes: 4600 cycles per 128 keys instead of 3400). The whole warp waits, one lane issues; the
            // shuffles tell the compiler that the operands are the same in all lanes (the tensor
            // instructions take them from uniform registers).
            auto uniform = [](uint32_t x) { return __shfl_sync(~0u, x, 0); };
            const uint32_t id_qk = uniform(idesc_f16(BF, TK, false)), id_pv = uniform(idesc_f16(BF, n_pv, true));
            const uint32_t q_lo = uniform(desc_lo(smem_u32(qbuf), 16)), steps = uniform(k_steps), tm = uniform(tmem);
            const uint32_t k_lo = uniform(desc_lo(smem_u32(ring), 16)), v_lo = uniform(desc_lo(smem_u32(ring), CHUNK));
            int pos[2] = {}, event[2] = {}, seg = 0;  // loads and arrivals taken, per stream; segments so far
            uint32_t p_parity = 0;
            bool ok = true;
            auto slot_of = [&](int st, int at) { return (DUAL ? 0 : st * NS) + at % NS; };
            auto wait_full = [&](int st, int e) { return warp_wait(&sh.full[slot_of(st, e)], e / NS & 1); };
            auto qk = [&](int st, uint32_t b, uint64_t *free) {
                const uint32_t a = q_lo + (DUAL ? st : 0) * (QTILE >> 4), d = tm + TM_S + st * 128;
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < 4 * HC; k++)
                        if (k < steps)
                            mma_ss(d, a + (((k / 4) * QCHUNK + (k % 4) * 32) >> 4), b + (((k / 4) * CHUNK + (k % 4) * 32) >> 4), id_qk, k > 0);
                    mma_commit(&sh.s_full[st]);
                    if (!DUAL || st == 1) mma_commit(free);
                }
            };
            for (; ok && more; more = share.next(g, groups)) {
                const int all = g.t1 - g.t0;
                auto tiles = [&](int st) { return DUAL ? all : (all + 1 - st) / 2; };  // of a stream
                for (int st = 0; ok && st < NQ; st++) ok = warp_wait(&sh.q_ready[st], seg & 1);
                fence_after();
#pragma unroll
                for (int st = 0; st < 2; st++) {
                    if (!ok || !tiles(st)) continue;
                    const int slot = slot_of(st, pos[st]);
                    if ((ok = wait_full(st, event[st]))) qk(st, uniform(k_lo + slot * (TILE >> 4)), &sh.empty[slot]);
                    pos[st]++, event[st]++;
                }
                for (int i = 0; ok && i < tiles(0); i++) {
#pragma unroll
                    for (int st = 0; st < 2; st++) {
                        if (!ok || i >= tiles(st)) continue;
                        const bool last = i + 1 == tiles(st);
                        const int v_slot = slot_of(st, pos[st]), k_slot = slot_of(st, pos[st] + 1);
                        const uint32_t v = uniform(v_lo + v_slot * (TILE >> 4)), k = uniform(k_lo + k_slot * (TILE >> 4)), again = uniform(i > 0);
                        if (!DUAL || st == 0) ok = wait_full(st, event[st]);
                        pos[st] += last ? 1 : 2, event[st]++;
                        ok = ok && warp_wait(&sh.p_ready[st], p_parity >> st & 1);
                        if (!ok) continue;
                        p_parity ^= 1u << st;
                        fence_after();
                        if (elect_one()) {
                            const uint32_t d = tm + TM_O + st * 128, a = tm + TM_S + st * 128;
#pragma unroll
                            for (int c = 0; c < TK / 16; c++) mma_ts(d, a + 8 * c, v + (2048 * c >> 4), id_pv, c > 0 ? 1u : again);
                            if (!DUAL || st == 1) mma_commit(&sh.empty[v_slot]);
                            if (last) mma_commit(&sh.o_done[st]);
                        }
                        if (!last) qk(st, k, &sh.empty[k_slot]);  // over P, which the MMAs before have read by then
                    }
                }
                seg++;
            }
            if (!ok) {  // the MMAs in flight end before the tensor memory is freed
                if (lane == 0) atomicOr(&g_tree_status, 1u);
                if (elect_one()) mma_commit(&sh.drain);
                warp_wait(&sh.drain, 0);
            }
        }
        __syncwarp();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;\n" ::);
        const int st = (warp - 4) / 4, tid = threadIdx.x - 128 - 128 * st;  // stream, row of its tile
        const uint32_t lanes = (uint32_t)(warp % 4) << 21;                  // 32 lanes to a warp
        const uint32_t tm_s = tmem + TM_S + st * 128 + lanes, tm_o = tmem + TM_O + st * 128 + lanes;
        // (a scale of zero: queries of zero, since a masked score's -inf times zero would be NaN)
        const float c = p.scale == 0.0f ? 1.0f : fabsf(p.scale) * 1.4426950408889634f;
        const uint32_t flip = p.scale < 0.0f ? 0x80008000u : 0u;
        const int chunks = p.head_dim / 8;  // 16-byte pieces of a row
        int base = 0, arrived = 0, seg = 0;  // loads, arrivals and segments before this one
        uint32_t s_parity = 0, o_parity = 0;
        bool ok = true;
        for (; ok && more; more = share.next(g, groups)) {
            const int n = (g.t1 - g.t0 + STEP - 1 - (DUAL ? 0 : st)) / STEP;  // the stream's tiles
            const Lengths len = lengths_of(p, g.s, g.past);
            const int32_t *parent = p.parent ? p.parent + (int64_t)g.s * p.n_node : nullptr;
            const int row = g.group * ROWS + (DUAL ? st * TR : 0) + tid;
            const bool real = row < rows;
            const int node = real ? row / rep : 0, head = g.head * rep + (real ? row - node * rep : 0);
            const bool busy = __any_sync(~0u, real);  // a warp without rows does no arithmetic
            const bool edges = g.t1 * TK > len.cached;  // drafted rows, or none at all, in the last tiles
            int parent_of[2] = {-2, -2};                // of nodes lane and lane + 32
            if (edges && p.n_node <= 64)
                for (int w = 0; w < 2; w++)
                    if (lane + 32 * w < p.n_node) parent_of[w] = node_up(parent, lane + 32 * w);
            const int64_t q_at = g.s * p.q_seq + node * p.q_node + head * p.q_head;
            if (DUAL || st == 0) {  // the warp's rows of Q into the swizzled tile, a run of lanes to a row
                constexpr int PER = HC * 8;  // lanes to a row: 16 bytes each
                uint8_t *dst = qbuf + (DUAL ? st : 0) * QTILE + (warp % 4) * 32 * 128;
                const int j = lane % PER, rows_left = rows - (row - lane);
                // (copies, so that all are in flight at once; what is no query is zero)
#pragma unroll
                for (int i = 0; i < PER; i++) {
                    const int r = i * (32 / PER) + lane / PER;
                    const int64_t at = __shfl_sync(~0u, q_at, r);
                    const bool some = r < rows_left && j < chunks && p.scale != 0.0f;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(
                                     smem_u32(dst + r * 128 + (j / 8) * QCHUNK + (((j & 7) ^ (r & 7)) << 4))),
                                 "l"((const uint4 *)((const T *)p.q + (some ? at : 0)) + (some ? j : 0)), "r"(some ? 16 : 0)
                                 : "memory");
                }
                asm volatile("cp.async.wait_all;\n" ::: "memory");
                if (flip) {
#pragma unroll 1
                    for (int i = 0; i < PER; i++) {
                        const int r = i * (32 / PER) + lane / PER;
                        uint4 *x = (uint4 *)(dst + r * 128 + (j / 8) * QCHUNK + (((j & 7) ^ (r & 7)) << 4));
                        *x = make_uint4(x->x ^ flip, x->y ^ flip, x->z ^ flip, x->w ^ flip);
                    }
                }
                fence_async_smem();
                mbar_arrive(&sh.q_ready[st]);
            }
            float m = -INFINITY, l = 0.0f;
            bool live = true;
            uint64_t path = 0, alive = 0;  // up to 64 nodes: this row's path, and the nodes that are no padding
            if (edges && p.n_node <= 64) {
                warp_paths(parent_of, p.n_node, node, path, alive);
                if (len.keys - len.past < 64) path &= len.keys > len.past ? (1ull << (len.keys - len.past)) - 1 : 0;
                live = real && (alive >> node & 1);
            } else if (edges) {
                load_tree(sh.up[st], parent, p.n_node);
                live = walk_tree(sh.up[st], real ? node : -2, [](int) {});
                __syncwarp();
            }
            for (int i = 0; i < n; i++) {
                const int j0 = (g.t0 + (DUAL ? i : 2 * i + st)) * TK;
                const bool edge = j0 + TK > len.cached;  // not all of its keys are cached ones
                constexpr int MW = (TK + 31) / 32;
                uint32_t sees[MW];  // the keys this row sees
#pragma unroll
                for (int w = 0; w < MW; w++) sees[w] = ~0u;
                if (edge) {
#pragma unroll
                    for (int w = 0; w < MW; w++) {
                        const int k = len.cached - j0 - 32 * w;
                        sees[w] = !live ? 0u : k >= 32 ? ~0u : k <= 0 ? 0u : (1u << k) - 1u;
                    }
                    if (p.n_node <= 64) {
                        const uint64_t mine = live ? path : 0;
                        const int at = len.past - j0;  // of node 0, from -63 on where any is in this tile
#pragma unroll
                        for (int w = 0; w < MW; w++) {
                            const int up = at - 32 * w;
                            if (up >= 0 && up < 32) sees[w] |= (uint32_t)(mine << up);
                            if (up < 0 && up > -64) sees[w] |= (uint32_t)(mine >> -up);
                        }
                    } else {
                        walk_tree(sh.up[st], live && real ? node : -1, [&](int j) {
                            const int64_t row_at = (int64_t)len.past + j, at = row_at - j0;
                            if (at < 0 || at >= TK || row_at >= p.max_seq) return;
#pragma unroll
                            for (int w = 0; w < MW; w++)
                                if (at >> 5 == w) sees[w] |= 1u << (at & 31);
                        });
                        __syncwarp();
                    }
                    // The warp's V rows: nothing of them may meet a weight of zero unless it is finite.
                    const int vp = base + 2 * i + 1, slot = (DUAL ? 0 : st * NS) + vp % NS, ve = arrived + 1 + i;
                    if (!(ok = warp_wait(&sh.full[(DUAL ? 0 : st * NS) + ve % NS], ve / NS & 1))) break;
                    const int j = j0 + tid, d = j - len.past;
                    const bool drafted = j >= len.cached && j < len.keys;
                    const bool keep = tid >= TK || j < len.cached || (drafted && (p.n_node <= 64 ? alive >> d & 1 : walk_tree(sh.up[st], d, [](int) {})));
                    const uint32_t gone = ~__ballot_sync(~0u, keep), look = __ballot_sync(~0u, tid < TK && drafted && keep);
                    if (gone | look) {
                        constexpr int PER = HC * 8;  // lanes to a row: 16 bytes each
                        const int e = lane % PER;
                        uint4 *v = (uint4 *)(ring + slot * TILE + (warp % 4) * 32 * 128 + (e / 8) * CHUNK) + (e & 7);
                        uint32_t bad = 0;
#pragma unroll
                        for (int r = lane / PER; r < 32; r += 32 / PER) {
                            if (look >> r & 1) {
                                const uint4 x = v[8 * r];
                                bad |= infinite2<T>(x.x) | infinite2<T>(x.y) | infinite2<T>(x.z) | infinite2<T>(x.w);
                            } else if (gone >> r & 1) {
                                v[8 * r] = make_uint4(0, 0, 0, 0);
                            }
                        }
                        if (__any_sync(~0u, bad)) {
                            for (int r = lane / PER; r < 32; r += 32 / PER)
                                if (look >> r & 1) {
                                    const uint4 x = v[8 * r];
                                    v[8 * r] = make_uint4(finite2<T>(x.x), finite2<T>(x.y), finite2<T>(x.z), finite2<T>(x.w));
                                }
                            *(volatile int *)&sh.odd = seg + 1;
                        }
                        __syncwarp();
                    }
                    fence_async_smem();
                }
                if (!(ok = warp_wait(&sh.s_full[st], s_parity))) break;
                s_parity ^= 1;
                fence_after();
                if (busy) {
                    float s[TK];
#pragma unroll
                    for (int k = 0; k < TK; k += 32) tmem_ld(tm_s + k, s + k);
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
                        if (i) {  // O holds something (the S that has arrived came after the last P V)
                            for (int d = 0; d < n_pv; d += 16) {
                                float o[16];
                                tmem_ld16(tm_o + d, o);
                                tmem_ld_wait();
#pragma unroll
                                for (int e = 0; e < 16; e++) o[e] *= f;
                                tmem_st16(tm_o + d, (const uint32_t *)o);
                            }
                        }
                    }
                    const float off = m == -INFINITY ? 0.0f : m;
                    float l0 = 0.0f, l1 = 0.0f, l2 = 0.0f, l3 = 0.0f;
#pragma unroll
                    for (int b = 0; b < TK; b += 32) {
                        uint32_t w[16];
#pragma unroll
                        for (int k = b; k < b + 32; k += 4) {
                            const float e0 = exp2_fast(fmaf(s[k], c, -off)), e1 = exp2_fast(fmaf(s[k + 1], c, -off));
                            const float e2 = exp2_fast(fmaf(s[k + 2], c, -off)), e3 = exp2_fast(fmaf(s[k + 3], c, -off));
                            l0 += e0, l1 += e1, l2 += e2, l3 += e3;
                            w[(k - b) / 2] = pack2<T>(e0, e1);
                            w[(k - b) / 2 + 1] = pack2<T>(e2, e3);
                        }
                        tmem_st16(tm_s + b / 2, w);
                    }
                    l += (l0 + l1) + (l2 + l3);
                    tmem_st_wait();
                }
                fence_before();
                mbar_arrive(&sh.p_ready[st]);
            }
            if (!ok) break;
            // the segment's end: O of this stream, then of both, is complete
            if (n) {
                if (!(ok = warp_wait(&sh.o_done[st], o_parity))) break;
                o_parity ^= 1;
            }
            fence_after();
            float f = 1.0f, f1 = 0.0f;  // factors of this stream's O and the other's
            if (!DUAL) {
                if (st == 1) {
                    sh.ml[tid] = make_float2(m, l);
                    fence_before();
                    mbar_arrive(&sh.merge_full);
                    if (!(ok = warp_wait(&sh.merge_done, seg & 1))) break;
                    seg++;
                    base += 2 * n, arrived += n ? n + 1 : 0;
                    continue;
                }
                if (!(ok = warp_wait(&sh.merge_full, seg & 1))) break;
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
                uint8_t *stage = qbuf + (DUAL ? st : 0) * QTILE + (warp % 4) * 32 * 128;  // the rows of Q, no longer needed
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
                    if (odd) {  // what this row sees of the values that were left out
                        const T *v = (const T *)p.v_cache + g.s * p.cache_seq + g.head * p.cache_head + d;
                        for (int j = live && real ? node : -1; j >= 0; j = node_up(parent, j)) {
                            const int64_t r = (int64_t)len.past + j;
                            if (r < (int64_t)g.t0 * TK || r >= (int64_t)g.t1 * TK || r >= p.max_seq) continue;
#pragma unroll
                            for (int e = 0; e < 32; e++) {
                                const float x = d + e < p.head_dim ? to_f32(v[r * p.cache_row + e]) : 0.0f;
                                if (!isfinite(x)) o[e] += x;
                            }
                        }
                    }
                    if (whole) {
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            // a padding node's zero, whatever its sums hold
#pragma unroll
                            for (int b = 0; b < 8; b++) o[e + b] = inv == 0.0f ? 0.0f : o[e + b] * inv;
                            const int piece = (d + e) / 8;
                            *(uint4 *)(stage + lane * 128 + (piece / 8) * QCHUNK + (((piece & 7) ^ (lane & 7)) << 4)) =
                                make_uint4(pack2<T>(o[e], o[e + 1]), pack2<T>(o[e + 2], o[e + 3]), pack2<T>(o[e + 4], o[e + 5]),
                                           pack2<T>(o[e + 6], o[e + 7]));
                        }
                    } else {  // 32 elements of 32 rows through shared memory, so that rows are written in runs
                        __syncwarp();
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            *(float4 *)(stage + lane * 128 + (((e / 4) ^ (lane & 7)) << 4)) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                        __syncwarp();
                        const int e = lane % 8, rows_left = rows - (row - lane);
                        float *dst = part_o + slot * part_stride(ROWS, p.head_dim) + (int64_t)(in_group - lane) * p.head_dim + d + 4 * e;
                        if (d + 4 * e < p.head_dim)
#pragma unroll
                            for (int r = lane / 8; r < 32; r += 4)
                                if (r < rows_left)
                                    *(float4 *)(dst + r * p.head_dim) = *(const float4 *)(stage + r * 128 + ((e ^ (r & 7)) << 4));
                    }
                }
            }
            __syncwarp();
            if (busy && g.t0 == 0 && g.t1 == g.tiles) {
                constexpr int PER = HC * 8;
                const uint8_t *src = qbuf + (DUAL ? st : 0) * QTILE + (warp % 4) * 32 * 128;
                const int64_t o_at = g.s * p.out_seq + node * p.out_node + head * p.out_head;
                const int j = lane % PER, rows_left = rows - (row - lane);
#pragma unroll
                for (int i = 0; i < PER; i++) {
                    const int r = i * (32 / PER) + lane / PER;
                    const int64_t at = __shfl_sync(~0u, o_at, r);
                    const uint4 v = *(const uint4 *)(src + r * 128 + (j / 8) * QCHUNK + (((j & 7) ^ (r & 7)) << 4));
                    if (r < rows_left && j < chunks) *((uint4 *)((T *)p.out + at) + j) = v;
                }
                __syncwarp();
            }
            fence_before();
            if (!DUAL) mbar_arrive(&sh.merge_done);
            seg++;
            base += 2 * n, arrived += n ? n + 1 : 0;
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
    launch(tree_tc_kernel<T, DUAL, HC>, TA_CTAS, TT, tc_smem(DUAL, HC), s, a, k, v, sp.cuts, sp.o, sp.ml);
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
    return a.type != T_F32 && a.head_dim <= TC_MAX_DIM && mappable(a.cache_row, a.max_seq) && mappable(a.cache_head, a.n_kv_head) &&
           mappable(a.cache_seq, a.n_seq);
}

int tree_tc_rows(const sdy_tree_attention_args &a) { return a.n_node * (a.n_head / a.n_kv_head) > TR ? 2 * TR : TR; }

void tree_tc(const sdy_tree_attention_args &a, cudaStream_t s) {
    CUtensorMap k, v;
    if (!cache_map(&k, a, a.k_cache) || !cache_map(&v, a, a.v_cache)) return;
    const TreeSpace sp = tree_space(a, tree_tc_rows(a));
    if (a.type == T_F16) tc_pick<__half>(a, sp, k, v, s);
    else tc_pick<__nv_bfloat16>(a, sp, k, v, s);
    tree_join(a, sp, tree_tc_rows(a), s);
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
