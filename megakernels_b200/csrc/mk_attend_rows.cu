// Attention of many queries per request over a paged cache (declarations and rule: include/mk_serve.h).
//
// attend_rows: a CTA owns 128 rows, the (token, query head) pairs of one KV head for 128 / (query heads per KV head) tokens; two neighbouring CTAs
// of a request are a pair that multiplies together (cta_group::2, 256 rows; heads of 64: one CTA alone).  They pass over the keys that any of
// their rows sees in tiles of 128.  Warps 0-7: two threads per row (64 keys each), softmax and output; warps 8 on: producers, which bring keys and
// values into a ring of shared memory in the tensor core's swizzled order; the last warp's lane, of the pair's first CTA, issues the products:
//   S = Q K^T    Q and K from shared memory (both K-major), 128 scores a row into one of two accumulators in tensor memory;
//   O += P V     P from tensor memory, where the row's threads put it over its scores, V from shared memory as it lies (MN-major).
// Each CTA of a pair brings half of a tile: 64 of its keys, and half of the dims of all its values.  So a 4-bit tile is turned into halves once per 256 rows
// (two prompts of 1500 of 4000 positions, 24 / 4 heads of 256: 423 us alone, 283 in pairs), and a prompt of 8192 moves 1.08 GB through the L2, not 1.31.
//   While the softmax works on tile i, the products of S(i + 1) and P(i - 1) V run.  Two threads of a row exchange its maximum over a barrier of their two
// warps: a barrier of all eight, or a whole row per thread with the warps by turns over the tiles, both take longer (prompt of 8192: 216 and 226 us, 198 so).
// Outputs are scaled again only when a row's maximum rises by 2^8 (in tensor memory, by the row's threads, behind the product before).
//   What bounds it: a tile of heads of 256 takes 3200 cycles, of which the two products are 2050; S(i + 1) waits for P(i - 1) V, whose probabilities lie in its
// accumulator, and that wait and the issue behind it are the rest (tensor memory holds no third accumulator).  A prompt of 8192 with 16 / 8 heads of 256 and a
// window of 1024: 178 us, 0.77 PFLOP/s of what the window needs.  4 bits: 292 us, the producers' instructions.
//   16 bits: tiled TMA loads straight into place (a box is a page's rows, 64 dims), chunks by turns over three warps, as issuing one's loads takes as long as multiplying it.
// Rows of values that no query of the pair may see can hold anything, so the warp writes zeros over them before it hands the tile on; keys need
// no such care, their scores are masked.  Probabilities are rounded to the operands' type, as the product takes both of one type (bf16: half of the output's own rounding again).
//   4 bits: four warps turn the codes of keys into halves and four those of values, one rounding (2^-11) each: the values of 16 keys times a power of two of their own, 2^-E, so
// that any bf16 scale fits.  Keys' E scales the scores; values' E is added to the scores' exponent (sum of p v = sum of (p 2^E)(v 2^-E)) and taken out of the denominator.
// Codes 0 .. 7 of a word come out in the order 0 4 1 5 2 6 3 7; queries are stored and outputs read in the same order.
#include <cuda.h>

#include "mk_attend.cuh"
#include "mk_device.cuh"

namespace mkv {

constexpr int R_ROWS = 128, R_KEYS = 128;
enum { WA_EMPTY = 401, WA_FULL, WA_SCORES, WA_PROBS, WA_DONE, WA_QUERIES, WA_LANDED, WA_TOLD };

template <int HD, int KIND> struct RowsLayout {
    static constexpr int CG = HD >= 128 ? 2 : 1;                      // CTAs that multiply together
    static constexpr int PRODUCERS = KIND == K_INT4 ? 8 : 3;          // warps
    static constexpr int THREADS = (8 + PRODUCERS + 1) * 32;
    // One block per pair, or a pair for each two SMs that goes from block to block, so that queries and keys come in while the last block's outputs go.
    // 16 bits: a prompt of 8192 takes 178 us so, 205 one by one.  4 bits: 17 warps have 96 registers each, and the loop wants some of them (352 us, not 283).
    static constexpr bool LOOP = KIND != K_INT4;
    static constexpr int KN = R_KEYS / CG, VD = HD / CG;              // this CTA's keys of a tile, and dims of its values
    static constexpr int SLOT = KN * HD * 2, DEPTH = HD == 256 ? 4 : 8, Q_BYTES = R_ROWS * HD * 2;
    // A producer at step q has seen step q - (warps by turns) - DEPTH consumed; the parity it waits for is that of one phase only if step q - 2 DEPTH is among those.
    static_assert(DEPTH >= (KIND == K_INT4 ? 2 : PRODUCERS), "a slower ring would let a producer pass a phase early");
};
// The tiles of 128 keys that the queries at positions lo .. hi see: `front` of them hold sinks, the others run from tile `from`.
struct Tiles {
    int n, front, from;
};
// A block of rows, as the CTA sees it: its request and KV head, the request's tokens, context and this CTA's first token, its rows; of the pair the
// first and last position, the first key of its windows and its tiles.
struct Block {
    int r, head, first, count, context, token0, rows, pos_lo, pos_hi, win_lo;
    Tiles tl;
    int walk_r, walk_blocks;             // requests before walk_r have walk_blocks blocks
};
struct RowsShared {
    uint64_t full[8], empty[8], told[8], scores[2], probs[2], done, queries, q_free, landed[3];
    uint32_t tmem;
    volatile int dead;
    int warp_sums[20], items;            // blocks of all requests and KV heads
    Block blocks[20];                    // every warp's own
    float tops[2][2][R_ROWS], sums[2][2][R_ROWS];        // of either half of a tile, by turns over the tiles: a row's largest score; of a block: its sum
    int q_exp[R_ROWS];                   // 4 bits: the queries' powers of two
    int exps[8][16];                     // of a tile (mod 8: the ring holds five ahead at most): E of its eight runs of 16 keys, and of values
    uint32_t valid[8];                   // of a tile (mod 8): which runs lie in pages of the cache
};

// Where shared memory that threads have written is handed on (full, queries), both sides have the cluster's scope, as either CTA may have written it.
// Tensor memory is ordered by its own fences and the loads by their bytes: the other barriers do with a relaxed arrival, as a release of the
// cluster's scope first waits for every store before it.  What producers tell the softmax of a tile (valid, exps) has a barrier within the CTA (told).
__device__ __forceinline__ bool try_wait_cluster(uint64_t* b, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(ok) : "r"(smem_u32(b)), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ uint32_t of_first(const void* p) {          // the address in the pair's first CTA
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(0));
    return r;
}
__device__ __forceinline__ void arrive(uint32_t b) { asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(b) : "memory"); }
__device__ __forceinline__ void arrive_relaxed(uint32_t b) { asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(b) : "memory"); }
__device__ __forceinline__ void arrive_expect(uint32_t b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.relaxed.cluster.shared::cluster.b64 _, [%0], %1;" ::"r"(b), "r"(bytes) : "memory");
}
template <bool CLUSTER> static __device__ __noinline__ bool rows_wait_slow(RowsShared& S, const AttendArgs& A, uint64_t* b, uint32_t parity, int site) {
    unsigned long long t0 = 0;
#pragma unroll 1
    for (unsigned it = 0;; it++) {
        if (CLUSTER ? try_wait_cluster(b, parity) : mk::mbar_try_wait(b, parity)) return true;
        if ((it & 63u) == 63u) {
            if (S.dead) return false;
            const unsigned long long now = mk::globaltimer();
            if (!t0) t0 = now;
            else if (now - t0 > (unsigned long long)A.spin_limit_ns) {
                S.dead = 1;
                if (atomicCAS(A.status, 0, MK_ERR_TIMEOUT) == 0) A.status[1] = site, A.status[2] = (int)blockIdx.x, A.status[3] = (int)threadIdx.x;
                return false;
            }
        }
    }
}
template <bool CLUSTER = false> __device__ __forceinline__ bool rows_wait(RowsShared& S, const AttendArgs& A, uint64_t* b, uint32_t parity, int site) {
    return (CLUSTER ? try_wait_cluster(b, parity) : mk::mbar_try_wait(b, parity)) || rows_wait_slow<CLUSTER>(S, A, b, parity, site);
}
__device__ __forceinline__ void pair_sync() { asm volatile("barrier.cluster.arrive.release;\n barrier.cluster.wait.acquire;" ::: "memory"); }

template <int N> struct Const {
    static constexpr int value = N;
};

// SWIZZLE_128B operands in shared memory.  K-major: rows of 128 bytes, eight-row groups 1024 bytes apart.  MN-major: a row of 128 bytes holds 64
// neighbouring M (N) of one k; eight k 1024 bytes apart, the next 64 M (N) `lead` bytes apart.
__device__ __forceinline__ uint64_t k_major(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFF) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint64_t mn_major(uint32_t saddr, uint32_t lead) {
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// The barrier in every CTA of the pair.
template <int CG> __device__ __forceinline__ void commit(uint64_t* b) {
    if constexpr (CG == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(b)), "h"((uint16_t)3) : "memory");
    else asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(b)) : "memory");
}
template <int CG> __device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CG == 2)
        asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
    else asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
template <int CG> __device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CG == 2)
        asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate));
    else asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ void tmem_ld32(uint32_t (&r)[32], uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
                   "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
                   "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(addr));
}
// The registers of a load are its own until this wait: naming them here keeps every use behind it.
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
                 "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
                 "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
                 "r"(r[31])
                 : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float power(int e) { return __int_as_float((e + 127) << 23); }           // 2^e, -126 <= e <= 127
__device__ __forceinline__ uint32_t fma_half2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
// The exponent by which values of magnitude x are taken down, so that they stay below 2.
__device__ __forceinline__ int exponent_of(float x) { return x > 0.f && x < INFINITY ? min(max((int)(__float_as_uint(x) >> 23) - 127, -100), 100) : 0; }

// How the tensor maps of a 16-bit cache see it: dims (d, positions of a page and KV heads in the order of their strides, pages), boxes of 64 d and `box` positions.
struct Maps {
    CUtensorMap k, v, q;                 // q: (d, query heads, tokens), boxes of 64 d, a KV head's query heads and a block's tokens
    int box, heads_inside;               // heads_inside: the KV head is the second dim, the position the third
};
// Loads into this CTA; the bytes count on `bar`, an address of the cluster's window.
template <int CG> __device__ __forceinline__ void tile_load(uint32_t dst, const CUtensorMap* map, int d, int second, int third, int page, uint32_t bar) {
    if constexpr (CG == 2)
        asm volatile("cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(map), "r"(d), "r"(second),
                     "r"(third), "r"(page), "r"(bar)
                     : "memory");
    else
        asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(map), "r"(d), "r"(second), "r"(third),
                     "r"(page), "r"(bar)
                     : "memory");
}
template <int CG> __device__ __forceinline__ void queries_load(uint32_t dst, const CUtensorMap* map, int d, int head, int token, uint32_t bar) {
    if constexpr (CG == 2)
        asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map), "r"(d), "r"(head),
                     "r"(token), "r"(bar)
                     : "memory");
    else
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map), "r"(d), "r"(head), "r"(token), "r"(bar)
                     : "memory");
}

__device__ __forceinline__ Tiles tiles_of(const AttendArgs& A, int lo, int hi) {
    Tiles t;
    const int low = A.window ? max(0, lo - A.window + 1) : 0;
    t.from = low / R_KEYS;
    t.front = A.window ? min((A.sinks + R_KEYS - 1) / R_KEYS, t.from) : 0;
    t.n = hi < 0 ? 0 : t.front + hi / R_KEYS - t.from + 1;
    return t;
}

template <int CG> __device__ __forceinline__ int blocks_of(const AttendArgs& A, int per_tile, int r) {         // of a request, for one KV head
    const int a = A.starts ? min(max(__ldg(A.starts + r), 0), A.T) : r, b = A.starts ? min(max(__ldg(A.starts + r + 1), a), A.T) : r + 1;
    return (b - a + CG * per_tile - 1) / (CG * per_tile);
}
// The warp's next block, in shared memory (a call of its own and no registers of its own: the loops over tiles want them).
template <int CG> static __device__ __noinline__ void block_at(RowsShared& S, const AttendArgs& A, int item) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = CG == 2 ? (int)blockIdx.x & 1 : 0, per_tile = R_ROWS / A.per;
    Block& B = S.blocks[warp];
    __syncwarp();
    const int nth = item / A.nkv, head = item - nth * A.nkv;
    int walk_r = B.walk_r, walk_blocks = B.walk_blocks, n, upto, which;
    if (nth < walk_blocks) walk_r = walk_blocks = 0;
    for (;;) {
        n = walk_r + lane < A.R ? blocks_of<CG>(A, per_tile, walk_r + lane) : 0, upto = n;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int v = __shfl_up_sync(~0u, upto, d);
            if (lane >= d) upto += v;
        }
        const uint32_t over = __ballot_sync(~0u, walk_blocks + upto > nth);
        which = max(__ffs(over) - 1, 0);
        if (over || walk_r + 32 >= A.R) break;
        walk_blocks += __shfl_sync(~0u, upto, 31), walk_r += 32;
    }
    const int r = walk_r + which, block = max(__shfl_sync(~0u, walk_blocks + upto - 1, which) - nth, 0);
    const int first = A.starts ? min(max(__ldg(A.starts + r), 0), A.T) : r, count = A.starts ? min(max(__ldg(A.starts + r + 1), first), A.T) - first : 1;
    const int context = (int)min((long long)max(__ldg(A.context + r), 0), (long long)A.max_pages << A.page_shift);
    const int pair0 = block * CG * per_tile, token0 = pair0 + rank * per_tile;
    const int pos_lo = context - count + pair0, pos_hi = context - count + min(pair0 + CG * per_tile, count) - 1;
    if (lane == 0) {
        B.r = r, B.head = head, B.first = first, B.count = count, B.context = context, B.token0 = token0;
        B.rows = max(0, min(per_tile, count - token0)) * A.per;
        B.pos_lo = pos_lo, B.pos_hi = pos_hi, B.win_lo = A.window ? pos_lo - A.window + 1 : 0;
        B.tl = tiles_of(A, pos_lo, pos_hi);
        B.walk_r = walk_r, B.walk_blocks = walk_blocks;
    }
    __syncwarp();
}

template <int HD, int KIND>
static __global__ void __launch_bounds__(RowsLayout<HD, KIND>::THREADS, 1) attend_rows(const __grid_constant__ AttendArgs A, const __grid_constant__ Maps M) {
    using L = RowsLayout<HD, KIND>;
    constexpr bool I4 = KIND == K_INT4, BF = KIND == K_BF16;
    constexpr int G = HD / 64, CG = L::CG, KN = L::KN, VD = L::VD, DEPTH = L::DEPTH, MMA_WARP = 8 + L::PRODUCERS;
    constexpr uint32_t T_O = 256;                                      // tensor memory: scores 0-127, 128-255, outputs behind
    extern __shared__ __align__(16) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t *q_s = smem, *ring = smem + L::Q_BYTES;
    RowsShared& S = *reinterpret_cast<RowsShared*>(ring + DEPTH * L::SLOT);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int per_tile = R_ROWS / A.per;                               // tokens of a CTA
    const int rank = CG == 2 ? (int)blockIdx.x & 1 : 0, pair = (int)blockIdx.x / CG;

    if (tid == 0) S.dead = 0;
    {
        int mine = 0;
        for (int r = tid; r < A.R; r += L::THREADS) mine += blocks_of<CG>(A, per_tile, r);
        mine = __reduce_add_sync(~0u, mine);
        if (lane == 0) S.warp_sums[warp] = mine;
    }
    if (tid == 32) {
        // (full, probs and queries count the arrivals of both CTAs in the first one)
        for (int i = 0; i < DEPTH; i++) mk::mbar_init(&S.full[i], I4 ? 4 * CG : CG), mk::mbar_init(&S.empty[i], 1);
        for (int i = 0; i < 2; i++) mk::mbar_init(&S.scores[i], 1), mk::mbar_init(&S.probs[i], 8 * CG);
        for (int i = 0; i < 3; i++) mk::mbar_init(&S.landed[i], 1);
        for (int i = 0; i < 8; i++) mk::mbar_init(&S.told[i], I4 ? 4 : 1);
        mk::mbar_init(&S.done, 1);
        mk::mbar_init(&S.queries, I4 ? 8 * CG : CG);
        mk::mbar_init(&S.q_free, 1);
        mk::fence_barrier_init();
    }
    if (warp == MMA_WARP) {
        if constexpr (CG == 2) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&S.tmem)));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&S.tmem)));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    if (lane == 0) S.blocks[warp].walk_r = S.blocks[warp].walk_blocks = 0;
    __syncthreads();
    if (tid == 0) {
        int all = 0;
        for (int w = 0; w < L::THREADS / 32; w++) all += S.warp_sums[w];
        S.items = all * A.nkv;
    }
    __syncthreads();
    if constexpr (CG == 2) pair_sync();                                // the other CTA's barriers are there
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = S.tmem;
    const int items = S.items;

    // ---- the blocks, a request's last ones first (they see most), KV heads fastest; every warp walks over those of its pair by itself.  The pairs take
    // them in rounds, back and forth, so that who begins with a long one goes on with a short one.
    // Barriers and buffers go on from block to block: `tiles` counts the tiles before this one's.
    Block& B = S.blocks[warp];
    const int pairs = (int)gridDim.x / CG;
    auto item_of = [&](int round) { return round * pairs + (round & 1 ? pairs - 1 - pair : pair); };

    if (warp >= 8 && warp < MMA_WARP) {
        // ================= producers: chunks in the order K0, K1 V0, K2 V1, ... ====================================
        const int pw = warp - 8;
        uint32_t slot = 0, phase = 0, patches = 0, tiles = 0;
        int nth = 0;
        bool ok = true;
        auto room = [&](uint32_t s, uint32_t ph) { return __all_sync(~0u, rows_wait(S, A, &S.empty[s], ph ^ 1u, WA_EMPTY)) != 0; };
        for (int item; (item = item_of(nth)) < items && ok; nth++) {
        block_at<CG>(S, A, item);
        const Tiles tl = B.tl;
        const int r = B.r, head = B.head, context = B.context, pos_hi = B.pos_hi, win_lo = B.win_lo;
        auto key0_of = [&](int tile) { return (tile < tl.front ? tile : tl.from + tile - tl.front) * R_KEYS; };
        auto pages_of = [&](int key0) {
            // lane l < 8: the page of the tile's keys 16 l ..., -1 outside the cache
            const int key = key0 + 16 * (lane & 7), n = key >> A.page_shift;
            const int page = n < A.max_pages ? __ldg(A.table + r * A.table_stride + n) : -1;
            return page >= 0 && page < A.pages ? page : -1;
        };
        auto seen = [&](int key) { return key <= pos_hi && (key >= win_lo || key < A.sinks); };
        if constexpr (!I4) {
            // the queries: a box of the CTA's tokens and the KV head's query heads is 128 rows or a few less (what the tensor holds behind
            // the request's tokens fills rows that go nowhere)
            if (pw == 0 && nth > 0) ok = __all_sync(~0u, rows_wait(S, A, &S.q_free, (nth - 1) & 1, WA_QUERIES));
            if (pw == 0 && lane == 0 && ok) {
                const uint32_t bar = of_first(&S.queries);
                arrive_expect(bar, (uint32_t)(per_tile * A.per * HD * 2));
                for (int x = 0; x < G; x++) queries_load<CG>(smem_u32(q_s) + x * R_ROWS * 128, &M.q, x * 64, head * A.per, min(B.first + B.token0, A.T - 1), bar);
            }
            __syncwarp();
        }
        // step 0: K0; then K(i + 1), V(i) by turns; the last one V(n - 1)
        const int steps = 2 * tl.n;
        auto is_value = [&](int step) { return step == steps - 1 || (step > 0 && (step & 1) == 0); };
        auto tile_at = [&](int step) { return step == 0 ? 0 : (step == steps - 1 ? tl.n - 1 : ((step & 1) ? (step + 1) / 2 : step / 2 - 1)); };
        auto tell_valid = [&](int tile, int my_page) {
            const uint32_t v = __ballot_sync(~0u, my_page >= 0) & 0xFFu;
            if (lane == 0) S.valid[tiles + tile & 7] = v;
        };
        auto tell = [&](int tile) {
            __syncwarp();
            if (lane == 0) mk::mbar_arrive(&S.told[tiles + tile & 7]);
        };
        if constexpr (I4) {
            // Warps 0-3 bring keys, 4-7 values.  Two threads a row, four runs of eight values of every group each.  Of keys the pair's CTAs turn 64 rows each into
            // halves, of values half of the groups of all rows, in two parts.  The next tile's codes are on their way while this one's are turned, and the pages of the tile behind.
            constexpr int VG = G / CG, KP = 2 / CG;                    // groups of values, parts of keys
            const int half = lane & 1, pr = pw & 3;
            // Two sets of rows: of keys, this CTA's and the other's (whose scales alone it wants; with one CTA, both its own); of values, both parts.
            uint32_t w[8 * G / CG], m[2][G], of_values[2][G];
            auto run_of = [&](bool value, int p) { return (value ? p : rank ^ p) * 4 + pr; };
            auto get = [&](auto value_, int tile, int my_page) {
                constexpr bool value = decltype(value_)::value != 0;
                const int key0 = key0_of(tile);
                if (!value && pr == 0) tell_valid(tile, my_page);
                auto scales = [&](uint32_t (&to)[G], const uint8_t* base, long long at, bool wanted) {
                    const uint8_t* p = base + at * (G * 4);
                    if constexpr (G == 4) *reinterpret_cast<uint4*>(to) = wanted ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
                    else if constexpr (G == 2) *reinterpret_cast<uint2*>(to) = wanted ? __ldg(reinterpret_cast<const uint2*>(p)) : make_uint2(0, 0);
                    else to[0] = wanted ? __ldg(reinterpret_cast<const uint32_t*>(p)) : 0u;
                };
#pragma unroll
                for (int p = 0; p < 2; p++) {
                    const int run = run_of(value, p), key = key0 + run * 16 + (lane >> 1), page = __shfl_sync(~0u, my_page, run);
                    const bool live = page >= 0 && seen(key);
                    const long long at = (((long long)max(page, 0) * A.nkv + head) << A.page_shift) + (key & ((1 << A.page_shift) - 1));
                    scales(m[p], value ? A.vs : A.ks, at, live);
                    const uint8_t* row = (value ? A.v : A.k) + at * (HD / 2) + half * (HD / 4);
                    if constexpr (!value) {
                        if (p < KP)
#pragma unroll
                            for (int j = 0; j < G; j++)
                                *reinterpret_cast<uint4*>(w + (p * G + j) * 4) = live ? __ldg(reinterpret_cast<const uint4*>(row) + j) : make_uint4(0, 0, 0, 0);
                        const int run_v = run_of(true, p), key_v = key0 + run_v * 16 + (lane >> 1), page_v = __shfl_sync(~0u, my_page, run_v);
                        scales(of_values[p], A.vs, (((long long)max(page_v, 0) * A.nkv + head) << A.page_shift) + (key_v & ((1 << A.page_shift) - 1)), page_v >= 0 && seen(key_v));
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const uint8_t* src = row + j * G * 4 + rank * VG * 4;
                            if constexpr (VG == 2) *reinterpret_cast<uint2*>(w + (p * 4 + j) * 2) = live ? __ldg(reinterpret_cast<const uint2*>(src)) : make_uint2(0, 0);
                            else w[p * 4 + j] = live ? __ldg(reinterpret_cast<const uint32_t*>(src)) : 0u;
                        }
                    }
                }
            };
            auto warp_exp = [&](const uint32_t (&s)[G]) {
                uint32_t big = 0;                                      // bf16 without a sign orders as a whole number does
#pragma unroll
                for (int g = 0; g < G; g++) big = __vmaxu2(big, s[g] & 0x7FFF7FFFu);
                return exponent_of(__uint_as_float(__reduce_max_sync(~0u, __float_as_uint(fmaxf(15.f * __uint_as_float(big << 16), __uint_as_float(big & 0xFFFF0000u))))));
            };
            auto turn = [&](uint32_t c, uint32_t s2, uint32_t l2) {
                return make_uint4(fma_half2(codes<0>(c), s2, l2), fma_half2(codes<1>(c), s2, l2), fma_half2(codes<2>(c), s2, l2), fma_half2(codes<3>(c), s2, l2));
            };
            auto both = [](float v) { return pack_half(v, v); };
            auto bring = [&](auto value_) {
                constexpr bool value = decltype(value_)::value != 0;
                if (!tl.n) return;
                int page_next = tl.n > 1 ? pages_of(key0_of(1)) : -1;
                get(value_, 0, pages_of(key0_of(0)));
                for (int tile = 0; tile < tl.n; tile++) {
                    const int step = value ? (tile == tl.n - 1 ? steps - 1 : 2 * tile + 2) : (tile ? 2 * tile - 1 : 0);
                    slot = (2 * tiles + step) % DEPTH, phase = (2 * tiles + step) / DEPTH & 1;
                    int e[2];
#pragma unroll
                    for (int p = 0; p < 2; p++) {
                        e[p] = warp_exp(m[p]);
                        if constexpr (!value) {
                            const int ev = warp_exp(of_values[p]);
                            if (lane == 0) S.exps[tiles + tile & 7][run_of(false, p)] = e[p], S.exps[tiles + tile & 7][8 + run_of(true, p)] = ev;
                        }
                    }
                    if constexpr (!value) tell(tile);
                    if (!(ok = room(slot, phase))) break;
                    uint8_t* to = ring + slot * L::SLOT;
#pragma unroll
                    for (int p = 0; p < (value ? 2 : KP); p++) {
                        const float down = power(-e[p]);
                        const int row = p * 64 + pr * 16 + (lane >> 1);
                        constexpr int GS = value ? VG : G, ROWS = value ? R_KEYS : KN;
#pragma unroll
                        for (int g = 0; g < GS; g++) {
                            const uint32_t sl = value && CG == 2 && rank ? m[p][(CG - 1) * VG + g % VG] : m[p][g];
                            const uint32_t s2 = both(__uint_as_float(sl << 16) * down), l2 = both(__uint_as_float(sl & 0xFFFF0000u) * down);
#pragma unroll
                            for (int j = 0; j < 4; j++) *reinterpret_cast<uint4*>(to + g * ROWS * 128 + row * 128 + (((half * 4 + j) ^ (row & 7)) << 4)) = turn(w[(p * 4 + j) * GS + g], s2, l2);
                        }
                    }
                    mk::fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) arrive(of_first(&S.full[slot]));    // (before the next loads, which its release would wait for)
                    if (tile + 1 < tl.n) {
                        get(value_, tile + 1, page_next);
                        page_next = tile + 2 < tl.n ? pages_of(key0_of(tile + 2)) : -1;
                    }
                }
            };
            if (pw < 4) bring(Const<0>{});
            else bring(Const<1>{});
        } else {
            const int box_shift = 31 - __clz(M.box);
            // (a warp's turns go on from block to block)
            for (int q = (pw + L::PRODUCERS - (int)(2 * tiles % L::PRODUCERS)) % L::PRODUCERS; q < steps && ok; q += L::PRODUCERS) {
                const int tile = tile_at(q), key0 = key0_of(tile), my_page = pages_of(key0);
                const bool value = is_value(q);
                slot = (2 * tiles + q) % DEPTH, phase = (2 * tiles + q) / DEPTH & 1;
                if (!value) tell_valid(tile, my_page), tell(tile);
                // keys that a query of the pair, or of a later one, sees hold values; so do all sinks
                const uint32_t pages = __ballot_sync(~0u, my_page >= 0);                               // a bit per run of 16 keys (boxes are whole pages, or parts of one)
                const bool clean = (pages & 0xFFu) == 0xFFu && key0 + R_KEYS <= context && (key0 >= win_lo || key0 + R_KEYS <= A.sinks);
                uint8_t* dst = ring + slot * L::SLOT;
                // keys: this CTA's, all dims; values: all 128 keys, this CTA's dims
                const int n = value ? R_KEYS : KN, from = value ? 0 : rank * KN, d0 = value ? rank * VD : 0;
                constexpr int K_SHIFT = G == 4 ? 2 : (G == 2 ? 1 : 0), V_SHIFT = VD == 128 ? 1 : 0;
                const int slab_shift = value ? V_SHIFT : K_SHIFT;
                const uint32_t bar = value && !clean ? smem_u32(&S.landed[pw]) : of_first(&S.full[slot]);
                const int x = lane & ((1 << slab_shift) - 1), row = (lane >> slab_shift) << box_shift, off = (key0 + from + row) & ((1 << A.page_shift) - 1);
                const int page = __shfl_sync(~0u, my_page, (from + row) >> 4 & 7);
                const bool mine = row < n && page >= 0;
                const uint32_t loads = __popc(__ballot_sync(~0u, mine));
                if (!(ok = room(slot, phase))) break;
                if (lane == 0) {
                    if (loads) arrive_expect(bar, loads * M.box * 128);
                    else arrive(bar);
                }
                __syncwarp();
                if (mine)
                    tile_load<CG>(smem_u32(dst) + x * n * 128 + row * 128, value ? &M.v : &M.k, d0 + x * 64, M.heads_inside ? head : off, M.heads_inside ? off : head, page, bar);
                __syncwarp();
                if (value && !clean) {
                    if (!(ok = __all_sync(~0u, rows_wait(S, A, &S.landed[pw], patches & 1, WA_LANDED)) != 0)) break;
                    patches++;
                    // a lane per row; the pieces by turns, so that the lanes' stores spread over the banks
                    for (int r0 = 0; r0 < n; r0 += 32) {
                        const int line = r0 + lane;
                        if (!(pages >> (line >> 4) & 1) || !seen(key0 + line))
#pragma unroll 8
                            for (int i = 0; i < 8 << V_SHIFT; i++) *reinterpret_cast<uint4*>(dst + (i >> 3) * n * 128 + line * 128 + ((i + lane & 7) << 4)) = make_uint4(0, 0, 0, 0);
                    }
                    mk::fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) arrive(of_first(&S.full[slot]));
                }
            }
        }
        tiles += tl.n;
        if constexpr (!L::LOOP) break;
        }
        if (!I4 && S.dead) {
            // loads under way still write shared memory: a bounded wait for them
            const unsigned long long t0 = mk::globaltimer();
            while (mk::globaltimer() - t0 < 1000000ull) {}
        }
    } else if (warp == MMA_WARP) {
        // ================= the products: the pair's first CTA issues them ==========================================
        constexpr uint32_t type = BF ? (1u << 7) | (1u << 10) : 0u, m = (uint32_t)(8 * CG) << 24;
        constexpr uint32_t id_s = (1u << 4) | type | ((R_KEYS >> 3) << 17) | m, id_o = (1u << 4) | type | (1u << 16) | ((HD >> 3) << 17) | m;
        uint32_t slot = 0, phase = 0, tiles = 0;
        int nth = 0;
        bool ok = rank == 0;
        for (int item; (item = item_of(nth)) < items && ok; nth++) {
            block_at<CG>(S, A, item);
            const int n = B.tl.n;
            if (lane == 0) {
                auto next = [&]() {
                    if (!rows_wait<(CG == 2)>(S, A, &S.full[slot], phase, WA_FULL)) return false;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    return true;
                };
                auto release = [&]() {
                    commit<CG>(&S.empty[slot]);
                    if (++slot == DEPTH) slot = 0, phase ^= 1u;
                };
                auto scores = [&](int i) {
                    const uint32_t t = tiles + i;
                    if (!next()) return false;
                    const uint32_t k = smem_u32(ring + slot * L::SLOT), q = smem_u32(q_s);
#pragma unroll
                    for (int x = 0; x < G; x++) {
                        const uint64_t da = k_major(q + x * R_ROWS * 128), db = k_major(k + x * KN * 128);
#pragma unroll
                        for (int j = 0; j < 4; j++) mma_ss<CG>(tmem + (t & 1) * 128, da + 2 * j, db + 2 * j, id_s, (uint32_t)(x + j > 0));
                    }
                    release();
                    commit<CG>(&S.scores[t & 1]);
                    if (i == n - 1) commit<CG>(&S.q_free);
                    return true;
                };
                ok = rows_wait<(CG == 2)>(S, A, &S.queries, nth & 1, WA_QUERIES);
                if (ok && n == 0) commit<CG>(&S.q_free);
                ok = ok && (n == 0 || scores(0));
                for (int i = 0; i < n && ok; i++) {
                    const uint32_t t = tiles + i;
                    // P(t - 1) V is done before S(t + 1) takes its accumulator (every tile waits for the one before, behind a block's last scores too:
                    // a parity names a phase only among two)
                    if (t > 0 && !(ok = rows_wait(S, A, &S.done, (t - 1) & 1, WA_DONE))) break;
                    if (i + 1 < n && !(ok = scores(i + 1))) break;
                    // (the softmax puts a block's first probabilities only when it has read the outputs of the block before)
                    if (!(ok = rows_wait(S, A, &S.probs[t & 1], (t >> 1) & 1, WA_PROBS) && next())) break;
                    const uint64_t db = mn_major(smem_u32(ring + slot * L::SLOT), R_KEYS * 128);
#pragma unroll
                    for (int x = 0; x < R_KEYS / 16; x++)
                        mma_ts<CG>(tmem + T_O, tmem + (t & 1) * 128 + x / 4 * 64 + x % 4 * 8, db + x * 128, id_o, (uint32_t)(i + x > 0));
                    release();
                    commit<CG>(&S.done);
                }
            }
            ok = __shfl_sync(~0u, (int)ok, 0) != 0;
            tiles += n;
            if constexpr (!L::LOOP) break;
        }
        __syncwarp();
    } else {
        // ================= softmax and output: two threads a row, 64 keys (later half of the dims) each; rows behind the last repeat it ====
        const int half = warp >> 2, row = tid & 127;
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        // barrier of the eight warps; whether any of them has given up, the same answer for all
        auto failed = [](bool mine) {
            uint32_t any;
            asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 q, %1, 0;\n bar.red.or.pred p, 9, 256, q;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(any) : "r"((uint32_t)mine) : "memory");
            return any != 0;
        };
        bool ok = true;
        uint32_t tiles = 0;
        int nth = 0;
        for (int item; (item = item_of(nth)) < items && ok; nth++) {
        block_at<CG>(S, A, item);
        const Tiles& tl = B.tl;
        const int &head = B.head, &context = B.context, &count = B.count, &rows = B.rows, &token0 = B.token0, &first = B.first;
        auto key0_of = [&](int tile) { return (tile < tl.front ? tile : tl.from + tile - tl.front) * R_KEYS; };
        const int n = max(0, min(row, rows - 1)), token = n / A.per, h = n - token * A.per, pos = context - count + token0 + token;
        // (a CTA without tokens of its own, the second of a request's last pair, does as if it had the tokens before)
        const int from_token = min(first + token0 + token, A.T - 1);
        if constexpr (I4) {
            static_assert(!L::LOOP, "the next block's queries would have to wait for q_free");
            // the queries: a warp's lanes turn 16 of its rows into halves one after the other
            const uint16_t* own = reinterpret_cast<const uint16_t*>(A.q) + from_token * A.q_tok + (long long)(head * A.per + h) * A.q_head;
            const bool has = lane < HD / 8;
#pragma unroll 1
            for (int i0 = half * 16; i0 < half * 16 + 16; i0 += 8) {
            uint4 x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint16_t* p = reinterpret_cast<const uint16_t*>(__shfl_sync(~0u, (unsigned long long)own, i0 + i)) + lane * 8;
                x[i] = has ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int at = (warp & 3) * 32 + i0 + i;
                float v[8], big = 0.f;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const uint32_t w = (&x[i].x)[j >> 1];
                    v[j] = from16((uint16_t)(j & 1 ? w >> 16 : w), A.q_f16);
                    big = fmaxf(big, fabsf(v[j]));
                }
                big = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(big)));
                const int e = exponent_of(big);
                const float down = power(-e);
                if (lane == 0) S.q_exp[at] = e;
                if (has)
                    *reinterpret_cast<uint4*>(q_s + (lane >> 3) * (R_ROWS * 128) + at * 128 + (((lane & 7) ^ (at & 7)) << 4)) =
                        make_uint4(pack_half(v[0] * down, v[4] * down), pack_half(v[1] * down, v[5] * down), pack_half(v[2] * down, v[6] * down), pack_half(v[3] * down, v[7] * down));
            }
            }
            mk::fence_proxy_async();
            __syncwarp();
            if (lane == 0) arrive(of_first(&S.queries));
        }
        if constexpr (I4) failed(false);
        const int own_lo = context - count + token0, own_hi = own_lo + per_tile - 1;                  // positions of the CTA's rows
        float ref = -INFINITY, sum = 0.f;
        const float scale = A.scale_log2 * (I4 ? power(S.q_exp[row]) : 1.f);
        // A warp that has given up goes on without waiting, as the warp that has the other halves of its rows waits for its maxima.
        for (int i = 0; i < tl.n; i++) {
            const uint32_t t = tiles + i;
            ok = ok && __all_sync(~0u, rows_wait(S, A, &S.scores[t & 1], (t >> 1) & 1, WA_SCORES));
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            ok = ok && __all_sync(~0u, rows_wait(S, A, &S.told[t & 7], (t >> 3) & 1, WA_TOLD));
            const int key0 = key0_of(i);
            const uint32_t at = lanes + (t & 1) * 128 + half * 64, valid = *(volatile uint32_t*)&S.valid[t & 7];
            const bool whole = valid == 0xFFu && key0 + R_KEYS - 1 <= own_lo && (!A.window || key0 > own_hi - A.window || key0 + R_KEYS <= A.sinks);
            const int* exps = S.exps[t & 7] + half * 4;
            // scores of keys that this row does not see become -inf
            auto mask = [&](uint32_t (&x)[32], int c) {
                if (!whole) {
                    const int w = half * 2 + c;
                    auto below = [&](int n) { return n >= 32 * w + 32 ? ~0u : (n <= 32 * w ? 0u : (1u << (n - 32 * w)) - 1); };                    // columns under n
                    uint32_t bits = below(pos - key0 + 1);
                    if (A.window) bits &= ~below(pos - A.window + 1 - key0) | below(A.sinks - key0);
                    bits &= (valid >> (2 * w) & 1 ? 0xFFFFu : 0u) | (valid >> (2 * w + 1) & 1 ? 0xFFFF0000u : 0u);
#pragma unroll
                    for (int j = 0; j < 32; j++) x[j] = bits >> j & 1 ? x[j] : 0xFF800000u;
                }
            };
            // (4 bits: fewer registers, so that the scores are read from tensor memory twice)
            uint32_t x[I4 ? 1 : 2][32];
            float top = -INFINITY;
            if constexpr (!I4) {
                tmem_ld32(x[0], at);
                tmem_ld32(x[1], at + 32);
                tmem_wait_ld(x[0]);
                tmem_wait_ld(x[1]);
            }
#pragma unroll
            for (int c = 0; c < 2; c++) {
                uint32_t (&y)[32] = x[I4 ? 0 : c];
                if constexpr (I4) tmem_ld32(y, at + c * 32), tmem_wait_ld(y);
                mask(y, c);
                float a[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < 32; j++) a[(j >> 4) * 2 + (j & 1)] = fmaxf(a[(j >> 4) * 2 + (j & 1)], __uint_as_float(y[j]));
                // (4 bits: a run of 16 keys has a factor of its scores, and an exponent of its values)
                if constexpr (I4) {
#pragma unroll
                    for (int j = 0; j < 2; j++) top = fmaxf(top, fmaf(fmaxf(a[2 * j], a[2 * j + 1]), scale * power(exps[2 * c + j]), (float)exps[8 + 2 * c + j]));
                } else
                    top = fmaxf(top, fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])) * scale);
            }
            S.tops[t & 1][half][row] = top;
            asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory");
            top = fmaxf(top, S.tops[t & 1][half ^ 1][row]);
            // the reference rises when a score exceeds it by 2^8 (in one of the warp's rows; those behind the last hold anything and have no say)
            // (a parity names a phase only among two: S(t) is there, so the product of t - 2 is done, and this tile's wants our probabilities)
            auto product_before = [&]() { ok = ok && __all_sync(~0u, rows_wait(S, A, &S.done, (t - 1) & 1, WA_DONE)); };
            if (__any_sync(~0u, row < rows && top > ref + 8.f)) {
                const float next = fmaxf(ref, top), turn = next == -INFINITY ? 1.f : exp2_fast(ref - next);
                sum *= turn;
                ref = next;
                if (i > 0) {
                    product_before();
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    uint32_t z[32];
#pragma unroll 1
                    for (int c = half * (HD / 64); c < (half + 1) * (HD / 64); c++) {
                        tmem_ld32(z, lanes + T_O + c * 32);
                        tmem_wait_ld(z);
#pragma unroll
                        for (int j = 0; j < 32; j++) z[j] = __float_as_uint(__uint_as_float(z[j]) * turn);
                        tmem_st32(lanes + T_O + c * 32, z);
                    }
                }
            }
            const float base = ref == -INFINITY ? 0.f : ref;
#pragma unroll
            for (int c = 0; c < 2; c++) {
                uint32_t (&y)[32] = x[I4 ? 0 : c];
                if constexpr (I4) {
                    tmem_ld32(y, at + c * 32);
                    tmem_wait_ld(y);
                    mask(y, c);
                }
                float part[4] = {0.f, 0.f, 0.f, 0.f}, f[2] = {scale, scale}, b[2] = {-base, -base};
                if constexpr (I4) {
#pragma unroll
                    for (int j = 0; j < 2; j++) f[j] = scale * power(exps[2 * c + j]), b[j] = (float)exps[8 + 2 * c + j] - base;
                }
                uint32_t p[16];
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    // (masked scores are -inf: their probability is 0)
                    const float u = exp2_fast(fmaf(__uint_as_float(y[j]), f[j >> 4], b[j >> 4])), v = exp2_fast(fmaf(__uint_as_float(y[j + 1]), f[j >> 4], b[j >> 4]));
                    part[j >> 4] += u, part[2 + (j >> 4)] += v;
                    p[j / 2] = BF ? pack_bf(u, v) : pack_half(u, v);
                }
                if constexpr (I4) sum += (part[0] + part[2]) * power(-exps[8 + 2 * c]) + (part[1] + part[3]) * power(-exps[9 + 2 * c]);
                else sum += (part[0] + part[2]) + (part[1] + part[3]);
                tmem_st16(at + c * 16, p);                             // over scores that this thread has read
            }
            tmem_wait_st();
            if (i > 0 && i + 1 == tl.n) product_before();              // (so that the wait for this one, below, has no other phase before it)
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) arrive_relaxed(of_first(&S.probs[t & 1]));
        }
        S.sums[nth & 1][half][row] = sum;
        if (tl.n > 0) ok = ok && __all_sync(~0u, rows_wait(S, A, &S.done, tiles + tl.n - 1 & 1, WA_DONE));
        if (failed(!ok)) ok = false;                                   // nothing is written then, and all eight warps leave together
        sum += S.sums[nth & 1][half ^ 1][row];
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (ok) {
            const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
            uint16_t* dst = reinterpret_cast<uint16_t*>(A.out) + (first + token0 + token) * A.out_tok + (long long)(head * A.per + h) * A.out_head;
#pragma unroll 1
            for (int c = half * (HD / 64); c < (half + 1) * (HD / 64); c++) {
                uint32_t x[32];
                if (tl.n > 0) {
                    tmem_ld32(x, lanes + T_O + c * 32);
                    tmem_wait_ld(x);
                }
                if (row < rows)
#pragma unroll
                for (int j = 0; j < 32; j += 8) {
                    uint4 o = make_uint4(0, 0, 0, 0);
                    if (tl.n > 0 && sum != 0.f) {
                        float v[8];
#pragma unroll
                        for (int y = 0; y < 8; y++) v[y] = __uint_as_float(x[j + (I4 ? (y & 3) * 2 + (y >> 2) : y)]) * inv;
#pragma unroll
                        for (int y = 0; y < 4; y++) (&o.x)[y] = A.q_f16 ? pack_half(v[2 * y], v[2 * y + 1]) : pack_bf(v[2 * y], v[2 * y + 1]);
                    }
                    *reinterpret_cast<uint4*>(dst + c * 32 + j) = o;
                }
                __syncwarp();
            }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        tiles += tl.n;
        if constexpr (!L::LOOP) break;
        }
    }
    if (warp == MMA_WARP && S.dead) {
        // a wait ran out: products under way still read shared and tensor memory, so this waits a bounded time for them
        const unsigned long long t0 = mk::globaltimer();
        while (mk::globaltimer() - t0 < 1000000ull) {}
    }
    __syncthreads();
    if constexpr (CG == 2) pair_sync();                                // nobody arrives at a CTA that has left, or multiplies in its memory
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if constexpr (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        return cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) == cudaSuccess && found == cudaDriverEntryPointSuccess ? reinterpret_cast<EncodeTiled>(p) : nullptr;
    }();
    return fn;
}

static int make_maps(const AttendArgs& A, int head_dim, bool f16, Maps* M) {
    memset(M, 0, sizeof *M);
    const EncodeTiled encode = encode_tiled();
    if (!encode) return vfail(MK_ERR_CUDA, "mk_attend: the driver has no cuTensorMapEncodeTiled");
    const int page = 1 << A.page_shift, most = head_dim >= 128 ? 64 : R_KEYS;          // (a pair's CTA takes 64 keys of a tile)
    M->box = page < most ? page : most;
    // (the stride of an extent of one says nothing, and may be 0)
    const long long s_head = A.nkv > 1 ? A.s_head : A.s_pos << A.page_shift, s_page = A.pages > 1 ? A.s_page : (A.s_pos << A.page_shift) * A.nkv;
    M->heads_inside = s_head < A.s_pos;
    const cuuint64_t size[4] = {(cuuint64_t)head_dim, (cuuint64_t)(M->heads_inside ? A.nkv : page), (cuuint64_t)(M->heads_inside ? page : A.nkv), (cuuint64_t)A.pages};
    const cuuint64_t stride[3] = {(cuuint64_t)(M->heads_inside ? s_head : A.s_pos), (cuuint64_t)(M->heads_inside ? A.s_pos : s_head), (cuuint64_t)s_page};
    const cuuint32_t box[4] = {64, (cuuint32_t)(M->heads_inside ? 1 : M->box), (cuuint32_t)(M->heads_inside ? M->box : 1), 1}, step[4] = {1, 1, 1, 1};
    for (int i = 0; i < 2; i++) {
        const CUresult rc = encode(i ? &M->v : &M->k, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<uint8_t*>(i ? A.v : A.k), size, stride, box, step,
                                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (rc != CUDA_SUCCESS) return vfail(MK_ERR_CUDA, "mk_attend: no tensor map for strides %lld, %lld, %lld bytes (error %d)", A.s_pos, A.s_head, A.s_page, (int)rc);
    }
    const int per_tile = R_ROWS / A.per;
    const cuuint64_t q_size[3] = {(cuuint64_t)head_dim, (cuuint64_t)A.nq, (cuuint64_t)A.T}, q_stride[2] = {(cuuint64_t)(A.nq > 1 ? A.q_head * 2 : head_dim * 2), (cuuint64_t)(A.T > 1 ? A.q_tok * 2 : A.nq * head_dim * 2)};
    const cuuint32_t q_box[3] = {64, (cuuint32_t)A.per, (cuuint32_t)per_tile};
    const CUresult rc = encode(&M->q, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(A.q), q_size, q_stride, q_box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) return vfail(MK_ERR_CUDA, "mk_attend: no tensor map for query strides %lld, %lld elements (error %d)", A.q_tok, A.q_head, (int)rc);
    return MK_OK;
}

template <int HD, int KIND>
static int launch_one(const AttendArgs& A, int sms, cudaStream_t st) {
    using L = RowsLayout<HD, KIND>;
    constexpr int smem = L::Q_BYTES + L::DEPTH * L::SLOT + (int)sizeof(RowsShared) + 1024;
    static_assert(smem <= 232448 && smem > 116 * 1024, "one CTA per SM: it takes all of the tensor memory");
    const int per_tile = R_ROWS / A.per;
    // (every request rounds up once)
    const long long blocks = ((long long)A.T / (per_tile * L::CG) + (A.T < A.R ? A.T : A.R)) * A.nkv, most = L::LOOP ? sms / L::CG : blocks;
    if (blocks >= (1 << 30)) return vfail(MK_ERR_UNSUPPORTED, "mk_attend: %d tokens of %d KV heads", A.T, A.nkv);
    const unsigned grid = (unsigned)((blocks < most ? blocks : most) * L::CG);
    Maps M;
    if (KIND == K_INT4) memset(&M, 0, sizeof M);
    else {
        const int rc = make_maps(A, HD, KIND == K_F16, &M);
        if (rc != MK_OK) return rc;
    }
    MKV_CUDA(cudaFuncSetAttribute(attend_rows<HD, KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    MKV_CUDA(launch(attend_rows<HD, KIND>, grid, L::THREADS, smem, L::CG, false, st, A, M));
    return MK_OK;
}
template <int HD>
static int launch_hd(const AttendArgs& A, int type, int sms, cudaStream_t st) {
    return type == MKV_INT4 ? launch_one<HD, K_INT4>(A, sms, st) : (type == MKV_F16 ? launch_one<HD, K_F16>(A, sms, st) : launch_one<HD, K_BF16>(A, sms, st));
}
int launch_rows(const AttendArgs& A, int type, int head_dim, int sms, cudaStream_t st) {
    return head_dim == 64 ? launch_hd<64>(A, type, sms, st) : (head_dim == 128 ? launch_hd<128>(A, type, sms, st) : launch_hd<256>(A, type, sms, st));
}

}  // namespace mkv
