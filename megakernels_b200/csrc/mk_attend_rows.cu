// Attention of many queries per request over a paged cache (declarations and rule: include/mk_serve.h).
//
// attend_rows: a CTA owns 128 rows, the (token, query head) pairs of one KV head for 128 / (query heads per KV head) tokens, and passes
// over the keys they see in tiles of 128.  Warps 0-7: two threads a row, softmax and output; warps 4 on: producers, which bring keys and values into a ring
// of shared memory in the tensor core's swizzled order; the last warp's lane issues the products:
//   S = Q K^T    Q and K from shared memory (both K-major), 128 x 128 scores into one of two accumulators in tensor memory;
//   O += P V     P from tensor memory, where the row's thread put it over its scores, V from shared memory as it lies (MN-major),
//                128 x dim outputs in tensor memory.
// While the softmax works on tile i, the products of S(i + 1) and P(i - 1) V run.  Outputs are scaled again only when a row's maximum rises
// by 2^8 (in tensor memory, by the row's thread, behind the product before).
//   Tiles of 128 keys because a product of 128 x 64 would read its operands from shared memory slower than it multiplies; keys (by dims) and values
// (by keys) of a head of 256 come in halves, so that four 32 KB slots beside the 64 KB of Q hold two products ahead.
//   16 bits: one warp's tiled TMA loads straight into place (a box is a page's rows, 64 dims).  Rows of values that no query of the block may see can hold anything, so the
// warp writes zeros over them before it hands the tile on; keys need no such care, their scores are masked.  Probabilities are rounded to the operands' type, as the product takes both of one type
// (bf16: half of the output's own rounding again).
//   4 bits: four warps turn codes into halves, one rounding (2^-11) each: the values of 16 keys times a power of two of their own, 2^-E, so
// that any bf16 scale fits.  Keys' E scales the scores; values' E is added to the scores' exponent (sum of p v = sum of (p 2^E)(v 2^-E)) and taken out of the denominator.
// Codes 0 .. 7 of a word come out in the order 0 4 1 5 2 6 3 7; queries are stored and outputs read in the same order.
#include <cuda.h>

#include "mk_attend.cuh"
#include "mk_device.cuh"

namespace mkv {

constexpr int R_ROWS = 128, R_KEYS = 128;
enum { WA_EMPTY = 401, WA_FULL, WA_SCORES, WA_PROBS, WA_DONE, WA_QUERIES, WA_LANDED };

template <int HD, int KIND> struct RowsLayout {
    static constexpr int PRODUCERS = KIND == K_INT4 ? 4 : 3;          // warps
    static constexpr int THREADS = (8 + PRODUCERS + 1) * 32;
    static constexpr int CH = HD == 256 ? 2 : 1;                      // chunks of a tile's keys, and of its values
    static constexpr int SLOT = R_KEYS * HD * 2 / CH, DEPTH = HD == 256 ? 4 : (HD == 128 ? 5 : 8), Q_BYTES = R_ROWS * HD * 2;
};
struct RowsShared {
    uint64_t full[8], empty[8], scores[2], probs[2], done, queries, landed[3];
    uint32_t tmem;
    volatile int dead;
    int request, block;
    int warp_sums[20];
    float tops[2][2][R_ROWS];            // a row's largest score of either half of a tile, by turns; at the end the sums
    int q_exp[R_ROWS];                   // 4 bits: the queries' powers of two
    int exps[8][16];                     // of a tile (mod 8: the ring holds five ahead at most): E of its eight runs of 16 keys, and of values
    uint32_t valid[8];                   // of a tile (mod 8): which runs lie in pages of the cache
};

static __device__ __noinline__ bool rows_wait_slow(RowsShared& S, const AttendArgs& A, uint64_t* b, uint32_t parity, int site) {
    unsigned long long t0 = 0;
#pragma unroll 1
    for (unsigned it = 0;; it++) {
        if (mk::mbar_try_wait(b, parity)) return true;
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
__device__ __forceinline__ bool rows_wait(RowsShared& S, const AttendArgs& A, uint64_t* b, uint32_t parity, int site) {
    return mk::mbar_try_wait(b, parity) || rows_wait_slow(S, A, b, parity, site);
}

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
__device__ __forceinline__ void commit(uint64_t* b) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(b)) : "memory");
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

// The tiles of 128 keys that the queries at positions lo .. hi see: `front` of them hold sinks, the others run from tile `from`.
struct Tiles {
    int n, front, from;
};
__device__ __forceinline__ Tiles tiles_of(const AttendArgs& A, int lo, int hi) {
    Tiles t;
    const int low = A.window ? max(0, lo - A.window + 1) : 0;
    t.from = low / R_KEYS;
    t.front = A.window ? min((A.sinks + R_KEYS - 1) / R_KEYS, t.from) : 0;
    t.n = hi < 0 ? 0 : t.front + hi / R_KEYS - t.from + 1;
    return t;
}

// How the tensor maps of a 16-bit cache see it: dims (d, positions of a page and KV heads in the order of their strides, pages), boxes of 64 d and `box` positions.
struct Maps {
    CUtensorMap k, v, q;                 // q: (d, query heads, tokens), boxes of 64 d, a KV head's query heads and a block's tokens
    int box, heads_inside;               // heads_inside: the KV head is the second dim, the position the third
};
__device__ __forceinline__ void tile_load(uint32_t dst, const CUtensorMap* map, int d, int second, int third, int page, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(map), "r"(d), "r"(second), "r"(third),
                 "r"(page), "r"(smem_u32(bar))
                 : "memory");
}

template <int HD, int KIND>
static __global__ void __launch_bounds__(RowsLayout<HD, KIND>::THREADS, 1) attend_rows(const __grid_constant__ AttendArgs A, const __grid_constant__ Maps M) {
    using L = RowsLayout<HD, KIND>;
    constexpr bool I4 = KIND == K_INT4, BF = KIND == K_BF16;
    constexpr int G = HD / 64, CH = L::CH, DEPTH = L::DEPTH, MMA_WARP = 8 + L::PRODUCERS;
    constexpr uint32_t T_O = 256;                                      // tensor memory: scores 0-127, 128-255, outputs behind
    extern __shared__ __align__(16) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t *q_s = smem, *ring = smem + L::Q_BYTES;
    RowsShared& S = *reinterpret_cast<RowsShared*>(ring + DEPTH * L::SLOT);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int per_tile = R_ROWS / A.per;                               // tokens of a block

    // ---- which request and block this CTA has (blocks of a request last first: they see most)
    if (tid == 0) S.request = -1, S.dead = 0;
    {
        const int each = (A.R + L::THREADS - 1) / L::THREADS, r0 = min(A.R, tid * each), r1 = min(A.R, r0 + each);
        auto blocks = [&](int r) {
            const int a = A.starts ? min(max(__ldg(A.starts + r), 0), A.T) : r, b = A.starts ? min(max(__ldg(A.starts + r + 1), a), A.T) : r + 1;
            return (b - a + per_tile - 1) / per_tile;
        };
        int mine = 0;
        for (int r = r0; r < r1; r++) mine += blocks(r);
        int upto = mine;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int v = __shfl_up_sync(~0u, upto, d);
            if (lane >= d) upto += v;
        }
        if (lane == 31) S.warp_sums[warp] = upto;
        __syncthreads();
        for (int w = 0; w < warp; w++) upto += S.warp_sums[w];
        int before = upto - mine;
        if ((int)blockIdx.x >= before && (int)blockIdx.x < upto)
            for (int r = r0; r < r1; r++) {
                const int n = blocks(r);
                if ((int)blockIdx.x < before + n) {
                    S.request = r;
                    S.block = n - 1 - ((int)blockIdx.x - before);
                    break;
                }
                before += n;
            }
    }
    if (tid == 32) {
        for (int i = 0; i < DEPTH; i++) mk::mbar_init(&S.full[i], I4 ? L::PRODUCERS : 1), mk::mbar_init(&S.empty[i], 1);
        for (int i = 0; i < 2; i++) mk::mbar_init(&S.scores[i], 1), mk::mbar_init(&S.probs[i], 8);
        mk::mbar_init(&S.done, 1);
        mk::mbar_init(&S.queries, I4 ? 8 : 1);
        for (int i = 0; i < 3; i++) mk::mbar_init(&S.landed[i], 1);
        mk::fence_barrier_init();
    }
    __syncthreads();
    if (S.request < 0) return;                                         // the grid is an upper bound
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&S.tmem)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    const int r = S.request, head = blockIdx.y;
    const int first = A.starts ? min(max(__ldg(A.starts + r), 0), A.T) : r, count = A.starts ? min(max(__ldg(A.starts + r + 1), first), A.T) - first : 1;
    const int context = (int)min((long long)max(__ldg(A.context + r), 0), (long long)A.max_pages << A.page_shift);
    const int token0 = S.block * per_tile, tokens = min(per_tile, count - token0), rows = tokens * A.per;
    const int pos_lo = context - count + token0, pos_hi = pos_lo + tokens - 1;
    const Tiles tl = tiles_of(A, pos_lo, pos_hi);
    const int win_lo = A.window ? pos_lo - A.window + 1 : 0;
    auto key0_of = [&](int tile) { return (tile < tl.front ? tile : tl.from + tile - tl.front) * R_KEYS; };

    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = S.tmem;

    if (warp >= 8 && warp < MMA_WARP) {
        // ================= producers: chunks in the order K0, K1 V0, K2 V1, ... (CH of each) ======================
        const int pw = warp - 8;
        uint32_t slot = 0, phase = 0, patches = 0;
        bool ok = true;
        auto room = [&](uint32_t s, uint32_t ph) { return __all_sync(~0u, rows_wait(S, A, &S.empty[s], ph ^ 1u, WA_EMPTY)) != 0; };
        auto pages_of = [&](int key0) {
            // lane l < 8: the page of the tile's keys 16 l ..., -1 outside the cache
            const int key = key0 + 16 * (lane & 7), n = key >> A.page_shift;
            const int page = n < A.max_pages ? __ldg(A.table + r * A.table_stride + n) : -1;
            return page >= 0 && page < A.pages ? page : -1;
        };
        auto seen = [&](int key) { return key <= pos_hi && (key >= win_lo || key < A.sinks); };
        if constexpr (!I4) {
            // the queries: a box of the block's tokens and the KV head's query heads is 128 rows or a few less (what the tensor holds behind
            // the block's tokens fills rows that go nowhere)
            if (pw == 0 && lane == 0) {
                mk::mbar_expect_tx(&S.queries, (uint32_t)(per_tile * A.per * HD * 2));
                for (int x = 0; x < G; x++)
                    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(q_s) + x * R_ROWS * 128), "l"(&M.q),
                                 "r"(x * 64), "r"(head * A.per), "r"(first + token0), "r"(smem_u32(&S.queries))
                                 : "memory");
            }
            __syncwarp();
        }
        // step 0: K0; then K(i + 1), V(i) by turns; the last one V(n - 1)
        const int steps = 2 * tl.n;
        auto is_value = [&](int step) { return step == steps - 1 || (step > 0 && (step & 1) == 0); };
        auto tile_at = [&](int step) { return step == 0 ? 0 : (step == steps - 1 ? tl.n - 1 : ((step & 1) ? (step + 1) / 2 : step / 2 - 1)); };
        auto tell_valid = [&](int tile, int my_page) {
            const uint32_t v = __ballot_sync(~0u, my_page >= 0) & 0xFFu;
            if (lane == 0) S.valid[tile & 7] = v;
        };
        if constexpr (I4) {
            // Half a step at a time, 64 rows, two threads a row (four runs of eight values of every group each).  The codes of the next two halves
            // are on their way while this one's are turned into halves, and the pages of the tile behind.
            const int half = lane & 1;
            int page_v = -1, page_k = tl.n ? pages_of(key0_of(0)) : -1, page_next = tl.n > 1 ? pages_of(key0_of(1)) : -1;      // of V(i), K(i + 1) and K(i + 2)
            struct Raw {
                uint32_t w[4 * G], m[G], of_values[G];
            };
            auto get = [&](int part, Raw& x) {
                const int step = part >> 1, tile = tile_at(step), run = (part & 1) * 4 + pw, key = key0_of(tile) + run * 16 + (lane >> 1);
                const bool value = is_value(step);
                if (!value && !(part & 1) && step > 0) {                // on to the next tile's keys
                    page_v = page_k, page_k = page_next;
                    page_next = tile + 1 < tl.n ? pages_of(key0_of(tile + 1)) : -1;
                }
                const int my_page = value && step != steps - 1 ? page_v : page_k;                      // (the last values are those of the last keys)
                if (!value && pw == 0 && !(part & 1)) tell_valid(tile, my_page);
                const int page = __shfl_sync(~0u, my_page, run);
                const bool live = page >= 0 && seen(key);
                const long long at = (((long long)max(page, 0) * A.nkv + head) << A.page_shift) + (key & ((1 << A.page_shift) - 1));
                const uint8_t* src = (value ? A.v : A.k) + at * (HD / 2) + half * (HD / 4);
#pragma unroll
                for (int j = 0; j < G; j++) *reinterpret_cast<uint4*>(x.w + 4 * j) = live ? __ldg(reinterpret_cast<const uint4*>(src) + j) : make_uint4(0, 0, 0, 0);
                auto scales = [&](uint32_t (&to)[G], const uint8_t* base, bool wanted) {
                    const uint8_t* p = base + at * (G * 4);
                    if constexpr (G == 4) *reinterpret_cast<uint4*>(to) = wanted ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
                    else if constexpr (G == 2) *reinterpret_cast<uint2*>(to) = wanted ? __ldg(reinterpret_cast<const uint2*>(p)) : make_uint2(0, 0);
                    else to[0] = wanted ? __ldg(reinterpret_cast<const uint32_t*>(p)) : 0u;
                };
                scales(x.m, value ? A.vs : A.ks, live);
                scales(x.of_values, A.vs, live && !value);
            };
            auto warp_exp = [&](const uint32_t (&s)[G]) {
                float big = 0.f;
#pragma unroll
                for (int g = 0; g < G; g++) big = fmaxf(big, fmaxf(15.f * __uint_as_float(s[g] << 16), fabsf(__uint_as_float(s[g] & 0xFFFF0000u))));
                return exponent_of(__uint_as_float(__reduce_max_sync(~0u, __float_as_uint(big))));
            };
            uint32_t sl[CH];
            auto put = [&](int part, const Raw& x) {
                const int step = part >> 1, p = part & 1;
                const bool value = is_value(step);
                const int e = warp_exp(x.m);
                if (!value) {
                    const int ev = warp_exp(x.of_values), tile = tile_at(step) & 7;
                    if (lane == 0) S.exps[tile][p * 4 + pw] = e, S.exps[tile][8 + p * 4 + pw] = ev;
                }
                if (p == 0) {
                    uint32_t ph[CH];
#pragma unroll
                    for (int c = 0; c < CH; c++) {
                        sl[c] = slot, ph[c] = phase;
                        if (++slot == DEPTH) slot = 0, phase ^= 1u;
                    }
#pragma unroll
                    for (int c = 0; c < CH; c++) ok = ok && room(sl[c], ph[c]);
                    if (!ok) return;
                }
                const float down = power(-e);
                const int slab = (value ? R_KEYS / CH : R_KEYS) * 128, row = (p * 4 + pw) * 16 + (lane >> 1), row_in = value && CH == 2 ? row & 63 : row;   // (values: a chunk is 64 keys, keys: 128 dims)
#pragma unroll
                for (int g = 0; g < G; g++) {
                    const float s1 = __uint_as_float(x.m[g] << 16) * down, l1 = __uint_as_float(x.m[g] & 0xFFFF0000u) * down;
                    const uint32_t s2 = pack_half(s1, s1), l2 = pack_half(l1, l1);
                    const uint32_t to = CH == 1 ? sl[0] : (value ? (p ? sl[CH - 1] : sl[0]) : sl[g >> 1 & (CH - 1)]);
                    uint8_t* dst = ring + to * L::SLOT + (CH == 2 && !value ? g & 1 : g) * slab + row_in * 128;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const uint32_t c = x.w[j * G + g];
                        *reinterpret_cast<uint4*>(dst + (((half * 4 + j) ^ (row & 7)) << 4)) =
                            make_uint4(fma_half2(codes<0>(c), s2, l2), fma_half2(codes<1>(c), s2, l2), fma_half2(codes<2>(c), s2, l2), fma_half2(codes<3>(c), s2, l2));
                    }
                }
                if (p == 1) {
                    mk::fence_proxy_async();
                    __syncwarp();
                    if (lane == 0)
#pragma unroll
                        for (int c = 0; c < CH; c++) mk::mbar_arrive(&S.full[sl[c]]);
                }
            };
            Raw x, y, z;
            const int parts = 2 * steps;
            auto one = [&](int part, const Raw& now, Raw& far) {
                if (part >= parts || !ok) return;
                if (part + 2 < parts) get(part + 2, far);
                put(part, now);
            };
            if (parts) get(0, x), get(1, y);
            for (int part = 0; part < parts && ok; part += 3) {
                one(part, x, z);
                one(part + 1, y, x);
                one(part + 2, z, y);
            }
        } else {
            // the warps take chunks by turns: issuing one's loads takes as long as multiplying it
            const int box_shift = 31 - __clz(M.box);
            for (int q = pw; q < steps * CH && ok; q += L::PRODUCERS) {
                const int step = q / CH, c = q % CH, tile = tile_at(step), key0 = key0_of(tile), my_page = pages_of(key0);
                const bool value = is_value(step);
                slot = q % DEPTH, phase = q / DEPTH & 1;
                if (!value && c == 0) tell_valid(tile, my_page);
                // keys that a query of the block, or of a later one, sees hold values; so do all sinks
                const uint32_t pages = __ballot_sync(~0u, my_page >= 0);                                   // a bit per run of 16 keys (boxes are whole pages, or parts of one)
                const bool clean = (pages & 0xFFu) == 0xFFu && key0 + R_KEYS <= context && (key0 >= win_lo || key0 + R_KEYS <= A.sinks);
                uint8_t* dst = ring + slot * L::SLOT;
                // keys: all 128, dims 128 c ...; values (of a head of 256): keys 64 c ..., all dims
                const bool by_keys = value && CH == 2;
                const int n = by_keys ? 64 : R_KEYS, from = by_keys ? 64 * c : 0, d0 = by_keys ? 0 : c * 128, slab_shift = HD == 64 ? 0 : (by_keys ? 2 : 1);
                uint64_t* bar = value && !clean ? &S.landed[pw] : &S.full[slot];
                const int x = lane & ((1 << slab_shift) - 1), row = (lane >> slab_shift) << box_shift, off = (key0 + from + row) & ((1 << A.page_shift) - 1);
                const int page = __shfl_sync(~0u, my_page, (from + row) >> 4 & 7);
                const bool mine = row < n && page >= 0;
                const uint32_t loads = __popc(__ballot_sync(~0u, mine));
                if (!(ok = room(slot, phase))) break;
                if (lane == 0) {
                    if (loads) mk::mbar_expect_tx(bar, loads * M.box * 128);
                    else mk::mbar_arrive(bar);
                }
                __syncwarp();
                if (mine)
                    tile_load(smem_u32(dst) + x * n * 128 + row * 128, value ? &M.v : &M.k, d0 + x * 64, M.heads_inside ? head : off, M.heads_inside ? off : head, page, bar);
                __syncwarp();
                if (value && !clean) {
                    if (!(ok = __all_sync(~0u, rows_wait(S, A, &S.landed[pw], patches & 1, WA_LANDED)) != 0)) break;
                    patches++;
                    // a lane per row; the pieces by turns, so that the lanes' stores spread over the banks
                    for (int r0 = 0; r0 < n; r0 += 32) {
                        const int line = r0 + lane;
                        if (!(pages >> ((from + line) >> 4) & 1) || !seen(key0 + from + line))
#pragma unroll 8
                            for (int i = 0; i < 8 << slab_shift; i++) *reinterpret_cast<uint4*>(dst + (i >> 3) * n * 128 + line * 128 + ((i + lane & 7) << 4)) = make_uint4(0, 0, 0, 0);
                    }
                    mk::fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) mk::mbar_arrive(&S.full[slot]);
                }
            }
        }
        if (!I4 && S.dead) {
            // loads under way still write shared memory: a bounded wait for them
            const unsigned long long t0 = mk::globaltimer();
            while (mk::globaltimer() - t0 < 1000000ull) {}
        }
    } else if (warp == MMA_WARP) {
        // ================= the products ===============================================================================
        if (lane == 0) {
            constexpr uint32_t type = BF ? (1u << 7) | (1u << 10) : 0u, m128 = 8u << 24;
            constexpr uint32_t id_s = (1u << 4) | type | ((R_KEYS >> 3) << 17) | m128, id_o = (1u << 4) | type | (1u << 16) | ((HD >> 3) << 17) | m128;
            uint32_t slot = 0, phase = 0;
            bool ok = true;
            auto next = [&]() {
                if (!rows_wait(S, A, &S.full[slot], phase, WA_FULL)) return false;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                return true;
            };
            auto release = [&]() {
                commit(&S.empty[slot]);
                if (++slot == DEPTH) slot = 0, phase ^= 1u;
            };
            auto scores = [&](int tile) {
                for (int c = 0; c < CH; c++) {
                    if (!next()) return false;
                    const uint32_t k = smem_u32(ring + slot * L::SLOT), q = smem_u32(q_s) + c * 2 * R_ROWS * 128;
                    constexpr int SLABS = HD >= 128 ? 2 : 1;
#pragma unroll
                    for (int x = 0; x < SLABS; x++) {
                        const uint64_t da = k_major(q + x * R_ROWS * 128), db = k_major(k + x * R_KEYS * 128);
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
                                         ::"r"(tmem + (tile & 1) * 128), "l"(da + 2 * i), "l"(db + 2 * i), "r"(id_s), "r"((uint32_t)(c + x + i > 0)));
                    }
                    release();
                }
                commit(&S.scores[tile & 1]);
                return true;
            };
            ok = rows_wait(S, A, &S.queries, 0, WA_QUERIES);
            ok = ok && (tl.n == 0 || scores(0));
            for (int i = 0; i < tl.n && ok; i++) {
                if (i + 1 < tl.n) {
                    // the accumulator still holds the probabilities of tile i - 1
                    if (i > 0) ok = rows_wait(S, A, &S.done, (i - 1) & 1, WA_DONE);
                    if (!(ok = ok && scores(i + 1))) break;
                }
                if (!(ok = rows_wait(S, A, &S.probs[i & 1], (i >> 1) & 1, WA_PROBS))) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                for (int c = 0; c < CH && ok; c++) {
                    if (!(ok = next())) break;
                    constexpr int KEYS = R_KEYS / CH;
                    const uint64_t db = mn_major(smem_u32(ring + slot * L::SLOT), KEYS * 128);
#pragma unroll
                    for (int x = 0; x < KEYS / 16; x++)
                        asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
                                     ::"r"(tmem + T_O), "r"(tmem + (i & 1) * 128 + (c * KEYS + x * 16) / 64 * 64 + (c * KEYS + x * 16) % 64 / 2), "l"(db + x * 128), "r"(id_o), "r"((uint32_t)(i + c + x > 0)));
                    release();
                }
                if (ok) commit(&S.done);
            }
        }
        __syncwarp();
    } else {
        // ================= softmax and output: two threads a row, 64 keys (later half of the dims) each; rows behind the last repeat it ====
        const int half = warp >> 2, row = tid & 127, n = min(row, rows - 1), token = n / A.per, h = n - token * A.per, pos = pos_lo + token;
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        if constexpr (I4) {
            // the queries: a warp's lanes turn 16 of its rows into halves one after the other
            const uint16_t* own = reinterpret_cast<const uint16_t*>(A.q) + (first + token0 + token) * A.q_tok + (long long)(head * A.per + h) * A.q_head;
            const bool has = lane < HD / 8;
            uint4 x[16];
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const uint16_t* p = reinterpret_cast<const uint16_t*>(__shfl_sync(~0u, (unsigned long long)own, half * 16 + i)) + lane * 8;
                x[i] = has ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int at = (warp & 3) * 32 + half * 16 + i;
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
            mk::fence_proxy_async();
            __syncwarp();
            if (lane == 0) mk::mbar_arrive(&S.queries);
        }
        // barrier of the eight warps; whether any of them has given up, the same answer for all
        auto failed = [](bool mine) {
            uint32_t any;
            asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 q, %1, 0;\n bar.red.or.pred p, 1, 256, q;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(any) : "r"((uint32_t)mine) : "memory");
            return any != 0;
        };
        if constexpr (I4) failed(false);
        float ref = -INFINITY, sum = 0.f;
        const float scale = A.scale_log2 * (I4 ? power(S.q_exp[row]) : 1.f);
        bool ok = true;
        for (int i = 0; i < tl.n; i++) {
            ok = __all_sync(~0u, rows_wait(S, A, &S.scores[i & 1], (i >> 1) & 1, WA_SCORES)) && ok;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const int key0 = key0_of(i);
            const uint32_t at = lanes + (i & 1) * 128 + half * 64, valid = *(volatile uint32_t*)&S.valid[i & 7];
            const bool whole = valid == 0xFFu && key0 + R_KEYS - 1 <= pos_lo && (!A.window || key0 > pos_hi - A.window || key0 + R_KEYS <= A.sinks);
            // the keys this row sees, a bit each
            uint32_t bits[2] = {~0u, ~0u};
            if (!whole) {
                auto below = [](int n, int w) { return n >= 32 * w + 32 ? ~0u : (n <= 32 * w ? 0u : (1u << (n - 32 * w)) - 1); };      // columns under n
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const int w = half * 2 + c;
                    bits[c] = below(pos - key0 + 1, w);
                    if (A.window) bits[c] &= ~below(pos - A.window + 1 - key0, w) | below(A.sinks - key0, w);
                    bits[c] &= (valid >> (2 * w) & 1 ? 0xFFFFu : 0u) | (valid >> (2 * w + 1) & 1 ? 0xFFFF0000u : 0u);
                }
            }
            // factors of a run of 16 keys: of its scores, and the exponent of its values
            float f[4], ev[4];
            if constexpr (I4) {
#pragma unroll
                for (int j = 0; j < 4; j++) f[j] = scale * power(S.exps[i & 7][half * 4 + j]), ev[j] = (float)S.exps[i & 7][8 + half * 4 + j];
            }
            uint32_t x[2][32];
            float top = -INFINITY;
            tmem_ld32(x[0], at);
            tmem_ld32(x[1], at + 32);
            tmem_wait_ld(x[0]);
            tmem_wait_ld(x[1]);
            if (!whole) {
#pragma unroll
                for (int j = 0; j < 64; j++) x[j >> 5][j & 31] = bits[j >> 5] >> (j & 31) & 1 ? x[j >> 5][j & 31] : 0xFF800000u;                   // -inf
            }
            float a[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < 64; j++) a[j >> 4] = fmaxf(a[j >> 4], __uint_as_float(x[j >> 5][j & 31]));
            if constexpr (I4) {
#pragma unroll
                for (int j = 0; j < 4; j++) top = fmaxf(top, fmaf(a[j], f[j], ev[j]));
            } else
                top = fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])) * scale;
            S.tops[i & 1][half][row] = top;
            if (failed(!ok)) {                                         // (all eight warps leave together: they share this barrier)
                ok = false;
                break;
            }
            top = fmaxf(top, S.tops[i & 1][half ^ 1][row]);
            // the reference rises when a score exceeds it by 2^8
            if (__any_sync(~0u, top > ref + 8.f)) {
                const float next = fmaxf(ref, top), turn = next == -INFINITY ? 1.f : exp2_fast(ref - next);
                sum *= turn;
                ref = next;
                if (i > 0) {
                    ok = __all_sync(~0u, rows_wait(S, A, &S.done, (i - 1) & 1, WA_DONE)) && ok;
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
                    tmem_wait_st();
                }
            }
            const float base = ref == -INFINITY ? 0.f : ref;
#pragma unroll
            for (int c = 0; c < 2; c++) {
                float part[4] = {0.f, 0.f, 0.f, 0.f};
                uint32_t p[16];
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    const float fj = I4 ? f[2 * c + (j >> 4)] : scale, bj = I4 ? ev[2 * c + (j >> 4)] - base : -base;
                    // (masked scores are -inf: their probability is 0)
                    const float u = exp2_fast(fmaf(__uint_as_float(x[c][j]), fj, bj)), v = exp2_fast(fmaf(__uint_as_float(x[c][j + 1]), fj, bj));
                    part[j >> 4] += u, part[2 + (j >> 4)] += v;
                    p[j / 2] = BF ? pack_bf(u, v) : pack_half(u, v);
                }
                if constexpr (I4) sum += (part[0] + part[2]) * power(-S.exps[i & 7][8 + half * 4 + 2 * c]) + (part[1] + part[3]) * power(-S.exps[i & 7][9 + half * 4 + 2 * c]);
                else sum += (part[0] + part[2]) + (part[1] + part[3]);
                tmem_st16(at + c * 16, p);                             // over scores that this thread has read
            }
            tmem_wait_st();
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mk::mbar_arrive(&S.probs[i & 1]);
        }
        S.tops[tl.n & 1][half][row] = sum;
        if (failed(!ok)) ok = false;                                   // nothing is written then
        sum += S.tops[tl.n & 1][half ^ 1][row];
        // (one after the other: a parity names a phase only among two)
        for (int i = max(tl.n - 2, 0); i < tl.n && ok; i++) ok = __all_sync(~0u, rows_wait(S, A, &S.done, i & 1, WA_DONE));
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
    }
    __syncthreads();
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (S.dead) {
            // a wait ran out: products under way still read shared and tensor memory, so this waits a bounded time for them
            const unsigned long long t0 = mk::globaltimer();
            while (mk::globaltimer() - t0 < 1000000ull) {}
        }
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
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
    const int page = 1 << A.page_shift, most = head_dim == 256 ? 64 : R_KEYS;
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
static int launch_one(const AttendArgs& A, cudaStream_t st) {
    using L = RowsLayout<HD, KIND>;
    constexpr int smem = L::Q_BYTES + L::DEPTH * L::SLOT + (int)sizeof(RowsShared) + 1024;
    static_assert(smem <= 232448 && smem > 116 * 1024, "one CTA per SM: it takes all of the tensor memory");
    const int per_tile = R_ROWS / A.per;
    // every request rounds up once
    const long long blocks = (long long)A.T / per_tile + (A.T < A.R ? A.T : A.R);
    Maps M;
    if (KIND == K_INT4) memset(&M, 0, sizeof M);
    else {
        const int rc = make_maps(A, HD, KIND == K_F16, &M);
        if (rc != MK_OK) return rc;
    }
    MKV_CUDA(cudaFuncSetAttribute(attend_rows<HD, KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    MKV_CUDA(launch(attend_rows<HD, KIND>, dim3((unsigned)blocks, A.nkv), L::THREADS, smem, 1, false, st, A, M));
    return MK_OK;
}
template <int HD>
static int launch_hd(const AttendArgs& A, int type, cudaStream_t st) {
    return type == MKV_INT4 ? launch_one<HD, K_INT4>(A, st) : (type == MKV_F16 ? launch_one<HD, K_F16>(A, st) : launch_one<HD, K_BF16>(A, st));
}
int launch_rows(const AttendArgs& A, int type, int head_dim, cudaStream_t st) {
    return head_dim == 64 ? launch_hd<64>(A, type, st) : (head_dim == 128 ? launch_hd<128>(A, type, st) : launch_hd<256>(A, type, st));
}

}  // namespace mkv
