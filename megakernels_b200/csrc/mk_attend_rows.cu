// Attention of many queries per request over a paged cache (declarations and rule: include/mk_serve.h).
//
// attend_rows: a CTA owns 128 rows, the (token, query head) pairs of one KV head for 128 / (query heads per KV head) tokens, and passes
// over the keys they see in tiles of 128.  Warps 0-3: one row per thread, softmax and output; warps 4 on: producers, which bring keys and values into a ring
// of shared memory in the tensor core's swizzled order; the last warp's lane issues the products:
//   S = Q K^T    Q and K from shared memory (both K-major), 128 x 128 scores into one of two accumulators in tensor memory;
//   O += P V     P from tensor memory, where the row's thread put it over its scores, V from shared memory as it lies (MN-major),
//                128 x dim outputs in tensor memory.
// While the softmax works on tile i, the products of S(i + 1) and P(i - 1) V run.  Outputs are scaled again only when a row's maximum rises
// by 2^8 (in tensor memory, by the row's thread, behind the product before).
//   Tiles of 128 keys because a product of 128 x 64 would read its operands from shared memory slower than it multiplies; keys (by dims) and values
// (by keys) of a head of 256 come in halves, so that four 32 KB slots beside the 64 KB of Q hold two products ahead.
//   16 bits: cp.async straight into place, rows that nobody sees as zeros.  Probabilities are rounded to the operands' type, as the product takes both of one type
// (bf16: half of the output's own rounding again).
//   4 bits: eight warps turn codes into halves, one rounding (2^-11) each: the values of 16 keys times a power of two of their own, 2^-E, so
// that any bf16 scale fits.  Keys' E scales the scores; values' E is added to the scores' exponent (sum of p v = sum of (p 2^E)(v 2^-E)) and taken out of the denominator.
// Codes 0 .. 7 of a word come out in the order 0 4 1 5 2 6 3 7; queries are stored and outputs read in the same order.
#include "mk_attend.cuh"
#include "mk_device.cuh"

namespace mkv {

constexpr int R_ROWS = 128, R_KEYS = 128;
enum { WA_EMPTY = 401, WA_FULL, WA_SCORES, WA_PROBS, WA_DONE, WA_QUERIES };

template <int HD, int KIND> struct RowsLayout {
    static constexpr int PRODUCERS = KIND == K_INT4 ? 8 : 4;          // warps
    static constexpr int THREADS = (4 + PRODUCERS + 1) * 32;
    static constexpr int CH = HD == 256 ? 2 : 1;                      // chunks of a tile's keys, and of its values
    static constexpr int SLOT = R_KEYS * HD * 2 / CH, DEPTH = HD == 256 ? 4 : (HD == 128 ? 5 : 8), Q_BYTES = R_ROWS * HD * 2;
};
struct RowsShared {
    uint64_t full[8], empty[8], scores[2], probs[2], done, queries;
    uint32_t tmem;
    volatile int dead;
    int request, block;
    int warp_sums[16];
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

template <int HD, int KIND>
static __global__ void __launch_bounds__(RowsLayout<HD, KIND>::THREADS, 1) attend_rows(const __grid_constant__ AttendArgs A) {
    using L = RowsLayout<HD, KIND>;
    constexpr bool I4 = KIND == K_INT4, BF = KIND == K_BF16;
    constexpr int G = HD / 64, CH = L::CH, DEPTH = L::DEPTH, MMA_WARP = 4 + L::PRODUCERS;
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
        for (int i = 0; i < DEPTH; i++) mk::mbar_init(&S.full[i], L::PRODUCERS), mk::mbar_init(&S.empty[i], 1);
        for (int i = 0; i < 2; i++) mk::mbar_init(&S.scores[i], 1), mk::mbar_init(&S.probs[i], 4);
        mk::mbar_init(&S.done, 1);
        mk::mbar_init(&S.queries, 4);
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

    if (warp >= 4 && warp < MMA_WARP) {
        // ================= producers: chunks in the order K0, K1 V0, K2 V1, ... (CH of each) ======================
        const int pw = warp - 4;
        uint32_t slot = 0, phase = 0;
        int waiting = 0;                                               // chunks whose copies are under way: the last ones issued, two at most
        bool ok = true;
        auto arrived = [&](int back) {                                 // the chunk `back` before the next one has landed
            mk::fence_proxy_async();
            __syncwarp();
            if (lane == 0) mk::mbar_arrive(&S.full[(slot + DEPTH - back) % DEPTH]);
            waiting--;
        };
        auto land = [&]() {
            cp_wait<0>();
            while (waiting > 0) arrived(waiting);
        };
        auto room = [&](uint32_t s, uint32_t ph) {
            if (__all_sync(~0u, mk::mbar_try_wait(&S.empty[s], ph ^ 1u))) return true;
            land();                                                    // nobody is kept waiting for what has arrived
            return __all_sync(~0u, rows_wait(S, A, &S.empty[s], ph ^ 1u, WA_EMPTY)) != 0;
        };
        auto pages_of = [&](int key0) {
            // lane l < 8: the page of the tile's keys 16 l ..., -1 outside the cache
            const int key = key0 + 16 * (lane & 7), n = key >> A.page_shift;
            const int page = n < A.max_pages ? __ldg(A.table + r * A.table_stride + n) : -1;
            return page >= 0 && page < A.pages ? page : -1;
        };
        auto seen = [&](int key) { return key <= pos_hi && (key >= win_lo || key < A.sinks); };
        for (int step = 0; step <= 2 * tl.n - 1 && ok; step++) {
            // step 0: K0; then K(i + 1), V(i) by turns; the last one V(n - 1)
            const bool value = step == 2 * tl.n - 1 || (step > 0 && (step & 1) == 0);
            const int tile = step == 0 ? 0 : (value ? (step == 2 * tl.n - 1 ? tl.n - 1 : step / 2 - 1) : (step + 1) / 2);
            const int key0 = key0_of(tile), my_page = pages_of(key0);
            if (!value && pw == 0) {
                const uint32_t v = __ballot_sync(~0u, my_page >= 0) & 0xFFu;
                if (lane == 0) S.valid[tile & 7] = v;
            }
            if constexpr (I4) {
                // two threads a row: four runs of eight values of every group each
                const int row = pw * 16 + (lane >> 1), half = lane & 1, page = __shfl_sync(~0u, my_page, pw), key = key0 + row;
                const bool live = page >= 0 && seen(key);
                const long long at = (((long long)max(page, 0) * A.nkv + head) << A.page_shift) + (key & ((1 << A.page_shift) - 1));
                uint32_t mk_[G], mv_[G], w[4 * G];
                auto load = [&](uint32_t (&m)[G], const uint8_t* base) {
                    const uint8_t* p = base + at * (G * 4);
                    if constexpr (G == 4) *reinterpret_cast<uint4*>(m) = live ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
                    else if constexpr (G == 2) *reinterpret_cast<uint2*>(m) = live ? __ldg(reinterpret_cast<const uint2*>(p)) : make_uint2(0, 0);
                    else m[0] = live ? __ldg(reinterpret_cast<const uint32_t*>(p)) : 0u;
                };
                {
                    const uint8_t* p = (value ? A.v : A.k) + at * (HD / 2) + half * (HD / 4);
#pragma unroll
                    for (int j = 0; j < G; j++) *reinterpret_cast<uint4*>(w + 4 * j) = live ? __ldg(reinterpret_cast<const uint4*>(p) + j) : make_uint4(0, 0, 0, 0);
                }
                auto warp_exp = [&](const uint32_t (&m)[G]) {
                    float big = 0.f;
#pragma unroll
                    for (int g = 0; g < G; g++) big = fmaxf(big, fmaxf(15.f * __uint_as_float(m[g] << 16), fabsf(__uint_as_float(m[g] & 0xFFFF0000u))));
#pragma unroll
                    for (int d = 16; d; d >>= 1) big = fmaxf(big, __shfl_xor_sync(~0u, big, d));
                    return exponent_of(big);
                };
                int e;
                if (value) {
                    load(mv_, A.vs);
                    e = warp_exp(mv_);
                } else {
                    load(mk_, A.ks);
                    load(mv_, A.vs);
                    e = warp_exp(mk_);
                    const int ev = warp_exp(mv_);
                    if (lane == 0) S.exps[tile & 7][pw] = e, S.exps[tile & 7][8 + pw] = ev;
                }
                const float down = power(-e);
                uint32_t s2[G], l2[G];
#pragma unroll
                for (int g = 0; g < G; g++) {
                    const uint32_t m = value ? mv_[g] : mk_[g];
                    const float s = __uint_as_float(m << 16) * down, l = __uint_as_float(m & 0xFFFF0000u) * down;
                    s2[g] = pack_half(s, s), l2[g] = pack_half(l, l);
                }
                // both chunks' slots
                uint32_t sl[CH], ph[CH];
#pragma unroll
                for (int c = 0; c < CH; c++) {
                    sl[c] = slot, ph[c] = phase;
                    if (++slot == DEPTH) slot = 0, phase ^= 1u;
                }
#pragma unroll
                for (int c = 0; c < CH; c++) ok = ok && room(sl[c], ph[c]);
                if (!ok) break;
                const int mine = value && CH == 2 ? row >> 6 : 0, row_in = value && CH == 2 ? row & 63 : row;   // (values: a chunk is 64 keys, keys: 128 dims)
                const int slab = (value ? R_KEYS / CH : R_KEYS) * 128;
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int g = 0; g < G; g++) {
                        const uint32_t x = w[j * G + g];
                        const uint4 h = make_uint4(fma_half2(codes<0>(x), s2[g], l2[g]), fma_half2(codes<1>(x), s2[g], l2[g]), fma_half2(codes<2>(x), s2[g], l2[g]), fma_half2(codes<3>(x), s2[g], l2[g]));
                        const int chunk = value ? mine : (CH == 2 ? g >> 1 : 0), slab_no = value ? g : (CH == 2 ? g & 1 : g);
                        *reinterpret_cast<uint4*>(ring + sl[CH == 2 ? chunk : 0] * L::SLOT + slab_no * slab + row_in * 128 + (((half * 4 + j) ^ (row & 7)) << 4)) = h;
                    }
                mk::fence_proxy_async();
                __syncwarp();
                if (lane == 0)
#pragma unroll
                    for (int c = 0; c < CH; c++) mk::mbar_arrive(&S.full[sl[c]]);
            } else {
                // lane l < 8: where the tile's keys 16 l ... begin (they lie one after the other: a page holds whole runs of 16)
                const uint8_t* run = (value ? A.v : A.k) + head * A.s_head + max(my_page, 0) * A.s_page + ((key0 + 16 * (lane & 7)) & ((1 << A.page_shift) - 1)) * A.s_pos;
                const bool all_seen = key0 + R_KEYS - 1 <= pos_hi && (key0 >= win_lo || key0 + R_KEYS <= A.sinks) && __all_sync(~0u, my_page >= 0);
#pragma unroll
                for (int c = 0; c < CH; c++) {
                    if (!ok || !(ok = room(slot, phase))) break;
                    const uint32_t dst = smem_u32(ring + slot * L::SLOT);
                    // P pieces of 16 bytes of N rows from row_from; a warp copies 32 / P rows at a time
                    auto copy = [&](auto pieces_, auto rows_, int row_from, int byte_from) {
                        constexpr int P = decltype(pieces_)::value, N = decltype(rows_)::value, AT_ONCE = 32 / P, SLAB = N * 128, STEP = 4 * AT_ONCE;
                        const int piece = lane % P, row0 = pw * AT_ONCE + lane / P;
                        const long long off = row0 * A.s_pos + byte_from + piece * 16;
                        const uint32_t to = dst + (piece >> 3) * SLAB + row0 * 128;
#pragma unroll
                        for (int u = 0; u < N / 16; u++) {
                            const int from = row_from / 16 + u;
                            const uint8_t* src = reinterpret_cast<const uint8_t*>(__shfl_sync(~0u, (unsigned long long)run, from)) + off;
                            const bool there = all_seen || __shfl_sync(~0u, my_page, from) >= 0;
#pragma unroll
                            for (int i = 0; i < 16 / STEP; i++) {
                                const int row = i * STEP + row0;
                                const bool live = all_seen || (there && seen(key0 + from * 16 + row));
                                cp16(to + u * 2048 + i * STEP * 128 + (((piece & 7) ^ (row & 7)) << 4), src + i * STEP * A.s_pos, live);
                            }
                        }
                    };
                    if constexpr (HD == 256) {
                        if (value) copy(Const<32>{}, Const<64>{}, c * 64, 0);
                        else copy(Const<16>{}, Const<128>{}, 0, c * 256);
                    } else if constexpr (HD == 128) copy(Const<16>{}, Const<128>{}, 0, 0);
                    else copy(Const<8>{}, Const<128>{}, 0, 0);
                    cp_commit();
                    if (waiting == 2) {
                        cp_wait<2>();
                        arrived(2);
                    }
                    waiting++;
                    if (++slot == DEPTH) slot = 0, phase ^= 1u;
                }
            }
        }
        if (ok) land();
        cp_wait<0>();
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
                                     ::"r"(tmem + T_O), "r"(tmem + (i & 1) * 128 + c * (KEYS / 2) + x * 8), "l"(db + x * 128), "r"(id_o), "r"((uint32_t)(i + c + x > 0)));
                    release();
                }
                if (ok) commit(&S.done);
            }
        }
        __syncwarp();
    } else {
        // ================= softmax and output: thread = row (rows behind the last repeat it) ==============================
        const int row = tid, n = min(row, rows - 1), token = n / A.per, h = n - token * A.per, pos = pos_lo + token;
        const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
        {
            // the queries: a warp's lanes copy its 32 rows one after the other
            const uint16_t* own = reinterpret_cast<const uint16_t*>(A.q) + (first + token0 + token) * A.q_tok + (long long)(head * A.per + h) * A.q_head;
            const bool has = lane < HD / 8;
            auto from = [&](int i) { return reinterpret_cast<const uint16_t*>(__shfl_sync(~0u, (unsigned long long)own, i)) + lane * 8; };
            auto place = [&](int i) { return q_s + (lane >> 3) * (R_ROWS * 128) + (warp * 32 + i) * 128 + (((lane & 7) ^ (i & 7)) << 4); };
            if constexpr (I4) {
#pragma unroll 1
                for (int i0 = 0; i0 < 32; i0 += 8) {
                    uint4 x[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const uint16_t* p = from(i0 + i);
                        x[i] = has ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
                    }
#pragma unroll
                    for (int i = 0; i < 8; i++) {
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
                        if (lane == 0) S.q_exp[warp * 32 + i0 + i] = e;
                        if (has) *reinterpret_cast<uint4*>(place(i0 + i)) = make_uint4(pack_half(v[0] * down, v[4] * down), pack_half(v[1] * down, v[5] * down), pack_half(v[2] * down, v[6] * down), pack_half(v[3] * down, v[7] * down));
                    }
                }
            } else {
#pragma unroll 8
                for (int i = 0; i < 32; i++) {
                    const uint16_t* p = from(i);
                    if (has) cp16(smem_u32(place(i)), p, true);
                }
                cp_commit();
                cp_wait<0>();
            }
            mk::fence_proxy_async();
            __syncwarp();
            if (lane == 0) mk::mbar_arrive(&S.queries);
        }
        float ref = -INFINITY, sum = 0.f;
        const float scale = A.scale_log2 * (I4 ? power(S.q_exp[row]) : 1.f);
        bool ok = true;
        for (int i = 0; i < tl.n; i++) {
            if (!__all_sync(~0u, rows_wait(S, A, &S.scores[i & 1], (i >> 1) & 1, WA_SCORES))) {
                ok = false;
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const int key0 = key0_of(i);
            const uint32_t at = lanes + (i & 1) * 128, valid = *(volatile uint32_t*)&S.valid[i & 7];
            const bool whole = valid == 0xFFu && key0 + R_KEYS - 1 <= pos_lo && (!A.window || key0 > pos_hi - A.window || key0 + R_KEYS <= A.sinks);
            // the keys this row sees, a bit each
            uint32_t bits[4] = {~0u, ~0u, ~0u, ~0u};
            if (!whole) {
                auto below = [](int n, int w) { return n >= 32 * w + 32 ? ~0u : (n <= 32 * w ? 0u : (1u << (n - 32 * w)) - 1); };      // columns under n
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    bits[w] = below(pos - key0 + 1, w);
                    if (A.window) bits[w] &= ~below(pos - A.window + 1 - key0, w) | below(A.sinks - key0, w);
                    bits[w] &= (valid >> (2 * w) & 1 ? 0xFFFFu : 0u) | (valid >> (2 * w + 1) & 1 ? 0xFFFF0000u : 0u);
                }
            }
            // factors of a run of 16 keys: of its scores, and the exponent of its values
            float f[8], ev[8];
            if constexpr (I4) {
#pragma unroll
                for (int j = 0; j < 8; j++) f[j] = scale * power(S.exps[i & 7][j]), ev[j] = (float)S.exps[i & 7][8 + j];
            }
            uint32_t x[2][32];
            float top = -INFINITY;
            tmem_ld32(x[0], at);
#pragma unroll
            for (int c = 0; c < 4; c++) {
                tmem_wait_ld(x[c & 1]);
                if (c < 3) tmem_ld32(x[(c + 1) & 1], at + (c + 1) * 32);
                uint32_t (&y)[32] = x[c & 1];
                if (!whole) {
#pragma unroll
                    for (int j = 0; j < 32; j++) y[j] = bits[c] >> j & 1 ? y[j] : 0xFF800000u;                   // -inf
                }
                float a[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < 32; j++) a[j >> 4 | (j & 1) * 2] = fmaxf(a[j >> 4 | (j & 1) * 2], __uint_as_float(y[j]));
                if constexpr (I4) top = fmaxf(top, fmaxf(fmaf(fmaxf(a[0], a[2]), f[2 * c], ev[2 * c]), fmaf(fmaxf(a[1], a[3]), f[2 * c + 1], ev[2 * c + 1])));
                else top = fmaxf(top, fmaxf(fmaxf(a[0], a[2]), fmaxf(a[1], a[3])));
            }
            if constexpr (!I4) top *= scale;
            // the reference rises when a score exceeds it by 2^8
            if (__any_sync(~0u, top > ref + 8.f)) {
                const float next = fmaxf(ref, top), turn = next == -INFINITY ? 1.f : exp2_fast(ref - next);
                sum *= turn;
                ref = next;
                if (i > 0) {
                    if (!__all_sync(~0u, rows_wait(S, A, &S.done, (i - 1) & 1, WA_DONE))) {
                        ok = false;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                    for (int c = 0; c < HD / 32; c++) {
                        tmem_ld32(x[0], lanes + T_O + c * 32);
                        tmem_wait_ld(x[0]);
#pragma unroll
                        for (int j = 0; j < 32; j++) x[0][j] = __float_as_uint(__uint_as_float(x[0][j]) * turn);
                        tmem_st32(lanes + T_O + c * 32, x[0]);
                    }
                    tmem_wait_st();
                }
            }
            const float base = ref == -INFINITY ? 0.f : ref;
            tmem_ld32(x[0], at);
#pragma unroll
            for (int c = 0; c < 4; c++) {
                tmem_wait_ld(x[c & 1]);
                if (c < 3) tmem_ld32(x[(c + 1) & 1], at + (c + 1) * 32);
                uint32_t (&y)[32] = x[c & 1];
                float part[4] = {0.f, 0.f, 0.f, 0.f};
                uint32_t p[16];
#pragma unroll
                for (int j = 0; j < 32; j++) {
                    const float fj = I4 ? f[2 * c + (j >> 4)] : scale, bj = I4 ? ev[2 * c + (j >> 4)] - base : -base;
                    y[j] = __float_as_uint(exp2_fast(fmaf(__uint_as_float(y[j]), fj, bj)));
                }
                if (!whole) {
#pragma unroll
                    for (int j = 0; j < 32; j++) y[j] = bits[c] >> j & 1 ? y[j] : 0u;
                }
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    const float u = __uint_as_float(y[j]), v = __uint_as_float(y[j + 1]);
                    part[j >> 4] += u, part[2 + (j >> 4)] += v;
                    p[j / 2] = BF ? pack_bf(u, v) : pack_half(u, v);
                }
                if constexpr (I4) sum += (part[0] + part[2]) * power(-S.exps[i & 7][8 + 2 * c]) + (part[1] + part[3]) * power(-S.exps[i & 7][9 + 2 * c]);
                else sum += (part[0] + part[2]) + (part[1] + part[3]);
                tmem_st16(at + c * 16, p);
            }
            tmem_wait_st();
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mk::mbar_arrive(&S.probs[i & 1]);
        }
        // (one after the other: a parity names a phase only among two)
        for (int i = max(tl.n - 2, 0); i < tl.n && ok; i++) ok = __all_sync(~0u, rows_wait(S, A, &S.done, i & 1, WA_DONE));
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (ok) {
            const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
            uint16_t* dst = reinterpret_cast<uint16_t*>(A.out) + (first + token0 + token) * A.out_tok + (long long)(head * A.per + h) * A.out_head;
#pragma unroll 1
            for (int c = 0; c < HD / 32; c++) {
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

template <int HD, int KIND>
static int launch_one(const AttendArgs& A, cudaStream_t st) {
    using L = RowsLayout<HD, KIND>;
    constexpr int smem = L::Q_BYTES + L::DEPTH * L::SLOT + (int)sizeof(RowsShared) + 1024;
    static_assert(smem <= 232448 && smem > 116 * 1024, "one CTA per SM: it takes all of the tensor memory");
    const int per_tile = R_ROWS / A.per;
    // every request rounds up once
    const long long blocks = (long long)A.T / per_tile + (A.T < A.R ? A.T : A.R);
    MKV_CUDA(cudaFuncSetAttribute(attend_rows<HD, KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    MKV_CUDA(launch(attend_rows<HD, KIND>, dim3((unsigned)blocks, A.nkv), L::THREADS, smem, 1, false, st, A));
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
