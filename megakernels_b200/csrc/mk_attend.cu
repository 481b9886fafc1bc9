// Attention over a paged cache (declarations and rule: include/mk_serve.h).
//
// attend_step: few rows per SM (by_tiles).  Rows are the (token, query head) pairs of a KV head, eight at a time; a unit is (request, KV
// head, eight rows), and its work the tiles of 16 keys that they see.  All tiles of a call form one line, dealt to the CTAs in equal
// runs; inside a run a warp takes every eighth (sixth, twelfth) tile, on its own: it copies the tile's rows into a ring of its own (cp.async, no barrier),
// multiplies them as they lie and keeps running maxima, sums and outputs in registers.  Scores are keys x dims x queries with
// the 16 keys as rows of mma.sync (m16n8k16), outputs dims x keys x queries; which dims and keys stand for which
// row or column of a fragment is free, and chosen so that a lane multiplies whole 16-byte runs of the cache rows.
//   A 4-bit row is never turned into values: a code becomes a half by an OR and a subtraction, the product of codes is corrected per
// group (score = sum_g scale_g (q . c)_g + low_g sum(q)_g; output: p scale_g as the second operand, and one product with the lows).
//   What bounds it is the cache's bytes; the ring keeps 16 to 37 KB per SM in flight.
// attend_join: adds the parts of units that several CTAs share, in their order.
#include "mk_attend.cuh"

namespace mkv {

constexpr int A_ROWS = 8, A_KEYS = 16;

// What a request asks for: its queries and the tiles of 16 keys any of them sees.  The first `front` tiles hold the sinks, the others
// run from tile `from`.
struct Span {
    int first, count, context, tiles, front, from;
};
__device__ __forceinline__ Span span_of(const AttendArgs& A, int r) {
    Span s;
    s.first = A.starts ? min(max(__ldg(A.starts + r), 0), A.T) : r;
    s.count = A.starts ? min(max(__ldg(A.starts + r + 1), s.first), A.T) - s.first : 1;
    s.context = (int)min((long long)max(__ldg(A.context + r), 0), (long long)A.max_pages << A.page_shift);
    const int low = A.window ? max(0, s.context - s.count - A.window + 1) : 0;      // the first query's first key that is no sink
    s.from = low / A_KEYS;
    s.front = A.window ? min((A.sinks + A_KEYS - 1) / A_KEYS, s.from) : 0;
    s.tiles = s.count ? s.front + max((s.context + A_KEYS - 1) / A_KEYS - s.from, 1) : 0;
    return s;
}

// The line of all tiles: prefix[r] = tiles of all units of the requests before r.  Threads of the CTA together.
template <int WARPS>
__device__ __forceinline__ long long build_line(const AttendArgs& A, long long* prefix, long long* warps) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (A.R + WARPS * 32 - 1) / (WARPS * 32), r0 = min(A.R, tid * per), r1 = min(A.R, r0 + per);
    long long mine = 0;
    for (int r = r0; r < r1; r++) {
        const Span s = span_of(A, r);
        prefix[r] = mine;
        mine += (long long)s.tiles * A.nkv * ((s.count * A.per + A_ROWS - 1) / A_ROWS);
    }
    long long x = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const long long v = __shfl_up_sync(~0u, x, d);
        if (lane >= d) x += v;
    }
    if (lane == 31) warps[warp] = x;
    __syncthreads();
    long long before = x - mine, all = 0;
    for (int w = 0; w < WARPS; w++) {
        if (w < warp) before += warps[w];
        all += warps[w];
    }
    for (int r = r0; r < r1; r++) prefix[r] += before;
    if (tid == 0) prefix[A.R] = all;
    __syncthreads();
    return all;
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <int HD, int KIND> struct Layout {
    static constexpr int ROW = KIND == K_INT4 ? HD / 2 : HD * 2;                   // bytes of a cache row
    static constexpr int META = KIND == K_INT4 ? HD / 64 * 4 : 0;
    static constexpr int SLOT = A_KEYS * 2 * (ROW + META);
    static constexpr int WARPS = HD == 256 ? (KIND == K_INT4 ? 12 : 6) : 8;
    static constexpr int DEPTH = KIND == K_INT4 ? (HD == 256 ? 3 : 8) : (HD == 256 ? 2 : (HD == 128 ? 3 : 6));
    static constexpr int JOIN = WARPS * A_ROWS * (HD + 2) * 4;                     // what the warps leave for one another
    static constexpr int RING = WARPS * DEPTH * SLOT > JOIN ? WARPS * DEPTH * SLOT : JOIN;
    static constexpr int REC = 4 + A_ROWS * (HD + 2);                              // floats of a part: header, outputs, maxima, sums
};

// Byte offset of `byte` inside a staged row: the 16-byte pieces of a row are permuted with its number, so that the lanes of one shared-memory
// access (two keys' pieces t or 2 t as rows of the scores, four keys' pieces g and g + 1 as columns of the outputs) touch different banks.
template <int ROW> __device__ __forceinline__ int staged(int row, int byte) {
    if constexpr (ROW >= 128) {
        const int f = (row & 1) * 5 ^ (row >> 2 & 1) * 2 ^ (row >> 3 & 1) * 4;
        return row * ROW + (byte ^ (f << 4));
    } else if constexpr (ROW == 64) return row * ROW + (byte ^ ((row >> 2 & 3) << 4));
    else return row * ROW + (byte ^ ((row >> 2 & 1) << 4));
}

// A row's (scale, low) pairs.
template <int G> __device__ __forceinline__ void load_scales(uint32_t (&m)[G], const uint8_t* p) {
    if constexpr (G == 4) *reinterpret_cast<uint4*>(m) = *reinterpret_cast<const uint4*>(p);
    else if constexpr (G == 2) *reinterpret_cast<uint2*>(m) = *reinterpret_cast<const uint2*>(p);
    else m[0] = *reinterpret_cast<const uint32_t*>(p);
}

template <int HD, int KIND>
static __global__ void __launch_bounds__(Layout<HD, KIND>::WARPS * 32, 1) attend_step(const __grid_constant__ AttendArgs A) {
    using L = Layout<HD, KIND>;
    constexpr int G = HD / 64, A_WARPS = L::WARPS, A_THREADS = A_WARPS * 32;
    constexpr bool I4 = KIND == K_INT4, BF = KIND == K_BF16;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ long long warp_sums[A_WARPS];
    long long* prefix = reinterpret_cast<long long*>(smem + L::RING);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const long long all = build_line<A_WARPS>(A, prefix, warp_sums);
    // equal runs; none shorter than a tile per warp
    const long long ctas = min((long long)gridDim.x, (all + A_WARPS - 1) / A_WARPS), c = blockIdx.x;
    const long long w0 = c < ctas ? all * c / ctas : all, w1 = c < ctas ? all * (c + 1) / ctas : all;
    float* rec = A.part + (size_t)c * 2 * L::REC;
    if (tid < 2) *reinterpret_cast<int4*>(rec + tid * L::REC) = make_int4(0, 0, 0, 0);
    __syncthreads();
    uint8_t* ring = smem + warp * L::DEPTH * L::SLOT;
    const uint32_t ring_u = smem_u32(ring);

    for (long long at = w0; at < w1;) {
        // the unit that holds `at`
        int lo = 0, hi = A.R;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (prefix[mid] <= at) lo = mid;
            else hi = mid;
        }
        const int r = lo;
        const Span s = span_of(A, r);
        const long long in = at - prefix[r];
        const int unit = (int)(in / s.tiles), t0 = (int)(in - (long long)unit * s.tiles), t1 = (int)min((long long)s.tiles, t0 + (w1 - at));
        const int blocks = (s.count * A.per + A_ROWS - 1) / A_ROWS, head = unit / blocks, row0 = (unit - head * blocks) * A_ROWS;
        const int rows = min(A_ROWS, s.count * A.per - row0);
        at += t1 - t0;

        // ---- the queries: row n = g of the second operand
        uint32_t qf[HD / 16][2];
        float qsum[G][2], fix[2] = {1.f, 1.f};          // (of rows 2 t, 2 t + 1)
        const int my_token = (row0 + min(g, rows - 1)) / A.per, my_head = row0 + min(g, rows - 1) - my_token * A.per;
        {
            const uint16_t* src = reinterpret_cast<const uint16_t*>(A.q) + (s.first + my_token) * A.q_tok + (long long)(head * A.per + my_head) * A.q_head;
            if constexpr (I4) {
                // as halves, the row's largest below 2: dims 64 c + 16 t + 8 w + {p, p + 4}
                float big = 0.f;
                uint4 raw[G][2];
#pragma unroll
                for (int c2 = 0; c2 < G; c2++)
#pragma unroll
                    for (int w = 0; w < 2; w++) raw[c2][w] = *reinterpret_cast<const uint4*>(src + c2 * 64 + t * 16 + w * 8);
                auto val = [&](int c2, int w, int i) {
                    const uint32_t x = (&raw[c2][w].x)[i >> 1];
                    return from16((uint16_t)(i & 1 ? x >> 16 : x), A.q_f16);
                };
#pragma unroll
                for (int c2 = 0; c2 < G; c2++)
#pragma unroll
                    for (int w = 0; w < 2; w++)
#pragma unroll
                        for (int i = 0; i < 8; i++) big = fmaxf(big, fabsf(val(c2, w, i)));
                big = fmaxf(big, __shfl_xor_sync(~0u, big, 1));
                big = fmaxf(big, __shfl_xor_sync(~0u, big, 2));
                const int e = big > 0.f && big < INFINITY ? min(max(ilogbf(big), -100), 100) : 0;
                const float down = exp2f((float)-e), up = exp2f((float)e);
#pragma unroll
                for (int c2 = 0; c2 < G; c2++) {
                    float sum = 0.f;
#pragma unroll
                    for (int w = 0; w < 2; w++) {
#pragma unroll
                        for (int i = 0; i < 8; i++) sum += val(c2, w, i) * down;
#pragma unroll
                        for (int p = 0; p < 4; p++) qf[c2 * 4 + w * 2 + (p >> 1)][p & 1] = pack_half(val(c2, w, p) * down, val(c2, w, p + 4) * down);
                    }
                    sum += __shfl_xor_sync(~0u, sum, 1);
                    sum += __shfl_xor_sync(~0u, sum, 2);
                    qsum[c2][0] = __shfl_sync(~0u, sum, 8 * t);
                    qsum[c2][1] = __shfl_sync(~0u, sum, 8 * t + 4);
                }
                fix[0] = __shfl_sync(~0u, up, 8 * t) * A.scale_log2;
                fix[1] = __shfl_sync(~0u, up, 8 * t + 4) * A.scale_log2;
            } else {
                // dims 32 c + 8 t + 0 ... 7
#pragma unroll
                for (int c2 = 0; c2 < HD / 32; c2++) {
                    const uint4 x = *reinterpret_cast<const uint4*>(src + c2 * 32 + t * 8);
                    qf[2 * c2][0] = x.x, qf[2 * c2][1] = x.y, qf[2 * c2 + 1][0] = x.z, qf[2 * c2 + 1][1] = x.w;
                }
                fix[0] = fix[1] = A.scale_log2;
            }
        }
        // positions of the two rows whose scores this lane holds (columns behind the last row repeat it and go nowhere)
        int pos[2];
#pragma unroll
        for (int j = 0; j < 2; j++) pos[j] = s.context - s.count + (row0 + min(2 * t + j, rows - 1)) / A.per;
        const int pos_lo = s.context - s.count + row0 / A.per, pos_hi = s.context - s.count + (row0 + rows - 1) / A.per;
        // keys that no row of the block sees are not read: a page's rest, what lies before the window
        const int win_lo = A.window ? pos_lo - A.window + 1 : 0;

        float o[G * 4][4];
#pragma unroll
        for (int i = 0; i < G * 4; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        float low_acc[4] = {0.f, 0.f, 0.f, 0.f};
        float ref[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
        float v_unit = 0.f, v_inv = 0.f;                 // 4 bits: a power of two about the largest value so far, and its inverse

        auto key0_of = [&](int tile) { return (tile < s.front ? tile : s.from + tile - s.front) * A_KEYS; };
        auto page_of = [&](int key0) {
            const int n = key0 >> A.page_shift;
            const int page = n < A.max_pages ? __ldg(A.table + r * A.table_stride + n) : -1;
            return page >= 0 && page < A.pages ? page : -1;
        };
        // this lane's pieces of a tile: row0, row0 + AT_ONCE, ... (a 4-bit row's address is a compile-time distance from the one before)
        constexpr int P = L::ROW / 16, AT_ONCE = 32 / P > 0 ? 32 / P : 1, STEPS = A_KEYS * P / 32;
        const int row_l = P <= 32 ? lane / P : 0, byte_l = P <= 32 ? (lane % P) * 16 : lane * 16;
        auto place = [&](int j) { return P <= 32 ? staged<L::ROW>(row_l + j * AT_ONCE, byte_l) : staged<L::ROW>(j * 32 / P, byte_l + j * 32 % P * 16); };
        auto fetch = [&](int tile, int slot) {
            if (tile < t1) {
                const int key0 = key0_of(tile), page = page_of(key0), off = key0 & ((1 << A.page_shift) - 1);
                if (page >= 0) {
                    const uint32_t dst = ring_u + slot * L::SLOT;
                    const long long s_pos = I4 ? (long long)L::ROW : A.s_pos, at = page * A.s_page + head * A.s_head + off * s_pos + row_l * s_pos + byte_l;
                    const uint8_t *k = A.k + at, *v = A.v + at;
                    auto seen = [&](int row) { return key0 + row <= pos_hi && (key0 + row >= win_lo || key0 + row < A.sinks); };
                    const bool all = key0 + A_KEYS - 1 <= pos_hi && (key0 >= win_lo || key0 + A_KEYS <= A.sinks);
                    const uint8_t* meta = nullptr;
                    uint32_t meta_to = 0;
                    if constexpr (I4) {
                        const long long row = (((long long)page * A.nkv + head) << A.page_shift) + off + (lane & 15);
                        meta = (lane < 16 ? A.ks : A.vs) + row * L::META;
                        meta_to = dst + A_KEYS * 2 * L::ROW + lane * L::META;
                    }
                    if (all) {
#pragma unroll
                        for (int j = 0; j < STEPS; j++) {
                            const long long o2 = P <= 32 ? j * AT_ONCE * s_pos : (j * 32 / P) * s_pos + j * 32 % P * 16;
                            cp16(dst + place(j), k + o2);
                            cp16(dst + A_KEYS * L::ROW + place(j), v + o2);
                        }
                        if constexpr (I4) {
                            if constexpr (L::META == 16) cp16(meta_to, meta);
                            else cp_small<L::META>(meta_to, meta, true);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < STEPS; j++) {
                            const long long o2 = P <= 32 ? j * AT_ONCE * s_pos : (j * 32 / P) * s_pos + j * 32 % P * 16;
                            const bool live = seen(P <= 32 ? row_l + j * AT_ONCE : j * 32 / P);
                            cp16(dst + place(j), k + o2, live);
                            cp16(dst + A_KEYS * L::ROW + place(j), v + o2, live);
                        }
                        if constexpr (I4) {
                            const bool live = seen(lane & 15);
                            if constexpr (L::META == 16) cp16(meta_to, meta, live);
                            else cp_small<L::META>(meta_to, meta, live);
                        }
                    }
                }
            }
            cp_commit();
        };

        __syncwarp();
#pragma unroll
        for (int d = 0; d < L::DEPTH - 1; d++) fetch(t0 + warp + d * A_WARPS, d);
        int slot = 0;
#pragma unroll 1
        for (int tile = t0 + warp; tile < t1; tile += A_WARPS) {
            __syncwarp();                                                          // the slot's last readers are through
            fetch(tile + (L::DEPTH - 1) * A_WARPS, slot == 0 ? L::DEPTH - 1 : slot - 1);
            cp_wait<L::DEPTH - 1>();
            __syncwarp();
            const uint8_t *ks = ring + slot * L::SLOT, *vs = ks + A_KEYS * L::ROW;
            slot = slot + 1 == L::DEPTH ? 0 : slot + 1;
            const int key0 = key0_of(tile);
            if (page_of(key0) < 0) continue;
            // ---- scores: rows g and g + 8 of the tile are keys ka and ka + 2
            const int ka = 4 * (g >> 1) + (g & 1);
            float sc[4] = {0.f, 0.f, 0.f, 0.f};
            if constexpr (I4) {
                const uint8_t* ms = ks + A_KEYS * 2 * L::ROW;
                uint32_t ma[G], mb[G];
                load_scales<G>(ma, ms + ka * L::META);
                load_scales<G>(mb, ms + (ka + 2) * L::META);
                // a row's words are [8][G]: lane t multiplies words (2 t, .) and (2 t + 1, .)
                uint32_t wa[2 * G], wb[2 * G];
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const uint8_t* p = ks;
                    uint32_t* w = x ? wb : wa;
                    const int row = ka + 2 * x;
                    if constexpr (G == 4) {
                        *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p + staged<L::ROW>(row, t * 32));
                        *reinterpret_cast<uint4*>(w + 4) = *reinterpret_cast<const uint4*>(p + staged<L::ROW>(row, t * 32 + 16));
                    } else if constexpr (G == 2) {
                        *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p + staged<L::ROW>(row, t * 16));
                    } else {
                        *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p + staged<L::ROW>(row, t * 8));
                    }
                }
#pragma unroll
                for (int c2 = 0; c2 < G; c2++) {
                    float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int w = 0; w < 2; w++) {
                        const uint32_t a = wa[w * G + c2], b = wb[w * G + c2];
                        mma<false>(x, codes<0>(a), codes<0>(b), codes<1>(a), codes<1>(b), qf[c2 * 4 + w * 2][0], qf[c2 * 4 + w * 2][1]);
                        mma<false>(x, codes<2>(a), codes<2>(b), codes<3>(a), codes<3>(b), qf[c2 * 4 + w * 2 + 1][0], qf[c2 * 4 + w * 2 + 1][1]);
                    }
                    const float sa = __uint_as_float(ma[c2] << 16), la = __uint_as_float(ma[c2] & 0xFFFF0000u), sb = __uint_as_float(mb[c2] << 16), lb = __uint_as_float(mb[c2] & 0xFFFF0000u);
                    sc[0] = fmaf(sa, x[0], fmaf(la, qsum[c2][0], sc[0]));
                    sc[1] = fmaf(sa, x[1], fmaf(la, qsum[c2][1], sc[1]));
                    sc[2] = fmaf(sb, x[2], fmaf(lb, qsum[c2][0], sc[2]));
                    sc[3] = fmaf(sb, x[3], fmaf(lb, qsum[c2][1], sc[3]));
                }
            } else {
                float sd[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c2 = 0; c2 < HD / 32; c2++) {
                    const uint4 a = *reinterpret_cast<const uint4*>(ks + staged<L::ROW>(ka, c2 * 64 + t * 16)), b = *reinterpret_cast<const uint4*>(ks + staged<L::ROW>(ka + 2, c2 * 64 + t * 16));
                    mma<BF>(sc, a.x, b.x, a.y, b.y, qf[2 * c2][0], qf[2 * c2][1]);
                    mma<BF>(sd, a.z, b.z, a.w, b.w, qf[2 * c2 + 1][0], qf[2 * c2 + 1][1]);
                }
#pragma unroll
                for (int i = 0; i < 4; i++) sc[i] += sd[i];
            }
            // ---- mask, running maximum (raised only when a score exceeds it by 8: probabilities stay below 2^8), probabilities
            const bool whole = key0 + A_KEYS - 1 <= pos_lo && (!A.window || key0 > pos_hi - A.window || key0 + A_KEYS <= A.sinks);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int j = i & 1, key = key0 + ka + (i & 2);
                sc[i] *= fix[j];
                if (!whole && (key > pos[j] || (A.window && key <= pos[j] - A.window && key >= A.sinks))) sc[i] = -INFINITY;
            }
            float top[2] = {fmaxf(sc[0], sc[2]), fmaxf(sc[1], sc[3])};
            // 4 bits: the scales of this lane's four keys (4 t ... 4 t + 3), and the largest of scales and lows as the bits they are (bf16 without a sign orders
            // as a whole number does)
            uint32_t vm[4][G], vbits = 0u;
            const uint8_t* const ms_v = ks + A_KEYS * (2 * L::ROW + L::META);
            if constexpr (I4) {
#pragma unroll
                for (int j = 0; j < 4; j++) load_scales<G>(vm[j], ms_v + (4 * t + j) * L::META);
#pragma unroll
                for (int j = 0; j < 4; j += 2)
#pragma unroll
                    for (int c2 = 0; c2 < G; c2++) vbits = __vimax3_u16x2(vbits, vm[j][c2] & 0x7FFF7FFFu, vm[j + 1][c2] & 0x7FFF7FFFu);
            }
            const float vmax = fmaxf(15.f * __uint_as_float(vbits << 16), __uint_as_float(vbits & 0xFFFF0000u));
            if (__any_sync(~0u, top[0] > ref[0] + 8.f || top[1] > ref[1] + 8.f || (I4 && vmax > 16.f * v_unit))) {
                float f[2];
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    float m = top[j];
                    m = fmaxf(m, __shfl_xor_sync(~0u, m, 4));
                    m = fmaxf(m, __shfl_xor_sync(~0u, m, 8));
                    m = fmaxf(m, __shfl_xor_sync(~0u, m, 16));
                    m = fmaxf(m, ref[j]);
                    f[j] = m == -INFINITY ? 1.f : exp2_fast(ref[j] - m);               // (nothing so far: 0)
                    sum[j] *= f[j];
                    ref[j] = m;
                }
                if constexpr (I4) {
                    float m = vmax;
                    m = fmaxf(m, __shfl_xor_sync(~0u, m, 1));
                    m = fmaxf(m, __shfl_xor_sync(~0u, m, 2));
                    if (m > v_unit && m < INFINITY) {
                        const float next = exp2f((float)min(max(ilogbf(m), -120), 120));
                        if (next > v_unit) {
                            const float turn = v_unit / next;
                            f[0] *= turn, f[1] *= turn;
                            v_unit = next, v_inv = 1.f / next;
                        }
                    }
                    low_acc[0] *= f[0], low_acc[1] *= f[1];
                }
#pragma unroll
                for (int i = 0; i < G * 4; i++) o[i][0] *= f[0], o[i][1] *= f[1], o[i][2] *= f[0], o[i][3] *= f[1];
            }
            float p[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                p[i] = exp2_fast(sc[i] - (ref[i & 1] == -INFINITY ? 0.f : ref[i & 1]));     // (-inf: 0)
                sum[i & 1] += p[i];
            }
            // ---- outputs: rows are dims, this lane's keys 4 t ... 4 t + 3
            if constexpr (I4) {
                const uint32_t p0 = transpose8(pack_half(p[0], p[1])), p1 = transpose8(pack_half(p[2], p[3]));
                uint32_t w[4][G];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint8_t* src = vs + staged<L::ROW>(4 * t + j, g * 4 * G);
                    if constexpr (G == 4) *reinterpret_cast<uint4*>(w[j]) = *reinterpret_cast<const uint4*>(src);
                    else if constexpr (G == 2) *reinterpret_cast<uint2*>(w[j]) = *reinterpret_cast<const uint2*>(src);
                    else w[j][0] = *reinterpret_cast<const uint32_t*>(src);
                }
                // row g of the lows: those of group g (rows past the groups repeat them and go nowhere)
                uint32_t la, lb;
                {
                    float low[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) low[j] = __uint_as_float(*reinterpret_cast<const uint32_t*>(ms_v + (4 * t + j) * L::META + (g & (G - 1)) * 4) & 0xFFFF0000u) * v_inv;
                    la = pack_half(low[0], low[1]), lb = pack_half(low[2], low[3]);
                }
#pragma unroll
                for (int c2 = 0; c2 < G; c2++) {
                    float sv[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) sv[j] = __uint_as_float(vm[j][c2] << 16) * v_inv;
                    const uint32_t b0 = mul_half2(p0, pack_half(sv[0], sv[1])), b1 = mul_half2(p1, pack_half(sv[2], sv[3]));
                    const uint32_t x0 = __byte_perm(w[0][c2], w[1][c2], 0x5410), x1 = __byte_perm(w[0][c2], w[1][c2], 0x7632);
                    const uint32_t y0 = __byte_perm(w[2][c2], w[3][c2], 0x5410), y1 = __byte_perm(w[2][c2], w[3][c2], 0x7632);
                    mma<false>(o[c2 * 4 + 0], codes<0>(x0), codes<0>(x1), codes<0>(y0), codes<0>(y1), b0, b1);
                    mma<false>(o[c2 * 4 + 1], codes<1>(x0), codes<1>(x1), codes<1>(y0), codes<1>(y1), b0, b1);
                    mma<false>(o[c2 * 4 + 2], codes<2>(x0), codes<2>(x1), codes<2>(y0), codes<2>(y1), b0, b1);
                    mma<false>(o[c2 * 4 + 3], codes<3>(x0), codes<3>(x1), codes<3>(y0), codes<3>(y1), b0, b1);
                }
                mma<false>(low_acc, la, 0u, lb, 0u, p0, p1);                       // row g: sum of p low over group g
            } else {
                // probabilities as two bf16 pieces (16 bits), or one half (11)
                const uint32_t h0 = BF ? pack_bf(p[0], p[1]) : pack_half(p[0], p[1]), h1 = BF ? pack_bf(p[2], p[3]) : pack_half(p[2], p[3]);
                const uint32_t p0 = transpose8(h0), p1 = transpose8(h1);
                uint32_t e0 = 0u, e1 = 0u;
                if constexpr (BF) {
                    e0 = transpose8(pack_bf(p[0] - __uint_as_float(h0 << 16), p[1] - __uint_as_float(h0 & 0xFFFF0000u)));
                    e1 = transpose8(pack_bf(p[2] - __uint_as_float(h1 << 16), p[3] - __uint_as_float(h1 & 0xFFFF0000u)));
                }
#pragma unroll
                for (int c2 = 0; c2 < G; c2++) {
                    uint32_t w[4][4];
#pragma unroll
                    for (int j = 0; j < 4; j++) *reinterpret_cast<uint4*>(w[j]) = *reinterpret_cast<const uint4*>(vs + staged<L::ROW>(4 * t + j, c2 * 128 + g * 16));
#pragma unroll
                    for (int i = 0; i < 4; i++) {                                  // dims i and i + 4 of the lane's eight
                        const int sel = i & 1 ? 0x7632 : 0x5410, lo_w = i >> 1, hi_w = 2 + (i >> 1);
                        const uint32_t a0 = __byte_perm(w[0][lo_w], w[1][lo_w], sel), a1 = __byte_perm(w[0][hi_w], w[1][hi_w], sel);
                        const uint32_t a2 = __byte_perm(w[2][lo_w], w[3][lo_w], sel), a3 = __byte_perm(w[2][hi_w], w[3][hi_w], sel);
                        mma<BF>(o[c2 * 4 + i], a0, a1, a2, a3, p0, p1);
                        if constexpr (BF) mma<BF>(o[c2 * 4 + i], a0, a1, a2, a3, e0, e1);
                    }
                }
            }
        }
        cp_wait<0>();
        // ---- the warp's outputs complete: sums over its lanes, 4-bit lows and unit
#pragma unroll
        for (int j = 0; j < 2; j++) {
            sum[j] += __shfl_xor_sync(~0u, sum[j], 4);
            sum[j] += __shfl_xor_sync(~0u, sum[j], 8);
            sum[j] += __shfl_xor_sync(~0u, sum[j], 16);
        }
        if constexpr (I4) {
#pragma unroll
            for (int c2 = 0; c2 < G; c2++) {
                const float l0 = __shfl_sync(~0u, low_acc[0], c2 * 4 + t), l1 = __shfl_sync(~0u, low_acc[1], c2 * 4 + t);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float* x = o[c2 * 4 + i];
                    x[0] = (x[0] + l0) * v_unit, x[1] = (x[1] + l1) * v_unit, x[2] = (x[2] + l0) * v_unit, x[3] = (x[3] + l1) * v_unit;
                }
            }
        }
        __syncthreads();                                                           // nobody's ring is read any more
        float* join = reinterpret_cast<float*>(smem);                              // [warp][row][HD], then [warp][row] maxima, sums
        float *jm = join + A_WARPS * A_ROWS * HD, *js = jm + A_WARPS * A_ROWS;
#pragma unroll
        for (int c2 = 0; c2 < G; c2++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int x = 0; x < 4; x++) join[(warp * A_ROWS + 2 * t + (x & 1)) * HD + c2 * 64 + 8 * g + i + (x & 2 ? 4 : 0)] = o[c2 * 4 + i][x];
        if (g == 0) {
#pragma unroll
            for (int j = 0; j < 2; j++) jm[warp * A_ROWS + 2 * t + j] = ref[j], js[warp * A_ROWS + 2 * t + j] = sum[j];
        }
        __syncthreads();
        const bool begins = t0 == 0, ends = t1 == s.tiles;
        float* part = rec + (begins ? L::REC : 0);
        for (int i = tid; i < rows * HD / 2; i += A_THREADS) {
            const int n = i / (HD / 2), d = (i - n * (HD / 2)) * 2;
            float m = -INFINITY;
#pragma unroll
            for (int w = 0; w < A_WARPS; w++) m = fmaxf(m, jm[w * A_ROWS + n]);
            float l = 0.f, a = 0.f, b = 0.f;
            if (m > -INFINITY) {
#pragma unroll
                for (int w = 0; w < A_WARPS; w++) {
                    const float f = exp2f(jm[w * A_ROWS + n] - m);
                    const float2 x = *reinterpret_cast<const float2*>(join + (w * A_ROWS + n) * HD + d);
                    l = fmaf(f, js[w * A_ROWS + n], l);
                    if (f > 0.f) a = fmaf(f, x.x, a), b = fmaf(f, x.y, b);
                }
            }
            if (begins && ends) {
                const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);        // (a sum that is NaN stays one)
                const int token = (row0 + n) / A.per, h = row0 + n - token * A.per;
                uint16_t* dst = reinterpret_cast<uint16_t*>(A.out) + (s.first + token) * A.out_tok + (long long)(head * A.per + h) * A.out_head + d;
                *reinterpret_cast<uint32_t*>(dst) = A.q_f16 ? pack_half(a * inv, b * inv) : pack_bf(a * inv, b * inv);
            } else {
                *reinterpret_cast<float2*>(part + 4 + n * HD + d) = make_float2(a, b);
                if (d == 0) part[4 + A_ROWS * HD + n] = m, part[4 + A_ROWS * HD + A_ROWS + n] = l;
            }
        }
        if (!(begins && ends) && tid == 0) *reinterpret_cast<int4*>(part) = make_int4(1 | (ends ? 2 : 0), r, head, row0);
        __syncthreads();                                                           // the ring is written again
    }
    grid_release();
}

// Block (c, y) adds up 64 dims of the unit that starts in CTA c and does not end there: its part, then one part of every following CTA until the one that
// ends it.  Maxima and sums of all parts first, side by side, so that nothing is carried from part to part: a single long context is in as many parts
// as there are CTAs (30000 positions of one request, one part after the other: 93 us a call; so 21).
constexpr int J_GROUPS = 4, J_THREADS = J_GROUPS * 256, J_PARTS = 256;
template <int HD>
static __global__ void __launch_bounds__(J_THREADS) attend_join(const __grid_constant__ AttendArgs A, int ctas) {
    constexpr int REC = 4 + A_ROWS * (HD + 2);
    __shared__ float weight[J_PARTS][A_ROWS];
    __shared__ float2 sums[J_GROUPS - 1][256];
    __shared__ int last_s;
    grid_wait();
    const int c = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float* first = A.part + ((size_t)c * 2 + 1) * REC;
    const int4 head = *reinterpret_cast<const int4*>(first);
    if (!head.x || (head.x & 2)) return;
    if (tid == 0) last_s = ctas - 1;
    __syncthreads();
    for (int x = c + 1 + tid; x < ctas; x += J_THREADS)
        if (*reinterpret_cast<const int*>(A.part + (size_t)x * 2 * REC) & 2) atomicMin(&last_s, x);
    __syncthreads();
    const int parts = last_s - c + 1;
    auto part = [&](int i) { return i == 0 ? first : A.part + (size_t)(c + i) * 2 * REC; };
    for (int i = tid; i < parts * A_ROWS; i += J_THREADS) weight[i / A_ROWS][i % A_ROWS] = part(i / A_ROWS)[4 + A_ROWS * HD + i % A_ROWS];
    __syncthreads();
    if (warp < A_ROWS) {
        float m = -INFINITY, l = 0.f;
        for (int i = lane; i < parts; i += 32) m = fmaxf(m, weight[i][warp]);
#pragma unroll
        for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
        for (int i = lane; i < parts; i += 32) {
            const float pm = weight[i][warp], f = pm == -INFINITY ? 0.f : exp2_fast(pm - m);
            if (f > 0.f) l = fmaf(f, part(i)[4 + A_ROWS * HD + A_ROWS + warp], l);
            weight[i][warp] = f;
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) l += __shfl_xor_sync(~0u, l, d);
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);                // (a sum that is NaN stays one)
        for (int i = lane; i < parts; i += 32) weight[i][warp] *= inv;
    }
    __syncthreads();
    const Span s = span_of(A, head.y);
    const int row0 = head.w, rows = min(A_ROWS, s.count * A.per - row0), group = tid >> 8, at = tid & 255, n = at >> 5, d = blockIdx.y * 64 + (at & 31) * 2;
    float2 sum = make_float2(0.f, 0.f);
    if (n < rows) {
#pragma unroll 8
        for (int i = group; i < parts; i += J_GROUPS) {
            const float w = weight[i][n];
            const float2 v = *reinterpret_cast<const float2*>(part(i) + 4 + n * HD + d);
            if (w != 0.f) sum.x = fmaf(w, v.x, sum.x), sum.y = fmaf(w, v.y, sum.y);
        }
    }
    if (group) sums[group - 1][at] = sum;
    __syncthreads();
    if (group || n >= rows) return;
#pragma unroll
    for (int g = 0; g < J_GROUPS - 1; g++) sum.x += sums[g][at].x, sum.y += sums[g][at].y;
    const int token = (row0 + n) / A.per, h = row0 + n - token * A.per;
    uint16_t* dst = reinterpret_cast<uint16_t*>(A.out) + (s.first + token) * A.out_tok + (long long)(head.z * A.per + h) * A.out_head + d;
    *reinterpret_cast<uint32_t*>(dst) = A.q_f16 ? pack_half(sum.x, sum.y) : pack_bf(sum.x, sum.y);
}

static int sm_count(int device) {
    int n = 0;
    return cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) == cudaSuccess ? n : 0;
}

template <int HD, int KIND>
static int launch_step(const AttendArgs& A, int sms, cudaStream_t st) {
    using L = Layout<HD, KIND>;
    const size_t smem = L::RING + (size_t)(A.R + 1) * 8;
    if (sms > J_PARTS) return vfail(MK_ERR_UNSUPPORTED, "mk_attend: %d SMs", sms);
    MKV_CUDA(cudaFuncSetAttribute(attend_step<HD, KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    MKV_CUDA(launch(attend_step<HD, KIND>, dim3(sms), L::WARPS * 32, smem, 1, false, st, A));
    MKV_CUDA(launch(attend_join<HD>, dim3(sms, HD / 64), J_THREADS, 0, 1, true, st, A, sms));
    return MK_OK;
}
template <int HD>
static int launch_kind(const AttendArgs& A, int type, int sms, cudaStream_t st) {
    return type == MKV_INT4 ? launch_step<HD, K_INT4>(A, sms, st) : (type == MKV_F16 ? launch_step<HD, K_F16>(A, sms, st) : launch_step<HD, K_BF16>(A, sms, st));
}

// Which kernel: attend_step reads a request's keys once per eight rows, evenly over all SMs; attend_rows once per 256 (heads of 64: 128), but a pair of
// SMs (an SM) takes all keys of its rows, so the call lasts as many passes as pairs have blocks.  A unit of eight rows costs an SM about what a pass costs a pair: the step
// where there are no more units per SM than passes.  Requests may differ: counted from max_new, or as if half of the last unit (block) of each were empty.  Us, step and tiles, 16 requests of 4000 positions: 16 / 2 heads of 256, bf16, 8, 32, 64 rows
// 39 67, 68 68, 122 68; 24 / 4 heads, 12, 30 rows 68 70, 171 71 (4 bits 68 116, 116 116); 32 / 8 heads of 128, 16, 32 rows 92 104, 166 104 (4 bits 80 151, 146 149);
// 8 / 8 heads of 64, 8, 16 rows 36 54, 56 54.  One request of 8000, 16 / 2 heads of 256: 64, 128 rows 30 112, 41 114.
static bool by_tiles(const AttendArgs& A, int max_new, int head_dim, int sms) {
    const int cg = head_dim >= 128 ? 2 : 1;
    auto count = [&](long long rows) {
        const long long busy = A.R < A.T ? A.R : A.T, each = busy * (((long long)max_new * A.per + rows - 1) / rows), half = (long long)A.T * A.per / rows + busy / 2;
        const long long all = half > busy ? half : busy;
        return A.nkv * (each < all ? each : all);
    };
    const long long passes = (count(128 * cg) + sms / cg - 1) / (sms / cg);
    return count(8) > passes * sms;
}

static const char* bad_attend(const mk_attend_args* a) {
    if (const char* why = bad_cache(a->cache)) return why;
    const mk_cache& c = a->cache;
    if (a->type != MKV_BF16 && a->type != MKV_F16) return "type of the queries";
    if (c.type != MKV_INT4 && c.type != a->type) return "a cache of another 16-bit type than the queries";
    if (a->requests < 1 || a->requests > MKV_MAX_REQUESTS) return "number of requests";
    if (a->tokens < 0 || a->max_pages < 1 || (int64_t)a->max_pages * c.page > 1 << 30) return "tokens or pages per request (at most 2^30 tokens)";
    if ((int64_t)a->tokens * a->q_heads > 1 << 30) return "more than 2^30 query heads in a call";
    if (a->q_heads < 1 || c.kv_heads > 65535 || a->q_heads % c.kv_heads || a->q_heads / c.kv_heads > MKV_MAX_GROUP_HEADS) return "query heads per KV head";
    if (!a->starts && a->tokens != a->requests) return "one query per request, or starts";
    if (a->window < 0 || a->sinks < 0 || a->max_new < 1) return "window, sinks or max_new";
    if (!(a->scale > 0.f && a->scale < 1e30f)) return "scale (positive)";
    return nullptr;
}

}  // namespace mkv

using namespace mkv;

extern "C" int64_t mk_attend_bytes(const mk_attend_args* a) {
    if (!a) return vfail(MK_ERR_BADARG, "mk_attend_bytes: null argument");
    if (const char* why = bad_attend(a)) return vfail(MK_ERR_BADARG, "mk_attend_bytes: %s", why);
    const int sms = sm_count(a->device);
    if (!sms) return vfail(MK_ERR_CUDA, "mk_attend_bytes: no device %d", a->device);
    return (int64_t)sms * 2 * (4 + A_ROWS * (a->cache.head_dim + 2)) * 4;
}

extern "C" int mk_attend(const mk_attend_args* a, void* stream) {
    if (!a) return vfail(MK_ERR_BADARG, "mk_attend: null argument");
    if (const char* why = bad_attend(a)) return vfail(MK_ERR_BADARG, "mk_attend: %s", why);
    if (!a->q || !a->out || !a->table || !a->context || !a->workspace || !a->status) return vfail(MK_ERR_BADARG, "mk_attend: a buffer is missing");
    if (!aligned(a->q, 16) || !aligned(a->out, 16) || !aligned(a->workspace, 16)) return vfail(MK_ERR_BADARG, "mk_attend: queries, outputs or workspace not 16-byte aligned");
    const int64_t strides[] = {a->q_tok, a->q_head, a->out_tok, a->out_head};
    for (int64_t s : strides)
        if (s < 0 || s % 8) return vfail(MK_ERR_BADARG, "mk_attend: stride %lld (a multiple of 8 elements)", (long long)s);
    if ((a->tokens > 1 && a->out_tok < a->cache.head_dim) || (a->q_heads > 1 && a->out_head < a->cache.head_dim))
        return vfail(MK_ERR_BADARG, "mk_attend: rows of out overlap at strides %lld, %lld", (long long)a->out_tok, (long long)a->out_head);
    if (a->table_stride < a->max_pages && a->requests > 1) return vfail(MK_ERR_BADARG, "mk_attend: table rows %lld apart hold no %d pages", (long long)a->table_stride, a->max_pages);
    if (a->tokens == 0) return MK_OK;
    MKV_DEVICE(a->device);
    const int sms = sm_count(a->device);
    const mk_cache& c = a->cache;
    AttendArgs A;
    memset(&A, 0, sizeof A);
    A.q = reinterpret_cast<const void*>(a->q), A.out = reinterpret_cast<void*>(a->out);
    A.k = reinterpret_cast<const uint8_t*>(c.k), A.v = reinterpret_cast<const uint8_t*>(c.v);
    A.ks = reinterpret_cast<const uint8_t*>(c.k_scales), A.vs = reinterpret_cast<const uint8_t*>(c.v_scales);
    A.table = reinterpret_cast<const int*>(a->table), A.context = reinterpret_cast<const int*>(a->context), A.starts = reinterpret_cast<const int*>(a->starts);
    A.part = reinterpret_cast<float*>(a->workspace), A.status = reinterpret_cast<int*>(a->status);
    A.q_tok = a->q_tok, A.q_head = a->q_head, A.out_tok = a->out_tok, A.out_head = a->out_head, A.table_stride = a->table_stride;
    if (c.type == MKV_INT4) {
        A.s_pos = c.head_dim / 2, A.s_head = A.s_pos * c.page, A.s_page = A.s_head * c.kv_heads;
    } else {
        A.s_pos = c.s_pos * 2, A.s_head = c.s_head * 2, A.s_page = c.s_page * 2;
    }
    A.R = a->requests, A.T = a->tokens, A.nq = a->q_heads, A.nkv = c.kv_heads, A.per = a->q_heads / c.kv_heads, A.pages = c.pages;
    A.page_shift = 31 - __builtin_clz(c.page), A.max_pages = a->max_pages, A.q_f16 = a->type == MKV_F16;
    const int longest = a->max_pages * c.page;
    A.window = a->window < longest ? a->window : 0;                                // such a window hides nothing
    A.sinks = a->sinks < longest ? a->sinks : longest;
    A.spin_limit_ns = a->spin_limit_ns > 0 ? a->spin_limit_ns : 2000000000ll;
    A.scale_log2 = a->scale * 1.4426950408889634f;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (by_tiles(A, a->max_new, c.head_dim, sms)) return launch_rows(A, c.type, c.head_dim, sms, st);
    return c.head_dim == 64 ? launch_kind<64>(A, c.type, sms, st) : (c.head_dim == 128 ? launch_kind<128>(A, c.type, sms, st) : launch_kind<256>(A, c.type, sms, st));
}
