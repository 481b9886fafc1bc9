// Cache pages, and query and key heads on their way into the cache (declarations: include/mk_serve.h).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mk_serve_host.h"

namespace mkv {

// ---- cache pages -------------------------------------------------------------------------------------------------
// One cluster does the whole call, so it is one launch and one grid-wide order of its phases costs a cluster barrier each:
//   A  rank 0 scans the requests (pages returned, pages taken, tokens) and leaves every request's numbers in scratch;
//   B  returned pages go on the stack, a warp per request;
//   C  taken pages go into the tables, a warp per request;
//   D  a thread per token slot finds its request among the starts and looks its page up.
// What bounds it is the chain of four phases, not bytes (1000 requests and 16384 slots move 0.3 MB): a CTA of 1024 threads scans
// 4096 requests in one piece, and eight of them fill the slots.
constexpr int PLAN_THREADS = 1024;

struct PlanArgs {
    const int *lengths, *new_tokens;
    int *table, *held, *free_pages, *n_free;
    int4* scratch;                       // per request: {base, pages returned before it, pages taken before it, pages held before the call}
    int *slots, *positions, *rows, *starts, *context, *granted;
    int R, P, page_shift, n_pages, room;
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\n barrier.cluster.wait.acquire;" ::: "memory");
}

struct Sums {
    int back;                            // at most all pages
    long long take, tokens;              // as asked for, which may be more than there is
};

// Exclusive sums over the threads of a CTA, in thread order, and the totals.
__device__ Sums scan(Sums v, Sums* total, Sums* warps) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Sums x = v;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int a = __shfl_up_sync(~0u, x.back, d);
        const long long b = __shfl_up_sync(~0u, x.take, d), c = __shfl_up_sync(~0u, x.tokens, d);
        if (lane >= d) x.back += a, x.take += b, x.tokens += c;
    }
    __syncthreads();
    if (lane == 31) warps[warp] = x;
    __syncthreads();
    Sums before = {0, 0, 0}, all = {0, 0, 0};
    for (int w = 0; w < PLAN_THREADS / 32; w++) {
        const Sums s = warps[w];
        if (w < warp) before.back += s.back, before.take += s.take, before.tokens += s.tokens;
        all.back += s.back, all.take += s.take, all.tokens += s.tokens;
    }
    *total = all;
    return {before.back + x.back - v.back, before.take + x.take - v.take, before.tokens + x.tokens - v.tokens};
}

static __global__ void __launch_bounds__(PLAN_THREADS, 1) plan_pages(const __grid_constant__ PlanArgs A) {
    extern __shared__ int starts_s[];
    __shared__ Sums warps[PLAN_THREADS / 32];
    const int rank = cluster_rank(), ranks = cluster_size(), tid = threadIdx.x;
    const int page = 1 << A.page_shift;
    int* totals = reinterpret_cast<int*>(A.scratch + A.R);          // {stack height with the returned pages, pages taken}
    if (rank == 0) {
        const int per = (A.R + PLAN_THREADS - 1) / PLAN_THREADS, r0 = min(A.R, tid * per), r1 = min(A.R, r0 + per);
        struct Row {
            int base, back, take, tokens, held, length, need;
            bool valid;
        };
        auto row = [&](int r) {
            Row x;
            const int length = A.lengths[r], fresh = A.new_tokens[r], held = min(max(A.held[r], 0), A.P);
            const long long need = ((long long)length + fresh + page - 1) >> A.page_shift;
            x.valid = length >= 0 && fresh >= 0 && need <= A.P;
            x.need = x.valid ? (int)need : 0;
            x.length = length;
            x.held = held;
            x.base = (int)min((long long)held, ((long long)max(length, 0) + page - 1) >> A.page_shift);
            x.back = held - x.base;
            x.take = x.valid ? max(x.need - x.base, 0) : 0;
            x.tokens = x.valid ? fresh : 0;
            return x;
        };
        Sums mine = {0, 0, 0}, all;
        for (int r = r0; r < r1; r++) {
            const Row x = row(r);
            mine.back += x.back, mine.take += x.take, mine.tokens += x.tokens;
        }
        Sums before = scan(mine, &all, warps);
        const int height = A.n_free[0] + all.back;
        int taken = 0;
        for (int r = r0; r < r1; r++) {
            const Row x = row(r);
            const bool fits = before.take + x.take <= height && before.tokens + x.tokens <= A.room;
            const bool ok = x.valid && (fits || (x.take == 0 && x.tokens == 0));
            A.scratch[r] = make_int4(x.base, before.back, ok ? (int)min(before.take, (long long)height) : 0, x.held);
            A.context[r] = ok ? x.length + x.tokens : (x.valid ? x.length : 0);
            A.granted[r] = ok;
            A.held[r] = ok ? max(x.need, x.base) : x.base;
            if (ok) taken += x.take;
            before.back += x.back, before.take += x.take, before.tokens += x.tokens;
        }
        // tokens again, of the granted requests alone
        Sums got = {0, taken, 0};
        for (int r = r0; r < r1; r++)
            if (A.granted[r]) got.tokens += A.new_tokens[r];
        Sums at = scan(got, &all, warps);
        for (int r = r0; r < r1; r++) {
            A.starts[r] = (int)at.tokens;
            if (A.granted[r]) at.tokens += A.new_tokens[r];
        }
        if (tid == 0) {
            A.starts[A.R] = (int)all.tokens;
            totals[0] = height;
            totals[1] = (int)all.take;
        }
    }
    cluster_sync();
    const int warps_all = ranks * (PLAN_THREADS / 32), lane = tid & 31;
    const int height = __ldcg(totals), stack = A.n_pages - 1;
    int returned = 0;
    for (int r = rank * (PLAN_THREADS / 32) + (tid >> 5); r < A.R; r += warps_all) {
        const int4 x = __ldcg(A.scratch + r);
        for (int j = x.x + lane; j < x.w; j += 32) {
            const int to = height - 1 - (x.y + j - x.x);
            if (to >= 0 && to < stack) A.free_pages[to] = A.table[(size_t)r * A.P + j];
        }
        returned |= x.w - x.x;
    }
    cluster_sync();
    for (int r = rank * (PLAN_THREADS / 32) + (tid >> 5); r < A.R; r += warps_all) {
        const int4 x = __ldcg(A.scratch + r);
        const int holds = __ldcg(A.held + r), behind = max(holds, x.w);
        for (int j = x.x + lane; j < behind; j += 32) {
            const int from = height - 1 - (x.z + j - x.x);
            A.table[(size_t)r * A.P + j] = j < holds && from >= 0 && from < stack ? __ldcg(A.free_pages + from) : 0;
        }
    }
    for (int i = tid; i <= A.R; i += PLAN_THREADS) starts_s[i] = __ldcg(A.starts + i);
    cluster_sync();
    if (rank == 0 && tid == 0) A.n_free[0] = height - totals[1];
    const int tokens = starts_s[A.R];
    for (int i = rank * PLAN_THREADS + tid; i < A.room; i += ranks * PLAN_THREADS) {
        int slot = -1, position = 0, r = -1;
        if (i < tokens) {
            int lo = 0, hi = A.R;                                     // the last request that starts at or before i and has tokens
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (starts_s[mid] <= i) lo = mid;
                else hi = mid;
            }
            r = lo;
            position = __ldg(A.lengths + r) + i - starts_s[r];
            slot = (__ldcg(A.table + (size_t)r * A.P + (position >> A.page_shift)) << A.page_shift) + (position & (page - 1));
        }
        A.slots[i] = slot;
        A.positions[i] = position;
        A.rows[i] = r;
    }
}

// ---- heads -------------------------------------------------------------------------------------------------------
// A CTA takes a token (or a part of its heads), a warp one head at a time: lane l holds V neighbouring dims from V l (V = 4; 2 of a head of 64),
// and of a head of 256 the four that lie 128 further, too; the angles of its dims stay in registers for all the heads.
// The partner of a dim in a half-split rotation is rot / 2 away: in another lane of the same piece, or (rot 256) in this one.
// Sums and rotation in 32 bits, operation by operation as the formula has them (a 4-bit code next to a border would fall the other way otherwise:
// one in a million does for each last bit), one rounding to the output's type; a 4-bit cache is cut from the 32-bit values.
// The sum of squares adds a dim and the one 128 further, then a lane's four, then lanes in pairs.  Bound by bytes at many tokens, by the
// chain load - reduce - store at few.
struct HeadsArgs {
    const void *q, *k, *v;
    void *q_out, *k_out;
    const int *positions, *slots;
    const float *q_norm, *k_norm, *cos, *sin;
    long long q_tok, q_head, k_tok, k_head, v_tok, v_head;
    void *ck, *cv;
    uint32_t *ks, *vs;                   // (scale, low) pairs of a 4-bit cache
    long long s_page, s_head, s_pos;
    int cache_type, page_shift, n_slots; // cache_type -1: none
    float eps, offset;
    int tokens, nq, nkv, f16, rot, pairs, max_position, interleaved, v_norm;
};

__device__ __forceinline__ float2 unpack(uint32_t w, __nv_bfloat16) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }
__device__ __forceinline__ float2 unpack(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
// V neighbouring elements, as they lie and as values.
template <class T, int V> struct Piece {
    static constexpr int WORDS = V * sizeof(T) / 4;
    uint32_t w[WORDS];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (WORDS == 4) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p);
        else if constexpr (WORDS == 2) *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
        else w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < WORDS; i++) w[i] = 0u;
    }
    __device__ __forceinline__ void values(float* x) const {
#pragma unroll
        for (int i = 0; i < WORDS; i++) {
            if constexpr (sizeof(T) == 4) x[i] = __uint_as_float(w[i]);
            else {
                const float2 v = unpack(w[i], T());
                x[2 * i] = v.x, x[2 * i + 1] = v.y;
            }
        }
    }
};
template <int V> __device__ __forceinline__ void load_piece(float* x, const float* p) {
    Piece<float, V> v;
    v.load(p);
    v.values(x);
}
template <int V> __device__ __forceinline__ void store_piece(uint16_t* p, const float* x, bool f16) {
    uint32_t w[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; i++) {
        if (f16) {
            const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    if constexpr (V == 4) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(w);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
}
__device__ __forceinline__ float nan_min(float a, float b) { return a != a || b != b ? __int_as_float(0x7FC00000) : fminf(a, b); }
__device__ __forceinline__ float nan_max(float a, float b) { return a != a || b != b ? __int_as_float(0x7FC00000) : fmaxf(a, b); }

// The lanes' V values each of one piece (32 V dims from group `g0`) -> codes and (scale, low), rows of G groups.  The low end is rounded down and
// the step up to bf16, so all values lie within [low, low + 15 steps] (to a last bit of the fifteenth) and are off by half a step at
// most.  A group with a value that is not finite reads back as NaN.
template <int V, int G>
__device__ __forceinline__ void store_codes(uint8_t* row, uint32_t* scales, const float* x, int g0, int lane) {
    constexpr int LANES = 64 / V;                                     // of a group
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int i = 1; i < V; i++) lo = nan_min(lo, x[i]), hi = nan_max(hi, x[i]);
#pragma unroll
    for (int d = 1; d < LANES; d *= 2) lo = nan_min(lo, __shfl_xor_sync(~0u, lo, d)), hi = nan_max(hi, __shfl_xor_sync(~0u, hi, d));
    const __nv_bfloat16 low = __float2bfloat16_rd(lo);
    const float base = __bfloat162float(low);
    const __nv_bfloat16 step = __float2bfloat16_ru(__fmul_rn(__fadd_rn(hi, -base), 1.f / 15.f));
    const float s = __bfloat162float(step), inv = __frcp_rn(s);
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
        // the quotient rounded as a division would round it, at the price of a product: only one that lies near a half can fall the other way
        const float a = __fadd_rn(x[i], -base), q = a * inv;
        float c = rintf(q);
        if (fabsf(q - c) > 0.49999f) c = rintf(__fdiv_rn(a, s));
        if (!(s > 0.f)) c = 0.f;
        word |= (uint32_t)(c >= 0.f ? fminf(c, 15.f) : 0.f) << (4 * i);      // (a NaN compares false)
    }
    constexpr int SHARE = 8 / V;                                      // lanes of a word
    word <<= 4 * V * (lane & (SHARE - 1));
#pragma unroll
    for (int d = 1; d < SHARE; d *= 2) word |= __shfl_xor_sync(~0u, word, d);
    const int at = lane / SHARE;                                      // the piece's words: eight of a group
    if ((lane & (SHARE - 1)) == 0) reinterpret_cast<uint32_t*>(row)[(at & 7) * G + g0 + at / 8] = word;
    if (lane % LANES == 0) scales[g0 + lane / LANES] = (uint32_t)__bfloat16_as_ushort(step) | ((uint32_t)__bfloat16_as_ushort(low) << 16);
}

template <class T, int N>
static __global__ void __launch_bounds__(256, 4) heads_kernel(const __grid_constant__ HeadsArgs A) {
    constexpr int D = 32 * N, V = N < 4 ? N : 4, PIECES = N / V;
    const int t = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto dim_of = [&](int i) { return i / V * 128 + lane * V + i % V; };
    const int total = A.nq + (A.cache_type >= 0 ? 2 : 1) * A.nkv, stride = 8 * gridDim.y;
    // (the first head's row does not depend on where the token goes: it is asked for first)
    Piece<T, V> next[PIECES];
    auto fetch = [&](int h) {
        const T* src = h < A.nq ? reinterpret_cast<const T*>(A.q) + (long long)t * A.q_tok + h * A.q_head
                                : (h < A.nq + A.nkv ? reinterpret_cast<const T*>(A.k) + (long long)t * A.k_tok + (h - A.nq) * A.k_head
                                                    : reinterpret_cast<const T*>(A.v) + (long long)t * A.v_tok + (h - A.nq - A.nkv) * A.v_head);
#pragma unroll
        for (int p = 0; p < PIECES; p++) next[p].load(src + dim_of(p * V));
    };
    int h = blockIdx.y * 8 + warp;
    if (h < total) fetch(h);
    const int pos = A.positions[t];
    bool live = A.cos ? pos >= 0 && pos < A.max_position : true;
    int slot = 0;
    if (A.cache_type >= 0) {
        slot = A.slots[t];
        live = live && slot >= 0 && slot < A.n_slots;
    }
    // the angles of this lane's dims: turned = x * c + partner * s; `from`: the partner's lane, `other`: its piece
    float c[N], s[N];
    uint32_t turns = 0;
    int from[PIECES];
    bool other[PIECES];
    const int half = A.rot / 2;
    // (a piece's angles are neighbours; the tables' rows allow whole loads where a row is whole pieces)
    const bool wide = A.pairs % V == 0 && !A.interleaved;
#pragma unroll
    for (int p = 0; p < PIECES; p++) {
        const int d0 = dim_of(p * V), first = A.interleaved ? d0 >> 1 : (d0 < half ? d0 : d0 - half);      // (half is a multiple of V)
#pragma unroll
        for (int i = 0; i < V; i++) c[p * V + i] = 1.f, s[p * V + i] = 0.f;
        if (A.cos && live && d0 < A.rot) {
            const size_t row = (size_t)pos * A.pairs;
            if (wide) {
                if (first < A.pairs) {
                    load_piece<V>(c + p * V, A.cos + row + first);
                    load_piece<V>(s + p * V, A.sin + row + first);
                    turns |= ((1u << V) - 1) << (p * V);
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const int pair = A.interleaved ? (d0 + i) >> 1 : first + i;
                    if (pair < A.pairs) c[p * V + i] = __ldg(A.cos + row + pair), s[p * V + i] = __ldg(A.sin + row + pair), turns |= 1u << (p * V + i);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < V; i++)
            if (A.interleaved ? !(i & 1) : d0 < half) s[p * V + i] = -s[p * V + i];
        const int partner = d0 >= A.rot ? d0 : (d0 < half ? d0 + half : d0 - half);
        from[p] = (partner & 127) / V;
        other[p] = partner / 128 != p;
    }
    const bool near = PIECES == 1 || half <= 64;                      // partners in the same piece
    for (; h < total; h += stride) {
        const int kind = h < A.nq ? 0 : (h < A.nq + A.nkv ? 1 : 2), head = kind == 0 ? h : (kind == 1 ? h - A.nq : h - A.nq - A.nkv);
        float x[N];
#pragma unroll
        for (int p = 0; p < PIECES; p++) {
            if (!live) next[p].zero();
            next[p].values(x + p * V);
        }
        if (h + stride < total) fetch(h + stride);                    // the next head is on its way while this one is turned
        const float* w = kind == 0 ? A.q_norm : (kind == 1 ? A.k_norm : nullptr);
        if (w || (kind == 2 && A.v_norm)) {
            float sq[V];
#pragma unroll
            for (int i = 0; i < V; i++) sq[i] = PIECES == 2 ? x[i] * x[i] + x[V + i] * x[V + i] : x[i] * x[i];
            float sum = sq[0];
#pragma unroll
            for (int i = 1; i < V; i++) sum += sq[i];
#pragma unroll
            for (int d = 1; d < 32; d *= 2) sum += __shfl_xor_sync(~0u, sum, d);
            const float r = live ? rsqrtf(sum * (1.f / D) + A.eps) : 0.f;
#pragma unroll
            for (int p = 0; p < PIECES; p++) {
                float wv[V];
                if (w) load_piece<V>(wv, w + dim_of(p * V));
#pragma unroll
                for (int i = 0; i < V; i++) x[p * V + i] = x[p * V + i] * r * (w ? A.offset + wv[i] : 1.f);
            }
        }
        if (kind < 2 && A.cos) {
            float z[N];                                               // the partners
            if (A.interleaved) {
#pragma unroll
                for (int i = 0; i < N; i++) z[i] = x[i ^ 1];
            } else if (PIECES == 2 && half == 128) {
#pragma unroll
                for (int i = 0; i < N; i++) z[i] = x[(i + V) % N];
            } else if (near) {
#pragma unroll
                for (int i = 0; i < V; i++) z[i] = __shfl_sync(~0u, x[i], from[0]);
#pragma unroll
                for (int i = V; i < N; i++) z[i] = 0.f;               // (these dims are not turned: near ends at the first piece)
            } else {
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const float a = __shfl_sync(~0u, x[i], from[i / V]), b = __shfl_sync(~0u, x[(i + V) % N], from[i / V]);
                    z[i] = other[i / V] ? b : a;
                }
            }
#pragma unroll
            for (int i = 0; i < N; i++) {
                const float y = x[i] * c[i] + z[i] * s[i];
                x[i] = turns >> i & 1 ? y : x[i];
            }
        }
        if (kind == 0 || A.cache_type < 0) {
            uint16_t* out = reinterpret_cast<uint16_t*>(kind == 0 ? A.q_out : A.k_out) + ((size_t)t * (kind == 0 ? A.nq : A.nkv) + head) * D;
#pragma unroll
            for (int p = 0; p < PIECES; p++) store_piece<V>(out + dim_of(p * V), x + p * V, A.f16);
        } else if (live) {
            const int at = slot >> A.page_shift, off = slot & ((1 << A.page_shift) - 1);
            if (A.cache_type == MKV_INT4) {
                const size_t row = (((size_t)at * A.nkv + head) << A.page_shift) + off;
#pragma unroll
                for (int p = 0; p < PIECES; p++)
                    store_codes<V, N / 2>(reinterpret_cast<uint8_t*>(kind == 1 ? A.ck : A.cv) + row * (D / 2), (kind == 1 ? A.ks : A.vs) + row * (D / 64), x + p * V, p * 2, lane);
            } else {
                uint16_t* out = reinterpret_cast<uint16_t*>(kind == 1 ? A.ck : A.cv) + (at * A.s_page + head * A.s_head + off * A.s_pos);
#pragma unroll
                for (int p = 0; p < PIECES; p++) store_piece<V>(out + dim_of(p * V), x + p * V, A.cache_type == MKV_F16);
            }
        }
    }
}

// ---- rows of the cache as values -----------------------------------------------------------------------------------
template <int N>
static __global__ void __launch_bounds__(256) rows_kernel(const __grid_constant__ HeadsArgs A) {
    constexpr int D = 32 * N;
    const int t = blockIdx.x, lane = threadIdx.x & 31, slot = A.slots[t];
    const bool live = slot >= 0 && slot < A.n_slots;
    const int at = live ? slot >> A.page_shift : 0, off = slot & ((1 << A.page_shift) - 1);
    for (int h = blockIdx.y * 8 + (threadIdx.x >> 5); h < 2 * A.nkv; h += 8 * gridDim.y) {
        const bool key = h < A.nkv;
        const int head = key ? h : h - A.nkv;
        void* out = key ? A.q_out : A.k_out;
        const size_t o = ((size_t)t * A.nkv + head) * D + lane * N;
        if (A.cache_type == MKV_INT4) {
            const size_t row = (((size_t)at * A.nkv + head) << A.page_shift) + off;
            const int word = lane * N / 8, g = word / 8, i = word & 7;
            const uint32_t w = live ? __ldg(reinterpret_cast<const uint32_t*>(key ? A.ck : A.cv) + row * (D / 8) + i * (N / 2) + g) >> (N < 8 ? 4 * N * (lane & (8 / N - 1)) : 0) : 0u;
            const uint32_t sl = live ? __ldg((key ? A.ks : A.vs) + row * (D / 64) + g) : 0u;
            float x[N];
#pragma unroll
            for (int j = 0; j < N; j++) x[j] = (float)((w >> (4 * j)) & 15u) * __uint_as_float(sl << 16) + __uint_as_float(sl & 0xFFFF0000u);
            float* p = reinterpret_cast<float*>(out) + o;
            if constexpr (N % 4 == 0) {
#pragma unroll
                for (int j = 0; j < N; j += 4) *reinterpret_cast<float4*>(p + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
            } else
                *reinterpret_cast<float2*>(p) = make_float2(x[0], x[1]);
        } else {
            const uint16_t* src = reinterpret_cast<const uint16_t*>(key ? A.ck : A.cv) + (at * A.s_page + head * A.s_head + off * A.s_pos) + lane * N;
            uint32_t w[N / 2];
#pragma unroll
            for (int j = 0; j < N / 2; j++) w[j] = live ? reinterpret_cast<const uint32_t*>(src)[j] : 0u;
            uint32_t* p = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(out) + o);
#pragma unroll
            for (int j = 0; j < N / 2; j++) p[j] = w[j];
        }
    }
}

// CTAs along y: enough that the warps of all tokens cover the machine once (8 per CTA, one head each at least).  Us with one, by this rule and with one warp per head,
// 24 / 4 heads of 256 into 4 bits: 8 tokens 8.4 6.4 6.4, 300 tokens 12.1 12.4 13.0, 1000 tokens 18.7 18.6 24.8, 4000 tokens 61.6 61.6 84.2
static int head_parts(int tokens, int heads) {
    const int most = (heads + 7) / 8, want = (148 * 4 + tokens - 1) / tokens;
    return want < 1 ? 1 : (want < most ? want : most);
}
static int log2_of(int n) { return 31 - __builtin_clz(n); }

static void set_cache(HeadsArgs& H, const mk_cache& c) {
    H.ck = reinterpret_cast<void*>(c.k);
    H.cv = reinterpret_cast<void*>(c.v);
    H.ks = reinterpret_cast<uint32_t*>(c.k_scales);
    H.vs = reinterpret_cast<uint32_t*>(c.v_scales);
    H.s_page = c.s_page, H.s_head = c.s_head, H.s_pos = c.s_pos;
    H.cache_type = c.type;
    H.page_shift = log2_of(c.page);
    H.n_slots = c.pages * c.page;
    H.nkv = c.kv_heads;
}

template <class T>
static int launch_heads(const HeadsArgs& H, int dim, dim3 grid, cudaStream_t st) {
    cudaError_t e = dim == 64 ? launch(heads_kernel<T, 2>, grid, 256, 0, 1, false, st, H)
                              : (dim == 128 ? launch(heads_kernel<T, 4>, grid, 256, 0, 1, false, st, H) : launch(heads_kernel<T, 8>, grid, 256, 0, 1, false, st, H));
    MKV_CUDA(e);
    return MK_OK;
}

}  // namespace mkv

using namespace mkv;

extern "C" int mk_page_plan(const mk_plan_args* a, void* stream) {
    if (!a) return vfail(MK_ERR_BADARG, "mk_page_plan: null argument");
    if (a->requests < 1 || a->requests > MKV_MAX_REQUESTS) return vfail(MK_ERR_BADARG, "mk_page_plan: %d requests (1 to %d)", a->requests, MKV_MAX_REQUESTS);
    if (a->page < 1 || (a->page & (a->page - 1))) return vfail(MK_ERR_BADARG, "mk_page_plan: %d tokens per page (a power of two)", a->page);
    if (a->max_pages < 1 || a->pages < 2 || (int64_t)a->pages * a->page > INT32_MAX || (int64_t)a->max_pages * a->page > INT32_MAX)
        return vfail(MK_ERR_BADARG, "mk_page_plan: %d pages, at most %d per request, of %d tokens", a->pages, a->max_pages, a->page);
    if (a->room < 1) return vfail(MK_ERR_BADARG, "mk_page_plan: room for %d tokens", a->room);
    const uint64_t all[] = {a->lengths, a->new_tokens, a->table, a->held, a->free_pages, a->n_free, a->scratch, a->slots, a->positions, a->rows, a->starts, a->context, a->granted};
    for (uint64_t p : all)
        if (!p || !aligned(p, 4)) return vfail(MK_ERR_BADARG, "mk_page_plan: a buffer is missing or misaligned");
    if (!aligned(a->scratch, 16)) return vfail(MK_ERR_BADARG, "mk_page_plan: scratch not 16-byte aligned");
    MKV_DEVICE(a->device);
    PlanArgs A;
    A.lengths = reinterpret_cast<const int*>(a->lengths);
    A.new_tokens = reinterpret_cast<const int*>(a->new_tokens);
    A.table = reinterpret_cast<int*>(a->table);
    A.held = reinterpret_cast<int*>(a->held);
    A.free_pages = reinterpret_cast<int*>(a->free_pages);
    A.n_free = reinterpret_cast<int*>(a->n_free);
    A.scratch = reinterpret_cast<int4*>(a->scratch);
    A.slots = reinterpret_cast<int*>(a->slots);
    A.positions = reinterpret_cast<int*>(a->positions);
    A.rows = reinterpret_cast<int*>(a->rows);
    A.starts = reinterpret_cast<int*>(a->starts);
    A.context = reinterpret_cast<int*>(a->context);
    A.granted = reinterpret_cast<int*>(a->granted);
    A.R = a->requests, A.P = a->max_pages, A.page_shift = log2_of(a->page), A.n_pages = a->pages, A.room = a->room;
    // one CTA needs no barriers between CTAs, eight fill tables and slots faster: us with 1 and 8, one token each of 8, 64, 256, 1000 requests 8.4 10.4, 10.4 10.5, 12.5 12.0,
    // 24.7 14.6; 64 of 200 tokens 19.4 12.5
    const int ranks = a->requests <= 64 && a->room <= 1024 ? 1 : 8;
    MKV_CUDA(launch(plan_pages, dim3(ranks), PLAN_THREADS, (size_t)(A.R + 1) * 4, ranks, false, static_cast<cudaStream_t>(stream), A));
    return MK_OK;
}

extern "C" int mk_heads(const mk_heads_args* a, void* stream) {
    if (!a) return vfail(MK_ERR_BADARG, "mk_heads: null argument");
    if (a->tokens < 0 || a->q_heads < 0 || a->kv_heads < 1) return vfail(MK_ERR_BADARG, "mk_heads: %d tokens, %d and %d heads", a->tokens, a->q_heads, a->kv_heads);
    const int D = a->head_dim, V = D < 128 ? 2 : 4;
    if (D != 64 && D != 128 && D != 256) return vfail(MK_ERR_UNSUPPORTED, "mk_heads: head dim %d (64, 128 or 256)", D);
    if (a->source < 0 || a->source > MKV_F32) return vfail(MK_ERR_BADARG, "mk_heads: source type %d", a->source);
    if (a->type != MKV_BF16 && a->type != MKV_F16) return vfail(MK_ERR_BADARG, "mk_heads: output type %d", a->type);
    const bool cached = a->cache.k != 0;
    if ((a->q_heads && (!a->q || !a->q_out)) || !a->k || !a->positions || (cached && (!a->v || !a->slots)) || (!cached && !a->k_out)) return vfail(MK_ERR_BADARG, "mk_heads: a buffer is missing");
    if (cached) {
        if (const char* why = bad_cache(a->cache)) return vfail(MK_ERR_BADARG, "mk_heads: %s", why);
        if (a->cache.head_dim != D || a->cache.kv_heads != a->kv_heads) return vfail(MK_ERR_BADARG, "mk_heads: cache of %d heads of %d", a->cache.kv_heads, a->cache.head_dim);
    }
    const int size = a->source == MKV_F32 ? 4 : 2, unit = V * size;
    if (!aligned(a->q, unit) || !aligned(a->k, unit) || (cached && !aligned(a->v, unit)) || !aligned(a->q_out, 16) || !aligned(a->k_out, 16))
        return vfail(MK_ERR_BADARG, "mk_heads: an address is not %d-byte aligned", unit);
    const int64_t strides[] = {a->q_tok, a->q_head, a->k_tok, a->k_head, cached ? a->v_tok : 0, cached ? a->v_head : 0};
    for (int64_t s : strides)
        if (s < 0 || (s * size) % unit) return vfail(MK_ERR_BADARG, "mk_heads: stride %lld breaks the %d-byte alignment of rows", (long long)s, unit);
    if (a->cos || a->sin) {
        if (!a->cos || !a->sin || a->max_position < 1) return vfail(MK_ERR_BADARG, "mk_heads: rotation tables");
        if (a->rot < 2 || a->rot > D || a->pairs < 1 || a->pairs > a->rot / 2) return vfail(MK_ERR_BADARG, "mk_heads: %d rotated dims, %d angles", a->rot, a->pairs);
        if (a->rot % (D / 16)) return vfail(MK_ERR_UNSUPPORTED, "mk_heads: %d rotated dims of %d (a multiple of %d)", a->rot, D, D / 16);
    }
    if (!aligned(a->q_norm, 16) || !aligned(a->k_norm, 16)) return vfail(MK_ERR_BADARG, "mk_heads: norm weights not 16-byte aligned");
    if (a->tokens == 0) return MK_OK;
    MKV_DEVICE(a->device);
    HeadsArgs H;
    memset(&H, 0, sizeof H);
    H.cache_type = -1;
    if (cached) set_cache(H, a->cache);
    H.q = reinterpret_cast<const void*>(a->q), H.k = reinterpret_cast<const void*>(a->k), H.v = reinterpret_cast<const void*>(a->v);
    H.q_out = reinterpret_cast<void*>(a->q_out), H.k_out = reinterpret_cast<void*>(a->k_out);
    H.positions = reinterpret_cast<const int*>(a->positions), H.slots = reinterpret_cast<const int*>(a->slots);
    H.q_norm = reinterpret_cast<const float*>(a->q_norm), H.k_norm = reinterpret_cast<const float*>(a->k_norm);
    H.cos = reinterpret_cast<const float*>(a->cos), H.sin = reinterpret_cast<const float*>(a->sin);
    H.q_tok = a->q_tok, H.q_head = a->q_head, H.k_tok = a->k_tok, H.k_head = a->k_head, H.v_tok = a->v_tok, H.v_head = a->v_head;
    H.eps = a->eps, H.offset = a->norm_offset;
    H.tokens = a->tokens, H.nq = a->q_heads, H.nkv = a->kv_heads, H.f16 = a->type == MKV_F16, H.rot = a->rot, H.pairs = a->pairs;
    H.max_position = a->max_position, H.interleaved = a->interleaved, H.v_norm = a->v_norm;
    const dim3 grid(a->tokens, head_parts(a->tokens, a->q_heads + (cached ? 2 : 1) * a->kv_heads));
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return a->source == MKV_F32 ? launch_heads<float>(H, D, grid, st) : (a->source == MKV_BF16 ? launch_heads<__nv_bfloat16>(H, D, grid, st) : launch_heads<__half>(H, D, grid, st));
}

extern "C" int mk_cache_rows(const mk_cache* cache, uint64_t slots, int tokens, uint64_t k_out, uint64_t v_out, int device, void* stream) {
    if (!cache || !slots || !k_out || !v_out || tokens < 0) return vfail(MK_ERR_BADARG, "mk_cache_rows: a buffer is missing");
    if (const char* why = bad_cache(*cache)) return vfail(MK_ERR_BADARG, "mk_cache_rows: %s", why);
    if (!aligned(k_out, 16) || !aligned(v_out, 16)) return vfail(MK_ERR_BADARG, "mk_cache_rows: outputs not 16-byte aligned");
    if (tokens == 0) return MK_OK;
    MKV_DEVICE(device);
    HeadsArgs H;
    memset(&H, 0, sizeof H);
    set_cache(H, *cache);
    H.slots = reinterpret_cast<const int*>(slots);
    H.q_out = reinterpret_cast<void*>(k_out), H.k_out = reinterpret_cast<void*>(v_out);
    const dim3 grid(tokens, head_parts(tokens, 2 * cache->kv_heads));
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int D = cache->head_dim;
    MKV_CUDA(D == 64 ? launch(rows_kernel<2>, grid, 256, 0, 1, false, st, H) : (D == 128 ? launch(rows_kernel<4>, grid, 256, 0, 1, false, st, H) : launch(rows_kernel<8>, grid, 256, 0, 1, false, st, H)));
    return MK_OK;
}
