// The next token: temperature, top-k, top-p and min-p from given uniform numbers (declarations and rule: include/mk_serve.h).
//
// A cluster owns a row.  Its CTAs keep a contiguous piece of the row each in shared memory as order-preserving 32-bit keys, so the logits
// are read from memory once; everything after that is passes over shared memory with one exchange between the CTAs each.
//
//   keep = a prefix of the candidates in the order (key falling, index rising).  A prefix is a key and, among the equals of that
// key, how many of them (`need`), the lowest indexes first.  top-k wants the prefix of k candidates, top-p the shortest prefix whose weight reaches
// p times that of the first prefix: both are one search for the place where a running sum (of ones, or of weights) over falling keys
// reaches a target.  `search` narrows an interval of keys.  First by a handful of cuts of the value, whose sums stay in registers: they leave a few hundred
// candidates of most rows, where adding all of them to bins in shared memory would cost more than the rest of the call.  Then by 256 bins over what is left, counts
// and weights summed over the cluster, the bin that holds the place becoming the interval: equal steps of the value first (by leading bits
// all lanes would add to the same few), then of the key.
// An interval whose members all belong to the prefix ends the search.
//
// Weights are exp in 64 bits, counted in steps of 2^-44: integer sums, the same in any order, so a border falls the same way whatever the
// split.  (32-bit weights would move a border of a flat row of 250000 candidates once in some hundred rows.)
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mk_serve_host.h"

namespace mkv {

constexpr int S_THREADS = 512, S_WARPS = S_THREADS / 32, S_BINS = 256, S_RANKS = 16;
typedef unsigned long long u64;

struct SampleArgs {
    const void* logits;
    const float *u, *temperature, *top_p, *min_p;
    const int* top_k;
    int *ids, *kept;
    float* logprobs;
    long long stride;
    int rows, vocab, type, piece;        // piece: logits per CTA (a multiple of 32)
};

struct Bins {
    uint32_t count[S_BINS], lo[S_BINS], hi[S_BINS];        // weights as two words
};
constexpr int S_CUTS = 5;                // intervals of one round of cuts
struct alignas(16) Shared {              // (the keys behind it are written sixteen bytes at a time)
    double powers[32];                   // 2^(i / 32)
    Bins bins[2];
    u64 merged_w[S_BINS];
    uint32_t merged_n[S_BINS];
    u64 warp_w[S_WARPS];
    uint32_t warp_n[S_WARPS];
    u64 cut_w[S_WARPS][S_CUTS];
    uint32_t cut_n[S_WARPS][S_CUTS];
    // what every CTA of the cluster writes into every other one
    uint32_t key_of[S_RANKS], live_of[S_RANKS], ties_of[S_RANKS], kept_of[S_RANKS];
    u64 weight_of[S_RANKS], cut_w_of[2][S_CUTS][S_RANKS];
    uint32_t cut_n_of[2][S_CUTS][S_RANKS];
    u64 above;
    uint32_t bin, bin_n, border[2];
};

__device__ __forceinline__ uint32_t ctarank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t nctarank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release;\n barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t remote(const void* p, int rank) {
    uint32_t a = (uint32_t)__cvta_generic_to_shared(p), r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    return r;
}
__device__ __forceinline__ uint32_t remote_load(const uint32_t* p, int rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(remote(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ void remote_store(uint32_t* p, int rank, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote(p, rank)), "r"(v) : "memory");
}
__device__ __forceinline__ void remote_store(u64* p, int rank, u64 v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote(p, rank)), "l"(v) : "memory");
}

__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
constexpr uint32_t LOWEST = 0x00800000u;                   // the key of the lowest finite value
// Keys order as the values do; 0 is kept for what is masked (-inf, NaN).  -0 counts as 0.
__device__ __forceinline__ uint32_t key_of(float x) {
    if (!(x > -INFINITY)) return 0u;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key); }

// The weight of a key in steps of 2^-44: exp by a table of 2^(i / 32) and a polynomial of degree 5 on |r| <= ln 2 / 64 (the table-driven method of Tang, 1989; the
// terms left out are below 2^-48), rounded to a whole number by an addition of 2^52.
__device__ __forceinline__ u64 weight(uint32_t key, uint32_t top, double inv_t, const double* powers) {
    if (key == top) return 1ull << 44;                      // also where the largest is infinite
    const double y = ((double)value_of(key) - (double)value_of(top)) * inv_t;
    if (!(y >= -31.5)) return 0ull;
    const double magic = 6755399441055744.0, t = fma(y, 46.16624130844683, magic);     // 32 / ln 2; 1.5 * 2^52
    const int n = __double2loint(t);
    const double k = t - magic;
    double r = fma(k, -0.021660849392446835, y);            // ln 2 / 32 to 38 bits (k has 11: exact), and the rest of it
    r = fma(k, -5.1456092446553379e-14, r);
    double e = fma(r, 1.0 / 120, 1.0 / 24);
    e = fma(e, r, 1.0 / 6);
    e = fma(e, r, 0.5);
    e = fma(e, r, 1.0);
    e = fma(e, r, 1.0) * powers[n & 31];
    e = __hiloint2double(__double2hiint(e) + (((n >> 5) + 44) << 20), __double2loint(e));
    return (u64)(__double_as_longlong(e + 4503599627370496.0) & 0xFFFFFFFFFFFFFll);
}

static_assert(sizeof(Shared) % 16 == 0, "keys behind it");

struct Place {
    uint32_t key, need;                  // the prefix's last key, and how many of its equals belong to the prefix
    uint32_t equals;                     // how many there are, where `need` is not all of them
};
constexpr uint32_t ALL = 0xFFFFFFFFu;

struct Row {
    Shared* S;
    const uint32_t* keys;
    int n, rank, ranks, level, cuts;     // level, cuts: how many exchanges of bins and of cuts so far (they alternate between two buffers)
    uint32_t top;
    double inv_t;
};

__device__ __forceinline__ u64 warp_add(u64 v) {
    // (pieces of 24 bits, so that 32 of them fit a word)
    const uint32_t a = __reduce_add_sync(~0u, (uint32_t)v & 0xFFFFFFu), b = __reduce_add_sync(~0u, (uint32_t)(v >> 24) & 0xFFFFFFu), c = __reduce_add_sync(~0u, (uint32_t)(v >> 48));
    return (u64)a + ((u64)b << 24) + ((u64)c << 48);
}

// The bin of a key of the interval that ends with `hi`: equal steps of the value or of the key.  (The last one of values takes what rounding leaves over.)
__device__ __forceinline__ int bin_of(uint32_t key, uint32_t hi, float hi_value, float per_value, uint32_t step, bool by_value) {
    if (by_value) return min(S_BINS - 1, (int)((hi_value - value_of(key)) * per_value));
    return (int)((hi - key) / step);
}

// The prefix at which the running sum of ones (weights == false) reaches `share` > 0, or the running sum of weights `share` times that of
// the candidates down to `within` (of its equals only `within.need`).  The sum over all candidates is at least the target.
template <bool WEIGHTS>
__device__ Place search(Row& R, Place within, double share) {
    Shared& S = *R.S;
    const int tid = threadIdx.x, lane = tid & 31;
    uint32_t lo = within.key, hi = R.top;
    double target = share;                                   // in ones, or in steps of 2^-44
    u64 above = 0;                                           // the sum above the interval
    const u64 floor_w = WEIGHTS ? weight(within.key, R.top, R.inv_t, S.powers) : 0ull, excess = within.need == ALL ? 0ull : (u64)(within.equals - within.need);
    uint32_t members = 0;
    {
        // ---- the cuts: 1, 3, 6 and 12 temperatures below the largest
        const double t = 1.0 / R.inv_t, top = (double)value_of(hi);
        uint32_t cut[S_CUTS];
#pragma unroll
        for (int j = 0; j < S_CUTS - 1; j++) {
            const double below[S_CUTS - 1] = {1, 3, 6, 12};
            cut[j] = min(max(lo, key_of((float)(top - t * below[j]))), hi);              // (an infinite largest: its own key)
        }
        cut[S_CUTS - 1] = lo;
        u64 w[S_CUTS] = {};
        uint32_t n[S_CUTS] = {};
        for (int e = tid; e < R.n; e += S_THREADS) {
            const uint32_t key = R.keys[e];
            if (key < lo) continue;
            const u64 x = WEIGHTS ? weight(key, R.top, R.inv_t, S.powers) : 0ull;
#pragma unroll
            for (int j = 0; j < S_CUTS; j++)                 // running: down to every cut
                if (key >= cut[j]) n[j]++, w[j] += x;
        }
#pragma unroll
        for (int j = 0; j < S_CUTS; j++) {
            const uint32_t a = __reduce_add_sync(~0u, n[j]);
            const u64 b = WEIGHTS ? warp_add(w[j]) : 0ull;
            if (lane == 0) S.cut_n[tid >> 5][j] = a, S.cut_w[tid >> 5][j] = b;
        }
        __syncthreads();
        const int buffer = R.cuts++ & 1;
        if (tid < S_CUTS * R.ranks) {
            const int j = tid / R.ranks, to = tid - j * R.ranks;
            uint32_t a = 0;
            u64 b = 0;
            for (int x = 0; x < S_WARPS; x++) a += S.cut_n[x][j], b += S.cut_w[x][j];
            remote_store(&S.cut_n_of[buffer][j][R.rank], to, a);
            if (WEIGHTS) remote_store(&S.cut_w_of[buffer][j][R.rank], to, b);
        }
        cluster_barrier();
        u64 sum_w[S_CUTS];
        uint32_t sum_n[S_CUTS];
#pragma unroll
        for (int j = 0; j < S_CUTS; j++) {
            sum_w[j] = 0, sum_n[j] = 0;
            for (int r = 0; r < R.ranks; r++) {
                sum_n[j] += S.cut_n_of[buffer][j][r];
                if (WEIGHTS) sum_w[j] += S.cut_w_of[buffer][j][r];
            }
        }
        if (WEIGHTS) {
            target = share * (double)(sum_w[S_CUTS - 1] - excess * floor_w);
            if (!(target > 0)) return {R.top, 1u, 0u};       // the first candidate always stays
        }
        bool found = false;
#pragma unroll
        for (int j = 0; j < S_CUTS; j++) {
            if (found || cut[j] > hi) continue;
            const u64 upto = WEIGHTS ? sum_w[j] : (u64)sum_n[j];
            if ((double)upto >= target || cut[j] == lo) {
                members = sum_n[j] - (j ? sum_n[j - 1] : 0u);
                if (!WEIGHTS && (double)upto == target) return {cut[j], ALL, 0u};
                lo = cut[j], found = true;
            } else {
                above = upto;
                hi = cut[j] - 1;                             // (above lo, which the last cut is)
            }
        }
        if (members == 1) return {lo, ALL, 0u};
    }
    while (lo < hi) {
        Bins& B = S.bins[R.level & 1];
        R.level++;
        // equal steps of the value where the interval is one of ordinary values and many keys, else of the key
        const float hi_value = value_of(hi), width = hi_value - value_of(lo), per_value = (float)S_BINS / width;
        const bool by_value = (double)width * R.inv_t < 64 && hi - lo > 1u << 16 && per_value < 1e30f;
        const uint32_t step = (hi - lo) / S_BINS + 1;
        for (int i = tid; i < S_BINS; i += S_THREADS) B.count[i] = B.lo[i] = B.hi[i] = 0;
        __syncthreads();
        for (int e = tid; e < R.n; e += S_THREADS) {
            const uint32_t key = R.keys[e];
            if (key < lo || key > hi) continue;
            const int b = bin_of(key, hi, hi_value, per_value, step, by_value);
            atomicAdd(&B.count[b], 1u);
            if (WEIGHTS) {
                const u64 w = weight(key, R.top, R.inv_t, S.powers);
                const uint32_t w_lo = (uint32_t)w, old = atomicAdd(&B.lo[b], w_lo), w_hi = (uint32_t)(w >> 32) + (old + w_lo < old);
                if (w_hi) atomicAdd(&B.hi[b], w_hi);
            }
        }
        cluster_barrier();
        // every CTA adds up all of them (1 to 3 KB each); the buffer is written again two levels on, behind the next barrier
        for (int b = tid; b < S_BINS; b += S_THREADS) {
            uint32_t n = 0;
            u64 w = 0;
            for (int r = 0; r < R.ranks; r++) {
                n += remote_load(&B.count[b], r);
                if (WEIGHTS) w += (u64)remote_load(&B.lo[b], r) + ((u64)remote_load(&B.hi[b], r) << 32);
            }
            S.merged_n[b] = n;
            S.merged_w[b] = w;
        }
        __syncthreads();
        if (tid < 32) {
            // the bin in which the running sum reaches the target: eight bins per lane
            u64 mine = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) mine += WEIGHTS ? S.merged_w[tid * 8 + j] : (u64)S.merged_n[tid * 8 + j];
            u64 upto = mine;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const u64 v = __shfl_up_sync(~0u, upto, d);
                if (tid >= d) upto += v;
            }
            const uint32_t reached = __ballot_sync(~0u, (double)(above + upto) >= target);
            const int who = reached ? __ffs(reached) - 1 : 31;
            if (tid == who) {
                u64 run = above + upto - mine;
                int b = tid * 8;
                for (; b < tid * 8 + 7; b++) {
                    const u64 next = run + (WEIGHTS ? S.merged_w[b] : (u64)S.merged_n[b]);
                    if ((double)next >= target) break;
                    run = next;
                }
                S.bin = b;
                S.bin_n = S.merged_n[b];
                S.above = run;
            }
        }
        __syncthreads();
        const uint32_t b = S.bin;
        above = S.above;
        members = S.bin_n;
        __syncthreads();
        if (by_value) {
            // bin_of falls as the key rises: the smallest keys with a bin of b or less, and of b - 1 or less, by 32-fold division
            if (tid < 64) {
                const int want = (int)b - (tid >> 5);
                uint32_t l = lo, h = hi;                      // (hi itself is in bin 0; for b = 0 the second border is not used)
                while (l < h) {
                    const uint32_t part = (h - l) / 32 + 1, m = l + part * lane;
                    const uint32_t yes = __ballot_sync(~0u, m >= h || m < l || bin_of(m, hi, hi_value, per_value, step, true) <= want);
                    const int j = yes ? __ffs(yes) - 1 : 32;
                    const uint32_t at = l + part * j;
                    if (j < 32 && at < h && at >= l) h = at;
                    if (j > 0) l = min(h, l + part * (j - 1) + 1);
                }
                if (lane == 0) S.border[tid >> 5] = l;
            }
            __syncthreads();
            lo = S.border[0];
            if (b > 0) hi = max(lo, S.border[1] - 1);
        } else {
            const uint32_t top = hi - b * step;
            lo = top - lo >= step ? top - step + 1 : lo;
            hi = top;
        }
        if (members == 1 || (!WEIGHTS && (double)(above + members) == target)) return {lo, ALL, 0u};     // all of them: no key is cut
    }
    // one key: how many of its equals
    uint32_t n = 1;
    if (!WEIGHTS) n = (uint32_t)(target - (double)above);
    else {
        const u64 w = weight(lo, R.top, R.inv_t, S.powers);
        if (w) {
            n = (uint32_t)fmin(fmax(ceil((target - (double)above) / (double)w), 1.0), 4294967040.0);
            if (n > 1 && (double)(above + (u64)(n - 1) * w) >= target) n--;                // the division's rounding
            else if ((double)(above + (u64)n * w) < target) n++;
        }
        if (lo == within.key && within.need != ALL) n = min(n, within.need);
    }
    return {lo, n >= members ? ALL : n, members};
}

static __global__ void __launch_bounds__(S_THREADS, 2) sample_rows(const __grid_constant__ SampleArgs A) {
    extern __shared__ __align__(16) uint8_t smem[];
    Shared& S = *reinterpret_cast<Shared*>(smem);
    uint32_t* keys = reinterpret_cast<uint32_t*>(smem + sizeof(Shared));
    const int ranks = nctarank(), rank = ctarank(), row = blockIdx.x / ranks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int first = rank * A.piece, n = max(0, min(A.vocab - first, A.piece));
    if (tid < 32) S.powers[tid] = exp2((double)tid * (1.0 / 32));
    // ---- the piece as keys, its largest and how many are not masked
    uint32_t best = 0, live = 0;
    {
        const long long base = (long long)row * A.stride + first;
        auto take = [&](float x) {
            const uint32_t key = key_of(x);
            best = max(best, key);
            live += key != 0;
            return key;
        };
        auto read = [&](auto zero) {
            typedef decltype(zero) T;
            constexpr int V = 16 / sizeof(T);
            const T* src = reinterpret_cast<const T*>(A.logits) + base;
            auto value = [](T x) {
                if constexpr (sizeof(T) == 4) return (float)x;
                else return to_float(x);
            };
            const int wide = ((uintptr_t)src & 15) == 0 ? n / V : 0;      // rows that do not start on a 16-byte boundary are read one by one
#pragma unroll 4
            for (int e = tid; e < wide; e += S_THREADS) {
                const uint4 raw = __ldg(reinterpret_cast<const uint4*>(src) + e);
                alignas(16) T x[V];
                *reinterpret_cast<uint4*>(x) = raw;
                uint32_t k[V];
#pragma unroll
                for (int i = 0; i < V; i++) k[i] = take(value(x[i]));
#pragma unroll
                for (int i = 0; i < V; i += 4) *reinterpret_cast<uint4*>(keys + e * V + i) = make_uint4(k[i], k[i + 1], k[i + 2], k[i + 3]);
            }
#pragma unroll 4
            for (int e = wide * V + tid; e < n; e += S_THREADS) keys[e] = take(value(src[e]));
        };
        if (A.type == MKV_F32) read(0.f);
        else if (A.type == MKV_BF16) read(__nv_bfloat16());
        else read(__half());
    }
    best = __reduce_max_sync(~0u, best);
    live = __reduce_add_sync(~0u, live);
    if (lane == 0) S.warp_n[warp] = live, S.warp_w[warp] = best;
    cluster_barrier();                                        // (and every CTA of the cluster is there to be written to)
    if (tid < ranks) {
        uint32_t b = 0, l = 0;
        for (int w = 0; w < S_WARPS; w++) b = max(b, (uint32_t)S.warp_w[w]), l += S.warp_n[w];
        remote_store(&S.key_of[rank], tid, b);
        remote_store(&S.live_of[rank], tid, l);
    }
    cluster_barrier();
    uint32_t top = 0, total = 0;
    for (int r = 0; r < ranks; r++) top = max(top, S.key_of[r]), total += S.live_of[r];
    if (total == 0) {
        if (rank == 0 && tid == 0) A.ids[row] = -1, A.logprobs[row] = -INFINITY, A.kept[row] = 0;
        return;                                               // (the whole cluster: nobody reads this CTA any more)
    }
    const float t = A.temperature[row], p = A.top_p[row], asked = A.min_p[row], m = asked > 0.f ? fminf(asked, 1.f) : 0.f;
    int k = A.top_k[row];
    const bool greedy = !(t > 0.f);
    if (greedy) k = 1;
    Row R = {&S, keys, n, rank, ranks, 0, 0, top, greedy ? 1.0 : 1.0 / (double)t};
    // ---- the prefix
    Place at = {LOWEST, ALL, 0u};                             // all that is not masked
    const bool one = k == 1;
    if (one) at = {top, 1u, 0u};
    else if (k > 1 && (uint32_t)k < total) at = search<false>(R, at, (double)k);
    if (p < 1.f && !one) at = search<true>(R, at, (double)p);
    // of the equals of the cut key, the lowest indexes: how many lie in the CTAs in front
    uint32_t before = 0;
    if (at.need != ALL) {
        uint32_t mine = 0;
        for (int e = tid; e < n; e += S_THREADS) mine += keys[e] == at.key;
        mine = __reduce_add_sync(~0u, mine);
        __syncthreads();
        if (lane == 0) S.warp_n[warp] = mine;
        __syncthreads();
        if (tid < ranks) {
            uint32_t l = 0;
            for (int w = 0; w < S_WARPS; w++) l += S.warp_n[w];
            remote_store(&S.ties_of[rank], tid, l);
        }
        cluster_barrier();
        for (int r = 0; r < rank; r++) before += S.ties_of[r];
    }
    // ---- weights of the kept ones, in index order: a run of the piece per warp
    const int per_warp = ((n + S_WARPS - 1) / S_WARPS + 31) & ~31, w0 = min(n, warp * per_warp), w1 = min(n, w0 + per_warp);
    if (at.need != ALL) {
        uint32_t mine = 0;
        for (int e = w0 + lane; e < w1; e += 32) mine += keys[e] == at.key;
        mine = __reduce_add_sync(~0u, mine);
        __syncthreads();
        if (lane == 0) S.warp_n[warp] = mine;
        __syncthreads();
        for (int w = 0; w < warp; w++) before += S.warp_n[w];
    }
    const double floor_w = (double)m * 17592186044416.0;
    // the weight of entry e, or 0 where it is not kept; `seen`: equals of the cut key in front of this step
    auto kept_weight = [&](int e, uint32_t& seen, bool& stays) {
        const uint32_t key = e < w1 ? keys[e] : 0u;
        stays = key > at.key;
        const uint32_t equal = __ballot_sync(~0u, key == at.key && key != 0);
        if (key == at.key && key != 0) stays = at.need == ALL || seen + __popc(equal & ((1u << lane) - 1)) < at.need;
        seen += __popc(equal);
        u64 w = 0;
        if (stays) {
            w = weight(key, top, R.inv_t, S.powers);
            stays = (double)w >= floor_w;
        }
        return stays ? w : 0ull;
    };
    u64 sum = 0;
    uint32_t count = 0, seen = before;
    for (int e0 = w0; e0 < w1; e0 += 32) {
        bool stays;
        sum += kept_weight(e0 + lane, seen, stays);
        count += stays;
    }
    sum = warp_add(sum);
    count = __reduce_add_sync(~0u, count);
    __syncthreads();
    if (lane == 0) S.warp_w[warp] = sum, S.warp_n[warp] = count;
    __syncthreads();
    if (tid < ranks) {
        u64 s = 0;
        uint32_t c = 0;
        for (int w = 0; w < S_WARPS; w++) s += S.warp_w[w], c += S.warp_n[w];
        remote_store(&S.weight_of[rank], tid, s);
        remote_store(&S.kept_of[rank], tid, c);
    }
    cluster_barrier();
    u64 all = 0, front = 0;
    uint32_t kept = 0;
    for (int r = 0; r < ranks; r++) {
        if (r < rank) front += S.weight_of[r];
        all += S.weight_of[r];
        kept += S.kept_of[r];
    }
    // ---- the first entry at which the running sum exceeds u times the whole (u below 1, so there is one)
    const double target = (double)fminf(fmaxf(A.u[row], 0.f), 0.99999994f) * (double)all;
    for (int w = 0; w < warp; w++) front += S.warp_w[w];
    const u64 own = S.warp_w[warp];
    if (own && (double)front <= target && (double)(front + own) > target) {
        seen = before;
        for (int e0 = w0; e0 < w1; e0 += 32) {
            bool stays;
            const u64 w = kept_weight(e0 + lane, seen, stays);
            u64 upto = w;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const u64 v = __shfl_up_sync(~0u, upto, d);
                if (lane >= d) upto += v;
            }
            const uint32_t passed = __ballot_sync(~0u, (double)(front + upto) > target && w > 0);
            if (passed) {
                if (lane == __ffs(passed) - 1) {
                    A.ids[row] = first + e0 + lane;
                    // the share from the weight itself: its steps are too coarse for a logarithm of a small one
                    const uint32_t key = keys[e0 + lane];
                    const double y = key == top ? 0.0 : ((double)value_of(key) - (double)value_of(top)) * R.inv_t;
                    A.logprobs[row] = (float)(y - log((double)all * (1.0 / 17592186044416.0)));
                    A.kept[row] = (int)kept;
                }
                break;
            }
            front += __shfl_sync(~0u, upto, 31);
        }
    }
}

}  // namespace mkv

using namespace mkv;

extern "C" int mk_sample(const mk_sample_args* a, void* stream) {
    if (!a) return vfail(MK_ERR_BADARG, "mk_sample: null argument");
    if (a->rows < 0 || a->vocab < 1 || a->vocab > MKV_MAX_VOCAB) return vfail(MK_ERR_BADARG, "mk_sample: %d rows of %d logits (at most %d)", a->rows, a->vocab, MKV_MAX_VOCAB);
    if (a->type < 0 || a->type > MKV_F32) return vfail(MK_ERR_BADARG, "mk_sample: logits of type %d", a->type);
    if (a->stride < 0) return vfail(MK_ERR_BADARG, "mk_sample: stride %lld", (long long)a->stride);
    const uint64_t all[] = {a->logits, a->u, a->temperature, a->top_k, a->top_p, a->min_p, a->ids, a->logprobs, a->kept};
    for (uint64_t p : all)
        if (!p || (p & (p == a->logits && a->type != MKV_F32 ? 1 : 3))) return vfail(MK_ERR_BADARG, "mk_sample: a buffer is missing or misaligned");
    if (a->rows == 0) return MK_OK;
    MKV_DEVICE(a->device);
    SampleArgs A;
    A.logits = reinterpret_cast<const void*>(a->logits);
    A.u = reinterpret_cast<const float*>(a->u), A.temperature = reinterpret_cast<const float*>(a->temperature);
    A.top_p = reinterpret_cast<const float*>(a->top_p), A.min_p = reinterpret_cast<const float*>(a->min_p);
    A.top_k = reinterpret_cast<const int*>(a->top_k);
    A.ids = reinterpret_cast<int*>(a->ids), A.kept = reinterpret_cast<int*>(a->kept), A.logprobs = reinterpret_cast<float*>(a->logprobs);
    A.stride = a->stride, A.rows = a->rows, A.vocab = a->vocab, A.type = a->type;
    // CTAs of a row: more of them shorten its passes, but clusters wait for room (one of 16 takes a whole GPC's SMs), so all rows together take about
    // 256 CTAs, and more only where a piece would be longer than 20000 logits.  Greedy, us: 64 rows of 30000 with 2, 4, 8, 16 CTAs each 18, 15, 20, 39;
    // of 151936 with 4, 8, 16 64, 41, 55; of 248320 with 8, 16 87, 73; one row of 151936 with 4, 8, 16 24, 17, 12.
    int ranks = 1;
    while (ranks < S_RANKS && a->vocab > ranks * 2048 && ((int64_t)a->rows * ranks * 2 <= 256 || a->vocab > ranks * 20000)) ranks *= 2;
    A.piece = ((a->vocab + ranks - 1) / ranks + 31) & ~31;
    const size_t smem = sizeof(Shared) + (size_t)A.piece * 4;
    MKV_CUDA(cudaFuncSetAttribute(sample_rows, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    MKV_CUDA(cudaFuncSetAttribute(sample_rows, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    MKV_CUDA(launch(sample_rows, dim3((unsigned)a->rows * ranks), S_THREADS, smem, ranks, false, static_cast<cudaStream_t>(stream), A));
    return MK_OK;
}
