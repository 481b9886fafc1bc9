// The next token: temperature, top-k, top-p and min-p from given uniform numbers (declarations and rule: include/mk_serve.h).
//
// A cluster owns a row.  Its CTAs keep a contiguous piece of the row each in shared memory as order-preserving 32-bit keys, so the logits
// are read from memory once; everything after that is passes over shared memory with one exchange between the CTAs each.
//
//   keep = a prefix of the candidates in the order (key falling, index rising).  A prefix is a key and, among the equals of that
//   key, how many of them (`need`), the lowest indexes first.  top-k wants the prefix of k candidates, top-p the shortest prefix whose weight reaches
//   p times that of the first prefix: both are one search for the place where a running sum (of ones, or of weights) over falling keys
//   reaches a target.  `search` narrows an interval of keys: 256 bins over it, counts and weights per bin summed over the cluster,
//   the bin that holds the place becomes the interval.  The first level's bins are equal steps of the value (logits crowd into few octaves, so
//   bins by leading bits would make all lanes add to the same few), later ones equal steps of the key (at most four of those).
//   A bin whose members all belong to the prefix ends the search.
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
struct Shared {
    Bins bins[2];
    u64 merged_w[S_BINS];
    uint32_t merged_n[S_BINS];
    u64 warp_w[S_WARPS];
    uint32_t warp_n[S_WARPS];
    // what every CTA of the cluster writes into every other one
    uint32_t key_of[S_RANKS], live_of[S_RANKS], ties_of[S_RANKS], kept_of[S_RANKS];
    u64 weight_of[S_RANKS];
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

constexpr uint32_t LOWEST = 0x00800000u;                   // the key of the lowest finite value
// Keys order as the values do; 0 is kept for what is masked (-inf, NaN).  -0 counts as 0.
__device__ __forceinline__ uint32_t key_of(float x) {
    if (!(x > -INFINITY)) return 0u;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key); }

// The weight of a key in steps of 2^-44.
__device__ __forceinline__ u64 weight(uint32_t key, uint32_t top, double inv_t) {
    if (key == top) return 1ull << 44;                      // also where the largest is infinite
    const double y = ((double)value_of(key) - (double)value_of(top)) * inv_t;
    return y < -31.5 ? 0ull : (u64)__double2ll_rn(exp(y) * 17592186044416.0);
}

struct Place {
    uint32_t key, need;                  // the prefix's last key, and how many of its equals belong to the prefix
};

struct Row {
    Shared* S;
    const uint32_t* keys;
    int n, rank, ranks, level;           // level: how many exchanges of bins so far (they alternate between two buffers)
    uint32_t top;
    double inv_t;
};

// One level: bins over keys in [lo, hi], summed over the cluster.  `by_value`: bins are equal steps of the value.
__device__ __forceinline__ int bin_of(uint32_t key, uint32_t hi, float hi_value, float per_value, uint32_t step, bool by_value) {
    if (by_value) return min(S_BINS - 1, (int)((hi_value - value_of(key)) * per_value));
    return (int)((hi - key) / step);
}

// The prefix at which the running sum of ones (weights == false) or weights reaches `target` > 0, over candidates with keys in [lo, hi] (and of
// `lo` only `lo_need`, if weighted); the sum over all of them is at least the target.
template <bool WEIGHTS>
__device__ Place search(Row& R, uint32_t lo, uint32_t hi, double target, uint32_t lo_need) {
    Shared& S = *R.S;
    const int tid = threadIdx.x;
    const uint32_t floor_key = lo;
    double left = target;                                    // what the candidates above the interval leave of it
    u64 above = 0;
    bool by_value = value_of(hi) < INFINITY;                 // the first level
    for (;;) {
        if (lo == hi) break;
        Bins& B = S.bins[R.level & 1];
        R.level++;
        // equal steps of the value reach down to a weight of exp(-32), the last bin holds the rest
        const float hi_value = value_of(hi), per_value = (float)(S_BINS / 32 * R.inv_t);
        const uint32_t step = (hi - lo) / S_BINS + 1;
        const bool value_bins = by_value && per_value < 1e30f;
        for (int i = tid; i < S_BINS; i += S_THREADS) B.count[i] = B.lo[i] = B.hi[i] = 0;
        __syncthreads();
        for (int e = tid; e < R.n; e += S_THREADS) {
            const uint32_t key = R.keys[e];
            if (key < lo || key > hi) continue;
            const int b = bin_of(key, hi, hi_value, per_value, step, value_bins);
            atomicAdd(&B.count[b], 1u);
            if (WEIGHTS) {
                const u64 w = weight(key, R.top, R.inv_t);
                const uint32_t w_lo = (uint32_t)w, old = atomicAdd(&B.lo[b], w_lo), w_hi = (uint32_t)(w >> 32) + (old + w_lo < old);
                if (w_hi) atomicAdd(&B.hi[b], w_hi);
            }
        }
        cluster_barrier();
        // every CTA adds up all of them (8 to 12 KB); the buffer is written again two levels on, behind the next barrier
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
            const uint32_t reached = __ballot_sync(~0u, (double)(above + upto) >= left);
            const int who = reached ? __ffs(reached) - 1 : 31;
            if (tid == who) {
                u64 run = above + upto - mine;
                int b = tid * 8;
                for (; b < tid * 8 + 7; b++) {
                    const u64 next = run + (WEIGHTS ? S.merged_w[b] : (u64)S.merged_n[b]);
                    if ((double)next >= left) break;
                    run = next;
                }
                S.bin = b;
                S.bin_n = S.merged_n[b];
                S.above = run;
            }
        }
        __syncthreads();
        const int b = (int)S.bin;
        above = S.above;
        const uint32_t members = S.bin_n;
        __syncthreads();
        // the bin's interval of keys
        if (value_bins) {
            // bin_of falls as the key rises: the smallest keys with a bin of b or less, and of b - 1 or less
            if (tid < 64) {
                const int want = tid < 32 ? b : b - 1, at = tid & 31;
                uint32_t l = lo, h = hi;                      // (hi itself is in bin 0; for b = 0 the second border is not used)
                while (l < h) {
                    const uint32_t part = (h - l) / 32 + 1, m = l + part * at;
                    const bool beyond = m >= h || m < l;
                    const uint32_t yes = __ballot_sync(~0u, beyond || bin_of(m, hi, hi_value, per_value, step, true) <= want);
                    const int j = yes ? __ffs(yes) - 1 : 32;
                    const uint32_t new_h = j < 32 && l + part * j < h && l + part * j >= l ? l + part * j : h;
                    l = j > 0 ? l + part * (j - 1) + 1 : l;
                    h = new_h;
                    if (l > h) l = h;
                }
                if (at == 0) S.border[tid >> 5] = l;
            }
            __syncthreads();
            lo = S.border[0];
            if (b > 0) hi = max(lo, S.border[1] - 1);
        } else {
            const uint32_t top = hi - (uint32_t)b * step, width = step - 1;
            lo = top - lo > width ? top - width : lo;
            hi = top;
        }
        by_value = false;
        if (members == 1 || (!WEIGHTS && (double)(above + members) == left)) return {lo, 0xFFFFFFFFu};   // all of them: no key is cut
    }
    // one key: how many of its equals
    if (!WEIGHTS) return {lo, (uint32_t)(left - (double)above)};
    const u64 w = weight(lo, R.top, R.inv_t);
    uint32_t n = 1;
    if (w) {
        n = (uint32_t)fmin(fmax(ceil((left - (double)above) / (double)w), 1.0), 4294967040.0);
        if (n > 1 && (double)(above + (u64)(n - 1) * w) >= left) n--;              // the division's rounding
        else if ((double)(above + (u64)n * w) < left) n++;
    }
    return {lo, lo == floor_key && n > lo_need ? lo_need : n};
}

__device__ __forceinline__ u64 warp_add(u64 v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
    return v;
}

static __global__ void __launch_bounds__(S_THREADS) sample_rows(const __grid_constant__ SampleArgs A) {
    extern __shared__ __align__(16) uint8_t smem[];
    Shared& S = *reinterpret_cast<Shared*>(smem);
    uint32_t* keys = reinterpret_cast<uint32_t*>(smem + sizeof(Shared));
    const int ranks = nctarank(), rank = ctarank(), row = blockIdx.x / ranks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int first = rank * A.piece, n = max(0, min(A.vocab - first, A.piece));
    // ---- the piece as keys, its largest and how many are not masked
    uint32_t best = 0, live = 0;
    {
        const long long base = (long long)row * A.stride + first;
        for (int e = tid; e < n; e += S_THREADS) {
            const float x = A.type == MKV_F32 ? __ldg(reinterpret_cast<const float*>(A.logits) + base + e)
                                              : (A.type == MKV_BF16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(A.logits)[base + e])
                                                                    : __half2float(reinterpret_cast<const __half*>(A.logits)[base + e]));
            const uint32_t key = key_of(x);
            keys[e] = key;
            best = max(best, key);
            live += key != 0;
        }
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
    Row R = {&S, keys, n, rank, ranks, 0, top, greedy ? 1.0 : 1.0 / (double)t};
    // ---- the prefix
    Place at = {LOWEST, 0xFFFFFFFFu};                         // all that is not masked
    if (k == 1) at = {top, 1u};
    else if (k > 1 && (uint32_t)k < total) at = search<false>(R, LOWEST, top, (double)k, 0u);
    // how many equals of the cut key every CTA holds, and the weight of the prefix
    auto ties = [&](uint32_t key, uint32_t* before) {
        uint32_t mine = 0;
        for (int e = tid; e < n; e += S_THREADS) mine += keys[e] == key;
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
        uint32_t all = 0;
        *before = 0;
        for (int r = 0; r < ranks; r++) {
            if (r < rank) *before += S.ties_of[r];
            all += S.ties_of[r];
        }
        return all;
    };
    if (p < 1.f && !(at.key == top && at.need == 1u)) {
        u64 mine = 0;
        for (int e = tid; e < n; e += S_THREADS)
            if (keys[e] > at.key || (keys[e] == at.key && at.need == 0xFFFFFFFFu)) mine += weight(keys[e], top, R.inv_t);
        mine = warp_add(mine);
        __syncthreads();
        if (lane == 0) S.warp_w[warp] = mine;
        __syncthreads();
        if (tid < ranks) {
            u64 l = 0;
            for (int w = 0; w < S_WARPS; w++) l += S.warp_w[w];
            remote_store(&S.weight_of[rank], tid, l);
        }
        cluster_barrier();
        u64 all = 0;
        for (int r = 0; r < ranks; r++) all += S.weight_of[r];
        if (at.need != 0xFFFFFFFFu) all += (u64)at.need * weight(at.key, top, R.inv_t);
        const double target = (double)p * (double)all;
        // the first candidate always stays
        at = target > 0 ? search<true>(R, at.key, top, target, at.need) : Place{top, 1u};
    }
    uint32_t before = 0;
    if (at.need != 0xFFFFFFFFu && ties(at.key, &before) <= at.need) at.need = 0xFFFFFFFFu;
    // ---- weights of the kept ones, in index order: a run of the piece per warp
    const int per_warp = ((n + S_WARPS - 1) / S_WARPS + 31) & ~31, w0 = min(n, warp * per_warp), w1 = min(n, w0 + per_warp);
    if (at.need != 0xFFFFFFFFu) {
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
        if (key == at.key && key != 0) stays = at.need == 0xFFFFFFFFu || seen + __popc(equal & ((1u << lane) - 1)) < at.need;
        seen += __popc(equal);
        u64 w = 0;
        if (stays) {
            w = weight(key, top, R.inv_t);
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
    // CTAs of a row: as many as keep a piece at 2048 logits or more
    int ranks = 1;
    while (ranks < S_RANKS && a->vocab > ranks * 2048) ranks *= 2;
    A.piece = ((a->vocab + ranks - 1) / ranks + 31) & ~31;
    const size_t smem = sizeof(Shared) + (size_t)A.piece * 4;
    MKV_CUDA(cudaFuncSetAttribute(sample_rows, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    MKV_CUDA(cudaFuncSetAttribute(sample_rows, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    MKV_CUDA(launch(sample_rows, dim3((unsigned)a->rows * ranks), S_THREADS, smem, ranks, false, static_cast<cudaStream_t>(stream), A));
    return MK_OK;
}
