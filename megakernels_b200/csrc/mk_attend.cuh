// What the two attention kernels share (mk_attend.cu: few queries per request, mk_attend_rows.cu: many).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mk_serve_host.h"

namespace mkv {

struct AttendArgs {
    const void* q;
    void* out;
    const uint8_t *k, *v;
    const uint8_t *ks, *vs;
    const int *table, *context, *starts;
    float* part;                          // [grid][2][header 4 | A_ROWS x (dim + 2)]
    int* status;
    long long q_tok, q_head, out_tok, out_head, table_stride;
    long long s_page, s_head, s_pos;      // in bytes (codes: of a codes row's page, head, position)
    long long spin_limit_ns;
    int R, T, nq, nkv, per, pages, page_shift, max_pages, window, sinks, q_f16;
    float scale_log2;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
template <int B> __device__ __forceinline__ void cp_small(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(B), "r"(live ? B : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <bool BF>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (BF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_bf(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float from16(uint16_t x, bool f16) {
    return f16 ? __half2float(__ushort_as_half(x)) : __uint_as_float((uint32_t)x << 16);
}
__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// Codes i and i + 4 of a word's low and high halves (nibbles at bits 4 i), as two halves.  1024 + c and 1024 + 16 c are halves as they
// stand; what is left is one subtraction, exact.
template <int I> __device__ __forceinline__ uint32_t codes(uint32_t w) {
    uint32_t r;
    if constexpr (I == 0 || I == 2) {
        const uint32_t x = ((I == 2 ? w >> 8 : w) & 0x000F000Fu) | 0x64006400u;
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(0x64006400u));
    } else {
        const uint32_t x = ((I == 3 ? w >> 8 : w) & 0x00F000F0u) | 0x64006400u;
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(0x2C002C00u), "r"(0xD400D400u));      // x / 16 - 64
    }
    return r;
}

enum { K_BF16, K_F16, K_INT4 };

// mk_attend_rows.cu
int launch_rows(const AttendArgs& A, int type, int head_dim, int sms, cudaStream_t st);

}  // namespace mkv
