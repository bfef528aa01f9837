// Bounded loads of a matrix's rows: a buffer descriptor over the rows a step may
// read, moved along with the step in scalar registers, and per-thread byte
// offsets that stay the same from step to step.  Loads past the last row's end
// return zeros, so a step needs no branch around its loads and no 64-bit
// address arithmetic in vector registers.
#pragma once
#include "common.h"

typedef unsigned pt_uintx2 __attribute__((ext_vector_type(2)));
typedef unsigned pt_uintx4 __attribute__((ext_vector_type(4)));

constexpr int PT_NOWHERE = 0x7ffffff0;   // a byte offset past any descriptor's end

struct RowBuf {
    const char* base;
    int ld;        // bytes between rows
    int width;     // bytes read of a row, at most ld
    // rows [r, r1), at most `span` of them, from offset 0 (span * ld < 2^31)
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t rows(int r, int r1, int span) const {
        const int n = min(max(r1 - r, 0), span);
        return __builtin_amdgcn_make_buffer_rsrc((void*)(base + (long)r * ld), 0, max((n - 1) * ld + width, 0),
                                                 0x00020000);
    }
};
__device__ __forceinline__ pt_uintx4 ld_buf16(__amdgpu_buffer_rsrc_t rs, int off) {
    return __builtin_bit_cast(pt_uintx4, __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0));
}
__device__ __forceinline__ pt_uintx2 ld_buf8(__amdgpu_buffer_rsrc_t rs, int off) {
    return __builtin_bit_cast(pt_uintx2, __builtin_amdgcn_raw_buffer_load_b64(rs, off, 0, 0));
}
__device__ __forceinline__ unsigned ld_buf4(__amdgpu_buffer_rsrc_t rs, int off) {
    return __builtin_amdgcn_raw_buffer_load_b32(rs, off, 0, 0);
}
__device__ __forceinline__ unsigned ld_buf2(__amdgpu_buffer_rsrc_t rs, int off) {
    return (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(rs, off, 0, 0);
}
__device__ __forceinline__ unsigned ld_buf1(__amdgpu_buffer_rsrc_t rs, int off) {
    return (unsigned char)__builtin_amdgcn_raw_buffer_load_b8(rs, off, 0, 0);
}
