// Tile helpers shared by the attention kernels (attention.hip, attention_ext.hip): LDS images of [rows][HDT] bf16 and the
// MFMA 32x32x16 fragments read from them.
#pragma once
#include "common.h"

namespace pdt {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

typedef bf16x4 __attribute__((address_space(3))) * lds_bf16x4_ptr;

// accumulator tile regs [8*blk, 8*blk+8) -> bf16 A operand
__device__ __forceinline__ bf16x8 acc_to_a(const f32x16& t, int blk) {
    bf16x8 a;
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = (bf16)t[8 * blk + j];
    return a;
}
__device__ __forceinline__ int acc_row(int r, int half) { return (r & 3) + 8 * (r >> 2) + 4 * half; }

template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
}
// sum over the 64 lanes, the same in all, without LDS: pairs, quads, half rows, rows of 16, then rows into the last one
__device__ __forceinline__ float row_sum(float v) {
    v = dpp_add<0xB1, 0xf>(v);   // lanes ^ 1
    v = dpp_add<0x4E, 0xf>(v);   // lanes ^ 2
    v = dpp_add<0x141, 0xf>(v);  // mirrored within 8
    v = dpp_add<0x140, 0xf>(v);  // mirrored within 16
    v = dpp_add<0x142, 0xa>(v);  // row 0 into 1, 2 into 3
    v = dpp_add<0x143, 0xc>(v);  // rows 0 and 1 into 2 and 3
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

template <int HDT>
struct AttnGeo {
    static constexpr int ROWBYTES = HDT * 2, NCH = HDT / 8, STEPS = HDT / 16, DT = HDT / 32;
    static __device__ __forceinline__ int swz(int row, int chunk) {
        const int x = ((((row >> 1) & 1) << 2) | ((row >> 2) & 3)) & (NCH - 1);
        return row * ROWBYTES + ((chunk ^ x) << 4);
    }
    static __device__ __forceinline__ bf16x8 rows(const char* img, int row, int step, int half) {
        return *reinterpret_cast<const bf16x8*>(img + swz(row, 2 * step + half));
    }
    static __device__ __forceinline__ bf16x8 cols(const char* img, int r0, int colbase, int lane) {
        const int q4 = (lane & 15) >> 2, p = lane & 3, h16 = (lane >> 4) & 1, half = lane >> 5;
        const int col = colbase + h16 * 16 + p * 4;
        const int ra = r0 + 4 * half + q4, rb = ra + 8;
        const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4_ptr)(img + swz(ra, col >> 3) + (col & 7) * 2));
        const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4_ptr)(img + swz(rb, col >> 3) + (col & 7) * 2));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    // rows [r0, r0 + 64) of a [*, row_stride] tensor -> LDS image rows 0..63 (zeros past S); 256 threads
    static __device__ __forceinline__ void stage64(char* img, const bf16* src, long row_stride, int r0, int S, int tid) {
        // every load of the block is issued before the first LDS store (a load -> wait -> store loop pays the memory
        // latency once per chunk); rows past S read row S - 1 and are zeroed by a select, so no load sits behind a branch
        constexpr int IT = 64 * NCH / 256;
        static_assert(IT >= 1 && 64 * NCH % 256 == 0, "a block is a whole number of chunks per thread");
        bf16x8 v[IT];
#pragma unroll
        for (int t = 0; t < IT; ++t) {
            const int i = tid + 256 * t, row = i / NCH, ch = i % NCH;
            const int rr = r0 + row < S ? r0 + row : S - 1;
            v[t] = *reinterpret_cast<const bf16x8*>(src + (long)rr * row_stride + ch * 8);
        }
#pragma unroll
        for (int t = 0; t < IT; ++t) {
            const int i = tid + 256 * t, row = i / NCH, ch = i % NCH;
            if (r0 + row >= S) {
#pragma unroll
                for (int k = 0; k < 8; ++k) v[t][k] = (bf16)0.f;
            }
            *reinterpret_cast<bf16x8*>(img + swz(row, ch)) = v[t];
        }
    }
    // a wave's own 32 rows as MFMA fragments straight from global memory (lane = row, 8 elements per step and half)
    static __device__ __forceinline__ void own_rows(bf16x8* f, const bf16* src, long row_stride, int row, int S, int half) {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
#pragma unroll
            for (int k = 0; k < 8; ++k) f[s][k] = (bf16)0.f;
            if (row < S) f[s] = *reinterpret_cast<const bf16x8*>(src + (long)row * row_stride + s * 16 + half * 8);
        }
    }
};

}  // namespace
}  // namespace pdt
