// Pieces shared by the two forms of latent attention: the swizzled LDS
// images that LDS-DMA fills, their two kinds of fragment reads, and the
// step from a score column in registers to the next product's operand.
#pragma once

#include "common.h"

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned uint2_ __attribute__((ext_vector_type(2)));
typedef unsigned uint4_ __attribute__((ext_vector_type(4)));

template <typename T> struct LatentVec;
template <> struct LatentVec<__bf16> {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    typedef __bf16 v4 __attribute__((ext_vector_type(4)));
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
};
template <> struct LatentVec<_Float16> {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    typedef _Float16 v4 __attribute__((ext_vector_type(4)));
    typedef _Float16 v2 __attribute__((ext_vector_type(2)));
};

__device__ __forceinline__ f32x16 latent_mfma(LatentVec<__bf16>::v8 a,
                                              LatentVec<__bf16>::v8 b,
                                              f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 latent_mfma(LatentVec<_Float16>::v8 a,
                                              LatentVec<_Float16>::v8 b,
                                              f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// An LDS image holds rows (tokens) of CH 16-byte chunks without padding, as
// LDS-DMA writes it; chunk c of row r lies at chunk position c ^ key(r). The
// key makes both reads free of bank conflicts (64 banks of 4 B):
// - 16 consecutive rows at one chunk (the score product's operand),
// - 4 consecutive rows at 4 adjacent chunks (the transposing reads of the
//   value product).
// Rows of 16k chunks all start at bank 0, so 16 keys are needed and rows
// that differ in their low two bits go to different groups of 4 chunks; rows
// of 16k + 8 chunks alternate between two halves already, rows of 8k + 4
// between four quarters.
template <int CH>
__device__ __forceinline__ constexpr int latent_key(int row) {
    if constexpr (CH % 16 == 0)
        return ((row & 3) << 2) | ((row >> 2) & 3);
    else if constexpr (CH % 8 == 0)
        return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
    else
        return (row >> 2) & 3;
}

// 16 bytes a lane from global memory into LDS at base + lane * 16
__device__ __forceinline__ void latent_lds_load(const void* src, void* dst) {
    __builtin_amdgcn_global_load_lds(
        (const __attribute__((address_space(1))) unsigned int*)src,
        (__attribute__((address_space(3))) unsigned int*)dst, 16, 0, 0);
}

// Wait for this wave's LDS-DMA, then for all waves. The clobbers keep LDS
// accesses on their side of the barrier.
__device__ __forceinline__ void latent_arrive() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// chunk c of row r
template <typename T, int CH>
__device__ __forceinline__ typename LatentVec<T>::v8 latent_row_read(
        const T* image, int row, int chunk) {
    return *reinterpret_cast<const typename LatentVec<T>::v8*>(
        image + (row * CH + (chunk ^ latent_key<CH>(row))) * 8);
}

template <typename T>
__device__ __forceinline__ typename LatentVec<T>::v4 latent_tr_read(
        const T* p) {
    typedef __attribute__((address_space(3))) LatentVec<__bf16>::v4 lds_v4;
    const auto r = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
        reinterpret_cast<lds_v4*>(reinterpret_cast<uintptr_t>(p)));
    return __builtin_bit_cast(typename LatentVec<T>::v4, r);
}

// A-operand of the value product, V^T[32 columns from col0][16 tokens from
// row0]: lane l gets column l & 31 of tokens row0 + (l >> 5) * 8 + 0..7. A
// transposing read turns 4 rows of 16 columns, given as 4 adjacent elements
// by each of 16 lanes, into one column of 4 rows for each of them.
template <typename T, int CH>
__device__ __forceinline__ typename LatentVec<T>::v8 latent_column_read(
        const T* image, int row0, int col0, int lane) {
    const int row = row0 + (lane >> 5) * 8 + ((lane & 15) >> 2);
    const int col = col0 + (lane & 16) + (lane & 3) * 4;
    const auto at = [&](int r) {
        return image + (r * CH + ((col >> 3) ^ latent_key<CH>(r))) * 8
               + (col & 7);
    };
    const auto lo = latent_tr_read<T>(at(row));
    const auto hi = latent_tr_read<T>(at(row + 4));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

template <typename T>
__device__ __forceinline__ unsigned latent_pack(float lo, float hi) {
    typename LatentVec<T>::v2 v = {(T)lo, (T)hi};
    return __builtin_bit_cast(unsigned, v);
}

// B-operand of the value product for tokens 16c .. 16c+15 of a 32-token
// score column: a lane's scores are tokens (lane >> 5) * 4 + 8 * (i >> 2) +
// (i & 3), the operand wants (lane >> 5) * 8 + 0..7, so the two halves of
// the wave exchange four values each.
template <typename T>
__device__ __forceinline__ typename LatentVec<T>::v8 latent_weights(
        const f32x16& p, int c) {
    const unsigned u0 = latent_pack<T>(p[8 * c + 0], p[8 * c + 1]);
    const unsigned u1 = latent_pack<T>(p[8 * c + 2], p[8 * c + 3]);
    const unsigned v0 = latent_pack<T>(p[8 * c + 4], p[8 * c + 5]);
    const unsigned v1 = latent_pack<T>(p[8 * c + 6], p[8 * c + 7]);
    const uint2_ w0 = __builtin_amdgcn_permlane32_swap(u0, v0, false, false);
    const uint2_ w1 = __builtin_amdgcn_permlane32_swap(u1, v1, false, false);
    const uint4_ w = {w0.x, w1.x, w0.y, w1.y};
    return __builtin_bit_cast(typename LatentVec<T>::v8, w);
}

// Running reference of the softmax, in powers of two. Weights are kept as
// 2^(score - reference) and the reference moves only when a score exceeds it
// by more than SLACK, which leaves the accumulators alone in most tiles; the
// weights then stay below 2^SLACK above their usual range, and sums are held
// in 32 bits. fp16 weights end at 65504 and lose bits below 2^-14, so they
// are shifted up by BIAS.
template <typename T> struct LatentSoftmax {
    static constexpr float SLACK = 8.0f, BIAS = 0.0f;
};
template <> struct LatentSoftmax<_Float16> {
    static constexpr float SLACK = 5.0f, BIAS = 8.0f;
};

// Blocks go to the 8 XCDs in turn; give each XCD a contiguous range of the
// work, so that neighbours, which read the same keys, share its L2.
__device__ __forceinline__ int xcd_contiguous(int block, int blocks) {
    const int whole = blocks / 8, extra = blocks % 8;
    const int xcd = block % 8, i = block / 8;
    return xcd * whole + min(xcd, extra) + i;
}
