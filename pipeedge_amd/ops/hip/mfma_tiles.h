// Pieces shared by the kernels built from swizzled LDS images: LDS-DMA into
// them, the two kinds of fragment reads, and the running reference of a
// softmax.
#pragma once

#include "common.h"

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <typename T> struct TileVec;
template <> struct TileVec<__bf16> {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    typedef __bf16 v4 __attribute__((ext_vector_type(4)));
};
template <> struct TileVec<_Float16> {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    typedef _Float16 v4 __attribute__((ext_vector_type(4)));
};

__device__ __forceinline__ f32x16 tile_mfma(TileVec<__bf16>::v8 a,
                                              TileVec<__bf16>::v8 b,
                                              f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 tile_mfma(TileVec<_Float16>::v8 a,
                                              TileVec<_Float16>::v8 b,
                                              f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ f32x4 tile_mfma(TileVec<__bf16>::v8 a,
                                             TileVec<__bf16>::v8 b,
                                             f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 tile_mfma(TileVec<_Float16>::v8 a,
                                             TileVec<_Float16>::v8 b,
                                             f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// An LDS image holds rows of CH 16-byte chunks without padding, as LDS-DMA
// writes it; chunk c of row r lies at chunk position c ^ key(r). The key keeps
// both reads at full rate (64 banks of 4 B, 256 B a cycle):
// - rows at one chunk (M = 32) or at 4 adjacent ones (M = 16, the chunk from
//   lane / 16). A 16-byte read takes 16 lanes a cycle, 0-3, 12-15 and 20-27
//   of the first 32, then the other 16, so for M = 16 rows 0-3 and 12-15 at
//   one chunk meet rows 4-11 at the next one: the second lowest key bit tells
//   these row sets apart, and the lowest one is free to pair rows in a set
//   (124 B a cycle with the row's bits in order, 230 so);
// - 8 consecutive rows at 2 or 4 adjacent chunks (the transposing reads).
// Rows of 16k chunks all start at bank 0, so the low two bits of the row
// choose among groups of 4 chunks; rows of 16k + 8 chunks alternate between
// two halves already, rows of 8k + 4 between four quarters.
template <int CH>
__device__ __forceinline__ constexpr int tile_key(int row) {
    const int low = (((row >> 3) ^ (row >> 2)) & 1) * 2 + ((row >> 3) & 1);
    if constexpr (CH % 16 == 0)
        return ((row & 3) << 2) | low;
    else if constexpr (CH % 8 == 0)
        return (((row >> 1) & 1) << 2) | low;
    else
        return low;
}

// 16 bytes a lane from global memory into LDS at dst + lane * 16 (LDS-DMA).
// Written out because the compiler, which cannot tell the buffers of an image
// apart, would wait for all pieces on their way before each transposing read
// (with tiles of 32 tokens, three ahead, which that had ruled out, 64 ragged
// cached sequences of 16 heads went from 46 to 41 us). It does not count these
// loads, which only makes its own waits longer than they need to be; waiting
// for a piece is the caller's part, with an explicit s_waitcnt vmcnt and a
// barrier, whose clobbers also keep LDS accesses on their side. The load has
// no output register that could be reused early.
__device__ __forceinline__ void tile_load(const void* src, void* dst) {
    // dst is the same for all lanes, which the compiler may have lost
    const int to = __builtin_amdgcn_readfirstlane(
        (int)reinterpret_cast<uintptr_t>(dst));
    asm volatile("s_mov_b32 m0, %0\n\t"
                 "s_nop 0\n\t"
                 "global_load_lds_dwordx4 %1, off"
                 :
                 : "s"(to), "v"(src)
                 : "m0");
}
// the same from base + offset, base the same for all lanes
__device__ __forceinline__ void tile_load(const void* base, unsigned offset,
                                          void* dst) {
    const int to = __builtin_amdgcn_readfirstlane(
        (int)reinterpret_cast<uintptr_t>(dst));
    const uintptr_t b = reinterpret_cast<uintptr_t>(base);
    const uintptr_t from =
        (uintptr_t)(unsigned)__builtin_amdgcn_readfirstlane((int)b)
        | (uintptr_t)__builtin_amdgcn_readfirstlane((int)(b >> 32)) << 32;
    asm volatile("s_mov_b32 m0, %0\n\t"
                 "s_nop 0\n\t"
                 "global_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(to), "v"(offset), "s"(from)
                 : "m0");
}

// Makes the compiler wait for a loaded value here: at its first use inside a
// loop it would wait in every turn, and for the pieces on their way as well.
template <typename V>
__device__ __forceinline__ void tile_settle(V& v) {
    asm volatile("" : "+v"(v));
}

// At the head of a rare branch: without it the compiler computes the branch's
// values in every turn and selects, which costs more than the branch.
__device__ __forceinline__ void tile_rare() { asm volatile(""); }

// Wait for this wave's LDS-DMA, then for all waves. The clobbers keep LDS
// accesses on their side of the barrier.
__device__ __forceinline__ void tile_arrive() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Chunks that a key permutes among each other.
template <int CH>
__device__ __forceinline__ constexpr int tile_group() {
    return CH % 16 == 0 ? 16 : CH % 8 == 0 ? 8 : 4;
}

// Fragment addresses are kept as one register a tile: a chunk number known
// at compile time only flips address bits inside a group of chunks or adds a
// constant, since rows and images begin at multiples of a group.

__device__ __forceinline__ unsigned tile_lds(const void* p) {
    return (unsigned)reinterpret_cast<uintptr_t>(p);    // byte address
}

// Both products run on M x M MFMAs, M = 16 (k = 32) or 32 (k = 16); the 64
// lanes are 64 / M groups of M, and lane l gives k = 8 (l / M) + 0..7 of
// row l % M.

// Score operand: chunks (64 / M) i + l / M of row row0 + l % M
template <int CH, int M>
__device__ __forceinline__ unsigned tile_row_base(unsigned image,
                                                    int lane) {
    const int row = lane % M;
    return image + row * CH * 16 + (((lane / M) ^ tile_key<CH>(row)) << 4);
}
template <typename T, int CH, int M>
__device__ __forceinline__ typename TileVec<T>::v8 tile_row_read(
        unsigned base, int row0, int i) {
    constexpr int G = tile_group<CH>(), STEP = 64 / M;
    const unsigned at = (base ^ ((STEP * i % G) << 4))
                        + (STEP * i / G) * G * 16 + row0 * CH * 16;
    return *reinterpret_cast<const __attribute__((address_space(3)))
        typename TileVec<T>::v8*>((uintptr_t)at);
}

template <typename T>
__device__ __forceinline__ typename TileVec<T>::v4 tile_tr_read(
        unsigned at) {
    typedef __attribute__((address_space(3))) TileVec<__bf16>::v4 lds_v4;
    const auto r = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
        reinterpret_cast<lds_v4*>((uintptr_t)at));
    return __builtin_bit_cast(typename TileVec<T>::v4, r);
}

// Value operand, V^T[M columns from M n][tokens]: lane l gets column l % M.
// The sum over tokens may take them in any order, so the 8 values of a lane
// are those tokens whose scores the lane holds: 4 (l / M) + 0..3 and the same
// + 256 / M, counted from row0. No weight ever crosses lanes. A transposing
// read turns 4 rows of 16 columns, given as 4 adjacent elements by each of 16
// lanes, into one column of 4 rows for each of them.
template <int CH, int M>
__device__ __forceinline__ unsigned tile_column_base(unsigned image,
                                                       int lane) {
    const int row = lane / M * 4 + ((lane & 15) >> 2);
    const int chunk = (lane % M >= 16 ? 2 : 0) + ((lane & 3) >> 1);
    return image + row * CH * 16 + ((chunk ^ tile_key<CH>(row)) << 4)
           + (lane & 1) * 8;
}
template <typename T, int CH, int M>
__device__ __forceinline__ typename TileVec<T>::v8 tile_column_read(
        unsigned base, int row0, int n) {
    constexpr int G = tile_group<CH>(), STEP = M / 8;
    constexpr int NEXT = 256 / M;       // rows to the second read
    // 16 rows on, a row's key is the same; 8 rows on, the same bits differ
    constexpr unsigned flip8 =
        NEXT == 16 ? 0 : (tile_key<CH>(8) ^ tile_key<CH>(0)) << 4;
    const unsigned flip = (STEP * n % G) << 4;
    const unsigned add = (STEP * n / G) * G * 16 + row0 * CH * 16;
    const auto lo = tile_tr_read<T>((base ^ flip) + add);
    const auto hi = tile_tr_read<T>((base ^ flip ^ flip8) + add
                                      + NEXT * CH * 16);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// eight weights, rounded to the type of the values they multiply
template <typename T>
__device__ __forceinline__ typename TileVec<T>::v8 tile_weights(
        const float (&w)[8]) {
    typename TileVec<T>::v8 r;
    #pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = (T)w[j];
    return r;
}

// Running reference of the softmax, in powers of two. Weights are kept as
// 2^(score - reference) and the reference moves only when a score exceeds it
// by more than SLACK, which leaves the accumulators alone in most tiles; the
// weights then stay below 2^SLACK above their usual range, and sums are held
// in 32 bits. fp16 weights end at 65504 and lose bits below 2^-14, so they
// are shifted up by BIAS.
template <typename T> struct RunningTop {
    static constexpr float SLACK = 8.0f, BIAS = 0.0f;
};
template <> struct RunningTop<_Float16> {
    static constexpr float SLACK = 5.0f, BIAS = 8.0f;
};

// Blocks go to the 8 XCDs in turn; give each XCD a contiguous range of the
// work, so that neighbours, which read the same keys, share its L2.
__device__ __forceinline__ int xcd_contiguous(int block, int blocks) {
    const int whole = blocks / 8, extra = blocks % 8;
    const int xcd = block % 8, i = block / 8;
    return xcd * whole + min(xcd, extra) + i;
}
