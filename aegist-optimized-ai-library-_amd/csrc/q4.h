// Layout of a 4-bit weight matrix as the projections read it (Q4 weight), and the host-side launchers of
// q4.hip that other files call.
//
// A weight [N, K] in groups of G = 32, 64 or 128 consecutive k: w[n, k] = code * scale[n, k / G] + min[n, k / G],
// codes 0..15, scale and min in fp16. One block of memory with three sections:
//   codes   [N / 16][K / 128][64 lanes][16 bytes]: 1 KB holds 16 rows x 128 k in the order of the matrix
//           operand of v_mfma_f32_16x16x32_f16, so that a wave reads 1 KB in one contiguous piece and needs no
//           exchange between lanes. Lane 16 q + r has row r; its dword j has the 8 codes k = 32 j + 8 q + e,
//           element e from bit q4_bit(e) on (element 7 from bit 30 round to bit 1): in place, shifted by 4 either
//           way and turned by 8, two codes at a time come to lie at bits 6 to 9 of a dword's halves.
//   scale   [N / 16][K / G / 8][16 rows][8 groups] fp16: 16 bytes are 8 consecutive groups of a row
//   min     the same
// Rows, k and groups past the matrix are zeros.
#pragma once

#include "common.h"

namespace aegist {

__host__ __device__ constexpr int q4_bit(int e) { return (e % 2) * 16 + (e < 2 ? 6 : e < 4 ? 2 : e < 6 ? 10 : 14); }
__host__ __device__ constexpr uint32_t q4_put(uint32_t code, int e) {
    return code << q4_bit(e) | (q4_bit(e) > 28 ? code >> (32 - q4_bit(e)) : 0);
}
__host__ __device__ constexpr uint32_t q4_get(uint32_t d, int e) {
    return (d >> q4_bit(e) | (q4_bit(e) > 28 ? d << (32 - q4_bit(e)) : 0)) & 15;
}

struct Q4Dims {
    int N, K, G;
    __host__ __device__ int tiles() const { return (N + 15) / 16; }
    __host__ __device__ int chunks() const { return (K + 127) / 128; }
    __host__ __device__ int blocks8() const { return (K / G + 7) / 8; }
    __host__ __device__ size_t code_bytes() const { return (size_t)tiles() * chunks() * 1024; }
    __host__ __device__ size_t scale_bytes() const { return (size_t)tiles() * blocks8() * 256; }
    __host__ __device__ size_t bytes() const { return code_bytes() + 2 * scale_bytes(); }
};

struct Q4Ptr {
    const unsigned char* codes;
    const _Float16 *scale, *mins;
};
__host__ __device__ inline Q4Ptr q4_ptr(const void* w, const Q4Dims& d) {
    const unsigned char* p = (const unsigned char*)w;
    return {p, (const _Float16*)(p + d.code_bytes()), (const _Float16*)(p + d.code_bytes() + d.scale_bytes())};
}

typedef uint32_t u4v __attribute__((ext_vector_type(4)));

// 8 consecutive values of a row (k a multiple of 8; rows 16-byte aligned). ONCE: read past the caches
template <typename T> struct X8;
template <> struct X8<float> {
    f32x4 v[2];
    // zeros where k is past the row's K (a multiple of 8)
    template <bool ONCE = false>
    __device__ __forceinline__ void load(const float* row, int k, int K) {
        const f32x4* p = (const f32x4*)(row + min(k, K - 8));
        const f32x4 a = ONCE ? __builtin_nontemporal_load(p) : p[0], b = ONCE ? __builtin_nontemporal_load(p + 1) : p[1];
        v[0] = k < K ? a : f32x4{0, 0, 0, 0};
        v[1] = k < K ? b : f32x4{0, 0, 0, 0};
    }
    __device__ __forceinline__ float get(int i) const { return v[i / 4][i % 4]; }
};
template <> struct X8<uint16_t> {
    u4v v;
    template <bool ONCE = false>
    __device__ __forceinline__ void load(const uint16_t* row, int k, int K) {
        const u4v* p = (const u4v*)(row + min(k, K - 8));
        const u4v a = ONCE ? __builtin_nontemporal_load(p) : *p;
        v = k < K ? a : u4v{0, 0, 0, 0};
    }
    __device__ __forceinline__ float get(int i) const { return i % 2 ? bf_hi(v[i / 2]) : bf_lo(v[i / 2]); }
};

// AEGIST_OK, or the error of sizes that no Q4 weight has.
int check_q4(const char* who, int N, int K, int G);
// The kernel that M rows (of more than 2^19, the first block) take: 0 the stream, else tiles of 2, 4 or 8 x 16 rows.
int linear_q4_form(int x_dtype, int M, int N, int K, int G);
size_t linear_q4_workspace(int x_dtype, int M, int N, int K, int G);
int launch_linear_q4(const void* X, int x_dtype, long long ldx, const void* W, float* Y, long long ldy, int M, int N,
                     int K, int G, int accumulate, void* ws, size_t ws_bytes, hipStream_t st);

}  // namespace aegist
