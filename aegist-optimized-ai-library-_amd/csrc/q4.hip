// The making of 4-bit weights: rounding, packing and reading back. (The product is q4_linear.hip.)
#include "q4.h"

#include <algorithm>

using namespace aegist;

namespace {

// index of (row n, group g) in the scale and min sections
__device__ __forceinline__ size_t q4_group(const Q4Dims& d, int n, int g) {
    return ((size_t)(n / 16) * d.blocks8() + g / 8) * 128 + (n % 16) * 8 + g % 8;
}

// (fminf and fmaxf would first make a quiet NaN of every value, an instruction each)
__device__ __forceinline__ float min3(float a, float b, float c) {
    asm("v_min3_f32 %0, %0, %1, %2" : "+v"(a) : "v"(b), "v"(c));
    return a;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    asm("v_max3_f32 %0, %0, %1, %2" : "+v"(a) : "v"(b), "v"(c));
    return a;
}

__device__ __forceinline__ float abs_max3(float a, float b, float c) {
    asm("v_max3_f32 %0, %0, |%1|, |%2|" : "+v"(a) : "v"(b), "v"(c));
    return a;
}

// largest of the lanes l, l ^ 16, l ^ 32 and l ^ 48
__device__ __forceinline__ float quad_max(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// The codes of 8 values: (w - mn) / sc rounded to the nearest, ties to even, in 0..15, as doubles decide it. In fp32, with
// inv = 1 / sc (0 for no scale) to a unit, the quotient is off by at most 15.5 * 4 * 2^-24 < 2^-18, so only within 2^-16
// of a half can doubles say otherwise: 1 value in 30000, and the division in doubles is left to the eights that hold
// one (2048 x 4096 bf16: 28 us with it for all).
template <typename TW>
__device__ __forceinline__ uint32_t q4_code8(const X8<TW>& w, _Float16 mn, _Float16 sc, float inv) {
    float c[8], off = 0.f;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const float q0 = (w.get(e) - (float)mn) * inv, q1 = (w.get(e + 1) - (float)mn) * inv;
        c[e] = __builtin_rintf(q0);
        c[e + 1] = __builtin_rintf(q1);
        off = abs_max3(off, q0 - c[e], q1 - c[e + 1]);
    }
    if (off > 0.5f - 0x1p-16f) {
#pragma unroll
        for (int e = 0; e < 8; e++) c[e] = (float)rint(((double)w.get(e) - (double)mn) / (double)sc);
    }
    uint32_t p = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) p |= q4_put((uint32_t)__builtin_amdgcn_fmed3f(c[e], 0.f, 15.f), e);
    return p;
}

// One wave per 16 rows x 128 k. Lane 16 q + r holds the runs k = 32 j + 8 q .. + 7 of row r, so a group's extremes
// are its own values' and, over the four q, two exchanges'.
template <typename TW>
__global__ void __launch_bounds__(256) q4_quantize_kernel(const TW* __restrict__ W, long long ldw, unsigned char* out,
                                                          const Q4Dims d) {
    const int lane = threadIdx.x % WAVE, r = lane % 16, q = lane / 16;
    const int c = blockIdx.x * 4 + threadIdx.x / WAVE, nt = blockIdx.y + blockIdx.z * 65535;
    if (c >= d.chunks() || nt >= d.tiles()) return;
    const int n = nt * 16 + r;
    const bool row = n < d.N;
    X8<TW> w[4];
#pragma unroll
    for (int j = 0; j < 4; j++) w[j].template load<true>(W + (size_t)min(n, d.N - 1) * ldw, c * 128 + 32 * j + 8 * q, d.K);
    float lo[4], hi[4];  // (hi is infinite where a value has no place in the format)
#pragma unroll
    for (int j = 0; j < 4; j++) {
        lo[j] = hi[j] = w[j].get(0);
        float bad = 0.f;  // NaN with a NaN or infinity among the values, which the extremes may pass over
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            lo[j] = min3(lo[j], w[j].get(e), w[j].get(e + 1));
            hi[j] = max3(hi[j], w[j].get(e), w[j].get(e + 1));
            bad = __builtin_fmaf(w[j].get(e), 0.f, __builtin_fmaf(w[j].get(e + 1), 0.f, bad));
        }
        if (!(bad == 0.f && hi[j] <= 65504.f && lo[j] >= -65504.f)) hi[j] = INFINITY;
        lo[j] = -quad_max(-lo[j]);
        hi[j] = quad_max(hi[j]);
    }
    const int span = d.G / 32;  // runs of 32 k per group
#pragma unroll
    for (int s = 1; s < 4; s *= 2)
        if (s < span) {
            float l2[4], h2[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                l2[j] = fminf(lo[j], lo[j ^ s]);
                h2[j] = fmaxf(hi[j], hi[j ^ s]);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) lo[j] = l2[j], hi[j] = h2[j];
        }
    // lane 16 q + r: the minimum and scale of run q
    const float h = q == 0 ? hi[0] : q == 1 ? hi[1] : q == 2 ? hi[2] : hi[3];
    const float l = q == 0 ? lo[0] : q == 1 ? lo[1] : q == 2 ? lo[2] : lo[3];
    const _Float16 mn = h == INFINITY ? (_Float16)__builtin_nanf("") : (_Float16)l;
    const double range = ((double)h - (double)mn) / 15.0;
    const _Float16 sc = range > 0.0 ? (_Float16)range : (_Float16)0.f;
    const uint32_t both = (uint32_t)__builtin_bit_cast(uint16_t, mn) | (uint32_t)__builtin_bit_cast(uint16_t, sc) << 16;
    u4v codes;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t u = __shfl(both, 16 * j + r, WAVE);
        const _Float16 sj = __builtin_bit_cast(_Float16, (uint16_t)(u >> 16));
        const float inv = sj > (_Float16)0.f ? __builtin_amdgcn_rcpf((float)sj) : 0.f;
        codes[j] = q4_code8(w[j], __builtin_bit_cast(_Float16, (uint16_t)u), sj, inv);
        if (!row || c * 128 + 32 * j >= d.K || inv == 0.f) codes[j] = 0;
    }
    _Float16* scale = (_Float16*)(out + d.code_bytes());
    _Float16* mins = (_Float16*)(out + d.code_bytes() + d.scale_bytes());
    const int k = c * 128 + 32 * q;
    // (the rows past N and the groups past K too: zeros)
    if (k % d.G == 0 && k / d.G < d.blocks8() * 8) {
        const bool in = row && k < d.K;
        scale[q4_group(d, n, k / d.G)] = in ? sc : (_Float16)0.f;
        mins[q4_group(d, n, k / d.G)] = in ? mn : (_Float16)0.f;
    }
    if (c == d.chunks() - 1 && q == 0)
        for (int g = d.chunks() * (128 / d.G); g < d.blocks8() * 8; g++) scale[q4_group(d, n, g)] = mins[q4_group(d, n, g)] = 0;
    ((u4v*)out)[((size_t)nt * d.chunks() + c) * 64 + lane] = codes;
}

// Codes of the engine's layout (two to a byte, the even element low) into the operand's order, one wave per 16
// rows x 128 k. min = -8 scale where none are given: (code - 8) * scale.
__global__ void __launch_bounds__(256) q4_pack_kernel(const unsigned char* __restrict__ codes, unsigned char* out,
                                                      const Q4Dims d) {
    const int lane = threadIdx.x % WAVE, r = lane % 16, q = lane / 16;
    const int c = blockIdx.x * 4 + threadIdx.x / WAVE, nt = blockIdx.y + blockIdx.z * 65535;
    if (c >= d.chunks() || nt >= d.tiles()) return;
    const int n = nt * 16 + r;
    u4v v;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int k = c * 128 + 32 * j + 8 * q;
        uint32_t s = 0, p = 0;
        if (n < d.N && k < d.K) s = *(const uint32_t*)(codes + ((size_t)n * d.K + k) / 2);
#pragma unroll
        for (int e = 0; e < 8; e++) p |= q4_put(s >> (4 * e) & 15, e);
        v[j] = p;
    }
    ((u4v*)out)[((size_t)nt * d.chunks() + c) * 64 + lane] = v;
}

// Scales and minima from rows [N, K / G], with zeros in the places that no group has.
__global__ void __launch_bounds__(256) q4_pack_groups_kernel(const _Float16* __restrict__ scale,
                                                             const _Float16* __restrict__ mins, unsigned char* out,
                                                             const Q4Dims d) {
    const size_t all = d.scale_bytes() / 2;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (size_t)gridDim.x * 256) {
        const int g = (int)(i / 128 % d.blocks8()) * 8 + i % 8, n = (int)(i / 128 / d.blocks8()) * 16 + i / 8 % 16;
        _Float16 s = 0, m = 0;
        if (n < d.N && g < d.K / d.G) {
            s = scale[(size_t)n * (d.K / d.G) + g];
            m = mins ? mins[(size_t)n * (d.K / d.G) + g] : (_Float16)(-8.f * (float)s);
        }
        ((_Float16*)(out + d.code_bytes()))[i] = s;
        ((_Float16*)(out + d.code_bytes() + d.scale_bytes()))[i] = m;
    }
}

__global__ void __launch_bounds__(256) q4_dequantize_kernel(const unsigned char* __restrict__ W, float* __restrict__ out,
                                                            const Q4Dims d) {
    const int lane = threadIdx.x % WAVE, r = lane % 16, q = lane / 16;
    const int c = blockIdx.x * 4 + threadIdx.x / WAVE, nt = blockIdx.y + blockIdx.z * 65535;
    if (c >= d.chunks() || nt >= d.tiles()) return;
    const int n = nt * 16 + r;
    if (n >= d.N) return;
    const Q4Ptr w = q4_ptr(W, d);
    const u4v v = ((const u4v*)w.codes)[((size_t)nt * d.chunks() + c) * 64 + lane];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int k = c * 128 + 32 * j + 8 * q;
        if (k >= d.K) continue;
        const size_t gi = q4_group(d, n, k / d.G);
        const float s = (float)w.scale[gi], m = (float)w.mins[gi];
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; e++) f[e] = fmaf((float)q4_get(v[j], e), s, m);
        float4* o = (float4*)(out + (size_t)n * d.K + k);
        o[0] = float4{f[0], f[1], f[2], f[3]};
        o[1] = float4{f[4], f[5], f[6], f[7]};
    }
}

// grid over (chunks / 4, tiles): tiles past 65535 go on along z
dim3 q4_grid(const Q4Dims& d) {
    return dim3((d.chunks() + 3) / 4, std::min(d.tiles(), 65535), (d.tiles() + 65534) / 65535);
}

}  // namespace

namespace aegist {

int check_q4(const char* who, int N, int K, int G) {
    const std::string w(who);
    if (G != 32 && G != 64 && G != 128) return fail(AEGIST_ERR_SHAPE, w + ": groups of 32, 64 or 128 values");
    if (N < 0 || K <= 0 || K % G) return fail(AEGIST_ERR_SHAPE, w + ": K must be a positive multiple of the group");
    if (N > 1 << 28 || K > 1 << 28) return fail(AEGIST_ERR_SHAPE, w + ": N and K are at most 2^28");
    return 0;
}

}  // namespace aegist

extern "C" size_t aegist_q4_bytes(int N, int K, int group) {
    if (check_q4("q4_bytes", N, K, group)) return 0;
    return Q4Dims{N, K, group}.bytes();
}

extern "C" int aegist_q4_quantize(const void* W, int w_dtype, long long ldw, void* q4, int N, int K, int group,
                                  void* stream) {
    int rc = check_q4("q4_quantize", N, K, group);
    if (rc) return rc;
    if (w_dtype != AEGIST_F32 && w_dtype != AEGIST_BF16)
        return fail(AEGIST_ERR_DTYPE, "q4_quantize: W must be AEGIST_F32 or AEGIST_BF16");
    if (N == 0) return 0;
    if (!W || !q4 || (uintptr_t)q4 % 16) return fail(AEGIST_ERR_SHAPE, "q4_quantize: null operand, or q4 not 16-byte aligned");
    const int es = w_dtype == AEGIST_F32 ? 4 : 2;
    if (ldw < K || (ldw * es) % 16 || (uintptr_t)W % 16)
        return fail(AEGIST_ERR_SHAPE, "q4_quantize: W needs 16-byte aligned rows (ldw >= K)");
    const Q4Dims d{N, K, group};
    const hipStream_t st = AEG_STREAM(stream);
    if (w_dtype == AEGIST_F32)
        q4_quantize_kernel<float><<<q4_grid(d), 256, 0, st>>>((const float*)W, ldw, (unsigned char*)q4, d);
    else
        q4_quantize_kernel<uint16_t><<<q4_grid(d), 256, 0, st>>>((const uint16_t*)W, ldw, (unsigned char*)q4, d);
    return after_launch("q4_quantize");
}

extern "C" int aegist_q4_pack(const void* codes, const uint16_t* scale, const uint16_t* mins, void* q4, int N, int K,
                              int group, void* stream) {
    int rc = check_q4("q4_pack", N, K, group);
    if (rc) return rc;
    if (N == 0) return 0;
    if (!codes || !scale || !q4 || (uintptr_t)q4 % 16 || (uintptr_t)codes % 4)
        return fail(AEGIST_ERR_SHAPE, "q4_pack: null operand, q4 not 16-byte or codes not 4-byte aligned");
    const Q4Dims d{N, K, group};
    const hipStream_t st = AEG_STREAM(stream);
    q4_pack_kernel<<<q4_grid(d), 256, 0, st>>>((const unsigned char*)codes, (unsigned char*)q4, d);
    if ((rc = after_launch("q4_pack"))) return rc;
    q4_pack_groups_kernel<<<(unsigned)std::min<size_t>((d.scale_bytes() / 2 + 255) / 256, 1 << 20), 256, 0, st>>>(
        (const _Float16*)scale, (const _Float16*)mins, (unsigned char*)q4, d);
    return after_launch("q4_pack");
}

extern "C" int aegist_q4_dequantize(const void* q4, float* out, int N, int K, int group, void* stream) {
    int rc = check_q4("q4_dequantize", N, K, group);
    if (rc) return rc;
    if (N == 0) return 0;
    if (!q4 || !out || (uintptr_t)q4 % 16 || (uintptr_t)out % 16)
        return fail(AEGIST_ERR_SHAPE, "q4_dequantize: null operand, or one not 16-byte aligned");
    const Q4Dims d{N, K, group};
    q4_dequantize_kernel<<<q4_grid(d), 256, 0, AEG_STREAM(stream)>>>((const unsigned char*)q4, out, d);
    return after_launch("q4_dequantize");
}
