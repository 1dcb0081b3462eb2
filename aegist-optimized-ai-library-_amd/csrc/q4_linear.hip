// Projections with 4-bit weights:
//   Y[m, n] (+)= sum_k X[m, k] (code[n, k] scale[n, g] + min[n, g])
//             =  sum_g scale[n, g] (sum_{k in g} X[m, k] code[n, k]) + sum_g min[n, g] (sum_{k in g} X[m, k])
//
// Both sums are products of the matrix cores in fp16, with fp32 accumulation:
//   - a code is an fp16 value as it stands: its 4 bits at bits 6 to 9 are the subnormal code * 2^-18, which
//     v_mfma_f32_16x16x32_f16 takes at full value. Eight codes are seven instructions (four masks, three shifts),
//     with no conversion and no offset to subtract. (At bits 0 to 3 five would do, but the unit aligns the
//     products of an instruction by their operands' exponents, which a subnormal's leading zeros do not lower: six
//     more of them cost as many bits, 3.5e-6 instead of 2e-7 of the output's 2-norm at 8192 x 2048);
//   - a row of X is scaled by a power of two so that its largest value lies in [2^14, 2^15). A bf16 value is then
//     exact in fp16, an fp32 one the sum of two (hi rounded, lo the remainder): 22 bits, where the products
//     of the codes are exact. Values below 2^-28 of the row's largest lose bits to fp16's subnormals, at
//     most 2^-39 of that largest;
//   - the sums of a group's X (fp32, rounded to 22 bits in two fp16 parts) against the minima are one more product
//     with K / G in the place of K.
// A group's products are summed apart and then join the row's sum with the group's scale, in fp32.
#include "q4.h"

#include <algorithm>
#include <type_traits>

using namespace aegist;

namespace {

typedef uint32_t u4v __attribute__((ext_vector_type(4)));
typedef uint32_t u2v __attribute__((ext_vector_type(2)));

// the four fp16 pairs of eight codes, in units of 2^-18
__device__ __forceinline__ half8 q4_codes(uint32_t d) {
    constexpr uint32_t m = 0x03c003c0u;
    return __builtin_bit_cast(half8, u4v{d & m, d << 4 & m, d >> 4 & m, __builtin_amdgcn_alignbit(d, d, 8) & m});
}
// what undoes the units of the code products (2^-18) beside those of the minima (X's sums in units of 2^7)
constexpr float kCodeUnit = 0x1p11f;

// power of two by which a row of X is scaled; 0 for rows without a finite largest value (their outputs are not)
__device__ __forceinline__ int row_exp(float amax) {
    return amax > 0.f && amax < INFINITY ? 14 - ((int)(__float_as_uint(amax) >= 0x00800000u
                                                        ? (__float_as_uint(amax) >> 23) - 127
                                                        : -118 - __builtin_clz(__float_as_uint(amax))))
                                         : 0;
}

// 8 consecutive values of X as floats
__device__ __forceinline__ void x8(const float* p, float (&f)[8]) {
    const float4 a = ((const float4*)p)[0], b = ((const float4*)p)[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
__device__ __forceinline__ void x8(const uint16_t* p, float (&f)[8]) {
    const uint4 a = *(const uint4*)p;
    f[0] = bf_lo(a.x); f[1] = bf_hi(a.x); f[2] = bf_lo(a.y); f[3] = bf_hi(a.y);
    f[4] = bf_lo(a.z); f[5] = bf_hi(a.z); f[6] = bf_lo(a.w); f[7] = bf_hi(a.w);
}

// 8 scaled values as fp16; `lo` gets the remainders
__device__ __forceinline__ half8 x_parts(const float (&f)[8], int e, half8* lo) {
    half8 hi;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float v = __builtin_ldexpf(f[i], e);
        hi[i] = (_Float16)v;
        if (lo) (*lo)[i] = (_Float16)(v - (float)hi[i]);
    }
    return hi;
}

struct Q4Args {
    const void* X;
    long long ldx;
    const unsigned char* W;
    float* Y;
    long long ldy;
    int M, accumulate;
    Q4Dims d;
};

// ---------------------------------------------------------------------------------------------
// Few rows: the weight stream. A workgroup stages X in LDS as fp16 rows and its waves then take whole 1 KB pieces
// of the weight as they lie in memory, PD pieces in flight each; KS waves share a tile of 16 rows of W, every KS-th
// piece each, and meet in LDS. The pieces of X are on their way from L2, and its rows are scaled, while the first
// pieces of the weight come from HBM.
constexpr int SW = 8;           // waves of a workgroup
constexpr int SPD = 8;          // pieces in flight per wave
constexpr int SK = 128;         // k per piece

struct StreamLds {              // byte offsets
    int rows, row_bytes, xs, xs_bytes, exps, red, total;
};
__host__ __device__ inline StreamLds stream_lds(int M, int parts, const Q4Dims& d, int ks) {
    StreamLds l;
    l.rows = 0;
    l.row_bytes = d.chunks() * SK * 2 + 16;  // (16 bytes on: the 16 rows of an operand read lie in different banks)
    l.xs = M * parts * l.row_bytes;
    l.xs_bytes = (d.K / d.G + 31) / 32 * 64 + 16;
    l.exps = l.xs + 2 * M * l.xs_bytes;
    l.red = l.exps + 64;
    l.total = l.red + (ks > 1 ? 2 * SW * 1024 : 0);
    return l;
}

// SPG: steps of 32 k per group. PK: fp32 X of up to 8 rows, its two parts as rows m and m + 8 of one operand.
template <typename TX, int SPG, bool PK, int KS>
__global__ void __launch_bounds__(64 * SW) q4_stream_kernel(const Q4Args a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    constexpr bool F32 = std::is_same<TX, float>::value;
    constexpr int PARTS = F32 ? 2 : 1, NA = F32 && !PK ? 2 : 1, TW = SW / KS;
    constexpr int GP = 4 / SPG;  // groups per piece
    const Q4Dims d = a.d;
    const Q4Ptr w = q4_ptr(a.W, d);
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int r = lane % 16, q = lane / 16, ks = wave % KS, tw = wave / KS;
    const int M = a.M, KC = d.chunks(), NG = d.K / d.G, B8 = d.blocks8(), tiles = d.tiles();
    const StreamLds sl = stream_lds(M, PARTS, d, KS);
    // a tile's items of this wave: pieces of codes, then blocks of 32 groups' minima
    const int ni = (KC + KS - 1) / KS, nb = ((NG + 31) / 32 + KS - 1) / KS, n1 = ni + nb;
    const int t0 = blockIdx.x * TW, tstep = gridDim.x * TW;
    const int its = (tiles - t0 + tstep - 1) / tstep;  // rounds of this workgroup's tiles (the same for its waves)

    u4v code[SPD];
    u2v sc[SPD];
    int lt = t0 + tw, li = 0;
    auto load = [&](int slot) {
        code[slot] = u4v{0, 0, 0, 0};
        sc[slot] = u2v{0, 0};
        if (lt < tiles) {
            if (li < ni) {
                const int c = ks + KS * li;
                if (c < KC) {
                    code[slot] = __builtin_nontemporal_load((const u4v*)w.codes + ((size_t)lt * KC + c) * 64 + lane);
                    const _Float16* p = w.scale + ((size_t)lt * B8 + c * GP / 8) * 128 + r * 8 + c * GP % 8;
                    if (GP == 4) sc[slot] = *(const u2v*)p;
                    else if (GP == 2) sc[slot][0] = *(const uint32_t*)p;
                    else sc[slot][0] = *(const uint16_t*)p;
                }
            } else {
                const int b8 = (ks + KS * (li - ni)) * 4 + q;
                if (b8 < B8) code[slot] = *(const u4v*)(w.mins + ((size_t)lt * B8 + b8) * 128 + r * 8);
            }
        }
        if (++li == n1) li = 0, lt += tstep;
    };
#pragma unroll
    for (int s = 0; s < SPD; s++) load(s);

    // X: `wpr` waves per row, 8 consecutive values per lane and step
    {
        int* exps = (int*)(lds + sl.exps);
        float* part = (float*)(lds + sl.exps);  // one maximum per wave, before the exponents take their place
        const int wpr = M == 1 ? 8 : M == 2 ? 4 : M <= 4 ? 2 : 1, seg = wave % wpr;
        const int KP = KC * SK;
        auto amax_of = [&](int m) {
            const TX* x = (const TX*)a.X + (size_t)m * a.ldx;
            float v = 0.f;
            for (int k = (seg * WAVE + lane) * 8; k < d.K; k += wpr * WAVE * 8) {
                float f[8];
                x8(x + k, f);
#pragma unroll
                for (int i = 0; i < 8; i++) v = fmaxf(v, fabsf(f[i]));
            }
            return wave_max(v);
        };
        auto convert = [&](int m, int e) {
            const TX* x = (const TX*)a.X + (size_t)m * a.ldx;
            for (int k0 = seg * WAVE * 8; k0 < KP; k0 += wpr * WAVE * 8) {
                const int k = k0 + lane * 8;
                float f[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                if (k < d.K) x8(x + k, f);
                half8 lo;
                const half8 hi = x_parts(f, e, F32 ? &lo : nullptr);
                if (k < KP) {
                    *(half8*)(lds + m * sl.row_bytes + 2 * k) = hi;
                    if (F32) *(half8*)(lds + (M + m) * sl.row_bytes + 2 * k) = lo;
                }
                // the group's sum: 4, 8 or 16 lanes
                float s = ((f[0] + f[1]) + (f[2] + f[3])) + ((f[4] + f[5]) + (f[6] + f[7]));
#pragma unroll
                for (int o = 1; o < 4 * SPG; o *= 2) s += __shfl_xor(s, o, WAVE);
                if (lane % (4 * SPG) == 0 && k < d.K) {
                    s = __builtin_ldexpf(s, e - 7);
                    const _Float16 h = (_Float16)s;
                    *(_Float16*)(lds + sl.xs + m * sl.xs_bytes + k / d.G * 2) = h;
                    *(_Float16*)(lds + sl.xs + (M + m) * sl.xs_bytes + k / d.G * 2) = (_Float16)(s - (float)h);
                }
            }
            if (seg == 0)
                for (int g = NG + lane; g < (NG + 31) / 32 * 32; g += WAVE) {
                    *(_Float16*)(lds + sl.xs + m * sl.xs_bytes + g * 2) = 0;
                    *(_Float16*)(lds + sl.xs + (M + m) * sl.xs_bytes + g * 2) = 0;
                }
        };
        if (wpr > 1) {
            const int m = wave / wpr;
            const float v = m < M ? amax_of(m) : 0.f;
            if (lane == 0) part[wave] = v;
            lds_barrier();
            float v2 = 0.f;
            for (int i = 0; i < wpr; i++) v2 = fmaxf(v2, part[wave / wpr * wpr + i]);
            const int e = row_exp(v2);
            lds_barrier();
            if (m < M) {
                convert(m, e);
                if (seg == 0 && lane == 0) exps[m] = e;
            }
        } else {
            for (int m = wave; m < M; m += SW) {
                const int e = row_exp(amax_of(m));
                convert(m, e);
                if (lane == 0) exps[m] = e;
            }
        }
        lds_barrier();
    }

    // LDS rows of this lane's operand row
    const int mr = min(PK ? r % 8 : r, M - 1);
    const unsigned char* xrow[NA];
    xrow[0] = lds + ((PK && r >= 8 ? M : 0) + mr) * sl.row_bytes + q * 16;
    if (NA == 2) xrow[NA - 1] = lds + (M + mr) * sl.row_bytes + q * 16;
    const unsigned char* srow = lds + sl.xs + min(r, M - 1) * sl.xs_bytes + q * 16;

    f32x4 acc{0.f, 0.f, 0.f, 0.f}, accm{0.f, 0.f, 0.f, 0.f};
    int ct = t0 + tw, ci = 0, it = 0;
    const int total = its * n1;
    for (int f = 0; f < total; f += SPD) {
#pragma unroll
        for (int s = 0; s < SPD; s++) {
            if (f + s >= total) break;
            if (ci < ni) {
                const int c = ks + KS * ci;
                if (c < KC) {
                    f32x4 p{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const half8 b = q4_codes(code[s][j]);
#pragma unroll
                        for (int n = 0; n < NA; n++) {
                            const half8 x = *(const half8*)(xrow[n] + c * (SK * 2) + j * 64);
                            p = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, b, p, 0, 0, 0);
                        }
                        if (j % SPG == SPG - 1) {
                            const int g = j / SPG;
                            const float scale = (float)__builtin_bit_cast(_Float16, (uint16_t)(sc[s][g / 2] >> (16 * (g % 2))));
                            acc += p * scale;
                            p = f32x4{0.f, 0.f, 0.f, 0.f};
                        }
                    }
                }
            } else {
                const int b = ks + KS * (ci - ni);
                if (b * 32 < NG) {
                    const half8 mn = __builtin_bit_cast(half8, code[s]);
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        const half8 x = *(const half8*)(srow + n * M * sl.xs_bytes + b * 64);
                        accm = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, mn, accm, 0, 0, 0);
                    }
                }
            }
            load(s);
            if (++ci < n1) continue;
            // the tile's last item: lane (r, q) holds rows 4 q .. 4 q + 3 of Y's column 16 ct + r
            f32x4 v = acc * kCodeUnit;
            if (PK) {
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] = pair_sum32(v[i]);
            }
            v += accm;
            bool mine = true;
            if (KS > 1) {
                f32x4* red = (f32x4*)(lds + sl.red + it % 2 * (SW * 1024));
                red[wave * 64 + lane] = v;
                lds_barrier();
                mine = ks == 0;
                if (mine) {
#pragma unroll
                    for (int i = 1; i < KS; i++) v += red[(wave + i) * 64 + lane];
                }
            }
            const int n = ct * 16 + r;
            if (mine && ct < tiles && n < d.N) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int m = 4 * q + i;
                    if (m < M) {
                        float* y = a.Y + (size_t)m * a.ldy + n;
                        const float o = __builtin_ldexpf(v[i], 7 - ((const int*)(lds + sl.exps))[m]);
                        *y = a.accumulate ? *y + o : o;
                    }
                }
            }
            acc = accm = f32x4{0.f, 0.f, 0.f, 0.f};
            ci = 0;
            ct += tstep;
            it++;
        }
    }
}

template <typename TX, int SPG, bool PK, int KS>
int launch_stream(const Q4Args& a, int grid, hipStream_t st) {
    const int bytes = stream_lds(a.M, std::is_same<TX, float>::value ? 2 : 1, a.d, KS).total;
    if (bytes > 65536)
        AEG_HIP(hipFuncSetAttribute((const void*)q4_stream_kernel<TX, SPG, PK, KS>,
                                    hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    q4_stream_kernel<TX, SPG, PK, KS><<<grid, 64 * SW, bytes, st>>>(a);
    return after_launch("linear_q4");
}

template <typename TX, int SPG, bool PK>
int stream_ks(const Q4Args& a, hipStream_t st) {
    const int tiles = a.d.tiles();
    // waves per tile
    const int ks = tiles >= 4096 ? 1 : tiles >= 1024 ? 4 : 8;
    auto grid = [&](int k) { return std::min((tiles + SW / k - 1) / (SW / k), 512); };
    switch (ks) {
        case 1: return launch_stream<TX, SPG, PK, 1>(a, grid(1), st);
        case 4: return launch_stream<TX, SPG, PK, 4>(a, grid(4), st);
        default: return launch_stream<TX, SPG, PK, 8>(a, grid(8), st);
    }
}

template <typename TX, bool PK>
int stream_spg(const Q4Args& a, hipStream_t st) {
    switch (a.d.G) {
        case 32: return stream_ks<TX, 1, PK>(a, st);
        case 64: return stream_ks<TX, 2, PK>(a, st);
        default: return stream_ks<TX, 4, PK>(a, st);
    }
}

// ---------------------------------------------------------------------------------------------
// 16 rows of W x 16 rows of X per workgroup, a product per thread.
template <typename TX>
__global__ void __launch_bounds__(256) linear_q4_kernel(const TX* __restrict__ X, long long ldx,
                                                        const unsigned char* __restrict__ W, float* __restrict__ Y,
                                                        long long ldy, int M, const Q4Dims d, int accumulate) {
    const int r = threadIdx.x % 16, n = blockIdx.x * 16 + r;
    const Q4Ptr w = q4_ptr(W, d);
    for (int m = blockIdx.y * 16 + threadIdx.x / 16; m < M; m += gridDim.y * 16) {
        if (n >= d.N) return;
        const TX* x = X + (size_t)m * ldx;
        float acc = 0.f;
        for (int g = 0; g < d.K / d.G; g++) {
            float p = 0.f, s = 0.f;
            for (int k = g * d.G; k < (g + 1) * d.G; k += 8) {
                const int lane = k % 32 / 8 * 16 + r;
                const uint32_t v = ((const uint32_t*)w.codes)[(((size_t)blockIdx.x * d.chunks() + k / 128) * 64 + lane) * 4 +
                                                              k % 128 / 32];
                for (int e = 0; e < 8; e++) {
                    const float f = Act<TX>::ld(x, k + e);
                    p = fmaf((float)q4_get(v, e), f, p);
                    s += f;
                }
            }
            const size_t gi = ((size_t)(n / 16) * d.blocks8() + g / 8) * 128 + (n % 16) * 8 + g % 8;
            acc = fmaf(p, (float)w.scale[gi], fmaf(s, (float)w.mins[gi], acc));
        }
        float* y = Y + (size_t)m * ldy + n;
        *y = accumulate ? *y + acc : acc;
    }
}

// LDS that a workgroup may take: 160 KB per CU
constexpr int kStreamLds = 160 * 1024;

bool stream_fits(int x_dtype, int M, const Q4Dims& d) {
    return M <= 16 && stream_lds(M, x_dtype == AEGIST_F32 ? 2 : 1, d, SW).total <= kStreamLds;
}

}  // namespace

namespace aegist {

size_t linear_q4_workspace(int x_dtype, int M, int N, int K, int G) {
    (void)x_dtype, (void)M, (void)N, (void)K, (void)G;
    return 0;
}

int launch_linear_q4(const void* X, int x_dtype, long long ldx, const void* W, float* Y, long long ldy, int M, int N,
                     int K, int G, int accumulate, void*, size_t, hipStream_t st) {
    int rc = check_q4("linear_q4", N, K, G);
    if (rc) return rc;
    if (x_dtype != AEGIST_F32 && x_dtype != AEGIST_BF16)
        return fail(AEGIST_ERR_DTYPE, "linear_q4: X must be AEGIST_F32 or AEGIST_BF16");
    if (M < 0) return fail(AEGIST_ERR_SHAPE, "linear_q4: negative size");
    if (M == 0 || N == 0) return 0;
    if (!X || !W || !Y) return fail(AEGIST_ERR_SHAPE, "linear_q4: null operand");
    const int xs = x_dtype == AEGIST_F32 ? 4 : 2;
    if (ldx < K || (ldx * xs) % 16 || (uintptr_t)X % 16)
        return fail(AEGIST_ERR_SHAPE, "linear_q4: X needs 16-byte aligned rows (ldx >= K)");
    if (ldy < N) return fail(AEGIST_ERR_SHAPE, "linear_q4: ldy < N");
    if ((uintptr_t)W % 16) return fail(AEGIST_ERR_SHAPE, "linear_q4: W must be 16-byte aligned");
    const Q4Dims d{N, K, G};
    if (stream_fits(x_dtype, M, d)) {
        const Q4Args a{X, ldx, (const unsigned char*)W, Y, ldy, M, accumulate, d};
        if (x_dtype == AEGIST_BF16) return stream_spg<uint16_t, false>(a, st);
        return M <= 8 ? stream_spg<float, true>(a, st) : stream_spg<float, false>(a, st);
    }
    const dim3 grid(d.tiles(), std::min((M + 15) / 16, 65535));
    if (x_dtype == AEGIST_F32)
        linear_q4_kernel<float><<<grid, 256, 0, st>>>((const float*)X, ldx, (const unsigned char*)W, Y, ldy, M, d, accumulate);
    else
        linear_q4_kernel<uint16_t><<<grid, 256, 0, st>>>((const uint16_t*)X, ldx, (const unsigned char*)W, Y, ldy, M, d, accumulate);
    return after_launch("linear_q4");
}

}  // namespace aegist

extern "C" size_t aegist_linear_q4_workspace_bytes(int x_dtype, int M, int N, int K, int group) {
    if (M < 0 || check_q4("linear_q4_workspace", N, K, group)) return 0;
    return linear_q4_workspace(x_dtype, M, N, K, group);
}

extern "C" int aegist_linear_q4(const void* X, int x_dtype, long long ldx, const void* q4, float* Y, long long ldy,
                                int M, int N, int K, int group, int accumulate, void* ws, size_t ws_bytes,
                                void* stream) {
    return launch_linear_q4(X, x_dtype, ldx, q4, Y, ldy, M, N, K, group, accumulate, ws, ws_bytes, AEG_STREAM(stream));
}
