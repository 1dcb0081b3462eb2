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

// 8 consecutive values of X
template <typename TX> struct X8;
template <> struct X8<float> {
    f32x4 v[2];
    // zeros where k is past the row's K (a multiple of 8)
    __device__ __forceinline__ void load(const float* row, int k, int K) {
        const f32x4* p = (const f32x4*)(row + min(k, K - 8));
        const f32x4 a = p[0], b = p[1];
        v[0] = k < K ? a : f32x4{0, 0, 0, 0};
        v[1] = k < K ? b : f32x4{0, 0, 0, 0};
    }
    __device__ __forceinline__ float get(int i) const { return v[i / 4][i % 4]; }
};
template <> struct X8<uint16_t> {
    u4v v;
    __device__ __forceinline__ void load(const uint16_t* row, int k, int K) {
        const u4v a = *(const u4v*)(row + min(k, K - 8));
        v = k < K ? a : u4v{0, 0, 0, 0};
    }
    __device__ __forceinline__ float get(int i) const { return i % 2 ? bf_hi(v[i / 2]) : bf_lo(v[i / 2]); }
};

// 8 scaled values as fp16; `lo` gets the remainders
template <typename TX>
__device__ __forceinline__ half8 x_parts(const X8<TX>& x, int e, half8* lo) {
    half8 hi;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float v = __builtin_ldexpf(x.get(i), e);
        hi[i] = (_Float16)v;
        if (lo) (*lo)[i] = (_Float16)(v - (float)hi[i]);
    }
    return hi;
}

struct Q4Args {
    const void* X;  // rows, or the operands made of them (XOps)
    long long ldx;
    const unsigned char* W;
    float* Y;
    long long ldy;
    int M, accumulate;
    Q4Dims d;
    int c0;         // first piece of K that a launch takes
};

// ---------------------------------------------------------------------------------------------
// More than a few rows: X is made into matrix operands once, in the workspace, in the order in which waves load
// them (1 KB for 16 rows x 32 k):
//   parts [M / 16][parts][K / 32][64 lanes][8 fp16]: lane 16 q + r has k = 32 j + 8 q .. + 7 of row r, with zeros
//         from K to a multiple of 256
//   sums  [M / 16][2 parts][K / G / 32][64 lanes][8 fp16]: the sums of the groups 32 b + 8 q .. + 7
//   exps  [M] int: the power of two each row was scaled by
struct XOps {
    int parts, steps, blocks;  // 32 k each, 32 groups each
    size_t tiles;
    __host__ __device__ XOps(int M, int parts, const Q4Dims& d)
        : parts(parts), steps((d.K + 255) / 256 * 8), blocks((d.K / d.G + 31) / 32), tiles((M + 15) / 16) {}
    __host__ __device__ size_t sums_at() const { return tiles * parts * steps * 1024; }
    __host__ __device__ size_t exps_at() const { return sums_at() + tiles * 2 * blocks * 1024; }
    __host__ __device__ size_t bytes() const { return exps_at() + (tiles * 64 + 255) / 256 * 256; }
};

// One workgroup per 16 rows; XW waves take the steps in turn, XJ of them held in registers between the row's maximum
// and its conversion (longer rows are read again, from L2).
constexpr int XW = 16, XJ = 4;

template <typename TX>
__global__ void __launch_bounds__(XW * WAVE) q4_rows_kernel(const Q4Args a, unsigned char* out) {
    constexpr bool F32 = std::is_same<TX, float>::value;
    __shared__ float top[XW][16];
    const Q4Dims d = a.d;
    const XOps o(a.M, F32 ? 2 : 1, d);
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int r = lane % 16, q = lane / 16, spg = d.G / 32, NG = d.K / d.G;
    const size_t mt = blockIdx.x;
    const TX* x = (const TX*)a.X + (mt * 16 + min(r, (int)(a.M - 1 - mt * 16))) * a.ldx;
    // consecutive steps of XJ = 4 hold whole groups
    const int rounds = (o.steps + XW * XJ - 1) / (XW * XJ);
    X8<TX> f[XJ];
    float amax = 0.f;
    for (int i = rounds - 1; i >= 0; i--) {  // (the first is read last and stays)
#pragma unroll
        for (int j = 0; j < XJ; j++) {
            const int k = ((i * XW + wave) * XJ + j) * 32 + 8 * q;
            f[j].load(x, k, d.K);
        }
#pragma unroll
        for (int j = 0; j < XJ; j++)
#pragma unroll
            for (int e = 0; e < 8; e++) amax = fmaxf(amax, fabsf(f[j].get(e)));
    }
    amax = fmaxf(amax, __shfl_xor(amax, 16, WAVE));
    amax = fmaxf(amax, __shfl_xor(amax, 32, WAVE));
    if (q == 0) top[wave][r] = amax;
    lds_barrier();
#pragma unroll
    for (int i = 0; i < XW; i++) amax = fmaxf(amax, top[i][r]);
    const int e = row_exp(amax);
    if (wave == 0 && q == 0) ((int*)(out + o.exps_at()))[mt * 16 + r] = e;
    half8* parts = (half8*)out;
    _Float16* sums = (_Float16*)(out + o.sums_at());
    for (int i = 0; i < rounds; i++) {
        const int j0 = (i * XW + wave) * XJ;
        if (j0 >= o.steps) break;
        if (i > 0) {
#pragma unroll
            for (int j = 0; j < XJ; j++) {
                const int k = (j0 + j) * 32 + 8 * q;
                f[j].load(x, k, d.K);
            }
        }
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < XJ; j++) {
            half8 lo;
            const half8 hi = x_parts(f[j], e, F32 ? &lo : nullptr);
            parts[(mt * o.parts * o.steps + j0 + j) * 64 + lane] = hi;
            if (F32) parts[((mt * o.parts + 1) * o.steps + j0 + j) * 64 + lane] = lo;
            s += ((f[j].get(0) + f[j].get(1)) + (f[j].get(2) + f[j].get(3))) + ((f[j].get(4) + f[j].get(5)) + (f[j].get(6) + f[j].get(7)));
            if ((j + 1) % spg) continue;
            s += __shfl_xor(s, 16, WAVE);
            s += __shfl_xor(s, 32, WAVE);
            s = __builtin_ldexpf(s, e - 7);
            const int g = (j0 + j) / spg;
            const _Float16 hs = (_Float16)s;
            if (q < 2 && g < NG)  // lane 16 q + r writes part q
                sums[(((mt * 2 + q) * o.blocks + g / 32) * 64 + g % 32 / 8 * 16 + r) * 8 + g % 8] = q ? (_Float16)(s - (float)hs) : hs;
            s = 0.f;
        }
    }
    // groups past the last
    for (int g = NG + wave; g < o.blocks * 32; g += XW)
        if (q < 2) sums[(((mt * 2 + q) * o.blocks + g / 32) * 64 + g % 32 / 8 * 16 + r) * 8 + g % 8] = 0;
}

// ---------------------------------------------------------------------------------------------
// Few rows: the weight as a stream, X in registers. The waves of a workgroup cut K into slices of CPS pieces (128 k
// each); a wave holds its slice of 16 RT rows of X as matrix operands and takes its pieces of one tile (16 rows of
// W) after the other, the next two in flight; per round of two tiles the waves' sums meet in LDS. So a weight
// is one contiguous 1 KB load and no more, nothing in the loop reads LDS but the sums, and a slice is
// scaled by its own largest value, which needs no exchange between waves.
//
// Waves that staged X in LDS, once per workgroup, and read it back per piece took 16.5 us at 16 rows of 2048 x 4096,
// mostly the staging (two rows per wave one after the other).

template <int SPG, int CPS>
struct Q4Slice {
    static constexpr int GROUPS = CPS * 4 / SPG;           // groups of a slice
    static constexpr int SB = (GROUPS + 7) / 8;            // blocks of 8 groups that they touch
    u4v code[CPS];
    u4v scale[SB], mins;
};

// SPG: steps of 32 k per group. PK: fp32 X of up to 8 rows, its two parts as rows m and m + 8 of one operand.
// MW: waves at most. PRE: X is there as operands (XOps), else every workgroup makes them of the rows.
template <typename TX, int SPG, bool PK, int RT, int CPS, int MW, bool PRE>
__global__ void __launch_bounds__(MW * WAVE) q4_stream_kernel(const Q4Args a) {
    constexpr bool F32 = std::is_same<TX, float>::value;
    constexpr int NA = F32 && !PK ? 2 : 1, NS = PK ? 1 : 2, ST = CPS * 4;
    constexpr int SUMS = RT < 2 ? 2 : RT;  // sums per meeting of the waves
    typedef Q4Slice<SPG, CPS> Slice;
    constexpr int NB = SUMS / RT;  // tiles of such a meeting
    extern __shared__ f32x4 red_raw[];  // [2][SUMS][KS][WAVE]
    const Q4Dims d = a.d;
    const Q4Ptr w = q4_ptr(a.W, d);
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int r = lane % 16, q = lane / 16, KS = blockDim.x / WAVE;
    const int KC = d.chunks(), B8 = d.blocks8(), tiles = d.tiles();
    const int c0 = a.c0 + wave * CPS, g0 = c0 * (4 / SPG);  // first piece and first group of the slice
    const int m0 = blockIdx.y * (16 * RT), M = a.M - m0;  // rows of this workgroup

    // tiles blockIdx.x, + gridDim.x, ... Pieces and groups past K repeat the last ones: X is zero there.
    Slice sl[2];
    const int cl = KC - 1 - c0, bl = B8 - 1 - g0 / 8;
    const int mb = PRE ? min(wave * 4 + q, B8 - 1) : g0 / 8 + min(q, min(Slice::SB - 1, bl));
    auto load = [&](Slice& s, int t) {
        if (t >= tiles) return;
        const u4v* cp = (const u4v*)w.codes + ((size_t)t * KC + c0) * 64 + lane;
        const _Float16* sp = w.scale + ((size_t)t * B8 + g0 / 8) * 128 + r * 8;
#pragma unroll
        for (int c = 0; c < CPS; c++) s.code[c] = __builtin_nontemporal_load(cp + min(c, cl) * 64);
#pragma unroll
        for (int b = 0; b < Slice::SB; b++) s.scale[b] = *(const u4v*)(sp + min(b, bl) * 128);
        s.mins = *(const u4v*)(w.mins + ((size_t)t * B8 + mb) * 128 + r * 8);
    };
    load(sl[0], blockIdx.x);
    load(sl[1], blockIdx.x + gridDim.x);

    // the slice of X: lane (r, q) has k = 32 j + 8 q .. + 7 of the steps j, of row r (PK: of row r % 8)
    half8 xa[RT][NA][ST], xs[PRE ? 1 : RT][NS];
    int e4[PRE ? 1 : RT][4];  // exponents of the rows 4 q + i whose sums this lane holds
    // PRE: the waves' blocks of sums [blocks][RT][2][WAVE], which a tile reads once
    half8* xsl = (half8*)(red_raw + 2 * SUMS * KS * WAVE);
    const int nblocks = a.c0 ? 0 : (d.K / d.G + 31) / 32;
#pragma unroll
    for (int t = 0; t < RT; t++) {
        if constexpr (PRE) {
            const XOps o(a.M, NA, d);
            const size_t mt = min((size_t)(m0 / 16 + t), o.tiles - 1);
            const half8* parts = (const half8*)a.X;
            const half8* sums = (const half8*)((const unsigned char*)a.X + o.sums_at());
#pragma unroll
            for (int n = 0; n < NA; n++)
#pragma unroll
                for (int j = 0; j < ST; j++) xa[t][n][j] = parts[((mt * NA + n) * o.steps + c0 * 4 + j) * 64 + lane];
            if (wave < nblocks) {
#pragma unroll
                for (int n = 0; n < 2; n++)
                    xsl[((wave * RT + t) * 2 + n) * WAVE + lane] = sums[((mt * 2 + n) * o.blocks + wave) * 64 + lane];
            }
            continue;
        }
        const int m = min(PK ? r % 8 : 16 * t + r, M - 1);
        const TX* x = (const TX*)a.X + (size_t)(m0 + m) * a.ldx;
        X8<TX> f[ST];
        float amax = 0.f;
#pragma unroll
        for (int j = 0; j < ST; j++) {
            const int k = c0 * 128 + 32 * j + 8 * q;
            f[j].load(x, k, d.K);
        }
#pragma unroll
        for (int j = 0; j < ST; j++)
#pragma unroll
            for (int i = 0; i < 8; i++) amax = fmaxf(amax, fabsf(f[j].get(i)));
        amax = fmaxf(amax, __shfl_xor(amax, 16, WAVE));
        amax = fmaxf(amax, __shfl_xor(amax, 32, WAVE));
        const int e = row_exp(amax);
#pragma unroll
        for (int i = 0; i < 4; i++) e4[t][i] = 7 - __shfl(e, (4 * q + i) % (PK ? 8 : 16), WAVE);
        float s = 0.f;
        half8 hi{}, lo{};
#pragma unroll
        for (int j = 0; j < ST; j++) {
            half8 l;
            const half8 h = x_parts(f[j], e, F32 ? &l : nullptr);
            if (PK) xa[t][0][j] = r < 8 ? h : l;
            else {
                xa[t][0][j] = h;
                if (NA == 2) xa[t][NA - 1][j] = l;
            }
            s += ((f[j].get(0) + f[j].get(1)) + (f[j].get(2) + f[j].get(3))) + ((f[j].get(4) + f[j].get(5)) + (f[j].get(6) + f[j].get(7)));
            if (j % SPG < SPG - 1) continue;
            // the group's sum, and its place among the 8 of the block that lanes q read the minima of
            s += __shfl_xor(s, 16, WAVE);
            s += __shfl_xor(s, 32, WAVE);
            s = __builtin_ldexpf(s, e - 7);
            const _Float16 sh = (_Float16)s, slo = (_Float16)(s - (float)sh);
            const int g = j / SPG;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const bool here = Slice::GROUPS >= 8 ? g % 8 == i && q == g / 8 : q == 0 && (g0 + g) % 8 == i;
                hi[i] = here ? sh : hi[i];
                lo[i] = here ? slo : lo[i];
            }
            s = 0.f;
        }
        if (PK) xs[t][0] = r < 8 ? hi : lo;
        else xs[t][0] = hi, xs[t][NS - 1] = lo;
    }

    // a tile: this wave's share of its sums, in units of Y
    auto product = [&](const Slice& s, f32x4 (&v)[RT]) {
        f32x4 acc[RT], p[RT];
#pragma unroll
        for (int t = 0; t < RT; t++) acc[t] = p[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < ST; j++) {
            const half8 b = q4_codes(s.code[j / 4][j % 4]);
#pragma unroll
            for (int n = 0; n < NA; n++)
#pragma unroll
                for (int t = 0; t < RT; t++) p[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xa[t][n][j], b, p[t], 0, 0, 0);
            if (j % SPG < SPG - 1) continue;
            const int g = j / SPG;
            uint32_t sw;  // (a slice of 4 or 2 groups begins in the middle of its block)
            if (Slice::GROUPS >= 8) sw = s.scale[g / 8][g % 8 / 2];
            else if (Slice::GROUPS == 4) sw = g0 % 8 ? s.scale[0][2 + g / 2] : s.scale[0][g / 2];
            else if (Slice::GROUPS == 2) sw = s.scale[0][g0 / 2 % 4];
            else sw = s.scale[0][g0 / 2 % 4] >> (16 * (g0 % 2));
            const float sc = (float)__builtin_bit_cast(_Float16, (uint16_t)(Slice::GROUPS > 1 ? sw >> (16 * (g % 2)) : sw));
#pragma unroll
            for (int t = 0; t < RT; t++) {
                acc[t] += p[t] * sc;
                asm volatile("" : "+v"(acc[t]));  // (here, not sunk past the tile with p kept till then)
                p[t] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
            __builtin_amdgcn_sched_barrier(0);  // (codes are unpacked a group at a time: registers)
        }
        const half8 mn = __builtin_bit_cast(half8, s.mins);
#pragma unroll
        for (int t = 0; t < RT; t++) {
            f32x4 am = acc[t] * kCodeUnit;
            if constexpr (PRE) {
                if (wave < nblocks) {
#pragma unroll
                    for (int n = 0; n < 2; n++)
                        am = __builtin_amdgcn_mfma_f32_16x16x32_f16(xsl[((wave * RT + t) * 2 + n) * WAVE + lane], mn, am, 0, 0, 0);
                }
                v[t] = am;
            } else {
#pragma unroll
                for (int n = 0; n < NS; n++) am = __builtin_amdgcn_mfma_f32_16x16x32_f16(xs[t][n], mn, am, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; i++) v[t][i] = __builtin_ldexpf(PK ? pair_sum32(am[i]) : am[i], e4[t][i]);
            }
        }
    };

    auto red = [&](int buf, int i, int k) -> f32x4& { return red_raw[((buf * SUMS + i) * KS + k) * WAVE + lane]; };
    int buf = 0;
    for (int t0 = blockIdx.x; t0 < tiles; t0 += 2 * gridDim.x) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int ct = t0 + h * gridDim.x;  // (the same for all waves)
            if (ct < tiles) {
                f32x4 v[RT];
                product(sl[h], v);
                load(sl[h], ct + 2 * gridDim.x);
#pragma unroll
                for (int t = 0; t < RT; t++) red(buf, h % NB + t, wave) = v[t];
            }
            if (h % NB < NB - 1) continue;
            lds_barrier();  // (the other buffer's readers are past it when they reach the next one)
            // the sums over the waves: lane (r, q) has rows 4 q .. 4 q + 3 of Y's column 16 ct + r
            for (int i = wave; i < SUMS; i += KS) {
                const int t = RT == 1 ? 0 : i, tt = RT == 1 ? t0 + i * gridDim.x : ct, n = tt * 16 + r;
                if (tt >= tiles) break;
                f32x4 v = red(buf, i, 0);
                for (int k = 1; k < KS; k++) v += red(buf, i, k);
                if constexpr (PRE) {  // (one power of two for all slices of a row)
                    const XOps o(a.M, NA, d);
                    const int4 e = *((const int4*)((const unsigned char*)a.X + o.exps_at()) + min((size_t)(m0 / 16 + t), o.tiles - 1) * 4 + q);
                    v = f32x4{__builtin_ldexpf(v[0], 7 - e.x), __builtin_ldexpf(v[1], 7 - e.y), __builtin_ldexpf(v[2], 7 - e.z),
                              __builtin_ldexpf(v[3], 7 - e.w)};
                }
                if (n >= d.N) continue;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int m = 16 * t + 4 * q + j;
                    if (m < M) {
                        float* y = a.Y + (size_t)(m0 + m) * a.ldy + n;
                        *y = a.accumulate ? *y + v[j] : v[j];
                    }
                }
            }
            buf ^= 1;
        }
    }
}

template <typename TX, int SPG, bool PK, int RT, int CPS, int MW, bool PRE>
int launch_stream(const Q4Args& a, hipStream_t st) {
    const int ks = std::min(MW, (a.d.chunks() - a.c0 + CPS - 1) / CPS), tiles = a.d.tiles(), gy = (a.M + 16 * RT - 1) / (16 * RT);
    // 16 waves per CU, or 8 with X's operands in twice the registers; every workgroup as many tiles as the others
    const int cu = PRE ? 8 : 16, most = std::max(1, 256 * std::max(1, cu / ks) / gy), rounds = (tiles + most - 1) / most;
    const int lds = ((RT < 2 ? 4 : 2 * RT) * ks + (PRE ? (a.d.K / a.d.G + 31) / 32 * 2 * RT : 0)) * 1024;
    if (lds > 65536)
        AEG_HIP(hipFuncSetAttribute((const void*)q4_stream_kernel<TX, SPG, PK, RT, CPS, MW, PRE>,
                                    hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    q4_stream_kernel<TX, SPG, PK, RT, CPS, MW, PRE><<<dim3((tiles + rounds - 1) / rounds, gy), ks * WAVE,
                                                      lds, st>>>(a);
    return after_launch("linear_q4");
}

template <typename TX, bool PK, int RT, int CPS, int MW, bool PRE>
int stream_spg(const Q4Args& a, hipStream_t st) {
    switch (a.d.G) {
        case 32: return launch_stream<TX, 1, PK, RT, CPS, MW, PRE>(a, st);
        case 64: return launch_stream<TX, 2, PK, RT, CPS, MW, PRE>(a, st);
        default: return launch_stream<TX, 4, PK, RT, CPS, MW, PRE>(a, st);
    }
}

// ---------------------------------------------------------------------------------------------
// Many rows: tiles of 128 rows of X x 256 of W, 8 waves of 64 x 64. X's operands go from the workspace straight into
// LDS (1 KB pieces as they lie there: no bank conflicts, no swizzle), 128 k to a stage; codes go from global memory to
// registers and are unpacked in the wave that uses them. Both are requested two stages ahead (fp32 X: one, of
// twice the products: LDS). The sums of a group join
// the tile's in fp32 (one FMA per 32 products and lane).
constexpr int GM = 128, GN = 256, GR = 4, GC = 4;  // tile; a wave's 16 x 16 tiles

// 16 bytes per lane straight from global memory into LDS at lds + 16 lane (lds uniform)
__device__ __forceinline__ void q4_g2lds(const void* src, void* lds) {
    __builtin_amdgcn_global_load_lds(src, (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}

template <int P, int SPG>
__global__ void __launch_bounds__(512) q4_gemm_kernel(const Q4Args a, int tiles_m, int tiles_n, int ntiles, int per_xcd) {
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];  // [NB][8 tiles][P][4 steps][1 KB]
    constexpr int NB = 2;  // stages in LDS and registers
    constexpr int BUF = GM / 16 * P * 4 * 1024, GP = 4 / SPG;
    // steps whose products are summed before they are scaled: two of one group, where X's operands leave the registers
    constexpr int U = P == 2 || SPG == 1 ? 1 : 2;
    // consecutive tiles on one XCD: 8 of M beside each other, then along N, so that its workgroups share both in L2
    const int li = (blockIdx.x % 8) * per_xcd + blockIdx.x / 8;
    if (li >= ntiles) return;
    const int gm = li / (8 * tiles_n) * 8, gw = min(8, tiles_m - gm), in = li - gm * tiles_n;
    const int bm = gm + in % gw, bn = in / gw;
    const Q4Dims d = a.d;
    const Q4Ptr w = q4_ptr(a.W, d);
    const XOps o(a.M, P, d);
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int r = lane % 16, q = lane / 16, wm = wave % 2, wn = wave / 2;
    const int KC = d.chunks(), B8 = d.blocks8(), tiles = d.tiles(), xt = (int)o.tiles;

    // this wave's pieces of X per stage: one tile of 16 rows, all its parts and steps
    const unsigned char* xsrc = (const unsigned char*)a.X + ((size_t)min(bm * 8 + wave, xt - 1) * P * o.steps) * 1024 + lane * 16;
    auto stage = [&](int buf, int c) {
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                q4_g2lds(xsrc + ((size_t)p * o.steps + c * 4 + j) * 1024, lds + buf * BUF + ((wave * P + p) * 4 + j) * 1024);
    };
    int nt[GC];
#pragma unroll
    for (int n = 0; n < GC; n++) nt[n] = min(bn * 16 + wn * 4 + n, tiles - 1);
    u4v code[NB][GC];
    u2v sc[NB][GC];
    auto load = [&](int buf, int c) {
#pragma unroll
        for (int n = 0; n < GC; n++) {
            code[buf][n] = ((const u4v*)w.codes)[((size_t)nt[n] * KC + c) * 64 + lane];
            const _Float16* p = w.scale + ((size_t)nt[n] * B8 + c * GP / 8) * 128 + r * 8 + c * GP % 8;
            if (GP == 4) sc[buf][n] = *(const u2v*)p;
            else if (GP == 2) sc[buf][n][0] = *(const uint32_t*)p;
            else sc[buf][n][0] = *(const uint16_t*)p;
        }
    };
#pragma unroll
    for (int c = 0; c < NB - 1; c++)
        if (c < KC) {
            stage(c, c);
            load(c, c);
        }

    // the minima's term first, in the units of the codes' sums
    f32x4 acc[GR][GC];
#pragma unroll
    for (int m = 0; m < GR; m++)
#pragma unroll
        for (int n = 0; n < GC; n++) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    const half8* sums = (const half8*)((const unsigned char*)a.X + o.sums_at());
    for (int b = 0; b < o.blocks; b++) {
        half8 mn[GC];
#pragma unroll
        for (int n = 0; n < GC; n++) mn[n] = *(const half8*)(w.mins + ((size_t)nt[n] * B8 + min(b * 4 + q, B8 - 1)) * 128 + r * 8);
#pragma unroll
        for (int m = 0; m < GR; m++)
#pragma unroll
            for (int p = 0; p < 2; p++) {
                const half8 x = sums[(((size_t)min(bm * 8 + wm * 4 + m, xt - 1) * 2 + p) * o.blocks + b) * 64 + lane];
#pragma unroll
                for (int n = 0; n < GC; n++) acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, mn[n], acc[m][n], 0, 0, 0);
            }
    }
#pragma unroll
    for (int m = 0; m < GR; m++)
#pragma unroll
        for (int n = 0; n < GC; n++) acc[m][n] *= 1.f / kCodeUnit;

    auto step = [&](int buf, int c) {
        // this wave's pieces of stage c are in LDS once only the later stage's loads are in flight
        if (NB == 3 && c + 1 < KC) __builtin_amdgcn_s_waitcnt(0x0f70 | (4 * P + 2 * GC));
        else __builtin_amdgcn_s_waitcnt(0x0f70);
        lds_barrier();  // all waves' are, and all have read stage c - 1
        if (c + NB - 1 < KC) {
            stage((buf + NB - 1) % NB, c + NB - 1);
            load((buf + NB - 1) % NB, c + NB - 1);
        }
        const unsigned char* x = lds + buf * BUF + wm * 4 * P * 4096 + lane * 16;
        half8 xa[2][P][U][GR];
        constexpr int XF = P * U * GR;  // operands of a unit, products of a unit's tile
        auto operand = [&](int u, int i) {
            const int m = i % GR, s = i / GR % U, pt = i / GR / U;
            xa[u % 2][pt][s][m] = *(const half8*)(x + ((m * P + pt) * 4 + u * U + s) * 1024);
        };
        half8 b[2][U];
        auto unpack = [&](int i) {
#pragma unroll
            for (int s = 0; s < U; s++) b[i % 2][s] = q4_codes(code[buf][i % GC][i / GC * U + s]);
        };
        f32x4 p[2][GR];
        auto join = [&](int i) {
            const int u = i / GC, n = i % GC, g = u * U / SPG;
            const float f = (float)__builtin_bit_cast(_Float16, (uint16_t)(sc[buf][n][g / 2] >> (16 * (g % 2))));
#pragma unroll
            for (int m = 0; m < GR; m++) {
                acc[m][n] += p[i % 2][m] * f;
                asm volatile("" : "+v"(acc[m][n]));  // (here, not sunk past the stage with p kept till then)
            }
        };
#pragma unroll
        for (int i = 0; i < XF; i++) operand(0, i);
        unpack(0);
        __builtin_amdgcn_sched_barrier(0);
        // tile i: its products, and between them the codes of the next one, the FMAs of the one before and a share of the
        // next unit's operands
        constexpr int IS = 4 / U * GC;
#pragma unroll
        for (int i = 0; i < IS; i++) {
            const int u = i / GC;
            if (u + 1 < 4 / U) {
#pragma unroll
                for (int k = 0; k < XF / GC; k++) operand(u + 1, i % GC * (XF / GC) + k);
            }
#pragma unroll
            for (int s = 0; s < U; s++)
#pragma unroll
                for (int pt = 0; pt < P; pt++)
#pragma unroll
                    for (int m = 0; m < GR; m++)
                        p[i % 2][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            xa[u % 2][pt][s][m], b[i % 2][s], s == 0 && pt == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : p[i % 2][m], 0, 0, 0);
            if (i + 1 < IS) unpack(i + 1);
            if (i > 0) join(i - 1);
            constexpr int VALU = (7 * U + 4 * GR + 2 + XF - 1) / XF;  // per product
#pragma unroll
            for (int k = 0; k < XF; k++) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                if (k < XF / GC) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, VALU, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        join(IS - 1);
    };
    for (int c = 0; c < KC; c += NB) {
#pragma unroll
        for (int i = 0; i < NB; i++)
            if (c + i < KC) step(i, c + i);
    }

    const int* exps = (const int*)((const unsigned char*)a.X + o.exps_at());
#pragma unroll
    for (int m = 0; m < GR; m++) {
        const int row = bm * GM + (wm * 4 + m) * 16 + 4 * q;
        const int4 e = *(const int4*)(exps + min(row, xt * 16 - 4));
        const int es[4] = {18 - e.x, 18 - e.y, 18 - e.z, 18 - e.w};
#pragma unroll
        for (int n = 0; n < GC; n++) {
            const int col = (bn * 16 + wn * 4 + n) * 16 + r;
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (row + i < a.M && col < d.N) {
                    float* y = a.Y + (size_t)(row + i) * a.ldy + col;
                    const float v = __builtin_ldexpf(acc[m][n][i], es[i]);
                    __builtin_nontemporal_store(a.accumulate ? *y + v : v, y);
                }
        }
    }
}

template <int P, int SPG>
int launch_gemm(const Q4Args& a, hipStream_t st) {
    const int tm = (a.M + GM - 1) / GM, tn = (a.d.N + GN - 1) / GN, n = tm * tn, per = (n + 7) / 8;
    constexpr int lds = 2 * (GM / 16 * P * 4 * 1024);
    if (lds > 65536)
        AEG_HIP(hipFuncSetAttribute((const void*)q4_gemm_kernel<P, SPG>, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    q4_gemm_kernel<P, SPG><<<8 * per, 512, lds, st>>>(a, tm, tn, n, per);
    return after_launch("linear_q4");
}
template <int P>
int gemm_spg(const Q4Args& a, hipStream_t st) {
    switch (a.d.G) {
        case 32: return launch_gemm<P, 1>(a, st);
        case 64: return launch_gemm<P, 2>(a, st);
        default: return launch_gemm<P, 4>(a, st);
    }
}

// Rows of X and K that the stream takes with X's rows as they are, and as operands (K in blocks of 2048, the minima of
// all of it in the first).
bool stream_fits(int M, const Q4Dims& d) { return M <= 16 && d.K <= 4096; }
bool pre_fits(int M, const Q4Dims& d) { return M <= 256 && d.K <= 8192; }

int run_stream(const Q4Args& a, int x_dtype, hipStream_t st) {
    if (x_dtype == AEGIST_BF16) return stream_spg<uint16_t, false, 1, 2, 16, false>(a, st);
    if (a.M <= 8) return stream_spg<float, true, 1, 2, 16, false>(a, st);
    return a.d.K > 2048 ? stream_spg<float, false, 1, 4, 8, false>(a, st) : stream_spg<float, false, 1, 2, 8, false>(a, st);
}

int run_rows(Q4Args a, int x_dtype, void* ws, hipStream_t st) {
    const int tiles = (a.M + 15) / 16;
    if (x_dtype == AEGIST_F32) q4_rows_kernel<float><<<tiles, XW * WAVE, 0, st>>>(a, (unsigned char*)ws);
    else q4_rows_kernel<uint16_t><<<tiles, XW * WAVE, 0, st>>>(a, (unsigned char*)ws);
    int rc = after_launch("linear_q4");
    if (rc) return rc;
    a.X = ws;
    if (!pre_fits(a.M, a.d)) return x_dtype == AEGIST_F32 ? gemm_spg<2>(a, st) : gemm_spg<1>(a, st);
    for (a.c0 = 0; a.c0 < a.d.chunks() && !rc; a.c0 += 16, a.accumulate = 1)
        rc = x_dtype == AEGIST_F32 ? stream_spg<float, false, 2, 2, 8, true>(a, st)
             : a.M <= 32           ? stream_spg<uint16_t, false, 2, 2, 8, true>(a, st)
                                   : stream_spg<uint16_t, false, 4, 2, 8, true>(a, st);
    return rc;
}

}  // namespace

namespace aegist {

size_t linear_q4_workspace(int x_dtype, int M, int N, int K, int G) {
    const Q4Dims d{N, K, G};
    return M == 0 || N == 0 || stream_fits(M, d) ? 0 : XOps(M, x_dtype == AEGIST_F32 ? 2 : 1, d).bytes();
}

int launch_linear_q4(const void* X, int x_dtype, long long ldx, const void* W, float* Y, long long ldy, int M, int N,
                     int K, int G, int accumulate, void* ws, size_t ws_bytes, hipStream_t st) {
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
    const Q4Args a{X, ldx, (const unsigned char*)W, Y, ldy, M, accumulate, d, 0};
    if (stream_fits(M, d)) return run_stream(a, x_dtype, st);
    if ((rc = check_workspace(ws, ws_bytes, linear_q4_workspace(x_dtype, M, N, K, G), "linear_q4"))) return rc;
    return run_rows(a, x_dtype, ws, st);
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
