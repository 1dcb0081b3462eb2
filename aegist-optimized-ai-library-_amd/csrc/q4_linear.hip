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
//     of the codes are exact (error of the product against 64 bits beside a plain fp32 product's, of the 2-norm: at K = 32
//     1.26e-7 and 1.02e-7, from K = 64 on the smaller). What fp16's subnormals cut off, an fp32 value below about 2^-17 of
//     its row's largest to fewer than 22 bits and a bf16 one below about 2^-31 to fewer than 8, is at most 2^-39 of
//     that largest;
//   - the sums of a group's X (fp32, rounded to 22 bits in two fp16 parts) against the minima are one more product
//     with K / G in the place of K.
// A group's products are summed apart and then join the row's sum with the group's scale, in fp32.
#include "q4.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

using namespace aegist;

namespace {

typedef uint32_t u2v __attribute__((ext_vector_type(2)));

// the four fp16 pairs of eight codes, in units of 2^-18
__device__ __forceinline__ half8 q4_codes(uint32_t d) {
    constexpr uint32_t m = 0x03c003c0u;
    return __builtin_bit_cast(half8, u4v{d & m, d << 4 & m, d >> 4 & m, __builtin_amdgcn_alignbit(d, d, 8) & m});
}
// The scale in the low half of w as a float in a register of its own (left to the compiler, every FMA converts it again).
__device__ __forceinline__ float q4_scale(uint32_t w) {
    float f = (float)__builtin_bit_cast(_Float16, (uint16_t)w);
    asm("" : "+v"(f));
    return f;
}
// what undoes the units of the code products (2^-18) beside those of the minima (X's sums in units of 2^7, in which the
// 128 values of a group stay within fp16)
constexpr float kCodeUnit = 0x1p11f, kSumUnit = 0x1p-7f;

// power of two by which a row of X is scaled; 0 for rows without a finite largest value (their outputs are not)
__device__ __forceinline__ int row_exp(float amax) {
    return amax > 0.f && amax < INFINITY ? 14 - ((int)(__float_as_uint(amax) >= 0x00800000u
                                                        ? (__float_as_uint(amax) >> 23) - 127
                                                        : -118 - __builtin_clz(__float_as_uint(amax))))
                                         : 0;
}

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

// Rows of a launch (of more, blocks of so many): their 16-row tiles fit a grid's second dimension, and their operands'
// workspace does not grow further.
constexpr int kMaxRows = 1 << 19;

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
//         from K to a multiple of 128
//   sums  [M / 16][2 parts][K / G / 32][64 lanes][8 fp16]: the sums of the groups 32 b + 8 q .. + 7
//   exps  [M] int: the power of two each row was scaled by
struct XOps {
    int parts, steps, blocks;  // 32 k each, 32 groups each
    size_t tiles;
    __host__ __device__ XOps(int M, int parts, const Q4Dims& d)
        : parts(parts), steps(d.chunks() * 4), blocks((d.K / d.G + 31) / 32), tiles((M + 15) / 16) {}
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
#pragma unroll
            for (int i = 0; i < 8; i++) s += __builtin_ldexpf(f[j].get(i), e);  // (scaled: it cannot overflow)
            parts[(mt * o.parts * o.steps + j0 + j) * 64 + lane] = hi;
            if (F32) parts[((mt * o.parts + 1) * o.steps + j0 + j) * 64 + lane] = lo;
            if ((j + 1) % spg) continue;
            s += __shfl_xor(s, 16, WAVE);
            s += __shfl_xor(s, 32, WAVE);
            s *= kSumUnit;
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
// each); a wave holds its slice of 16 rows of X as matrix operands and takes its pieces of one tile (16 rows of
// W) after the other, the next two in flight; per round of two tiles the waves' sums meet in LDS. So a weight
// is one contiguous 1 KB load and no more, nothing in the loop reads LDS but the sums, and a slice is
// scaled by its own largest value, which needs no exchange between waves.
//
// Waves that staged X in LDS, once per workgroup, and read it back per piece took 16.5 us at 16 rows of 2048 x 4096,
// mostly the staging (two rows per wave one after the other).

// Up to kStaged rows are scaled one after the other, 4 values of the slice per lane, and pass through the wave's own LDS
// into the operands: a lane that makes its operands itself makes those of row min(r, M - 1), the same as the others of that
// row (8192 x 2048, one row: 7.0 us so, 5.7 staged; three rows: no difference).
constexpr int kStaged = 2;
// per wave: rows [M][parts][256 fp16], sums [M][2][8 fp16], exponents [4]
__host__ __device__ constexpr int staged_bytes(int M, int parts) { return M * (parts * 512 + 32) + 16; }

template <int SPG, int CPS>
struct Q4Slice {
    static constexpr int GROUPS = CPS * 4 / SPG;           // groups of a slice
    static constexpr int SB = (GROUPS + 7) / 8;            // blocks of 8 groups that they touch
    u4v code[CPS];
    u4v scale[SB], mins;
};

// SPG: steps of 32 k per group. MW: waves at most. FEW: up to kStaged rows.
template <typename TX, int SPG, int CPS, int MW, bool FEW>
__global__ void __launch_bounds__(MW * WAVE) q4_stream_kernel(const Q4Args a) {
    constexpr bool F32 = std::is_same<TX, float>::value;
    constexpr bool PK = F32 && FEW;  // the two parts of row m as rows m and m + 8 of one operand
    constexpr int NA = F32 && !PK ? 2 : 1, NS = PK ? 1 : 2, ST = CPS * 4;
    typedef Q4Slice<SPG, CPS> Slice;
    extern __shared__ f32x4 red_raw[];  // [2][2 tiles][KS][WAVE]
    const Q4Dims d = a.d;
    const Q4Ptr w = q4_ptr(a.W, d);
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int r = lane % 16, q = lane / 16, KS = blockDim.x / WAVE;
    const int KC = d.chunks(), B8 = d.blocks8(), tiles = d.tiles();
    const int c0 = a.c0 + wave * CPS, g0 = c0 * (4 / SPG);  // first piece and first group of the slice
    const int m0 = blockIdx.y * 16, M = a.M - m0;  // rows of this workgroup

    // tiles blockIdx.x, + gridDim.x, ... Pieces and groups past K repeat the last ones: X is zero there.
    Slice sl[2];
    const int cl = KC - 1 - c0, bl = B8 - 1 - g0 / 8;
    const int mb = g0 / 8 + min(q, min(Slice::SB - 1, bl));
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
    half8 xa[NA][ST], xs[NS];
    int e4[4];  // exponents of the rows 4 q + i whose sums this lane holds
    if constexpr (FEW) {
        static_assert(CPS == 2, "4 values per lane");
        constexpr int PARTS = F32 ? 2 : 1;
        unsigned char* own = (unsigned char*)(red_raw + 4 * KS * WAVE) + wave * staged_bytes(M, PARTS);
        unsigned char *own_s = own + M * PARTS * 512, *own_e = own_s + M * 32;
        const int k = c0 * 128 + 4 * lane, kk = min(k, d.K - 4);
        float f[kStaged][4];
#pragma unroll
        for (int m = 0; m < kStaged; m++) {
            const TX* x = (const TX*)a.X + (size_t)(m0 + min(m, M - 1)) * a.ldx + kk;
            if constexpr (F32) {
                const f32x4 v = *(const f32x4*)x;
#pragma unroll
                for (int i = 0; i < 4; i++) f[m][i] = v[i];
            } else {
                const u2v v = *(const u2v*)x;
                f[m][0] = bf_lo(v[0]), f[m][1] = bf_hi(v[0]), f[m][2] = bf_lo(v[1]), f[m][3] = bf_hi(v[1]);
            }
        }
        if (lane < 8 * M) ((uint32_t*)own_s)[lane] = 0;
        wave_sync();
#pragma unroll
        for (int m = 0; m < kStaged; m++) {
            if (m >= M) break;  // (the same for all lanes)
#pragma unroll
            for (int i = 0; i < 4; i++) f[m][i] = k < d.K ? f[m][i] : 0.f;
            const int e = row_exp(wave_max(fmaxf(fmaxf(fabsf(f[m][0]), fabsf(f[m][1])), fmaxf(fabsf(f[m][2]), fabsf(f[m][3])))));
            half4 hi, lo;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                f[m][i] = __builtin_ldexpf(f[m][i], e);
                hi[i] = (_Float16)f[m][i];
                lo[i] = (_Float16)(f[m][i] - (float)hi[i]);
            }
            *(half4*)(own + m * PARTS * 512 + lane * 8) = hi;
            if (F32) *(half4*)(own + (m * PARTS + 1) * 512 + lane * 8) = lo;
            // the group's sum, from 8, 16 or 32 lanes, to its place among the 8 of its block
            float s = (f[m][0] + f[m][1]) + (f[m][2] + f[m][3]);
#pragma unroll
            for (int o = 1; o < 8 * SPG; o *= 2) s += __shfl_xor(s, o, WAVE);
            s *= kSumUnit;
            const _Float16 sh = (_Float16)s;
            if (lane % (8 * SPG) == 0) {
                const int g = (g0 + lane / (8 * SPG)) % 8;
                ((_Float16*)(own_s + m * 32))[g] = sh;
                ((_Float16*)(own_s + m * 32))[8 + g] = (_Float16)(s - (float)sh);
            }
            if (lane == 0) ((int*)own_e)[m] = e;
        }
        wave_sync();
        const int m = min(PK ? r % 8 : r, M - 1), part = PK ? r / 8 : 0;
#pragma unroll
        for (int n = 0; n < NA; n++)
#pragma unroll
            for (int j = 0; j < ST; j++) xa[n][j] = *(const half8*)(own + (m * PARTS + part + n) * 512 + (32 * j + 8 * q) * 2);
        const half8 none{};
#pragma unroll
        for (int n = 0; n < NS; n++) {
            xs[n] = *(const half8*)(own_s + m * 32 + (part + n) * 16);
            if (q > 0) xs[n] = none;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) e4[i] = 7 - ((const int*)own_e)[min((4 * q + i) % (PK ? 8 : 16), M - 1)];
    } else {
        const int m = min(r, M - 1);
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
        for (int i = 0; i < 4; i++) e4[i] = 7 - __shfl(e, 4 * q + i, WAVE);
        // the groups' sums as products with rows of ones: group g of row r in lane (r, g / 8), the value g % 4 of
        // sums[g % 8 / 4], which is the place that the product with the minima reads it from (a slice of 2 or 4 groups
        // begins within its block of 8)
        constexpr bool WHOLE = Slice::GROUPS >= 8;
        f32x4 sums[2]{};
#pragma unroll
        for (int j = 0; j < ST; j++) {
            half8 lo;
            xa[0][j] = x_parts(f[j], e, F32 ? &lo : nullptr);
            if (F32) xa[NA - 1][j] = lo;
            const int g = j / SPG;
            const uint32_t one = r == (WHOLE ? 4 * (g / 8) + g % 4 : (g0 + g) % 4) ? 0x3c003c00u : 0;
#pragma unroll
            for (int n = 0; n < NA; n++)
                sums[WHOLE ? g % 8 / 4 : 0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                    __builtin_bit_cast(half8, u4v{one, one, one, one}), xa[n][j], sums[WHOLE ? g % 8 / 4 : 0], 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float s = kSumUnit * (WHOLE ? sums[i / 4][i % 4] : i / 4 == g0 % 8 / 4 ? sums[0][i % 4] : 0.f);
            xs[0][i] = (_Float16)s;
            xs[NS - 1][i] = (_Float16)(s - (float)xs[0][i]);
        }
    }

    // a tile: this wave's share of its sums, in units of Y
    auto product = [&](const Slice& s) {
        f32x4 acc{0.f, 0.f, 0.f, 0.f}, p{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < ST; j++) {
            const half8 b = q4_codes(s.code[j / 4][j % 4]);
#pragma unroll
            for (int n = 0; n < NA; n++) p = __builtin_amdgcn_mfma_f32_16x16x32_f16(xa[n][j], b, p, 0, 0, 0);
            if (j % SPG < SPG - 1) continue;
            const int g = j / SPG;
            uint32_t sw;  // (a slice of 4 or 2 groups begins in the middle of its block)
            if (Slice::GROUPS >= 8) sw = s.scale[g / 8][g % 8 / 2];
            else if (Slice::GROUPS == 4) sw = g0 % 8 ? s.scale[0][2 + g / 2] : s.scale[0][g / 2];
            else sw = s.scale[0][g0 / 2 % 4];
            acc += p * q4_scale(sw >> (16 * (g % 2)));
            asm volatile("" : "+v"(acc));  // (here, not sunk past the tile with p kept till then)
            p = f32x4{0.f, 0.f, 0.f, 0.f};
            __builtin_amdgcn_sched_barrier(0);  // (codes are unpacked a group at a time: registers)
        }
        f32x4 v = acc * kCodeUnit;
#pragma unroll
        for (int n = 0; n < NS; n++) v = __builtin_amdgcn_mfma_f32_16x16x32_f16(xs[n], __builtin_bit_cast(half8, s.mins), v, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = __builtin_ldexpf(PK ? pair_sum32(v[i]) : v[i], e4[i]);
        return v;
    };

    auto red = [&](int buf, int i, int k) -> f32x4& { return red_raw[((buf * 2 + i) * KS + k) * WAVE + lane]; };
    int buf = 0;
    for (int t0 = blockIdx.x; t0 < tiles; t0 += 2 * gridDim.x, buf ^= 1) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int ct = t0 + h * gridDim.x;  // (the same for all waves)
            if (ct >= tiles) break;
            red(buf, h, wave) = product(sl[h]);
            load(sl[h], ct + 2 * gridDim.x);
        }
        lds_barrier();  // (the other buffer's readers are past it when they reach the next one)
        // the sums over the waves: lane (r, q) has rows 4 q .. 4 q + 3 of Y's column 16 ct + r
        for (int h = wave; h < 2; h += KS) {
            const int ct = t0 + h * gridDim.x, n = ct * 16 + r;
            if (ct >= tiles) break;
            f32x4 v = red(buf, h, 0);
            for (int k = 1; k < KS; k++) v += red(buf, h, k);
            if (n >= d.N) continue;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int m = 4 * q + j;
                if (m < M) {
                    float* y = a.Y + (size_t)(m0 + m) * a.ldy + n;
                    *y = a.accumulate ? *y + v[j] : v[j];
                }
            }
        }
    }
}

// Tiles that each workgroup takes, one after the other, where a CU holds `per` workgroups and gy of them share a tile: as
// many as fill the chip, every one as many tiles as the others. Workgroups go round the 8 XCDs, so with a multiple of 8
// of them side by side those that share a tile share it in one L2 (160 rows of 8192 x 2048: 26.4 us without).
int stream_rounds(int tiles, int gy, int per, int* gx = nullptr) {
    int most = std::max(1, 256 * per / gy);
    const bool whole = gy > 1 && most >= 8;
    if (whole) most = most / 8 * 8;
    const int rounds = (tiles + most - 1) / most, x = (tiles + rounds - 1) / rounds;
    if (gx) *gx = whole ? (x + 7) / 8 * 8 : x;
    return rounds;
}

template <typename TX, int SPG, int CPS, int MW, bool FEW>
int launch_stream(const Q4Args& a, hipStream_t st) {
    const int ks = std::min(MW, (a.d.chunks() - a.c0 + CPS - 1) / CPS), tiles = a.d.tiles(), gy = (a.M + 15) / 16;
    int gx;
    stream_rounds(tiles, gy, MW / ks, &gx);
    const int lds = 4 * ks * 1024 + (FEW ? ks * staged_bytes(a.M, std::is_same<TX, float>::value ? 2 : 1) : 0);
    if (lds > 65536)
        AEG_HIP(hipFuncSetAttribute((const void*)q4_stream_kernel<TX, SPG, CPS, MW, FEW>,
                                    hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    q4_stream_kernel<TX, SPG, CPS, MW, FEW><<<dim3(gx, gy), ks * WAVE, lds, st>>>(a);
    return after_launch("linear_q4");
}

// K in blocks that the waves' slices hold
template <typename TX, int CPS, int MW, bool FEW = false>
int run_stream(Q4Args a, hipStream_t st) {
    int rc = 0;
    for (a.c0 = 0; a.c0 < a.d.chunks() && !rc; a.c0 += CPS * MW, a.accumulate = 1) switch (a.d.G) {
            case 32: rc = launch_stream<TX, 1, CPS, MW, FEW>(a, st); break;
            case 64: rc = launch_stream<TX, 2, CPS, MW, FEW>(a, st); break;
            default: rc = launch_stream<TX, 4, CPS, MW, FEW>(a, st);
        }
    return rc;
}

int run_stream(const Q4Args& a, int x_dtype, hipStream_t st) {
    const bool few = a.M <= kStaged;
    if (x_dtype == AEGIST_BF16) return few ? run_stream<uint16_t, 2, 16, true>(a, st) : run_stream<uint16_t, 2, 16>(a, st);
    if (few) return run_stream<float, 2, 16, true>(a, st);
    // twice the registers per row: 8 waves
    return a.d.K > 2048 ? run_stream<float, 4, 8>(a, st) : run_stream<float, 2, 8>(a, st);
}

// ---------------------------------------------------------------------------------------------
// Many rows: tiles of 32, 64 or 128 rows of X x 256 of W, 8 waves of 32 columns (so that no two unpack the same codes).
// X's operands go from the workspace straight into LDS (1 KB pieces as they lie there: no bank conflicts, no swizzle),
// 128 k to a stage; codes go from global memory to registers and are unpacked in the wave that uses them. Both are
// requested a stage ahead. The sums of a group join the tile's in fp32 (one FMA per 32 products and lane).
constexpr int GN = 256, GC = 2;  // columns of a tile; a wave's 16-column tiles of them

// 16 bytes per lane straight from global memory into LDS at lds + 16 lane (lds uniform)
__device__ __forceinline__ void q4_g2lds(const void* src, void* lds) {
    __builtin_amdgcn_global_load_lds(src, (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}

// GR: 16-row tiles, of the workgroup and of each wave.
template <int P, int SPG, int GR>
__global__ void __launch_bounds__(512) q4_gemm_kernel(const Q4Args a, int tiles_m, int tiles_n, int ntiles, int per_xcd) {
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];  // [2 stages][GR][P][4 steps][1 KB], exponents [GM]
    constexpr int GM = 16 * GR, BUF = GR * P * 4 * 1024, GP = 4 / SPG;
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
    const int r = lane % 16, q = lane / 16;
    const int KC = d.chunks(), B8 = d.blocks8(), tiles = d.tiles(), xt = (int)o.tiles;

    // this wave's pieces of X per stage
    constexpr int XP = GR * P * 4 / 8;
    const unsigned char* xsrc[XP];
#pragma unroll
    for (int i = 0; i < XP; i++) {
        const int j = wave * XP + i;  // (tile, part, step)
        xsrc[i] = (const unsigned char*)a.X + (((size_t)min(bm * GR + j / (4 * P), xt - 1) * P + j / 4 % P) * o.steps + j % 4) * 1024 + lane * 16;
    }
    auto stage = [&](int buf, int c) {
#pragma unroll
        for (int i = 0; i < XP; i++) q4_g2lds(xsrc[i] + (size_t)c * 4096, lds + buf * BUF + (wave * XP + i) * 1024);
    };
    int nt[GC];
#pragma unroll
    for (int n = 0; n < GC; n++) nt[n] = min(bn * 16 + wave * GC + n, tiles - 1);
    u4v code[2][GC];
    u2v sc[2][GC];
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
    stage(0, 0);
    load(0, 0);
    // (the rows' exponents for the end, where their latency would stand alone)
    int* exps = (int*)(lds + 2 * BUF);
    if (threadIdx.x < GM)
        exps[threadIdx.x] = ((const int*)((const unsigned char*)a.X + o.exps_at()))[min(bm * GM + (int)threadIdx.x, xt * 16 - 1)];

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
                const half8 x = sums[(((size_t)min(bm * GR + m, xt - 1) * 2 + p) * o.blocks + b) * 64 + lane];
#pragma unroll
                for (int n = 0; n < GC; n++) acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, mn[n], acc[m][n], 0, 0, 0);
            }
    }
#pragma unroll
    for (int m = 0; m < GR; m++)
#pragma unroll
        for (int n = 0; n < GC; n++) acc[m][n] *= 1.f / kCodeUnit;

    auto step = [&](int buf, int c) {
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's pieces of stage c are in LDS
        lds_barrier();                       // all waves' are, and all have read stage c - 1
        if (c + 1 < KC) {
            stage(1 - buf, c + 1);
            load(1 - buf, c + 1);
        }
        const unsigned char* x = lds + buf * BUF + lane * 16;
        half8 xa[P][U][GR];
        constexpr int XF = P * U * GR;  // operands of a unit, products of a unit's tile
        auto operand = [&](int u, int s, int pt, int m) {
            xa[pt][s][m] = *(const half8*)(x + ((m * P + pt) * 4 + u * U + s) * 1024);
        };
        half8 b[2][U];
        auto unpack = [&](int i) {
#pragma unroll
            for (int s = 0; s < U; s++) b[i % 2][s] = q4_codes(code[buf][i % GC][i / GC * U + s]);
        };
        f32x4 p[2][GR];
        auto join = [&](int i) {
            const int u = i / GC, n = i % GC, g = u * U / SPG;
            const float f = q4_scale(sc[buf][n][g / 2] >> (16 * (g % 2)));
#pragma unroll
            for (int m = 0; m < GR; m++) {
                acc[m][n] += p[i % 2][m] * f;
                asm volatile("" : "+v"(acc[m][n]));  // (here, not sunk past the stage with p kept till then)
            }
        };
#pragma unroll
        for (int s = 0; s < U; s++)
#pragma unroll
            for (int pt = 0; pt < P; pt++)
#pragma unroll
                for (int m = 0; m < GR; m++) operand(0, s, pt, m);
        unpack(0);
        __builtin_amdgcn_sched_barrier(0);
        // tile i: its products, and between them the codes of the next one, the FMAs of the one before and, in a unit's
        // last tile, the next unit's operands in the place of those just used
        constexpr int IS = 4 / U * GC;
#pragma unroll
        for (int i = 0; i < IS; i++) {
            const int u = i / GC;
            const bool last = i % GC == GC - 1 && u + 1 < 4 / U;
#pragma unroll
            for (int s = 0; s < U; s++)
#pragma unroll
                for (int pt = 0; pt < P; pt++)
#pragma unroll
                    for (int m = 0; m < GR; m++) {
                        p[i % 2][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            xa[pt][s][m], b[i % 2][s], s == 0 && pt == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : p[i % 2][m], 0, 0, 0);
                        if (last) operand(u + 1, s, pt, m);
                    }
            if (i + 1 < IS) unpack(i + 1);
            if (i > 0) join(i - 1);
            constexpr int VALU = (7 * U + 4 * GR + 2 + XF - 1) / XF;  // per product
#pragma unroll
            for (int k = 0; k < XF; k++) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                if (last) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, VALU, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        join(IS - 1);
    };
    for (int c = 0; c < KC; c += 2) {
        step(0, c);
        if (c + 1 < KC) step(1, c + 1);
    }

#pragma unroll
    for (int m = 0; m < GR; m++) {
        const int row = bm * GM + m * 16 + 4 * q;
        const int4 e = *(const int4*)(exps + m * 16 + 4 * q);
        const int es[4] = {18 - e.x, 18 - e.y, 18 - e.z, 18 - e.w};
#pragma unroll
        for (int n = 0; n < GC; n++) {
            const int col = (bn * 16 + wave * GC + n) * 16 + r;
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

template <int P, int SPG, int GR>
int launch_gemm(const Q4Args& a, hipStream_t st) {
    const int tm = (a.M + 16 * GR - 1) / (16 * GR), tn = (a.d.N + GN - 1) / GN, n = tm * tn, per = (n + 7) / 8;
    constexpr int lds = 2 * (GR * P * 4 * 1024) + GR * 64;
    if (lds > 65536)
        AEG_HIP(hipFuncSetAttribute((const void*)q4_gemm_kernel<P, SPG, GR>, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    q4_gemm_kernel<P, SPG, GR><<<8 * per, 512, lds, st>>>(a, tm, tn, n, per);
    return after_launch("linear_q4");
}
template <int P, int GR>
int gemm_spg(const Q4Args& a, hipStream_t st) {
    switch (a.d.G) {
        case 32: return launch_gemm<P, 1, GR>(a, st);
        case 64: return launch_gemm<P, 2, GR>(a, st);
        default: return launch_gemm<P, 4, GR>(a, st);
    }
}

// The kernel of M rows: 0 for the stream, else the GR of the tiles (32, 64 or 128 rows of X x 256 of W), whichever the
// estimate is shortest for (us; fitted to M 64 to 4000, N 512 to 32768, K 512 to 4096; over 176 other sizes of these
// ranges the choice is at most 9% above the fastest). The stream: 1.2 per round of tiles (fp32 X 0.95, 1.4 in slices of
// 512), all rows of X at once. The tiles: rounds of 256 workgroups, each a walk along K; of the small ones, two of a CU
// overlap. Measured (bf16, K = 2048; stream, 32, 64, 128 rows): 1000 rows x 512 12.9, 22.6, 28.8, 43.6; 1000 x 4096
// 46.9, 33.9, 32.9, 45.3; 200 x 8192 31.6, 24.2, 28.6, 41.2; 4000 x 8192 300, 190, 184, 168.
int q4_form(int x_dtype, int M, const Q4Dims& d) {
    if (M <= 16) return 0;
    const bool f32 = x_dtype == AEGIST_F32;
    const int gy = (M + 15) / 16, KC = d.chunks(), cps = f32 && d.K > 2048 ? 4 : 2, mw = f32 ? 8 : 16;
    double best = 7;
    for (int c = 0; c < KC; c += cps * mw) {
        const int per = mw / std::min(mw, (KC - c + cps - 1) / cps), slots = 256 * per;
        best += (double)stream_rounds(d.tiles(), gy, per) * ((gy + slots - 1) / slots) * (f32 ? cps == 4 ? 1.4 : 0.95 : 1.2);
    }
    int form = 0;
    // {before the rounds, per round, per round and 128 k, a further round's share of the first}
    struct Cost { int gr; double base, round, k, more; };
    static constexpr Cost kBf16[3] = {{2, 8, 0.8, 6.9 / 8, 0.8}, {4, 8.5, 2, 10.3 / 8, 1}, {8, 4, 8, 17.5 / 8, 1}};
    static constexpr Cost kF32[3] = {{2, 10, 2, 9.8 / 8, 0.85}, {4, 10, 1, 17.3 / 8, 1}, {8, 4, 13, 28.0 / 8, 1}};
    for (const Cost& c : f32 ? kF32 : kBf16) {
        const double groups = std::ceil(M / (16.0 * c.gr)) * ((d.N + GN - 1) / GN), rounds = std::ceil(groups / 256);
        const double us = c.base + (c.round + c.k * KC) * (1 + c.more * (rounds - 1));
        if (us < best) best = us, form = c.gr;
    }
    return form;
}

int run_gemm(int form, Q4Args a, int x_dtype, void* ws, hipStream_t st) {
    const int tiles = (a.M + 15) / 16;
    if (x_dtype == AEGIST_F32) q4_rows_kernel<float><<<tiles, XW * WAVE, 0, st>>>(a, (unsigned char*)ws);
    else q4_rows_kernel<uint16_t><<<tiles, XW * WAVE, 0, st>>>(a, (unsigned char*)ws);
    int rc = after_launch("linear_q4");
    if (rc) return rc;
    a.X = ws;
    const bool f32 = x_dtype == AEGIST_F32;
    switch (form) {
        case 2: return f32 ? gemm_spg<2, 2>(a, st) : gemm_spg<1, 2>(a, st);
        case 4: return f32 ? gemm_spg<2, 4>(a, st) : gemm_spg<1, 4>(a, st);
        default: return f32 ? gemm_spg<2, 8>(a, st) : gemm_spg<1, 8>(a, st);
    }
}

}  // namespace

namespace aegist {

int linear_q4_form(int x_dtype, int M, int N, int K, int G) { return q4_form(x_dtype, std::min(M, kMaxRows), Q4Dims{N, K, G}); }

size_t linear_q4_workspace(int x_dtype, int M, int N, int K, int G) {
    const Q4Dims d{N, K, G};
    if (N == 0) return 0;
    M = std::min(M, kMaxRows);
    // (what the choice of any smaller M needs is enough for it)
    for (int m = 32; m < M + 16; m += 16)
        if (linear_q4_form(x_dtype, std::min(m, M), N, K, G)) return XOps(M, x_dtype == AEGIST_F32 ? 2 : 1, d).bytes();
    return 0;
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
    // (workgroups read X and W while others write their part of Y)
    const uintptr_t y0 = (uintptr_t)Y, y1 = y0 + ((M - 1) * (size_t)ldy + N) * 4;
    auto meets = [&](const void* p, size_t n) { return (uintptr_t)p < y1 && y0 < (uintptr_t)p + n; };
    if (meets(X, ((M - 1) * (size_t)ldx + K) * xs) || meets(W, d.bytes()))
        return fail(AEGIST_ERR_SHAPE, "linear_q4: Y overlaps X or W");
    for (int m = 0; m < M && !rc; m += std::min(kMaxRows, M - m)) {
        const Q4Args a{(const char*)X + (size_t)m * ldx * xs, ldx, (const unsigned char*)W, Y + (size_t)m * ldy, ldy,
                       std::min(kMaxRows, M - m), accumulate, d, 0};
        const int form = linear_q4_form(x_dtype, a.M, N, K, G);
        if (!form) rc = run_stream(a, x_dtype, st);
        else if (!(rc = check_workspace(ws, ws_bytes, XOps(a.M, x_dtype == AEGIST_F32 ? 2 : 1, d).bytes(), "linear_q4")))
            rc = run_gemm(form, a, x_dtype, ws, st);
    }
    return rc;
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
