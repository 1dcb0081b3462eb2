// Log probabilities of given tokens, the entropy and the most probable tokens of each row of logits, and the
// same straight from hidden rows and an output head.
//
//   m = max x,  z = sum e^(x - m),  logprob = x[token] - m - ln z,  entropy = ln z - sum e^(x - m) (x - m) / z
//
// (the entropy's sum is taken over x - m, not x, so that a common offset of the logits costs no digits). Exponentials are
// the hardware's 2^y of the rounded product y = (x - m) log2 e: an error of |x - m| 2^-24 and an ulp in a term, where a
// library exponential has an ulp or two; it is felt below an ulp of the log probability. Logits
// of -inf have no probability; a row of nothing else has logprob -inf for every token and entropy 0. NaN or
// +inf anywhere in a row makes its logprobs and entropy NaN.
//
// One pass: a workgroup holds a segment of a row in registers, so the maximum, the sums relative to it and the
// selection of the alternatives read it from there. Segments of a row are joined by their maxima in fixed order; few
// long rows are cut into splits, which a second launch joins.
//
// Bound by HBM for many rows of fp32 (2000 x 131072, 8 alternatives: 163 to 170 us, 6.2 to 6.4 TB/s with part of it in the
// last-level cache; without alternatives 165), by a segment's arithmetic, with nothing requested beside it, for as
// many of bf16 (the same size 125 to 130, without alternatives 103), by the latency of a launch or two for few: 61 rows of
// 100003 in bf16 take 10.6 us, with 5 alternatives 15.2.
#include "logprobs.h"
#include "q4.h"

#include <algorithm>

using namespace aegist;

namespace aegist {
int launch_proj(const void* X, int x_dtype, long long ldx, const void* W, int w_dtype, const uint16_t* scale, float* Y,
                long long ldy, int M, int N, int K, int accumulate, hipStream_t st);
bool proj_is_gemm_bf16(const void* X, int x_dtype, long long ldx, const void* W, int w_dtype, const uint16_t* scale, int M,
                       int N, int K);
int launch_gemm_bf16_stats(const uint16_t* X, long long ldx, const uint16_t* W, int M, int N, int K, const RowStats& stats,
                           hipStream_t st);
}

namespace {

constexpr int MAX_TOP = 64;
constexpr int MAX_V = 1 << 30;           // (a logit's index plus a segment stays an int)
constexpr int NT = 256, NW = NT / WAVE;  // threads, waves
constexpr int CAP = 512;                 // candidates that are ranked at once

__device__ __forceinline__ float lp_key_value(u64 k) {
    const uint32_t b = (uint32_t)(k >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ u64 max64(u64 a, u64 b) { return a > b ? a : b; }
__device__ __forceinline__ u64 wave_max64(u64 k) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) k = max64(k, __shfl_xor(k, o, WAVE));
    return k;
}

struct LogprobOut {
    const int* tokens;
    float *logprob, *entropy;
    int* top_ids;
    float* top_logprobs;
    int top;
};

__host__ __device__ inline size_t parts_bytes(int T, int splits, int top) {
    return ((size_t)T * splits * (sizeof(Part) + (size_t)top * sizeof(u64)) + 255) / 256 * 256;
}

__device__ __forceinline__ void join(Part& a, const Part& b) {
    const float m = fmaxf(a.m, b.m);
    // (a side that is empty, or any side of a bad row, is not scaled: no inf - inf)
    const float da = a.m == m ? 0.f : a.m - m, db = b.m == m ? 0.f : b.m - m;
    const float fa = a.m == -INFINITY ? 0.f : expf(da), fb = b.m == -INFINITY ? 0.f : expf(db);
    // s = sum e^(x - m') (x - m'), moved to m: e^d (s + d z)
    const float sa = fa > 0.f ? fa * fmaf(da, a.z, a.s) : 0.f, sb = fb > 0.f ? fb * fmaf(db, b.z, b.s) : 0.f;
    a.z = fa * a.z + fb * b.z;
    a.s = sa + sb;
    a.m = m;
    a.tok = b.tok > a.tok || b.tok != b.tok ? b.tok : a.tok;  // (-inf where the token is not)
    a.bad |= b.bad;
}

__device__ __forceinline__ void finish(const LogprobOut& o, int t, int V, const Part& p) {
    const bool bad = p.bad, empty = p.m == -INFINITY;
    const float lz = bad ? __builtin_nanf("") : logf(p.z);
    const int tok = o.tokens[t];
    float lp = tok < 0 ? 0.f : __builtin_nanf("");
    if (tok >= 0 && tok < V && !bad) lp = empty ? -INFINITY : p.tok - p.m - lz;
    o.logprob[t] = lp;
    o.entropy[t] = empty && !bad ? 0.f : lz - p.s / p.z;
}
__device__ __forceinline__ void finish_top(const LogprobOut& o, int t, int j, const Part& p, u64 key) {
    o.top_ids[(size_t)t * o.top + j] = (int)~(uint32_t)key;
    o.top_logprobs[(size_t)t * o.top + j] = p.bad              ? __builtin_nanf("")
                                            : p.m == -INFINITY ? -INFINITY
                                                               : lp_key_value(key) - p.m - logf(p.z);
}

// 4 consecutive logits. again(): what follows takes them from these registers anew (bf16 values would be kept unpacked as
// floats beside them, twice the registers)
template <typename T> struct L4;
template <> struct L4<float> {
    typedef float v __attribute__((ext_vector_type(4), aligned(4)));
    v x;
    __device__ __forceinline__ void load(const float* p) { x = __builtin_nontemporal_load((const v*)p); }
    __device__ __forceinline__ float get(int i) const { return x[i]; }
    __device__ __forceinline__ void set(int i, float f) { x[i] = f; }
    __device__ __forceinline__ void again() {}
};
template <> struct L4<uint16_t> {
    typedef uint32_t v __attribute__((ext_vector_type(2), aligned(2)));
    v x;
    __device__ __forceinline__ void load(const uint16_t* p) { x = __builtin_nontemporal_load((const v*)p); }
    __device__ __forceinline__ float get(int i) const { return i % 2 ? bf_hi(x[i / 2]) : bf_lo(x[i / 2]); }
    __device__ __forceinline__ void set(int i, float f) {
        const uint32_t h = __float_as_uint(f) >> 16;  // (a bf16 value)
        x[i / 2] = i % 2 ? (x[i / 2] & 0xffffu) | h << 16 : (x[i / 2] & 0xffff0000u) | h;
    }
    __device__ __forceinline__ void again() { asm volatile("" : "+v"(x)); }
};

struct Lds {
    float red[3][NW];
    Part part[NW];
    u64 key[NW];
    uint32_t thr[2][NW];
    int count;
    u64 cand[CAP + MAX_TOP];   // candidates, after the alternatives so far
    u64 list[MAX_TOP];         // the alternatives so far, descending
};

// (fmaxf would first make a quiet NaN of every value, an instruction each)
__device__ __forceinline__ float max3(float a, float b, float c) {
    asm("v_max3_f32 %0, %0, %1, %2" : "+v"(a) : "v"(b), "v"(c));
    return a;
}

// Largest value of the wave by DPP steps (as wave_sum_dpp), in every lane
__device__ __forceinline__ float wave_max_dpp(float v) {
#define AEG_DPP_MAX(CTRL, ROWS) \
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), CTRL, ROWS, 0xF, false)))
    AEG_DPP_MAX(0x111, 0xF);  // row_shr:1
    AEG_DPP_MAX(0x112, 0xF);
    AEG_DPP_MAX(0x114, 0xF);
    AEG_DPP_MAX(0x118, 0xF);
    AEG_DPP_MAX(0x142, 0xA);  // row_bcast:15 to rows 1 and 3
    AEG_DPP_MAX(0x143, 0xC);  // row_bcast:31 to rows 2 and 3
#undef AEG_DPP_MAX
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), WAVE - 1));
}
// The same of unsigned values
__device__ __forceinline__ uint32_t wave_umax_dpp(uint32_t v) {
#define AEG_DPP_MAX(CTRL, ROWS) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, ROWS, 0xF, false))
    AEG_DPP_MAX(0x111, 0xF);
    AEG_DPP_MAX(0x112, 0xF);
    AEG_DPP_MAX(0x114, 0xF);
    AEG_DPP_MAX(0x118, 0xF);
    AEG_DPP_MAX(0x142, 0xA);
    AEG_DPP_MAX(0x143, 0xC);
#undef AEG_DPP_MAX
    return (uint32_t)__builtin_amdgcn_readlane((int)v, WAVE - 1);
}

// Bounds from below of the `top`-th largest of a workgroup's values, where v is the largest of a lane's, as the upper
// halves of keys (0: below all). A wave's top-th largest lane is one: so many values of the wave are at or above it. The
// smallest, over the waves, of their (top / NW)-th largest is another, closer one where values are spread evenly
// (one row of 4000, 20 alternatives: 30 candidates are left instead of 80). Each wave leaves both in LDS. A few are taken
// by maxima one after the other, more by the ranks of all lanes (61 rows of 100003 bf16, 5 alternatives: 14.2 us, by ranks
// 16.7; 1 row of 131072 with 12 10.9 by ranks, 11.2).
constexpr int kFewTop = 8;
__device__ __forceinline__ void bound_part(Lds& s, uint32_t v, int top, int lane, int wave) {
    const int share = (top + NW - 1) / NW;
    uint32_t nth, part = 0;
    if (top <= kFewTop) {
        uint32_t rest = v;
        int n = 0;  // lanes so far
        do {
            nth = wave_umax_dpp(rest);
            const bool is = rest == nth;
            if (n < share) part = nth;
            n += (int)__popcll(__ballot(is));
            rest = is ? 0 : rest;
        } while (n < top);
    } else {
        int r = 0;
#pragma unroll 16
        for (int j = 0; j < WAVE; j++) r += (uint32_t)__builtin_amdgcn_readlane((int)v, j) > v;
        nth = ~wave_umax_dpp(r < top ? ~v : 0);
        part = ~wave_umax_dpp(r < share ? ~v : 0);
    }
    if (lane == 0) s.thr[0][wave] = nth, s.thr[1][wave] = part;
}
__device__ __forceinline__ uint32_t bound(const Lds& s) {
    uint32_t a = s.thr[0][0], b = s.thr[1][0];
#pragma unroll
    for (int w = 1; w < NW; w++) a = max(a, s.thr[0][w]), b = min(b, s.thr[1][w]);
    return max(a, b);
}

__device__ __forceinline__ void add_candidate(Lds& s, u64 k) {
    const int at = atomicAdd(&s.count, 1);
    if (at < CAP + MAX_TOP) s.cand[at] = k;
}

// Places for a wave's n candidates, behind the ones that are there already, in any order (they are ranked). -1 if there are
// more than are ranked (the count says so).
__device__ __forceinline__ int candidate_places(Lds& s, int n, int lane) {
    int at = 0;
    if (lane == 0) at = atomicAdd(&s.count, n);
    at = __builtin_amdgcn_readfirstlane(at);
    return at + n <= CAP + MAX_TOP ? at : -1;
}
__device__ __forceinline__ int lanes_below(u64 b) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0));
}

// The candidates among a segment's logits: those at or above thr. Few lanes hold any. Up to HITS of those
// at a time lay all their logits down in LDS, and the wave looks at 64 of them at once: a test and a branch per
// register would be paid by every wave that holds a single one. (1703 rows of 38708 bf16, 20 alternatives: 57 us (60 on other cards) with
// 4 lanes of 64 logits at a time, 64 with 2, 63 with 8.)
template <int VPT>
struct alignas(16) Hits {
    static constexpr int LANES = VPT == 4 ? 8 : 4, EACH = 4 * VPT, ROW = EACH + 4, J = LANES * EACH / WAVE;  // (rows 16 bytes apart in the banks)
    float x[LANES][ROW];
    int c[LANES];
};
template <int VPT, typename V>
__device__ __forceinline__ void add_candidates(Lds& s, Hits<VPT>& hits, const V (&v)[VPT], float mt, float thr, int c, int c1,
                                               int lane) {
    typedef Hits<VPT> H;
    u64 todo = __ballot(mt >= thr);
    while (todo) {
        const int at = lanes_below(todo), cnt = min((int)__popcll(todo), H::LANES);
        const bool mine = (todo >> lane & 1) && at < H::LANES;
        if (mine) {
#pragma unroll
            for (int i = 0; i < VPT; i++)
                *(f32x4*)&hits.x[at][4 * i] = f32x4{v[i].get(0), v[i].get(1), v[i].get(2), v[i].get(3)};
            hits.c[at] = c;
        }
        todo &= ~__ballot(mine);
        wave_sync();
        u64 key[H::J], is[H::J];
        int n = 0;
#pragma unroll
        for (int j = 0; j < H::J; j++) {
            const int id = lane + WAVE * j, h = id / H::EACH, k = id % H::EACH;
            const float f = hits.x[h][k];
            const int ce = hits.c[h] + 4 * NT * (k / 4) + k % 4;
            key[j] = lp_key(f, ce);
            is[j] = __ballot(h < cnt && ce < c1 && f >= thr);
            n += (int)__popcll(is[j]);
        }
        int to = candidate_places(s, n, lane);
        if (to < 0) return;
#pragma unroll
        for (int j = 0; j < H::J; j++) {
            if (is[j] >> lane & 1) s.cand[to + lanes_below(is[j])] = key[j];
            to += (int)__popcll(is[j]);
        }
        wave_sync();  // (the next ones' logits go where these were read)
    }
}

// the `top` largest of n <= CAP + MAX_TOP keys (all different, or 0) into the list, descending
__device__ __forceinline__ void rank_keys(Lds& s, int n, int top) {
    for (int i = threadIdx.x; i < n; i += NT) {
        const u64 k = s.cand[i];
        int r = 0;
#pragma unroll 8
        for (int j = 0; j < n; j++) r += s.cand[j] > k;
        if (r < top && k) s.list[r] = k;
    }
}

// The `top` largest of the list's `have` keys and the N keys that each thread gives (0: none), into the list. All
// threads call it; returns how many there are. Where the bound leaves too many (values all alike or in order), the
// largest is taken one after the other.
template <int N, int UNROLL, typename Key>
__device__ __forceinline__ int select_keys(Lds& s, int have, int top, Key key) {
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
    u64 k = 0;
#pragma unroll UNROLL
    for (int i = 0; i < N; i++) k = max64(k, key(i));
    if (top == 1) {  // (the largest, without a bound)
        k = wave_max64(k);
        if (lane == 0) s.key[wave] = k;
        __syncthreads();
        k = max64(max64(s.key[0], s.key[1]), max64(s.key[2], s.key[3]));
        if (threadIdx.x == 0) s.list[0] = have ? max64(k, s.list[0]) : k;
        __syncthreads();
        return have || k;
    }
    __syncthreads();
    bound_part(s, (uint32_t)(k >> 32), top, lane, wave);
    if ((int)threadIdx.x < have) s.cand[threadIdx.x] = s.list[threadIdx.x];
    if (threadIdx.x == 0) s.count = have;
    __syncthreads();
    u64 thr = max64((u64)bound(s) << 32, have == top ? max64(s.list[top - 1], 1) : 1);
    if (k >= thr) {
#pragma unroll UNROLL
        for (int i = 0; i < N; i++) {
            const u64 ki = key(i);
            if (ki >= thr) add_candidate(s, ki);
        }
    }
    __syncthreads();
    const int n = s.count;
    if (n <= CAP + MAX_TOP) {
        rank_keys(s, n, top);
        have = min(top, n);
    } else {
        u64 last = ~0ull;
        const u64 mine = (int)threadIdx.x < have ? s.cand[threadIdx.x] : 0;
        for (int j = 0; j < top; j++) {
            u64 best = mine < last ? mine : 0;
#pragma unroll UNROLL
            for (int i = 0; i < N; i++) {
                const u64 ki = key(i);
                if (ki < last) best = max64(best, ki);
            }
            best = wave_max64(best);
            __syncthreads();
            if (lane == 0) s.key[wave] = best;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < NW; w++) best = max64(best, s.key[w]);
            if (threadIdx.x == 0) s.list[j] = best;
            last = best;
        }
        have = top;
    }
    __syncthreads();
    return have;
}

// A workgroup's items: rows x splits, each `span` logits (the last fewer) in segments of 4 VPT NT. With one split the
// outputs are written here.
template <typename T, int VPT>
__global__ void __launch_bounds__(NT) logprobs_kernel(const T* __restrict__ L, long long ld, int rows, int V, int span,
                                                      int splits, Part* __restrict__ parts, u64* __restrict__ tops,
                                                      const LogprobOut o) {
    __shared__ Lds s;
    __shared__ Hits<VPT> hits[NW];
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE, top = o.top;
    constexpr int SEG = 4 * VPT * NT;
    constexpr float LOG2E = 1.44269504f, LN2 = 0.693147181f;
    for (long long item = blockIdx.x; item < (long long)rows * splits; item += gridDim.x) {
        const int t = (int)(item / splits), sp = (int)(item % splits);
        const int c0 = sp * span, c1 = min(V, c0 + span);
        const T* x = L + (size_t)t * ld;
        const int tok = o.tokens[t];
        Part p{-INFINITY, 0.f, 0.f, -INFINITY, 0, {}};
        int have = 0;  // alternatives so far (the same in all threads)
        for (int b = c0; b < c1; b += SEG) {
            L4<T> v[VPT];
            // the thread's logits: b + 4 (NT i + thread) ..
            const T* xb = x + b;
            uint32_t at = 4 * threadIdx.x;
            asm volatile("" : "+v"(at));  // (VPT offsets are not worth registers for the whole loop)
            const int c = b + (int)at;
            if (b + SEG <= c1) {
#pragma unroll
                for (int i = 0; i < VPT; i++) v[i].load(xb + 4 * NT * i + at);
            } else {
                // the last segment: whole fours as above, then the one that the end cuts, -inf past it
                const uint32_t n = c1 - b, whole = n & ~3u;
                L4<T> rest;
#pragma unroll
                for (int e = 0; e < 4; e++) rest.set(e, whole + e < n ? Act<T>::ld(xb, min(whole + e, n - 1)) : -INFINITY);
#pragma unroll
                for (int i = 0; i < VPT; i++) {
                    const uint32_t k = at + 4 * NT * i;
#pragma unroll
                    for (int e = 0; e < 4; e++) v[i].set(e, -INFINITY);
                    if (k < whole) v[i].load(xb + 4 * NT * i + at);
                    else if (k == whole) v[i] = rest;
                }
            }
            if (b == c0 && tok >= c0 && tok < c1) p.tok = Act<T>::ld(x, tok);  // (with the segment's, not after it)
            float mt = -INFINITY;  // the thread's largest (quiet NaN apart)
#pragma unroll
            for (int i = 0; i < VPT; i++)
                mt = max3(max3(mt, v[i].get(0), v[i].get(1)), v[i].get(2), v[i].get(3));
#pragma unroll
            for (int i = 0; i < VPT; i++) v[i].again();
            const float mw = wave_max_dpp(mt);
            if (lane == 0) s.red[0][wave] = mw;
            __syncthreads();
            const float m = fmaxf(fmaxf(s.red[0][0], s.red[0][1]), fmaxf(s.red[0][2], s.red[0][3]));
            // e^(x - m) = 2^y. The entropy's y is held at -200, so that a masked logit's term is 0, not 0 times -inf;
            // NaN reaches z.
            const float mz = m > -INFINITY ? m : 0.f;
            Part q{m, 0.f, 0.f, -INFINITY, !(m < INFINITY), {}};
            if (m < INFINITY) {
                float z[2] = {0.f, 0.f}, y2[2] = {0.f, 0.f};
#pragma unroll
                for (int i = 0; i < VPT; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float y = (v[i].get(e) - mz) * LOG2E, ex = __builtin_amdgcn_exp2f(y);
                        z[e % 2] += ex;
                        y2[e % 2] = __builtin_fmaf(ex, fmaxf(y, -200.f), y2[e % 2]);
                    }
                q.z = z[0] + z[1];
                q.s = (y2[0] + y2[1]) * LN2;
#pragma unroll
                for (int i = 0; i < VPT; i++) v[i].again();
            }
            q.z = wave_sum_dpp(q.z);
            q.s = wave_sum_dpp(q.s);
            if (lane == 0) s.red[1][wave] = q.z, s.red[2][wave] = q.s;
            if (threadIdx.x == 0) s.count = have;
            // the alternatives' lower bound: from the first segment's lanes (of one: the maximum), then from the list
            if (top > 1 && have < top) bound_part(s, (uint32_t)(lp_key(mt, 0) >> 32), top, lane, wave);
            __syncthreads();
            q.z = (s.red[1][0] + s.red[1][1]) + (s.red[1][2] + s.red[1][3]);
            q.s = (s.red[2][0] + s.red[2][1]) + (s.red[2][2] + s.red[2][3]);
            if (!(q.z < INFINITY)) q.bad = 1;
            const uint32_t most = (uint32_t)(lp_key(m, 0) >> 32);
            if (top && (have < top || q.bad || most > (uint32_t)(s.list[top - 1] >> 32))) {
                // later tokens lose ties with the list's, so after it come values above its last. Where fewer logits than
                // asked for are not masked, those are all of them and masked ones of the lowest tokens: of the first 2
                // top, at least top are
                uint32_t low = have == top ? (uint32_t)(s.list[top - 1] >> 32) : top == 1 ? most : bound(s);
                const bool masked = have < top && low == (uint32_t)(lp_key(-INFINITY, 0) >> 32);
                if (have == top || masked) low++;
                const float thr = lp_key_value((u64)low << 32);  // (past +inf: NaN, which nothing is above)
                if ((int)threadIdx.x < have) s.cand[threadIdx.x] = s.list[threadIdx.x];
                if (masked) {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (4 * (int)threadIdx.x + e < 2 * top && c + e < c1 && v[0].get(e) == -INFINITY)
                            add_candidate(s, lp_key(-INFINITY, c + e));
                }
                add_candidates(s, hits[wave], v, mt, thr, c, c1, lane);
                __syncthreads();
                int n = s.count, least = 0;
                if (n > CAP + MAX_TOP && have < top && !q.bad) {
                    // too many, as where masks are the type's lowest value: values above the bound, and of those equal to
                    // it the ones among the first 2 top tokens, which are the lowest, if that makes enough. (Read
                    // again. 1000 rows of 32768 with all but 16 masked, 20 alternatives: 55 us, by maxima one after the other
                    // 503, masked with -inf 28.)
                    __syncthreads();
                    if (threadIdx.x == 0) s.count = have;
                    __syncthreads();
#pragma unroll 4
                    for (int i = 0; i < 4 * VPT; i++) {
                        const int ce = c + 4 * NT * (i / 4) + i % 4;
                        const u64 k = ce < c1 ? lp_key(Act<T>::ld(x, ce), ce) : 0;
                        if ((uint32_t)(k >> 32) > low || ((uint32_t)(k >> 32) == low && ce - b < 2 * top)) add_candidate(s, k);
                    }
                    __syncthreads();
                    n = s.count;
                    least = min(top, c1 - b);
                }
                if (n >= least && n <= CAP + MAX_TOP && !q.bad) {  // (NaN comes first, and no float comparison finds it)
                    if (n > have) rank_keys(s, n, top);
                    have = min(top, n);
                } else {
                    // (read again: keys of a whole segment would take two registers per logit)
                    have = select_keys<4 * VPT, 1>(s, have, top, [&](int i) {
                        const int ce = c + 4 * NT * (i / 4) + i % 4;
                        return ce < c1 ? lp_key(Act<T>::ld(x, ce), ce) : 0;
                    });
                }
            }
            join(p, q);
        }
        if (top) __syncthreads();
        if (splits == 1) {
            if (threadIdx.x == 0) finish(o, t, V, p);
            if ((int)threadIdx.x < top) finish_top(o, t, threadIdx.x, p, s.list[threadIdx.x]);
        } else {
            const size_t at = (size_t)item;
            if (threadIdx.x == 0) parts[at] = p;
            if ((int)threadIdx.x < top) tops[at * top + threadIdx.x] = (int)threadIdx.x < have ? s.list[threadIdx.x] : 0;
        }
    }
}

// One workgroup per row joins its splits: each thread's in order, then all lanes' in a fixed tree.
__global__ void __launch_bounds__(NT) logprobs_join_kernel(const Part* __restrict__ parts, const u64* __restrict__ tops,
                                                           int rows, int V, int splits, const LogprobOut o) {
    __shared__ Lds s;
    constexpr int N = 4;
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
    for (int t = blockIdx.x; t < rows; t += gridDim.x) {
        const u64* keys = tops + (size_t)t * splits * o.top;
        const int n = splits * o.top;
        u64 k[N];  // the first block's, requested with the parts
#pragma unroll
        for (int i = 0; i < N; i++) k[i] = (int)threadIdx.x + NT * i < n ? keys[threadIdx.x + NT * i] : 0;
        Part p{-INFINITY, 0.f, 0.f, -INFINITY, 0, {}};
        for (int i = threadIdx.x; i < splits; i += NT) join(p, parts[(size_t)t * splits + i]);
        const float m = wave_max_dpp(p.m), f = p.m == -INFINITY ? 0.f : p.m == m ? 1.f : expf(p.m - m);
        p.s = wave_sum_dpp(f > 0.f ? f * fmaf(p.m - m, p.z, p.s) : 0.f);
        p.z = wave_sum_dpp(f * p.z);
        p.tok = wave_max_dpp(p.tok);
        p.bad = __any(p.bad);
        p.m = m;
        if (splits > WAVE) {
            if (lane == 0) s.part[wave] = p;
            __syncthreads();
            p = s.part[0];
#pragma unroll
            for (int w = 1; w < NW; w++) join(p, s.part[w]);
        }
        if (threadIdx.x == 0) finish(o, t, V, p);
        if (o.top) {
            int have = 0;
            for (int b = 0; b < n; b += N * NT) {
                if (b > 0) {
#pragma unroll
                    for (int i = 0; i < N; i++) k[i] = b + (int)threadIdx.x + NT * i < n ? keys[b + threadIdx.x + NT * i] : 0;
                }
                have = select_keys<N, N>(s, have, o.top, [&](int i) { return k[i]; });
            }
            if ((int)threadIdx.x < o.top) finish_top(o, t, threadIdx.x, p, s.list[threadIdx.x]);
        }
        __syncthreads();
    }
}

// fp32 rows [rows, K] (K a multiple of 16) as A + R, A the first 16 bits of each value and R the other 8, which bf16 holds:
// the projections of several rows count an fp32 value with 16 bits, so A's product is one of all its bits and R's adds the
// rest. (An infinity leaves a NaN in R.)
template <typename TR>
__global__ void __launch_bounds__(256) split_rows_kernel(const float* __restrict__ X, long long ldx, int rows, int K,
                                                         float* __restrict__ A, TR* __restrict__ R) {
    const int k4 = K / 4;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < (size_t)rows * k4; i += (size_t)gridDim.x * 256) {
        const f32x4 x = *(const f32x4*)(X + (i / k4) * ldx + i % k4 * 4);
        f32x4 a, r;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            a[e] = __uint_as_float(__float_as_uint(x[e]) & 0xffffff00u);
            r[e] = x[e] - a[e];  // (exact)
        }
        *(f32x4*)(A + i * 4) = a;
        if constexpr (sizeof(TR) == 4) {
            *(f32x4*)(R + i * 4) = r;
        } else {
            uint32_t h[4];
#pragma unroll
            for (int e = 0; e < 4; e++) h[e] = __float_as_uint(r[e]) >> 16;
            *(uint2*)(R + i * 4) = uint2{h[0] | h[1] << 16, h[2] | h[3] << 16};
        }
    }
}

// Y += Z over n values
__global__ void __launch_bounds__(256) add_logits_kernel(float* __restrict__ Y, const float* __restrict__ Z, size_t n) {
    typedef L4<float>::v v4;
    for (size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (size_t)gridDim.x * 1024) {
        if (i + 4 <= n) {
            *(v4*)(Y + i) += *(const v4*)(Z + i);
        } else {
            for (size_t j = i; j < n; j++) Y[j] += Z[j];
        }
    }
}

int check_out(const char* who, int T, int V, const LogprobOut& o) {
    const std::string w(who);
    if (T < 0 || V < 1 || V > MAX_V)
        return fail(AEGIST_ERR_SHAPE, w + ": negative size, or a vocabulary of none or more than 2^30 tokens");
    if (o.top < 0 || o.top > MAX_TOP || o.top > V)
        return fail(AEGIST_ERR_SHAPE, w + ": 0 to 64 alternatives, no more than the vocabulary has");
    if (T == 0) return 0;
    if (!o.tokens || !o.logprob || !o.entropy || (o.top && (!o.top_ids || !o.top_logprobs)))
        return fail(AEGIST_ERR_SHAPE, w + ": null operand");
    return 0;
}

// How T rows are taken: segments of 1024 vpt logits, `splits` of `span` logits.
//   - up to 8192 logits: one workgroup per row, small segments (1 row of 8000, 20 alternatives: 8.8 us, large segments
//     9.5, two splits 10.3; 1000 rows with 5: 12, 14, 18);
//   - up to 16384, and 32768 from 128 rows on: one workgroup per row, large segments (1 row of 16000 with 20: 9.1 us and one
//     launch, four splits 11.2 and two launches; 200 rows of 32768 with 5: 13.0, in 8 splits 15.4. But 1 row of 32000
//     with 20: 14.4, in 8 splits 11.0);
//   - longer rows, fewer than 384: so many splits that about 1536 workgroups share them (6 per CU); of the small
//     segments if those are up to 8192 logits (1 row of 131072 with 20: 11.9 us, in 8 large splits 15.3);
//   - more rows: one workgroup each. Without alternatives and with 5, against 3 or 4 splits, us:
//       rows x logits   384 x 40000         450 x 100003        512 x 262144        384 x 2^20          600 x 2^20
//       fp32            16, 22 (17, 23)     34, 43 (39, 44)     86, 89 (88, 96)     237, 273 (240, 245) 447, 440 (388, 394)
//       bf16            16, 23 (16, 22)     35, 46 (35, 46)     65, 84 (64, 81)     233, 269 (159, 186) 309, 340 (246, 284)
//     At 700 x 40000 it is 24, 27 (29, 37). What it costs: bf16 rows longer than about 200000 at up to 700 rows (700 x 2^20:
//     317, 343 against 289, 320), where a workgroup's segments follow one another by their latency.
struct Form {
    int vpt, span, splits;
};
Form form_of(int T, int V) {
    auto cut = [&](int vpt, long long want) {
        const int seg = 4 * vpt * NT;
        const long long span = ((V + want - 1) / want + seg - 1) / seg * seg;
        return Form{vpt, (int)span, (int)((V + span - 1) / span)};
    };
    if (V <= 8192) return cut(4, 1);
    if (V <= (T < 128 ? 16384 : 32768) || T >= 384) return cut(16, 1);
    const long long want = 1536 / T;
    const Form f = cut(4, want);
    return f.span <= 8192 ? f : cut(16, want);
}

size_t splits_bytes(int T, int V, int top) {
    const Form f = form_of(T, V);
    return f.splits > 1 ? parts_bytes(T, f.splits, top) : 0;
}

int run_join(const Part* parts, const u64* tops, int T, int V, int splits, const LogprobOut& o, hipStream_t st) {
    logprobs_join_kernel<<<std::min(T, 1 << 20), NT, 0, st>>>(parts, tops, T, V, splits, o);
    return after_launch("token_logprobs");
}

int run_logprobs(const void* L, int dtype, long long ld, int T, int V, void* ws, const LogprobOut& o, hipStream_t st) {
    const Form f = form_of(T, V);
    Part* parts = (Part*)ws;
    u64* tops = (u64*)(parts + (size_t)T * f.splits);
    const int grid = (int)std::min<long long>((long long)T * f.splits, 1 << 20);
#define AEG_LP(TY, VPT) logprobs_kernel<TY, VPT><<<grid, NT, 0, st>>>((const TY*)L, ld, T, V, f.span, f.splits, parts, tops, o)
    if (dtype == AEGIST_F32) {
        if (f.vpt == 4) AEG_LP(float, 4);
        else AEG_LP(float, 16);
    } else {
        if (f.vpt == 4) AEG_LP(uint16_t, 4);
        else AEG_LP(uint16_t, 16);
    }
#undef AEG_LP
    int rc = after_launch("token_logprobs");
    return rc || f.splits == 1 ? rc : run_join(parts, tops, T, V, f.splits, o, st);
}

// Whether `rows` rows go to the product as A + R: fp32 ones on int8 or bf16 weights, where the projection does not take all
// their bits as it is (it does for one row, and for two on bf16 weights).
bool head_splits(int x_dtype, int w_dtype, int rows) {
    return x_dtype == AEGIST_F32 && w_dtype != AEGIST_Q4 && rows > (w_dtype == AEGIST_BF16 ? 2 : 1);
}
// Up to so many rows A and R are the rows of one product, so that it reads the weight once, and their logits are added; more
// rows take two products. Us, of the products alone, one (two), 131072 x 2048: bf16 16 rows 129 (228), 64 191 (301), 128 332 (368),
// 300 752 (689); int8 16 rows 65 (118), 64 138 (160), 128 262 (252). 32768 x 2048: bf16 64 rows 46 (60), int8 44 (53).
constexpr int kStackedRows = 64;
size_t round256(size_t n) { return (n + 255) / 256 * 256; }
// (a last block of fewer rows may be stacked where the others are not)
size_t head_logits_bytes(int x_dtype, int w_dtype, int rows, int V) {
    const int n = head_splits(x_dtype, w_dtype, rows) ? std::max(rows, 2 * std::min(rows, kStackedRows)) : rows;
    return round256((size_t)n * V * 4);
}
size_t head_a_bytes(int rows, int K) { return round256((size_t)rows * K * 4); }
size_t head_split_bytes(int x_dtype, int w_dtype, int rows, int K) {
    if (!head_splits(x_dtype, w_dtype, rows)) return 0;
    return std::max(head_a_bytes(rows, K) + round256((size_t)rows * K * 2), head_a_bytes(2 * std::min(rows, kStackedRows), K));
}
// Rows of a block: 256 MiB of logits, and no more of split rows.
int head_rows(int x_dtype, int w_dtype, int T, int V, int K) {
    long long rows = (256LL << 20) / (4LL * V);
    if (head_splits(x_dtype, w_dtype, T)) rows = std::min(rows, (256LL << 20) / (6LL * K));
    return (int)std::max(1LL, std::min<long long>(T, rows));
}

}  // namespace

extern "C" size_t aegist_token_logprobs_workspace_bytes(int T, int V, int top) {
    if (T < 1 || V < 1 || V > MAX_V || top < 0 || top > MAX_TOP) return 0;
    // no T up to this needs more: rows of up to 16384 logits are not cut, others into splits of at least 4096 and of no more
    // than 1536 in all
    if (V <= 16384) return 0;
    return parts_bytes((int)std::min(1536LL, T * ((V + 4095LL) / 4096)), 1, top);
}

extern "C" int aegist_token_logprobs(const void* logits, int dtype, long long ld, const int* tokens, float* logprob,
                                     float* entropy, int* top_ids, float* top_logprobs, int T, int V, int top, void* ws,
                                     size_t ws_bytes, void* stream) {
    const LogprobOut o{tokens, logprob, entropy, top_ids, top_logprobs, top};
    int rc = check_out("token_logprobs", T, V, o);
    if (rc) return rc;
    if (dtype != AEGIST_F32 && dtype != AEGIST_BF16)
        return fail(AEGIST_ERR_DTYPE, "token_logprobs: logits must be AEGIST_F32 or AEGIST_BF16");
    if (T == 0) return 0;
    if (!logits || ld < V) return fail(AEGIST_ERR_SHAPE, "token_logprobs: null logits, or ld < V");
    rc = check_workspace(ws, ws_bytes, splits_bytes(T, V, top), "token_logprobs");
    return rc ? rc : run_logprobs(logits, dtype, ld, T, V, ws, o, AEG_STREAM(stream));
}

extern "C" size_t aegist_head_logprobs_workspace_bytes(int x_dtype, int w_dtype, int T, int V, int K, int group, int top) {
    if (T < 1 || V < 1 || V > MAX_V || K < 1) return 0;
    const int rows = head_rows(x_dtype, w_dtype, T, V, K);
    // (the logits also where the product could leave statistics in their place: that takes an alignment, a stride and a weight
    // without scales, which are not known here)
    return head_logits_bytes(x_dtype, w_dtype, rows, V) + aegist_token_logprobs_workspace_bytes(rows, V, top) +
           head_split_bytes(x_dtype, w_dtype, rows, K) +
           (w_dtype == AEGIST_Q4 ? aegist_linear_q4_workspace_bytes(x_dtype, rows, V, K, group) : 0);
}

extern "C" int aegist_head_logprobs(const void* X, int x_dtype, long long ldx, const void* W, int w_dtype,
                                    const uint16_t* scale, const int* tokens, float* logprob, float* entropy,
                                    int* top_ids, float* top_logprobs, int T, int V, int K, int group, int top, void* ws,
                                    size_t ws_bytes, void* stream) {
    const LogprobOut o{tokens, logprob, entropy, top_ids, top_logprobs, top};
    int rc = check_out("head_logprobs", T, V, o);
    if (rc) return rc;
    if (x_dtype != AEGIST_F32 && x_dtype != AEGIST_BF16)
        return fail(AEGIST_ERR_DTYPE, "head_logprobs: X must be AEGIST_F32 or AEGIST_BF16");
    if (w_dtype != AEGIST_I8 && w_dtype != AEGIST_BF16 && w_dtype != AEGIST_Q4)
        return fail(AEGIST_ERR_DTYPE, "head_logprobs: W must be AEGIST_I8, AEGIST_BF16 or AEGIST_Q4");
    if (w_dtype == AEGIST_Q4 && (rc = check_q4("head_logprobs", V, K, group))) return rc;
    if (T == 0) return 0;
    if (!X || !W || K < 1) return fail(AEGIST_ERR_SHAPE, "head_logprobs: null operand or K < 1");
    if (w_dtype != AEGIST_Q4 && (K % 16 || ldx < K || ldx * (x_dtype == AEGIST_F32 ? 4 : 2) % 16 || (uintptr_t)X % 16))
        return fail(AEGIST_ERR_SHAPE, "head_logprobs: X needs 16-byte aligned rows (ldx >= K), K a multiple of 16");
    const hipStream_t st = AEG_STREAM(stream);
    const int block = head_rows(x_dtype, w_dtype, T, V, K), xs = x_dtype == AEGIST_F32 ? 4 : 2;
    const size_t lb = head_logits_bytes(x_dtype, w_dtype, block, V), pb = aegist_token_logprobs_workspace_bytes(block, V, top);
    rc = check_workspace(ws, ws_bytes, lb + pb + head_split_bytes(x_dtype, w_dtype, block, K), "head_logprobs");
    if (rc) return rc;  // (what a 4-bit product needs behind them linear_q4 checks)
    float* logits = (float*)ws;
    char *pws = (char*)ws + lb, *lws = pws + pb;
    float* xa = (float*)lws;
    uint16_t* xr = (uint16_t*)(lws + head_a_bytes(block, K));
    const int splits = row_stats_splits(V);
    Part* parts = (Part*)ws;
    u64* keys = (u64*)(parts + (size_t)block * splits);
    for (int t = 0; t < T; t += block) {
        const int m = std::min(block, T - t);
        const void* x = (const char*)X + (size_t)t * ldx * xs;
        const LogprobOut part{tokens + t, logprob + t, entropy + t, top_ids ? top_ids + (size_t)t * top : nullptr,
                              top_logprobs ? top_logprobs + (size_t)t * top : nullptr, top};
        // At most one alternative, on the tiles of gemm_bf16: the product leaves the rows' statistics in the place of the
        // logits (40 bytes per 128 columns), which a lane has nearly to itself: it holds 32 columns of a row (1000 rows of
        // 32768 x 2048: 114 us, 110 without alternatives, by way of the logits 155; their product alone takes 127).
        if (top <= 1 && V >= 256 && proj_is_gemm_bf16(x, x_dtype, ldx, W, w_dtype, scale, m, V, K)) {
            rc = launch_gemm_bf16_stats((const uint16_t*)x, ldx, (const uint16_t*)W, m, V, K,
                                        RowStats{part.tokens, parts, top ? keys : nullptr, splits}, st);
            if (rc || (rc = run_join(parts, keys, m, V, splits, part, st))) return rc;
            continue;
        }
        if (head_splits(x_dtype, w_dtype, m)) {
            const bool stacked = m <= kStackedRows;
            const int grid = (int)std::min<size_t>(((size_t)m * K / 4 + 255) / 256, 1 << 16);
            if (stacked) split_rows_kernel<float><<<grid, 256, 0, st>>>((const float*)x, ldx, m, K, xa, xa + (size_t)m * K);
            else split_rows_kernel<uint16_t><<<grid, 256, 0, st>>>((const float*)x, ldx, m, K, xa, xr);
            if ((rc = after_launch("head_logprobs"))) return rc;
            if (stacked) {
                const size_t n = (size_t)m * V;
                if ((rc = launch_proj(xa, AEGIST_F32, K, W, w_dtype, scale, logits, V, 2 * m, V, K, 0, st))) return rc;
                add_logits_kernel<<<(int)std::min<size_t>((n + 1023) / 1024, 1 << 16), 256, 0, st>>>(logits, logits + n, n);
                rc = after_launch("head_logprobs");
            } else {
                rc = launch_proj(xr, AEGIST_BF16, K, W, w_dtype, scale, logits, V, m, V, K, 0, st);
                if (!rc) rc = launch_proj(xa, AEGIST_F32, K, W, w_dtype, scale, logits, V, m, V, K, 1, st);
            }
        } else
            rc = w_dtype == AEGIST_Q4 ? launch_linear_q4(x, x_dtype, ldx, W, logits, V, m, V, K, group, 0, lws, ws_bytes - lb - pb, st)
                                      : launch_proj(x, x_dtype, ldx, W, w_dtype, scale, logits, V, m, V, K, 0, st);
        if (rc) return rc;
        if ((rc = run_logprobs(logits, AEGIST_F32, V, m, V, pws, part, st))) return rc;
    }
    return 0;
}
