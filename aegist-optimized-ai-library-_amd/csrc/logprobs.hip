// Log probabilities of given tokens, the entropy and the most probable tokens of each row of logits, and the
// same straight from hidden rows and an output head.
//
//   m = max x,  z = sum e^(x - m),  logprob = x[token] - m - ln z,  entropy = ln z - sum e^(x - m) (x - m) / z
//
// (the entropy's sum is taken over x - m, not x, so that a common offset of the logits costs no digits). Logits
// of -inf have no probability; a row of nothing else has logprob -inf for every token and entropy 0. NaN or
// +inf anywhere in a row makes its logprobs and entropy NaN.
#include "q4.h"

#include <algorithm>

using namespace aegist;

namespace aegist {
int launch_proj(const void* X, int x_dtype, long long ldx, const void* W, int w_dtype, const uint16_t* scale, float* Y,
                long long ldy, int M, int N, int K, int accumulate, hipStream_t st);
}

namespace {

constexpr int MAX_TOP = 64;

// Order of the alternatives as one number: the larger value first (NaN before all, -0 as +0), then the lower
// token. Larger keys come first; 0 is below every element's.
__device__ __forceinline__ uint64_t lp_key(float v, uint32_t id) {
    const uint32_t b = v != v ? 0x7fc00000u : __float_as_uint(v + 0.f);
    return (uint64_t)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (uint32_t)~id;
}
__device__ __forceinline__ float lp_key_value(uint64_t k) {
    const uint32_t b = (uint32_t)(k >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}

struct LogprobOut {
    const int* tokens;
    float *logprob, *entropy;
    int* top_ids;
    float* top_logprobs;
    int top;
};

// one workgroup per row
template <typename T>
__global__ void __launch_bounds__(256) logprobs_kernel(const T* __restrict__ L, long long ld, int rows, int V,
                                                       const LogprobOut o) {
    __shared__ float red[4];
    __shared__ uint64_t best[4];
    for (int t = blockIdx.x; t < rows; t += gridDim.x) {
        const T* x = L + (size_t)t * ld;
        float m = -INFINITY;
        bool bad = false;
        for (int i = threadIdx.x; i < V; i += 256) {
            const float v = Act<T>::ld(x, i);
            m = fmaxf(m, v);
            bad |= v != v || v == INFINITY;
        }
        bad = __syncthreads_or(bad);
        m = wave_max(m);
        if (threadIdx.x % WAVE == 0) red[threadIdx.x / WAVE] = m;
        __syncthreads();
        m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const bool empty = m == -INFINITY;
        float z = 0.f, s = 0.f;
        if (!empty && !bad)
            for (int i = threadIdx.x; i < V; i += 256) {
                const float d = Act<T>::ld(x, i) - m, e = expf(d);
                z += e;
                if (e > 0.f) s = fmaf(e, d, s);
            }
        z = block_sum(z, red);
        s = block_sum(s, red);
        const float lz = bad ? __builtin_nanf("") : logf(z);
        if (threadIdx.x == 0) {
            const int tok = o.tokens[t];
            float lp = tok < 0 ? 0.f : __builtin_nanf("");
            if (tok >= 0 && tok < V && !bad) lp = empty ? -INFINITY : Act<T>::ld(x, tok) - m - lz;
            o.logprob[t] = lp;
            o.entropy[t] = empty && !bad ? 0.f : lz - s / z;
        }
        uint64_t last = ~0ull;
        for (int j = 0; j < o.top; j++) {
            uint64_t k = 0;
            for (int i = threadIdx.x; i < V; i += 256) {
                const uint64_t ki = lp_key(Act<T>::ld(x, i), i);
                if (ki < last && ki > k) k = ki;
            }
            for (int w = 32; w > 0; w >>= 1) {
                const uint64_t k2 = __shfl_xor((unsigned long long)k, w, WAVE);
                k = k2 > k ? k2 : k;
            }
            __syncthreads();
            if (threadIdx.x % WAVE == 0) best[threadIdx.x / WAVE] = k;
            __syncthreads();
            for (int w = 0; w < 4; w++) k = best[w] > k ? best[w] : k;
            if (threadIdx.x == 0) {
                o.top_ids[(size_t)t * o.top + j] = (int)~(uint32_t)k;
                o.top_logprobs[(size_t)t * o.top + j] =
                    bad ? __builtin_nanf("") : empty ? -INFINITY : lp_key_value(k) - m - lz;
            }
            last = k;
        }
        __syncthreads();
    }
}

int check_out(const char* who, int T, int V, const LogprobOut& o) {
    const std::string w(who);
    if (T < 0 || V < 1) return fail(AEGIST_ERR_SHAPE, w + ": negative size or empty vocabulary");
    if (o.top < 0 || o.top > MAX_TOP || o.top > V)
        return fail(AEGIST_ERR_SHAPE, w + ": 0 to 64 alternatives, no more than the vocabulary has");
    if (T == 0) return 0;
    if (!o.tokens || !o.logprob || !o.entropy || (o.top && (!o.top_ids || !o.top_logprobs)))
        return fail(AEGIST_ERR_SHAPE, w + ": null operand");
    return 0;
}

int run_logprobs(const void* L, int dtype, long long ld, int T, int V, const LogprobOut& o, hipStream_t st) {
    const int grid = std::min(T, 1 << 20);
    if (dtype == AEGIST_F32) logprobs_kernel<float><<<grid, 256, 0, st>>>((const float*)L, ld, T, V, o);
    else logprobs_kernel<uint16_t><<<grid, 256, 0, st>>>((const uint16_t*)L, ld, T, V, o);
    return after_launch("token_logprobs");
}

// rows of logits that are whole at a time: 256 MiB
int head_rows(int T, int V) { return (int)std::max(1LL, std::min<long long>(T, (256LL << 20) / (4LL * V))); }

size_t head_logits_bytes(int T, int V) { return ((size_t)head_rows(T, V) * V * 4 + 255) / 256 * 256; }

}  // namespace

extern "C" size_t aegist_token_logprobs_workspace_bytes(int T, int V, int top) { return 0; }

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
    return run_logprobs(logits, dtype, ld, T, V, o, AEG_STREAM(stream));
}

extern "C" size_t aegist_head_logprobs_workspace_bytes(int x_dtype, int w_dtype, int T, int V, int K, int group, int top) {
    if (T < 1 || V < 1 || K < 1) return 0;
    return head_logits_bytes(T, V) + (w_dtype == AEGIST_Q4 ? aegist_linear_q4_workspace_bytes(x_dtype, head_rows(T, V), V, K, group) : 0);
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
    rc = check_workspace(ws, ws_bytes, aegist_head_logprobs_workspace_bytes(x_dtype, w_dtype, T, V, K, group, top),
                         "head_logprobs");
    if (rc) return rc;
    const hipStream_t st = AEG_STREAM(stream);
    const int block = head_rows(T, V), xs = x_dtype == AEGIST_F32 ? 4 : 2;
    const size_t lb = head_logits_bytes(T, V);
    float* logits = (float*)ws;
    for (int t = 0; t < T; t += block) {
        const int m = std::min(block, T - t);
        const void* x = (const char*)X + (size_t)t * ldx * xs;
        rc = w_dtype == AEGIST_Q4 ? launch_linear_q4(x, x_dtype, ldx, W, logits, V, m, V, K, group, 0, (char*)ws + lb,
                                                     ws_bytes - lb, st)
                                  : launch_proj(x, x_dtype, ldx, W, w_dtype, scale, logits, V, m, V, K, 0, st);
        if (rc) return rc;
        const LogprobOut part{tokens + t, logprob + t, entropy + t, top_ids ? top_ids + (size_t)t * top : nullptr,
                              top_logprobs ? top_logprobs + (size_t)t * top : nullptr, top};
        if ((rc = run_logprobs(logits, AEGIST_F32, V, m, V, part, st))) return rc;
    }
    return 0;
}
