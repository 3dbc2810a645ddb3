// Token log-probabilities on the device: rows of scores over a vocabulary -> the log-probability
// of given tokens, the entropy of the row's distribution, and its top alternatives.
//
// Per row, with A the allowed tokens (bit set in the mask, or no mask; logit above -inf) and
// y = x / temperature:
//   lse = m + log S,  S = sum over A of e^(y - m),  m = max over A of y;
//   log-probability of token t: y_t - lse;  entropy: log S - (sum over A of e^(y - m) (y - m)) / S;
//   alternatives: the `top` largest logits of A, equal ones by the lower id.
#include "heads.cuh"
#include "kernels.h"

namespace shipk {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// What a logit is among the alternatives: 0, none, for -inf and NaN.
__device__ __forceinline__ uint64_t logit_key(float x, int id) { return x > -INFINITY ? choice_key(x, id) : 0; }

struct Args {
    const void* logits;
    int vocab;
    int64_t row_stride;
    const int64_t* tokens;
    int n_tokens;
    const uint32_t* allowed;
    int64_t allowed_stride;
    float temperature;
    int top;
    float* logprobs;
    float* entropy;
    float* top_logprobs;
    int64_t* top_ids;
};

// A part of a row's sums: its largest logit m, the sum of e^d and that of e^d d, d = (x - m) / temperature.
struct Part {
    float m, s, h;
};

__device__ __forceinline__ Part join(const Part& a, const Part& b, float inv_t) {
    const float m = fmaxf(a.m, b.m);
    Part r{m, 0.f, 0.f};
    // a part that holds nothing adds nothing (its -inf would meet another); NaN sums stay NaN
    if (!(a.s == 0.f)) {
        const float d = fmaxf((a.m - m) * inv_t, -1e4f), e = expf(d);
        r.s += e * a.s;
        r.h += e * (a.h + d * a.s);
    }
    if (!(b.s == 0.f)) {
        const float d = fmaxf((b.m - m) * inv_t, -1e4f), e = expf(d);
        r.s += e * b.s;
        r.h += e * (b.h + d * b.s);
    }
    return r;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(const __grid_constant__ Args a) {
    __shared__ Part parts[kWarps];
    __shared__ uint64_t best[kWarps];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
    const uint32_t* allowed = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
    auto logit = [&](int v) {
        const bool on = !allowed || (__ldg(allowed + (v >> 5)) >> (v & 31)) & 1u;
        return on ? to_f32(x[v]) : -INFINITY;
    };

    const float inv_t = __fdiv_rn(1.f, a.temperature);
    Part p{-INFINITY, 0.f, 0.f};
    for (int v = tid; v < a.vocab; v += kThreads) {
        const float l = logit(v);
        if (l == -INFINITY) continue;
        p = join(p, Part{l, 1.f + 0.f * l, 0.f}, inv_t);  // NaN for NaN and +inf
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        p = join(p, Part{__shfl_xor_sync(0xffffffffu, p.m, o), __shfl_xor_sync(0xffffffffu, p.s, o),
                         __shfl_xor_sync(0xffffffffu, p.h, o)}, inv_t);
    if (lane == 0) parts[warp] = p;
    __syncthreads();
    p = parts[0];
    for (int w = 1; w < kWarps; ++w) p = join(p, parts[w], inv_t);
    const bool empty = p.s == 0.f;
    const float log_s = empty ? 0.f : logf(p.s);
    auto logprob = [&](float l) {
        if (empty || l == -INFINITY) return empty || p.s == p.s ? -INFINITY : p.s;
        return (l - p.m) * inv_t - log_s;
    };
    if (tid == 0) a.entropy[row] = empty ? 0.f : log_s - p.h / p.s;
    for (int j = tid; j < a.n_tokens; j += kThreads) {
        const int64_t t = a.tokens[row * a.n_tokens + j];
        a.logprobs[row * a.n_tokens + j] = t < 0 ? 0.f : t >= a.vocab ? NAN : logprob(logit((int)t));
    }
    uint64_t last = ~0ull;
    for (int j = 0; j < a.top; ++j) {
        uint64_t k = 0;
        for (int v = tid; v < a.vocab; v += kThreads) {
            const uint64_t c = logit_key(logit(v), v);
            if (c < last && c > k) k = c;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const uint64_t c = __shfl_xor_sync(0xffffffffu, k, o);
            k = c > k ? c : k;
        }
        __syncthreads();
        if (lane == 0) best[warp] = k;
        __syncthreads();
        for (int w = 0; w < kWarps; ++w) k = best[w] > k ? best[w] : k;
        if (tid == 0) {
            a.top_ids[row * a.top + j] = k ? key_index(k) : -1;
            a.top_logprobs[row * a.top + j] = k ? logprob(key_value(k)) : -INFINITY;
        }
        last = k;
    }
}

}  // namespace

Status launch_token_logprobs(const void* logits, int dtype, int rows, int vocab, int64_t row_stride,
                             const int64_t* tokens, int n_tokens, const uint32_t* allowed, int64_t allowed_stride,
                             float temperature, int top, float* logprobs, float* entropy, float* top_logprobs,
                             int64_t* top_ids, cudaStream_t stream) {
    const Args a{logits, vocab, row_stride, tokens, n_tokens, allowed, allowed_stride, temperature,
                 top, logprobs, entropy, top_logprobs, top_ids};
    if (dtype == SHIPK_DTYPE_F32) logprobs_kernel<float><<<rows, kThreads, 0, stream>>>(a);
    else if (dtype == SHIPK_DTYPE_F16) logprobs_kernel<__half><<<rows, kThreads, 0, stream>>>(a);
    else logprobs_kernel<__nv_bfloat16><<<rows, kThreads, 0, stream>>>(a);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return Status{SHIPK_ECUDA, cudaGetErrorString(e)};
    return Status{SHIPK_OK, nullptr};
}

}  // namespace shipk
