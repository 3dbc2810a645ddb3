// Routing rows to experts: a gate's scores -> the experts of each row with their weights, the
// rows grouped by expert, and the experts' results joined per row.
//
// route: per row, with A the experts whose logit and bias are neither -inf nor NaN,
//   s_e = 1 / (1 + e^-x_e), or e^x_e / (sum over A of e^x); c_e = s_e + bias_e;
//   a group's score: the largest c of its experts in A, or the sum of its two largest; the
//   top_groups groups with the largest scores (ties: the lower group) stay, then the top_k
//   largest c among their experts in A (ties: the lower expert) are chosen;
//   weight: s_e, divided by the sum of the chosen s when renormalising, times scale.
// The scores decide an order, so they are exactly rounded: computed in 64 bits and rounded once
// to 32, c_e and a group's sum with one 32-bit rounding each. Any way of computing them that keeps
// those roundings chooses the same experts.
//
// plan: a stable counting sort of the (row, j) assignments by expert. combine: the weighted sum
// of each row's results, in 32 bits in the order of j, rounded once to the output's type.
#include "heads.cuh"
#include "kernels.h"

namespace shipk {

namespace {

// ---- route ----------------------------------------------------------------------------------

constexpr int kRouteThreads = 128;
constexpr int kRouteWarps = kRouteThreads / 32;

struct RouteArgs {
    const void* logits;
    int rows, experts;
    int64_t row_stride;
    const float* bias;
    int top_k, sigmoid, groups, top_groups, group_top2, renormalise;
    float scale;
    float* weights;
    int32_t* ids;
};

__device__ __forceinline__ uint64_t warp_max(uint64_t k) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const uint64_t c = __shfl_xor_sync(0xffffffffu, k, o);
        k = c > k ? c : k;
    }
    return k;
}

// One warp per row; the scores and choices of its row stand in shared memory.
template <typename T>
__global__ void __launch_bounds__(kRouteThreads) route_kernel(const __grid_constant__ RouteArgs a) {
    extern __shared__ float route_smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = (int64_t)blockIdx.x * kRouteWarps + warp;
    if (row >= a.rows) return;
    float* score = route_smem + warp * 2 * a.experts;
    float* choice = score + a.experts;  // -inf: not in A, or its group was not chosen
    const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;

    double m = -INFINITY, sum = 0.0;
    if (!a.sigmoid) {
        for (int e = lane; e < a.experts; e += 32) {
            const double l = fmin((double)to_f32(x[e]), (double)3.402823466e38f);  // NaN: not in A
            const float b = a.bias ? __ldg(a.bias + e) : 0.f;
            if (to_f32(x[e]) > -INFINITY && b > -INFINITY) m = fmax(m, l);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, o));
        for (int e = lane; e < a.experts; e += 32) {
            const double l = fmin((double)to_f32(x[e]), (double)3.402823466e38f);
            const float b = a.bias ? __ldg(a.bias + e) : 0.f;
            if (to_f32(x[e]) > -INFINITY && b > -INFINITY) sum += exp(l - m);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    for (int e = lane; e < a.experts; e += 32) {
        const float l = to_f32(x[e]), b = a.bias ? __ldg(a.bias + e) : 0.f;
        const double d = fmin((double)l, (double)3.402823466e38f);  // +inf as the largest logit
        const bool in = l > -INFINITY && b > -INFINITY;
        const float s = !in ? 0.f : (float)(a.sigmoid ? 1.0 / (1.0 + exp(-d)) : exp(d - m) / sum);
        score[e] = s;
        choice[e] = in ? __fadd_rn(s, b) : -INFINITY;
    }
    __syncwarp();
    if (a.groups > 1) {
        const int size = a.experts / a.groups;
        uint64_t mine = 0;
        if (lane < a.groups) {
            float first = -INFINITY, second = -INFINITY;
            for (int i = 0; i < size; ++i) {
                const float c = choice[lane * size + i];
                if (c > first) {
                    second = first;
                    first = c;
                } else if (c > second) {
                    second = c;
                }
            }
            if (first > -INFINITY)
                mine = choice_key(a.group_top2 && second > -INFINITY ? __fadd_rn(first, second) : first, lane);
        }
        int rank = 0;
        for (int g = 0; g < a.groups; ++g) rank += __shfl_sync(0xffffffffu, mine, g) > mine;
        if (lane < a.groups && rank >= a.top_groups)
            for (int i = 0; i < size; ++i) choice[lane * size + i] = -INFINITY;
        __syncwarp();
    }
    double total = 0.0;
    uint64_t mine = 0, last = ~0ull;  // lane j keeps the j-th chosen
    for (int j = 0; j < a.top_k; ++j) {
        uint64_t k = 0;
        for (int e = lane; e < a.experts; e += 32) {
            if (!(choice[e] > -INFINITY)) continue;
            const uint64_t c = choice_key(choice[e], e);
            if (c < last && c > k) k = c;
        }
        k = warp_max(k);
        if (k) total += (double)score[key_index(k)];
        if (lane == j) mine = k;
        last = k;
    }
    if (lane < a.top_k) {
        const int e = mine ? key_index(mine) : -1;
        double w = 0.0;
        if (e >= 0) {
            w = score[e];
            if (a.renormalise) w = total > 0.0 ? w / total : 0.0;
            w *= (double)a.scale;
        }
        a.ids[row * a.top_k + lane] = e;
        a.weights[row * a.top_k + lane] = (float)w;
    }
}

// ---- plan -----------------------------------------------------------------------------------

constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;

struct PlanArgs {
    const int32_t* ids;
    int pairs, k, experts;
    int32_t* order;
    int32_t* slots;
    int32_t* offsets;
};

// One CTA. Each warp owns a run of assignments and a row of counters: it counts its run's experts,
// the counters become the places before which this warp's assignments of each expert go, and it
// walks its run again in order, so that the sort is stable and no atomic decides a place.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const __grid_constant__ PlanArgs a) {
    extern __shared__ int plan_smem[];  // [kPlanWarps][experts]
    __shared__ int scan[kPlanWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int* mine = plan_smem + warp * a.experts;
    for (int e = lane; e < a.experts; e += 32) mine[e] = 0;
    __syncwarp();
    const int64_t run = ((((int64_t)a.pairs + kPlanWarps - 1) / kPlanWarps) + 31) & ~(int64_t)31;
    const int64_t lo = min((int64_t)a.pairs, run * warp), hi = min((int64_t)a.pairs, lo + run);
    for (int64_t i = lo + lane; i - lane < hi; i += 32) {
        int id = i < hi ? a.ids[i] : -1;
        if (id < 0 || id >= a.experts) id = -1;
        const unsigned peers = __match_any_sync(0xffffffffu, id);
        if (id >= 0 && lane == __ffs(peers) - 1) mine[id] += __popc(peers);
        __syncwarp();
    }
    __syncthreads();
    int total = 0;
    if (tid < a.experts) {
        for (int w = 0; w < kPlanWarps; ++w) {
            const int c = plan_smem[w * a.experts + tid];
            plan_smem[w * a.experts + tid] = total;
            total += c;
        }
    }
    int incl = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    int before = 0, kept = 0;
    for (int w = 0; w < kPlanWarps; ++w) {
        if (w < warp) before += scan[w];
        kept += scan[w];
    }
    const int first = before + incl - total;
    if (tid < a.experts) {
        a.offsets[tid] = first;
        for (int w = 0; w < kPlanWarps; ++w) plan_smem[w * a.experts + tid] += first;
    }
    if (tid == 0) a.offsets[a.experts] = kept;
    __syncthreads();
    for (int64_t i = lo + lane; i - lane < hi; i += 32) {
        int id = i < hi ? a.ids[i] : -1;
        if (id < 0 || id >= a.experts) id = -1;
        const unsigned peers = __match_any_sync(0xffffffffu, id);
        const int place = id >= 0 ? mine[id] + __popc(peers & ((1u << lane) - 1u)) : -1;
        __syncwarp();
        if (id >= 0 && lane == __ffs(peers) - 1) mine[id] += __popc(peers);
        __syncwarp();
        if (i < hi) a.slots[i] = place;
        if (place >= 0) a.order[place] = (int)(i / a.k);
    }
    for (int64_t i = (int64_t)kept + tid; i < a.pairs; i += kPlanThreads) a.order[i] = -1;
}

// ---- combine --------------------------------------------------------------------------------

constexpr int kCombineThreads = 256;

struct CombineArgs {
    const void* rows;
    int n_rows;
    int64_t row_stride;
    const float* weights;
    const int32_t* slots;
    int n, k, width;
    void* out;
};

template <typename T>
__global__ void __launch_bounds__(kCombineThreads) combine_kernel(const __grid_constant__ CombineArgs a) {
    const int64_t i = (int64_t)blockIdx.x * kCombineThreads + threadIdx.x;
    if (i >= (int64_t)a.n * a.width) return;
    const int64_t row = i / a.width, c = i - row * a.width;
    float sum = 0.f;
    for (int j = 0; j < a.k; ++j) {
        const int slot = __ldg(a.slots + row * a.k + j);
        if (slot < 0 || slot >= a.n_rows) continue;
        sum = __fmaf_rn(__ldg(a.weights + row * a.k + j), to_f32(static_cast<const T*>(a.rows)[slot * a.row_stride + c]), sum);
    }
    from_f32(sum, static_cast<T*>(a.out) + i);
}

Status launched() {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? Status{SHIPK_OK, nullptr} : Status{SHIPK_ECUDA, cudaGetErrorString(e)};
}

}  // namespace

Status launch_route(const void* logits, int dtype, int rows, int experts, int64_t row_stride, const float* bias,
                    int top_k, int sigmoid, int groups, int top_groups, int group_top2, int renormalise, float scale,
                    float* weights, int32_t* ids, cudaStream_t stream) {
    const RouteArgs a{logits, rows, experts, row_stride, bias, top_k, sigmoid, groups,
                      top_groups, group_top2, renormalise, scale, weights, ids};
    const int ctas = (int)(((int64_t)rows + kRouteWarps - 1) / kRouteWarps);
    const int smem = kRouteWarps * 2 * experts * (int)sizeof(float);  // at most 32 KB
    if (dtype == SHIPK_DTYPE_F32) route_kernel<float><<<ctas, kRouteThreads, smem, stream>>>(a);
    else if (dtype == SHIPK_DTYPE_F16) route_kernel<__half><<<ctas, kRouteThreads, smem, stream>>>(a);
    else route_kernel<__nv_bfloat16><<<ctas, kRouteThreads, smem, stream>>>(a);
    return launched();
}

Status launch_plan(const int32_t* ids, int rows, int k, int experts, int32_t* order, int32_t* slots, int32_t* offsets,
                   cudaStream_t stream) {
    const PlanArgs a{ids, rows * k, k, experts, order, slots, offsets};
    const int smem = kPlanWarps * experts * (int)sizeof(int);
    const cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(plan_kernel), kPlanWarps * kMaxExperts * (int)sizeof(int));
    if (e != cudaSuccess) return Status{SHIPK_ECUDA, cudaGetErrorString(e)};
    plan_kernel<<<1, kPlanThreads, smem, stream>>>(a);
    return launched();
}

Status launch_combine(const void* in, int dtype, int n_in, int64_t row_stride, const float* weights, const int32_t* slots,
                      int rows, int k, int width, void* out, cudaStream_t stream) {
    const CombineArgs a{in, n_in, row_stride, weights, slots, rows, k, width, out};
    const int64_t ctas = ((int64_t)rows * width + kCombineThreads - 1) / kCombineThreads;
    if (ctas > 0x7fffffff) return Status{SHIPK_ERANGE, "more than 2^39 output values"};
    if (dtype == SHIPK_DTYPE_F32) combine_kernel<float><<<(int)ctas, kCombineThreads, 0, stream>>>(a);
    else if (dtype == SHIPK_DTYPE_F16) combine_kernel<__half><<<(int)ctas, kCombineThreads, 0, stream>>>(a);
    else combine_kernel<__nv_bfloat16><<<(int)ctas, kCombineThreads, 0, stream>>>(a);
    return launched();
}

}  // namespace shipk
