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

#include <cooperative_groups.h>

#include <algorithm>
#include <map>
#include <mutex>

namespace cg = cooperative_groups;

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
    int top_k, groups, top_groups, group_top2, renormalise;
    int each;  // experts of a lane
    int size, span;  // experts of a group; its lanes, 0 where groups share lanes
    int wide, wide_bias;  // a lane's logits, and its biases, 16 bytes at a time
    float scale;
    float* weights;
    int32_t* ids;
};

__device__ __forceinline__ double exact_logit(float x) { return (double)fminf(x, 3.402823466e38f); }  // +inf: the largest
__device__ __forceinline__ float exact_sigmoid(float x) { return (float)(1.0 / (1.0 + exp(-exact_logit(x)))); }

// What a warp holds of a row: expert lane * each + i in slot i of a lane. Slots past the experts and
// experts that cannot be chosen hold a choice of -inf.
template <int NS>
struct Choices {
    float c[NS];

    __device__ __forceinline__ float best() const {
        float m = c[0];
#pragma unroll
        for (int i = 1; i < NS; ++i) m = fmaxf(m, c[i]);
        return m;
    }
};

// Shared by a warp: the choices that reach a bound, in any order.
constexpr int kListed = 64;
struct Listed {
    uint64_t keys[kListed];
    float x[kListed];       // their logits
    int8_t order[kListed];  // the entry of each rank
};

// The larger two of two descending pairs.
__device__ __forceinline__ void merge2(float& first, float& second, float f, float s) {
    second = fmaxf(fminf(first, f), fmaxf(second, s));
    first = fmaxf(first, f);
}

// Closes every group but the top_groups best. With groups of whole lanes a group's score meets in
// its lanes; else through `row` (shared memory, one float for each expert). Returns how far the last
// group kept is above the next one.
template <int NS>
__device__ __forceinline__ float keep_groups(const RouteArgs& a, Choices<NS>& k, float* row, int lane) {
    float first = k.c[0], second = -INFINITY;
    const int span = a.span;
    if (span) {
#pragma unroll
        for (int i = 1; i < NS; ++i) {
            second = fmaxf(second, fminf(first, k.c[i]));
            first = fmaxf(first, k.c[i]);
        }
        if ((span & (span - 1)) == 0) {
            for (int o = 1; o < span; o *= 2)
                merge2(first, second, __shfl_xor_sync(0xffffffffu, first, o), __shfl_xor_sync(0xffffffffu, second, o));
        } else {  // a group's first lane gathers the others'
            const float f = first, s = second;
            for (int o = 1; o < span; ++o)
                merge2(first, second, __shfl_down_sync(0xffffffffu, f, o), __shfl_down_sync(0xffffffffu, s, o));
        }
    } else {
#pragma unroll
        for (int i = 0; i < NS; ++i)
            if (i < a.each && lane * a.each + i < a.experts) row[lane * a.each + i] = k.c[i];
        __syncwarp();
        first = -INFINITY;
        if (lane < a.groups)
            for (int i = 0; i < a.size; ++i) merge2(first, second, row[lane * a.size + i], -INFINITY);
    }
    // lane g takes group g's score; 0: nothing in it can be chosen
    const float value = a.group_top2 && second > -INFINITY ? __fadd_rn(first, second) : first;
    uint32_t ord = first > -INFINITY ? order_bits(value) : 0u;
    if (span) ord = __shfl_sync(0xffffffffu, ord, (lane * span) & 31);
    if (lane >= a.groups) ord = 0;
    int above = 0;
    for (int g = 0; g < a.groups; ++g) {
        const uint32_t other = __shfl_sync(0xffffffffu, ord, g);
        above += other > ord || (other == ord && g < lane);
    }
    const bool kept = ord && above < a.top_groups;
    const unsigned open = __ballot_sync(0xffffffffu, kept);
    // the least kept and the best left out
    const uint32_t low = __reduce_min_sync(0xffffffffu, kept ? ord : 0xffffffffu);
    const uint32_t high = __reduce_max_sync(0xffffffffu, kept ? 0u : ord);
    if (span) {
        const int g = lane / span;
        if (!(open >> g & 1u))
#pragma unroll
            for (int i = 0; i < NS; ++i) k.c[i] = -INFINITY;
    } else {
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int g = (lane * a.each + i) / a.size;
            if (g < 32 && !(open >> g & 1u)) k.c[i] = -INFINITY;
        }
    }
    return high && open ? from_order_bits(low) - from_order_bits(high) : INFINITY;
}

// The top_k best, ties to the lower expert, the j-th in lane j. `margin`: how far two choices have
// to be apart for their order to be sure, or 0 where they are exact; false when some two that decide
// are nearer without being equal by their inputs (the logit, and no bias).
//
// The top_k-th largest of the lanes' maxima bounds the choices: at least top_k reach it, and few
// more. Those that do (or come within the margin of it) are listed and ranked. More than the list holds,
// by ties or many of them: taken one at a time.
template <int NS>
__device__ __forceinline__ bool take_best(const RouteArgs& a, Choices<NS>& k, const float (&x)[NS], float margin, int lane,
                                          Listed& list, int& chosen) {
    const float m = k.best();
    const uint32_t mine = m > -INFINITY ? order_bits(m) : 0u;
    uint32_t left = mine, t = 0;
    for (int j = 0; j < a.top_k; ++j) {
        t = __reduce_max_sync(0xffffffffu, left);
        if (lane == __ffs(__ballot_sync(0xffffffffu, left == t)) - 1) left = 0;
    }
    float least = t ? from_order_bits(t) : -INFINITY;
    if (margin > 0.f) least = least - (margin + 0x1p-21f * fabsf(least));  // NaN, which nothing reaches, for +inf
    int n = 0;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const bool in = k.c[i] >= least && k.c[i] > -INFINITY;
        const unsigned who = __ballot_sync(0xffffffffu, in);
        const int at = n + __popc(who & ((1u << lane) - 1u));
        if (in && at < kListed) {
            list.keys[at] = choice_key(k.c[i], lane * a.each + i);
            list.x[at] = x[i];
        }
        n += __popc(who);
    }
    __syncwarp();
    chosen = -1;
    if (n <= kListed) {
        const uint64_t k0 = lane < n ? list.keys[lane] : 0, k1 = lane + 32 < n ? list.keys[lane + 32] : 0;
        int r0 = 0, r1 = 0;
        for (int q = 0; q < n; ++q) {
            const uint64_t other = list.keys[q];
            r0 += other > k0;
            r1 += other > k1;
        }
        if (lane < n) list.order[r0] = (int8_t)lane;
        if (lane + 32 < n) list.order[r1] = (int8_t)(lane + 32);
        __syncwarp();
        if (lane < min(n, a.top_k)) chosen = key_index(list.keys[list.order[lane]]);
        if (margin > 0.f) {
            // each choice against the one behind it; what is not listed is further than the margin.
            // Equal inputs are equal choices, but behind the last one others may follow that are near.
            if (!(least > -INFINITY) && t) return false;
            bool sure = true;
            if (lane < min(n - 1, a.top_k)) {
                const int u = list.order[lane], v = list.order[lane + 1];
                const float hi = key_value(list.keys[u]), lo = key_value(list.keys[v]);
                const bool equal = list.x[u] == list.x[v] && !a.bias && lane + 1 < a.top_k;
                sure = hi - lo > margin + 0x1p-21f * fabsf(lo) || equal;
            }
            return __all_sync(0xffffffffu, sure);
        }
        return true;
    }
    if (margin > 0.f) return false;
    uint32_t o = mine;
    for (int j = 0; j < a.top_k; ++j) {
        const uint32_t high = __reduce_max_sync(0xffffffffu, o);
        if (!high) break;
        int slot = 0;
#pragma unroll
        for (int i = NS - 1; i >= 0; --i) slot = k.c[i] > -INFINITY && order_bits(k.c[i]) == o ? i : slot;
        const int e = __reduce_min_sync(0xffffffffu, o == high ? lane * a.each + slot : 0x7fffffff);
        if (lane == j) chosen = e;
        const bool own = o == high && lane * a.each + slot == e;
#pragma unroll
        for (int i = 0; i < NS; ++i) k.c[i] = own && i == slot ? -INFINITY : k.c[i];
        const float next = k.best();
        o = next > -INFINITY ? order_bits(next) : 0u;
    }
    return true;
}

// A warp per row. Softmax scores are computed in 64 bits. Sigmoid scores are computed in 32 first
// (2 units in the last place for the exponential, 2 for the quotient, the sum's rounding: 2^-20.6 of
// the score) and where all the choices that decide are further apart than two such errors they
// stand as they would in 64 bits; only else are all of the row's scores computed in 64. The weights
// always come from the exact scores of the chosen. Bound by issue slots (77% busy): 16,384 rows of 256
// experts in 8 groups, 1160 instructions a row, take 25 us where the logits alone are 2.6; 64 bits
// for every score and choices in shared memory took 55.
template <typename T, int NS, bool SIGMOID>
__global__ void __launch_bounds__(kRouteThreads) route_kernel(const __grid_constant__ RouteArgs a) {
    extern __shared__ float route_smem[];
    __shared__ Listed lists[kRouteWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = (int64_t)blockIdx.x * kRouteWarps + warp;
    if (row >= a.rows) return;
    Listed& list = lists[warp];
    const T* logits = static_cast<const T*>(a.logits) + row * a.row_stride;
    float* const by_expert = route_smem + warp * a.experts;

    float x[NS];
    const int e0 = lane * a.each;
    constexpr int kVec = 16 / sizeof(T);
    if (NS >= kVec && a.wide) {  // each == NS
        if constexpr (NS >= kVec) {
#pragma unroll
            for (int i = 0; i < NS; i += kVec) {
                const uint4 u = __ldg(reinterpret_cast<const uint4*>(logits + e0 + i));
                T v[kVec];
                *reinterpret_cast<uint4*>(v) = u;
#pragma unroll
                for (int j = 0; j < kVec; ++j) x[i + j] = to_f32(v[j]);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < NS; ++i) x[i] = i < a.each && e0 + i < a.experts ? to_f32(logits[e0 + i]) : -INFINITY;
    }
    float b[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) b[i] = 0.f;
    if (a.bias) {
        if (NS >= 4 && a.wide_bias) {  // each == NS
#pragma unroll
            for (int i = 0; i + 3 < NS; i += 4) {
                const float4 v = __ldg(reinterpret_cast<const float4*>(a.bias + e0 + i));
                b[i] = v.x;
                b[i + 1] = v.y;
                b[i + 2] = v.z;
                b[i + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NS; ++i) b[i] = i < a.each && e0 + i < a.experts ? __ldg(a.bias + e0 + i) : 0.f;
        }
    }
#pragma unroll
    for (int i = 0; i < NS; ++i) x[i] = x[i] > -INFINITY && b[i] > -INFINITY ? x[i] : -INFINITY;  // NaN too

    Choices<NS> k;
    int chosen = -1;
    double m = 0.0, inv = 1.0;
    double e[SIGMOID || NS > 8 ? 1 : NS];  // more would cost the warps that hide the exponentials
    bool sure = false;
    if (SIGMOID) {
        float high = 0.f;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const float s = __fdividef(1.f, 1.f + expf(fminf(-x[i], 80.f)));
            k.c[i] = x[i] > -INFINITY ? __fadd_rn(s, b[i]) : -INFINITY;
            if (x[i] > -INFINITY) high = fmaxf(high, s);
        }
        high = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(high)));
        const float margin = fmaxf(0x1p-19f * high, 4e-35f);  // e^-80 stands for all below it
        const float gap = a.groups > 1 ? keep_groups(a, k, by_expert, lane) : INFINITY;
        sure = take_best(a, k, x, margin, lane, list, chosen) && gap > 4.f * margin;
        if (a.groups > 1 && sure) {
            // a group's sum may be large by its bias: its own rounding counts too
            float large = 0.f;
#pragma unroll
            for (int i = 0; i < NS; ++i) large = fmaxf(large, fabsf(b[i]) < INFINITY ? fabsf(b[i]) : 0.f);
            large = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(large)));
            sure = gap > 4.f * margin + 0x1p-19f * large;
        }
    } else {
        float high = -INFINITY;
#pragma unroll
        for (int i = 0; i < NS; ++i) high = fmaxf(high, x[i]);
        const uint32_t top = __reduce_max_sync(0xffffffffu, order_bits(high));
        m = exact_logit(from_order_bits(top));
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            double v = 0.0;
            if (x[i] > -INFINITY) v = exp(exact_logit(x[i]) - m);
            if (NS <= 8) e[i < (int)(sizeof(e) / sizeof(double)) ? i : 0] = v;
            sum += v;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        inv = 1.0 / sum;
    }
    auto exact = [&](float v) { return SIGMOID ? exact_sigmoid(v) : (float)(exp(exact_logit(v) - m) * inv); };
    if (!sure) {  // the whole warp
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            float s = 0.f;
            if (!SIGMOID && NS <= 8) s = (float)(e[i < (int)(sizeof(e) / sizeof(double)) ? i : 0] * inv);
            else if (x[i] > -INFINITY) s = exact(x[i]);
            k.c[i] = x[i] > -INFINITY ? __fadd_rn(s, b[i]) : -INFINITY;
        }
        if (a.groups > 1) {
            __syncwarp();
            keep_groups(a, k, by_expert, lane);
        }
        take_best(a, k, x, 0.f, lane, list, chosen);
    }

    const double score = chosen >= 0 ? (double)exact(to_f32(logits[chosen])) : 0.0;
    double w = score;
    if (a.renormalise) {
        double total = 0.0;
        for (int j = 0; j < a.top_k; ++j) total += __shfl_sync(0xffffffffu, score, j);
        w = total > 0.0 ? w / total : 0.0;
    }
    if (lane < a.top_k) {
        a.ids[row * a.top_k + lane] = chosen;
        a.weights[row * a.top_k + lane] = (float)(w * (double)a.scale);
    }
}

template <typename T, int NS>
void launch_route_slots(const RouteArgs& a, bool sigmoid, cudaStream_t stream) {
    const unsigned ctas = (unsigned)(((int64_t)a.rows + kRouteWarps - 1) / kRouteWarps);
    const int smem = a.groups > 1 && !a.span ? kRouteWarps * a.experts * (int)sizeof(float) : 0;
    if (sigmoid) route_kernel<T, NS, true><<<ctas, kRouteThreads, smem, stream>>>(a);
    else route_kernel<T, NS, false><<<ctas, kRouteThreads, smem, stream>>>(a);
}

template <typename T>
void launch_route_type(RouteArgs a, bool sigmoid, cudaStream_t stream) {
    a.each = (a.experts + 31) / 32;
    a.size = a.experts / a.groups;
    a.span = a.size % a.each ? 0 : a.size / a.each;
    int ns = 1;
    while (ns < a.each) ns *= 2;
    a.wide = a.each == ns && a.experts == 32 * ns && ns * sizeof(T) >= 16 &&
             (reinterpret_cast<uintptr_t>(a.logits) | (uintptr_t)(a.row_stride * (int64_t)sizeof(T))) % 16 == 0;
    a.wide_bias = a.each == ns && a.experts == 32 * ns && ns >= 4 && reinterpret_cast<uintptr_t>(a.bias) % 16 == 0;
    if (ns == 1) launch_route_slots<T, 1>(a, sigmoid, stream);
    else if (ns == 2) launch_route_slots<T, 2>(a, sigmoid, stream);
    else if (ns == 4) launch_route_slots<T, 4>(a, sigmoid, stream);
    else if (ns == 8) launch_route_slots<T, 8>(a, sigmoid, stream);
    else if (ns == 16) launch_route_slots<T, 16>(a, sigmoid, stream);
    else launch_route_slots<T, 32>(a, sigmoid, stream);
}

// ---- plan -----------------------------------------------------------------------------------

constexpr int kPlanCluster = 16;  // where the device places it; else the 8 that every one does
constexpr int kPlanAhead = 4;  // ids a lane has in flight

struct PlanArgs {
    const int32_t* ids;
    int pairs, k, experts;
    int32_t* order;
    int32_t* slots;
    int32_t* offsets;
};

// One CTA, or one cluster of them. Each warp owns a run of assignments and a row of counters: it
// counts its run's experts, the counters become the places before which this warp's assignments
// of each expert go (after those of earlier warps, earlier CTAs and lower experts), and it walks its
// run again in order, so that the sort is stable and no atomic decides a place. Bound by what an SM
// issues and scatters, so by how many SMs a cluster has: 131,072 assignments of 256 experts take 273
// us on one CTA (with a 64-bit division for each), 21 on a cluster of 8 and 14 on one of 16, the most
// there is; two launches with the counts in memory between them could use more SMs, for a workspace
// and a second launch. Equal ids by one ballot a bit: __match_any_sync took 25 us on the cluster of 8.
__global__ void __launch_bounds__(1024) plan_kernel(const __grid_constant__ PlanArgs a) {
    extern __shared__ int plan_smem[];
    __shared__ int scan[32];
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int threads = blockDim.x, warps = threads / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int* const totals = plan_smem;             // [experts] of this CTA, read by the others
    int* const base = totals + a.experts;      // [experts]
    int* const counts = base + a.experts;      // [warps][experts]
    int* const mine = counts + warp * a.experts;
    for (int e = lane; e < a.experts; e += 32) mine[e] = 0;
    __syncwarp();
    const int64_t run = (((int64_t)a.pairs + ranks * warps - 1) / (ranks * warps) + 31) & ~(int64_t)31;
    const int lo = (int)min((int64_t)a.pairs, run * (rank * warps + warp)), hi = (int)min((int64_t)a.pairs, lo + run);
    auto read = [&](int i) {
        const int id = i < hi ? __ldg(a.ids + i) : a.experts;
        return id >= 0 && id < a.experts ? id : a.experts;  // nobody's
    };
    const int bits = 32 - __clz(a.experts);
    for (int i0 = lo; i0 < hi; i0 += 32 * kPlanAhead) {
        int id[kPlanAhead];
#pragma unroll
        for (int q = 0; q < kPlanAhead; ++q) id[q] = read(i0 + 32 * q + lane);
#pragma unroll
        for (int q = 0; q < kPlanAhead; ++q)
            if (id[q] < a.experts) atomicAdd(mine + id[q], 1);
    }
    __syncthreads();
    for (int e = tid; e < a.experts; e += threads) {
        int total = 0;
        for (int w0 = 0; w0 < warps; w0 += 4) {  // warps come in fours
            int c[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) c[w] = counts[(w0 + w) * a.experts + e];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                counts[(w0 + w) * a.experts + e] = total;
                total += c[w];
            }
        }
        totals[e] = total;
    }
    // every expert's count over the CTAs, and over those before this one; a thread has a run of experts
    if (ranks > 1) cluster.sync();
    else __syncthreads();
    const int each = (a.experts + threads - 1) / threads;
    const int e0 = min(a.experts, tid * each), e1 = min(a.experts, e0 + each);
    int sum = 0;
    for (int e = e0; e < e1; ++e) {
        int before = 0, all = ranks > 1 ? 0 : totals[e];
        for (int r0 = 0; ranks > 1 && r0 < ranks; r0 += 8) {  // clusters are of 8 or 16
            int c[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) c[r] = *cluster.map_shared_rank(totals + e, r0 + r);
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                before += r0 + r < rank ? c[r] : 0;
                all += c[r];
            }
        }
        base[e] = sum + before;
        sum += all;
    }
    if (ranks > 1) cluster.barrier_arrive();  // the others' totals have been read
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    int first = incl - sum, kept = 0;
    for (int w = 0; w < warps; ++w) {
        first += w < warp ? scan[w] : 0;
        kept += scan[w];
    }
    for (int e = e0; e < e1; ++e) {
        base[e] += first;
        if (rank == 0) a.offsets[e] = base[e];  // nothing comes before the first CTA's
    }
    if (rank == 0 && tid == 0) a.offsets[a.experts] = kept;
    __syncthreads();
    for (int i0 = lo; i0 < hi; i0 += 32 * kPlanAhead) {
        int id[kPlanAhead];
#pragma unroll
        for (int q = 0; q < kPlanAhead; ++q) id[q] = read(i0 + 32 * q + lane);
#pragma unroll
        for (int q = 0; q < kPlanAhead; ++q) {
            const int i = i0 + 32 * q + lane;
            // the lanes with the same id, one ballot for each of its bits
            unsigned peers = 0xffffffffu;
            for (int b = 0; b < bits; ++b) {
                const bool on = id[q] >> b & 1;
                const unsigned who = __ballot_sync(0xffffffffu, on);
                peers &= on ? who : ~who;
            }
            int place = -1;
            if (id[q] < a.experts) place = base[id[q]] + mine[id[q]] + __popc(peers & ((1u << lane) - 1u));
            __syncwarp();
            if (id[q] < a.experts && lane == __ffs(peers) - 1) mine[id[q]] += __popc(peers);
            __syncwarp();
            if (i < hi) a.slots[i] = place;
            // below pairs always, but where another stream's call changes the ids between their two readings
            if ((unsigned)place < (unsigned)a.pairs) a.order[place] = (int)((unsigned)i / (unsigned)a.k);
        }
    }
    for (int64_t i = (int64_t)kept + rank * threads + tid; i < a.pairs; i += ranks * threads) a.order[i] = -1;
    if (ranks > 1) cluster.barrier_wait();  // no CTA leaves while its totals are read
}

// ---- combine --------------------------------------------------------------------------------

constexpr int kCombineThreads = 256;
constexpr int kCombineAhead = 4;  // results a thread has in flight

struct CombineArgs {
    const void* rows;
    int n_rows;
    int64_t row_stride;
    const float* weights;
    const int32_t* slots;
    int n, k, width;
    int per_cta;  // rows of a CTA
    void* out;
};

template <typename T, int VEC>
struct alignas(VEC * sizeof(T)) Pack {
    T v[VEC];
};

// A thread per row and VEC adjacent columns. Bound by memory: each result is read once. A row's loads
// wait for its slots, so many threads with few loads each serve better than the other way: 16,384 rows
// of 8 x 2048 bfloat16 took 117 us with 8 loads ahead, 104 with 4 CTAs of them forced on an SM, 91 (the
// memory's 6.6 TB/s) with 4 loads and 6 CTAs.
template <typename T, int VEC>
__global__ void __launch_bounds__(kCombineThreads, 6) combine_kernel(const __grid_constant__ CombineArgs a) {
    using P = Pack<T, VEC>;
    const unsigned cols = (unsigned)(a.width / VEC);
    const unsigned in_cta = a.per_cta > 1 ? threadIdx.x / cols : 0;
    const int64_t row = (int64_t)blockIdx.x * a.per_cta + in_cta;
    if (in_cta >= (unsigned)a.per_cta || row >= a.n) return;
    const float* weights = a.weights + row * a.k;
    const int32_t* slots = a.slots + row * a.k;
    for (unsigned c = a.per_cta > 1 ? threadIdx.x - in_cta * cols : blockIdx.y * kCombineThreads + threadIdx.x; c < cols;
         c += gridDim.y * kCombineThreads) {
        float sum[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[i] = 0.f;
        for (int j0 = 0; j0 < a.k; j0 += kCombineAhead) {
            P p[kCombineAhead];
            float w[kCombineAhead];
#pragma unroll
            for (int j = 0; j < kCombineAhead; ++j) {
                const int slot = j0 + j < a.k ? __ldg(slots + j0 + j) : -1;
                w[j] = 0.f;
#pragma unroll
                for (int i = 0; i < VEC; ++i) from_f32(0.f, &p[j].v[i]);
                if (slot >= 0 && slot < a.n_rows) {
                    w[j] = __ldg(weights + j0 + j);
                    p[j] = *reinterpret_cast<const P*>(static_cast<const T*>(a.rows) + slot * a.row_stride + (int64_t)c * VEC);
                }
            }
#pragma unroll
            for (int j = 0; j < kCombineAhead; ++j)
#pragma unroll
                for (int i = 0; i < VEC; ++i) sum[i] = __fmaf_rn(w[j], to_f32(p[j].v[i]), sum[i]);
        }
        P out;
#pragma unroll
        for (int i = 0; i < VEC; ++i) from_f32(sum[i], &out.v[i]);
        *reinterpret_cast<P*>(static_cast<T*>(a.out) + row * a.width + (int64_t)c * VEC) = out;
    }
}

template <typename T, int VEC>
void launch_combine_vec(CombineArgs a, cudaStream_t stream) {
    const int64_t cols = a.width / VEC;
    a.per_cta = cols < kCombineThreads ? (int)(kCombineThreads / cols) : 1;
    const dim3 grid((unsigned)(((int64_t)a.n + a.per_cta - 1) / a.per_cta),
                    (unsigned)std::min<int64_t>((cols + kCombineThreads - 1) / kCombineThreads, 65535));
    combine_kernel<T, VEC><<<grid, kCombineThreads, 0, stream>>>(a);
}

// The widest loads that every row's start, in and out, allows.
template <typename T>
void launch_combine_type(const CombineArgs& a, cudaStream_t stream) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.rows) | reinterpret_cast<uintptr_t>(a.out) |
                         (uintptr_t)(a.row_stride * (int64_t)sizeof(T)) | (uintptr_t)((int64_t)a.width * sizeof(T));
    if (at % 16 == 0) launch_combine_vec<T, 16 / sizeof(T)>(a, stream);
    else if (sizeof(T) == 2 && at % 4 == 0) launch_combine_vec<T, sizeof(T) == 2 ? 2 : 1>(a, stream);
    else launch_combine_vec<T, 1>(a, stream);
}

Status launched() {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? Status{SHIPK_OK, nullptr} : Status{SHIPK_ECUDA, cudaGetErrorString(e)};
}

}  // namespace

Status launch_route(const void* logits, int dtype, int rows, int experts, int64_t row_stride, const float* bias,
                    int top_k, int sigmoid, int groups, int top_groups, int group_top2, int renormalise, float scale,
                    float* weights, int32_t* ids, cudaStream_t stream) {
    const RouteArgs a{logits, rows, experts, row_stride, bias, top_k, groups, top_groups, group_top2,
                      renormalise, 0, 0, 0, 0, 0, scale, weights, ids};
    if (dtype == SHIPK_DTYPE_F32) launch_route_type<float>(a, sigmoid, stream);
    else if (dtype == SHIPK_DTYPE_F16) launch_route_type<__half>(a, sigmoid, stream);
    else launch_route_type<__nv_bfloat16>(a, sigmoid, stream);
    return launched();
}

// Whether a cluster of 16 of these CTAs fits the current device (it need not fit a part of one).
static bool wide_cluster_fits(cudaLaunchConfig_t config) {
    static std::mutex mu;
    static std::map<int, bool> known;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return false;
    std::lock_guard<std::mutex> lock(mu);
    const auto it = known.find(dev);
    if (it != known.end()) return it->second;
    const void* kernel = reinterpret_cast<const void*>(plan_kernel);
    int n = 0;
    config.blockDim = dim3(1024);
    config.dynamicSmemBytes = (size_t)(2 + 32) * kMaxExperts * sizeof(int);
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, kernel, &config) != cudaSuccess)
        cudaGetLastError();  // not fatal: the smaller cluster
    return known[dev] = n > 0;
}

Status launch_plan(const int32_t* ids, int rows, int k, int experts, int32_t* order, int32_t* slots, int32_t* offsets,
                   cudaStream_t stream) {
    const PlanArgs a{ids, rows * k, k, experts, order, slots, offsets};
    cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(plan_kernel), (2 + 32) * kMaxExperts * (int)sizeof(int));
    if (e != cudaSuccess) return Status{SHIPK_ECUDA, cudaGetErrorString(e)};
    cudaLaunchConfig_t config{};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {kPlanCluster, 1, 1};
    config.gridDim = dim3(kPlanCluster);
    config.stream = stream;
    config.attrs = &attr;
    config.numAttrs = 1;
    // a cluster once one CTA's warps would walk for long (CTA against cluster of 16 in us, 256 experts: 512
    // assignments 4.1 and 5.7, 2048 5.2 and 6.3, 4096 8.6 and 6.6); a warp for every 128 assignments
    const int ranks = a.pairs <= 2048 ? 1 : wide_cluster_fits(config) ? kPlanCluster : 8;
    const int64_t warps = ((int64_t)a.pairs / ranks + 127) / 128;
    const int threads = 128 * (int)std::min<int64_t>(std::max<int64_t>((warps + 3) / 4, 1), 8);
    attr.val.clusterDim.x = (unsigned)ranks;
    config.gridDim = dim3((unsigned)ranks);
    config.blockDim = dim3((unsigned)threads);
    config.dynamicSmemBytes = (size_t)(2 + threads / 32) * experts * sizeof(int);
    e = cudaLaunchKernelEx(&config, plan_kernel, a);
    const Status s = launched();
    return e == cudaSuccess ? s : Status{SHIPK_ECUDA, cudaGetErrorString(e)};
}

Status launch_combine(const void* in, int dtype, int n_in, int64_t row_stride, const float* weights, const int32_t* slots,
                      int rows, int k, int width, void* out, cudaStream_t stream) {
    const CombineArgs a{in, n_in, row_stride, weights, slots, rows, k, width, 1, out};
    if (dtype == SHIPK_DTYPE_F32) launch_combine_type<float>(a, stream);
    else if (dtype == SHIPK_DTYPE_F16) launch_combine_type<__half>(a, stream);
    else launch_combine_type<__nv_bfloat16>(a, stream);
    return launched();
}

}  // namespace shipk
