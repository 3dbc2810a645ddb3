// Token log-probabilities on the device: rows of scores over a vocabulary -> the log-probability
// of given tokens, the entropy of the row's distribution, and its top alternatives.
//
// Per row, with A the allowed tokens (bit set in the mask, or no mask; logit above -inf), m the
// largest logit of A and d = (x - m) / temperature:
//   S = sum over A of e^d;  log-probability of token t: d_t - log S;
//   entropy: log S - (sum over A of e^d d) / S;
//   alternatives: the `top` largest logits of A, equal ones by the lower id.
//
// One pass over the scores, by a warp, a CTA or a cluster of CTAs per row. Each thread keeps sums
// relative to a logit of its own (in base 2: the hardware's exponential), which it raises only
// when a logit is so far above it that the sums could overflow: a raise rescales them, as a
// running maximum would at every new one. The threads' sums meet by one rescaling each.
//
// The alternatives come out of the same pass. It keeps each thread's largest logit, with its
// place, and a 16-bit mark for each run of granules that the thread read: the largest logit there. A
// bound t that at least `top` of the threads' maxima reach is reached by every alternative, and
// only runs whose mark reaches it can hold one. These few runs are read again (from L2), what
// reaches t is collected, and the few dozen collected are ranked.
#include "heads.cuh"
#include "kernels.h"

#include <cooperative_groups.h>

#include <algorithm>

namespace cg = cooperative_groups;

namespace shipk {

namespace {

constexpr int kThreads = 256;  // per CTA
constexpr int kMaxCluster = 8;
constexpr int kUnroll = 4;     // 16-byte loads of a stage
constexpr int kStages = 2;     // stages a thread has in flight
static_assert(kUnroll == 4, "a stage is 2^2 granules of a thread");

struct Args {
    const void* logits;
    int rows, vocab;
    int64_t row_stride;
    const int64_t* tokens;
    int n_tokens;
    const uint32_t* allowed;
    int64_t allowed_stride;
    float inv_t;    // 1 / temperature
    float scale;    // log2(e) / temperature
    float headroom; // a thread raises its reference when a logit is this far above it
    int top;
    float* logprobs;
    float* entropy;
    float* top_logprobs;
    int64_t* top_ids;
};

// A part of a row's sums relative to the logit m: of 2^y and of 2^y y, y = (x - m) scale.
struct Part {
    float m, s, h;
};

__device__ __forceinline__ float exp2_fast(float y) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y));
    return e;
}
// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Two 32-bit values to one instruction: a * b + c, a * b and a + b, each rounded once.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t&>(r))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t&>(r))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t&>(r))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return r;
}

// 2^y below this adds nothing to a sum that holds its reference; the clamp keeps 0 * -inf out.
constexpr float kLowest = -150.f;

// The parts of LANES neighbouring lanes as one, in each of them: their maximum first, then every
// part rescaled to it once, then plain sums.
template <int LANES>
__device__ __forceinline__ Part join(Part p, float scale) {
    uint32_t m = order_bits(p.m);
    if (LANES == 32) {
        m = __reduce_max_sync(0xffffffffu, m);
    } else {
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    }
    Part r{from_order_bits(m), 0.f, 0.f};
    if (!(p.s == 0.f)) {  // a part that holds nothing adds nothing (its -inf would meet another); NaN stays
        const float d = fmaxf((p.m - r.m) * scale, -1e4f), e = exp2_fast(d);
        r.s = e * p.s;
        r.h = e * (p.h + d * p.s);
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
        r.s += __shfl_xor_sync(0xffffffffu, r.s, o);
        r.h += __shfl_xor_sync(0xffffffffu, r.h, o);
    }
    return r;
}

// The 16 bytes at a granule of the row's memory as float values.
__device__ __forceinline__ void unpack(const uint4& u, float (&x)[4], const float*) {
    x[0] = __uint_as_float(u.x);
    x[1] = __uint_as_float(u.y);
    x[2] = __uint_as_float(u.z);
    x[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void unpack(const uint4& u, float (&x)[8], const __half*) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(reinterpret_cast<const __half2&>(w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void unpack(const uint4& u, float (&x)[8], const __nv_bfloat16*) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

__device__ __forceinline__ void copy_async(uint4* to, const uint4* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from)
                 : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A row's memory in 16-byte granules from the one that holds its first value: granule g holds
// the values [g kVec - shift, (g + 1) kVec - shift) of the row, those of the first and the last
// granule that lie outside it excepted.
template <typename T, bool MASK>
struct Row {
    static constexpr int kVec = 16 / sizeof(T);
    const T* x;
    const uint4* base;
    const uint32_t* allowed;
    int vocab, shift, granules, full0, full1;  // granules [full0, full1) hold kVec values each

    __device__ __forceinline__ Row(const Args& a, int64_t row) {
        x = static_cast<const T*>(a.logits) + row * a.row_stride;
        const uintptr_t at = reinterpret_cast<uintptr_t>(x);
        base = reinterpret_cast<const uint4*>(at & ~(uintptr_t)15);
        shift = (int)(at & 15) / (int)sizeof(T);
        vocab = a.vocab;
        granules = (shift + vocab + kVec - 1) / kVec;
        full0 = shift ? 1 : 0;
        full1 = (shift + vocab) / kVec;
        allowed = MASK ? a.allowed + row * a.allowed_stride : nullptr;
    }
    __device__ __forceinline__ bool on(int v) const { return !MASK || ((__ldg(allowed + (v >> 5)) >> (v & 31)) & 1u); }
    __device__ __forceinline__ float logit(int v) const { return on(v) ? to_f32(x[v]) : -INFINITY; }
    __device__ __forceinline__ uint32_t bits(int g) const {  // of a full granule
        const int v = g * kVec - shift, off = v & 31;
        const uint32_t* w = allowed + (v >> 5);
        return __funnelshift_r(__ldg(w), off + kVec > 32 ? __ldg(w + 1) : 0u, off);
    }
    __device__ __forceinline__ void cover(int g, float (&v)[kVec]) const {
        if (MASK) {
            const uint32_t b = bits(g);
#pragma unroll
            for (int i = 0; i < kVec; ++i) v[i] = (b >> i) & 1u ? v[i] : -INFINITY;
        }
    }
    // any granule; -inf outside the row
    __device__ __forceinline__ void read(int g, float (&v)[kVec]) const {
        if (g >= full0 && g < full1) {
            unpack(__ldg(base + g), v, x);
            cover(g, v);
            return;
        }
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            const int k = g * kVec - shift + i;
            v[i] = k >= 0 && k < vocab ? logit(k) : -INFINITY;
        }
    }
};

// What a group of THREADS threads shares while it works on a row (or a cluster's part of one).
template <int THREADS>
struct Shared {
    static constexpr int kCollect = THREADS == 32 ? 128 : 512;
    static constexpr int kMarks = THREADS == 32 ? 8 : 16;  // of a thread
    uint64_t keys[kCollect];           // the logits that reach the bound
    uint64_t chosen[kMaxTop];
    uint64_t rounds[THREADS / 32];     // a warp's contribution to the bound
    Part parts[THREADS / 32];
    uint32_t ord[THREADS];             // order bits of the threads' maxima, 0: none
    int at[THREADS];                   // and their granules
    uint16_t marks[kMarks * THREADS];  // upper half of the order bits of a run's largest logit
    uint16_t runs[kCollect];           // marked runs to read again: mark * THREADS + thread
    int marked, collected;
    uint64_t bound;
};

template <int THREADS>
__device__ __forceinline__ void group_sync() {
    if (THREADS == 32) __syncwarp();
    else __syncthreads();
}

// A bound is a key: order bits of a logit, then its granule, the lower the better. What reaches it
// is a larger logit, or the same one in that granule or before; 0 is reached by every logit.
__device__ __forceinline__ uint64_t bound_key(uint32_t ord, int at) {
    return ord ? ((uint64_t)ord << 32) | (0xffffffffu - (uint32_t)at) : 0;
}

// A bound that at least `wanted` of the threads' maxima reach, and few more: the search ends as soon
// as their number is within an eighth. Run by one warp, on g.ord and g.at. 0 when fewer than `wanted` threads
// have any logit.
template <int THREADS>
__device__ __forceinline__ uint64_t find_bound(const Shared<THREADS>& g, int wanted, int lane) {
    constexpr int N = THREADS / 32;
    auto sum = [](int n) {
        if constexpr (N == 1) return __popc(__ballot_sync(0xffffffffu, n));
        else return __reduce_add_sync(0xffffffffu, n);
    };
    uint32_t o[N];
    uint32_t any = 0, all = ~0u;
    int have = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        o[i] = g.ord[lane + 32 * i];
        if (o[i]) {
            any |= o[i];
            all &= o[i];
            ++have;
        }
    }
    have = sum(have);
    if (have < wanted) return 0;
    any = __reduce_or_sync(0xffffffffu, any);
    all = __reduce_and_sync(0xffffffffu, all);
    const int enough = wanted + wanted / 8;
    const uint32_t differ = any ^ all;
    int bit = differ ? 31 - __clz(differ) : -1;
    uint32_t t = bit < 0 ? all : all & ~((2u << bit) - 1u);  // the bits they share; bit -1: all of them
    int reach = have;
    for (; bit >= 0 && reach > enough; --bit) {
        const uint32_t u = t | (1u << bit);
        int n = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) n += o[i] >= u;
        n = sum(n);
        if (n >= wanted) {
            t = u;
            reach = n;
        }
    }
    int last = 0x7fffffff;
    if (reach > enough) {  // many equal ones: those in the first granules
        int above = 0, lo = 0x7fffffff, hi = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            above += o[i] > t;
            if (o[i] == t) {
                lo = min(lo, g.at[lane + 32 * i]);
                hi = max(hi, g.at[lane + 32 * i]);
            }
        }
        above = sum(above);
        lo = __reduce_min_sync(0xffffffffu, lo) - 1;
        last = __reduce_max_sync(0xffffffffu, hi);
        while (last - lo > 1 && reach > enough) {  // those up to `last` suffice, those up to `lo` do not
            const int mid = lo + (last - lo) / 2;
            int n = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) n += o[i] == t && g.at[lane + 32 * i] <= mid;
            n = above + sum(n);
            if (n >= wanted) {
                last = mid;
                reach = n;
            } else {
                lo = mid;
            }
        }
    }
    return bound_key(t, last);
}

// The same for a group of several warps without a search: with q = wanted / warps rounded up, the least
// of the warps' q-th largest maxima. Looser (some two times `wanted` reach it), far shorter. 0 when a
// warp has fewer than q. The warp's part: its q-th largest.
__device__ __forceinline__ uint64_t nth_largest(uint32_t ord, int at, int q, int lane) {
    uint32_t high = 0;
    int low = 0;
    for (int i = 0; i < q; ++i) {
        high = __reduce_max_sync(0xffffffffu, ord);
        low = __reduce_min_sync(0xffffffffu, ord == high ? at : 0x7fffffff);
        if (ord == high && at == low) ord = 0;
    }
    return bound_key(high, low);
}

template <int VEC>
__device__ __forceinline__ float largest(const float (&x)[VEC]) {
    const float m = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    if constexpr (VEC == 8) return fmaxf(m, fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
    return m;
}

// What a thread has of a row's sums and its largest logit while it reads its granules.
template <int VEC>
struct Running {
    float ref = -INFINITY, limit = -INFINITY, best = -INFINITY;
    int best_at = 0;
    float2 s2 = {0.f, 0.f}, h2 = {0.f, 0.f}, minus_ref = {0.f, 0.f};

    __device__ __forceinline__ float take(const float (&x)[VEC], int at, float scale, float headroom) {
        const float top = largest(x);
        if (top > best) {
            best = top;
            best_at = at;
        }
        if (top > limit) {  // the first logit, or one far above the reference
            const float d = fmaxf((ref - top) * scale, -1e4f);
            if (ref > -INFINITY) {
                const float e = exp2_fast(d);
                h2 = {e * (h2.x + d * s2.x), e * (h2.y + d * s2.y)};
                s2 = {e * s2.x, e * s2.y};
            }
            ref = top;
            limit = top + headroom;
            minus_ref = {-top, -top};
        }
        const float2 scale2 = {scale, scale};
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
            // the difference first: a product with the scale may round away what is left of it
            float2 y = mul2(add2(float2{x[i], x[i + 1]}, minus_ref), scale2);
            y = {max_nan(y.x, kLowest), max_nan(y.y, kLowest)};
            const float2 e = {exp2_fast(y.x), exp2_fast(y.y)};
            s2 = add2(s2, e);
            h2 = fma2(e, y, h2);
        }
        return top;
    }
    __device__ __forceinline__ Part part() const { return Part{ref, s2.x + s2.y, h2.x + h2.y}; }
};

// The granules [g0, g1) of a row that a group works on: the full ones in strides of THREADS, and
// the row's first and last one, where they are shared with other rows, by the first and the last
// thread.
template <typename T, bool MASK, int THREADS>
struct Run {
    int g0, g1, from, to;

    __device__ __forceinline__ Run(const Row<T, MASK>& r, unsigned rank, unsigned ranks) {
        const int each = ranks == 1 ? r.granules : ((r.granules + (int)ranks - 1) / (int)ranks + 7) & ~7;
        g0 = min(r.granules, each * (int)rank);
        g1 = min(r.granules, g0 + each);
        from = max(g0, r.full0);
        to = min(g1, r.full1);
    }
    __device__ __forceinline__ bool first(const Row<T, MASK>& r, int thread) const {
        return thread == 0 && g0 < min(g1, r.full0);
    }
    __device__ __forceinline__ bool last(const Row<T, MASK>& r, int thread) const {
        return thread == THREADS - 1 && g0 < g1 && r.full1 < g1 && r.full1 >= r.full0;
    }
};

// The alternatives among a run's granules into g.chosen, best first, 0 past the last; called by the
// whole group with each thread's largest logit and its granule, which are in g.ord and g.at, and, for
// more than one warp, with the warps' parts of the bound in g.rounds. `marks` runs of 2^shift granules of each thread have marks.
template <typename T, bool MASK, int THREADS>
__device__ __forceinline__ void choose(Shared<THREADS>& g, const Row<T, MASK>& r, const Run<T, MASK, THREADS>& run,
                                       int wanted, int tid, uint32_t ord, int best_at, int marks, int shift) {
    constexpr int kVec = Row<T, MASK>::kVec;
    constexpr int kWarps = THREADS / 32;
    const int lane = tid & 31, warp = tid / 32;
    uint64_t bound;
    if (kWarps == 1) {
        bound = find_bound<THREADS>(g, wanted, lane);
    } else {
        bound = g.rounds[0];
        for (int w = 1; w < kWarps; ++w) bound = min(bound, g.rounds[w]);
        if (!bound) {  // warps with few logits, or none: uniform over the group
            if (warp == 0) {
                bound = find_bound<THREADS>(g, wanted, lane);
                if (lane == 0) g.bound = bound;
            }
            group_sync<THREADS>();
            bound = g.bound;
        }
    }
    const uint32_t t = (uint32_t)(bound >> 32);
    const int last = key_index(bound);
    auto look = [&](const float (&x)[kVec], int at) {
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            if (!(x[i] > -INFINITY)) continue;
            const uint32_t o = order_bits(x[i]);
            if (o < t || (o == t && at > last)) continue;
            const int n = atomicAdd(&g.collected, 1);
            if (n < Shared<THREADS>::kCollect) g.keys[n] = choice_key(x[i], at * kVec - r.shift + i);
        }
    };
    if (ord && bound_key(ord, best_at) >= bound) {
        for (int m = 0; m < marks; ++m) {
            if (g.marks[m * THREADS + tid] < t >> 16) continue;
            const int n = atomicAdd(&g.marked, 1);
            if (n < Shared<THREADS>::kCollect) g.runs[n] = (uint16_t)(m * THREADS + tid);
        }
        if (run.first(r, tid) || run.last(r, tid)) {
            float x[kVec];
            const int at = tid == 0 ? 0 : run.g1 - 1;
            r.read(at, x);
            look(x, at);
        }
    }
    group_sync<THREADS>();
    const int looks = min(g.marked, Shared<THREADS>::kCollect) << shift;
    for (int q = tid; q < looks; q += THREADS) {
        const int of = g.runs[q >> shift], k = q & ((1 << shift) - 1);
        const int at = run.from + of % THREADS + (((of / THREADS) << shift) + k) * THREADS;
        if (at >= run.to) continue;
        float x[kVec];
        unpack(__ldg(r.base + at), x, r.x);
        r.cover(at, x);
        look(x, at);
    }
    group_sync<THREADS>();
    const int n = g.collected;
    if (n <= Shared<THREADS>::kCollect && g.marked <= Shared<THREADS>::kCollect) {
        for (int i = tid; i < n; i += THREADS) {
            const uint64_t k = g.keys[i];
            int better = 0;
            for (int j = 0; j < n; ++j) better += g.keys[j] > k;
            if (better < wanted) g.chosen[better] = k;
        }
    } else {
        // more than the group can hold reach the bound (large logits gathered in few threads'
        // places): the best below the one before, again and again
        uint64_t before = ~0ull;
        for (int j = 0; j < wanted && before; ++j) {
            uint64_t k = 0;
            for (int at = run.g0 + tid; at < run.g1; at += THREADS) {
                float x[kVec];
                r.read(at, x);
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    if (!(x[i] > -INFINITY)) continue;
                    const uint64_t c = choice_key(x[i], at * kVec - r.shift + i);
                    if (c < before && c > k) k = c;
                }
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const uint64_t c = __shfl_xor_sync(0xffffffffu, k, o);
                k = c > k ? c : k;
            }
            group_sync<THREADS>();
            if (lane == 0) g.keys[warp] = k;
            group_sync<THREADS>();
            for (int w = 0; w < kWarps; ++w) k = g.keys[w] > k ? g.keys[w] : k;
            if (tid == 0) g.chosen[j] = k;
            before = k;
        }
    }
    group_sync<THREADS>();
}

// The row's results from its sums and its alternatives' keys.
template <typename T, bool MASK, int THREADS>
__device__ __forceinline__ void write_row(const Args& a, const Row<T, MASK>& r, int64_t row, const Part& p,
                                          const uint64_t* chosen, int tid) {
    const bool empty = p.s == 0.f;
    const float log_s = empty ? 0.f : logf(p.s);
    auto logprob = [&](float x) {
        if (empty || (x == -INFINITY && p.s == p.s)) return -INFINITY;
        return (x - p.m) * a.inv_t - log_s;  // NaN where S is
    };
    if (tid == 0) a.entropy[row] = empty ? 0.f : log_s - 0.693147180559945f * (p.h / p.s);
    for (int j = tid; j < a.n_tokens; j += THREADS) {
        const int64_t t = a.tokens[row * a.n_tokens + j];
        a.logprobs[row * a.n_tokens + j] = t < 0 ? 0.f : t >= a.vocab ? NAN : logprob(r.logit((int)t));
    }
    for (int j = tid; j < a.top; j += THREADS) {
        const uint64_t k = chosen[j];
        a.top_ids[row * a.top + j] = k ? key_index(k) : -1;
        a.top_logprobs[row * a.top + j] = k ? logprob(key_value(k)) : -INFINITY;
    }
}

// A group of THREADS threads per row: a warp, a CTA, or (CLUSTER) a CTA for each part of a row.
// Groups walk over the rows. Each thread copies its granules into places of its own in shared
// memory, kStages stages of kUnroll ahead of where it reads, past the end of a row into the next
// one: what a row needs beyond its pass runs while the next row arrives. No thread reads what
// another copied, so the copies need no barrier.
template <typename T, int THREADS, bool MASK, bool CLUSTER>
__global__ void __launch_bounds__(kThreads, 4) logprobs_kernel(const __grid_constant__ Args a) {
    constexpr int kVec = Row<T, MASK>::kVec;
    constexpr int kWarps = THREADS / 32, kGroups = kThreads / THREADS;
    extern __shared__ uint4 rings[];  // [kGroups][kStages][kUnroll][THREADS]
    __shared__ Shared<THREADS> shared[kGroups];
    __shared__ uint64_t cluster_keys[CLUSTER ? kMaxCluster * kMaxTop : 1];
    __shared__ Part cluster_parts[CLUSTER ? kMaxCluster : 1];
    const int group = threadIdx.x / THREADS, tid = threadIdx.x % THREADS, lane = tid & 31;
    Shared<THREADS>& g = shared[group];
    uint4* const ring = rings + group * kStages * kUnroll * THREADS + tid;
    unsigned part = 0, parts = 1;
    if (CLUSTER) {
        cg::cluster_group cluster = cg::this_cluster();
        part = cluster.block_rank();
        parts = cluster.num_blocks();
        cluster.barrier_arrive();  // every CTA runs before one writes into another's memory
    }
    const int64_t first = CLUSTER ? blockIdx.x / parts : (int64_t)blockIdx.x * kGroups + group;
    const int64_t step = CLUSTER ? gridDim.x / parts : (int64_t)gridDim.x * kGroups;

    // the next stage to copy: of row `ahead`, granules from `next` to `end`
    int64_t ahead = first;
    const uint4* ahead_base = nullptr;
    int next = 0, end = 0;
    auto enter = [&]() {
        const Row<T, MASK> r(a, ahead);
        const Run<T, MASK, THREADS> run(r, part, parts);
        ahead_base = r.base + tid;
        next = run.from;
        end = run.to;
    };
    if (ahead < a.rows) enter();
    auto copy_stage = [&](int stage) {
        while (ahead < a.rows && next >= end) {
            ahead += step;
            if (ahead < a.rows) enter();
        }
        if (ahead < a.rows) {
#pragma unroll
            for (int k = 0; k < kUnroll; ++k)
                if (next + k * THREADS + tid < end)
                    copy_async(ring + (stage * kUnroll + k) * THREADS, ahead_base + next + k * THREADS);
            next += kUnroll * THREADS;
        }
        copies_commit();
    };
#pragma unroll
    for (int k = 0; k < kStages; ++k) copy_stage(k);
    int stage = 0;

    for (int64_t row = first; row < a.rows; row += step) {
        const Row<T, MASK> r(a, row);
        const Run<T, MASK, THREADS> run(r, part, parts);
        Running<kVec> sums;
        float x[kVec];
        if (run.first(r, tid)) {
            r.read(0, x);
            sums.take(x, 0, a.scale, a.headroom);
        }
        // marks of 2^per stages each
        const int stages = (max(0, run.to - run.from) + kUnroll * THREADS - 1) / (kUnroll * THREADS);
        const int per = stages > Shared<THREADS>::kMarks ? 32 - __clz((stages - 1) / Shared<THREADS>::kMarks) : 0;
        float marked = -INFINITY;
        for (int k0 = 0; k0 < stages; ++k0) {
            copies_wait<kStages - 1>();
            const uint4* held = ring + stage * kUnroll * THREADS;
            const int at = run.from + k0 * kUnroll * THREADS + tid;
            if (at - tid + kUnroll * THREADS <= run.to) {
#pragma unroll
                for (int k = 0; k < kUnroll; ++k) {
                    unpack(held[k * THREADS], x, r.x);
                    r.cover(at + k * THREADS, x);
                    marked = fmaxf(marked, sums.take(x, at + k * THREADS, a.scale, a.headroom));
                }
            } else {
                for (int k = 0; k < kUnroll && at + k * THREADS < run.to; ++k) {
                    unpack(held[k * THREADS], x, r.x);
                    r.cover(at + k * THREADS, x);
                    marked = fmaxf(marked, sums.take(x, at + k * THREADS, a.scale, a.headroom));
                }
            }
            copy_stage(stage);
            stage = stage + 1 == kStages ? 0 : stage + 1;
            if (((k0 + 1) & ((1 << per) - 1)) == 0 || k0 + 1 == stages) {
                g.marks[(k0 >> per) * THREADS + tid] = (uint16_t)(order_bits(marked) >> 16);
                marked = -INFINITY;
            }
        }
        if (run.last(r, tid)) {
            r.read(run.g1 - 1, x);
            sums.take(x, run.g1 - 1, a.scale, a.headroom);
        }
        Part p = join<32>(sums.part(), a.scale);
        const uint32_t ord = sums.best > -INFINITY ? order_bits(sums.best) : 0u;
        if (kWarps > 1 && lane == 0) g.parts[tid / 32] = p;
        if (a.top > 0) {
            g.ord[tid] = ord;
            g.at[tid] = sums.best_at;
            if (tid == 0) g.marked = g.collected = 0;
            for (int j = tid; j < a.top; j += THREADS) g.chosen[j] = 0;
            if (kWarps > 1) {
                const uint64_t nth = nth_largest(ord, sums.best_at, (a.top + kWarps - 1) / kWarps, lane);
                if (lane == 0) g.rounds[tid / 32] = nth;
            }
        }
        group_sync<THREADS>();
        if (kWarps > 1) p = join<kWarps>(g.parts[lane % kWarps], a.scale);
        if (a.top > 0)
            choose<T, MASK, THREADS>(g, r, run, a.top, tid, ord, sums.best_at, (stages + (1 << per) - 1) >> per,
                                     per + 2);
        if (CLUSTER) {  // its parts meet in its first CTA
            cg::cluster_group cluster = cg::this_cluster();
            cluster.barrier_wait();
            if (tid == 0) cluster.map_shared_rank(cluster_parts, 0)[part] = p;
            uint64_t* keys = cluster.map_shared_rank(cluster_keys, 0);
            for (int j = tid; j < a.top; j += THREADS) keys[part * a.top + j] = g.chosen[j];
            cluster.sync();
            if (part) return;
            p = join<kMaxCluster>(lane % kMaxCluster < parts ? cluster_parts[lane % kMaxCluster]
                                                             : Part{-INFINITY, 0.f, 0.f}, a.scale);
            const int n = (int)parts * a.top;
            for (int j = tid; j < a.top; j += THREADS) g.chosen[j] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += THREADS) {
                const uint64_t k = cluster_keys[i];
                int better = 0;
                for (int j = 0; j < n; ++j) better += cluster_keys[j] > k;
                if (k && better < a.top) g.chosen[better] = k;
            }
            __syncthreads();
        }
        write_row<T, MASK, THREADS>(a, r, row, p, g.chosen, tid);
        if (CLUSTER) return;    // one row for a cluster
        group_sync<THREADS>();  // the next row's threads write where this row's read
    }
}

constexpr int kSms = 148;
constexpr int kCtas = 4;          // per SM, by the launch bounds and the rings
constexpr int kWarpVocab = 4096;  // a warp takes rows of up to this many scores
constexpr int kWarpTop = 20;      // and this many alternatives of its 32 threads' maxima

template <typename T, bool MASK>
cudaError_t launch(const Args& a, cudaStream_t stream) {
    constexpr int ring = kStages * kUnroll * kThreads * (int)sizeof(uint4);
    if (a.vocab <= kWarpVocab && a.top <= kWarpTop) {
        constexpr int rows = kThreads / 32;
        auto kernel = logprobs_kernel<T, 32, MASK, false>;
        const cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kernel), ring);
        if (e != cudaSuccess) return e;
        const int64_t ctas = std::min<int64_t>(((int64_t)a.rows + rows - 1) / rows, kSms * kCtas);
        kernel<<<(unsigned)ctas, kThreads, ring, stream>>>(a);
        return cudaGetLastError();
    }
    int cluster = 1;
    while (cluster < kMaxCluster && (int64_t)a.rows * cluster < kSms * 8 && a.vocab / cluster > 4096) cluster *= 2;
    if (cluster == 1) {
        auto kernel = logprobs_kernel<T, kThreads, MASK, false>;
        const cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kernel), ring);
        if (e != cudaSuccess) return e;
        kernel<<<std::min(a.rows, kSms * kCtas), kThreads, ring, stream>>>(a);
        return cudaGetLastError();
    }
    auto kernel = logprobs_kernel<T, kThreads, MASK, true>;
    cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kernel), ring);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned)(a.rows * cluster));
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = ring;
    config.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {(unsigned)cluster, 1, 1};
    config.attrs = &attr;
    config.numAttrs = 1;
    e = cudaLaunchKernelEx(&config, kernel, a);
    const cudaError_t last = cudaGetLastError();
    return e != cudaSuccess ? e : last;
}

template <typename T>
cudaError_t launch(const Args& a, cudaStream_t stream) {
    return a.allowed ? launch<T, true>(a, stream) : launch<T, false>(a, stream);
}

}  // namespace

Status launch_token_logprobs(const void* logits, int dtype, int rows, int vocab, int64_t row_stride,
                             const int64_t* tokens, int n_tokens, const uint32_t* allowed, int64_t allowed_stride,
                             float temperature, int top, float* logprobs, float* entropy, float* top_logprobs,
                             int64_t* top_ids, cudaStream_t stream) {
    const float scale = 1.44269504088896f / temperature;
    // The headroom is 40 in base 2, and at most twice that once reference + headroom is rounded:
    // sums of 2^25 terms of up to 2^80, and of y times as much, stay finite.
    const Args a{logits, rows, vocab, row_stride, tokens, n_tokens, allowed, allowed_stride, 1.f / temperature, scale,
                 40.f / scale, top, logprobs, entropy, top_logprobs, top_ids};
    const cudaError_t e = dtype == SHIPK_DTYPE_F32   ? launch<float>(a, stream)
                          : dtype == SHIPK_DTYPE_F16 ? launch<__half>(a, stream)
                                                     : launch<__nv_bfloat16>(a, stream);
    return e == cudaSuccess ? Status{SHIPK_OK, nullptr} : Status{SHIPK_ECUDA, cudaGetErrorString(e)};
}

}  // namespace shipk
