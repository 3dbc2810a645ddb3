// Token log-probabilities on the device: rows of scores over a vocabulary -> the log-probability
// of given tokens, the entropy of the row's distribution, and its top alternatives.
//
// Per row, with A the allowed tokens (bit set in the mask, or no mask; logit above -inf), m the
// largest logit of A and d = (x - m) / temperature:
//   S = sum over A of e^d;  log-probability of token t: d_t - log S;
//   entropy: log S - (sum over A of e^d d) / S;
//   alternatives: the `top` largest logits of A, equal ones by the lower id.
//
// One pass over the scores. Each thread keeps sums relative to a logit of its own (in base 2: the
// hardware's exponential), which it raises only when a logit is so far above it that the sums
// could overflow: a raise rescales them, as a running maximum would at every new one. Partial
// sums meet by one rescaling each. The same pass keeps each thread's largest logit and where it
// was. Those bound the alternatives: with t the top-th largest of the threads' maxima, at least
// `top` logits reach t, and only the threads whose own maximum does can hold them, so a second
// look at these few threads' places (from L2) collects every logit that reaches t, ranks the few
// dozen collected and has the alternatives exactly.
#include "heads.cuh"
#include "kernels.h"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace shipk {

namespace {

constexpr int kThreads = 256;  // per CTA
constexpr int kMaxCluster = 8;
constexpr int kUnroll = 4;     // 16-byte loads a thread has in flight

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

__device__ __forceinline__ void add_part(Part& r, const Part& a, float scale) {
    // a part that holds nothing adds nothing (its -inf would meet another); NaN sums stay NaN
    if (a.s == 0.f) return;
    const float d = fmaxf((a.m - r.m) * scale, -1e4f), e = exp2_fast(d);
    r.s += e * a.s;
    r.h += e * (a.h + d * a.s);
}
__device__ __forceinline__ Part join(const Part& a, const Part& b, float scale) {
    Part r{fmaxf(a.m, b.m), 0.f, 0.f};
    add_part(r, a, scale);
    add_part(r, b, scale);
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

__device__ __forceinline__ uint4 load_streaming(const uint4* p) {
    uint4 u;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                 : "l"(p));
    return u;
}

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
    static constexpr int kCollect = THREADS == 32 ? 256 : 1024;
    uint64_t keys[kCollect];  // the logits that reach the bound
    uint64_t chosen[kMaxTop];
    uint32_t ord[THREADS];    // order bits of the threads' maxima, 0: none
    int at[THREADS];          // and their granules
    uint16_t holder[THREADS]; // threads whose maximum reaches the bound
    Part parts[THREADS / 32];
    int holders, collected, last;
    uint32_t bound;
};

template <int THREADS>
__device__ __forceinline__ void group_sync() {
    if (THREADS == 32) __syncwarp();
    else __syncthreads();
}

// The bound (t, last): at least `top` of the threads' maxima are above t, or equal to t in a
// granule up to `last`, and few more: the search ends as soon as their number is within an eighth. Run by
// one warp. t = 0 when fewer than `top` threads have any logit.
template <int THREADS>
__device__ __forceinline__ void find_bound(Shared<THREADS>& g, int top, int lane) {
    constexpr int N = THREADS / 32;
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
    have = __reduce_add_sync(0xffffffffu, have);
    any = __reduce_or_sync(0xffffffffu, any);
    all = __reduce_and_sync(0xffffffffu, all);
    uint32_t t = 0;
    int last = 0x7fffffff;
    if (have >= top) {
        const int enough = top + top / 8;
        const uint32_t differ = any ^ all;
        int bit = differ ? 31 - __clz(differ) : -1;
        t = bit < 0 ? all : all & ~((2u << bit) - 1u);  // the bits they share; bit -1: all of them
        int reach = have;  // maxima that reach t
        for (; bit >= 0 && reach > enough; --bit) {
            const uint32_t u = t | (1u << bit);
            int n = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) n += o[i] >= u;
            n = __reduce_add_sync(0xffffffffu, n);
            if (n >= top) {
                t = u;
                reach = n;
            }
        }
        if (reach > enough) {  // many equal ones: those in the first granules
            int above = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) above += o[i] > t;
            above = __reduce_add_sync(0xffffffffu, above);
            int lo = -1, hi = 0x7fffffff;  // `last` in (lo, hi]
            while (hi - lo > 1) {
                const int mid = lo + (hi - lo) / 2;
                int n = 0;
#pragma unroll
                for (int i = 0; i < N; ++i) n += o[i] == t && g.at[lane + 32 * i] <= mid;
                n = __reduce_add_sync(0xffffffffu, n);
                if (above + n >= top) hi = mid;
                else lo = mid;
            }
            last = hi;
        }
    }
    if (lane == 0) {
        g.bound = t;
        g.last = last;
    }
}

// One group of THREADS threads per row (32: a warp), or, in clusters, per run of a row's granules.
template <typename T, int THREADS, bool MASK, bool CLUSTER>
__global__ void __launch_bounds__(kThreads, 4) logprobs_kernel(const __grid_constant__ Args a) {
    constexpr int kGroups = kThreads / THREADS;
    constexpr int kVec = Row<T, MASK>::kVec;
    __shared__ Shared<THREADS> shared[kGroups];
    __shared__ uint64_t cluster_keys[CLUSTER ? kMaxCluster * kMaxTop : 1];
    __shared__ Part cluster_parts[CLUSTER ? kMaxCluster : 1];
    const int group = threadIdx.x / THREADS, tid = threadIdx.x % THREADS, lane = tid & 31;
    Shared<THREADS>& g = shared[group];
    unsigned rank = 0, ranks = 1;
    int64_t row = (int64_t)blockIdx.x * kGroups + group;
    if (CLUSTER) {
        cg::cluster_group cluster = cg::this_cluster();
        rank = cluster.block_rank();
        ranks = cluster.num_blocks();
        row = blockIdx.x / ranks;
        cluster.barrier_arrive();  // every CTA runs before one writes into another's memory
    }
    if (row >= a.rows) return;  // a whole warp's row: groups of 32 share no barrier

    const Row<T, MASK> r(a, row);
    const int run = CLUSTER ? ((r.granules + (int)ranks - 1) / (int)ranks + 7) & ~7 : r.granules;
    const int g0 = min(r.granules, run * (int)rank), g1 = min(r.granules, g0 + run);

    // ---- one pass: sums and the largest logit
    float ref = -INFINITY, limit = -INFINITY, best = -INFINITY;
    int best_at = 0;
    float2 s2 = {0.f, 0.f}, h2 = {0.f, 0.f}, minus_ref = {0.f, 0.f};
    const float2 scale2 = {a.scale, a.scale};
    auto take = [&](float (&x)[kVec], int at) {
        float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
        if (kVec == 8) top = fmaxf(top, fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
        if (top > best) {
            best = top;
            best_at = at;
        }
        if (top > limit) {  // the first logit, or one far above the reference
            const float d = fmaxf((ref - top) * a.scale, -1e4f);
            if (ref > -INFINITY) {
                const float e = exp2_fast(d);
                h2 = {e * (h2.x + d * s2.x), e * (h2.y + d * s2.y)};
                s2 = {e * s2.x, e * s2.y};
            }
            ref = top;
            limit = top + a.headroom;
            minus_ref = {-top, -top};
        }
#pragma unroll
        for (int i = 0; i < kVec; i += 2) {
            // the difference first: a product with the scale may round away what is left of it
            float2 y = mul2(add2(float2{x[i], x[i + 1]}, minus_ref), scale2);
            y = {max_nan(y.x, kLowest), max_nan(y.y, kLowest)};
            const float2 e = {exp2_fast(y.x), exp2_fast(y.y)};
            s2 = add2(s2, e);
            h2 = fma2(e, y, h2);
        }
    };
    // the row's first and last granule, where values of other rows share them
    const bool first = tid == 0 && g0 < min(g1, r.full0);
    const bool final = tid == THREADS - 1 && g0 < g1 && r.full1 < g1 && r.full1 >= r.full0;
    if (first) {
        float x[kVec];
        r.read(0, x);
        take(x, 0);
    }
    {
        const int from = max(g0, r.full0), to = min(g1, r.full1);
        int at = from + tid;
        for (; at + (kUnroll - 1) * THREADS < to; at += kUnroll * THREADS) {
            uint4 u[kUnroll];
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) u[k] = load_streaming(r.base + at + k * THREADS);
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) {
                float x[kVec];
                unpack(u[k], x, r.x);
                r.cover(at + k * THREADS, x);
                take(x, at + k * THREADS);
            }
        }
        for (; at < to; at += THREADS) {
            float x[kVec];
            unpack(load_streaming(r.base + at), x, r.x);
            r.cover(at, x);
            take(x, at);
        }
    }
    if (final) {
        float x[kVec];
        r.read(g1 - 1, x);
        take(x, g1 - 1);
    }
    Part p{ref, s2.x + s2.y, h2.x + h2.y};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        p = join(p, Part{__shfl_xor_sync(0xffffffffu, p.m, o), __shfl_xor_sync(0xffffffffu, p.s, o),
                         __shfl_xor_sync(0xffffffffu, p.h, o)}, a.scale);
    if (THREADS > 32 && lane == 0) g.parts[tid / 32] = p;

    // ---- the alternatives of this group's granules, best first, into g.chosen
    const uint32_t ord = best > -INFINITY ? order_bits(best) : 0u;
    if (a.top > 0) {
        g.ord[tid] = ord;
        g.at[tid] = best_at;
        if (tid == 0) g.holders = g.collected = 0;
        for (int j = tid; j < a.top; j += THREADS) g.chosen[j] = 0;
    }
    group_sync<THREADS>();
    if (THREADS > 32) {
        p = g.parts[0];
        for (int w = 1; w < THREADS / 32; ++w) p = join(p, g.parts[w], a.scale);
    }
    if (a.top > 0) {
        if (tid < 32) find_bound<THREADS>(g, a.top, lane);
        group_sync<THREADS>();
        const uint32_t t = g.bound;
        const int last = g.last;
        if (ord > t || (ord == t && ord && best_at <= last)) g.holder[atomicAdd(&g.holders, 1)] = (uint16_t)tid;
        group_sync<THREADS>();
        // a thread's granules: its strided ones of the full run, and the edges of the row, which
        // the first and the last thread took
        const int from = max(g0, r.full0), to = min(g1, r.full1);
        const int steps = (max(0, to - from) + THREADS - 1) / THREADS + 2;
        const int looks = g.holders * steps;
        for (int q = tid; q < looks; q += THREADS) {
            const int h = g.holder[q / steps], k = q % steps;
            int at = from + h + (k - 2) * THREADS;
            bool own = k >= 2 && at < to;
            if (k == 0) at = 0, own = h == 0 && g0 < min(g1, r.full0);
            if (k == 1) at = g1 - 1, own = h == THREADS - 1 && g0 < g1 && r.full1 < g1 && r.full1 >= r.full0;
            if (!own) continue;
            float x[kVec];
            r.read(at, x);
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                if (!(x[i] > -INFINITY)) continue;
                const uint32_t o = order_bits(x[i]);
                if (o < t || (o == t && at > last)) continue;
                const int n = atomicAdd(&g.collected, 1);
                if (n < Shared<THREADS>::kCollect) g.keys[n] = choice_key(x[i], at * kVec - r.shift + i);
            }
        }
        group_sync<THREADS>();
        const int n = g.collected;
        if (n <= Shared<THREADS>::kCollect) {
            for (int i = tid; i < n; i += THREADS) {
                const uint64_t k = g.keys[i];
                int better = 0;
                for (int j = 0; j < n && better < a.top; ++j) better += g.keys[j] > k;
                if (better < a.top) g.chosen[better] = k;
            }
            group_sync<THREADS>();
        } else {
            // more than the group can hold reach the bound (large logits gathered in few threads'
            // places): the best below the one before, again and again
            uint64_t before = ~0ull;
            for (int j = 0; j < a.top && before; ++j) {
                uint64_t k = 0;
                for (int at = g0 + tid; at < g1; at += THREADS) {
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
                if (lane == 0) g.keys[tid / 32] = k;
                group_sync<THREADS>();
                for (int w = 0; w < THREADS / 32; ++w) k = g.keys[w] > k ? g.keys[w] : k;
                if (tid == 0) g.chosen[j] = k;
                before = k;
            }
            group_sync<THREADS>();
        }
    }

    // ---- a cluster's parts meet in its first CTA
    uint64_t* chosen = g.chosen;
    if (CLUSTER) {
        cg::cluster_group cluster = cg::this_cluster();
        cluster.barrier_wait();
        if (tid == 0) cluster.map_shared_rank(cluster_parts, 0)[rank] = p;
        uint64_t* keys = cluster.map_shared_rank(cluster_keys, 0);
        for (int j = tid; j < a.top; j += THREADS) keys[rank * a.top + j] = g.chosen[j];
        cluster.sync();
        if (rank) return;
        p = cluster_parts[0];
        for (unsigned w = 1; w < ranks; ++w) p = join(p, cluster_parts[w], a.scale);
        const int n = (int)ranks * a.top;
        for (int j = tid; j < a.top; j += THREADS) g.chosen[j] = 0;
        __syncthreads();
        for (int i = tid; i < n; i += THREADS) {
            const uint64_t k = cluster_keys[i];
            if (!k) continue;
            int better = 0;
            for (int j = 0; j < n && better < a.top; ++j) better += cluster_keys[j] > k;
            if (better < a.top) g.chosen[better] = k;
        }
        __syncthreads();
    }

    // ---- the row's results
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

constexpr int kWarpVocab = 4096;  // a warp takes rows of up to this many scores
constexpr int kWarpTop = 20;      // and this many alternatives of its 32 threads' maxima

template <typename T, bool MASK>
cudaError_t launch(const Args& a, cudaStream_t stream) {
    if (a.vocab <= kWarpVocab && a.top <= kWarpTop) {
        constexpr int rows = kThreads / 32;
        logprobs_kernel<T, 32, MASK, false><<<(unsigned)(((int64_t)a.rows + rows - 1) / rows), kThreads, 0, stream>>>(a);
        return cudaGetLastError();
    }
    int cluster = 1;
    while (cluster < kMaxCluster && (int64_t)a.rows * cluster < 148 * 8 && a.vocab / cluster > 4096) cluster *= 2;
    if (cluster == 1) {
        logprobs_kernel<T, kThreads, MASK, false><<<a.rows, kThreads, 0, stream>>>(a);
        return cudaGetLastError();
    }
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned)(a.rows * cluster));
    config.blockDim = dim3(kThreads);
    config.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {(unsigned)cluster, 1, 1};
    config.attrs = &attr;
    config.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&config, logprobs_kernel<T, kThreads, MASK, true>, a);
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
