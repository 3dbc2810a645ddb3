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
// when a logit is well above it: a raise rescales them, as a running maximum would at every new one. The threads' sums meet by one rescaling each.
//
// The alternatives come out of the same pass. It keeps each thread's largest logit, and a 16-bit
// mark for each run of granules that the thread read: the upper half of the largest logit there. A
// bound t that at least `top` of the threads' maxima reach is reached by every alternative, and
// only runs whose mark reaches it can hold one. These few runs are read again (from L2), what
// reaches t is collected, and the few dozen collected are ranked.
#include "heads.cuh"
#include "kernels.h"

#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

namespace cg = cooperative_groups;

namespace shipk {

namespace {

constexpr int kWarpCta = 256;  // threads of a CTA whose warps each have a row of their own
constexpr int kMaxCluster = 8;
constexpr int kUnroll = 4;     // granules (16 bytes) of a thread in a stage
constexpr int kUnrollLog = 2;
constexpr int kStages = 2;     // stages a thread has in flight
static_assert(kUnroll == 1 << kUnrollLog, "");
constexpr int kTurns = 8;      // of tightening a bound
constexpr int kMaxRounds = kMaxTop / 8 + 4;  // maxima that a warp of eight offers for the bound

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

// Two 32-bit values to one instruction: a * b + c and a + b, each rounded once.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t&>(r))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t&>(r))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return r;
}

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

// ---- 16 bytes of scores: one granule ----------------------------------------------------------

// Bits 0 to 3 as the signs of a word's bytes, which a byte permutation spreads over a score.
__device__ __forceinline__ uint32_t byte_signs(uint32_t bits) { return ((bits & 15u) * 0x10204080u) & 0x80808080u; }
template <uint32_t SELECTOR>  // a nibble above 7: the sign of that byte, eight times
__device__ __forceinline__ uint32_t spread(uint32_t signs) {
    uint32_t r;
    asm("prmt.b32 %0, %1, 0, %2;" : "=r"(r) : "r"(signs), "n"(SELECTOR));
    return r;
}
__device__ __forceinline__ uint32_t pick(uint32_t on, uint32_t off, uint32_t mask) { return (on & mask) | (off & ~mask); }

template <typename T>
struct Granule;

// 32-bit scores. What has no probability has its y clamped: 2^y is 0 then, and y 2^y no NaN.
template <>
struct Granule<float> {
    static constexpr int kVec = 4;
    static __device__ __forceinline__ uint4 empty() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
    static __device__ __forceinline__ void unpack(const uint4& u, float (&x)[4]) {
        x[0] = __uint_as_float(u.x);
        x[1] = __uint_as_float(u.y);
        x[2] = __uint_as_float(u.z);
        x[3] = __uint_as_float(u.w);
    }
    static __device__ __forceinline__ float largest(const uint4 (&u)[kUnroll]) {
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < kUnroll; ++k)
            m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(u[k].x), __uint_as_float(u[k].y)),
                               fmaxf(__uint_as_float(u[k].z), __uint_as_float(u[k].w))));
        return m;
    }
    // y = x scale + offset of each score, at least -150
    static __device__ __forceinline__ void scaled(const uint4& u, float2 scale, float2 offset, float2 (&y)[2]) {
        y[0] = fma2(float2{__uint_as_float(u.x), __uint_as_float(u.y)}, scale, offset);
        y[1] = fma2(float2{__uint_as_float(u.z), __uint_as_float(u.w)}, scale, offset);
#pragma unroll
        for (int i = 0; i < 2; ++i) y[i] = {max_nan(y[i].x, -150.f), max_nan(y[i].y, -150.f)};
    }
    // whether scaled() may be used with a reference: x scale does not overflow above, -inf is no trouble
    static __device__ __forceinline__ bool plain(float, float) { return true; }
    static __device__ __forceinline__ uint4 cover(const uint4& u, uint32_t bits) {
        const uint32_t signs = byte_signs(bits), none = 0xff800000u;
        return make_uint4(pick(u.x, none, spread<0x8888>(signs)), pick(u.y, none, spread<0x9999>(signs)),
                          pick(u.z, none, spread<0xaaaa>(signs)), pick(u.w, none, spread<0xbbbb>(signs)));
    }
};

// 16-bit scores, two to a register: the maximum and the clamp at `kLow` are taken on both at once.
template <typename T>
struct Granule16 {
    static constexpr int kVec = 8;
    static __device__ __forceinline__ uint4 empty() { return make_uint4(T::kNone, T::kNone, T::kNone, T::kNone); }
    static __device__ __forceinline__ void unpack(const uint4& u, float (&x)[8]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = T::both(w[i]);
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ float largest(const uint4 (&u)[kUnroll]) {
        uint32_t m = T::max2(T::max2(u[0].x, u[0].y), T::max2(u[0].z, u[0].w));
#pragma unroll
        for (int k = 1; k < kUnroll; ++k)
            m = T::max2(m, T::max2(T::max2(u[k].x, u[k].y), T::max2(u[k].z, u[k].w)));
        const float2 f = T::both(m);
        return fmaxf(fmaxf(f.x, f.y), -INFINITY);
    }
    static __device__ __forceinline__ void scaled(const uint4& u, float2 scale, float2 offset, float2 (&y)[4]) {
        y[0] = fma2(T::both(T::raise(u.x)), scale, offset);
        y[1] = fma2(T::both(T::raise(u.y)), scale, offset);
        y[2] = fma2(T::both(T::raise(u.z)), scale, offset);
        y[3] = fma2(T::both(T::raise(u.w)), scale, offset);
    }
    // with this reference, a score at the clamp or below has no probability
    static __device__ __forceinline__ bool plain(float ref, float scale) { return (T::kLow - ref) * scale < -150.f; }
    static __device__ __forceinline__ uint4 cover(const uint4& u, uint32_t bits) {
        const uint32_t low = byte_signs(bits), high = byte_signs(bits >> 4);
        return make_uint4(pick(u.x, T::kNone, spread<0x9988>(low)), pick(u.y, T::kNone, spread<0xbbaa>(low)),
                          pick(u.z, T::kNone, spread<0x9988>(high)),
                          pick(u.w, T::kNone, spread<0xbbaa>(high)));
    }
};
struct Bf16Pair {
    static constexpr uint32_t kNone = 0xff80ff80u;
    static constexpr float kLow = -1.0101590720568703e30f;  // 0xf14c: any far value whose y stays finite
    static __device__ __forceinline__ float2 both(uint32_t w) {
        return {__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
    }
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ uint32_t raise(uint32_t a) {
        uint32_t r;
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(0xf14cf14cu));
        return r;
    }
};
struct HalfPair {
    static constexpr uint32_t kNone = 0xfc00fc00u;
    static constexpr float kLow = -65504.f;
    static __device__ __forceinline__ float2 both(uint32_t w) { return __half22float2(reinterpret_cast<const __half2&>(w)); }
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ uint32_t raise(uint32_t a) {
        uint32_t r;
        asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(0xfbfffbffu));
        return r;
    }
};
template <>
struct Granule<__nv_bfloat16> : Granule16<Bf16Pair> {};
template <>
struct Granule<__half> : Granule16<HalfPair> {};

__device__ __forceinline__ void copy_async(uint32_t to, const uint4* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_async4(uint32_t to, const uint32_t* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// ---- a row ------------------------------------------------------------------------------------

// A row's memory in 16-byte granules from the one that holds its first value: granule g holds
// the values [g kVec - shift, (g + 1) kVec - shift) of the row, those of the first and the last
// granule that lie outside it excepted.
template <typename T, bool MASK>
struct Row {
    static constexpr int kVec = Granule<T>::kVec;
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
    // a full granule's bytes with what is not allowed at -inf
    __device__ __forceinline__ uint4 cover(const uint4& u, int g) const {
        if (!MASK) return u;
        const int v = g * kVec - shift, off = v & 31;
        const uint32_t* w = allowed + (v >> 5);
        return Granule<T>::cover(u, __funnelshift_r(__ldg(w), off + kVec > 32 ? __ldg(w + 1) : 0u, off));
    }
    // any granule's scores; -inf outside the row
    __device__ __forceinline__ void read(int g, float (&v)[kVec]) const {
        if (g >= full0 && g < full1) {
            Granule<T>::unpack(cover(__ldg(base + g), g), v);
            return;
        }
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            const int k = g * kVec - shift + i;
            v[i] = k >= 0 && k < vocab ? logit(k) : -INFINITY;
        }
    }
};

// The granules [g0, g1) of a row that a group works on: the full ones, [from, to), in strides of
// THREADS, and the row's first and last one, where they are shared with other rows, by the first
// and the last thread.
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

// What a thread has of a row while it reads its granules: the sums relative to `ref`, in pairs, and
// its largest logit. Two ways to add scores. The plain one takes y = x scale + offset in one
// rounding, with offset = -ref scale rounded: the sums are then relative to the logit whose y is
// exactly 0, `slip` (in y) away from ref, which part() puts right. The careful one takes
// (x - ref) scale and clamps each y: where there is no reference yet, for references so large that
// ref scale says nothing about x scale, and, in 16 bits, for references so low that a score of -inf
// clamped to a finite one would count.
template <typename T>
struct Running {
    static constexpr int kVec = Granule<T>::kVec;
    float ref = -INFINITY, best = -INFINITY;
    float limit = NAN;  // what a logit may reach the plain way; NaN: the careful way
    float offset = 0.f;
    float2 s2 = {0.f, 0.f}, h2 = {0.f, 0.f};

    __device__ __forceinline__ void shift(float d) {  // to a reference d lower, in y
        const float e = exp2_fast(d);
        h2 = {e * (h2.x + d * s2.x), e * (h2.y + d * s2.y)};
        s2 = {e * s2.x, e * s2.y};
    }
    __device__ __forceinline__ float slip(float scale) const { return -__fmaf_rn(ref, scale, offset); }

    // a reference that suits scores of up to `top`, and whether it serves the plain way
    __device__ __forceinline__ void raise(float top, float scale, float headroom) {
        if (limit == limit) {
            shift(slip(scale));
            limit = NAN;
        }
        if (ref == -INFINITY) {
            ref = top;
        } else if (top > ref + headroom) {
            shift(fmaxf((ref - top) * scale, -1e4f));
            ref = top;
        }
        const float y = ref * scale;
        if (fabsf(y) < 4194304.f && Granule<T>::plain(ref, scale)) {  // slip below a half
            offset = -y;
            shift(-slip(scale));
            limit = ref + headroom;
        }
    }
    __device__ __forceinline__ void add_carefully(const float (&x)[kVec], float scale) {
        const float from = ref == -INFINITY ? 0.f : ref;
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            const float y = max_nan((x[i] - from) * scale, -150.f), e = exp2_fast(y);
            s2.x += e;
            h2.x = __fmaf_rn(e, y, h2.x);
        }
    }
    // a stage; returns its largest logit. A row's first one: the warp's largest is every lane's
    // reference, which few later logits are well above (with each lane's own, 4096 rows of 128,256
    // bfloat16 scores took 17 us more).
    __device__ __forceinline__ float take(const uint4 (&u)[kUnroll], float scale, float headroom, bool first) {
        const float top = Granule<T>::largest(u);
        best = fmaxf(best, top);
        float lead = top;
        if (first) lead = from_order_bits(__reduce_max_sync(0xffffffffu, order_bits(top)));
        if (__builtin_expect(!(lead <= limit), 0)) {
            raise(lead, scale, headroom);
            if (limit != limit) {
#pragma unroll 1
                for (int k = 0; k < kUnroll; ++k) {
                    uint4 v = u[0];
#pragma unroll
                    for (int i = 1; i < kUnroll; ++i) v = i == k ? u[i] : v;
                    float x[kVec];
                    Granule<T>::unpack(v, x);
                    add_carefully(x, scale);
                }
                return top;
            }
        }
        const float2 scale2 = {scale, scale}, offset2 = {offset, offset};
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            float2 y[kVec / 2];
            Granule<T>::scaled(u[k], scale2, offset2, y);
#pragma unroll
            for (int i = 0; i < kVec / 2; ++i) {
                const float2 e = {exp2_fast(y[i].x), exp2_fast(y[i].y)};
                s2 = add2(s2, e);
                h2 = fma2(e, y[i], h2);
            }
        }
        return top;
    }
    __device__ __forceinline__ void take_edge(const float (&x)[kVec], float scale, float headroom) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < kVec; ++i) top = fmaxf(top, x[i]);
        best = fmaxf(best, top);
        // sums relative to ref itself, then the careful way
        raise(top, scale, headroom);
        if (limit == limit) shift(slip(scale));
        add_carefully(x, scale);
        if (limit == limit) shift(-slip(scale));
    }
    __device__ __forceinline__ Part part(float scale) {
        if (limit == limit) shift(slip(scale));
        return Part{ref, s2.x + s2.y, h2.x + h2.y};
    }
};

// What a group of THREADS threads shares while it works on a row (or a cluster's part of one).
template <int THREADS>
struct Shared {
    static constexpr int kCollect = THREADS == 32 ? 128 : 512;
    static constexpr int kMarks = THREADS == 32 ? 8 : 16;  // of a thread
    uint64_t keys[kCollect];           // the logits that reach the bound
    uint64_t chosen[kMaxTop];
    Part parts[THREADS / 32];
    uint32_t rounds[THREADS / 32];     // a warp's contribution to the bound
    uint32_t ord[THREADS];             // order bits of the threads' maxima, 0: none
    uint16_t marks[kMarks * THREADS];  // upper half of a run's largest logit
    uint16_t runs[kCollect];           // marked runs to read again: mark * THREADS + thread
    int marked, collected;
    uint32_t bound;
};

// What a CTA that walks over its rows also keeps: the largest maxima of each warp, and, while the
// next row is read, what it is still to do for the one before.
struct Walk {
    static constexpr int kLooks = 256;  // granules that are read again, one for each thread
    uint4 again[kLooks];
    int at[kLooks];
    uint32_t maxima[8 * kMaxRounds];
    Part sums;
    int looks;
};

template <int THREADS>
__device__ __forceinline__ void group_sync() {
    if (THREADS == 32) __syncwarp();
    else __syncthreads();
}

// Order bits that at least `wanted` of the threads' maxima reach, and few more where they differ: the
// search ends as soon as their number is within an eighth. Run by one warp, on g.ord. 0 when
// fewer than `wanted` threads have any logit.
template <int THREADS>
__device__ __forceinline__ uint32_t find_bound(const Shared<THREADS>& g, int wanted, int lane) {
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
    return t;
}

// A group of several warps has a bound without that search: with q = wanted / warps rounded up, the
// least of the warps' q-th largest maxima. Looser (some two times `wanted` reach it where the large logits
// are spread, thousands where they lie together), far shorter. 0 when a warp has fewer than q logits. This is
// a warp's part of it.
__device__ __forceinline__ uint32_t nth_largest(uint32_t ord, int q, int lane) {
    uint32_t high = 0;
    for (int i = 0; i < q; ++i) {
        high = __reduce_max_sync(0xffffffffu, ord);
        if (lane == __ffs(__ballot_sync(0xffffffffu, ord == high)) - 1) ord = 0;
    }
    return high;
}

template <int THREADS>
__device__ __forceinline__ uint64_t group_max(Shared<THREADS>& g, uint64_t k, int tid) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const uint64_t c = __shfl_xor_sync(0xffffffffu, k, o);
        k = c > k ? c : k;
    }
    if (THREADS == 32) return k;
    __syncthreads();
    if ((tid & 31) == 0) g.keys[tid / 32] = k;
    __syncthreads();
    for (int w = 0; w < THREADS / 32; ++w) k = g.keys[w] > k ? g.keys[w] : k;
    return k;
}

// The alternatives one after another, the best below the one before each time: for rows where more
// reaches the bound than the group can hold (large logits gathered in few threads' places).
template <typename T, bool MASK, int THREADS>
__device__ __noinline__ void choose_slowly(Shared<THREADS>& g, Row<T, MASK> r, Run<T, MASK, THREADS> run,
                                           int wanted, int tid) {
    constexpr int kVec = Row<T, MASK>::kVec;
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
        k = group_max<THREADS>(g, k, tid);
        if (tid == 0) g.chosen[j] = k;
        before = k;
    }
}

// More reaches the bound t than the group can hold: where large logits lie together few threads read
// them all, and the threads' maxima say little about them (a vocabulary sorted by frequency has such rows);
// or where many are equal (rows of one value, zeros). The wanted-th best of what is held is a bound as well, and
// each turn a tighter one: what is above it is collected from the whole row. Then the first that equal it,
// found in the row's order until there are enough. False if more is above the last bound than the group can
// hold. One or two readings of the row more, where one for each alternative took (float16, 20 alternatives,
// logits of -log(id) and noise) 64 x 128,256 from 45 to 223 us and 8192 x 32,000 from 230 to 1515; ordinary rows
// take 13 and 172. The row's main pass feels this function's registers, so it is kept narrow: order bits
// instead of keys (52 and 235 with keys), loops that are not unrolled further. With that 4096 x 128,256 bfloat16
// take 209 us, 207 without this way.
template <typename T, bool MASK, int THREADS>
__device__ __noinline__ bool collect_tighter(Shared<THREADS>& g, Row<T, MASK> r, Run<T, MASK, THREADS> run,
                                             int wanted, int tid, uint32_t t) {
    constexpr int kVec = Row<T, MASK>::kVec;
    constexpr int kHold = Shared<THREADS>::kCollect;
#pragma unroll 1
    for (int turn = 0;; ++turn) {
        group_sync<THREADS>();
        const int n = min(g.collected, kHold);
        if (n >= wanted) {
            if (tid == 0) g.bound = ~0u;
            group_sync<THREADS>();
            auto held = [&](int i) { return (uint32_t)(g.keys[i] >> 32); };
#pragma unroll 1
            for (int i = tid; i < n; i += THREADS) {
                const uint32_t k = held(i);
                int better = 0;
#pragma unroll 4
                for (int j = 0; j < n; ++j) better += held(j) > k;
                if (better < wanted) atomicMin(&g.bound, k);
            }
            group_sync<THREADS>();
            t = g.bound;
        }
        group_sync<THREADS>();
        if (tid == 0) g.collected = 0;
        group_sync<THREADS>();
        for (int at = run.g0 + tid; at < run.g1; at += THREADS) {
            float x[kVec];
            r.read(at, x);
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                if (!(x[i] > -INFINITY && order_bits(x[i]) > t)) continue;
                const int n = atomicAdd(&g.collected, 1);
                if (n < kHold) g.keys[n] = choice_key(x[i], at * kVec - r.shift + i);
            }
        }
        group_sync<THREADS>();
        if (g.collected <= kHold - kMaxTop) break;
        if (turn == kTurns) return false;
    }
    // THREADS granules at a time, in order; each thread's equals are numbered before they are kept
    int missing = wanted - g.collected;
    for (int at0 = run.g0; at0 < run.g1 && missing > 0; at0 += THREADS) {
        float x[kVec];
        int mine = 0;
        const int at = at0 + tid;
        if (at < run.g1) {
            r.read(at, x);
#pragma unroll
            for (int i = 0; i < kVec; ++i) mine += x[i] > -INFINITY && order_bits(x[i]) == t;
        }
        group_sync<THREADS>();
        g.ord[tid] = (uint32_t)mine;
        group_sync<THREADS>();
        int before = 0, total = 0;
        for (int i = 0; i < THREADS; ++i) {
            const int n = (int)g.ord[i];
            before += i < tid ? n : 0;
            total += n;
        }
        if (mine) {
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                if (!(x[i] > -INFINITY && order_bits(x[i]) == t)) continue;
                if (before < missing) {
                    const int n = atomicAdd(&g.collected, 1);
                    g.keys[n] = choice_key(x[i], at * kVec - r.shift + i);
                }
                ++before;
            }
        }
        missing -= total;
    }
    group_sync<THREADS>();
    return true;
}

// What is collected, best first, into g.chosen; by the ways for more than was held where it was more.
template <typename T, bool MASK, int THREADS>
__device__ __forceinline__ void rank(Shared<THREADS>& g, const Row<T, MASK>& r, const Run<T, MASK, THREADS>& run,
                                     int wanted, int tid, uint32_t t) {
    constexpr int kHold = Shared<THREADS>::kCollect;
    bool held = g.collected <= kHold && g.marked <= kHold;
    if (!held) held = collect_tighter<T, MASK, THREADS>(g, r, run, wanted, tid, t);
    if (held) {
        const int n = g.collected;
        for (int i = tid; i < n; i += THREADS) {
            const uint64_t k = g.keys[i];
            int better = 0;
            for (int j = 0; j < n; ++j) better += g.keys[j] > k;
            if (better < wanted) g.chosen[better] = k;
        }
    } else {
        choose_slowly<T, MASK, THREADS>(g, r, run, wanted, tid);
    }
    group_sync<THREADS>();
}

// Collect what reaches the bound among a granule's scores.
template <int VEC, int THREADS>
__device__ __forceinline__ void collect(Shared<THREADS>& g, const float (&x)[VEC], int at, int shift, uint32_t t) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        if (!(x[i] > -INFINITY && order_bits(x[i]) >= t)) continue;
        const int n = atomicAdd(&g.collected, 1);
        if (n < Shared<THREADS>::kCollect) g.keys[n] = choice_key(x[i], at * VEC - shift + i);
    }
}

// This thread's runs whose marks reach the bound, if its maximum does, and its ends of the row.
template <typename T, bool MASK, int THREADS>
__device__ __forceinline__ void mark_runs(Shared<THREADS>& g, const Row<T, MASK>& r, const Run<T, MASK, THREADS>& run,
                                          int tid, uint32_t ord, uint32_t t, int marks) {
    constexpr int kVec = Row<T, MASK>::kVec;
    if (!(ord && ord >= t)) return;
    // Both cut towards zero, which keeps their order: a run with a logit that reaches t has a mark
    // that reaches t's upper half.
    const float least = t ? __uint_as_float(__float_as_uint(from_order_bits(t)) & 0xffff0000u) : -INFINITY;
    for (int m = 0; m < marks; ++m) {
        if (!(__uint_as_float((uint32_t)g.marks[m * THREADS + tid] << 16) >= least)) continue;
        const int n = atomicAdd(&g.marked, 1);
        if (n < Shared<THREADS>::kCollect) g.runs[n] = (uint16_t)(m * THREADS + tid);
    }
    if (run.first(r, tid) || run.last(r, tid)) {
        float x[kVec];
        const int at = tid == 0 ? 0 : run.g1 - 1;
        r.read(at, x);
        collect<kVec, THREADS>(g, x, at, r.shift, t);
    }
}

// The granule of the q-th look at the marked runs of 2^shift granules each; run.to: none.
template <typename T, bool MASK, int THREADS>
__device__ __forceinline__ int look_at(const Shared<THREADS>& g, const Run<T, MASK, THREADS>& run, int q, int shift) {
    const int of = g.runs[q >> shift], k = q & ((1 << shift) - 1);
    return min(run.to, run.from + of % THREADS + (((of / THREADS) << shift) + k) * THREADS);
}

// The alternatives among a run's granules into g.chosen, best first, 0 past the last; called by the
// whole group with each thread's largest logit, which is in g.ord, and, for more than one warp,
// with the warps' parts of the bound in g.rounds. Each of a thread's `marks` marks stands for
// 2^shift granules.
template <typename T, bool MASK, int THREADS>
__device__ __forceinline__ void choose(Shared<THREADS>& g, const Row<T, MASK>& r, const Run<T, MASK, THREADS>& run,
                                       int wanted, int tid, uint32_t ord, int marks, int shift) {
    constexpr int kVec = Row<T, MASK>::kVec;
    constexpr int kWarps = THREADS / 32;
    uint32_t t;
    if (kWarps == 1) {
        t = find_bound<THREADS>(g, wanted, tid);
    } else {
        t = g.rounds[0];
        for (int w = 1; w < kWarps; ++w) t = min(t, g.rounds[w]);
        if (!t) {  // warps with few logits, or none: uniform over the group
            if (tid < 32) {
                t = find_bound<THREADS>(g, wanted, tid);
                if (tid == 0) g.bound = t;
            }
            __syncthreads();
            t = g.bound;
        }
    }
    mark_runs<T, MASK, THREADS>(g, r, run, tid, ord, t, marks);
    group_sync<THREADS>();
    const int looks = min(g.marked, Shared<THREADS>::kCollect) << shift;
    for (int q = tid; q < looks; q += THREADS) {
        const int at = look_at<T, MASK, THREADS>(g, run, q, shift);
        if (at >= run.to) continue;
        float x[kVec];
        Granule<T>::unpack(r.cover(__ldg(r.base + at), at), x);
        collect<kVec, THREADS>(g, x, at, r.shift, t);
    }
    group_sync<THREADS>();
    rank<T, MASK, THREADS>(g, r, run, wanted, tid, t);
}

// The row's results from its sums and its alternatives' keys. The sums' own roundings (a reference's y
// is not exactly 0, nor is it the row's maximum) leave a sure row on either side of 0, by one step: what
// the definition bounds by 0 is cut off there, which brings no value further from the definition.
template <typename T, bool MASK, int THREADS>
__device__ __forceinline__ void write_row(const Args& a, const Row<T, MASK>& r, int64_t row, const Part& p,
                                          const uint64_t* chosen, int tid) {
    const bool empty = p.s == 0.f;
    const float log_s = empty ? 0.f : logf(p.s);
    auto logprob = [&](float x) {
        if (empty || (x == -INFINITY && p.s == p.s)) return -INFINITY;
        const float v = (x - p.m) * a.inv_t - log_s;
        return v > 0.f ? 0.f : v;  // NaN where S is
    };
    if (tid == 0) {
        const float v = empty ? 0.f : log_s - 0.693147180559945f * (p.h / p.s);
        a.entropy[row] = v < 0.f ? 0.f : v;
    }
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

// What a walking CTA does for a row while it reads the next one. The granules that it asked for when
// the row ended have come: collect what reaches the bound. Each thread looks at its own copies only.
template <typename T, bool MASK, int THREADS>
__device__ __noinline__ void collect_again(const Args& a, Shared<THREADS>& g, const Walk& w, int row, int tid) {
    constexpr int kVec = Row<T, MASK>::kVec;
    if (tid >= w.looks || w.at[tid] < 0) return;
    const Row<T, MASK> r(a, row);
    float x[kVec];
    Granule<T>::unpack(r.cover(w.again[tid], w.at[tid]), x);
    collect<kVec, THREADS>(g, x, w.at[tid], r.shift, g.bound);
}
// And then rank it and write the row's results.
template <typename T, bool MASK, int THREADS>
__device__ __noinline__ void finish(const Args& a, Shared<THREADS>& g, const Walk& w, int row, int tid) {
    const Row<T, MASK> r(a, row);
    const Run<T, MASK, THREADS> run(r, 0, 1);
    group_sync<THREADS>();
    rank<T, MASK, THREADS>(g, r, run, a.top, tid, g.bound);
    write_row<T, MASK, THREADS>(a, r, row, w.sums, g.chosen, tid);
}

// A group of THREADS threads per row: a warp, a CTA, or (CLUSTER) a CTA for each part of a row.
// Groups walk over the rows. Each thread copies its granules into places of its own in shared
// memory, kStages stages of kUnroll ahead of where it reads, past the end of a row into the next
// one. No thread reads what another copied (but for the mask's words, which a warp shares), so the
// copies need no barrier. A walking CTA does not wait for the granules that it reads again (they
// take 4 us from a busy memory, an eighth of a row of 128,256 bfloat16 scores): it asks for them
// when the row ends, looks at them after the next row's second stage and ranks them after its third.
//
// No unit is full: with 20 alternatives, 4096 rows of 128,256 bfloat16 scores keep the issue slots busy 69% of the
// time, the exponential unit 61% and the memory 60% (without alternatives 70, 68 and 68), and a CTA's warps wait most
// at the barriers of its rows' ends. A thread's stage of 32 such scores is 231 instructions, 32 of them
// exponentials, of which an SM starts 16 a clock. These rows take 182 us without alternatives and 209 with 20 of
// them, 2048 rows of float32 174; the scores alone take 161 at the memory's 6.55 TB/s. Dropped, each with
// 20 alternatives against the kernel of its time: loads into registers, a bound's holders read again
// whole (276 us); stages half as long (241 against 218), three CTAs of three stages (221), CTAs of 128
// threads (233), two warps of a CTA that finish what eight read (212 against 214, slower for few
// rows), a share of the exponentials by multiply-adds (213 to 232 against 213).
template <int THREADS>
constexpr int kCta = THREADS == 32 ? kWarpCta : THREADS;

template <typename T, int THREADS, bool MASK, bool CLUSTER>
__global__ void __launch_bounds__(kCta<THREADS>, 1024 / kCta<THREADS>) logprobs_kernel(const __grid_constant__ Args a) {
    constexpr int kVec = Row<T, MASK>::kVec;
    constexpr int kWarps = THREADS / 32, kGroups = kCta<THREADS> / THREADS;
    constexpr int kStage = kUnroll * THREADS;  // granules
    // of 32 granules in a row: the words that hold their bits, and one that may be read beside them
    constexpr int kWords = kVec + 2;
    static_assert(THREADS * kVec % 32 == 0, "the granules of a thread are whole words apart");
    extern __shared__ uint4 rings[];  // [kGroups][kStages][kUnroll][THREADS]
    __shared__ uint32_t mask_rings[MASK ? kCta<THREADS> / 32 * kStages * kUnroll * kWords : 1];
    constexpr bool kWalks = kGroups == 1 && !CLUSTER;
    __shared__ Shared<THREADS> shared[kGroups];
    __shared__ std::conditional_t<kWalks, Walk, int> walk;
    int owed = -1;  // the row that is still to be ranked and written
    __shared__ uint64_t cluster_keys[CLUSTER ? kMaxCluster * kMaxTop : 1];
    __shared__ Part cluster_parts[CLUSTER ? kMaxCluster : 1];
    const int group = threadIdx.x / THREADS, tid = threadIdx.x % THREADS, lane = tid & 31;
    Shared<THREADS>& g = shared[group];
    const uint4* const ring = rings + group * kStages * kStage + tid;
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
    unsigned part = 0, parts = 1;
    if (CLUSTER) {
        cg::cluster_group cluster = cg::this_cluster();
        part = cluster.block_rank();
        parts = cluster.num_blocks();
        cluster.barrier_arrive();  // every CTA runs before one writes into another's memory
    }
    const int64_t first = CLUSTER ? blockIdx.x / parts : (int64_t)blockIdx.x * kGroups + group;
    const int64_t step = CLUSTER ? gridDim.x / parts : (int64_t)gridDim.x * kGroups;

    // the next stage to copy: of row `ahead`, its `left` granules from `next` on
    int64_t ahead = first;
    const uint4* next = nullptr;
    int left = 0;
    const uint32_t* mask = nullptr;  // and the row's mask
    int next_word = 0;               // with the word of this warp's first granule in it
    const int last_word = (a.vocab - 1) >> 5;
    uint32_t* const mask_ring = mask_rings + (MASK ? threadIdx.x / 32 * kStages * kUnroll * kWords : 0);
    const uint32_t mask_at = (uint32_t)__cvta_generic_to_shared(mask_ring);
    // the words that a lane copies: how far from the stage's first, and from its place in the ring in bytes
    constexpr int kNeeded = kUnroll * (kWords - 1);
    auto word_of = [](int w) {
        const int k = w / (kWords - 1), i = w % (kWords - 1);
        return int2{k * (THREADS * kVec / 32) + i, (k * kWords + i) * (int)sizeof(uint32_t)};
    };
    const int2 words = word_of(lane), more = word_of(lane + 32);
    auto enter = [&]() {
        const Row<T, MASK> r(a, ahead);
        const Run<T, MASK, THREADS> run(r, part, parts);
        next = r.base + run.from + tid;
        left = run.to - run.from;
        if (MASK) {
            mask = r.allowed;
            next_word = ((run.from + tid - lane) * kVec - r.shift) >> 5;
        }
    };
    if (ahead < a.rows) enter();
    auto copy_stage = [&](int slot) {
        const uint32_t to = ring_at + (uint32_t)(slot * sizeof(uint4));
        if (left < kStage) {
            while (left <= 0 && ahead < a.rows) {
                ahead += step;
                if (ahead < a.rows) enter();
            }
        }
        if (left >= kStage) {
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) copy_async(to + k * THREADS * sizeof(uint4), next + k * THREADS);
        } else {
#pragma unroll
            for (int k = 0; k < kUnroll; ++k)
                if (k * THREADS + tid < left) copy_async(to + k * THREADS * sizeof(uint4), next + k * THREADS);
        }
        if (MASK && left > 0) {  // a lane for each word that the warp's granules of this stage need
            const uint32_t at = mask_at + (uint32_t)(slot / THREADS * kWords * sizeof(uint32_t));
            if (lane < kNeeded && next_word + words.x <= last_word) copy_async4(at + words.y, mask + next_word + words.x);
            if (kNeeded > 32 && lane + 32 < kNeeded && next_word + more.x <= last_word)
                copy_async4(at + more.y, mask + next_word + more.x);
            next_word += kStage * kVec / 32;
        }
        next += kStage;
        left -= kStage;
        copies_commit();
    };
#pragma unroll
    for (int k = 0; k < kStages; ++k) copy_stage(k * kStage);
    int slot = 0;  // where the next stage to read is in the ring

    for (int64_t row = first; row < a.rows; row += step) {
        const Row<T, MASK> r(a, row);
        const Run<T, MASK, THREADS> run(r, part, parts);
        Running<T> sums;
        if (run.first(r, tid)) {
            float x[kVec];
            r.read(0, x);
            sums.take_edge(x, a.scale, a.headroom);
        }
        // marks of 2^per stages each
        const int stages = (max(0, run.to - run.from) + kStage - 1) / kStage;
        const int per = stages > Shared<THREADS>::kMarks ? 32 - __clz((stages - 1) / Shared<THREADS>::kMarks) : 0;
        float marked = -INFINITY;
        const int granules = run.to - run.from;
        // where this thread's bits are among its warp's words: a stage is whole words, so always there
        const int warp_bit = ((run.from + tid - lane) * kVec - r.shift) & 31, my_bit = (warp_bit + lane * kVec) & 31;
        const uint32_t* const my_mask = mask_ring + (warp_bit + lane * kVec) / 32;
        for (int k0 = 0; k0 < stages; ++k0) {
            copies_wait<kStages - 1>();
            if (MASK) __syncwarp();  // the mask's words are other lanes' copies
            const uint4* held = ring + slot;
            const int done = k0 * kStage;
            uint4 u[kUnroll];
            auto covered = [&](int k) {
                if (!MASK) return held[k * THREADS];
                const uint32_t* w = my_mask + (slot / THREADS + k) * kWords;
                return Granule<T>::cover(held[k * THREADS], __funnelshift_r(w[0], w[1], my_bit));
            };
            if (done + kStage <= granules) {
#pragma unroll
                for (int k = 0; k < kUnroll; ++k) u[k] = covered(k);
            } else {
#pragma unroll
                for (int k = 0; k < kUnroll; ++k) u[k] = done + k * THREADS + tid < granules ? covered(k) : Granule<T>::empty();
            }
            if (MASK) __syncwarp();  // and this stage's are read before the next copies replace them
            const float top = sums.take(u, a.scale, a.headroom, k0 == 0);
            copy_stage(slot);
            slot = slot == (kStages - 1) * kStage ? 0 : slot + kStage;
            marked = k0 & ((1 << per) - 1) ? fmaxf(marked, top) : top;
            g.marks[(k0 >> per) * THREADS + tid] = (uint16_t)(__float_as_uint(marked) >> 16);
            if constexpr (kWalks) {
                if (__builtin_expect(owed >= 0, 0)) {
                    if (k0 == 1) collect_again<T, MASK, THREADS>(a, g, walk, owed, tid);
                    if (k0 == 2) {
                        finish<T, MASK, THREADS>(a, g, walk, owed, tid);
                        owed = -1;
                    }
                }
            }
        }
        if (run.last(r, tid)) {
            float x[kVec];
            r.read(run.g1 - 1, x);
            sums.take_edge(x, a.scale, a.headroom);
        }
        Part p = join<32>(sums.part(a.scale), a.scale);
        const uint32_t ord = sums.best > -INFINITY ? order_bits(sums.best) : 0u;
        const int marks = (stages + (1 << per) - 1) >> per, shift = per + kUnrollLog;
        if constexpr (kWalks) {
            if (owed >= 0) {  // this row was a short one
                copies_wait<0>();
                if (stages < 2) collect_again<T, MASK, THREADS>(a, g, walk, owed, tid);
                finish<T, MASK, THREADS>(a, g, walk, owed, tid);
                owed = -1;
            }
            // Each warp offers its largest maxima; the top-th largest of these is the bound: as good
            // as that of all the maxima unless a warp has more of the best than it offers.
            const int rounds = (a.top + kWarps - 1) / kWarps + 4;
            if (lane == 0) g.parts[tid / 32] = p;
            if (a.top > 0) {
                g.ord[tid] = ord;
                if (tid == 0) g.marked = g.collected = 0;
                uint32_t left = ord;
                for (int i = 0; i < rounds; ++i) {
                    const uint32_t high = __reduce_max_sync(0xffffffffu, left);
                    if (lane == __ffs(__ballot_sync(0xffffffffu, left == high)) - 1) left = 0;
                    if (lane == 0) walk.maxima[tid / 32 * rounds + i] = high;
                }
            }
            __syncthreads();
            p = join<kWarps>(g.parts[lane % kWarps], a.scale);
            if (a.top > 0) {
                for (int j = tid; j < a.top; j += THREADS) g.chosen[j] = 0;
                const int offered = kWarps * rounds;
                if (tid < offered) {
                    const uint32_t v = walk.maxima[tid];
                    int before = 0;
                    for (int j = 0; j < offered; ++j) before += walk.maxima[j] > v || (walk.maxima[j] == v && j < tid);
                    if (before == a.top - 1) g.bound = v;
                }
                __syncthreads();
                uint32_t t = g.bound;
                if (!t) {  // warps with few logits, or none: uniform over the CTA
                    __syncthreads();
                    if (tid < 32) {
                        t = find_bound<THREADS>(g, a.top, tid);
                        if (tid == 0) g.bound = t;
                    }
                    __syncthreads();
                    t = g.bound;
                }
                mark_runs<T, MASK, THREADS>(g, r, run, tid, ord, t, marks);
                __syncthreads();
                const int looks = min(g.marked, Shared<THREADS>::kCollect) << shift;
                if (looks <= Walk::kLooks && row + step < a.rows) {  // another row follows
                    if (tid < looks) {
                        const int at = look_at<T, MASK, THREADS>(g, run, tid, shift);
                        walk.at[tid] = at < run.to ? at : -1;
                        if (at < run.to) copy_async((uint32_t)__cvta_generic_to_shared(walk.again + tid), r.base + at);
                    }
                    copies_commit();
                    if (tid == 0) {
                        walk.sums = p;
                        walk.looks = looks;
                    }
                    owed = (int)row;
                    __syncthreads();
                    continue;
                }
                for (int q = tid; q < looks; q += THREADS) {
                    const int at = look_at<T, MASK, THREADS>(g, run, q, shift);
                    if (at >= run.to) continue;
                    float x[Row<T, MASK>::kVec];
                    Granule<T>::unpack(r.cover(__ldg(r.base + at), at), x);
                    collect<Row<T, MASK>::kVec, THREADS>(g, x, at, r.shift, t);
                }
                __syncthreads();
                rank<T, MASK, THREADS>(g, r, run, a.top, tid, t);
            }
            write_row<T, MASK, THREADS>(a, r, row, p, g.chosen, tid);
            __syncthreads();  // the next row's threads write where this row's read
            continue;
        }
        if (kWarps > 1 && lane == 0) g.parts[tid / 32] = p;
        if (a.top > 0) {
            g.ord[tid] = ord;
            if (tid == 0) g.marked = g.collected = 0;
            for (int j = tid; j < a.top; j += THREADS) g.chosen[j] = 0;
            if (kWarps > 1) {
                const uint32_t nth = nth_largest(ord, (a.top + kWarps - 1) / kWarps, lane);
                if (lane == 0) g.rounds[tid / 32] = nth;
            }
        }
        group_sync<THREADS>();
        if (kWarps > 1) p = join<kWarps>(g.parts[lane % kWarps], a.scale);
        if (a.top > 0) choose<T, MASK, THREADS>(g, r, run, a.top, tid, ord, marks, shift);
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

// Rows of up to 1024 scores: a warp each, bound by the latency of its few steps (4096 rows of 97 float32
// scores, 3 alternatives, in 4.2 us; the kernel above took 10.5). Every score is in a register: score 32 i + lane in slot i, so a
// slot's 32 bits of the mask are one word. Two passes over the registers, the maximum first; the
// alternatives one after another.
template <typename T, int NS, bool MASK>
__global__ void __launch_bounds__(kWarpCta) logprobs_small_kernel(const __grid_constant__ Args a) {
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * (kWarpCta / 32) + threadIdx.x / 32;
    if (row >= a.rows) return;
    const T* logits = static_cast<const T*>(a.logits) + row * a.row_stride;
    const uint32_t* allowed = MASK ? a.allowed + row * a.allowed_stride : nullptr;
    float x[NS];
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < NS; ++i) x[i] = 32 * i + lane < a.vocab ? to_f32(logits[32 * i + lane]) : -INFINITY;
    // the first given token of this lane, on its way while the row is summed
    int64_t token = -1;
    float given = -INFINITY;
    if (lane < a.n_tokens) {
        token = a.tokens[row * a.n_tokens + lane];
        if (token >= 0 && token < a.vocab && (!MASK || (allowed[token >> 5] >> (token & 31)) & 1u)) given = to_f32(logits[token]);
    }
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        if (MASK && 32 * i < a.vocab) x[i] = (__ldg(allowed + i) >> lane) & 1u ? x[i] : -INFINITY;
        m = fmaxf(m, x[i]);
    }
    uint32_t ord = m > -INFINITY ? order_bits(m) : 0u;  // of the lane's largest left
    uint32_t high = __reduce_max_sync(0xffffffffu, ord);
    const float top = high ? from_order_bits(high) : 0.f;
    float s = 0.f, h = 0.f;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const float y = max_nan((x[i] - top) * a.scale, -150.f), e = exp2_fast(y);
        s += e;
        h = __fmaf_rn(e, y, h);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        h += __shfl_xor_sync(0xffffffffu, h, o);
    }
    const bool empty = s == 0.f;
    const float log_s = empty ? 0.f : logf(s);
    auto logprob = [&](float v) {
        if (empty || (v == -INFINITY && s == s)) return -INFINITY;
        return (v - top) * a.inv_t - log_s;  // NaN where S is
    };
    if (lane == 0) a.entropy[row] = empty ? 0.f : log_s - 0.693147180559945f * (h / s);
    for (int j = lane; j < a.n_tokens; j += 32) {
        if (j >= 32) {
            token = a.tokens[row * a.n_tokens + j];
            given = -INFINITY;
            if (token >= 0 && token < a.vocab && (!MASK || (allowed[token >> 5] >> (token & 31)) & 1u)) given = to_f32(logits[token]);
        }
        a.logprobs[row * a.n_tokens + j] = token < 0 ? 0.f : token >= a.vocab ? NAN : logprob(given);
    }
    float alternative = 0.f;  // lane j keeps the j-th of each 32
    int id = -1;
    for (int j = 0; j < a.top; ++j) {
        int e = -1;
        if (high) {
            // the lowest id with this logit: every lane's lowest slot that has it, then the least of them
            int slot = 0;
#pragma unroll
            for (int i = NS - 1; i >= 0; --i) slot = x[i] >= m ? i : slot;  // m is the lane's largest: never NaN
            e = __reduce_min_sync(0xffffffffu, ord == high ? 32 * slot + lane : 0x7fffffff);
            const bool own = ord == high && 32 * slot + lane == e;
            if (NS > 1) {
                m = -INFINITY;
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    x[i] = own && i == slot ? -INFINITY : x[i];
                    m = fmaxf(m, x[i]);
                }
            } else if (own) {
                m = x[0] = -INFINITY;
            }
        }
        if ((j & 31) == lane) {
            id = e;
            alternative = high ? from_order_bits(high) : 0.f;
        }
        ord = m > -INFINITY ? order_bits(m) : 0u;
        high = __reduce_max_sync(0xffffffffu, ord);
        if ((j & 31) == 31 || j + 1 == a.top) {
            const int k = (j & ~31) + lane;
            if (k <= j) {
                a.top_ids[row * a.top + k] = id;
                a.top_logprobs[row * a.top + k] = id >= 0 ? logprob(alternative) : -INFINITY;
            }
        }
    }
}

// Alternatives for which the maxima of a warp's 32 threads are a bound that few scores pass: warp against CTA in us,
// bfloat16, with 20 16,384 x 1500 53 and 230, 2048 x 8000 19 and 30, 8192 x 32,000 172 and 168; with 24 63 and 242, 23
// and 30, 204 and 172; with 28 109 and 250, 63 and 31, 463 and 177.
constexpr int kWarpTop = 20;

template <typename T, int THREADS, bool MASK, bool CLUSTER>
cudaError_t launch(const Args& a, int cluster, cudaStream_t stream) {
    constexpr int kThreads = kCta<THREADS>, kRows = kThreads / THREADS;
    constexpr int ring = kStages * kUnroll * kThreads * (int)sizeof(uint4);
    auto kernel = logprobs_kernel<T, THREADS, MASK, CLUSTER>;
    cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kernel), ring);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t config{};
    // as many CTAs as run at once, which walk over the rows; with clusters, all of them
    config.gridDim = CLUSTER ? dim3((unsigned)(a.rows * cluster))
                             : dim3((unsigned)std::min<int64_t>(((int64_t)a.rows + kRows - 1) / kRows,
                                                                (int64_t)sm_count() * (1024 / kThreads)));
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = ring;
    config.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {(unsigned)cluster, 1, 1};
    config.attrs = &attr;
    config.numAttrs = CLUSTER ? 1 : 0;
    e = cudaLaunchKernelEx(&config, kernel, a);
    const cudaError_t last = cudaGetLastError();
    return e != cudaSuccess ? e : last;
}

template <typename T, int NS, bool MASK>
cudaError_t launch_small(const Args& a, cudaStream_t stream) {
    constexpr int rows = kWarpCta / 32;
    logprobs_small_kernel<T, NS, MASK><<<(unsigned)(((int64_t)a.rows + rows - 1) / rows), kWarpCta, 0, stream>>>(a);
    return cudaGetLastError();
}

template <typename T, bool MASK>
cudaError_t launch(const Args& a, cudaStream_t stream) {
    // A row in a warp's registers: up to where two passes over them cost more than a warp's or a CTA's one over memory.
    // 1000 scores, registers against logprobs_kernel in us: float32 64 rows, 3 alternatives 3.8 and 5.7, 4096
    // rows 10.4 and 10.2; bfloat16 16,384 rows 29.9 and 26.4. 300 scores: 2.9 and 5.4, 5.8 and 8.1. Each alternative is a pass
    // more, so with 20 of them 4096 x 300 takes 19.4 and 10.7, 4096 x 1000 33.5 and 13.9.
    if (a.vocab <= 32) return launch_small<T, 1, MASK>(a, stream);
    if (a.vocab <= 128) return launch_small<T, 4, MASK>(a, stream);
    if (a.vocab <= 256) return launch_small<T, 8, MASK>(a, stream);
    if (a.vocab <= 512) return launch_small<T, 16, MASK>(a, stream);
    if (a.vocab <= 1024) return launch_small<T, 32, MASK>(a, stream);
    // A warp per row has no barriers and its row's end is hidden by the other 31 warps of its SM, but
    // a row takes it eight times as long: it wins once there are about as many rows as granules in
    // one. bfloat16, 8 alternatives, warp against CTA in us: 2048 x 8000 15 and 25, 592 x 8000 12 and
    // 9; 8192 x 32,000 123 and 152, 1024 x 32,000 29 and 25; 16,384 x 1500 40 and 209, 148 x 1500 8.4
    // and 8.3.
    const int granules = (int)((int64_t)a.vocab * (int)sizeof(T) / 16);
    if (a.rows >= granules && a.top <= kWarpTop) return launch<T, 32, MASK, false>(a, 1, stream);
    // Parts of a row pay where there are CTAs to spare and the pass is long against what a part costs
    // beyond it. In us, 1, 2, 4 and 8 parts as far as the rule's border is lowered, 8 alternatives, bfloat16: 64 x 128,000
    // 16.2 and 11.8 (4 parts), 1 x 128,000 15.1, 9.2 (4) and 8.5 (8); 64 x 50,257 11.0, 10.3 (2) and 10.0 (4); 64 x 32,000
    // 8.1 and 8.5 (2). More CTAs than SMs: 148 x 50,257 11.5 and 12.7 (2), 148 x 128,000 16.9 and 15.7.
    const int sms = sm_count();
    int cluster = 1;
    while (cluster < kMaxCluster && (int64_t)a.rows * cluster <= sms && granules / cluster > 4000) cluster *= 2;
    if (cluster == 1) return launch<T, 256, MASK, false>(a, 1, stream);
    return launch<T, 256, MASK, true>(a, cluster, stream);
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
    // The headroom is 4 in base 2, and at most twice that once reference + headroom is rounded. More
    // would still not overflow, but a lone high logit would have its y 2^y summed as a large number
    // that the reference's move takes away again, and the entropy of a sure row is what is left: at
    // 40 it was off by 40 roundings. Less would raise the reference more often for nothing.
    const Args a{logits, rows, vocab, row_stride, tokens, n_tokens, allowed, allowed_stride, 1.f / temperature, scale,
                 4.f / scale, top, logprobs, entropy, top_logprobs, top_ids};
    const cudaError_t e = dtype == SHIPK_DTYPE_F32   ? launch<float>(a, stream)
                          : dtype == SHIPK_DTYPE_F16 ? launch<__half>(a, stream)
                                                     : launch<__nv_bfloat16>(a, stream);
    return e == cudaSuccess ? Status{SHIPK_OK, nullptr} : Status{SHIPK_ECUDA, cudaGetErrorString(e)};
}

}  // namespace shipk
