// Losses over rows of logits and the gradients they send back: log-probabilities of labels, distillation from a
// teacher's top logits, clipped policy loss, preference loss.
//
// With x a row of logits over C classes, T the temperature, m = max x, t_j = (x_j - m) / T, e_j = exp(t_j), s = sum e:
//   log p_j = t_j - log s,   H = log s - (sum e_j t_j) / s   (entropy)
// and the gradient of every loss here with respect to x has the form
//   d_j = e_j (a + b t_j)  for all j,  plus a correction at the label or at the classes of the teacher's list.
// So a row is read for (m, s, sum e t), a few numbers per row are computed, and the gradient is written from the same
// values. A thread keeps a running maximum and the sums relative to it, which are rescaled when the maximum grows; the
// partial results of the threads meet once per row. Exponents are taken to base 2 with the factor log2(e) / T.
#pragma once

#include "sk_device.cuh"
#include "sk_epilogue.cuh"
#include "sk_tc_ptx.cuh"

namespace sk {
namespace loss {

constexpr int kThreads = 256, kWarps = kThreads / 32;      // of the pair kernel
constexpr uint32_t kMaxList = 512;          // entries of a teacher's list
constexpr uint32_t kMaxListClasses = 1u << 20;   // a bit for each class fits shared memory
constexpr float kLn2 = 0.693147180559945f;
// A teacher's mass outside its list below this counts as none: rounding its log-sum-exp to f32 leaves as much.
constexpr double kLeastTail = 1e-6;
enum : int { kErrLabel = 1, kErrList = 2, kErrOffsets = 4 };

// The matrix of logits. log2(e) / T is the sum of two floats: with one, its rounding (up to 6e-8) times an exponent
// of -10 would be a common factor of 6e-7 on most of a wide row's sum. c_lo > 0, so that -inf stays -inf.
struct Rows {
    const void *x;
    void *d;                                // gradient, or nullptr
    uint32_t rows, cols, classes;
    float c_hi, c_lo;
    double inv_t;
    float k;                                // loss scale / T: factor on every gradient
    int *err;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// log of a positive f32 in 64 bits: the mantissa's logarithm is below 0.35, so that its f32 rounding is below 2e-8
// where that of log(s) itself would be 5e-7. Log-probabilities are differences that the losses take exponentials of, and
// sums over a thousand rows.
__device__ __forceinline__ double log_wide(float s) {
    int e;
    float f = frexpf(s, &e);
    if (f < 0.70710678f) { f *= 2.0f; --e; }
    return (double)e * 0.69314718055994531 + (double)logf(f);
}
// What ex2 lacks: its results are 5.1e-8 too small on average (measured over [-32, 0), weighted by size, the same in every
// octave; 1.4e-7 at most), and exact for the exponent 0 of a thread's own maximum. It is the same sign in every row, which
// the sum over a sequence does not average out: it made 8e-6 of a preference margin of sequences that differ by hundreds
// of rows. A thread's sum is lifted by it; what is left is below 1.7e-8 of a sum (4000 rows of 20 to 20000 classes).
constexpr float kEx2Low = 5.0e-8f;

// The largest of a warp's values, in every lane; one instruction on sm_100a. NaN only if all are.
__device__ __forceinline__ float max_of_warp(float v) {
    float r;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
// The same with NaN as soon as one of them is.
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_of_warp_or_nan(float v) {
    float r;
    asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

// ---- 16 bytes of a row, and pairs of f32 values ------------------------------------------------
// Arithmetic is on pairs (add / mul / fma.rn.f32x2: two round-to-nearest operations in one instruction), because wide
// rows of 16-bit logits are bound by instruction issue as much as by memory.
using f32x2 = uint64_t;
__device__ __forceinline__ f32x2 pair(float lo, float hi) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 halves(f32x2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) { f32x2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) { f32x2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) { f32x2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ f32x2 ex2_2(f32x2 t) { const float2 v = halves(t); return pair(ex2(v.x), ex2(v.y)); }

template <typename T> struct Unit;
template <> struct Unit<float> {
    static constexpr int V = 4;
    uint4 q;
    static constexpr uint32_t kNone = 0xFF800000u;        // -inf
    __device__ __forceinline__ float max() const {
        return fmaxf(fmaxf(__uint_as_float(q.x), __uint_as_float(q.y)), fmaxf(__uint_as_float(q.z), __uint_as_float(q.w)));
    }
    __device__ __forceinline__ f32x2 get(int i) const {
        return i ? pair(__uint_as_float(q.z), __uint_as_float(q.w)) : pair(__uint_as_float(q.x), __uint_as_float(q.y));
    }
    __device__ __forceinline__ void set(int i, f32x2 v) {
        const float2 f = halves(v);
        if (i) { q.z = __float_as_uint(f.x); q.w = __float_as_uint(f.y); } else { q.x = __float_as_uint(f.x); q.y = __float_as_uint(f.y); }
    }
    __device__ __forceinline__ void drop(int j) { (&q.x)[j] = kNone; }
};
template <> struct Unit<__nv_bfloat16> {
    static constexpr int V = 8;
    uint4 q;
    static constexpr uint32_t kNone = 0xFF80FF80u;
    __device__ __forceinline__ float max() const {
        auto h = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162 *>(&w); };
        const __nv_bfloat162 m = __hmax2(__hmax2(h(q.x), h(q.y)), __hmax2(h(q.z), h(q.w)));
        return fmaxf(__low2float(m), __high2float(m));
    }
    __device__ __forceinline__ f32x2 get(int i) const {
        const uint32_t w = (&q.x)[i];
        return pair(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    }
    __device__ __forceinline__ void set(int i, f32x2 v) {
        const float2 f = halves(v);
        const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
        (&q.x)[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
    __device__ __forceinline__ void drop(int j) {
        uint32_t &w = (&q.x)[j / 2];
        w = j & 1 ? (w & 0xFFFFu) | (kNone & 0xFFFF0000u) : (w & 0xFFFF0000u) | (kNone & 0xFFFFu);
    }
};
template <> struct Unit<__half> {
    static constexpr int V = 8;
    uint4 q;
    static constexpr uint32_t kNone = 0xFC00FC00u;
    __device__ __forceinline__ float max() const {
        auto h = [](uint32_t w) { return *reinterpret_cast<const __half2 *>(&w); };
        const __half2 m = __hmax2(__hmax2(h(q.x), h(q.y)), __hmax2(h(q.z), h(q.w)));
        return fmaxf(__low2float(m), __high2float(m));
    }
    __device__ __forceinline__ f32x2 get(int i) const {
        const uint32_t w = (&q.x)[i];
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
        return pair(f.x, f.y);
    }
    __device__ __forceinline__ void set(int i, f32x2 v) {
        const float2 f = halves(v);
        const __half2 h = __floats2half2_rn(f.x, f.y);
        (&q.x)[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
    __device__ __forceinline__ void drop(int j) {
        uint32_t &w = (&q.x)[j / 2];
        w = j & 1 ? (w & 0xFFFFu) | (kNone & 0xFFFF0000u) : (w & 0xFFFF0000u) | (kNone & 0xFFFFu);
    }
};
template <typename T> __device__ __forceinline__ Unit<T> no_unit() {
    constexpr uint32_t n = Unit<T>::kNone;
    return Unit<T>{make_uint4(n, n, n, n)};
}

// ---- a row as aligned 16-byte units -------------------------------------------------------------
// Rows of odd widths start anywhere: up to V - 1 elements before the first 16-byte boundary (head) and behind the last
// one (tail) are taken one by one, each by one thread; nothing outside the row is touched.
template <typename T> struct Span {
    static constexpr int V = Unit<T>::V;
    const T *p;
    uint32_t n, head, units, tail;
    __device__ __forceinline__ Span(const T *first, uint32_t count) : p(first), n(count) {
        head = (uint32_t)((16 - reinterpret_cast<uintptr_t>(first) % 16) % 16 / sizeof(T));
        head = head < n ? head : n;
        units = (n - head) / V;
        tail = n - head - units * V;
    }
    __device__ __forceinline__ Unit<T> load(uint32_t u) const { return Unit<T>{*reinterpret_cast<const uint4 *>(p + head + (size_t)u * V)}; }
    __device__ __forceinline__ const T *tail_at() const { return p + (n - tail); }
};
// `count` < V elements from `p` on, -inf behind them.
template <typename T> __device__ __forceinline__ Unit<T> part_unit(const T *p, uint32_t count) {
    Unit<T> u = no_unit<T>();
    T *e = reinterpret_cast<T *>(&u.q);
#pragma unroll
    for (int j = 0; j < Unit<T>::V - 1; ++j)
        if ((uint32_t)j < count) e[j] = p[j];
    return u;
}

// ---- row statistics ------------------------------------------------------------------------
// Of the classes that a thread has seen: the maximum, sum e and sum e t2 (t2 = t log2 e), relative to it.
struct Share { float m, s, u; };
// Of a part of a row: instead of sum e what it is beyond the 1 of one class at the maximum. Of a label that is nearly
// certain, log p is the log1p of that, of which 1 + it would keep the f32 places of 1 only.
struct Stat {
    float m, more, u;
    __device__ __forceinline__ float s() const { return m == -INFINITY ? more : 1.0f + more; }      // no class: 0 (or NaN)
    __device__ __forceinline__ double log_s() const { return more < 0.4f ? (double)log1pf(more) : log_wide(1.0f + more); }
};

// What is summed beside e. kSums: nothing; the exponent is the product with both parts of log2(e) / T. kEntropy: e t2 as
// well, from which the second part's effect on s follows at once (with_low), so that one product is enough. A class at
// -inf makes NaN of e t2 = 0 * -inf; such a row is taken again with kMasked, which bounds t2 at -200, where e is 0 already.
enum Sums : int { kSums = 0, kEntropy = 1, kMasked = 2 };
// 2^t for t <= 0, from its power series in the fraction: right to a rounding of either sign. With ex2 for the factors of
// partial sums, even lifted, up to 1.1e-7 of a row's sum was left; with this 1.7e-8.
__device__ __forceinline__ float pow2(float t) {
    if (t < -126.0f) return 0.0f;
    const float n = rintf(t), r = (t - n) * kLn2, r2 = r * r;
    const float upper = fmaf(r2, fmaf(r, 1.0f / 5040.0f, 1.0f / 720.0f), fmaf(r, 1.0f / 120.0f, 1.0f / 24.0f));
    const float p = 1.0f + fmaf(r2 * r2, upper, fmaf(r2, fmaf(r, 1.0f / 6.0f, 0.5f), r));
    return p * __int_as_float(((int)n + 127) << 23);
}
// log2 of the factor that takes sums relative to m to the larger maximum `to`. Beyond f32 it makes NaN of u as one class's
// does, unless that is bounded.
template <int SUMS> __device__ __forceinline__ float factor_log(float m, float to, float c_hi, float c_lo) {
    const float by = m - to;
    return SUMS == kSums ? fmaf(by, c_hi, by * c_lo) : by * c_hi;
}
template <int SUMS> __device__ __forceinline__ float moved_u(float u, float s, float d, float f) {
    return f * fmaf(SUMS == kMasked ? fmaxf(d, -200.0f) : d, s, u);
}

__device__ __forceinline__ f32x2 floor2(f32x2 t) { const float2 v = halves(t); return pair(fmaxf(v.x, -200.0f), fmaxf(v.y, -200.0f)); }

template <typename T, int U, int SUMS> __device__ __forceinline__ void accumulate(Share &a, const Unit<T> (&q)[U], float c_hi, float c_lo) {
    float mx = q[0].max();
#pragma unroll
    for (int k = 1; k < U; ++k) mx = fmaxf(mx, q[k].max());
    if (mx > a.m) {
        if (a.m != -INFINITY) {
            const float d = factor_log<SUMS>(a.m, mx, c_hi, c_lo), f = ex2(d);
            if (SUMS) a.u = moved_u<SUMS>(a.u, a.s, d, f);
            a.s *= f;                       // lifted with the rest at the end; by itself as well, it would be 2e-8 too much
        }
        a.m = mx;
    }
    const float ref = a.m == -INFINITY ? 0.0f : a.m;
    const f32x2 less = pair(-ref, -ref), hi = pair(c_hi, c_hi), lo = pair(c_lo, c_lo);
    f32x2 s = 0, u = 0;
#pragma unroll
    for (int k = 0; k < U; ++k) {
#pragma unroll
        for (int i = 0; i < Unit<T>::V / 2; ++i) {
            const f32x2 d = add2(q[k].get(i), less), t = SUMS == kSums ? fma2(d, hi, mul2(d, lo)) : mul2(d, hi), e = ex2_2(t);
            s = add2(s, e);
            if (SUMS) u = fma2(e, SUMS == kMasked ? floor2(t) : t, u);
        }
    }
    const float2 ss = halves(s);
    a.s += ss.x + ss.y;
    if (SUMS) {
        const float2 us = halves(u);
        a.u += us.x + us.y;
    }
}
// The statistics of n parts (a power of two), in every lane, in a fixed order; each group of n lanes holds the same parts.
template <int SUMS> __device__ __forceinline__ Stat join(Stat a, uint32_t n, float c_hi, float c_lo) {
    float m = a.m;
    if (n == 32) m = max_of_warp(m);
    else for (uint32_t o = n / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const uint32_t keeps = __ffs(__ballot_sync(0xffffffffu, a.m == m)) - 1;     // the part whose 1 is left out
    if (a.m != -INFINITY) {
        const float d = factor_log<SUMS>(a.m, m, c_hi, c_lo), f = pow2(d);
        if (SUMS) a.u = moved_u<SUMS>(a.u, 1.0f + a.more, d, f);
        if ((threadIdx.x & (n - 1)) != keeps) a.more = fmaf(a.more, f, f);
    }
    a.m = m;
    for (uint32_t o = n / 2; o > 0; o >>= 1) {
        a.more += __shfl_xor_sync(0xffffffffu, a.more, o);
        if (SUMS) a.u += __shfl_xor_sync(0xffffffffu, a.u, o);
    }
    return a;
}
// A warp's from the shares of its lanes, which are lifted by what ex2 lacks on the way.
template <int SUMS> __device__ __forceinline__ Stat join_lanes(const Share &a, float c_hi, float c_lo) {
    const float beyond = a.s - 1.0f;
    return join<SUMS>(Stat{a.m, a.m == -INFINITY ? a.s : fmaf(beyond, kEx2Low, beyond), a.u}, 32, c_hi, c_lo);
}
// sum 2^(d (c_hi + c_lo)) = sum e (1 + ln2 d c_lo) up to 1e-12
__device__ __forceinline__ void with_low(Stat &a, float c_hi, float c_lo) { a.more = fmaf(kLn2 * c_lo / c_hi, a.u, a.more); }
__device__ __forceinline__ bool masked(const Stat &a) { return a.u != a.u && a.more == a.more; }

// A row all of whose classes are -inf has no distribution.
__device__ __forceinline__ bool nothing(const Stat &a) { return a.m == -INFINITY && a.more == 0.0f; }

// ---- who works on a row -----------------------------------------------------------------------------
// A row of up to 4 KB is held by one warp in registers. Wider ones belong to a block, which reads them again for the
// gradient, from the L2 cache: at 256 bytes of a row per thread the rows in flight fit it and there are still enough warps.
// Measured with gradients (log-probability, 1 GiB read and written, 164 us of memory): 16384 bf16 columns 185 us with 128
// threads, 231 with 256; 32768 columns 241, 190, 234 with 128, 256, 512. Above 64 KB a cluster shares the row: 131072
// columns 215 us on four blocks, 246 on one, whose rows in flight leave the cache. Without a gradient nothing is read
// again and one block is faster (131072 columns 90 us against 111).
// Tried and slower: rows kept in shared memory, copied ahead of time by a warp of its own (32768 columns 216 us and
// more): one block per SM has too few warps to hide its reductions and exponentials.
constexpr int kAhead = 4;                   // units of a thread whose loads are in flight together
constexpr uint32_t kMaxCluster = 8;
constexpr int kWarpUnits = 8;               // units of a lane of a row held by a warp
struct alignas(16) Message { float m, more, u; int flag; };

// A block's part of a row: units [first, first + units) of its span, with the head before unit 0 and the tail behind the last.
template <typename T> struct Part {
    static constexpr int V = Unit<T>::V;
    uint32_t begin, head, units, tail;      // begin: element of the row at which the units start
    __device__ __forceinline__ Part(const Span<T> &sp, uint32_t rank, uint32_t ranks) {
        const uint32_t u0 = (uint32_t)((uint64_t)sp.units * rank / ranks), u1 = (uint32_t)((uint64_t)sp.units * (rank + 1) / ranks);
        begin = sp.head + u0 * V;
        units = u1 - u0;
        head = rank == 0 ? sp.head : 0;
        tail = rank == ranks - 1 ? sp.tail : 0;
    }
    __device__ __forceinline__ Unit<T> load(const T *x, uint32_t u) const { return Unit<T>{*reinterpret_cast<const uint4 *>(x + begin + (size_t)u * V)}; }
    __device__ __forceinline__ bool holds(uint32_t j) const { return j + head >= begin && j < begin + units * V + tail; }
    // place of element j among bits or units: the head's unit, the units, the tail's unit; elements count from the head's end
    __device__ __forceinline__ uint32_t place(uint32_t j) const { return j - begin + V; }
};

struct Coef { float a, b, at_label; };      // d_j = e_j (a + b t2_j), plus at_label at the label

// NT threads that work on one row together.
template <int NT> struct Team {
    struct Shared { Stat red[2][NT / 32]; Message box[2][kMaxCluster]; Coef coef; };
    Shared &sh;
    uint32_t tid, lane, rank, ranks, merged, met;
    __device__ __forceinline__ explicit Team(Shared &s) : sh(s), tid(threadIdx.x), lane(threadIdx.x & 31), rank(tc::cluster_rank()), ranks(tc::cluster_size()), merged(0), met(0) {
        if (ranks > 1) tc::cluster_sync<false>();
    }
    // Every team that was set up either meets or leaves.
    __device__ __forceinline__ void leave() { if (ranks > 1 && met == 0) tc::cluster_wait(); }
    // The block's statistics from those of its threads, in every thread, in a fixed order. Every warp joins all the
    // warps' parts, a lane to each: one after the other they took 10 % of a row of 64 KB.
    template <int SUMS> __device__ __forceinline__ Stat merge(const Share &share, float c_hi, float c_lo) {
        Stat(&red)[NT / 32] = sh.red[merged++ & 1];      // the other one may still be read
        const Stat a = join_lanes<SUMS>(share, c_hi, c_lo);
        if (lane == 0) red[tid / 32] = a;
        __syncthreads();
        return join<SUMS>(red[lane % (NT / 32)], NT / 32, c_hi, c_lo);
    }
    // The cluster's from those of its blocks, in a fixed order. All blocks of the cluster, the same number of times.
    template <int SUMS> __device__ __forceinline__ Stat meet(const Stat &a, int flag, float c_hi, float c_lo, int *any) {
        if (ranks == 1) { *any = flag; return a; }
        if (met == 0) tc::cluster_wait();                    // every block runs: its shared memory may be written
        Message(&box)[kMaxCluster] = sh.box[met++ & 1];  // of the other one a block may still be reading
        if (tid < ranks) {
            const uint32_t at = tc::map_shared(tc::smem_u32(&box[rank]), tid);
            asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(__float_as_uint(a.m)), "r"(__float_as_uint(a.more)), "r"(__float_as_uint(a.u)), "r"(flag) : "memory");
        }
        tc::cluster_sync();
        const Message &b = box[lane & (ranks - 1)];      // a lane to each again; ranks is a power of two
        *any = __any_sync(0xffffffffu, b.flag);
        return join<SUMS>(Stat{b.m, b.more, b.u}, ranks, c_hi, c_lo);
    }
    // A thread's share of the statistics of this block's part of the row at x. Units that do not fill a group are summed one
    // by one, the head and the tail by the form that takes places that are no classes. `leave` takes (unit, its place).
    template <typename T, int SUMS, class Leave>
    __device__ __forceinline__ Share scan(const T *x, const Part<T> &p, float c_hi, float c_lo, const Leave &leave) const {
        constexpr uint32_t V = Part<T>::V;
        Share a{-INFINITY, 0.0f, 0.0f};
        for (uint32_t u = tid; u < p.units; u += NT * kAhead) {
            Unit<T> q[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (u + k * NT < p.units) q[k] = p.load(x, u + k * NT);
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (u + k * NT < p.units) leave(q[k], (u + k * NT + 1) * V);
            if (u + (kAhead - 1) * NT < p.units) {
                accumulate<T, kAhead, SUMS>(a, q, c_hi, c_lo);
            } else {
#pragma unroll
                for (int k = 0; k < kAhead - 1; ++k)
                    if (u + k * NT < p.units) accumulate<T, 1, SUMS>(a, reinterpret_cast<const Unit<T>(&)[1]>(q[k]), c_hi, c_lo);
            }
        }
        constexpr int kEdge = SUMS ? kMasked : kSums;
        if (tid == 0 && p.head) {
            Unit<T> q[1] = {part_unit<T>(x, p.head)};
            leave(q[0], V - p.head);
            accumulate<T, 1, kEdge>(a, q, c_hi, c_lo);
        }
        if (tid == NT - 1 && p.tail) {
            Unit<T> q[1] = {part_unit<T>(x + p.begin + p.units * V, p.tail)};
            leave(q[0], (p.units + 1) * V);
            accumulate<T, 1, kEdge>(a, q, c_hi, c_lo);
        }
        return a;
    }
};
struct LeaveNone {
    template <typename U> __device__ __forceinline__ void operator()(U &, uint32_t) const {}
};

// ---- gradient rows ---------------------------------------------------------------------------
// Columns [from, to) of row `row`: zero.
template <typename T, int NT> __device__ __forceinline__ void zero_row(const Rows &r, uint32_t row, uint32_t from, uint32_t to, uint32_t tid) {
    if (from >= to) return;
    T *d = reinterpret_cast<T *>(r.d) + (size_t)row * r.cols + from;
    const Span<T> sp(d, to - from);
    for (uint32_t u = tid; u < sp.units; u += NT) *reinterpret_cast<uint4 *>(d + sp.head + (size_t)u * Span<T>::V) = make_uint4(0, 0, 0, 0);
    if (tid < sp.head) d[tid] = from_f32<T>(0.0f);
    if (tid < sp.tail) d[sp.n - sp.tail + tid] = from_f32<T>(0.0f);
}

template <typename T, int SUMS> __device__ __forceinline__ float gradient_of(float x, const Rows &r, float m, const Coef &k) {
    const float d = x - m, t = sizeof(T) == 4 ? fmaf(d, r.c_hi, d * r.c_lo) : d * r.c_hi;   // 16 bits hide the second part
    return ex2(t) * (SUMS ? fmaf(k.b, SUMS == kMasked ? fmaxf(t, -200.0f) : t, k.a) : k.a);
}
template <typename T, int SUMS> __device__ __forceinline__ void gradient_unit(Unit<T> &q, const Rows &r, float m, const Coef &k) {
    const f32x2 less = pair(-m, -m), hi = pair(r.c_hi, r.c_hi), ka = pair(k.a, k.a), kb = pair(k.b, k.b);
#pragma unroll
    for (int i = 0; i < Unit<T>::V / 2; ++i) {
        const f32x2 d = add2(q.get(i), less), t = sizeof(T) == 4 ? fma2(d, hi, mul2(d, pair(r.c_lo, r.c_lo))) : mul2(d, hi);
        q.set(i, mul2(ex2_2(t), SUMS ? fma2(kb, SUMS == kMasked ? floor2(t) : t, ka) : ka));
    }
}

// Up to V - 1 elements of a row at its head or tail.
template <typename T, int SUMS>
__device__ __forceinline__ void write_edge(const Rows &r, T *d, Unit<T> q, uint32_t first, uint32_t count, float m, const Coef &k, int32_t label, T at_label) {
    gradient_unit<T, SUMS ? kMasked : kSums>(q, r, m, k);
    const T *e = reinterpret_cast<const T *>(&q.q);
#pragma unroll
    for (uint32_t j = 0; j < Unit<T>::V - 1; ++j)
        if (j < count) d[first + j] = e[j];
    if (label >= 0 && (uint32_t)label - first < count) d[label] = at_label;
}
// One unit at element `at` of the row; the label's element is written behind its unit by the thread that wrote that.
template <typename T> __device__ __forceinline__ void write_unit(T *d, const Unit<T> &q, size_t at, bool whole, bool has_label, int32_t label, T at_label) {
    if (whole) {
        *reinterpret_cast<uint4 *>(d + at) = q.q;
    } else {                                // the gradient lies on another offset within 16 bytes than the logits
        const T *e = reinterpret_cast<const T *>(&q.q);
#pragma unroll
        for (int j = 0; j < Unit<T>::V; ++j) d[at + j] = e[j];
    }
    if (has_label) d[label] = at_label;
}
// The gradient of this block's part of a row from its logits; label < 0: none. It may lie where the logits lie: a thread
// stores a unit after it has read it.
template <typename T, int NT, int SUMS>
__device__ __forceinline__ void write_row(const Rows &r, uint32_t row, const Part<T> &p, uint32_t rank, uint32_t ranks, float m, const Coef &k, int32_t label, float at) {
    constexpr uint32_t V = Part<T>::V;
    const size_t base = (size_t)row * r.cols;
    const T *x = reinterpret_cast<const T *>(r.x) + base;
    T *d = reinterpret_cast<T *>(r.d) + base;
    const bool whole = reinterpret_cast<uintptr_t>(d + p.begin) % 16 == 0;
    const uint32_t label_unit = (uint32_t)(label - (int32_t)p.begin) / V;      // beyond all units if it is not here
    const T at_label = from_f32<T>(gradient_of<T, SUMS ? kMasked : kSums>(at, r, m, k) + k.at_label);
    for (uint32_t u = threadIdx.x; u < p.units; u += NT * kAhead) {
        Unit<T> q[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (u + j * NT < p.units) q[j] = p.load(x, u + j * NT);
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (u + j * NT >= p.units) break;
            gradient_unit<T, SUMS>(q[j], r, m, k);
            write_unit<T>(d, q[j], p.begin + (size_t)(u + j * NT) * V, whole, label_unit == u + j * NT, label, at_label);
        }
    }
    if (threadIdx.x == 0 && p.head) write_edge<T, SUMS>(r, d, part_unit<T>(x, p.head), 0, p.head, m, k, label, at_label);
    if (threadIdx.x == NT - 1 && p.tail)
        write_edge<T, SUMS>(r, d, part_unit<T>(x + p.begin + p.units * V, p.tail), p.begin + p.units * V, p.tail, m, k, label, at_label);
    if (rank == ranks - 1) zero_row<T, NT>(r, row, r.classes, r.cols, threadIdx.x);
}

// ---- losses on the log-probability of one class per row ------------------------------------------
// Each fetches what a row brings along (fetch), says which class it asks for (label_of; below 0: the row does not count),
// and turns its statistics into outputs and the coefficients of its gradient (finish; called by a warp with the same
// values, `first` is one of its threads).
__device__ __forceinline__ int32_t checked_label(const Rows &r, int32_t label, bool first) {
    if (label >= 0 && (uint32_t)label >= r.classes) {
        if (first) atomicOr(r.err, kErrLabel);
        return -1;
    }
    return label;
}
// log p of the label, and sum e t / s in natural units
__device__ __forceinline__ double log_prob(const Rows &r, const Stat &a, double log_s, float x) { return ((double)x - (double)a.m) * r.inv_t - log_s; }

struct LabelLogprob {
    const int32_t *labels;
    float *logp, *entropy;
    struct In { int32_t label; };
    __device__ __forceinline__ In fetch(uint32_t row) const { return In{labels[row]}; }
    static __device__ __forceinline__ int32_t label_of(const In &in) { return in.label; }
    __device__ __forceinline__ void skip(uint32_t row) const {
        logp[row] = 0.0f;
        if (entropy) entropy[row] = 0.0f;
    }
    __device__ __forceinline__ Coef finish(const Rows &r, uint32_t row, const Stat &a, float x, const In &, bool first) const {
        if (first) {
            const double log_s = a.log_s();
            logp[row] = (float)log_prob(r, a, log_s, x);
            if (entropy) entropy[row] = (float)(log_s - (double)(a.u / a.s() * kLn2));
        }
        return Coef{0.0f, 0.0f, 0.0f};
    }
};

// d = k [ g (1[j = l] - p_j) - h p_j (log p_j + H) ],  log p_j + H = ln2 (t2_j - u / s)
struct LabelLogprobBackward {
    const int32_t *labels;
    const float *d_logp, *d_entropy;
    struct In { int32_t label; float g, h; };
    __device__ __forceinline__ In fetch(uint32_t row) const { return In{labels[row], d_logp[row], d_entropy ? d_entropy[row] * kLn2 : 0.0f}; }
    static __device__ __forceinline__ int32_t label_of(const In &in) { return in.label; }
    __device__ __forceinline__ void skip(uint32_t) const {}
    __device__ __forceinline__ Coef finish(const Rows &r, uint32_t, const Stat &a, float, const In &in, bool) const {
        const float f = r.k / a.s();
        return Coef{f * (in.h * (a.u / a.s()) - in.g), -f * in.h, r.k * in.g};
    }
};

// rho = exp(logp - old), loss = w [ -min(rho A, clip(rho) A) + beta (exp(d) - d - 1) - eta H ], d = ref - logp
struct Policy {
    const int32_t *actions;
    const float *old, *advantages, *ref, *weights;
    float lo, hi, beta, eta;
    float *loss, *logp, *kl, *entropy;
    struct In { int32_t label; float w, old, adv, ref; };
    __device__ __forceinline__ In fetch(uint32_t row) const {
        return In{actions[row], weights ? weights[row] : 1.0f, old[row], advantages[row], ref ? ref[row] : 0.0f};
    }
    static __device__ __forceinline__ int32_t label_of(const In &in) { return in.w == 0.0f ? -1 : in.label; }
    __device__ __forceinline__ void skip(uint32_t row) const {
        loss[row] = logp[row] = kl[row] = 0.0f;
        if (entropy) entropy[row] = 0.0f;
    }
    // exp(d) - 1 - d without the cancellation of small d; infinite for an action that is masked (d = inf)
    static __device__ __forceinline__ float expm1_less(float d) {
        if (fabsf(d) > 0.5f) {
            const float e = expm1f(d);
            return e == INFINITY ? e : e - d;
        }
        float p = 1.0f / 40320.0f;
        p = fmaf(p, d, 1.0f / 5040.0f); p = fmaf(p, d, 1.0f / 720.0f); p = fmaf(p, d, 1.0f / 120.0f);
        p = fmaf(p, d, 1.0f / 24.0f); p = fmaf(p, d, 1.0f / 6.0f); p = fmaf(p, d, 0.5f);
        return p * d * d;
    }
    __device__ __forceinline__ Coef finish(const Rows &r, uint32_t row, const Stat &a, float x, const In &in, bool first) const {
        const double log_s = a.log_s(), lp = log_prob(r, a, log_s, x);
        const float w = in.w, adv = in.adv;
        const float rho = expf((float)(lp - (double)in.old));
        const float d = ref ? (float)((double)in.ref - lp) : 0.0f, h = (float)(log_s - (double)(a.u / a.s() * kLn2));
        const float plain = adv == 0.0f && rho == INFINITY ? 0.0f : rho * adv, held = fminf(fmaxf(rho, lo), hi) * adv;
        const bool clipped = (adv > 0.0f && rho > hi) || (adv < 0.0f && rho < lo);
        float g = clipped ? 0.0f : -plain;
        if (beta != 0.0f) g -= beta * expm1f(d);      // not 0 * inf: without the factor the KL is reported only
        const float kl_v = ref ? expm1_less(d) : 0.0f;
        if (first) {
            float l = clipped ? -held : -plain;      // the larger one, or NaN, which a maximum would drop
            if (beta != 0.0f) l += beta * kl_v;
            if (eta != 0.0f) l -= eta * h;
            loss[row] = w * l;
            logp[row] = (float)lp;
            kl[row] = kl_v;
            if (entropy) entropy[row] = h;
        }
        g *= w;
        const float f = r.k / a.s(), q = w * eta * kLn2;
        return Coef{f * (-g - q * (a.u / a.s())), f * q, r.k * g};
    }
};

// Log-probabilities of the rows of packed sequences, with what later kernels need of a row: its maximum and sum (0: the
// row does not count), what f32 leaves of the log-probability, and room for the factor on its gradient. Rows outside
// the sequences do not count.
struct alignas(16) Kept { float m, s, low, g; };
struct SequenceLogprob {
    const int32_t *labels, *offsets;
    uint32_t sequences;
    float *row_logp;
    Kept *kept;
    struct In { int32_t label; };
    __device__ __forceinline__ In fetch(uint32_t row) const {
        const bool inside = (int64_t)offsets[0] <= (int64_t)row && (int64_t)row < (int64_t)offsets[sequences];
        return In{inside ? labels[row] : -1};
    }
    static __device__ __forceinline__ int32_t label_of(const In &in) { return in.label; }
    __device__ __forceinline__ void skip(uint32_t row) const {
        row_logp[row] = 0.0f;
        kept[row] = Kept{0.0f, 0.0f, 0.0f, 0.0f};
    }
    __device__ __forceinline__ Coef finish(const Rows &r, uint32_t row, const Stat &a, float x, const In &, bool first) const {
        if (first) {
            const double lp = log_prob(r, a, a.log_s(), x);
            row_logp[row] = (float)lp;
            Kept k{a.m, a.s(), 0.0f, 0.0f};
            if (isfinite(lp)) k.low = (float)(lp - (double)(float)lp);
            kept[row] = k;
        }
        return Coef{0.0f, 0.0f, 0.0f};
    }
};

// A cluster (mostly of one block) per row.
template <typename T, int NT, class Op, int SUMS, bool GRAD>
__global__ void __launch_bounds__(NT) row_kernel(Rows r, Op op) {
    __shared__ typename Team<NT>::Shared shared;
    Team<NT> team(shared);
    const uint32_t row = blockIdx.x / team.ranks;
    const bool first = team.tid == 0 && team.rank == 0;
    grid_ready();
    const T *x = reinterpret_cast<const T *>(r.x) + (size_t)row * r.cols;
    const typename Op::In in = op.fetch(row);
    const int32_t label = checked_label(r, Op::label_of(in), first);
    auto skip = [&] {
        team.leave();
        if (first) op.skip(row);
        if (GRAD) zero_row<T, NT>(r, row, (uint32_t)((uint64_t)r.cols * team.rank / team.ranks), (uint32_t)((uint64_t)r.cols * (team.rank + 1) / team.ranks), team.tid);
    };
    if (label < 0) return skip();
    const float at = to_f32(x[label]);
    const Part<T> part(Span<T>(x, r.classes), team.rank, team.ranks);
    int any;
    Stat a = team.template merge<SUMS>(team.template scan<T, SUMS>(x, part, r.c_hi, r.c_lo, LeaveNone()), r.c_hi, r.c_lo);
    a = team.template meet<SUMS>(a, 0, r.c_hi, r.c_lo, &any);
    bool again = false;
    if (SUMS == kEntropy && masked(a)) {
        again = true;
        a = team.template merge<kMasked>(team.template scan<T, kMasked>(x, part, r.c_hi, r.c_lo, LeaveNone()), r.c_hi, r.c_lo);
        a = team.template meet<kMasked>(a, 0, r.c_hi, r.c_lo, &any);
    }
    if (SUMS) with_low(a, r.c_hi, r.c_lo);
    if (nothing(a)) return skip();
    // a few hundred instructions: one warp's
    if (team.tid < 32) {
        const Coef k = op.finish(r, row, a, at, in, first);
        if (GRAD && team.tid == 0) shared.coef = k;
    }
    if (!GRAD) return;
    __syncthreads();
    const Coef k = shared.coef;
    if (SUMS == kEntropy && again) write_row<T, NT, kMasked>(r, row, part, team.rank, team.ranks, a.m, k, label, at);
    else write_row<T, NT, SUMS>(r, row, part, team.rank, team.ranks, a.m, k, label, at);
}

// A warp per row, which it holds in registers: up to 32 x kWarpUnits units and the edges. SUMS: kSums or kMasked.
template <typename T, class Op, int SUMS, bool GRAD>
__global__ void __launch_bounds__(kThreads) warp_kernel(Rows r, Op op) {
    constexpr uint32_t V = Part<T>::V;
    const uint32_t lane = threadIdx.x & 31, row = blockIdx.x * kWarps + threadIdx.x / 32;
    const bool first = lane == 0;
    grid_ready();
    if (row >= r.rows) return;
    const T *x = reinterpret_cast<const T *>(r.x) + (size_t)row * r.cols;
    const typename Op::In in = op.fetch(row);
    const Part<T> p(Span<T>(x, r.classes), 0, 1);
    Unit<T> q[kWarpUnits], edge = no_unit<T>();
#pragma unroll
    for (int k = 0; k < kWarpUnits; ++k) q[k] = lane + k * 32 < p.units ? p.load(x, lane + k * 32) : no_unit<T>();
    const uint32_t side = lane == 0 ? p.head : lane == 31 ? p.tail : 0, from = lane == 0 ? 0 : p.begin + p.units * V;
    if (side) edge = part_unit<T>(x + from, side);
    const int32_t label = checked_label(r, Op::label_of(in), first);
    float at = 0.0f;
    Stat a{-INFINITY, 0.0f, 0.0f};
    if (label >= 0) {
        at = to_f32(x[label]);
        Share share{-INFINITY, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < kWarpUnits; k += 2)
            if (k * 32 < p.units) accumulate<T, 2, SUMS>(share, reinterpret_cast<const Unit<T>(&)[2]>(q[k]), r.c_hi, r.c_lo);
        if (side) accumulate<T, 1, SUMS>(share, reinterpret_cast<const Unit<T>(&)[1]>(edge), r.c_hi, r.c_lo);
        a = join_lanes<SUMS>(share, r.c_hi, r.c_lo);
        if (SUMS) with_low(a, r.c_hi, r.c_lo);
    }
    T *d = reinterpret_cast<T *>(r.d) + (size_t)row * r.cols;
    if (label < 0 || nothing(a)) {
        if (first) op.skip(row);
        if (GRAD) zero_row<T, 32>(r, row, 0, r.cols, lane);
        return;
    }
    const Coef k = op.finish(r, row, a, at, in, first);
    if (!GRAD) return;
    const bool whole = reinterpret_cast<uintptr_t>(d + p.begin) % 16 == 0;
    const uint32_t label_unit = (uint32_t)(label - (int32_t)p.begin) / V;
    const T at_label = from_f32<T>(gradient_of<T, SUMS>(at, r, a.m, k) + k.at_label);
#pragma unroll
    for (int j = 0; j < kWarpUnits; ++j) {
        const uint32_t u = lane + j * 32;
        if (u >= p.units) break;
        gradient_unit<T, SUMS>(q[j], r, a.m, k);
        write_unit<T>(d, q[j], p.begin + (size_t)u * V, whole, label_unit == u, label, at_label);
    }
    if (side) write_edge<T, SUMS>(r, d, edge, from, side, a.m, k, label, at_label);
    zero_row<T, 32>(r, row, r.classes, r.cols, lane);
}

// ---- preference loss: sequences ---------------------------------------------------------------------
struct Pairs {
    const int32_t *offsets;
    uint32_t pairs, rows, form, average;
    const float *ref, *weights, *row_logp;
    Kept *kept;
    double beta, smooth, margin;
    float *loss, *margins, *logp;
    int *err;
};

// One block per pair: the sums of both sequences in 64 bits (a thousand terms of ten lose four digits in 32), the
// loss as a function of their difference, and the factor on the gradient of each row's log-probability.
__global__ void __launch_bounds__(kThreads) pair_kernel(Pairs p) {
    __shared__ double sum_red[2][kWarps];
    __shared__ uint32_t n_red[2][kWarps];
    const uint32_t pair = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    grid_ready();
    int32_t from[2], to[2];
    double sum[2];
    uint32_t n[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        from[h] = p.offsets[2 * pair + h];
        to[h] = p.offsets[2 * pair + h + 1];
        if (from[h] < 0 || to[h] < from[h] || (uint32_t)to[h] > p.rows) {
            if (threadIdx.x == 0) atomicOr(p.err, kErrOffsets);
            from[h] = to[h] = 0;
        }
        double s = 0.0;
        uint32_t c = 0;
        for (int32_t r = from[h] + (int32_t)threadIdx.x; r < to[h]; r += kThreads)
            if (p.kept[r].s != 0.0f) { s += (double)p.row_logp[r] + (double)p.kept[r].low; ++c; }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, o);
            c += __shfl_xor_sync(0xffffffffu, c, o);
        }
        if (lane == 0) { sum_red[h][warp] = s; n_red[h][warp] = c; }
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        sum[h] = 0.0;
        n[h] = 0;
        for (int w = 0; w < kWarps; ++w) { sum[h] += sum_red[h][w]; n[h] += n_red[h][w]; }
        if (p.average && n[h]) sum[h] /= (double)n[h];
    }
    const double diff = (sum[0] - (p.ref ? (double)p.ref[2 * pair] : 0.0)) - (sum[1] - (p.ref ? (double)p.ref[2 * pair + 1] : 0.0));
    const double m = p.beta * diff - p.margin, w = p.weights ? (double)p.weights[pair] : 1.0;
    double value, slope;
    if (p.form == SK_PREFERENCE_SIGMOID) {
        const double l = log1p(exp(-fabs(m)));           // -log sigmoid(m) = l + max(-m, 0), -log sigmoid(-m) = l + max(m, 0)
        value = p.smooth < 1.0 ? (1.0 - p.smooth) * (l + fmax(-m, 0.0)) : 0.0;
        if (p.smooth > 0.0) value += p.smooth * (l + fmax(m, 0.0));   // not 0 * inf
        slope = p.smooth - 1.0 / (1.0 + exp(m));
    } else if (p.form == SK_PREFERENCE_HINGE) {
        value = m >= 1.0 ? 0.0 : 1.0 - m;                // not fmax, which drops NaN
        slope = m < 1.0 ? -1.0 : m >= 1.0 ? 0.0 : m;
    } else {
        value = (m - 0.5) * (m - 0.5);
        slope = 2.0 * (m - 0.5);
    }
    if (w == 0.0) value = slope = 0.0;                    // a pair that does not count, whatever it holds
    if (threadIdx.x == 0) {
        p.loss[pair] = (float)(w * value);
        p.margins[pair] = (float)m;
        p.logp[2 * pair] = (float)sum[0];
        p.logp[2 * pair + 1] = (float)sum[1];
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        double g = w * slope * (h ? -p.beta : p.beta);
        if (p.average && n[h]) g /= (double)n[h];
        for (int32_t r = from[h] + (int32_t)threadIdx.x; r < to[h]; r += kThreads)
            if (p.kept[r].s != 0.0f) atomicAdd(&p.kept[r].g, (float)g);      // 0 before: its pair's alone, unless offsets fall and pairs overlap
    }
}

// d = k g (1[j = l] - p_j) from the kept maximum and sum. A row without a sum got no log-probability.
template <typename T, int NT>
__global__ void __launch_bounds__(NT) sequence_gradient_kernel(Rows r, const int32_t *labels, const Kept *kept) {
    const uint32_t row = r.rows - 1 - blockIdx.x;       // the rows read last are still in the L2 cache
    grid_ready();
    const Kept k = kept[row];
    if (k.s == 0.0f || k.g == 0.0f) {
        zero_row<T, NT>(r, row, 0, r.cols, threadIdx.x);
        return;
    }
    const T *x = reinterpret_cast<const T *>(r.x) + (size_t)row * r.cols;
    const int32_t label = labels[row];
    write_row<T, NT, kSums>(r, row, Part<T>(Span<T>(x, r.classes), 0, 1), 0, 1, k.m, Coef{-r.k * k.g / k.s, 0.0f, r.k * k.g}, label, to_f32(x[label]));
}

// ---- distillation --------------------------------------------------------------------------------
struct Distill {
    const int32_t *indices;
    const void *values;
    uint32_t values_type, k;
    const float *lse, *weights;
    float *loss;
    double factor;                          // T^2
};
__device__ __forceinline__ float teacher_value(const Distill &d, size_t i) {
    return d.values_type == SK_F32 ? reinterpret_cast<const float *>(d.values)[i]
           : d.values_type == SK_F16 ? to_f32(reinterpret_cast<const __half *>(d.values)[i])
                                     : to_f32(reinterpret_cast<const __nv_bfloat16 *>(d.values)[i]);
}

// With q_k the teacher's probabilities of its list (a softmax over it, or exp(v_k / T - lse)), Q their sum, r = 1 - Q the
// mass outside (given lse; else 0) and S the student's probability outside the list,
//   loss = w T^2 [ sum q_k (log q_k - log p_k) + r (log r - log S) ]
//   d_j  = w T loss_scale [ (Q + r) p_j - r e_j / (sum of e outside)   outside the list ]
//                         [ (Q + r) p_j - q_j                          at its classes   ]
// S is a sum of its own over the classes outside (1 - sum p_k would cancel): a bit for each class of the block's part says
// which are listed, and these count as -inf where the row is summed; they are written by themselves behind the rest of the
// gradient. Setting its bit also tells an entry whether its class was given before; the masses then add at the class.
// The classes outside keep their own maximum: relative to the row's they vanish where the student holds the list 87 (in
// (x - m) / T) or more above them, and with them log S and the term r e_j / (sum of e outside), whose sum is r all the same.
template <int NT> struct DistillShared {
    typename Team<NT>::Shared team;
    int32_t idx[kMaxList];
    struct { double to_mass; float m, m_out, f, of_s, outside; bool dead; } found;   // what the list's warp made of it
    double share[kMaxList];                 // the teacher's share (not normalised): the mass outside the list is 1 less their sum
    float val[kMaxList], sx[kMaxList];      // the teacher's logit, the student's
};
// Bytes of the bits of one of `ranks` parts of a row: one per class, the head and the tail in units of their own.
template <typename T> inline size_t bit_bytes(uint32_t classes, uint32_t ranks) {
    const size_t units = (size_t)classes / Unit<T>::V, words = (((units + ranks - 1) / ranks + 2) * Unit<T>::V + 31) / 32;
    return words * 4;
}
template <typename T, int NT>
__global__ void __launch_bounds__(NT, 1536 / NT) distill_kernel(Rows r, Distill t) {
    constexpr uint32_t V = Unit<T>::V;
    extern __shared__ uint32_t bits[];
    __shared__ DistillShared<NT> sh;
    auto &idx = sh.idx;
    auto &found = sh.found;
    auto &share = sh.share;
    auto &val = sh.val, &sx = sh.sx;
    Team<NT> team(sh.team);
    const uint32_t row = blockIdx.x / team.ranks, tid = team.tid, lane = team.lane;
    const bool first = tid == 0 && team.rank == 0;
    grid_ready();
    const T *x = reinterpret_cast<const T *>(r.x) + (size_t)row * r.cols;
    const float w = t.weights ? t.weights[row] : 1.0f;
    const int32_t early = tid < t.k ? t.indices[(size_t)row * t.k + tid] : -1;      // the longest chain of loads starts first
    auto nothing_to_learn = [&] {
        team.leave();
        if (first) t.loss[row] = 0.0f;
        if (r.d) zero_row<T, NT>(r, row, (uint32_t)((uint64_t)r.cols * team.rank / team.ranks), (uint32_t)((uint64_t)r.cols * (team.rank + 1) / team.ranks), tid);
    };
    if (w == 0.0f) return nothing_to_learn();
    const Part<T> part(Span<T>(x, r.classes), team.rank, team.ranks);
    const uint32_t words = ((part.units + 2) * V + 31) / 32;
    for (uint32_t i = tid; i < words; i += NT) bits[i] = 0;
    for (uint32_t i = tid; i < t.k; i += NT) {
        int32_t c = i == tid ? early : t.indices[(size_t)row * t.k + i];
        if (c >= 0 && (uint32_t)c >= r.classes) { if (team.rank == 0) atomicOr(r.err, kErrList); c = -1; }
        idx[i] = c;
        val[i] = c >= 0 ? teacher_value(t, (size_t)row * t.k + i) : -INFINITY;
        sx[i] = c >= 0 ? to_f32(x[c]) : -INFINITY;
    }
    __syncthreads();
    auto mine = [&](uint32_t i) { return idx[i] >= 0 && part.holds((uint32_t)idx[i]); };
    float top = -INFINITY;
    bool some = false;
    for (uint32_t i = lane; i < t.k; i += 32) { top = fmaxf(top, val[i]); some |= idx[i] >= 0; }
    top = max_of_warp(top);
    some = __any_sync(0xffffffffu, some);
    const double shift = t.lse ? (double)t.lse[row] : (double)top * r.inv_t;
    bool twice = false;
    for (uint32_t i = tid; i < t.k; i += NT) {
        if (mine(i)) {
            const uint32_t b = part.place((uint32_t)idx[i]);
            twice |= (atomicOr(&bits[b / 32], 1u << (b % 32)) >> (b % 32)) & 1u;
        }
        share[i] = val[i] == -INFINITY ? 0.0 : exp((double)val[i] * r.inv_t - shift);
    }
    twice = __syncthreads_or(twice);
    Stat a = team.template merge<kSums>(team.template scan<T, kSums>(x, part, r.c_hi, r.c_lo, [&](Unit<T> &q, uint32_t place) {
        const uint32_t mark = bits[place / 32] >> (place % 32) & ((1u << V) - 1u);
        if (mark)
#pragma unroll
            for (int j = 0; j < (int)V; ++j) if (mark >> j & 1u) q.drop(j);
    }), r.c_hi, r.c_lo);
    int any;
    a = team.template meet<kSums>(a, twice, r.c_hi, r.c_lo, &any);
    twice = any;
    auto leads = [&](uint32_t i) {          // the first entry of its class
        if (twice)
            for (uint32_t o = 0; o < i; ++o)
                if (idx[o] == idx[i]) return false;
        return idx[i] >= 0;
    };
    if (tid < 32) {                         // the list is one warp's
        float best = -INFINITY, listed = 0.0f;
        for (uint32_t i = lane; i < t.k; i += 32) best = max_or_nan(best, sx[i]);
        // NaN beside classes at -inf alone is no empty row
        const float m = max_or_nan(a.m == -INFINITY ? a.m + a.more : a.m, max_of_warp_or_nan(best));
        const bool dead = (!t.lse && (!some || top == -INFINITY)) || (m == -INFINITY && a.more == 0.0f);
        const float outside = a.m == -INFINITY ? a.more : a.s() * pow2(factor_log<kSums>(a.m, m, r.c_hi, r.c_lo));
        double mass = 0.0;
        for (uint32_t i = lane; i < t.k; i += 32) {
            const float d = sx[i] - m, e = pow2(fmaf(d, r.c_hi, d * r.c_lo));
            if (leads(i)) listed += e;
            mass += share[i];
        }
        listed = warp_sum(listed);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mass += __shfl_xor_sync(0xffffffffu, mass, o);
        const float s = outside + listed;
        const double to_mass = t.lse ? 1.0 : (double)(1.0f / (float)mass);
        double rest = t.lse ? 1.0 - mass : 0.0;
        if (rest <= kLeastTail) rest = 0.0;
        if (team.rank == 0 && !dead) {
            const double log_s = log_wide(s), log_mass = t.lse ? 0.0 : log_wide((float)mass);
            double l = 0.0;
            for (uint32_t i = lane; i < t.k; i += 32) {
                const double log_q = (double)val[i] * r.inv_t - shift - log_mass;
                const double q = share[i] * to_mass;
                if (q != 0.0) l += q * (log_q - (((double)sx[i] - (double)m) * r.inv_t - log_s));
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
            if (rest > 0.0) l += rest * (log(rest) - (a.m == -INFINITY ? (a.more == 0.0f ? -INFINITY : (double)a.more) : ((double)a.m - (double)m) * r.inv_t + a.log_s() - log_s));
            if (first) t.loss[row] = (float)(t.factor * (double)w * l);
        }
        if (tid == 0) {
            // k = loss scale / T, the gradient's factor w T loss scale = w k T^2
            found.m = m;
            found.to_mass = to_mass;
            found.f = (float)((double)w * (double)r.k * t.factor);
            const double total = t.lse ? mass + rest : 1.0;
            found.of_s = (float)total / s;
            found.m_out = a.m == -INFINITY ? m - m : a.m;      // none: 0, or NaN for the row
            found.outside = a.m == -INFINITY ? 0.0f : (float)(total * (double)(outside / s) - rest) / a.s();
            found.dead = dead;
        }
    }
    if (!r.d && team.ranks == 1) {
        if (tid == 0 && found.dead) t.loss[row] = 0.0f;
        return;
    }
    __syncthreads();
    if (found.dead) return nothing_to_learn();
    if (!r.d) return;
    write_row<T, NT, kSums>(r, row, part, team.rank, team.ranks, found.m_out, Coef{found.f * found.outside, 0.0f, 0.0f}, -1, 0.0f);
    __syncthreads();                        // the list's classes are written again, with their own values
    T *d = reinterpret_cast<T *>(r.d) + (size_t)row * r.cols;
    for (uint32_t i = tid; i < t.k; i += NT) {
        if (!mine(i) || !leads(i)) continue;
        double q = 0.0;
        for (uint32_t o = i; o < (twice ? t.k : i + 1); ++o)
            if (idx[o] == idx[i]) q += share[o] * found.to_mass;
        const float df = sx[i] - found.m, e = ex2(fmaf(df, r.c_hi, df * r.c_lo));
        d[idx[i]] = from_f32<T>(found.f * (found.of_s * e - (float)q));
    }
}

} // namespace loss
} // namespace sk
