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

namespace sk {
namespace loss {

constexpr int kThreads = 256, kWarps = kThreads / 32;
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
// log of a sum of ex2 results of which the largest is 1. The instruction's results are 5.0e-8 too small on average
// (measured over [-32, 0), the same in every octave; 1.4e-7 at most, and exact for 1): the same sign in every row, which
// the sum over a sequence would not average out. It made 8e-6 of a preference margin of sequences that differ by
// hundreds of rows.
constexpr double kEx2Low = 5.0e-8;
__device__ __forceinline__ double log_sum(float s) { return log_wide(s) + kEx2Low * (1.0 - 1.0 / (double)s); }

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
// at least -200, where 2^t is 0 already: 0 * -inf does not arise
__device__ __forceinline__ f32x2 floor2(f32x2 t) { const float2 v = halves(t); return pair(fmaxf(v.x, -200.0f), fmaxf(v.y, -200.0f)); }

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
    __device__ __forceinline__ void put(int j, float v) { (&q.x)[j] = __float_as_uint(v); }
    __device__ __forceinline__ float at(int j) const { return __uint_as_float((&q.x)[j]); }
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
    __device__ __forceinline__ float at(int j) const { const float2 f = halves(get(j / 2)); return j & 1 ? f.y : f.x; }
    __device__ __forceinline__ void drop(int j) { uint32_t &w = (&q.x)[j / 2]; w = j & 1 ? (w & 0xFFFFu) | (kNone & 0xFFFF0000u) : (w & 0xFFFF0000u) | (kNone & 0xFFFFu); }
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
    __device__ __forceinline__ float at(int j) const { const float2 f = halves(get(j / 2)); return j & 1 ? f.y : f.x; }
    __device__ __forceinline__ void drop(int j) { uint32_t &w = (&q.x)[j / 2]; w = j & 1 ? (w & 0xFFFFu) | (kNone & 0xFFFF0000u) : (w & 0xFFFF0000u) | (kNone & 0xFFFFu); }
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
struct Stat { float m, s, u; };             // maximum, sum e, sum e t2 (t2 = t log2 e), relative to m

// (s, u) of a partial sum relative to m, seen from the larger maximum `to`.
__device__ __forceinline__ void rescale(Stat &a, float to, float c) {
    if (a.m == -INFINITY) { a.m = to; return; }   // holds no class (or only NaN, which s keeps)
    const float d = (a.m - to) * c, f = ex2(d);
    a.u = f * (a.u + fmaxf(d, -200.0f) * a.s);
    a.s *= f;
    a.m = to;
}

template <typename T, int U, bool ENT> __device__ __forceinline__ void accumulate(Stat &a, const Unit<T> (&q)[U], float c_hi, float c_lo) {
    float mx = q[0].max();
#pragma unroll
    for (int k = 1; k < U; ++k) mx = fmaxf(mx, q[k].max());
    if (mx > a.m) rescale(a, mx, c_hi);
    const float ref = a.m == -INFINITY ? 0.0f : a.m;
    const f32x2 less = pair(-ref, -ref), hi = pair(c_hi, c_hi), lo = pair(c_lo, c_lo);
    f32x2 s = 0, u = 0;
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
        for (int i = 0; i < Unit<T>::V / 2; ++i) {
            const f32x2 d = add2(q[k].get(i), less), t = fma2(d, hi, mul2(d, lo)), e = ex2_2(t);
            s = add2(s, e);
            if (ENT) u = fma2(e, floor2(t), u);
        }
    const float2 ss = halves(s);
    a.s += ss.x + ss.y;
    if (ENT) {
        const float2 us = halves(u);
        a.u += us.x + us.y;
    }
}

// Units of one thread taken at once: their loads are in flight together.
constexpr int kAhead = 4;

// A thread's share of a row's statistics. `leave` takes (unit, first bit of the unit) and may drop classes from it.
template <typename T, int NT, bool ENT, class Leave>
__device__ __forceinline__ Stat scan_row(const Span<T> &sp, float c_hi, float c_lo, const Leave &leave) {
    constexpr uint32_t V = Span<T>::V;
    Stat a{-INFINITY, 0.0f, 0.0f};
    for (uint32_t u = threadIdx.x; u < sp.units; u += NT * kAhead) {
        Unit<T> q[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) q[k] = u + k * NT < sp.units ? sp.load(u + k * NT) : no_unit<T>();
#pragma unroll
        for (int k = 0; k < kAhead; ++k) leave(q[k], (u + k * NT + 1) * V, u + k * NT < sp.units);
        accumulate<T, kAhead, ENT>(a, q, c_hi, c_lo);
    }
    if (threadIdx.x == 0 && sp.head) {
        Unit<T> q[1] = {part_unit<T>(sp.p, sp.head)};
        leave(q[0], V - sp.head, true);
        accumulate<T, 1, ENT>(a, q, c_hi, c_lo);
    }
    if (threadIdx.x == NT - 1 && sp.tail) {
        Unit<T> q[1] = {part_unit<T>(sp.tail_at(), sp.tail)};
        leave(q[0], (sp.units + 1) * V, true);
        accumulate<T, 1, ENT>(a, q, c_hi, c_lo);
    }
    return a;
}
struct LeaveNone {
    template <typename U> __device__ __forceinline__ void operator()(U &, uint32_t, bool) const {}
};

// One result from those of all threads of the block, in a fixed order.
template <int NT, bool ENT> __device__ __forceinline__ Stat merge(Stat a, Stat (&red)[NT / 32], float c) {
    rescale(a, warp_max(a.m), c);
    a.s = warp_sum(a.s);
    if (ENT) a.u = warp_sum(a.u);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = a;
    __syncthreads();
    Stat b{-INFINITY, 0.0f, 0.0f};
    const uint32_t lane = threadIdx.x & 31;
    if (lane < NT / 32) b = red[lane];
    rescale(b, warp_max(b.m), c);
    b.s = warp_sum(b.s);
    if (ENT) b.u = warp_sum(b.u);
    return b;
}
// A row all of whose classes are -inf has no distribution.
__device__ __forceinline__ bool nothing(const Stat &a) { return a.m == -INFINITY && a.s == 0.0f; }

// ---- gradient rows ---------------------------------------------------------------------------
// Columns [from, cols) of row `row`: zero.
template <typename T, int NT> __device__ __forceinline__ void zero_row(const Rows &r, uint32_t row, uint32_t from) {
    T *d = reinterpret_cast<T *>(r.d) + (size_t)row * r.cols + from;
    const Span<T> sp(d, r.cols - from);
    for (uint32_t u = threadIdx.x; u < sp.units; u += NT) *reinterpret_cast<uint4 *>(d + sp.head + (size_t)u * Span<T>::V) = make_uint4(0, 0, 0, 0);
    if (threadIdx.x < sp.head) d[threadIdx.x] = from_f32<T>(0.0f);
    if (threadIdx.x < sp.tail) d[sp.n - sp.tail + threadIdx.x] = from_f32<T>(0.0f);
}

struct Coef { float a, b, at_label; };      // d_j = e_j (a + b t2_j), plus at_label at the label

// One unit of the gradient; `at`: place of the label in it, or none.
template <typename T, bool ENT> __device__ __forceinline__ void gradient_unit(Unit<T> &q, const Rows &r, float m, const Coef &k, uint32_t at) {
    const f32x2 less = pair(-m, -m), hi = pair(r.c_hi, r.c_hi);
#pragma unroll
    for (int i = 0; i < Unit<T>::V / 2; ++i) {
        const f32x2 d = add2(q.get(i), less), t = sizeof(T) == 4 ? fma2(d, hi, mul2(d, pair(r.c_lo, r.c_lo))) : mul2(d, hi), e = ex2_2(t);
        f32x2 g = mul2(e, ENT ? fma2(floor2(t), pair(k.b, k.b), pair(k.a, k.a)) : pair(k.a, k.a));
        if (at / 2 == (uint32_t)i) g = add2(g, at & 1 ? pair(0.0f, k.at_label) : pair(k.at_label, 0.0f));
        q.set(i, g);
    }
}

// The gradient of one row from its logits; `label` < 0: no correction. The gradient may lie where the logits lie: a
// thread stores a unit after it has read it.
template <typename T, int NT, bool ENT>
__device__ __forceinline__ void write_row(const Rows &r, uint32_t row, float m, const Coef &k, int32_t label) {
    constexpr uint32_t V = Span<T>::V;
    const size_t base = (size_t)row * r.cols;
    const T *x = reinterpret_cast<const T *>(r.x) + base;
    T *d = reinterpret_cast<T *>(r.d) + base;
    const Span<T> sp(x, r.classes);
    const uint32_t rel = (uint32_t)(label - (int32_t)sp.head);         // huge for a label in the head, or none
    if ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(d)) % 16 == 0) {
        for (uint32_t u = threadIdx.x; u < sp.units; u += NT * kAhead) {
            Unit<T> q[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
                if (u + j * NT < sp.units) q[j] = sp.load(u + j * NT);
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                if (u + j * NT >= sp.units) break;
                gradient_unit<T, ENT>(q[j], r, m, k, rel / V == u + j * NT ? rel % V : V);
                *reinterpret_cast<uint4 *>(d + sp.head + (size_t)(u + j * NT) * V) = q[j].q;
            }
        }
    } else {
        for (uint32_t u = threadIdx.x; u < sp.units; u += NT) {
            Unit<T> q = sp.load(u);
            gradient_unit<T, ENT>(q, r, m, k, rel / V == u ? rel % V : V);
            const T *e = reinterpret_cast<const T *>(&q.q);
#pragma unroll
            for (int j = 0; j < (int)V; ++j) d[sp.head + (size_t)u * V + j] = e[j];
        }
    }
    if ((threadIdx.x == 0 && sp.head) || (threadIdx.x == NT - 1 && sp.tail)) {
        for (int side = 0; side < 2; ++side) {
            if (threadIdx.x != (side ? NT - 1 : 0)) continue;
            const uint32_t first = side ? sp.n - sp.tail : 0, count = side ? sp.tail : sp.head;
            Unit<T> q = part_unit<T>(x + first, count);
            const uint32_t in = (uint32_t)(label - (int32_t)first);
            gradient_unit<T, ENT>(q, r, m, k, label >= 0 && in < count ? in : V);
            const T *e = reinterpret_cast<const T *>(&q.q);
#pragma unroll
            for (int j = 0; j < (int)V - 1; ++j)
                if ((uint32_t)j < count) d[first + j] = e[j];
        }
    }
    if (r.cols > r.classes) zero_row<T, NT>(r, row, r.classes);
}

// ---- losses on the log-probability of one class per row ------------------------------------------
// Each says which rows count and which class they ask for (begin), and turns a row's statistics into outputs and the
// coefficients of its gradient (finish; called by every thread with the same values, `first` is one of them).
struct RowIn { float x; int32_t label; };
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
    __device__ __forceinline__ int32_t begin(const Rows &r, uint32_t row, bool first) const { return checked_label(r, labels[row], first); }
    __device__ __forceinline__ void skip(uint32_t row) const {
        logp[row] = 0.0f;
        if (entropy) entropy[row] = 0.0f;
    }
    __device__ __forceinline__ Coef finish(const Rows &r, uint32_t row, const Stat &a, float x, bool first) const {
        if (first) {
            const double log_s = log_sum(a.s);
            logp[row] = (float)log_prob(r, a, log_s, x);
            if (entropy) entropy[row] = (float)(log_s - (double)(a.u / a.s * kLn2));
        }
        return Coef{0.0f, 0.0f, 0.0f};
    }
};

// d = k [ g (1[j = l] - p_j) - h p_j (log p_j + H) ],  log p_j + H = ln2 (t2_j - u / s)
struct LabelLogprobBackward {
    const int32_t *labels;
    const float *d_logp, *d_entropy;
    __device__ __forceinline__ int32_t begin(const Rows &r, uint32_t row, bool first) const { return checked_label(r, labels[row], first); }
    __device__ __forceinline__ void skip(uint32_t) const {}
    __device__ __forceinline__ Coef finish(const Rows &r, uint32_t row, const Stat &a, float, bool) const {
        const float g = d_logp[row], h = d_entropy ? d_entropy[row] * kLn2 : 0.0f, f = r.k / a.s;
        return Coef{f * (h * (a.u / a.s) - g), -f * h, r.k * g};
    }
};

// rho = exp(logp - old), loss = w [ -min(rho A, clip(rho) A) + beta (exp(d) - d - 1) - eta H ], d = ref - logp
struct Policy {
    const int32_t *actions;
    const float *old, *advantages, *ref, *weights;
    float lo, hi, beta, eta;
    float *loss, *logp, *kl, *entropy;
    __device__ __forceinline__ int32_t begin(const Rows &r, uint32_t row, bool first) const {
        return weights && weights[row] == 0.0f ? -1 : checked_label(r, actions[row], first);
    }
    __device__ __forceinline__ void skip(uint32_t row) const {
        loss[row] = logp[row] = kl[row] = 0.0f;
        if (entropy) entropy[row] = 0.0f;
    }
    // exp(d) - 1 - d without the cancellation of small d
    static __device__ __forceinline__ float expm1_less(float d) {
        if (fabsf(d) > 0.5f) return expm1f(d) - d;
        float p = 1.0f / 40320.0f;
        p = fmaf(p, d, 1.0f / 5040.0f); p = fmaf(p, d, 1.0f / 720.0f); p = fmaf(p, d, 1.0f / 120.0f);
        p = fmaf(p, d, 1.0f / 24.0f); p = fmaf(p, d, 1.0f / 6.0f); p = fmaf(p, d, 0.5f);
        return p * d * d;
    }
    __device__ __forceinline__ Coef finish(const Rows &r, uint32_t row, const Stat &a, float x, bool first) const {
        const double log_s = log_sum(a.s), lp = log_prob(r, a, log_s, x);
        const float w = weights ? weights[row] : 1.0f, adv = advantages[row];
        const float rho = expf((float)(lp - (double)old[row]));
        const float d = ref ? (float)((double)ref[row] - lp) : 0.0f, h = (float)(log_s - (double)(a.u / a.s * kLn2));
        const float plain = rho * adv, held = fminf(fmaxf(rho, lo), hi) * adv;
        const bool clipped = (adv > 0.0f && rho > hi) || (adv < 0.0f && rho < lo);
        float g = clipped ? 0.0f : -plain;
        if (ref) g -= beta * expm1f(d);
        const float kl_v = ref ? expm1_less(d) : 0.0f;
        if (first) {
            float l = fmaxf(-plain, -held);
            if (ref) l += beta * kl_v;
            if (eta != 0.0f) l -= eta * h;
            loss[row] = w * l;
            logp[row] = (float)lp;
            kl[row] = kl_v;
            if (entropy) entropy[row] = h;
        }
        g *= w;
        const float f = r.k / a.s, q = w * eta * kLn2;
        return Coef{f * (-g - q * (a.u / a.s)), f * q, r.k * g};
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
    __device__ __forceinline__ int32_t begin(const Rows &r, uint32_t row, bool first) const {
        const bool inside = (int64_t)offsets[0] <= (int64_t)row && (int64_t)row < (int64_t)offsets[sequences];
        return inside ? checked_label(r, labels[row], first) : -1;
    }
    __device__ __forceinline__ void skip(uint32_t row) const {
        row_logp[row] = 0.0f;
        kept[row] = Kept{0.0f, 0.0f, 0.0f, 0.0f};
    }
    __device__ __forceinline__ Coef finish(const Rows &r, uint32_t row, const Stat &a, float x, bool first) const {
        if (first) {
            const double lp = log_prob(r, a, log_sum(a.s), x);
            row_logp[row] = (float)lp;
            Kept k{a.m, a.s, 0.0f, 0.0f};
            if (isfinite(lp)) k.low = (float)(lp - (double)(float)lp);
            kept[row] = k;
        }
        return Coef{0.0f, 0.0f, 0.0f};
    }
};

// One block per row.
template <typename T, int NT, class Op, bool ENT, bool GRAD>
__global__ void __launch_bounds__(NT) row_kernel(Rows r, Op op) {
    __shared__ Stat red[NT / 32];
    const uint32_t row = blockIdx.x;
    const bool first = threadIdx.x == 0;
    grid_ready();
    const T *x = reinterpret_cast<const T *>(r.x) + (size_t)row * r.cols;
    const int32_t label = op.begin(r, row, first);
    Stat a{-INFINITY, 0.0f, 0.0f};
    float at = 0.0f;
    if (label >= 0) {
        at = to_f32(x[label]);
        a = merge<NT, ENT>(scan_row<T, NT, ENT>(Span<T>(x, r.classes), r.c_hi, r.c_lo, LeaveNone()), red, r.c_hi);
    }
    if (label < 0 || nothing(a)) {
        if (first) op.skip(row);
        if (GRAD) zero_row<T, NT>(r, row, 0);
        return;
    }
    const Coef k = op.finish(r, row, a, at, first);
    if (GRAD) write_row<T, NT, ENT>(r, row, a.m, k, label);
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
        value = fmax(1.0 - m, 0.0);
        slope = m < 1.0 ? -1.0 : 0.0;
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
            if (p.kept[r].s != 0.0f) p.kept[r].g = (float)g;
    }
}

// d = k g (1[j = l] - p_j) from the kept maximum and sum. A row without a sum got no log-probability.
template <typename T, int NT>
__global__ void __launch_bounds__(NT) sequence_gradient_kernel(Rows r, const int32_t *labels, const Kept *kept) {
    const uint32_t row = blockIdx.x;
    grid_ready();
    const Kept k = kept[row];
    if (k.s == 0.0f || k.g == 0.0f) {
        zero_row<T, NT>(r, row, 0);
        return;
    }
    write_row<T, NT, false>(r, row, k.m, Coef{-r.k * k.g / k.s, 0.0f, r.k * k.g}, labels[row]);
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

// One block per row. With q_k the teacher's probabilities of its list (a softmax over it, or exp(v_k / T - lse)), Q
// their sum, r = 1 - Q the mass outside (given lse; else 0) and S the student's probability outside the list,
//   loss = w T^2 [ sum q_k (log q_k - log p_k) + r (log r - log S) ]
//   d_j  = w T loss_scale [ (Q + r) p_j - r e_j / (sum of e outside)   outside the list ]
//                         [ (Q + r) p_j - q_j                          at its classes   ]
// S is a sum of its own over the classes outside: 1 - sum p_k would cancel. A bit per class in shared memory says which
// those are; it also finds indices given twice, whose masses add at their class.
template <typename T, int NT>
__global__ void __launch_bounds__(NT) distill_kernel(Rows r, Distill t) {
    constexpr uint32_t V = Span<T>::V;
    extern __shared__ uint32_t bits[];
    __shared__ Stat red[NT / 32];
    __shared__ int32_t idx[kMaxList];
    __shared__ float val[kMaxList], sx[kMaxList];
    const uint32_t row = blockIdx.x, lane = threadIdx.x & 31;
    const bool first = threadIdx.x == 0;
    grid_ready();
    const T *x = reinterpret_cast<const T *>(r.x) + (size_t)row * r.cols;
    const Span<T> sp(x, r.classes);
    const uint32_t words = ((sp.units + 1) * V + sp.tail + 31) / 32;   // unit u has bits from (u + 1) V on, the head those below V
    const float w = t.weights ? t.weights[row] : 1.0f;
    auto nothing_to_learn = [&] {
        if (first) t.loss[row] = 0.0f;
        if (r.d) zero_row<T, NT>(r, row, 0);
    };
    if (w == 0.0f) return nothing_to_learn();
    for (uint32_t i = threadIdx.x; i < words; i += NT) bits[i] = 0;
    __syncthreads();
    bool twice = false;
    for (uint32_t i = threadIdx.x; i < t.k; i += NT) {
        int32_t c = t.indices[(size_t)row * t.k + i];
        if (c >= 0 && (uint32_t)c >= r.classes) { atomicOr(r.err, kErrList); c = -1; }
        idx[i] = c;
        val[i] = c >= 0 ? teacher_value(t, (size_t)row * t.k + i) : -INFINITY;
        sx[i] = c >= 0 ? to_f32(x[c]) : -INFINITY;
        if (c >= 0) {
            const uint32_t b = (uint32_t)c + V - sp.head;
            twice |= (atomicOr(&bits[b / 32], 1u << (b % 32)) >> (b % 32)) & 1u;
        }
    }
    twice = __syncthreads_or(twice);
    auto leads = [&](uint32_t i) {          // the first entry of its class
        if (twice)
            for (uint32_t o = 0; o < i; ++o)
                if (idx[o] == idx[i]) return false;
        return idx[i] >= 0;
    };
    const Stat outside_list = scan_row<T, NT, false>(sp, r.c_hi, r.c_lo, [&](Unit<T> &q, uint32_t bit, bool there) {
        const uint32_t mark = there ? bits[bit / 32] >> (bit % 32) & ((1u << V) - 1u) : 0;
        if (mark)
#pragma unroll
            for (int j = 0; j < (int)V; ++j) if (mark >> j & 1u) q.drop(j);
    });
    Stat a = merge<NT, false>(outside_list, red, r.c_hi);
    // the list: every warp goes through it for itself
    float top = -INFINITY, best = -INFINITY;
    for (uint32_t i = lane; i < t.k; i += 32) { top = fmaxf(top, val[i]); best = fmaxf(best, sx[i]); }
    top = warp_max(top);
    best = warp_max(best);
    const bool lost = __any_sync(0xffffffffu, [&] { bool n = false; for (uint32_t i = lane; i < t.k; i += 32) n |= idx[i] >= 0; return n; }());
    const float m = fmaxf(a.m, best);
    if ((!t.lse && (!lost || top == -INFINITY)) || (m == -INFINITY && a.s == 0.0f)) return nothing_to_learn();
    rescale(a, m, r.c_hi);
    const double shift = t.lse ? (double)t.lse[row] : (double)top * r.inv_t;
    auto raw_q = [&](uint32_t i) { return val[i] == -INFINITY ? 0.0f : expf((float)((double)val[i] * r.inv_t - shift)); };
    float listed = 0.0f;
    double mass = 0.0;
    for (uint32_t i = lane; i < t.k; i += 32) {
        const float d = sx[i] - m, e = ex2(fmaf(d, r.c_hi, d * r.c_lo));
        if (leads(i)) listed += e;
        mass += (double)raw_q(i);
    }
    listed = warp_sum(listed);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mass += __shfl_xor_sync(0xffffffffu, mass, o);
    const float s = a.s + listed, to_mass = t.lse ? 1.0f : (float)(1.0 / mass);
    double rest = t.lse ? 1.0 - mass : 0.0;
    if (rest <= kLeastTail) rest = 0.0;
    const float total = t.lse ? (float)(mass + rest) : 1.0f;
    if (threadIdx.x < 32) {
        const double log_s = log_sum(s), log_mass = t.lse ? 0.0 : log_wide((float)mass);
        double l = 0.0;
        for (uint32_t i = lane; i < t.k; i += 32) {
            const double log_q = (double)val[i] * r.inv_t - shift - log_mass;
            const float q = raw_q(i) * to_mass;
            if (q != 0.0f) l += (double)q * (log_q - (((double)sx[i] - (double)m) * r.inv_t - log_s));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if (rest > 0.0) l += rest * (log(rest) - (a.s > 0.0f ? log_wide(a.s) + kEx2Low - log_s : -INFINITY));
        if (first) t.loss[row] = (float)(t.factor * (double)w * l);
    }
    if (!r.d) return;
    // k = loss scale / T, the gradient's factor w T loss scale = w k T^2
    const float f = (float)((double)w * (double)r.k * t.factor);
    const float outside = a.s > 0.0f ? (float)((double)total / (double)s - rest / (double)a.s) : 0.0f;
    write_row<T, NT, false>(r, row, m, Coef{f * outside, 0.0f, 0.0f}, -1);
    __syncthreads();                        // the list's classes are written again, with their own values
    T *d = reinterpret_cast<T *>(r.d) + (size_t)row * r.cols;
    for (uint32_t i = threadIdx.x; i < t.k; i += NT) {
        if (!leads(i)) continue;
        float q = 0.0f;
        for (uint32_t o = i; o < (twice ? t.k : i + 1); ++o)
            if (idx[o] == idx[i]) q += raw_q(o) * to_mass;
        const float df = sx[i] - m, e = ex2(fmaf(df, r.c_hi, df * r.c_lo));
        d[idx[i]] = from_f32<T>(f * (total * e / s - q));
    }
}

} // namespace loss
} // namespace sk
