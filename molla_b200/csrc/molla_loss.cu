// Logprobs of given tokens, their gradient, and the losses over them (the formulas: include/molla_sample.h).
//
// With M = max x, c = log2(e)/T, t_j = c (x_j - M) and e_j = 2^t_j, S = sum e_j and W = sum e_j t_j:
//     logprob = (x_t - M)/T - ln S        entropy = ln S - W/(S c T)        p_j = e_j/S
// and for g = dL/dlogprob, h = dL/dentropy the gradient by logit j is
//     g [j = t]/T - e_j (A + H t_j)   with  H = h/(c T T S),  A = (g - h W/(S c T))/(T S)
// so a row needs three numbers (M, S, W) for everything. What multiplies e_j is counted in its exponent, not in x_j - M: t_j can be held at a
// number as small as -160, where e_j is 0 whatever the temperature, so that no product of a masked logit leaves 32 bits. Differences from M are exact for the logits that matter. Whatever
// rounding e_j has is the same in S, in W and in the gradient, where it cancels to first order; what it has in the mean is known (EX2_LOW, rounding_of), kept
// beside S and counted in ln S alone.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/molla_sample.h"
#include "molla_device.cuh"
#include "molla_loss.h"

using namespace molla;

#ifdef MOLLA_SAMPLE_TESTING
#define LOSS_KNOB(a, bit) (((a).knobs & (bit)) != 0)
#else
#define LOSS_KNOB(a, bit) false
#endif

namespace {

constexpr double LOG2E_64 = 1.44269504088896340736;
constexpr float LOG2E = (float)LOG2E_64, LOG2E_LEFT = (float)(LOG2E_64 - (double)LOG2E);
constexpr float DEEP = -160.0f;   // where an exponent is held as a factor: 2^t is 0 below -126 (-150 with subnormals), and 0 * t stays 0 for logits of -inf
constexpr unsigned int ROW_ERRORS = MOLLA_ROW_BAD_TOKEN | MOLLA_ROW_EMPTY | MOLLA_ROW_INVALID_CONFIG | MOLLA_ROW_LOAD_TIMEOUT;

// The later kernels of a call are launched while the one before runs, and wait here until it has ended: what is saved is their launch. (Nothing lets them begin
// any earlier.)
__device__ __forceinline__ void wait_for_launch_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <class T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(float v) { return v; }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }

// ---- a row's scalars ------------------------------------------------------------------------------

// A row's inputs; a lane fetches a row's, 32 rows ahead.
struct RowIn {
    int token;
    float T, per_T, old, advantage, weight, ref, xt;   // temperature and its inverse; the policy loss's; the token's logit
    unsigned int status; // why the row cannot be answered, before it is read
    bool idle;           // nothing to answer: no token, or no weight
};

__device__ __forceinline__ RowIn row_in(const LossArgs &a, int r) {
    RowIn in;
    in.token = a.tokens[r];
    in.T = a.temperature ? a.temperature[r] : 1.0f;
    in.per_T = 1.0f / in.T;
    in.weight = a.weight ? a.weight[r] : 1.0f;
    in.old = in.advantage = in.ref = in.xt = 0.0f;
    in.idle = in.token == -1 || in.weight == 0.0f;
    in.status = 0;
    if (!in.idle) {
        if (in.token < 0 || in.token >= a.V) in.status |= MOLLA_ROW_BAD_TOKEN;
        const float c = LOG2E / in.T;
        if (!(in.T > 0.0f) || !(c > 0.0f) || isinf(c)) in.status |= MOLLA_ROW_INVALID_CONFIG;
    }
    return in;
}

// 1/(c T): ln 2, but for what rounding left out of c.
__device__ __forceinline__ float nats_of(float c, float T) { return __frcp_rn(__fmul_rn(c, T)); }

// The gradient's three numbers: add at the token, and A and H of the formula; `mean` is W/(S c T). Finite derivatives over a temperature near
// the least one would leave 32 bits: the three are held at what a probability of 0 still makes 0 of (|H| 160 + |A| is below the largest float).
struct RowGrad { float token, A, H; };

__device__ __forceinline__ bool ordinary(float x) { return fabsf(x) < 3e38f; }
__device__ __forceinline__ float held_at(float x, float most) { return fabsf(x) > most ? copysignf(most, x) : x; }   // (NaN stays)

__device__ __forceinline__ RowGrad row_grad(float g, float h, float per_T, float per_S, float mean, float nats) {
    RowGrad o;
    const float inv = per_T * per_S;
    o.token = g * per_T;
    o.A = __fmaf_rn(-h, mean, g) * inv;
    o.H = h * inv * nats;
    if (ordinary(g) && ordinary(h)) { o.token = held_at(o.token, 1.6e38f); o.A = held_at(o.A, 1.6e38f); o.H = held_at(o.H, 1e36f); }
    return o;
}

// A value in two floats, the second below the first's last bit.
struct Two { float hi, lo; };
__device__ __forceinline__ Two two_sum(float a, float b) {
    const float s = __fadd_rn(a, b), bb = __fsub_rn(s, a);
    return Two{s, __fadd_rn(__fsub_rn(a, __fsub_rn(s, bb)), __fsub_rn(b, bb))};
}

constexpr float LN2 = 0.693147180559945309f;
constexpr float LN2_SHORT = 0.693145751953125f, LN2_REST = (float)(0.693147180559945309 - 0.693145751953125);   // 17 bits, times a small integer exact

// ln S, S > 0: the power of two apart; what is left lies within a factor of the square root of two of one, its logarithm is below 0.35 and
// good to 3e-8.
__device__ __forceinline__ Two ln_of(float S) {
    if (!(S > 0.0f) || !ordinary(S)) return Two{S == 0.0f ? -INFINITY : S, 0.0f};   // (NaN stays)
    const int k = (__float_as_int(S) - 0x3f3504f3) >> 23;
    const float y = log1pf(__fsub_rn(__int_as_float(__float_as_int(S) - (k << 23)), 1.0f)), n = (float)k;
    return two_sum(n * LN2_SHORT, __fmaf_rn(n, LN2_REST, y));
}

// exp(q) - 1 - q, for small q from its series, which the difference would lose, and exp(q) - 1
__device__ __forceinline__ float exp_less_line(float q, float &less_one) {
    if (fabsf(q) > 0.5f) {
        less_one = expm1f(q);
        return isinf(less_one) ? less_one : __fsub_rn(less_one, q);
    }
    float p = 1.0f / 3628800.0f;
    p = __fmaf_rn(p, q, 1.0f / 362880.0f); p = __fmaf_rn(p, q, 1.0f / 40320.0f); p = __fmaf_rn(p, q, 1.0f / 5040.0f);
    p = __fmaf_rn(p, q, 1.0f / 720.0f); p = __fmaf_rn(p, q, 1.0f / 120.0f); p = __fmaf_rn(p, q, 1.0f / 24.0f);
    p = __fmaf_rn(p, q, 1.0f / 6.0f); p = __fmaf_rn(p, q, 0.5f);
    p = p * q * q;
    less_one = p + q;
    return p;
}

// What a row answers once its maximum M, sum S and, where entropies are wanted, W are known: first what its gradient
// waits for, all of it in 32 bits (conversions to 64 run where the exponentials do, behind theirs: with 64 bits, logarithm, exponential and
// divisions a row's blocks waited 6200 cycles, with conversions alone 2400), then the rest.
struct Answer { unsigned int status; Two l, lnS; float mean, ratio, kl; bool held; };

template <bool ENT>
__device__ __forceinline__ RowGrad row_answer(const LossArgs &a, const RowIn &in, float M, Two S, float W, float c, Answer &o) {
    o.status = in.status | (M == -INFINITY && S.hi == 0.0f && !in.status ? MOLLA_ROW_EMPTY : 0u);
    const float per_S = __frcp_rn(S.hi);
    o.lnS = ln_of(S.hi);
    o.lnS.lo = __fmaf_rn(S.lo, per_S, o.lnS.lo);
    const float nats = in.per_T, nats_lo = __fmaf_rn(-in.T, nats, 1.0f) * nats, dx = __fsub_rn(in.xt, M);
    const float per_cT = ENT ? nats_of(c, in.T) : 0.0f;
    o.mean = ENT ? W * per_S * per_cT : 0.0f;
    const float p = dx * nats;
    if (ordinary(p) && ordinary(o.lnS.hi)) {
        const Two d = two_sum(in.xt, -M);
        const float p_lo = __fmaf_rn(dx, nats, -p) + __fmaf_rn(dx, nats_lo, d.lo * nats);
        const Two s = two_sum(p, -o.lnS.hi);
        o.l = two_sum(s.hi, s.lo + (p_lo - o.lnS.lo));
    } else {
        o.l = Two{p - o.lnS.hi, 0.0f};
    }
    o.ratio = o.kl = 0.0f;
    o.held = false;
    if (!a.row_loss) return RowGrad{0.0f, 0.0f, 0.0f};
    o.ratio = expf((o.l.hi - in.old) + o.l.lo);
    o.held = (in.advantage > 0.0f && o.ratio > 1.0f + a.clip_high) || (in.advantage < 0.0f && o.ratio < 1.0f - a.clip_low);   // (not a NaN)
    float g = o.held ? 0.0f : -(o.ratio * in.advantage);
    if (a.ref_logprob) {
        float less_one;
        o.kl = exp_less_line((in.ref - o.l.hi) - o.l.lo, less_one);
        if (a.kl_coef != 0.0f) g = __fmaf_rn(-a.kl_coef, less_one, g);
    }
    const float by = in.weight * a.scale * a.grad_scale;
    return o.status ? RowGrad{0.0f, 0.0f, 0.0f} : row_grad(g * by, ENT ? -a.entropy_coef * by : 0.0f, in.per_T, per_S, o.mean, per_cT);
}

__device__ __forceinline__ void row_write(const LossArgs &a, int r, const RowIn &in, float M, float S, const Answer &o) {
    const unsigned int status = o.status;
    const double H = ((double)o.lnS.hi + (double)o.lnS.lo) - (double)o.mean;
    a.status[r] = status;
    a.logprob[r] = status ? NAN : o.l.hi;
    if (a.logprob_lo) a.logprob_lo[r] = status ? 0.0f : o.l.lo;
    if (a.entropy) a.entropy[r] = status ? NAN : (float)H;
    if (a.depth) a.depth[r] = status ? NAN : 0.0f - o.mean;
    if (a.stats) { a.stats[2 * r] = status ? NAN : M; a.stats[2 * r + 1] = status ? 0.0f : S; }
    if (!a.row_loss) return;
    const double bound = o.held ? (in.advantage > 0.0f ? 1.0 + (double)a.clip_high : 1.0 - (double)a.clip_low) : (double)o.ratio;
    double term = -bound * (double)in.advantage;
    if (a.kl) a.kl[r] = status ? NAN : o.kl;
    if (a.kl_coef != 0.0f) term += (double)a.kl_coef * (double)o.kl;
    if (a.entropy_coef != 0.0f) term -= (double)a.entropy_coef * H;
    a.row_loss[r] = status ? NAN : (float)((double)in.weight * term);
    if (a.clipped) a.clipped[r] = !status && o.held;
}

// a row that cannot be answered, and is not read
__device__ __forceinline__ void row_refused(const LossArgs &a, int r, const RowIn &in) {
    Answer o = {};
    o.status = in.status;
    row_write(a, r, in, 0.0f, 1.0f, o);
}

__device__ void row_idle(const LossArgs &a, int r) {
    a.status[r] = 0;
    a.logprob[r] = 0.0f;
    if (a.logprob_lo) a.logprob_lo[r] = 0.0f;
    if (a.entropy) a.entropy[r] = 0.0f;
    if (a.depth) a.depth[r] = 0.0f;
    if (a.stats) { a.stats[2 * r] = 0.0f; a.stats[2 * r + 1] = 1.0f; }
    if (a.row_loss) a.row_loss[r] = 0.0f;
    if (a.kl) a.kl[r] = 0.0f;
    if (a.clipped) a.clipped[r] = 0;
}

// ---- a 16-byte chunk of logits -----------------------------------------------------------------------
// (Sums of pairs in packed 64-bit registers were tried: half of the additions, and three moves an element to pack them.)

__device__ __forceinline__ unsigned int word(const uint4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ void set_word(uint4 &v, int i, unsigned int w) { if (i == 0) v.x = w; else if (i == 1) v.y = w; else if (i == 2) v.z = w; else v.w = w; }
template <class V> __device__ __forceinline__ V as(unsigned int w) { return *reinterpret_cast<const V *>(&w); }
template <class V> __device__ __forceinline__ unsigned int bits(const V &v) { return *reinterpret_cast<const unsigned int *>(&v); }

// max: the larger of words of two chunks; top: the largest of a word; get and put: an element
template <class T> struct Chunk;
template <> struct Chunk<float> {
    static constexpr int N = 4;
    __device__ static __forceinline__ unsigned int max(unsigned int a, unsigned int b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }
    __device__ static __forceinline__ float top(unsigned int w) { return __uint_as_float(w); }
    __device__ static __forceinline__ void get(const uint4 &v, float (&x)[N]) {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = __uint_as_float(word(v, i));
    }
    __device__ static __forceinline__ uint4 put(const float (&x)[N]) {
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    }
    static constexpr unsigned int LOWEST = 0xff800000u;   // -inf
};
template <> struct Chunk<__nv_bfloat16> {
    static constexpr int N = 8;
    __device__ static __forceinline__ unsigned int max(unsigned int a, unsigned int b) { return bits(__hmax2(as<__nv_bfloat162>(a), as<__nv_bfloat162>(b))); }
    __device__ static __forceinline__ float top(unsigned int w) { return fmaxf(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
    __device__ static __forceinline__ void get(const uint4 &v, float (&x)[N]) {
#pragma unroll
        for (int i = 0; i < 4; i++) { const unsigned int w = word(v, i); x[2 * i] = __uint_as_float(w << 16); x[2 * i + 1] = __uint_as_float(w & 0xffff0000u); }
    }
    __device__ static __forceinline__ uint4 put(const float (&x)[N]) {
        uint4 o;
#pragma unroll
        for (int i = 0; i < 4; i++) set_word(o, i, bits(__floats2bfloat162_rn(x[2 * i], x[2 * i + 1])));
        return o;
    }
    static constexpr unsigned int LOWEST = 0xff80ff80u;
};
template <> struct Chunk<__half> {
    static constexpr int N = 8;
    __device__ static __forceinline__ unsigned int max(unsigned int a, unsigned int b) { return bits(__hmax2(as<__half2>(a), as<__half2>(b))); }
    __device__ static __forceinline__ float top(unsigned int w) { const float2 f = __half22float2(as<__half2>(w)); return fmaxf(f.x, f.y); }
    __device__ static __forceinline__ void get(const uint4 &v, float (&x)[N]) {
#pragma unroll
        for (int i = 0; i < 4; i++) { const float2 f = __half22float2(as<__half2>(word(v, i))); x[2 * i] = f.x; x[2 * i + 1] = f.y; }
    }
    __device__ static __forceinline__ uint4 put(const float (&x)[N]) {
        uint4 o;
#pragma unroll
        for (int i = 0; i < 4; i++) set_word(o, i, bits(__floats2half2_rn(x[2 * i], x[2 * i + 1])));
        return o;
    }
    static constexpr unsigned int LOWEST = 0xfc00fc00u;
};

// ---- rows by clusters, a unit of 4096 bytes by a warp ---------------------------------------------------

constexpr int UB = 4096;                    // a unit's bytes: eight chunks a lane
constexpr int KU = UB / 512;
template <class T> constexpr int UNIT = UB / (int)sizeof(T);   // and logits
constexpr int MAX_WARPS = 16;      // with the one that answers
constexpr int WAIT_TRIES = 1 << 22;   // of a bounded wait
__device__ __forceinline__ int tries_of(const LossArgs &a) { return LOSS_KNOB(a, 256 | 512 | 1024) ? 1 << 14 : WAIT_TRIES; }   // (testing build: waits that are meant to run out)

// How a launch lays its rows out: C blocks of W warps a row, R units of shared memory a warp, `rows_at_once` rows
// in flight. Nothing in a row's results depends on it: a unit is always one warp's, in the same order of additions, and
// the units are put together in theirs.
struct Layout { int C, W, R, rows_at_once, table; bool resident, ahead; };   // table: places for a row's sums

// The row's logits in memory: what lies before the first 16-byte boundary and behind the last (the edge, at most 14 logits), and
// whole 16-byte chunks in between, in units.
template <class T> struct RowSpan {
    const T *x; int head, units, full, tail; int bytes;
    __device__ __forceinline__ RowSpan(const T *row, int V) {
        const int off = (int)((uintptr_t)row & 15);
        head = off ? (16 - off) / (int)sizeof(T) : 0;
        if (head > V) head = V;
        x = row + head;
        bytes = ((V - head) * (int)sizeof(T)) & ~15;
        tail = V - head - bytes / (int)sizeof(T);
        units = (bytes + UB - 1) / UB;
        full = bytes / UB;
    }
    __device__ __forceinline__ int last_chunks() const { return (bytes - full * UB) >> 4; }   // of the unit that is not full
    __device__ __forceinline__ bool edge() const { return head + tail > 0; }
    // the edge's logit of a lane: the first lanes have the head, those from 16 on the tail; -1 if it has none
    __device__ __forceinline__ int edge_at(int lane) const {
        if (lane < head) return lane - head;
        const int t = lane - 16;
        return t >= 0 && t < tail ? bytes / (int)sizeof(T) + t : INT32_MIN;
    }
};

__device__ __forceinline__ float warp_max(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) v += __shfl_xor_sync(0xffffffffu, v, i);
    return v;
}
// 2^t for t <= 0 without ex2's bias: the nearest integer apart, the Taylor series of 2^f = e^(f ln 2) for the rest (|f| <= 1/2; the first term
// left out is below 6e-9 of the sum).
__device__ __forceinline__ float exp2_series(float t) {
    const float n = rintf(t < -127.0f ? -127.0f : t), f = __fmul_rn(t < -127.0f ? 0.0f : __fsub_rn(t, n), 0.693147180559945f);
    float p = 1.0f / 5040.0f;
    p = __fmaf_rn(p, f, 1.0f / 720.0f); p = __fmaf_rn(p, f, 1.0f / 120.0f); p = __fmaf_rn(p, f, 1.0f / 24.0f);
    p = __fmaf_rn(p, f, 1.0f / 6.0f); p = __fmaf_rn(p, f, 0.5f); p = __fmaf_rn(p, f, 1.0f); p = __fmaf_rn(p, f, 1.0f);
    return p * __int_as_float(((int)n + 127) << 23);   // 0 from 2^-127 down; NaN stays in p
}

// ex2.approx is low by 5.2e-8 in the mean, alike in every binade (4 million arguments from -32 to 0; by 2e-8 to 7e-8 in a sixteenth of one, which rows
// whose exponents all lie in such a part keep the difference of), which a sum of many terms
// keeps: uncorrected, the log ratio of a sequence of 200 rows was off by 1e-5. Its value at 0 is exact: of a unit's sum one term, its
// largest, is left out of the correction, and a sum that is a whole number (logits that are all alike, but for those of -inf) is not corrected at all. Where
// a unit's largest logit comes many times among others that count, its sum is high by up to 5.2e-8 of them.
constexpr float EX2_LOW = 5.2e-8f;

// 16 bytes of shared memory by their address there (pointers into it cost 64-bit arithmetic)
__device__ __forceinline__ uint4 lds16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
template <class T> __device__ __forceinline__ float lds_element(uint32_t at);
template <> __device__ __forceinline__ float lds_element<float>(uint32_t at) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ unsigned short lds2(uint32_t at) {
    unsigned short v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at) : "memory");
    return v;
}
template <> __device__ __forceinline__ float lds_element<__nv_bfloat16>(uint32_t at) { return __uint_as_float((unsigned int)lds2(at) << 16); }
template <> __device__ __forceinline__ float lds_element<__half>(uint32_t at) { return __half2float(__ushort_as_half(lds2(at))); }

// maximum, sum (in two floats) and weighted sum of a unit; where a wait ran out s_lo is LATE
struct Stat { float m, s, w, s_lo; };
constexpr float LATE = -1.0f;

// A lane's sum of values from 0 to 16, up to 64 altogether, without loss: 128 and what is above it in one float, whose last bit is 2^-16, and what each
// addition to it rounds off, up to 2^-17, in another.
struct Sum {
    float high = 128.0f, low = 0.0f;
    __device__ __forceinline__ void add(float v) {
        const float h = __fadd_rn(high, v);
        low = low + __fsub_rn(v, __fsub_rn(h, high));
        high = h;
    }
};
// Those of a warp: in integers of 2^-16 and, of what is left (up to four times 2^-17), of 2^-36 (the bits that an addition to 1.5 2^-13 ends in), which add
// up exactly in whatever order. (A tree of 32-bit sums loses what is below half a step of the largest value, always downwards: 5e-8 of a unit,
// which the log ratio of a long sequence adds up.) A NaN stays.
__device__ __forceinline__ Two warp_sum_exact(const Sum &t) {
    const float low = __fadd_rn(t.low, 1.5f / 8192.0f);
    const int A = __reduce_add_sync(0xffffffffu, __float_as_int(t.high) - __float_as_int(128.0f));
    const int B = __reduce_add_sync(0xffffffffu, __float_as_int(low) - __float_as_int(1.5f / 8192.0f));
    const Two s = two_sum((float)(A >> 8) * (1.0f / 256.0f), __fmaf_rn((float)B, 1.0f / 68719476736.0f, (float)(A & 255) * (1.0f / 65536.0f)));
    return __any_sync(0xffffffffu, !(t.high < 256.0f)) ? Two{NAN, 0.0f} : s;
}
__device__ __forceinline__ void put_sum(Stat &o, const Sum &t) {
    const Two s = warp_sum_exact(t);
    o.s = s.hi;
    o.s_lo = s.lo;
}

// A unit's, from shared memory twice: once for its maximum, then for the sums (four of either a lane). PART: how many sums of a unit that is not full
// are unrolled: as many as of a full one (8288 x 128256 bf16 392 to 383 us) but with a gradient, whose registers would spill (1 % slower).
template <class T, bool ENT, bool FULL, int PART>
__device__ __forceinline__ Stat unit_stat(uint32_t slot, int chunks, float c) {
    const int lane = threadIdx.x & 31;
    constexpr unsigned int low = Chunk<T>::LOWEST;
    uint4 most = make_uint4(low, low, low, low);
#pragma unroll(FULL ? KU / 2 : PART)
    for (int k = 0; k < KU; k++)
        if (FULL || k * 32 + lane < chunks) {
            const uint4 v = lds16(slot + k * 512 + lane * 16);
            most = make_uint4(Chunk<T>::max(most.x, v.x), Chunk<T>::max(most.y, v.y), Chunk<T>::max(most.z, v.z), Chunk<T>::max(most.w, v.w));
        }
    Stat o;
    o.m = warp_max(Chunk<T>::top(Chunk<T>::max(Chunk<T>::max(most.x, most.y), Chunk<T>::max(most.z, most.w))));
    const float m = o.m == -INFINITY ? 0.0f : o.m;   // nothing but -inf (and NaN): sums of 0 (and NaN)
    // Sixteen logits at a time are added up in 32 bits, their sums with what that rounds off: where one logit has most of the sum, every addition to
    // it would lose up to half a step, and what is smaller than that altogether (the logprobs of 128256 bf16 logits were low by 1.5e-8 on the
    // average, with a standard error of 3.8e-8; so they are right to 1e-9 on the average, with 2.7e-8, for 1 % of the time).
    constexpr int CHUNKS = 16 / Chunk<T>::N;
    Sum sum;
    float w[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll(FULL ? KU / 2 / CHUNKS : PART)
    for (int k0 = 0; k0 < KU; k0 += CHUNKS) {
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = k0; k < k0 + CHUNKS; k++)
            if (FULL || k * 32 + lane < chunks) {
                float x[Chunk<T>::N];
                Chunk<T>::get(lds16(slot + k * 512 + lane * 16), x);
#pragma unroll
                for (int i = 0; i < Chunk<T>::N; i++) {
                    const float t = __fsub_rn(x[i], m) * c, e = ex2(t);
                    s[i & 3] = k == k0 && i < 4 ? e : s[i & 3] + e;
                    if (ENT) w[i & 3] = __fmaf_rn(e, fmaxf(t, DEEP), w[i & 3]);
                }
            }
        sum.add((s[0] + s[1]) + (s[2] + s[3]));
    }
    put_sum(o, sum);
    o.w = 0.0f;
    if (ENT) o.w = warp_sum((w[0] + w[1]) + (w[2] + w[3]));
    return o;
}

// The edge's, a logit a lane (-inf where there is none).
template <bool ENT> __device__ __forceinline__ Stat edge_stat(float x, float c) {
    Stat o;
    o.m = warp_max(x);
    const float m = o.m == -INFINITY ? 0.0f : o.m, t = __fsub_rn(x, m) * c, e = ex2(t);
    Sum sum;
    sum.add(e);
    put_sum(o, sum);
    o.w = ENT ? warp_sum(e * fmaxf(t, DEEP)) : 0.0f;
    return o;
}

// A number n of logits: ln n, and -3/4 of its square's inverse.
struct Count { float ln, curve; };
__device__ __forceinline__ Count count_of(int n) {
    const float ln = __logf((float)n);
    return Count{ln, n > 1 ? -__fdividef(0.75f, ln * ln) : 0.0f};
}
// ln s to 0.03 for s from 1 to 4096: its bits are its logarithm, but for a curve. (None of this runs where the exponentials do.)
__device__ __forceinline__ float about_ln(float s) {
    const float bits = __int_as_float(0x4b000000 | (__float_as_int(s) >> 8));
    return __fmaf_rn(__fsub_rn(bits, 8388608.0f + 0x3f8000), LN2 / 32768.0f, 0.03f);
}
// What a unit's sum s of n logits lacks: the part EX2_LOW of all but its largest term, and `off` (rounding_of) of sum e (max - z). That is about
// s - 1 times how far in nats the others lie below the largest. No distribution has them further than ln(n/s) on the average: nearly that where they are much
// alike, less the more of s belongs to a few. With 1 - 3/4 (ln(n/s) / ln n)^2 of it normal tails of any width are met to 0.2, exponential
// ones to 0.7, a unit that is half masked to 0.6. Logits that are all alike have a whole number for their sum, which lacks nothing.
__device__ __forceinline__ float lacks(const Stat &o, const Count &n, float off) {
    const float far = n.ln - about_ln(o.s), whole = __fsub_rn(__fadd_rn(o.s, 12582912.0f), 12582912.0f);
    const float by = __fmaf_rn(off * far, __fmaf_rn(n.curve * far, far, 1.0f), EX2_LOW);
    return whole == o.s && o.s_lo == 0.0f ? 0.0f : (o.s - 1.0f) * by;
}

// c is log2(e)/T rounded: off by this part of it, up to 2^-24 (1.3e-8 at T = 1, 5.8e-8 at 1.1).
__device__ __forceinline__ float rounding_of(float c, float T) { return (__fmaf_rn(c, T, -LOG2E) - LOG2E_LEFT) * LN2; }

// All units of a row: a warp, the units in turn over the lanes, then a tree; S in two floats: the sum of what has been added up, and what that lost or lacks.
// What is `off` in c (rounding_of) puts ln S off by that times how far in nats the logits are below M on the average of the distribution: of a logprob an
// error of 4e-8 at T = 1, always to the same side.
template <class T, bool ENT>
__device__ __forceinline__ void row_stat(const Stat *st, const RowSpan<T> &span, const Count &of_last, const Count &of_edge, float c, float off, float &M,
                                         Two &S, float &W, bool &late) {
    const int n = span.units + (span.edge() ? 1 : 0);
    constexpr float LN_UNIT = sizeof(T) == 4 ? 6.93147181f : 7.62461899f;   // ln 1024, ln 2048
    const auto count = [&](int u) { return u < span.full ? Count{LN_UNIT, -0.75f / (LN_UNIT * LN_UNIT)} : u < span.units ? of_last : of_edge; };
    const int lane = threadIdx.x & 31;
    constexpr int HELD = 3;   // units a lane that stay in registers
    Stat v[HELD];
    float m = -INFINITY;
    bool l = false;
#pragma unroll
    for (int k = 0; k < HELD; k++) {
        v[k] = Stat{-INFINITY, 0.0f, 0.0f, 0.0f};
        if (k > 0 && k * 32 >= n) continue;
        if (k * 32 + lane < n) v[k] = st[k * 32 + lane];
        m = fmaxf(m, v[k].m);
        l |= v[k].s_lo == LATE;
    }
    for (int u = HELD * 32 + lane; u < n; u += 32) { m = fmaxf(m, st[u].m); l |= st[u].s_lo == LATE; }
    M = warp_max(m);
    late = __any_sync(0xffffffffu, l);
    S = Two{0.0f, 0.0f};
    W = 0.0f;
    const auto add = [&](const Stat &o, int u) {
        const float d = o.m == -INFINITY ? 0.0f : __fsub_rn(o.m, M);   // (a unit of -inf: sums of 0, or NaN)
        const float t = d * c, f = exp2_series(t), p = f * o.s, held = fmaxf(t, DEEP);   // (a NaN stays in f)
        const Two s = two_sum(S.hi, p);
        const float left = __fmaf_rn(off * LN2 * held, -o.s, o.s_lo + lacks(o, count(u), off));
        S = Two{s.hi, S.lo + (s.lo + __fmaf_rn(f, left, __fmaf_rn(f, o.s, -p)))};
        if (ENT) W = __fmaf_rn(f, __fmaf_rn(held, o.s, o.w), W);
    };
#pragma unroll
    for (int k = 0; k < HELD; k++)
        if (k == 0 || k * 32 < n) add(v[k], k * 32 + lane);
    for (int u = HELD * 32 + lane; u < n; u += 32) add(st[u], u);
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) {
        const float hi = __shfl_xor_sync(0xffffffffu, S.hi, i), lo = __shfl_xor_sync(0xffffffffu, S.lo, i);
        const Two s = two_sum(S.hi, hi);
        S = Two{s.hi, (S.lo + lo) + s.lo};
    }
    if (ENT) W = warp_sum(W);
}

template <class T, bool ENT>
__device__ __forceinline__ float gradient_of(float x, float M, float c, float A, float H) {
    const float t = __fsub_rn(x, M) * c, e = ex2(t);
    return ENT ? -(e * __fmaf_rn(H, fmaxf(t, DEEP), A)) : -(e * A);
}

// One unit's gradient: `to` is where its first logit's goes.
template <class T, bool ENT, bool FULL>
__device__ __forceinline__ void unit_gradient(uint32_t slot, int chunks, T *to, bool wide, float M, float c, float A, float H) {
    constexpr int N = Chunk<T>::N;
    const int lane = threadIdx.x & 31;
#pragma unroll(FULL ? KU / 2 : 1)
    for (int k = 0; k < KU; k++)
        if (FULL || k * 32 + lane < chunks) {
            float x[N];
            Chunk<T>::get(lds16(slot + k * 512 + lane * 16), x);
#pragma unroll
            for (int i = 0; i < N; i++) x[i] = gradient_of<T, ENT>(x[i], M, c, A, H);
            const uint4 o = Chunk<T>::put(x);
            if (wide) {
                __stcs(reinterpret_cast<uint4 *>(to) + k * 32 + lane, o);
            } else {
                const T *e = reinterpret_cast<const T *>(&o);
#pragma unroll
                for (int i = 0; i < N; i++) to[(k * 32 + lane) * N + i] = e[i];
            }
        }
}

__device__ __forceinline__ uint4 zero4() { return make_uint4(0u, 0u, 0u, 0u); }

// A row of zeros, by the warps of its blocks.
template <class T> __device__ void zero_row(T *out, int V, int warp, int warps) {
    const int lane = threadIdx.x & 31;
    const int off = (int)((uintptr_t)out & 15), head = min(off ? (16 - off) / (int)sizeof(T) : 0, V);
    const int chunks = (V - head) / Chunk<T>::N, tail = V - head - chunks * Chunk<T>::N;
    uint4 *to = reinterpret_cast<uint4 *>(out + head);
    for (int k = warp * 32 + lane; k < chunks; k += warps * 32) __stcs(to + k, zero4());
    if (warp == 0) {
        if (lane < head) out[lane] = from_f32<T>(0.0f);
        if (lane < tail) out[head + chunks * Chunk<T>::N + lane] = from_f32<T>(0.0f);
    }
}

// What a row's gradient is made of, where it is given (the backward pass).
struct RowShare { float M, c, A, H, token_add; int token; int zero, pad; };
__device__ __forceinline__ RowShare row_given(const LossArgs &a, int r) {
    RowShare o = {};
    const float T = a.temperature ? a.temperature[r] : 1.0f, S = a.in_stats[2 * r + 1];
    const float g = a.g_logprob[r], h = a.g_entropy ? a.g_entropy[r] : 0.0f;
    o.token = a.tokens[r];
    o.M = a.in_stats[2 * r];
    o.c = LOG2E / T;
    float mean = 0.0f;
    if (h != 0.0f && a.in_depth) {
        mean = -a.in_depth[r];
    } else if (h != 0.0f) {   // (what rounding the entropy left out comes with it)
        const Two lnS = ln_of(S);
        mean = (lnS.hi - a.in_entropy[r]) + lnS.lo;
    }
    const RowGrad q = row_grad(g, h, 1.0f / T, __frcp_rn(S), mean, nats_of(o.c, T));
    o.A = q.A; o.H = q.H; o.token_add = q.token;
    return o;
}

// Whether a row's logits are read at all.
template <bool STATS> __device__ __forceinline__ bool row_read(const LossArgs &a, int r) {
    if (STATS) {
        const RowIn in = row_in(a, r);
        return !in.idle && !in.status;
    }
    const int token = a.tokens[r];
    return !(token < 0 || token >= a.V || (a.g_logprob[r] == 0.0f && !(a.g_entropy && a.g_entropy[r] != 0.0f)) || a.in_stats[2 * r + 1] == 0.0f);
}

// A bulk copy of global memory to shared, with what L2 is told about the lines: nothing, that they will be read once more before long, or
// that this is the last time.
enum Lines { ANY, KEEP, LAST };
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar, Lines lines) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
    if (lines == ANY) {
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                     : "memory");
    } else {
        uint64_t policy;
        if (lines == KEEP) asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(policy));
        else asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(dst), "l"(src),
                     "r"(bytes), "r"(bar), "l"(policy)
                     : "memory");
    }
}

// A bounded wait for a phase of a barrier to end (all lanes alike). A try lets the warp sleep for up to a microsecond.
__device__ __forceinline__ bool try_for(uint32_t bar, int parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 1000;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return __all_sync(0xffffffffu, ok != 0);
}
__device__ __forceinline__ bool wait_for(uint32_t bar, int parity, int tries) {
    if (try_for(bar, parity)) return true;
    for (int i = 0; i < tries; i++)
        if (try_for(bar, parity)) return true;
    return false;
}
__device__ __forceinline__ bool wait_for(uint64_t *bar, int parity, int tries) { return wait_for(smem_u32(bar), parity, tries); }

// A warp's units of shared memory, filled in the order in which it will want them, row after row.
template <class T, bool STATS, bool GRAD> struct Feed {
    const LossArgs &a; const Layout &L;
    uint32_t slots, bars;      // in shared memory
    int warp, stride;          // of the row's warps; bytes from one of its units to the next
    int row0, step;            // this cluster's rows are row0, row0 + step, ...
    int i, base; unsigned int mask;   // the row that is being fetched, and which of 32 rows are read
    int row;                   // -1 before the first
    const char *src; int left; // the next unit, and the bytes from there to its row's end
    bool second;               // the row comes again, for its gradient
    int ahead;                 // units fetched or on their way, not given back
    int put, get, parity;      // slots
    bool more, late;
    int owed, owed_slot, owed_parity;   // copies on their way when a wait ran out

    __device__ __forceinline__ Feed(const LossArgs &a_, const Layout &L_, uint32_t s, uint32_t b, int w, int ws, int r0, int st)
        : a(a_), L(L_), slots(s), bars(b), warp(w), stride(ws * UB), row0(r0), step(st), i(-1), base(-32), mask(0), row(-1), src(nullptr), left(0), second(true),
          ahead(0), put(0), get(0), parity(0), more(true), late(false), owed(0) {
        next();
        while (more && ahead < L.R) fetch();
    }
    __device__ __forceinline__ bool row_ok(int k) const { return (long long)row0 + (long long)k * step < a.B; }
    // A gradient that follows another pass over the logits takes the rows from the last to the first: those are still in L2.
    __device__ __forceinline__ int row_of(int k) const { return !STATS && a.follows ? a.B - 1 - (row0 + k * step) : row0 + k * step; }
    __device__ __forceinline__ void start(int r) {
        const RowSpan<T> span((const T *)a.logits + (long long)r * a.row_stride, a.V);
        src = (const char *)span.x + warp * UB;
        left = span.bytes - warp * UB;
    }
    // The next row that is read, or -1.
    __device__ int next_row() {
        for (;;) {
            i++;
            if (!row_ok(i)) return -1;
            if (i - base >= 32) {
                base = i;
                const int lane = threadIdx.x & 31;
                mask = __ballot_sync(0xffffffffu, row_ok(i + lane) && row_read<STATS>(a, row_of(i + lane)));
            }
            if (mask >> (i - base) & 1) return row_of(i);
        }
    }
    // From the end of one row's units to the first of another, or, where units do not stay (see rows_kernel), of the same row for its gradient.
    __device__ void next() {
        do {
            second = STATS && GRAD && !L.resident && !second;
            if (!second) row = next_row();
            if (row < 0) { more = false; return; }
            start(row);
        } while (left <= 0);
    }
    // one more unit, where there is room
    __device__ __forceinline__ void fetch() {
        if (!more || ahead >= L.R) return;
        if ((threadIdx.x & 31) == 0) {
            const uint32_t to = slots + put * UB, bar = bars + put * 8, bytes = (uint32_t)min(left, UB);
            if (LOSS_KNOB(a, second || a.follows ? 1024 : 512) && warp == 0 && row == a.B / 2) {   // (testing build: a copy that never comes)
            } else if (!(STATS && GRAD) || L.resident) bulk_copy(to, src, bytes, bar, ANY);
            else if (second) bulk_copy(to, src, bytes, bar, LAST);
            else bulk_copy(to, src, bytes, bar, KEEP);
        }
        ahead++;
        put = put + 1 == L.R ? 0 : put + 1;
        src += stride;
        left -= stride;
        if (left <= 0) next();
    }
    // the k-th unit from the oldest that has not been given back: when it has arrived, or as it was
    __device__ __forceinline__ uint32_t wait(int k) {
        int s = get + k, p = parity;
        if (s >= L.R) { s -= L.R; p ^= 1; }
        if (!late && !wait_for(bars + s * 8, p, tries_of(a))) lose(k);
        return slots + s * UB;
    }
    __device__ __forceinline__ uint32_t oldest() const { return slots + get * UB; }
    __device__ __forceinline__ void give_back() {
        __syncwarp();
        ahead--;
        if (++get == L.R) { get = 0; parity ^= 1; }
        fetch();
    }
    // a wait ran out, with the units from the k-th on still on their way: nothing more is waited for or fetched
    __device__ __forceinline__ void lose(int k = 0) {
        if (late) return;
        late = true; more = false;
        owed = ahead - k; owed_slot = get + k; owed_parity = parity;
        if (owed_slot >= L.R) { owed_slot -= L.R; owed_parity ^= 1; }
    }
    // before the block's shared memory goes back, what is on its way is waited for once more
    __device__ __forceinline__ void drain() {
        for (; late && owed > 0; owed--) {
            wait_for(bars + owed_slot * 8, owed_parity, tries_of(a));
            if (++owed_slot == L.R) { owed_slot = 0; owed_parity ^= 1; }
        }
    }
};

// ---- the kernel ------------------------------------------------------------------------------------------
//
// STATS: a row's maximum and sums, logprob, entropy and loss. GRAD: its gradient, from those (the policy loss) or, without
// STATS, from the ones of an earlier pass. ENT: entropies take part.
//
// A warp has a ring of shared memory to itself and fills it with bulk copies, units of 4096 bytes that only it reads: nothing
// waits for another warp but the row's sums. Where the row fits the rings of its cluster (resident) it is read from memory once: the units stay
// until the gradient has been taken from them; else they come a second time, out of L2. Where the rings hold two rows (ahead: up to 8000 logits of 16
// bits, 4000 of 32, a block) the sums of a row come before the gradient of the row before it, whose answer arrives meanwhile; all others wait, between a
// row's sums and its gradient, for the row's answer, with the next copies on their way where a warp has two units or more.
//
// The sums of all units go to every block that waits for the row's answer; one warp there does nothing but put them together and answer; it has fetched
// the rows' inputs beforehand. (As a part of one of the ordinary warps' work, between two barriers, that took 12 of 29 thousand cycles a row.)
//
// The least a call can take is one read of the logits and one write of the gradient. In bf16 rows with a gradient nothing is at its limit: nineteen instructions a
// logit (104 M of a warp for 1184 x 151936) keep the issue slots 62 % busy, two exponentials a logit half of their unit, DRAM is at 74 % of the copy rate
// (4096 x 151936 in 517 us); the warps wait for the row's answer, for one another's turn at the exponentials and for second reads that miss L2 (a quarter).
// Their logprobs alone, 8288 x 128256, take 371 us, 89 %, with the issue slots 73 % busy; fp32 rows and the backward pass are bounded by HBM and by what the second read
// finds in L2 (2072 x 128256 fp32 404 us, 81 %; backward 3600 x 128256 bf16 316 us, 90 %). fp16 takes what bf16 takes (4096 x 151936 514 us). A gradient whose rows begin
// elsewhere within 16 bytes than their logits is stored an element at a time: backward 2048 x 128256 bf16 185 us, one element off 569; policy 227 / 496, 1800 x 128256 fp32 356 / 405.
constexpr int DEPTH = 4;   // rows whose sums may be on their way

struct alignas(16) Control {
    RowShare share[DEPTH];
    uint64_t sums[DEPTH];      // the sums of all of a row's units are there (used in the cluster's first block)
    uint64_t answered[DEPTH];  // ... and have been read, and `share` has what they came to
};

__device__ __forceinline__ void cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t at_rank(const void *p, int rank) {
    uint32_t to;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(p)), "r"(rank));
    return to;
}
// 16 bytes into a block's shared memory. In a cluster of several they are counted by a barrier there, which needs no fence (one
// would also wait for this thread's stores to global memory), and nobody may leave before all that is under way to it is there; a
// block by itself stores them, and arrives at the barrier when it has.
__device__ __forceinline__ void put16(bool alone, const void *at, int rank, float x, float y, float z, float w, const void *bar) {
    if (alone) {
        asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(smem_u32(at)), "f"(x), "f"(y), "f"(z), "f"(w) : "memory");
    } else {
        asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(at_rank(at, rank)),
                     "r"(__float_as_uint(x)), "r"(__float_as_uint(y)), "r"(__float_as_uint(z)), "r"(__float_as_uint(w)), "r"(at_rank(bar, rank)) : "memory");
    }
}
__device__ __forceinline__ void arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

size_t smem_of(const Layout &L) {
    return (size_t)L.W * L.R * (UB + 8) + DEPTH * (size_t)L.table * sizeof(Stat);
}

// The warp that answers for the rows of a cluster: one in every block where a gradient waits, else one in the first.
template <class T, bool GRAD, bool ENT>
__device__ __forceinline__ void answer_rows(const LossArgs &a, const Layout &L, Control &ctl, Stat *stats, int rank, int row0, int step) {
    const int lane = threadIdx.x & 31;
    const bool alone = L.C == 1, first = rank == 0;
    bool late = false;
    int n = 0;   // rows that are read
    int head = -1, tail = -1;   // of the row before, and the logits of its last units
    Count of_last{}, of_edge{};
    RowIn mine = {};
    unsigned int mask = 0;
    for (int i = 0; (long long)row0 + (long long)i * step < a.B; i++) {
        if (i % 32 == 0) {
            const long long r = (long long)row0 + (long long)(i + lane) * step;
            bool read = false;
            if (r < a.B) {
                mine = row_in(a, (int)r);
                read = !mine.idle && !mine.status;
                if (read && first) mine.xt = to_f32(((const T *)a.logits)[r * a.row_stride + mine.token]);
                if (a.row_loss) {
                    mine.old = a.old_logprob[r]; mine.advantage = a.advantage[r];
                    if (a.ref_logprob) mine.ref = a.ref_logprob[r];
                }
                if (first && mine.idle) row_idle(a, (int)r);
                else if (first && mine.status) row_refused(a, (int)r, mine);
            }
            mask = __ballot_sync(0xffffffffu, read);
        }
        if (!(mask >> (i % 32) & 1)) continue;
        const int r = row0 + i * step, from = i % 32, s = n % DEPTH;
        Stat *st = stats + s * L.table;
        RowIn in;
        in.token = __shfl_sync(0xffffffffu, mine.token, from); in.T = __shfl_sync(0xffffffffu, mine.T, from);
        in.per_T = __shfl_sync(0xffffffffu, mine.per_T, from);
        in.old = __shfl_sync(0xffffffffu, mine.old, from); in.advantage = __shfl_sync(0xffffffffu, mine.advantage, from);
        in.weight = __shfl_sync(0xffffffffu, mine.weight, from); in.ref = __shfl_sync(0xffffffffu, mine.ref, from);
        in.xt = __shfl_sync(0xffffffffu, mine.xt, from);
        in.status = 0; in.idle = false;
        const RowSpan<T> span((const T *)a.logits + (long long)r * a.row_stride, a.V);
        const float c = LOG2E / in.T;
        const int units = span.units + (span.edge() ? 1 : 0);
        // The token's logit is the first block's to fetch: where the gradient takes the logits' place nobody may write before it has been read,
        // and nobody does before it has the answer, which needs it.
        if (!alone && !late) {
            if (lane == 0) mbar_expect_tx(&ctl.sums[s], (uint32_t)((max(units, L.C * L.W) + (GRAD ? 1 : 0)) * (int)sizeof(Stat)));
            if (GRAD && first && lane < L.C) put16(false, st + L.table - 1, lane, in.xt, 0.0f, 0.0f, 0.0f, &ctl.sums[s]);
        }
        if (span.head != head || span.tail != tail) {   // (seldom: the rows' sizes are alike where they begin alike)
            head = span.head; tail = span.tail;
            of_last = count_of(span.last_chunks() * Chunk<T>::N); of_edge = count_of(head + tail);
        }
        const float off = rounding_of(c, in.T);
        if (!late) late = !wait_for(&ctl.sums[s], (n / DEPTH) & 1, tries_of(a));
        if (late) {   // the barriers are out of step: this warp answers no more, and whoever waits for it gives up in turn
            in.status = MOLLA_ROW_LOAD_TIMEOUT;
            if (first && lane == 0) row_refused(a, r, in);
            continue;
        }
        if (GRAD && !alone) in.xt = st[L.table - 1].m;
        float M, W;
        Two S;
        bool missed;
        row_stat<T, ENT>(st, span, of_last, of_edge, c, off, M, S, W, missed);
        if (missed) in.status |= MOLLA_ROW_LOAD_TIMEOUT;
        Answer o;
        const RowGrad q = row_answer<ENT>(a, in, M, S, W, c, o);
        __syncwarp();
        if (LOSS_KNOB(a, 256) && r == a.B / 2 && rank == L.C - 1) {   // (testing build: an answer that never comes)
        } else if (GRAD || alone) {
            if (lane == 0) {
                ctl.share[s] = RowShare{M, c, q.A, q.H, q.token, in.token, q.A == 0.0f && q.H == 0.0f && q.token == 0.0f, 0};
                arrive(&ctl.answered[s]);
            }
        } else if (lane < L.C) {   // nothing but the news that the table is free again
            put16(false, &ctl.share[s], lane, 0.0f, 0.0f, 0.0f, 0.0f, &ctl.answered[s]);
        }
        if (first && lane == 0) row_write(a, r, in, M, S.hi, o);
        n++;
    }
}

// Rows from `first` on whose gradient a warp could not take. With STATS nobody else writes to them any more, and their gradient becomes zeros; a
// backward pass, whose warps do not wait for one another, leaves NaN in it and says so where it has been given the places.
template <class T, bool STATS> __device__ __noinline__ void give_up(const LossArgs &a, int first, int step) {
    for (long long r = first; r >= 0 && r < a.B; r += step) {
        if (!row_read<STATS>(a, (int)r)) continue;
        if ((threadIdx.x & 31) == 0) {
            if (a.status) a.status[r] = MOLLA_ROW_LOAD_TIMEOUT;
            if (a.logprob) a.logprob[r] = NAN;
            if (a.entropy) a.entropy[r] = NAN;
            if (a.kl) a.kl[r] = NAN;
            if (a.clipped) a.clipped[r] = 0;
            if (a.row_loss) a.row_loss[r] = NAN;
            else if (a.loss) *a.loss = NAN;
        }
        if (STATS) zero_row<T>((T *)a.grad + r * a.grad_stride, a.V, 0, 1);
    }
}

template <class T, bool STATS, bool GRAD, bool ENT>
__global__ void __launch_bounds__(MAX_WARPS * 32, 2) rows_kernel(const __grid_constant__ LossArgs a, const __grid_constant__ Layout L) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ Control ctl;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, rank = blockIdx.x % L.C;
    const int warp = rank * L.W + w, warps = L.C * L.W;
    const int row0 = blockIdx.x / L.C, step = L.rows_at_once;
    const bool alone = L.C == 1;
    wait_for_launch_before();
    const uint32_t slots = smem_u32(smem) + w * L.R * UB;
    Stat *stats = reinterpret_cast<Stat *>(smem + (size_t)L.W * L.R * UB);   // [DEPTH][table]
    uint64_t *bars = reinterpret_cast<uint64_t *>(stats + DEPTH * L.table) + w * L.R;
    if (STATS) {
        if (threadIdx.x < DEPTH) {
            mbar_init(&ctl.sums[threadIdx.x], L.C == 1 ? warps : 1);
            mbar_init(&ctl.answered[threadIdx.x], 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (w < L.W)
        for (int i = lane; i < L.R; i += 32) mbar_init(&bars[i], 1);
    fence_proxy_async();
    if (STATS) cluster_sync();
    else __syncwarp();
    if (STATS && w == L.W) {
        if (GRAD || rank == 0) answer_rows<T, GRAD, ENT>(a, L, ctl, stats, rank, row0, step);
        cluster_sync();
        return;
    }
    Feed<T, STATS, GRAD> feed(a, L, slots, smem_u32(bars), warp, warps, row0, step);
    unsigned int mask = 0;
    RowShare mine = {};   // a row a lane: without STATS all of it, else c
    int n = 0;            // rows that are read
    int held = 0;         // units that stay for the gradient of the row before
    int before = -1;      // that row
    bool cut_off = false; // a row's answer, or room for its sums, did not come in time: this warp has no part in any further row
    int lost = -1;        // the first row whose gradient it has not taken
    for (int i = 0;; i++) {
        const int r = feed.row_of(i), from = i % 32;
        const bool last = !feed.row_ok(i);
        if (last && before < 0) break;
        if (from == 0 && !last) {
            const bool ok = feed.row_ok(i + lane), read = ok && row_read<STATS>(a, feed.row_of(i + lane));
            mask = __ballot_sync(0xffffffffu, read);
            if (!STATS && read) mine = row_given(a, feed.row_of(i + lane));
            if (STATS) mine.c = LOG2E / (read && a.temperature ? a.temperature[feed.row_of(i + lane)] : 1.0f);
        }
        if (!last && !(mask >> from & 1)) {
            if (GRAD) zero_row<T>((T *)a.grad + (long long)r * a.grad_stride, a.V, warp, warps);
            continue;
        }
        int units = 0;   // of this row that stay
        if (STATS && !last) {
            const RowSpan<T> span((const T *)a.logits + (long long)r * a.row_stride, a.V);
            const int s = n % DEPTH;
            const float c = __shfl_sync(0xffffffffu, mine.c, from);
            // without a gradient nobody waits for a row's answer: its table has to be free again
            if (!GRAD && n >= DEPTH && !cut_off && !wait_for(&ctl.answered[s], (n / DEPTH + 1) & 1, tries_of(a))) { feed.lose(); cut_off = true; }
            if (!GRAD && w == 0 && lane == 0 && !alone && !cut_off) mbar_expect_tx(&ctl.answered[s], 16);
            const Stat *st = stats + s * L.table;
            const bool tell = lane < (GRAD ? L.C : 1) && !cut_off;   // a lane a block that wants to know
            for (int u = warp; u < span.units; u += warps) {
                const uint32_t slot = feed.wait(held + units);
                Stat o = u < span.full ? unit_stat<T, ENT, true, 1>(slot, 0, c) : unit_stat<T, ENT, false, GRAD ? 1 : 2>(slot, span.last_chunks(), c);
                if (feed.late || LOSS_KNOB(a, 16)) o.s_lo = LATE;   // (testing build: a wait that ran out)
                if (tell) put16(alone, st + u, lane, o.m, o.s, o.w, o.s_lo, &ctl.sums[s]);
                if (GRAD && L.resident) units++;
                else feed.give_back();
            }
            if (span.edge() && warp == span.units % warps) {
                const int at = span.edge_at(lane);
                const Stat o = edge_stat<ENT>(at != INT32_MIN ? to_f32(span.x[at]) : -INFINITY, c);
                if (tell) put16(alone, st + span.units, lane, o.m, o.s, o.w, o.s_lo, &ctl.sums[s]);
            }
            // a warp without a unit says so: no row's answer may come before every warp is done with the rows before it
            __syncwarp();
            if (alone) { if (lane == 0 && !cut_off) arrive(&ctl.sums[s]); }
            else if (tell && warp >= span.units + (span.edge() ? 1 : 0)) put16(false, st + warp, lane, 0.0f, 0.0f, 0.0f, 0.0f, &ctl.sums[s]);
            n++;
        }
        if (!GRAD) continue;
        // The gradient: of the row before, whose answer came meanwhile (of this one where it is given)
        int g = r;
        if (STATS && L.ahead) { g = before; before = last ? -1 : r; held = units; }
        if (g < 0) continue;
        RowShare q;
        if (STATS) {
            const int k = last || !L.ahead ? n - 1 : n - 2, s = k % DEPTH;
            if (!cut_off && !wait_for(&ctl.answered[s], (k / DEPTH) & 1, tries_of(a))) { feed.lose(); cut_off = true; if (lost < 0) lost = g; }
            if (cut_off) continue;
            q = ctl.share[s];
        } else {
            q.M = __shfl_sync(0xffffffffu, mine.M, from); q.c = __shfl_sync(0xffffffffu, mine.c, from);
            q.A = __shfl_sync(0xffffffffu, mine.A, from); q.H = __shfl_sync(0xffffffffu, mine.H, from);
            q.token_add = __shfl_sync(0xffffffffu, mine.token_add, from); q.token = __shfl_sync(0xffffffffu, mine.token, from);
            q.zero = 0;
        }
        const RowSpan<T> span((const T *)a.logits + (long long)g * a.row_stride, a.V);
        T *out = (T *)a.grad + (long long)g * a.grad_stride, *to = out + span.head;
        const bool wide = ((uintptr_t)to & 15) == 0;
        const int edge_at = span.edge() && warp == span.units % warps ? span.edge_at(lane) : INT32_MIN;
        const float edge = edge_at != INT32_MIN ? to_f32(span.x[edge_at]) : 0.0f;
        if (q.zero) zero_row<T>(out, a.V, warp, warps);
        const int at_token = q.token - span.head, token_unit = at_token < 0 ? -1 : at_token / UNIT<T>;
        T *at = to + warp * UNIT<T>;
        for (int u = warp; u < span.units; u += warps, at += warps * UNIT<T>) {
            const uint32_t slot = STATS && L.resident ? feed.oldest() : feed.wait(0);
            const bool gone = feed.late && !(STATS && L.resident);   // (units that stay are there)
            const float A = !STATS && gone ? NAN : q.A;
            if (gone && !q.zero && lost < 0) lost = g;
            if (!q.zero && !(STATS && gone)) {
                if (u < span.full && wide) unit_gradient<T, ENT, true>(slot, 0, at, true, q.M, q.c, A, q.H);
                else unit_gradient<T, ENT, false>(slot, u < span.full ? UB / 16 : span.last_chunks(), at, wide, q.M, q.c, A, q.H);
                if (u == token_unit) {
                    const int t = at_token - u * UNIT<T>;
                    __syncwarp();   // behind the store of the whole chunk
                    if (lane == 0 && t * (int)sizeof(T) < span.bytes - u * UB)
                        at[t] = from_f32<T>(gradient_of<T, ENT>(lds_element<T>(slot + t * (int)sizeof(T)), q.M, q.c, A, q.H) + q.token_add);
                }
            }
            feed.give_back();
        }
        if (edge_at != INT32_MIN && !q.zero)
            to[edge_at] = from_f32<T>(gradient_of<T, ENT>(edge, q.M, q.c, q.A, q.H) + (edge_at == q.token - span.head ? q.token_add : 0.0f));
    }
    feed.drain();
    if (STATS) {
        // The last answers, which without a gradient nobody has waited for; nobody leaves while another block has something for it.
        for (int k = max(n - DEPTH, 0); k < n; k++)
            if (!wait_for(&ctl.answered[k % DEPTH], (k / DEPTH) & 1, tries_of(a))) break;
        cluster_sync();
    }
    if (GRAD && lost >= 0) give_up<T, STATS>(a, lost, !STATS && a.follows ? -step : step);
}

// ---- sums over rows ---------------------------------------------------------------------------------

constexpr int ST = 1024;

__device__ double sum_1024(double v, double *ws) {
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) v += __shfl_xor_sync(0xffffffffu, v, i);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) ws[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = ws[threadIdx.x & 31];
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) s += __shfl_xor_sync(0xffffffffu, s, i);
    return s;
}

__global__ void __launch_bounds__(ST) row_sum_kernel(const float *row_loss, int B, float scale, float *loss) {
    __shared__ double ws[ST / 32];
    wait_for_launch_before();
    double v = 0.0;
    for (int i = threadIdx.x; i < B; i += ST) v += (double)row_loss[i];
    v = sum_1024(v, ws);
    if (threadIdx.x == 0) *loss = (float)(v * (double)scale);
}

// Warps adds up the log ratios of a sequence's rows: each lane every so-manieth, then the lanes in the order of a tree.
__device__ double sequence_sum(const PairArgs &a, int from, int to, int step, unsigned int *status) {
    double v = 0.0;
#pragma unroll 4
    for (int r = from; r < to; r += step) {
        *status |= a.row_status[r] & ROW_ERRORS;
        if (a.tokens[r] != -1) v += ((double)a.logprob[r] - (a.ref_logprob ? (double)a.ref_logprob[r] : 0.0)) + (double)a.logprob_lo[r];
    }
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) v += __shfl_xor_sync(0xffffffffu, v, i);
    return v;
}

// ln(1 + exp(m)), and the sigmoid
__device__ __forceinline__ double soft(double m) { return fmax(m, 0.0) + log1p(exp(-fabs(m))); }
__device__ __forceinline__ double sigmoid(double m) { return m >= 0.0 ? 1.0 / (1.0 + exp(-m)) : exp(m) / (1.0 + exp(m)); }

// One block: the pairs a warp each, or, if they are few, as many warps as there are for each.
// Bound by latency: offsets, rows and sums in 64 bits one after the other, then the launch (12 us for 8 pairs of 450 rows; it begins while the score ends). One
// block, so that the loss is added up in one order without another launch.
__global__ void __launch_bounds__(ST) pairs_kernel(const __grid_constant__ PairArgs a) {
    __shared__ double ws[ST / 32], chosen[ST / 32], rejected[ST / 32];
    __shared__ unsigned int statuses[ST / 32];
    wait_for_launch_before();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, S = 2 * a.n_pairs;
    int bad = 0;
    for (int s = threadIdx.x; s < S; s += ST) bad |= a.off[s] < 0 || a.off[s + 1] < a.off[s] || a.off[s + 1] > a.B;
    const bool broken = __syncthreads_or(bad) != 0;
    if (a.g_logprob) {   // rows of no sequence
        const int first = broken || S == 0 ? a.B : a.off[0], last = broken || S == 0 ? a.B : a.off[S];
        for (int r = threadIdx.x; r < first; r += ST) a.g_logprob[r] = 0.0f;
        for (int r = last + threadIdx.x; r < a.B; r += ST) a.g_logprob[r] = 0.0f;
    }
    int at_once = 1;   // pairs, of `each` warps
    while (at_once < a.n_pairs && at_once < ST / 32) at_once *= 2;
    const int each = ST / 32 / at_once, group = warp / each, of_pair = threadIdx.x - group * each * 32, step = each * 32;
    double total = 0.0;
    for (int p0 = 0; p0 < a.n_pairs; p0 += at_once) {
        const int p = p0 + group;
        const bool mine = p < a.n_pairs && !broken;
        const int o0 = mine ? a.off[2 * p] : 0, o1 = mine ? a.off[2 * p + 1] : 0, o2 = mine ? a.off[2 * p + 2] : 0;
        unsigned int status = 0;
        const double c = sequence_sum(a, o0 + of_pair, o1, step, &status), d = sequence_sum(a, o1 + of_pair, o2, step, &status);
        status = __reduce_or_sync(0xffffffffu, status);
        __syncthreads();
        if (lane == 0) { chosen[warp] = c; rejected[warp] = d; statuses[warp] = status; }
        __syncthreads();
        if (p >= a.n_pairs) continue;
        if (broken) {
            if (of_pair == 0) {
                const int *o = a.off + 2 * p;
                a.pair_status[p] = o[0] < 0 || o[1] < o[0] || o[2] < o[1] || o[2] > a.B ? MOLLA_ROW_INVALID_CONFIG : 0u;
                a.pair_loss[p] = a.margin[p] = a.seq_logratio[2 * p] = a.seq_logratio[2 * p + 1] = NAN;
            }
            total = NAN;
            continue;
        }
        double sc = 0.0, sr = 0.0;
        status = 0;
        for (int k = group * each; k < (group + 1) * each; k++) { sc += chosen[k]; sr += rejected[k]; status |= statuses[k]; }
        const double beta = a.beta, eps = a.smoothing, w = a.weight ? (double)a.weight[p] : 1.0, m = beta * (sc - sr);
        const double l = w == 0.0 ? 0.0 : w * ((1.0 - eps) * soft(-m) + (eps == 0.0 ? 0.0 : eps * soft(m)));   // (of an infinite margin too)
        const double dm = status || w == 0.0 ? 0.0 : w * (eps * sigmoid(m) - (1.0 - eps) * sigmoid(-m));
        if (of_pair == 0) {
            total += l;
            a.pair_status[p] = status;
            a.pair_loss[p] = (float)l; a.margin[p] = (float)m;
            a.seq_logratio[2 * p] = (float)sc; a.seq_logratio[2 * p + 1] = (float)sr;
        }
        if (a.g_logprob) {
            const float g = (float)(beta * dm * (double)a.scale * (double)a.grad_scale);
            for (int r = o0 + of_pair; r < o1; r += step) a.g_logprob[r] = g;
            for (int r = o1 + of_pair; r < o2; r += step) a.g_logprob[r] = -g;
        }
    }
    total = sum_1024(lane == 0 ? total : 0.0, ws);
    if (threadIdx.x == 0) *a.loss = (float)(total * (double)a.scale);
}

// ---- launches --------------------------------------------------------------------------------------------

constexpr int MAX_DEVICES = 64;

struct Fits { int threads, smem, n; };

int sm_count_of(int &dev) {
    int sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) { dev = -1; return 0; }
    return sms;
}

constexpr size_t block_smem(int per_sm) { return (size_t)(228 / per_sm - 2) * 1024; }   // of a block's dynamic shared memory: an SM's 228 KB less what each block takes besides

// W warps, or as many fewer as share a block's units evenly (6 % of the rounds idle).
int even(int share, int W) {
    int best = 0x7fffffff, chosen = 1;
    if (W > share) W = share;
    for (int w = W; w > W / 2; w--) {
        const int rounds = (share + w - 1) / w * w;
        if (rounds < best && (best == 0x7fffffff || best * 16 > share * 17)) { best = rounds; chosen = w; }
    }
    return chosen;
}

// C blocks a row, at most W warps a block, and the shared memory of `per_sm` blocks an SM.
Layout layout_with(int C, int W, int per_sm, int V, int size) {
    Layout L{};
    const int unit = UB / size, most = (int)(((long long)V * size + UB - 1) / UB), share = (most + C - 1) / C;   // units of a row, and of a block
    L.C = C;
    L.table = max((V + unit - 1) / unit + 1, C * W) + 1;   // (an unaligned row's whole chunks and its edge, or a place a warp; the token's logit)
    const auto room = [&] { const size_t all = block_smem(per_sm), tables = DEPTH * (size_t)L.table * sizeof(Stat); return all > tables ? (int)((all - tables) / (UB + 8)) : 0; };
    while (per_sm > 1 && room() < (W < share ? W : share)) per_sm--;   // (the widest rows' tables)
    const int slots = room();
    L.W = even(share, W < slots ? W : slots);
    const int each = (share + L.W - 1) / L.W;
    L.R = slots / L.W;
    if (L.R > 32) L.R = 32;
    L.ahead = 2 * each <= L.R;
    L.resident = each <= L.R;
    return L;
}

// Long rows have 13 warps in two blocks an SM, with two units of shared memory each (one where the tables of sums leave no more, and then
// nothing is on its way while the warp works: fp32 rows of 125 to 133, 150 to 159, 197 to 212 and 250 to 262 thousand logits, 16-bit ones from 250 thousand); rows (or a block's part of them) of up to 18 units as many
// warps as leave two units to a warp, in as many more blocks an SM, so that they stay in shared memory; rows of up to 4 units a warp a unit.
// Policy loss with its gradient, us, in 2 / 3 / 5 / 6 / 10 blocks an SM: 4096 x 32000 bf16 146 / 124 / 126 / 126 / 135, 8192 x 50304 bf16
// 357 / 433 / - / - / -, 16384 x 8000 bf16 296 / 228 / 165 / 165 / 168, 32768 x 2000 bf16 554 / 386 / 259 / 222 / 161.
//
// Without a gradient nothing waits for an answer, and more blocks of fewer warps are better: 13 warps in two blocks an SM, 7 in four, us: 2048 x 128256 bf16
// 123 / 111, 8288 x 128256 bf16 395 / 381, 4096 x 128256 fp32 350 / 339.
//
// Where a row's units come a second time, out of L2, as many blocks share a row as keep what is in flight below 96 MB: 1 / 2 / 4 blocks a row took
// 532 / 575 / 675 us for 4096 x 151936 bf16 (304 KB a row), 507 / 468 / - for 2048 x 262144 bf16 (524 KB), 480 / 402 / 418 for 2072 x 128256 fp32
// (513 KB), 519 / 495 / 413 for 1024 x 262144 fp32 (1 MB). Of fp32 rows, which have less to compute and so feel what L2 loses more, two share a row from 60 MB on:
// 329 / 288 for 3000 x 65536 (77 MB), 200 / 223 for 4096 x 32000 (38 MB). Few rows are shared by as many blocks as there is room for: 4 x 32000 fp32
// 19.5 / 17.4 / 15.4, by eight 15.4.
//
// Many rows of a block each: five or nine warps with the one that answers leave one of an SM's four schedulers most of the work, and where the rounds of
// 13 do not come out even, seven in four blocks idle less. Usual / as here, us, 400 MB of logits: score, bf16, units a row 10, 15, 19, 25: 115 / 97, 107 / 94,
// 98 / 94, 101 / 96 (13: 98 / 96, and 40 / 45 with only 2450 rows: seven stay); backward 4, 10, 18: 162 / 151, 156 / 149, 150 / 145; policy loss with
// its gradient, bf16, four in six blocks though the units do not stay, 15, 18, 20, 24: 228 / 196, 208 / 191, 218 / 187, 189 / 181 (16, eight in three: 198 / 202;
// fp32, 15, 18: 158 / 168, 145 / 176); seven in four for 28, 40: 224 / 189, 202 / 187, fp32 173 / 159, 160 / 178; eleven in two, whose rounds are
// three warps a scheduler, not four, of bf16 63, 75: 185 / 179, 530 / 516 (4096 rows), and of 700 MB 63, 64, 65, 74, 75, 76, 77: 324 / 321, 321 / 326, 320 / 315,
// 327 / 318, 334 / 332, 333 / 330, 336 / 330; wider rows lose by it (86, 87, 98: 346 / 348, 329 / 332, 355 / 360), and so does 50, 16 rounds against 15: 188 / 203.
template <class T, bool STATS, bool GRAD> Layout layout_of(int B, int V, int sms) {
    const int size = (int)sizeof(T), most = (int)(((long long)V * size + UB - 1) / UB);
    int C = 1;
    if (STATS && GRAD)
        while (C < 8 && (most + C - 1) / C > 18 && 2ll * sms / C * most * UB > (size == 4 && C == 1 ? 60ll : 96ll) << 20) C *= 2;
    while (C < 8 && 2ll * B * C <= 2ll * sms * 15 / 16 && most >= 8 * C) C *= 2;
    const int share = (most + C - 1) / C;
    int W = share <= 4 ? share : share <= 18 ? (share + 1) / 2 : STATS ? 13 : 16;
    if (STATS && !GRAD && (long long)B * C > sms) W = even(share, share <= 6 ? (share + 1) / 2 : 7);
    else if (W < 13) W = even(share, W);
    int per_sm = W >= 13 ? 2 : 32 / (W + 1);
    const auto rounds = [&](int w) { return (share + w - 1) / w; };
    const long long rows_per_sm = C == 1 ? B / sms : 0;
    if (!STATS && W != 7 && share >= 4 && share <= 18 && rows_per_sm >= 16) {
        W = 4;
        per_sm = 8;
    } else if (STATS && !GRAD && size == 2 && W != 7 && share > 7 && share <= 32 && rows_per_sm >= 16) {
        W = 3;
        per_sm = 8;
    } else if (STATS && GRAD && size == 2 && W != 7 && W != 8 && share >= 13 && share <= 24 && rows_per_sm >= 12) {
        W = 4;
        per_sm = 6;
    } else if (STATS && GRAD && share > 18 && rows_per_sm >= 8) {
        const int usual = even(share, W);
        if (share <= (size == 4 ? 28 : 41) && even(share, 7) == 7 && 40 * rounds(usual) > 23 * rounds(7)) {
            W = 7;
            per_sm = 4;
        } else if (size == 2 && share > 41 && share <= 80 && even(share, 11) == 11 && 10 * 3 * rounds(11) <= 9 * ((usual + 3) / 4) * rounds(usual)) {
            W = 11;
        }
    }
    return layout_with(C, W, per_sm < 10 ? per_sm : 10, V, size);
}

template <class T, bool STATS, bool GRAD, bool ENT> cudaError_t launch_rows(const LossArgs &a, cudaStream_t st) {
    int dev = 0;
    const int sms = sm_count_of(dev);
    if (sms <= 0) return cudaErrorInvalidDevice;
    Layout L = layout_of<T, STATS, GRAD>(a.B, a.V, sms);
    const size_t smem = smem_of(L);
    auto kernel = rows_kernel<T, STATS, GRAD, ENT>;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[2];
    cfg.blockDim = dim3(32u * (unsigned int)(L.W + (STATS ? 1 : 0))); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned int)L.C; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    const bool clusters = STATS && L.C > 1;
    cfg.attrs = at; cfg.numAttrs = clusters ? 1 : 0;
    // How many clusters the device holds at a time, asked once per device and layout: one too many would wait for all
    // rows of another (72 of four blocks, two an SM, fit where 74 would fill the SMs).
    static thread_local Fits known[MAX_DEVICES][4] = {};
    const int kind = L.C == 1 ? 0 : L.C == 2 ? 1 : L.C == 4 ? 2 : 3;
    Fits fits = dev < MAX_DEVICES ? known[dev][kind] : Fits{};
    if (fits.threads != (int)cfg.blockDim.x || fits.smem != (int)smem) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)block_smem(1));
        if (e != cudaSuccess) return e;
        fits = Fits{(int)cfg.blockDim.x, (int)smem, 0};
        if (clusters) {
            cfg.gridDim = dim3((unsigned int)L.C);
            e = cudaOccupancyMaxActiveClusters(&fits.n, kernel, &cfg);
        } else {
            e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fits.n, kernel, (int)cfg.blockDim.x, smem);
            fits.n = fits.n * sms / L.C;
        }
        if (e != cudaSuccess) return e;
        if (fits.n < 1) return cudaErrorLaunchOutOfResources;
        if (dev < MAX_DEVICES) known[dev][kind] = fits;
    }
    L.rows_at_once = fits.n < a.B ? fits.n : a.B;
    cfg.gridDim = dim3((unsigned int)(L.rows_at_once * L.C));
    if (a.follows) { cfg.attrs = clusters ? at : at + 1; cfg.numAttrs++; }
    return cudaLaunchKernelEx(&cfg, kernel, a, (const Layout)L);
}

// one block behind another kernel of the same call
template <class... P> cudaError_t launch_one_block(void (*kernel)(P...), cudaStream_t st, P... args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(1); cfg.blockDim = dim3(ST); cfg.stream = st; cfg.attrs = at; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <bool STATS, bool GRAD> cudaError_t launch_type(const LossArgs &a, bool ent, cudaStream_t st) {
    if (a.B == 0) return cudaSuccess;
    switch (a.type) {
        case MOLLA_LOGITS_FP32: return ent ? launch_rows<float, STATS, GRAD, true>(a, st) : launch_rows<float, STATS, GRAD, false>(a, st);
        case MOLLA_LOGITS_BF16: return ent ? launch_rows<__nv_bfloat16, STATS, GRAD, true>(a, st) : launch_rows<__nv_bfloat16, STATS, GRAD, false>(a, st);
        default: return ent ? launch_rows<__half, STATS, GRAD, true>(a, st) : launch_rows<__half, STATS, GRAD, false>(a, st);
    }
}

}  // namespace

cudaError_t molla_loss_score(const LossArgs &a, cudaStream_t st) { return launch_type<true, false>(a, a.entropy || a.depth, st); }

cudaError_t molla_loss_backward(const LossArgs &a, cudaStream_t st) { return launch_type<false, true>(a, a.g_entropy != nullptr, st); }

cudaError_t molla_loss_policy(const LossArgs &a, cudaStream_t st) {
    const bool ent = a.entropy != nullptr || a.entropy_coef != 0.0f;
    const cudaError_t e = a.grad ? launch_type<true, true>(a, ent, st) : launch_type<true, false>(a, ent, st);
    if (e != cudaSuccess) return e;
    return launch_one_block(row_sum_kernel, st, (const float *)a.row_loss, a.B, a.scale, a.loss);
}

cudaError_t molla_loss_pairs(const PairArgs &a, cudaStream_t st) {
    return launch_one_block(pairs_kernel, st, a);
}
