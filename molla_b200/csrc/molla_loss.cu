// Logprobs of given tokens, their gradient, and the losses over them (the formulas: include/molla_sample.h).
//
// With M = max x, c = log2(e)/T and e_j = 2^(c (x_j - M)), S = sum e_j and W = sum e_j (x_j - M):
//     logprob = (x_t - M)/T - ln S        entropy = ln S - W/(S T)        p_j = e_j/S
// and for g = dL/dlogprob, h = dL/dentropy the gradient by logit j is
//     g [j = t]/T - e_j (A + H (x_j - M))   with  H = h/(T T S),  A = (g - h W/(S T))/(T S)
// so a row needs three numbers (M, S, W) for everything. Differences from M are exact for the logits that matter, and
// whatever rounding e_j has is the same in S and in the gradient, where it cancels to first order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/molla_sample.h"
#include "molla_loss.h"

namespace {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float DEEP = -1e30f;    // where x - M is held, so that 0 * (x - M) is 0 for logits of -inf too
constexpr unsigned int ROW_ERRORS = MOLLA_ROW_BAD_TOKEN | MOLLA_ROW_EMPTY | MOLLA_ROW_INVALID_CONFIG | MOLLA_ROW_LOAD_TIMEOUT;

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

struct RowIn {
    int token;
    float T;             // temperature
    unsigned int status; // why the row cannot be answered, before it is read
    bool idle;           // nothing to answer: no token, or no weight
};

__device__ __forceinline__ RowIn row_in(const LossArgs &a, int r) {
    RowIn in;
    in.token = a.tokens[r];
    in.T = a.temperature ? a.temperature[r] : 1.0f;
    in.idle = in.token == -1 || (a.weight && a.weight[r] == 0.0f);
    in.status = 0;
    if (!in.idle) {
        if (in.token < 0 || in.token >= a.V) in.status |= MOLLA_ROW_BAD_TOKEN;
        const float c = LOG2E / in.T;
        if (!(in.T > 0.0f) || !(c > 0.0f) || isinf(c)) in.status |= MOLLA_ROW_INVALID_CONFIG;
    }
    return in;
}

// The gradient's three numbers: add at the token, and A and H of the formula.
struct RowGrad { float token, A, H; };

__device__ __forceinline__ RowGrad row_grad(double g, double h, float T, float S, double w_over_st) {
    RowGrad o;
    const double inv = 1.0 / ((double)T * (double)S);
    o.token = (float)(g / (double)T);
    o.A = (float)((g - h * w_over_st) * inv);
    o.H = (float)(h * inv / (double)T);
    return o;
}

// What a row answers once its maximum M, sum S and, where entropies are wanted, W are known. One thread.
__device__ RowGrad row_answer(const LossArgs &a, int r, const RowIn &in, float xt, float M, float S, float W) {
    const bool empty = M == -INFINITY;
    const unsigned int status = in.status | (empty && !in.status ? MOLLA_ROW_EMPTY : 0u);
    const double T = in.T, lnS = log((double)S);
    const double l = ((double)xt - (double)M) / T - lnS;
    const bool want_entropy = a.entropy != nullptr || a.entropy_coef != 0.0f;
    const double w_over_st = want_entropy ? (double)W / ((double)S * T) : 0.0;
    const double H = lnS - w_over_st;
    RowGrad o{0.0f, 0.0f, 0.0f};
    a.status[r] = status;
    a.logprob[r] = status ? NAN : (float)l;
    if (a.entropy) a.entropy[r] = status ? NAN : (float)H;
    if (a.stats) { a.stats[2 * r] = status ? NAN : M; a.stats[2 * r + 1] = status ? 0.0f : S; }
    if (!a.row_loss) return o;
    // the policy loss
    const double w = a.weight ? (double)a.weight[r] : 1.0;
    const double ratio = exp(l - (double)a.old_logprob[r]), adv = a.advantage[r];
    const double lo = 1.0 - (double)a.clip_low, hi = 1.0 + (double)a.clip_high;
    const double u = ratio * adv, c = fmin(fmax(ratio, lo), hi) * adv;
    const bool held = c < u;
    double term = -(held ? c : u), g = held ? 0.0 : -u;   // (a ratio that is NaN is not held)
    if (a.ref_logprob) {
        const double q = (double)a.ref_logprob[r] - l, eq = expm1(q), kl = eq - q;
        if (a.kl) a.kl[r] = status ? NAN : (float)kl;
        if (a.kl_coef != 0.0f) { term += (double)a.kl_coef * kl; g -= (double)a.kl_coef * eq; }
    }
    double h = 0.0;
    if (a.entropy_coef != 0.0f) { term -= (double)a.entropy_coef * H; h = -w * (double)a.entropy_coef; }
    a.row_loss[r] = status ? NAN : (float)(w * term);
    if (a.clipped) a.clipped[r] = !status && held;
    const double gs = (double)a.scale * (double)a.grad_scale;
    if (!status) o = row_grad(g * w * gs, h * gs, in.T, S, w_over_st);
    return o;
}

__device__ void row_idle(const LossArgs &a, int r) {
    a.status[r] = 0;
    a.logprob[r] = 0.0f;
    if (a.entropy) a.entropy[r] = 0.0f;
    if (a.stats) { a.stats[2 * r] = 0.0f; a.stats[2 * r + 1] = 1.0f; }
    if (a.row_loss) a.row_loss[r] = 0.0f;
    if (a.kl) a.kl[r] = 0.0f;
    if (a.clipped) a.clipped[r] = 0;
}

// ---- a block a row --------------------------------------------------------------------------------

constexpr int NT = 512;

__device__ float block_max(float v, float *ws) {
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, i));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) ws[threadIdx.x >> 5] = v;
    __syncthreads();
    float m = ws[0];
    for (int i = 1; i < NT / 32; i++) m = fmaxf(m, ws[i]);
    return m;
}
__device__ float block_sum(float v, float *ws) {
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) v += __shfl_xor_sync(0xffffffffu, v, i);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) ws[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = ws[0];
    for (int i = 1; i < NT / 32; i++) s += ws[i];
    return s;
}

template <class T>
__device__ void write_gradient(const LossArgs &a, int r, const T *x, int token, float M, float c, const RowGrad &q, bool zero) {
    T *out = (T *)a.grad + (long long)r * a.grad_stride;
    for (int j = threadIdx.x; j < a.V; j += NT) {
        float v = 0.0f;
        if (!zero) {
            const float raw = __fsub_rn(to_f32(x[j]), M), d = raw < DEEP ? DEEP : raw;
            v = -ex2(d * c) * __fmaf_rn(q.H, d, q.A);
            if (j == token) v += q.token;
        }
        out[j] = from_f32<T>(v);
    }
}

// Everything a row's logits are read for: logprob, and with `a.grad` the policy loss's gradient.
template <class T>
__global__ void __launch_bounds__(NT) rows_kernel(const __grid_constant__ LossArgs a) {
    __shared__ float ws[NT / 32];
    __shared__ RowGrad s_grad;
    const int r = blockIdx.x;
    const T *x = (const T *)a.logits + (long long)r * a.row_stride;
    const RowIn in = row_in(a, r);
    float M = 0.0f, S = 1.0f, W = 0.0f;
    const float c = LOG2E / in.T;
    if (in.idle) {
        if (threadIdx.x == 0) { row_idle(a, r); s_grad = RowGrad{0.0f, 0.0f, 0.0f}; }
    } else {
        if (!in.status) {
            float m = -INFINITY;
            for (int j = threadIdx.x; j < a.V; j += NT) m = fmaxf(m, to_f32(x[j]));
            M = block_max(m, ws);
            float s = 0.0f, w = 0.0f;
            if (M > -INFINITY)
                for (int j = threadIdx.x; j < a.V; j += NT) {
                    const float raw = __fsub_rn(to_f32(x[j]), M), d = raw < DEEP ? DEEP : raw, e = ex2(d * c);
                    s += e;
                    w = __fmaf_rn(e, d, w);
                }
            S = block_sum(s, ws);
            W = block_sum(w, ws);
        }
        if (threadIdx.x == 0) s_grad = row_answer(a, r, in, in.status ? 0.0f : to_f32(x[in.token]), M, S, W);
    }
    if (!a.grad) return;
    __syncthreads();
    const RowGrad q = s_grad;
    write_gradient<T>(a, r, x, in.token, M, c, q, q.token == 0.0f && q.A == 0.0f && q.H == 0.0f);
}

// The gradient from the stats of an earlier pass.
template <class T>
__global__ void __launch_bounds__(NT) backward_kernel(const __grid_constant__ LossArgs a) {
    const int r = blockIdx.x;
    const T *x = (const T *)a.logits + (long long)r * a.row_stride;
    const int token = a.tokens[r];
    const float temp = a.temperature ? a.temperature[r] : 1.0f, M = a.in_stats[2 * r], S = a.in_stats[2 * r + 1];
    const float g = a.g_logprob[r], h = a.g_entropy ? a.g_entropy[r] : 0.0f;
    const bool zero = token < 0 || token >= a.V || (g == 0.0f && h == 0.0f) || S == 0.0f;
    RowGrad q{0.0f, 0.0f, 0.0f};
    if (!zero) q = row_grad(g, h, temp, S, h != 0.0f ? log((double)S) - (double)a.in_entropy[r] : 0.0);
    write_gradient<T>(a, r, x, token, M, LOG2E / temp, q, zero);
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
    double v = 0.0;
    for (int i = threadIdx.x; i < B; i += ST) v += (double)row_loss[i];
    v = sum_1024(v, ws);
    if (threadIdx.x == 0) *loss = (float)(v * (double)scale);
}

// A warp adds up the log ratios of a sequence's rows, each lane every 32nd, then the lanes in the order of a tree.
__device__ double sequence_sum(const PairArgs &a, int from, int to, unsigned int *status) {
    const int lane = threadIdx.x & 31;
    double v = 0.0;
    for (int r = from + lane; r < to; r += 32) {
        *status |= a.row_status[r] & ROW_ERRORS;
        if (a.tokens[r] != -1) v += (double)a.logprob[r] - (a.ref_logprob ? (double)a.ref_logprob[r] : 0.0);
    }
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) v += __shfl_xor_sync(0xffffffffu, v, i);
    return v;
}

// ln(1 + exp(m)), and the sigmoid
__device__ __forceinline__ double soft(double m) { return fmax(m, 0.0) + log1p(exp(-fabs(m))); }
__device__ __forceinline__ double sigmoid(double m) { return m >= 0.0 ? 1.0 / (1.0 + exp(-m)) : exp(m) / (1.0 + exp(m)); }

// One block: the pairs a warp each, in turn.
__global__ void __launch_bounds__(ST) pairs_kernel(const __grid_constant__ PairArgs a) {
    __shared__ double ws[ST / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, S = 2 * a.n_pairs;
    int bad = 0;
    for (int s = threadIdx.x; s < S; s += ST) bad |= a.off[s] < 0 || a.off[s + 1] < a.off[s] || a.off[s + 1] > a.B;
    const bool broken = __syncthreads_or(bad) != 0;
    if (a.g_logprob) {   // rows of no sequence
        const int first = broken || S == 0 ? a.B : a.off[0], last = broken || S == 0 ? a.B : a.off[S];
        for (int r = threadIdx.x; r < first; r += ST) a.g_logprob[r] = 0.0f;
        for (int r = last + threadIdx.x; r < a.B; r += ST) a.g_logprob[r] = 0.0f;
    }
    double total = 0.0;
    for (int p = warp; p < a.n_pairs; p += ST / 32) {
        if (broken) {
            if (lane == 0) {
                const int *o = a.off + 2 * p;
                a.pair_status[p] = o[0] < 0 || o[1] < o[0] || o[2] < o[1] || o[2] > a.B ? MOLLA_ROW_INVALID_CONFIG : 0u;
                a.pair_loss[p] = a.margin[p] = a.seq_logratio[2 * p] = a.seq_logratio[2 * p + 1] = NAN;
            }
            total = NAN;
            continue;
        }
        const int o0 = a.off[2 * p], o1 = a.off[2 * p + 1], o2 = a.off[2 * p + 2];
        unsigned int status = 0;
        const double sc = sequence_sum(a, o0, o1, &status), sr = sequence_sum(a, o1, o2, &status);
        status = __reduce_or_sync(0xffffffffu, status);
        const double beta = a.beta, eps = a.smoothing, w = a.weight ? (double)a.weight[p] : 1.0, m = beta * (sc - sr);
        const double l = w == 0.0 ? 0.0 : w * ((1.0 - eps) * soft(-m) + eps * soft(m));
        const double dm = status || w == 0.0 ? 0.0 : w * (eps * sigmoid(m) - (1.0 - eps) * sigmoid(-m));
        total += l;
        if (lane == 0) {
            a.pair_status[p] = status;
            a.pair_loss[p] = (float)l; a.margin[p] = (float)m;
            a.seq_logratio[2 * p] = (float)sc; a.seq_logratio[2 * p + 1] = (float)sr;
        }
        if (a.g_logprob) {
            const float g = (float)(beta * dm * (double)a.scale * (double)a.grad_scale);
            for (int r = o0 + lane; r < o1; r += 32) a.g_logprob[r] = g;
            for (int r = o1 + lane; r < o2; r += 32) a.g_logprob[r] = -g;
        }
    }
    total = sum_1024(lane == 0 ? total : 0.0, ws);
    if (threadIdx.x == 0) *a.loss = (float)(total * (double)a.scale);
}

template <class K> cudaError_t launch_rows(K f32, K bf16, K fp16, const LossArgs &a, cudaStream_t st) {
    if (a.B == 0) return cudaSuccess;
    (a.type == MOLLA_LOGITS_FP32 ? f32 : a.type == MOLLA_LOGITS_BF16 ? bf16 : fp16)<<<a.B, NT, 0, st>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t molla_loss_score(const LossArgs &a, cudaStream_t st) {
    return launch_rows(rows_kernel<float>, rows_kernel<__nv_bfloat16>, rows_kernel<__half>, a, st);
}

cudaError_t molla_loss_backward(const LossArgs &a, cudaStream_t st) {
    return launch_rows(backward_kernel<float>, backward_kernel<__nv_bfloat16>, backward_kernel<__half>, a, st);
}

cudaError_t molla_loss_policy(const LossArgs &a, cudaStream_t st) {
    const cudaError_t e = molla_loss_score(a, st);
    if (e != cudaSuccess) return e;
    row_sum_kernel<<<1, ST, 0, st>>>(a.row_loss, a.B, a.scale, a.loss);
    return cudaGetLastError();
}

cudaError_t molla_loss_pairs(const PairArgs &a, cudaStream_t st) {
    pairs_kernel<<<1, ST, 0, st>>>(a);
    return cudaGetLastError();
}
