// Losses over the log-probabilities of given labels: label log-probabilities with their gradient, the preference loss
// (paired log ratios against a reference policy) and the clipped policy loss with a KL term.
//
// Positions (n, l) of N sequences (or pictures) of L labels each carry C logits x_c.  With z = x / T, m = max x and
// s = sum_c exp((x_c - m) / T):
//   logp = (x_label - m) / T - log s,      d logp / d x_c = ([c == label] - exp((x_c - m) / T) / s) / T.
// Everything is held in fp32 (sums over positions in fp64); logits are rounded nowhere, gradients once, when they are
// stored in the logits' type.
#include "common.h"

#include <math.h>

namespace spice {
namespace {

constexpr int kTokThreads = 256;
constexpr int kTokChunk = 4096;      // positions of one workgroup of the passes over positions
constexpr int kTokFold = 1024;       // threads of the one workgroup that folds their partial sums

// The logits as the kernels see them: element strides of sequence, position and class.
struct Logits {
    const void *x;
    int64_t n, l, c;
    int64_t sn, sl, sc;
};

struct Labels {
    const int64_t *y;
    int64_t sn, sl;
    int64_t ignore;
};

// exp((x - m) / T) = exp2(d * k + d * k_lo), d = x - m.  k + k_lo is log2(e) / T to twice fp32's precision: the rounding
// of the constant alone would scale every exponent alike, and a sequence's log ratio, a small difference of thousands of
// log-probabilities, adds that bias up instead of averaging it out.
struct Temper {
    float k, k_lo, inv;
};

static Temper temper(float t) {
    const double k = 1.4426950408889634074 / (double)t;
    Temper r;
    r.k = (float)k;
    r.k_lo = (float)(k - (double)r.k);
    r.inv = (float)(1.0 / (double)t);
    return r;
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(__bf16 v) { return (float)v; }

__device__ __forceinline__ float exp_of(float d, Temper t) {
    return __builtin_amdgcn_exp2f(__builtin_fmaf(d, t.k, d * t.k_lo));
}

// ln s for s > 0: s = 2^e f with f in [sqrt(1/2), sqrt(2)), ln f = 2 atanh(t), t = (f - 1) / (f + 1), |t| < 0.1716, by its
// series up to t^9 / 9 (the next term is below 2^-29 of ln f), e ln 2 in two parts.  logf ends in the hardware's logarithm,
// whose error keeps one sign over a whole binade: the log ratio of 500 tokens was off by 1.9e-4 with it, 4e-6 with this.
__device__ __forceinline__ float log_of(float s) {
    int e;
    float f = frexpf(s, &e);
    if (f < 0.70710678f) {
        f += f;
        e -= 1;
    }
    if (!(s > 0.f) || s == INFINITY) return s == 0.f ? -INFINITY : s;   // (NaN, or an infinite sum: as it is)
    const float t = (f - 1.f) / (f + 1.f), q = t * t;
    float r = __builtin_fmaf(q, 1.f / 9.f, 1.f / 7.f);
    r = __builtin_fmaf(r, q, 1.f / 5.f);
    r = __builtin_fmaf(r, q, 1.f / 3.f);
    const float g = t + t, low = __builtin_fmaf(g * q, r, (float)e * 1.42860682e-6f);   // ln 2 - 0.693145751953125
    return __builtin_fmaf((float)e, 0.693145751953125f, g + low);
}

// What a position's label says.
enum { kCounted = 0, kIgnored = 1, kBad = 2 };
__device__ __forceinline__ int label_kind(int64_t y, int64_t ignore, int64_t c) {
    return y == ignore ? kIgnored : (y >= 0 && y < c) ? kCounted : kBad;
}

// A maximum to subtract: -inf (nothing finite seen) would make -inf - -inf out of an excluded class.
__device__ __forceinline__ float shift_of(float m) { return m == -INFINITY ? 0.f : m; }

// What a sum of exponentials over maximum m is worth over maximum `to` >= m: nothing where nothing finite was seen (its
// place holder 0 may lie far above `to`).
__device__ __forceinline__ float rescale(float m, float to, Temper t) { return m == -INFINITY ? 0.f : exp_of(m - to, t); }

// (m, s) of the workgroup from every thread's running maximum and sum; in every thread afterwards.
template <int THREADS>
__device__ __forceinline__ void fold_max_sum(float &m, float &s, Temper t, float *lds) {
    constexpr int waves = THREADS / kWave;
    float all = m;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor(all, o, kWave));
    s *= rescale(m, all, t);
    s = wave_sum(s);
    if (waves > 1) {
        __syncthreads();   // (the last fold's reads)
        if ((threadIdx.x & 63) == 0) {
            lds[threadIdx.x / kWave] = all;
            lds[waves + threadIdx.x / kWave] = s;
        }
        __syncthreads();
        float top = lds[0];
#pragma unroll
        for (int w = 1; w < waves; ++w) top = fmaxf(top, lds[w]);
        s = 0.f;
#pragma unroll
        for (int w = 0; w < waves; ++w) s += lds[waves + w] * rescale(lds[w], top, t);
        all = top;
    }
    m = all;
}

// The clipped policy loss of one position and its derivative by logp.
struct Policy {
    const float *old_logp, *adv, *ref;   // ref: NULL without a KL term
    int64_t adv_sn, adv_sl;
    float low, high, kl;                 // ratio bounds 1 - clip_low, 1 + clip_high; weight of the KL term
};

struct PolicyTerm {
    float surrogate, far, dlogp;
    bool over;
};

__device__ __forceinline__ PolicyTerm policy_term(const Policy &p, float logp, int64_t at, int64_t n, int64_t l) {
    PolicyTerm r;
    const float a = p.adv[n * p.adv_sn + l * p.adv_sl];
    const float ratio = expf(logp - p.old_logp[at]);
    const float free = ratio * a;
    const float held = fminf(fmaxf(ratio, p.low), p.high) * a;
    r.over = free > held;
    r.surrogate = r.over ? -held : -free;
    r.dlogp = r.over ? 0.f : -free;
    r.far = 0.f;
    if (p.ref) {
        const float q = p.ref[at] - logp;   // log of how much likelier the reference finds the label
        const float e = expf(q);
        r.far = e - q - 1.f;
        if (p.kl != 0.f) r.dlogp += p.kl * (1.f - e);
    }
    return r;
}

// ---- one position a workgroup, any strides ----

// LOGP: logp and (max, sum) of each position.  GRAD: weight * d logp / d x from them.  POLICY: logp, and the policy loss's
// gradient behind it.
enum { kModeLogp = 0, kModeGrad = 1, kModePolicy = 2, kModePolicyGrad = 3 };

struct TokArgs {
    Logits x;
    Labels y;
    Temper t;
    float *logp;            // [n, l]
    float2 *stats;          // [n, l] (max, sum), may be NULL
    const float2 *stats_in;
    const float *weight;    // kModeGrad: factor of each position
    int64_t w_sn, w_sl;
    const float *scale;     // device factor of the gradient, may be NULL
    int unless_one;         // nothing to do where that factor is 1
    float *weight_out;      // kModePolicy*: d loss / d logp of each position, may be NULL
    float host_scale;
    void *grad;
    int64_t g_sn, g_sl, g_sc;
    Policy policy;
    const float *share;     // [n] what a position of sequence n counts in the mean
};

template <typename T, int MODE>
__global__ __launch_bounds__(kTokThreads) void tok_any_kernel(TokArgs a) {
    __shared__ float lds[2 * kTokThreads / kWave];
    if (MODE == kModeGrad && a.unless_one && *a.scale == 1.f) return;
    const int64_t total = a.x.n * a.x.l;
    for (int64_t at = blockIdx.x; at < total; at += gridDim.x) {
        const int64_t n = at / a.x.l, l = at - n * a.x.l;
        const T *x = (const T *)a.x.x + n * a.x.sn + l * a.x.sl;
        const int64_t y = a.y.y[n * a.y.sn + l * a.y.sl];
        const int kind = label_kind(y, a.y.ignore, a.x.c);
        T *g = MODE == kModeGrad || MODE == kModePolicyGrad ? (T *)a.grad + n * a.g_sn + l * a.g_sl : nullptr;
        float m = -INFINITY, s = 0.f, logp = 0.f;
        if (MODE != kModeGrad) {
            if (kind == kCounted) {
                for (int64_t c = threadIdx.x; c < a.x.c; c += kTokThreads) {
                    const float v = to_f32(x[c * a.x.sc]);
                    if (v > m) {
                        s *= rescale(m, v, a.t);
                        m = v;
                    }
                    s += exp_of(v - shift_of(m), a.t);
                }
                fold_max_sum<kTokThreads>(m, s, a.t, lds);
                logp = (to_f32(x[y * a.x.sc]) - shift_of(m)) * a.t.inv - log_of(s);
            } else if (kind == kBad) {
                logp = NAN;
            }
            if (threadIdx.x == 0) {
                a.logp[at] = logp;
                if (a.stats) a.stats[at] = make_float2(m, s);
            }
        } else if (kind == kCounted) {
            const float2 st = a.stats_in[at];
            m = st.x;
            s = st.y;
        }
        if (MODE == kModeGrad || MODE == kModePolicyGrad) {
            float w = 0.f;
            if (kind == kBad)
                w = NAN;
            else if (kind == kCounted && MODE == kModeGrad)
                w = a.weight[n * a.w_sn + l * a.w_sl];
            else if (kind == kCounted)
                w = policy_term(a.policy, logp, at, n, l).dlogp * a.share[n];
            if (MODE == kModePolicyGrad && a.weight_out && threadIdx.x == 0) a.weight_out[at] = w;
            if (kind == kCounted) w *= a.t.inv * a.host_scale * (a.scale ? *a.scale : 1.f);
            const float each = kind == kCounted ? w / s : w;
            for (int64_t c = threadIdx.x; c < a.x.c; c += kTokThreads) {
                float v = kind == kIgnored ? 0.f : kind == kBad ? w : -each * exp_of(to_f32(x[c * a.x.sc]) - shift_of(m), a.t);
                if (kind == kCounted && c == y) v += w;
                g[c * a.g_sc] = (T)v;
            }
        }
    }
}

// ---- passes over positions ----

template <int K>
__device__ __forceinline__ void block_sums(double (&v)[K], double *lds, int threads) {
    const int waves = threads / kWave;
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = wave_sum(v[k]);
    if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int k = 0; k < K; ++k) lds[(threadIdx.x / kWave) * K + k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = 0.0;
    for (int w = 0; w < waves; ++w)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += lds[w * K + k];
    __syncthreads();
}

struct SumArgs {
    const float *logp;
    const float *ref;       // preference
    Labels y;
    int64_t n, l, c, chunks;
    Policy policy;
    double *part;           // [n, chunks, K]
};

// Positions counted of sequence blockIdx.y's chunk blockIdx.x, and their sums:
//   kSumCount: {count};  kSumPreference: {sum logp - ref, count};  kSumPolicy: {sum surrogate, sum far, clipped, count}.
enum { kSumCount = 0, kSumPreference = 1, kSumPolicy = 2 };
template <int WHAT>
constexpr int sum_terms() { return WHAT == kSumCount ? 1 : WHAT == kSumPreference ? 2 : 4; }

template <int WHAT>
__global__ __launch_bounds__(kTokThreads) void tok_sum_kernel(SumArgs a) {
    constexpr int K = sum_terms<WHAT>();
    __shared__ double lds[K * kTokThreads / kWave];
    for (int64_t item = blockIdx.x; item < a.n * a.chunks; item += gridDim.x) {
        const int64_t n = item / a.chunks, chunk = item - n * a.chunks;
        const int64_t end = min(a.l, (chunk + 1) * (int64_t)kTokChunk);
        double v[K];
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = 0.0;
        for (int64_t l = chunk * (int64_t)kTokChunk + threadIdx.x; l < end; l += kTokThreads) {
            const int64_t at = n * a.l + l;
            if (a.y.y[n * a.y.sn + l * a.y.sl] == a.y.ignore) continue;
            v[K - 1] += 1.0;
            if (WHAT == kSumPreference) v[0] += (double)a.logp[at] - (double)a.ref[at];
            if (WHAT == kSumPolicy) {
                const PolicyTerm t = policy_term(a.policy, a.logp[at], at, n, l);
                v[0] += t.surrogate;
                v[1 % K] += t.far;
                v[2 % K] += t.over ? 1.0 : 0.0;
            }
        }
        block_sums<K>(v, lds, kTokThreads);
        if (threadIdx.x == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) a.part[item * K + k] = v[k];
    }
}

// share[n]: what one position of sequence n counts in the mean over all counted positions (token), or in the mean over
// sequences of each one's mean.
__global__ __launch_bounds__(kTokFold) void tok_share_kernel(const double *part, int64_t n, int64_t chunks, int per_sequence,
                                                             float *share) {
    __shared__ double lds[kTokFold / kWave];
    double all = 0.0;
    if (!per_sequence) {
        double v[1] = {0.0};
        for (int64_t i = threadIdx.x; i < n * chunks; i += kTokFold) v[0] += part[i];
        block_sums<1>(v, lds, kTokFold);
        all = v[0];
    }
    for (int64_t i = threadIdx.x; i < n; i += kTokFold) {
        double count = all, weight = 1.0;
        if (per_sequence) {
            count = 0.0;
            weight = (double)n;
            for (int64_t k = 0; k < chunks; ++k) count += part[i * chunks + k];
        }
        share[i] = (float)(1.0 / (fmax(count, 1.0) * weight));
    }
}

struct PreferenceEnd {
    const double *part;     // [n, chunks, 2]
    int64_t n, chunks;
    float beta, smoothing;
    int ipo, average;
    float *total, *rewards, *weight;   // [1], [n], [n]: d total / d logp of every counted position of sequence n
};

__device__ __forceinline__ double sequence_total(const PreferenceEnd &e, int64_t i, double &count) {
    double sum = 0.0;
    count = 0.0;
    for (int64_t k = 0; k < e.chunks; ++k) {
        sum += e.part[(i * e.chunks + k) * 2];
        count += e.part[(i * e.chunks + k) * 2 + 1];
    }
    count = e.average ? fmax(count, 1.0) : 1.0;
    return sum / count;
}

// softplus(-x) = -log sigmoid(x), and sigmoid, without overflow on either side.
__device__ __forceinline__ double minus_log_sigmoid(double x) { return log1p(exp(-fabs(x))) + fmax(-x, 0.0); }
__device__ __forceinline__ double sigmoid(double x) {
    const double e = exp(-fabs(x));
    return x >= 0.0 ? 1.0 / (1.0 + e) : e / (1.0 + e);
}

__global__ __launch_bounds__(kTokFold) void tok_preference_kernel(PreferenceEnd e) {
    __shared__ double lds[kTokFold / kWave];
    const int64_t half = e.n / 2;
    double v[1] = {0.0};
    for (int64_t i = threadIdx.x; i < half; i += kTokFold) {
        double na, nb;
        const double sa = sequence_total(e, i, na), sb = sequence_total(e, half + i, nb);
        const double h = sa - sb, b = (double)e.beta, eps = (double)e.smoothing;
        double dh;
        if (e.ipo) {
            const double off = h - 0.5 / b;
            v[0] += off * off;
            dh = 2.0 * off;
        } else {
            v[0] += (1.0 - eps) * minus_log_sigmoid(b * h) + (eps != 0.0 ? eps * minus_log_sigmoid(-b * h) : 0.0);
            dh = -b * ((1.0 - eps) * sigmoid(-b * h) - eps * sigmoid(b * h));
        }
        e.rewards[i] = (float)(b * sa);
        e.rewards[half + i] = (float)(b * sb);
        e.weight[i] = (float)(dh / (double)half / na);
        e.weight[half + i] = (float)(-dh / (double)half / nb);
    }
    block_sums<1>(v, lds, kTokFold);
    if (threadIdx.x == 0) *e.total = (float)(v[0] / (double)half);
}

// out4 = {total, surrogate, kl, share of the counted positions where the clipping holds}
__global__ __launch_bounds__(kTokFold) void tok_policy_end_kernel(const double *part, int64_t n, int64_t chunks, const float *share,
                                                                  float kl, float *out4) {
    __shared__ double lds[4 * kTokFold / kWave];
    double v[4] = {0.0, 0.0, 0.0, 0.0};
    for (int64_t i = threadIdx.x; i < n * chunks; i += kTokFold) {
        const double each = (double)share[i / chunks];
        v[0] += part[i * 4] * each;
        v[1] += part[i * 4 + 1] * each;
        v[2] += part[i * 4 + 2];
        v[3] += part[i * 4 + 3];
    }
    block_sums<4>(v, lds, kTokFold);
    if (threadIdx.x == 0) {
        out4[0] = (float)(kl != 0.f ? v[0] + (double)kl * v[1] : v[0]);
        out4[1] = (float)v[0];
        out4[2] = (float)v[1];
        out4[3] = (float)(v[2] / fmax(v[3], 1.0));
    }
}

int64_t chunks_of(int64_t l) { return l > kTokChunk ? ceil_div(l, kTokChunk) : 1; }
unsigned grid_of(int64_t blocks) { return (unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)); }

bool logits_ok(const spice_logits *x) {
    return x && x->n >= 0 && x->l >= 0 && x->c >= 1 && x->dtype >= 0 && x->dtype <= 2 &&
           (x->data || x->n == 0 || x->l == 0) &&
           (x->n == 0 || x->l <= ((int64_t)1 << 40) / x->n);
}

bool labels_ok(const spice_logits *x, const spice_labels *y) {
    return y && (y->data || x->n == 0 || x->l == 0) && (y->ignore_index < 0 || y->ignore_index >= x->c);
}

bool temperature_ok(float t) { return t > 0.f && t <= 3.0e38f && 1.f / t <= 3.0e38f; }

TokArgs args_of(const spice_logits *x, const spice_labels *y, float t) {
    TokArgs a = {};
    a.x = Logits{x->data, x->n, x->l, x->c, x->n_stride, x->l_stride, x->c_stride};
    a.y = Labels{y->data, y->n_stride, y->l_stride, y->ignore_index};
    a.t = temper(t);
    a.host_scale = 1.f;
    return a;
}

// The gradient is dense, in the logits' own order of axes.
void grad_layout(TokArgs &a, void *grad, int32_t class_last) {
    a.grad = grad;
    a.g_sn = a.x.l * a.x.c;
    a.g_sl = class_last ? a.x.c : 1;
    a.g_sc = class_last ? 1 : a.x.l;
}

template <int MODE>
int launch_positions(const TokArgs &a, int32_t dtype, hipStream_t stream) {
    const int64_t total = a.x.n * a.x.l;
    if (total == 0) return SPICE_OK;
    const unsigned grid = grid_of(total);
    if (dtype == 0)
        tok_any_kernel<float, MODE><<<grid, kTokThreads, 0, stream>>>(a);
    else if (dtype == 1)
        tok_any_kernel<_Float16, MODE><<<grid, kTokThreads, 0, stream>>>(a);
    else
        tok_any_kernel<__bf16, MODE><<<grid, kTokThreads, 0, stream>>>(a);
    SPICE_LAUNCH_CHECK();
    return SPICE_OK;
}

SumArgs sums_of(const TokArgs &a, double *part) {
    SumArgs s = {};
    s.logp = a.logp;
    s.y = a.y;
    s.n = a.x.n;
    s.l = a.x.l;
    s.c = a.x.c;
    s.chunks = chunks_of(a.x.l);
    s.policy = a.policy;
    s.part = part;
    return s;
}

template <int WHAT>
int launch_sums(const SumArgs &s, hipStream_t stream) {
    if (s.n == 0) return SPICE_OK;
    tok_sum_kernel<WHAT><<<grid_of(s.n * s.chunks), kTokThreads, 0, stream>>>(s);
    SPICE_LAUNCH_CHECK();
    return SPICE_OK;
}

}  // namespace
}  // namespace spice

using namespace spice;

extern "C" size_t spice_token_loss_workspace_bytes(int64_t n, int64_t l) {
    if (n < 0 || l < 0) return 0;
    return (size_t)(n * chunks_of(l) * 4 * (int64_t)sizeof(double) + ((n + 1) / 2) * 8 + 64);
}

extern "C" int spice_token_logprobs(const spice_logits *x, const spice_labels *y, float temperature, float *logp, float *stats,
                                    void *stream) {
    if (!logits_ok(x) || !labels_ok(x, y) || !temperature_ok(temperature) || (!logp && x->n * x->l) || !aligned8(stats))
        return SPICE_ERR_ARG;
    TokArgs a = args_of(x, y, temperature);
    a.logp = logp;
    a.stats = (float2 *)stats;
    return launch_positions<kModeLogp>(a, x->dtype, (hipStream_t)stream);
}

extern "C" int spice_token_logprobs_grad(const spice_logits *x, const spice_labels *y, float temperature, const float *stats,
                                         const float *weight, int64_t w_n_stride, int64_t w_l_stride, float scale,
                                         const float *device_scale, int32_t unless_one, int32_t class_last, void *grad,
                                         void *stream) {
    if (!logits_ok(x) || !labels_ok(x, y) || !temperature_ok(temperature) || !aligned8(stats) || (unless_one && !device_scale) ||
        ((!stats || !weight || !grad) && x->n * x->l))
        return SPICE_ERR_ARG;
    TokArgs a = args_of(x, y, temperature);
    a.stats_in = (const float2 *)stats;
    a.weight = weight;
    a.w_sn = w_n_stride;
    a.w_sl = w_l_stride;
    a.host_scale = scale;
    a.scale = device_scale;
    a.unless_one = unless_one;
    grad_layout(a, grad, class_last);
    return launch_positions<kModeGrad>(a, x->dtype, (hipStream_t)stream);
}

extern "C" int spice_preference_loss(const spice_logits *x, const spice_labels *y, const float *ref_logp,
                                     const spice_preference_params *p, float *total, float *rewards, float *weight, float *logp,
                                     float *stats, void *workspace, size_t workspace_bytes, void *stream) {
    if (!logits_ok(x) || !labels_ok(x, y) || !p || x->n < 2 || x->n % 2 || !total || !rewards || !weight || !workspace ||
        !aligned8(workspace) || ((!ref_logp || !logp) && x->l) || !aligned8(stats) || !(p->beta > 0.f) ||
        !(p->smoothing >= 0.f && p->smoothing < 0.5f) || p->loss_type < 0 || p->loss_type > 1 ||
        (p->loss_type == SPICE_PREFERENCE_IPO && p->smoothing != 0.f) || !temperature_ok(p->temperature))
        return SPICE_ERR_ARG;
    if (workspace_bytes < spice_token_loss_workspace_bytes(x->n, x->l)) return SPICE_ERR_WORKSPACE;
    hipStream_t s = (hipStream_t)stream;
    TokArgs a = args_of(x, y, p->temperature);
    a.logp = logp;
    a.stats = (float2 *)stats;
    int rc = launch_positions<kModeLogp>(a, x->dtype, s);
    if (rc) return rc;
    SumArgs sums = sums_of(a, (double *)workspace);
    sums.ref = ref_logp;
    rc = launch_sums<kSumPreference>(sums, s);
    if (rc) return rc;
    PreferenceEnd e = {sums.part, x->n, sums.chunks, p->beta, p->smoothing, p->loss_type == SPICE_PREFERENCE_IPO, p->average != 0,
                       total, rewards, weight};
    tok_preference_kernel<<<1, kTokFold, 0, s>>>(e);
    SPICE_LAUNCH_CHECK();
    return SPICE_OK;
}

extern "C" int spice_policy_loss(const spice_logits *x, const spice_labels *y, const float *old_logp, const float *advantages,
                                 int64_t adv_n_stride, int64_t adv_l_stride, const float *ref_logp, const spice_policy_params *p,
                                 float *out4, float *logp, float *stats, float *weight, int32_t class_last, void *grad,
                                 void *workspace, size_t workspace_bytes, void *stream) {
    if (!logits_ok(x) || !labels_ok(x, y) || !p || !out4 || !workspace || !aligned8(workspace) ||
        ((!old_logp || !advantages || !logp) && x->n * x->l) || !(p->clip_low >= 0.f && p->clip_low <= 1.f) ||
        !(p->clip_high >= 0.f) || !(p->kl_weight >= 0.f) || (p->kl_weight > 0.f && !ref_logp && x->n * x->l) ||
        p->reduction < 0 || p->reduction > 1 || !aligned8(stats) || !temperature_ok(p->temperature))
        return SPICE_ERR_ARG;
    if (workspace_bytes < spice_token_loss_workspace_bytes(x->n, x->l)) return SPICE_ERR_WORKSPACE;
    hipStream_t s = (hipStream_t)stream;
    TokArgs a = args_of(x, y, p->temperature);
    a.logp = logp;
    a.stats = (float2 *)stats;
    a.weight_out = weight;
    a.host_scale = p->grad_scale;
    a.policy = Policy{old_logp, advantages, ref_logp, adv_n_stride, adv_l_stride, 1.f - p->clip_low, 1.f + p->clip_high,
                      p->kl_weight};
    SumArgs sums = sums_of(a, (double *)workspace);
    float *share = (float *)((double *)workspace + x->n * sums.chunks * 4);
    a.share = share;
    int rc = launch_sums<kSumCount>(sums, s);
    if (rc) return rc;
    tok_share_kernel<<<1, kTokFold, 0, s>>>(sums.part, x->n, sums.chunks, p->reduction == SPICE_POLICY_SEQUENCE, share);
    SPICE_LAUNCH_CHECK();
    if (grad) {
        grad_layout(a, grad, class_last);
        rc = launch_positions<kModePolicyGrad>(a, x->dtype, s);
    } else {
        rc = launch_positions<kModePolicy>(a, x->dtype, s);
    }
    if (rc) return rc;
    rc = launch_sums<kSumPolicy>(sums, s);
    if (rc) return rc;
    tok_policy_end_kernel<<<1, kTokFold, 0, s>>>(sums.part, x->n, sums.chunks, share, p->kl_weight, out4);
    SPICE_LAUNCH_CHECK();
    return SPICE_OK;
}
