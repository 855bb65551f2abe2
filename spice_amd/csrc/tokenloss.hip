// Losses over the log-probabilities of given labels: label log-probabilities with their gradient, the preference loss
// (paired log ratios against a reference policy) and the clipped policy loss with a KL term.
//
// Positions (n, l) of N sequences (or pictures) of L labels each carry C logits x_c.  With z = x / T, m = max x and
// s = sum_c exp((x_c - m) / T):
//   logp = (x_label - m) / T - log s,      d logp / d x_c = ([c == label] - exp((x_c - m) / T) / s) / T.
// Logits are rounded nowhere; an exponential is fp32, a sum of them short fp32 trees or chains (four roundings at most)
// joined in fp64, a label's log-probability, a log ratio and what is summed over positions fp64; what leaves (logp, the
// statistics, the factor of a position's gradient) rounds to fp32, and gradients once, when they are stored in the logits'
// type.  (One fp32 chain a lane loses what lies 2^-25 below its sum; the trees cost 0 to 3 % of a forward pass over it, every
// exponential added in fp64 by itself 5 to 16 %.)
#include "common.h"

#include <math.h>

namespace spice {
namespace {

constexpr int kTokThreads = 256;
constexpr int kTokChunk = 2048;      // positions of one workgroup of the passes over positions
constexpr int kTokFold = 1024;       // threads of the one workgroup that folds their partial sums
constexpr int64_t kTokCount = 2048;  // positions that every workgroup counts for itself: a launch less ([1,7,32000] fp16: 14.8 us, 17.4 with)
constexpr int64_t kTokHere = 4096;   // positions that this workgroup sums itself: 4 a thread

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
    double exact_inv;
};

static Temper temper(double t) {
    const double k = 1.4426950408889634074 / t;
    Temper r;
    r.k = (float)k;
    if ((double)r.k >= k) r.k = nextafterf(r.k, 0.f);   // k_lo > 0: an excluded class's d = -inf stays -inf in both products
    r.k_lo = (float)(k - (double)r.k);
    r.exact_inv = 1.0 / t;
    r.inv = (float)r.exact_inv;
    return r;
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(__bf16 v) { return (float)v; }

__device__ __forceinline__ float exp_of(float d, Temper t) {
    return __builtin_amdgcn_exp2f(__builtin_fmaf(d, t.k, d * t.k_lo));
}

// ln s for s > 0, in fp64: s = 2^e f with f in [sqrt(1/2), sqrt(2)), ln f = 2 atanh(t), t = (f - 1) / (f + 1), |t| < 0.1716,
// by its series up to t^9 / 9 (the next term is below 2^-29 of ln f); the terms behind 2 t in fp32.  logf ends in the
// hardware's logarithm, whose error keeps one sign over a whole binade: the log ratio of 500 tokens was off by 1.9e-4 with it.
__device__ __forceinline__ double log_of(float s) {
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
    // t to fp64's precision: one Newton step of the quotient
    const double num = (double)f - 1.0, den = (double)f + 1.0, exact = (double)t + (num - (double)t * den) * (double)(1.f / (f + 1.f));
    return (double)e * 0.69314718055994530942 + (2.0 * exact + (double)(2.f * t * q * r));
}

// A label's log-probability from its logit, the maximum and the sum, in fp64: a sequence's log ratio is a small difference of
// thousands of them, and rounding each, or the logit's distance to the maximum, to fp32 (2^-22 at 4 to 8) would show in it.
__device__ __forceinline__ double logp_of(float xl, float shift, double s, Temper t) {
    const float near = (float)s;
    const double rest = near > 0.f && near < INFINITY ? (s - (double)near) / s : 0.0;
    return ((double)xl - (double)shift) * t.exact_inv - (log_of(near) + rest);
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

// The sum of K exponentials as a tree, log2 K roundings deep.  A row's trees add up in fp64: a sum that has reached 1 in fp32
// takes up no class below 2^-25 of it (255 classes 17 below the top in chains of four lanes: a quarter of 1 - p lost).
template <int K>
__device__ __forceinline__ double tree_sum(float (&e)[K]) {
#pragma unroll
    for (int o = K / 2; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < o; ++k) e[k] += e[k + o];
    return (double)e[0];
}

// The sum of exponentials of a row beyond fp32's precision: what the logarithm is taken of.
__device__ __forceinline__ double wide_sum(double v, int lanes) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        if (o < lanes) v += __shfl_xor(v, o, kWave);
    return v;
}

// (m, s) of the workgroup from every thread's running maximum and sum; in every thread afterwards.
template <int THREADS>
__device__ __forceinline__ double fold_max_sum(float &m, double s, Temper t, double *lds) {
    constexpr int waves = THREADS / kWave;
    float all = m;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor(all, o, kWave));
    double sum = wide_sum(s * (double)rescale(m, all, t), kWave);
    if (waves > 1) {
        __syncthreads();   // (the last fold's reads)
        if ((threadIdx.x & 63) == 0) {
            lds[threadIdx.x / kWave] = sum;
            lds[waves + threadIdx.x / kWave] = (double)all;
        }
        __syncthreads();
        // every lane takes one wave's pair: all of them in every thread cost 16 exponentials a thread, 2 us of a row
        const int w = threadIdx.x & (waves - 1);
        const float mine = (float)lds[waves + w];
        float top = mine;
#pragma unroll
        for (int o = waves / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, kWave));
        sum = wide_sum(lds[w] * (double)rescale(mine, top, t), waves);
        all = top;
    }
    m = all;
    return sum;
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

// What a position brings along: read early, so that nothing waits for it behind the logits' sums.
struct PolicyIn {
    float adv, old_logp, ref;
};

__device__ __forceinline__ PolicyIn policy_in(const Policy &p, int64_t at, int64_t n, int64_t l) {
    return PolicyIn{p.adv[n * p.adv_sn + l * p.adv_sl], p.old_logp[at], p.ref ? p.ref[at] : 0.f};
}

// exp(q) - q - 1 and exp(q) - 1.  Where a policy has hardly left its reference the first is about q^2 / 2, which differences of
// numbers near 1 would round to steps of 2^-24 (2^21 positions 1e-4 apart: a mean of -4e-9 for 5e-9): for |q| <= 1 its series,
// q^2 sum_n q^n / (n + 2)! up to q^11 / 11! (the next term is below 2^-27 of it).
__device__ __forceinline__ void far_of(float q, float &far, float &e1) {
    if (fabsf(q) <= 1.f) {
        float r = 1.f / 39916800.f;
        r = __builtin_fmaf(r, q, 1.f / 3628800.f);
        r = __builtin_fmaf(r, q, 1.f / 362880.f);
        r = __builtin_fmaf(r, q, 1.f / 40320.f);
        r = __builtin_fmaf(r, q, 1.f / 5040.f);
        r = __builtin_fmaf(r, q, 1.f / 720.f);
        r = __builtin_fmaf(r, q, 1.f / 120.f);
        r = __builtin_fmaf(r, q, 1.f / 24.f);
        r = __builtin_fmaf(r, q, 1.f / 6.f);
        r = __builtin_fmaf(r, q, 0.5f);
        far = q * q * r;
        e1 = q + far;
    } else {
        e1 = expf(q) - 1.f;
        far = e1 - q;
    }
}

__device__ __forceinline__ PolicyTerm policy_term(const Policy &p, const PolicyIn &in, float logp) {
    PolicyTerm r;
    const float a = in.adv;
    const float moved = logp - in.old_logp, ratio = expf(moved);
    const float free = a == 0.f && moved < INFINITY ? 0.f : ratio * a;   // (a ratio past fp32's range is finite all the same)
    const float held = fminf(fmaxf(ratio, p.low), p.high) * a;
    r.over = free > held;
    r.surrogate = r.over ? -held : -free;
    r.dlogp = r.over ? 0.f : -free;
    r.far = 0.f;
    if (p.ref) {
        const float q = in.ref - logp;   // log of how much likelier the reference finds the label
        float e1;                        // exp(q) - 1
        far_of(q, r.far, e1);
        if (p.kl != 0.f) r.dlogp -= p.kl * e1;
    }
    return r;
}

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

struct TokArgs {
    Logits x;
    Labels y;
    Temper t;
    float *logp;            // [n, l], may be NULL
    double *ratio;          // [n, l] logp - ref, may be NULL
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
    const float *ref;       // kModePreference
    const float *share;     // [n] what a position of sequence n counts in the mean; NULL: counted where it is needed
    int per_sequence;
    double *part;           // sums of each workgroup's item
};

// What a position leaves: its log-probability, or the preference loss's log ratio, and its statistics.
__device__ __forceinline__ void leave_logp(const TokArgs &a, int64_t at, double logp, float m, float s, float ref) {
    if (a.logp) a.logp[at] = (float)logp;
    if (a.ratio) a.ratio[at] = logp - (double)ref;   // (where ignored it is not read)
    if (a.stats) a.stats[at] = make_float2(m, s);
}

// What a position of sequence n counts in the mean, from the labels: THREADS threads count all of them (few: kTokCount),
// a wave by itself or a workgroup with `lds`.
template <int THREADS>
__device__ __forceinline__ float share_here(const TokArgs &a, int64_t n, int *lds) {
    const int64_t first = a.per_sequence ? n * a.x.l : 0, end = a.per_sequence ? first + a.x.l : a.x.n * a.x.l;
    int count = 0;
    for (int64_t i = first + threadIdx.x % THREADS; i < end; i += THREADS) {
        const int64_t k = (uint32_t)i / (uint32_t)a.x.l;
        count += a.y.y[k * a.y.sn + (i - k * a.x.l) * a.y.sl] != a.y.ignore;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) count += __shfl_xor(count, o, kWave);
    if (THREADS > kWave) {
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x / kWave] = count;
        __syncthreads();
        count = 0;
#pragma unroll
        for (int w = 0; w < THREADS / kWave; ++w) count += lds[w];
    }
    return (float)(1.0 / ((double)(count > 1 ? count : 1) * (a.per_sequence ? (double)a.x.n : 1.0)));
}

// ---- one position a workgroup, any strides ----

// Logp: logp and (max, sum) of each position.  Grad: weight * d logp / d x from them.  Preference, Policy: logp, and what the
// loss sums over positions.  PolicyGrad: the policy loss's gradient behind that.
enum { kModeLogp = 0, kModeGrad = 1, kModePreference = 2, kModePolicy = 3, kModePolicyGrad = 4 };

// For few positions of many classes at any stride, where a workgroup a position is what fills the chip (route_of); bound by
// latency: one pass for maximum and sum, a second over the same lines for the gradient.  fp32 [1,3001,256] planes: forward
// 8.4 us, gradient 16, policy loss with both and its end launch 28.
template <typename T, int MODE>
__global__ __launch_bounds__(kTokThreads) void tok_any_kernel(TokArgs a) {
    __shared__ double lds[2 * kTokThreads / kWave];
    __shared__ int counts[kTokThreads / kWave];
    if (MODE == kModeGrad && a.unless_one && *a.scale == 1.f) return;
    const int64_t total = a.x.n * a.x.l;
    for (int64_t at = blockIdx.x; at < total; at += gridDim.x) {
        const int64_t n = at / a.x.l, l = at - n * a.x.l;
        const T *x = (const T *)a.x.x + n * a.x.sn + l * a.x.sl;
        const int64_t y = a.y.y[n * a.y.sn + l * a.y.sl];
        const int kind = label_kind(y, a.y.ignore, a.x.c);
        T *g = MODE == kModeGrad || MODE == kModePolicyGrad ? (T *)a.grad + n * a.g_sn + l * a.g_sl : nullptr;
        float m = -INFINITY, s = 0.f;
        double logp = 0.0;
        if (MODE != kModeGrad) {
            if (kind == kCounted) {
                double own = 0.0;
                for (int64_t c = threadIdx.x; c < a.x.c; c += kTokThreads) {
                    const float v = to_f32(x[c * a.x.sc]);
                    if (v > m) {
                        own *= (double)rescale(m, v, a.t);
                        m = v;
                    }
                    own += (double)exp_of(v - shift_of(m), a.t);
                }
                const double sum = fold_max_sum<kTokThreads>(m, own, a.t, lds);
                logp = logp_of(to_f32(x[y * a.x.sc]), shift_of(m), sum, a.t);
                s = (float)sum;
            } else if (kind == kBad) {
                logp = NAN;
            }
            if (threadIdx.x == 0) leave_logp(a, at, logp, m, s, a.ratio ? a.ref[at] : 0.f);
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
                w = policy_term(a.policy, policy_in(a.policy, at, n, l), (float)logp).dlogp *
                    (a.share ? a.share[n] : share_here<kTokThreads>(a, n, counts));
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

// ---- classes next to each other in memory: LANES lanes hold a row in registers ----

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
struct __attribute__((packed, aligned(2))) Vec16 { u32x4 v; };   // 16 bytes at any element's address

template <typename T> constexpr int vec_elements() { return 16 / (int)sizeof(T); }

__device__ __forceinline__ void unpack(u32x4 r, float (&v)[4], float) {
    typedef float f4 __attribute__((ext_vector_type(4)));
    const f4 f = __builtin_bit_cast(f4, r);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = f[k];
}
__device__ __forceinline__ void unpack(u32x4 r, float (&v)[8], _Float16) {
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    const h8 h = __builtin_bit_cast(h8, r);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = (float)h[k];
}
__device__ __forceinline__ void unpack(u32x4 r, float (&v)[8], __bf16) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const unsigned low = r[k] << 16, high = r[k] & 0xffff0000u;   // (bfloat16 is fp32's upper half)
        v[2 * k] = __builtin_bit_cast(float, low);
        v[2 * k + 1] = __builtin_bit_cast(float, high);
    }
}

template <typename T, int K>
__device__ __forceinline__ u32x4 pack(const float (&v)[K]) {
    typedef T tk __attribute__((ext_vector_type(K)));
    tk t;
#pragma unroll
    for (int k = 0; k < K; ++k) t[k] = (T)v[k];
    return __builtin_bit_cast(u32x4, t);
}

template <typename T>
__device__ __forceinline__ u32x4 load_vec(const T *p, int32_t left) {
    constexpr int K = vec_elements<T>();
    if (left >= K) return reinterpret_cast<const Vec16 *>(p)->v;
    float v[K];     // the row's last classes, or none of them, and -inf behind: they add nothing
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = k < left ? to_f32(p[k]) : -INFINITY;
    return pack<T, K>(v);
}

// ONCE: nothing reads these logits again (the policy loss takes its gradient in the same pass): past the caches, so that
// they displace nothing.  The other passes leave them in the memory-side cache for the gradient pass.
template <bool ONCE, typename T>
__device__ __forceinline__ u32x4 read_vec(const T *p) {
    const Vec16 *at = reinterpret_cast<const Vec16 *>(p);
    return ONCE ? __builtin_nontemporal_load(&at->v) : at->v;
}

// Gradients are stored past the caches: through them, a gradient's 256 MB of dirty lines in the memory-side cache were
// written back under the next call's reads ([8,1024,32000] bf16, loss + gradient: 240 us, 198 with these stores).
template <bool ONCE, typename T, int K>
__device__ __forceinline__ void store_vec(T *p, int32_t left, const float (&v)[K]) {
    if (left >= K) {
        if (ONCE)
            __builtin_nontemporal_store(pack<T, K>(v), &reinterpret_cast<Vec16 *>(p)->v);
        else
            reinterpret_cast<Vec16 *>(p)->v = pack<T, K>(v);
        return;
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (k < left) p[k] = (T)v[k];
}

// The gradient of K classes from c0 on.
template <int K>
__device__ __forceinline__ void grad_of(float (&v)[K], float m, float each, float w, int32_t y, int32_t c0, Temper t) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = each * exp_of(v[k] - m, t);
    if ((uint32_t)(y - c0) < (uint32_t)K) {
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = y - c0 == k ? v[k] + w : v[k];   // (+ 0 elsewhere would make -0 of a softmax of 0 a +0,
                                                                            // and a class that two lanes store is one value)
    }
}

// (m, s) of LANES neighbouring lanes; LANES > 64: of the workgroup.
template <int LANES>
__device__ __forceinline__ double fold_row(float &m, double s, Temper t, double *lds) {
    if (LANES <= kWave) {
        float all = m;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor(all, o, kWave));
        const double sum = wide_sum(s * (double)rescale(m, all, t), LANES);
        m = all;
        return sum;
    }
    return fold_max_sum<LANES>(m, s, t, lds);
}

// The packed row is all that is kept from one phase to the next: unpacked values that the compiler would carry along
// take twice the registers for 16-bit logits.
template <int NV>
__device__ __forceinline__ void forget(u32x4 (&raw)[NV]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) asm volatile("" : "+v"(raw[i]));
}

// A row is read once, as 16-byte loads at whatever address it starts, and stays packed in registers: maximum, exponentials
// and gradient are taken from there, so the bytes of the logits (and of the gradient) bound it.  LANES and NV: launch_rows.
// bf16, 5.9 TB/s being the card's large copy:
//   [1,1,32000] forward 5.0 us (one workgroup: a load, two barriers);   [8,1024,32000] forward 104 us (5.0 TB/s);
//   [4,1023,50001] forward 65 us, a third of the rows ignored (4.1 TB/s: rows start at odd addresses);
//   [8,512,131072] policy loss, logits in and gradient out, two fifths ignored, 307 us (5.5 TB/s; one row fills a compute
//   unit's registers, so its loads do not run under the last row's stores).
// A wave's fixed work (labels, fold, logarithm: about 1000 cycles) bounds rows of under 256 classes: 2^20 of 21 bf16 classes
// take 33 us where their bytes are 7.
//
// Vector i of lane j holds the classes from (i LANES + j) K on: the first `whole` are full in every lane (the same count in
// all of them), the one behind is ragged: it reaches back (value by value, bf16, 894,784 rows of 150: policy loss 205 us, 154
// so), or is filled up with -inf.  Fewer than 64 lanes: several rows a wave.
template <typename T, int LANES, int NV, int MODE>
__global__ __launch_bounds__(LANES < kTokThreads ? kTokThreads : LANES, NV <= 8 ? 6 : 4) void tok_row_kernel(TokArgs a, int64_t first) {
    constexpr int K = vec_elements<T>();
    constexpr int kBlock = LANES < kTokThreads ? kTokThreads : LANES;
    constexpr bool kGrad = MODE == kModeGrad || MODE == kModePolicyGrad, kStats = MODE == kModeGrad;
    constexpr bool kLong = LANES >= kWave;     // rows of many lines each, read and stored past the caches
    __shared__ double lds[2 * kBlock / kWave];
    __shared__ int counts[kBlock / kWave];
    if (kStats && a.unless_one && *a.scale == 1.f) return;
    float share = 0.f;
    if constexpr (MODE == kModePolicyGrad && !kLong)      // (all of the workgroup's waves are here)
        if (!a.share) share = share_here<kTokThreads>(a, 0, counts);
    const int row = kLong ? __builtin_amdgcn_readfirstlane(threadIdx.x / LANES) : threadIdx.x / LANES;
    const int64_t at = first + (int64_t)blockIdx.x * (kBlock / LANES) + row;
    if (at >= a.x.n * a.x.l) return;
    const int32_t lane = threadIdx.x % LANES, classes = (int32_t)a.x.c, whole = classes / (LANES * K);
    const int32_t tail = (whole * LANES + lane) * K, left = classes - tail;
    // the row's last classes, fewer than a vector: the row's last K instead, whose first `again` are another lane's too
    const int32_t again = left > 0 && left < K && classes >= K ? K - left : 0, from = tail - again;
    const int64_t n = at / a.x.l, l = at - n * a.x.l;
    const T *x = (const T *)a.x.x + n * a.x.sn + l * a.x.sl;
    const int64_t y = a.y.y[n * a.y.sn + l * a.y.sl];
    const float ref = !kGrad && a.ratio ? a.ref[at] : 0.f;
    PolicyIn in = {};
    if (MODE == kModePolicyGrad) in = policy_in(a.policy, at, n, l);
    const int kind = label_kind(y, a.y.ignore, a.x.c);
    float m = -INFINITY, s = 0.f;
    double logp = kind == kBad ? NAN : 0.0;
    u32x4 raw[NV], last;
    if (kind == kCounted) {
        const T *mine = x + lane * K;
        const float xl = kStats ? 0.f : to_f32(x[y]);
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (i < whole) raw[i] = read_vec<MODE == kModePolicyGrad && kLong>(mine + i * LANES * K);
        last = load_vec<T>(x + from, left + again);
        if constexpr (kStats) {
            const float2 st = a.stats_in[at];
            m = st.x;
            s = st.y;
        } else {
            if (MODE == kModePolicyGrad) {      // (under the logits' loads)
                if constexpr (kLong)
                    share = a.share ? a.share[n] : share_here<LANES>(a, n, counts);
                else if (a.share)
                    share = a.share[n];
            }
            float v[K];
            unpack(last, v, T());
#pragma unroll
            for (int k = 0; k < K; ++k) m = fmaxf(m, v[k]);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (i < whole) {
                    unpack(raw[i], v, T());
#pragma unroll
                    for (int k = 0; k < K; ++k) m = fmaxf(m, v[k]);
                }
            const float shift = shift_of(m);
            forget<NV>(raw);
            unpack(last, v, T());
#pragma unroll
            for (int k = 0; k < K; ++k) v[k] = k < again ? 0.f : exp_of(v[k] - shift, a.t);
            double own = tree_sum(v);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (i < whole) {
                    unpack(raw[i], v, T());
#pragma unroll
                    for (int k = 0; k < K; ++k) v[k] = exp_of(v[k] - shift, a.t);
                    own += tree_sum(v);
                }
            const double sum = fold_row<LANES>(m, own, a.t, lds);
            if (kGrad || lane == 0) logp = logp_of(xl, shift_of(m), sum, a.t);
            s = (float)sum;
        }
    }
    if (!kStats && lane == 0) leave_logp(a, at, logp, m, s, ref);
    if (kGrad) {
        T *g = (T *)a.grad + n * a.g_sn + l * a.g_sl;
        float w = kind == kBad ? NAN : 0.f;
        if (kind == kCounted)
            w = kStats ? a.weight[n * a.w_sn + l * a.w_sl] : policy_term(a.policy, in, (float)logp).dlogp * share;
        if (!kStats && a.weight_out && lane == 0) a.weight_out[at] = w;
        const float shift = shift_of(m);
        if (kind == kCounted) w *= a.t.inv * a.host_scale * (kStats && a.scale ? *a.scale : 1.f);   // (elsewhere 0 under any factor)
        const float each = kind == kCounted ? -w / s : w;
        float v[K];
        if (kind == kCounted) {
            T *mine = g + lane * K;
            forget<NV>(raw);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (i < whole) {
                    unpack(raw[i], v, T());
                    grad_of<K>(v, shift, each, w, (int32_t)y, (i * LANES + lane) * K, a.t);
                    store_vec<kLong>(mine + i * LANES * K, K, v);
                }
            unpack(last, v, T());
            grad_of<K>(v, shift, each, w, (int32_t)y, from, a.t);
            if (left > 0) store_vec<kLong>(g + from, left + again, v);      // (two lanes store the same values there)
        } else {
#pragma unroll
            for (int k = 0; k < K; ++k) v[k] = each;
            for (int32_t c0 = lane * K; c0 < classes; c0 += LANES * K) store_vec<kLong>(g + c0, classes - c0, v);
        }
    }
}

// Rows longer than the registers of a workgroup: four vectors a thread at a time, the maximum and sum running along (one
// rescaling a step), and for the gradient read again, mostly from the memory-side cache.  Bound by the bytes: bf16
// [1,4096,200000] forward 405 us (4.0 TB/s: each step's loads wait for the step before), policy loss 819 (the logits twice and
// the gradient: 6.0 TB/s).
template <typename T, int MODE>
__global__ __launch_bounds__(1024) void tok_long_row_kernel(TokArgs a) {
    constexpr int K = vec_elements<T>(), kBlock = 1024, kStep = 4;
    constexpr bool kGrad = MODE == kModePolicyGrad;
    __shared__ double lds[2 * kBlock / kWave];
    __shared__ int counts[kBlock / kWave];
    const int64_t total = a.x.n * a.x.l;
    const int32_t classes = (int32_t)a.x.c;
    for (int64_t at = blockIdx.x; at < total; at += gridDim.x) {
        const int64_t n = at / a.x.l, l = at - n * a.x.l;
        const T *x = (const T *)a.x.x + n * a.x.sn + l * a.x.sl;
        const int64_t y = a.y.y[n * a.y.sn + l * a.y.sl];
        const float ref = !kGrad && a.ratio ? a.ref[at] : 0.f;
        PolicyIn in = {};
        if (kGrad) in = policy_in(a.policy, at, n, l);
        const int kind = label_kind(y, a.y.ignore, a.x.c);
        float m = -INFINITY, s = 0.f;
        double logp = kind == kBad ? NAN : 0.0;
        if (kind == kCounted) {
            double own = 0.0;
            for (int64_t base = 0; base < classes; base += (int64_t)kStep * kBlock * K) {
                u32x4 raw[kStep];
                float top = m;
#pragma unroll
                for (int i = 0; i < kStep; ++i) {
                    const int64_t c0 = base + (i * kBlock + (int)threadIdx.x) * K;
                    if (c0 < classes) raw[i] = load_vec<T>(x + c0, (int32_t)(classes - c0));
                }
#pragma unroll
                for (int i = 0; i < kStep; ++i)
                    if (base + (i * kBlock + (int)threadIdx.x) * K < classes) {
                        float v[K];
                        unpack(raw[i], v, T());
#pragma unroll
                        for (int k = 0; k < K; ++k) top = fmaxf(top, v[k]);
                    }
                own *= (double)rescale(m, top, a.t);
                m = top;
                const float shift = shift_of(m);
#pragma unroll
                for (int i = 0; i < kStep; ++i)
                    if (base + (i * kBlock + (int)threadIdx.x) * K < classes) {
                        float v[K];
                        unpack(raw[i], v, T());
#pragma unroll
                        for (int k = 0; k < K; ++k) v[k] = exp_of(v[k] - shift, a.t);
                        own += tree_sum(v);
                    }
            }
            const double sum = fold_row<kBlock>(m, own, a.t, lds);
            logp = logp_of(to_f32(x[y]), shift_of(m), sum, a.t);
            s = (float)sum;
        }
        if (threadIdx.x == 0) leave_logp(a, at, logp, m, s, ref);
        if (kGrad) {
            T *g = (T *)a.grad + n * a.g_sn + l * a.g_sl;
            float w = kind == kBad ? NAN : 0.f;
            if (kind == kCounted)
                w = policy_term(a.policy, in, (float)logp).dlogp * (a.share ? a.share[n] : share_here<kBlock>(a, n, counts));
            if (a.weight_out && threadIdx.x == 0) a.weight_out[at] = w;
            const float shift = shift_of(m);
            if (kind == kCounted) w *= a.t.inv * a.host_scale;
            const float each = kind == kCounted ? -w / s : w;
            for (int64_t c0 = threadIdx.x * K; c0 < classes; c0 += kBlock * K) {
                float v[K];
                if (kind == kCounted) {
                    unpack(load_vec<T>(x + c0, (int32_t)(classes - c0)), v, T());
                    grad_of<K>(v, shift, each, w, (int32_t)y, (int32_t)c0, a.t);
                } else {
#pragma unroll
                    for (int k = 0; k < K; ++k) v[k] = each;
                }
                store_vec<true>(g + c0, (int32_t)(classes - c0), v);
            }
        }
    }
}

// weight * d logp / d x of rows whose maximum and sum are known: a stream, nothing to fold, so a workgroup takes kGradVecs
// vectors a lane of one row, whatever the row's length ([8,1024,32000] bf16, loss + gradient: 241 us with 1, 181 with 2, 188
// with 4 and 8).  Bound by the bytes: bf16 [8,1024,32000] 184 us (5.7 TB/s); behind a preference loss that ignores two fifths
// of the rows 116 us (7.1, part of the reads from the memory-side cache); [4,1023,50001], a third ignored, 104 us (6.5).
constexpr int kGradVecs = 2;

template <typename T>
__global__ __launch_bounds__(kTokThreads) void tok_row_grad_kernel(TokArgs a, int64_t pieces) {
    constexpr int K = vec_elements<T>();
    if (a.unless_one && *a.scale == 1.f) return;
    const int32_t classes = (int32_t)a.x.c;
    const float out_scale = a.t.inv * a.host_scale * (a.scale ? *a.scale : 1.f);
    for (int64_t turn = blockIdx.x; turn < a.x.n * a.x.l * pieces; turn += gridDim.x) {
        // from the last row to the first: what the loss's own pass read last is still in the memory-side cache
        // ([8,1024,32000] bf16, loss + gradient: 198 us in the loss's order, 188 in this one)
        const int64_t item = a.x.n * a.x.l * pieces - 1 - turn;
        const int64_t at = item / pieces, n = at / a.x.l, l = at - n * a.x.l;
        const int32_t c1 = (int32_t)((item - at * pieces) * (kGradVecs * kTokThreads * K)) + (int32_t)threadIdx.x * K;
        const T *x = (const T *)a.x.x + n * a.x.sn + l * a.x.sl;
        T *g = (T *)a.grad + n * a.g_sn + l * a.g_sl;
        const int64_t y = a.y.y[n * a.y.sn + l * a.y.sl];
        const int kind = label_kind(y, a.y.ignore, a.x.c);
        if (kind == kCounted) {
            u32x4 raw[kGradVecs];
#pragma unroll
            for (int i = 0; i < kGradVecs; ++i) {
                const int32_t c0 = c1 + i * kTokThreads * K;
                if (c0 < classes) raw[i] = load_vec<T>(x + c0, classes - c0);
            }
            const float2 st = a.stats_in[at];
            const float w = a.weight[n * a.w_sn + l * a.w_sl] * out_scale, each = -w / st.y, shift = shift_of(st.x);
#pragma unroll
            for (int i = 0; i < kGradVecs; ++i) {
                const int32_t c0 = c1 + i * kTokThreads * K;
                if (c0 < classes) {
                    float v[K];
                    unpack(raw[i], v, T());
                    grad_of<K>(v, shift, each, w, (int32_t)y, c0, a.t);
                    store_vec<true>(g + c0, classes - c0, v);
                }
            }
        } else {
            float v[K];
#pragma unroll
            for (int k = 0; k < K; ++k) v[k] = kind == kBad ? NAN : 0.f;
#pragma unroll
            for (int i = 0; i < kGradVecs; ++i) {
                const int32_t c0 = c1 + i * kTokThreads * K;
                if (c0 < classes) store_vec<true>(g + c0, classes - c0, v);
            }
        }
    }
}

// ---- positions next to each other in memory: a lane takes VEC of them, walking the class planes ----

// A position group's logits of one class as they lie in memory, and their values.
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
template <typename T, int VEC> struct GroupOf;
template <> struct GroupOf<float, 4> { typedef u32x4 type; };
template <> struct GroupOf<_Float16, 4> { typedef u32x2 type; };
template <> struct GroupOf<__bf16, 4> { typedef u32x2 type; };
template <typename T> struct GroupOf<T, 1> { typedef T type; };

template <typename T, int VEC>
__device__ __forceinline__ void values(const typename GroupOf<T, VEC>::type &r, float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        v[0] = to_f32(r);
    } else if constexpr (sizeof(T) == 4) {
        unpack(r, v, T());
    } else {
        float w[8];
        const u32x4 wide = {r[0], r[1], 0u, 0u};
        unpack(wide, w, T());
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = w[k];
    }
}

template <typename T, int VEC>
__device__ __forceinline__ typename GroupOf<T, VEC>::type grouped(const float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        return (T)v[0];
    } else if constexpr (sizeof(T) == 4) {
        return pack<T, VEC>(v);
    } else {
        typedef T t4 __attribute__((ext_vector_type(4)));
        const t4 t = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
        return __builtin_bit_cast(u32x2, t);
    }
}

// A group at any element's address.
template <typename T, int VEC>
struct __attribute__((packed, aligned(sizeof(T)))) GroupAt { typename GroupOf<T, VEC>::type v; };

// ONCE: see read_vec.
template <bool ONCE, typename T, int VEC>
__device__ __forceinline__ typename GroupOf<T, VEC>::type read_group(const T *p) {
    const GroupAt<T, VEC> *at = reinterpret_cast<const GroupAt<T, VEC> *>(p);
    return ONCE ? __builtin_nontemporal_load(&at->v) : at->v;
}

// Positions from `from` on of a group's gradient (the ones in front of it are another lane's).
template <typename T, int VEC>
__device__ __forceinline__ void store_group(T *p, int from, const float (&v)[VEC]) {
    if (from == 0) {
        __builtin_nontemporal_store(grouped<T, VEC>(v), &reinterpret_cast<GroupAt<T, VEC> *>(p)->v);
        return;
    }
#pragma unroll
    for (int k = 0; k < VEC; ++k)
        if (k >= from) p[k] = (T)v[k];
}

// As in the row kernel: packed logits from phase to phase.
template <typename G, int N>
__device__ __forceinline__ void forget_groups(G (&raw)[N]) {
    if constexpr (sizeof(G) >= 8) {
#pragma unroll
        for (int i = 0; i < N; ++i) asm volatile("" : "+v"(raw[i]));
    }
}

// CREG > 0: at most CREG classes, a position group's logits in registers, read once for maximum, sum and gradient.
// CREG = 0: the gradient alone, eight planes at a time.
// Four positions a lane make a wave's load of a plane 1 KB (fp32) in one instruction; all classes of a lane are in flight at
// once, nothing is exchanged between lanes, and the loss's sums leave as one item a workgroup.  Bound by the bytes: fp32
// [8,21,512x512] forward of the preference loss 43 us and its gradient 54 (218 and 386 MB with labels and statistics: 5.1 and
// 7.2 TB/s, the reads partly from the memory-side cache), policy loss with gradient 62 (394 MB: 6.3).  Workgroups of 64, 128,
// 512: 84, 84, 86 us for the whole policy loss, 77 with 256.  VEC = 1 takes any strides: channels last with a gradient in
// planes, the same size, policy loss 150 us in all (each lane reads its own row's lines, the gradient's stores are whole).
template <typename T, int VEC, int CREG, int MODE>
__global__ __launch_bounds__(kTokThreads, VEC == 1 || CREG <= 8 ? 4 : CREG <= 24 ? 3 : 2) void tok_planes_kernel(TokArgs a, int64_t tiles,
                                                                                                                int64_t first) {
    static_assert(CREG > 0 || MODE == kModeGrad, "without registers for the classes there is only the gradient");
    constexpr bool kGrad = MODE == kModeGrad || MODE == kModePolicyGrad;
    constexpr bool kStats = MODE == kModeGrad;          // (max, sum) given
    constexpr int K = MODE == kModePreference ? 2 : 4;  // sums of a workgroup
    constexpr bool kSums = MODE == kModePreference || MODE == kModePolicy || MODE == kModePolicyGrad;
    constexpr bool kOnce = MODE == kModePolicyGrad && CREG > 0 && VEC > 1;   // the logits' only reader (see read_vec)
    constexpr int kStep = 8;
    typedef typename GroupOf<T, VEC>::type G;
    __shared__ double lds[kSums ? K * kTokThreads / kWave : 1];
    __shared__ int counts[kTokThreads / kWave];
    if (MODE == kModeGrad && a.unless_one && *a.scale == 1.f) return;
    const int32_t classes = (int32_t)a.x.c;
    const int64_t item = first + blockIdx.x, n = item / tiles;
    int64_t l0 = ((item - n * tiles) * kTokThreads + threadIdx.x) * VEC;
    const bool live = l0 < a.x.l;
    const int dup = live && l0 + VEC > a.x.l ? (int)(l0 + VEC - a.x.l) : 0;   // the last group reaches back into the one before
    l0 -= dup;
    float share = 0.f;
    if (MODE == kModePolicyGrad) share = a.share ? a.share[n] : share_here<kTokThreads>(a, n, counts);
    double sums[K];
#pragma unroll
    for (int k = 0; k < K; ++k) sums[k] = 0.0;
    if (live) {
        const T *x = (const T *)a.x.x + n * a.x.sn + l0 * a.x.sl;
        const int64_t at = n * a.x.l + l0;
        const auto plane = [&](int32_t c) { return read_group<kOnce, T, VEC>(x + (int64_t)c * a.x.sc); };
        int32_t y[VEC];         // the label, or -1
        int kind[VEC];
        bool any = false;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            const int64_t label = a.y.y[n * a.y.sn + (l0 + k) * a.y.sl];
            kind[k] = label_kind(label, a.y.ignore, a.x.c);
            y[k] = kind[k] == kCounted ? (int32_t)label : -1;
            any |= kind[k] == kCounted;
        }
        float m[VEC], s[VEC], xl[VEC], w[VEC], v[VEC];
        double sum[VEC] = {};
        G raw[CREG > 0 ? CREG : kStep];
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            m[k] = -INFINITY;
            s[k] = xl[k] = w[k] = 0.f;
        }
        if (any && kStats) {
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                if (kind[k] == kCounted) {
                    const float2 st = a.stats_in[at + k];
                    m[k] = st.x;
                    s[k] = st.y;
                }
        }
        PolicyIn in[VEC] = {};
        if (MODE == kModePolicy || MODE == kModePolicyGrad) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) in[k] = policy_in(a.policy, at + k, n, l0 + k);
        }
        if (any && CREG > 0) {
#pragma unroll
            for (int c = 0; c < CREG; ++c)
                if (c < classes) raw[c] = plane(c);
            if (!kStats) {
#pragma unroll
                for (int c = 0; c < CREG; ++c)
                    if (c < classes) {
                        values<T, VEC>(raw[c], v);
#pragma unroll
                        for (int k = 0; k < VEC; ++k) {
                            m[k] = fmaxf(m[k], v[k]);
                            xl[k] = y[k] == c ? v[k] : xl[k];
                        }
                    }
                forget_groups(raw);
                // four short chains a position, joined in fp64 (see the split kernel)
#pragma unroll
                for (int c0 = 0; c0 < CREG; c0 += 16) {
                    float e[VEC][4] = {};
#pragma unroll
                    for (int c = c0; c < (c0 + 16 < CREG ? c0 + 16 : CREG); ++c)
                        if (c < classes) {
                            values<T, VEC>(raw[c], v);
#pragma unroll
                            for (int k = 0; k < VEC; ++k) e[k][c % 4] += exp_of(v[k] - shift_of(m[k]), a.t);
                        }
#pragma unroll
                    for (int k = 0; k < VEC; ++k) sum[k] += (double)(e[k][0] + e[k][1]) + (double)(e[k][2] + e[k][3]);
                }
#pragma unroll
                for (int k = 0; k < VEC; ++k) s[k] = (float)sum[k];
            }
        }
        float each[VEC];     // factor of a class's exponential in the gradient; where nothing is counted the value itself
        const float out_scale = kGrad ? a.t.inv * a.host_scale * (a.scale ? *a.scale : 1.f) : 0.f;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            const int64_t l = l0 + k;
            each[k] = 0.f;
            if (!kStats) {
                const double logp = kind[k] == kCounted ? logp_of(xl[k], shift_of(m[k]), sum[k], a.t) : kind[k] == kBad ? NAN : 0.0;
                if (k >= dup) leave_logp(a, at + k, logp, m[k], s[k], 0.f);
                if (MODE == kModePreference && kind[k] != kIgnored && k >= dup) {
                    sums[0] += logp - (double)a.ref[at + k];
                    sums[1] += 1.0;
                }
                if ((MODE == kModePolicy || MODE == kModePolicyGrad) && kind[k] != kIgnored) {
                    const PolicyTerm t = policy_term(a.policy, in[k], (float)logp);
                    if (k >= dup) {
                        sums[0] += t.surrogate;
                        sums[1] += t.far;
                        sums[2 % K] += t.over ? 1.0 : 0.0;
                        sums[3 % K] += 1.0;
                    }
                    w[k] = kind[k] == kBad ? NAN : t.dlogp * share;
                }
                if (MODE == kModePolicyGrad && a.weight_out && k >= dup) a.weight_out[at + k] = w[k];
            } else if (kind[k] == kCounted) {
                w[k] = a.weight[n * a.w_sn + l * a.w_sl];
            } else {
                w[k] = kind[k] == kBad ? NAN : 0.f;
            }
            if (kGrad) {
                if (kind[k] == kCounted) w[k] *= out_scale;
                each[k] = kind[k] == kCounted ? -w[k] / s[k] : w[k];
            }
        }
        if (kGrad) {
            T *g = (T *)a.grad + n * a.g_sn + l0 * a.g_sl;
            const auto store = [&](const G &from, int32_t c) {
                values<T, VEC>(from, v);
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    const float e = each[k] * exp_of(v[k] - shift_of(m[k]), a.t);
                    v[k] = kind[k] == kCounted ? (y[k] == c ? e + w[k] : e) : each[k];
                }
                store_group<T, VEC>(g + (int64_t)c * a.g_sc, dup, v);
            };
            if (CREG > 0) {
                forget_groups(raw);
#pragma unroll
                for (int c = 0; c < CREG; ++c)
                    if (c < classes) store(raw[c], c);
            } else {
                for (int32_t c0 = 0; c0 < classes; c0 += kStep) {
#pragma unroll
                    for (int j = 0; j < kStep; ++j)
                        if (any && c0 + j < classes) raw[j] = plane(c0 + j);
#pragma unroll
                    for (int j = 0; j < kStep; ++j)
                        if (c0 + j < classes) store(raw[j], c0 + j);
                }
            }
        }
    }
    if (kSums) {
        block_sums<K>(sums, lds, kTokThreads);
        if (threadIdx.x == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) a.part[item * K + k] = sums[k];
    }
}

// ---- the same for many classes: the class planes shared among the lane groups of a workgroup ----

// 64 neighbouring positions a workgroup: RUN lanes of VEC positions, and kTokThreads / RUN groups of them that take every
// kTokThreads / RUN-th class, eight planes in flight a lane.  The groups' maxima and sums meet in LDS, where one wave
// finishes the positions.  HOLD > 0: at most HOLD classes a group, kept for the gradient; HOLD = 0: any number, read again.
// (One lane walking all classes: [1,150,1024] fp32 26 / 24 / 56 us forward / gradient / policy, so 6.4 / 6.0 / 13.)  Bound by
// the bytes on large calls, 64 positions being 256 bytes a plane and load: fp32 [8,150,128x128] forward 17.5 us (4.5 TB/s),
// gradient 26.4 (6.0), policy loss 44.9 with its count and end; [1,1000,512x512] 191 (5.5), 424 (4.9), 529.  (Four
// chains a position, not a tree of the HOLD values: with it fp32 HOLD = 16 spilled 65 registers, policy loss 60 us.)
constexpr int kSplitTile = 64;

template <typename T, int VEC, int HOLD, int MODE>
__global__ __launch_bounds__(kTokThreads, HOLD > 0 ? 4 : 3) void tok_split_kernel(TokArgs a, int64_t tiles, int64_t first) {
    constexpr int RUN = kSplitTile / VEC, GROUPS = kTokThreads / RUN, kStep = HOLD > 0 ? HOLD : 8;
    constexpr bool kGrad = MODE == kModeGrad || MODE == kModePolicyGrad;
    constexpr bool kStats = MODE == kModeGrad;
    constexpr bool kOnce = MODE == kModePolicyGrad && HOLD > 0 && VEC > 1;
    constexpr int K = MODE == kModePreference ? 2 : 4;
    constexpr bool kSums = MODE == kModePreference || MODE == kModePolicy || MODE == kModePolicyGrad;
    typedef typename GroupOf<T, VEC>::type G;
    __shared__ float part_max[GROUPS][kSplitTile];      // of a group's classes
    __shared__ double part_sum[GROUPS][kSplitTile];
    __shared__ float at_label[kSplitTile], top_of[kSplitTile], each_of[kSplitTile], w_of[kSplitTile];
    __shared__ int label_of[kSplitTile];                // >= 0: counted; -1: ignored; -2: no class
    __shared__ int counts[kTokThreads / kWave];
    if (MODE == kModeGrad && a.unless_one && *a.scale == 1.f) return;
    const int32_t classes = (int32_t)a.x.c;
    // the last tile reaches back into the one before it, whose positions (the first `dup`) are that one's to write
    const int64_t item = first + blockIdx.x, n = item / tiles, tile = (item - n * tiles) * kSplitTile;
    const int dup = a.x.l >= kSplitTile && tile + kSplitTile > a.x.l ? (int)(tile + kSplitTile - a.x.l) : 0;
    const int64_t start = tile - dup;
    const int32_t group = threadIdx.x / RUN, pos = (threadIdx.x % RUN) * VEC;
    const int64_t l0 = start + pos;
    const bool live = l0 < a.x.l;
    float share = 0.f;
    if (MODE == kModePolicyGrad) share = a.share ? a.share[n] : share_here<kTokThreads>(a, n, counts);
    if (threadIdx.x < kSplitTile) {
        int y = -1;
        if (start + threadIdx.x < a.x.l) {
            const int64_t label = a.y.y[n * a.y.sn + (start + threadIdx.x) * a.y.sl];
            const int kind = label_kind(label, a.y.ignore, a.x.c);
            y = kind == kCounted ? (int)label : kind == kIgnored ? -1 : -2;
        }
        label_of[threadIdx.x] = y;
    }
    __syncthreads();
    int32_t y[VEC];
    bool any = false;
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
        y[k] = live ? label_of[pos + k] : -1;
        any |= y[k] >= 0;
    }
    const T *x = (const T *)a.x.x + n * a.x.sn + l0 * a.x.sl;
    const auto plane = [&](int32_t c) { return read_group<kOnce, T, VEC>(x + (int64_t)c * a.x.sc); };
    G raw[kStep];
    float v[VEC];
    if (!kStats) {
        float m[VEC];
        double s[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            m[k] = -INFINITY;
            s[k] = 0.0;
        }
        if (any) {
            for (int32_t c0 = group; c0 < classes; c0 += kStep * GROUPS) {
                float top[VEC];
#pragma unroll
                for (int k = 0; k < VEC; ++k) top[k] = m[k];
#pragma unroll
                for (int j = 0; j < kStep; ++j)
                    if (c0 + j * GROUPS < classes) raw[j] = plane(c0 + j * GROUPS);
#pragma unroll
                for (int j = 0; j < kStep; ++j)
                    if (c0 + j * GROUPS < classes) {
                        values<T, VEC>(raw[j], v);
#pragma unroll
                        for (int k = 0; k < VEC; ++k) {
                            top[k] = fmaxf(top[k], v[k]);
                            if (y[k] == c0 + j * GROUPS) at_label[pos + k] = v[k];
                        }
                    }
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    s[k] *= (double)rescale(m[k], top[k], a.t);
                    m[k] = top[k];
                }
                forget_groups(raw);
                // Four short chains a position, joined in fp64: once a sum in fp32 has reached 1, every class below 2^-25 adds
                // nothing to it (one chain over 32,000 classes 17 below the top: logp a quarter off).
                float e[VEC][4] = {};
#pragma unroll
                for (int j = 0; j < kStep; ++j)
                    if (c0 + j * GROUPS < classes) {
                        values<T, VEC>(raw[j], v);
#pragma unroll
                        for (int k = 0; k < VEC; ++k) e[k][j % 4] += exp_of(v[k] - shift_of(m[k]), a.t);
                    }
#pragma unroll
                for (int k = 0; k < VEC; ++k) s[k] += (double)(e[k][0] + e[k][1]) + (double)(e[k][2] + e[k][3]);
                if (HOLD > 0) break;
            }
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            part_max[group][pos + k] = m[k];
            part_sum[group][pos + k] = s[k];
        }
        __syncthreads();
    }
    double sums[K];
#pragma unroll
    for (int k = 0; k < K; ++k) sums[k] = 0.0;
    if (threadIdx.x < kSplitTile && start + threadIdx.x < a.x.l) {
        const int32_t q = threadIdx.x, yq = label_of[q];
        const int64_t l = start + q, at = n * a.x.l + l;
        float m = -INFINITY, s = 0.f, w = 0.f;
        if (kStats) {
            if (yq >= 0) {
                const float2 st = a.stats_in[at];
                m = st.x;
                s = st.y;
            }
            w = yq >= 0 ? a.weight[n * a.w_sn + l * a.w_sl] : yq == -2 ? NAN : 0.f;
        } else {
            for (int g = 0; g < GROUPS; ++g) m = fmaxf(m, part_max[g][q]);
            double sum = 0.0;
            for (int g = 0; g < GROUPS; ++g) sum += part_sum[g][q] * (double)rescale(part_max[g][q], m, a.t);
            s = (float)sum;
            const double exact = yq >= 0 ? logp_of(at_label[q], shift_of(m), sum, a.t) : yq == -2 ? (double)NAN : 0.0;
            if (q >= dup) leave_logp(a, at, exact, m, s, 0.f);
            if (MODE == kModePreference && yq != -1 && q >= dup) {
                sums[0] += exact - (double)a.ref[at];
                sums[1] += 1.0;
            }
            if ((MODE == kModePolicy || MODE == kModePolicyGrad) && yq != -1) {
                const PolicyTerm t = policy_term(a.policy, policy_in(a.policy, at, n, l), (float)exact);
                if (q >= dup) {
                    sums[0] += t.surrogate;
                    sums[1] += t.far;
                    sums[2 % K] += t.over ? 1.0 : 0.0;
                    sums[3 % K] += 1.0;
                }
                w = yq == -2 ? NAN : t.dlogp * share;
            }
            if (MODE == kModePolicyGrad && a.weight_out && q >= dup) a.weight_out[at] = w;
        }
        if (kGrad) {
            if (yq >= 0) w *= a.t.inv * a.host_scale * (a.scale ? *a.scale : 1.f);
            top_of[q] = shift_of(m);
            w_of[q] = w;
            each_of[q] = yq >= 0 ? -w / s : w;
        }
    }
    if (kSums && threadIdx.x < kWave) {     // (the wave that finished the positions)
#pragma unroll
        for (int k = 0; k < K; ++k) sums[k] = wave_sum(sums[k]);
        if (threadIdx.x == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) a.part[item * K + k] = sums[k];
    }
    if (kGrad) {
        __syncthreads();
        if (!live || pos + VEC <= dup) return;
        const int from = dup > pos ? dup - pos : 0;
        T *g = (T *)a.grad + n * a.g_sn + l0 * a.g_sl;
        float m[VEC], each[VEC], w[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            m[k] = top_of[pos + k];
            each[k] = each_of[pos + k];
            w[k] = w_of[pos + k];
        }
        if (HOLD > 0 && !kStats) forget_groups(raw);
#pragma nounroll
        for (int32_t c0 = group; c0 < classes; c0 += kStep * GROUPS) {
            if (any && (HOLD == 0 || kStats)) {
#pragma unroll
                for (int j = 0; j < kStep; ++j)
                    if (c0 + j * GROUPS < classes) raw[j] = plane(c0 + j * GROUPS);
            }
#pragma unroll
            for (int j = 0; j < kStep; ++j)
                if (c0 + j * GROUPS < classes) {
                    values<T, VEC>(raw[j], v);
#pragma unroll
                    for (int k = 0; k < VEC; ++k) {
                        const float e = each[k] * exp_of(v[k] - m[k], a.t);
                        v[k] = y[k] >= 0 ? (y[k] == c0 + j * GROUPS ? e + w[k] : e) : each[k];
                    }
                    store_group<T, VEC>(g + (int64_t)(c0 + j * GROUPS) * a.g_sc, from, v);
                }
            if (HOLD > 0) break;
        }
    }
}

// ---- passes over positions ----

struct SumArgs {
    const float *logp;
    const double *ratio;    // preference: logp - ref, in fp64: pairs of sequences are subtracted from each other
    Labels y;
    int64_t n, l, chunks;
    Policy policy;
    double *part;           // [n, chunks, K]
};

// What is summed over the counted positions of a sequence (the count is the last term):
//   kSumCount: {count};  kSumPreference: {sum logp - ref, count};  kSumPolicy: {sum surrogate, sum far, clipped, count}.
enum { kSumCount = 0, kSumPreference = 1, kSumPolicy = 2 };
template <int WHAT>
constexpr int sum_terms() { return WHAT == kSumCount ? 1 : WHAT == kSumPreference ? 2 : 4; }

template <int WHAT>
__device__ __forceinline__ void sum_position(const SumArgs &a, int64_t n, int64_t l, double (&v)[sum_terms<WHAT>()]) {
    constexpr int K = sum_terms<WHAT>();
    const int64_t at = n * a.l + l;
    if (a.y.y[n * a.y.sn + l * a.y.sl] == a.y.ignore) return;
    v[K - 1] += 1.0;
    if (WHAT == kSumPreference) v[0] += a.ratio[at];
    if (WHAT == kSumPolicy) {
        const PolicyTerm t = policy_term(a.policy, policy_in(a.policy, at, n, l), a.logp[at]);
        v[0] += t.surrogate;
        v[1 % K] += t.far;
        v[2 % K] += t.over ? 1.0 : 0.0;
    }
}

// A pass over labels and log-probabilities, kTokChunk positions a workgroup; latency bounds it: 5 us for 8192 positions of a
// loss as for the labels of 2^21 (17 MB).
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
#pragma unroll 8
        for (int64_t l = chunk * (int64_t)kTokChunk + threadIdx.x; l < end; l += kTokThreads) sum_position<WHAT>(a, n, l, v);
        block_sums<K>(v, lds, kTokThreads);
        if (threadIdx.x == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) a.part[item * K + k] = v[k];
    }
}

// The sums of every sequence by one workgroup of kTokFold threads, for calls of few positions: part[n, ways, K], a wave each.
template <int WHAT>
__device__ __forceinline__ void sums_here(const SumArgs &a, int64_t ways) {
    constexpr int K = sum_terms<WHAT>();
    for (int64_t item = threadIdx.x / kWave; item < a.n * ways; item += kTokFold / kWave) {
        const int64_t n = item / ways, way = item - n * ways;
        double v[K];
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = 0.0;
#pragma nounroll
        for (int64_t l = way * kWave + (threadIdx.x & 63); l < a.l; l += ways * kWave) sum_position<WHAT>(a, n, l, v);
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = wave_sum(v[k]);
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) a.part[item * K + k] = v[k];
    }
    __threadfence_block();
    __syncthreads();
}

// Each sequence's partial sums, folded by the lanes of a wave and handed to `take(n, sums)` in its first lane.
template <int K, typename F>
__device__ __forceinline__ void fold_sequences(const double *part, int64_t n, int64_t chunks, F take) {
    for (int64_t i = threadIdx.x / kWave; i < n; i += kTokFold / kWave) {
        double v[K];
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = 0.0;
        for (int64_t c = threadIdx.x & 63; c < chunks; c += kWave)
#pragma unroll
            for (int k = 0; k < K; ++k) v[k] += part[(i * chunks + c) * K + k];
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = wave_sum(v[k]);
        if ((threadIdx.x & 63) == 0) take(i, v);
    }
}

// share[n]: what one position of sequence n counts in the mean over all counted positions (token), or in the mean over
// sequences of each one's mean.  `ways` > 0: the positions are counted here.  One workgroup, latency: 4.5 us.  (Counts added
// up by every workgroup of the loss's pass: [8,21,512x512] 78 to 84 us, 75 with this launch: each waits for them.)
__global__ __launch_bounds__(kTokFold) void tok_share_kernel(SumArgs a, int64_t ways, int per_sequence, float *share) {
    __shared__ double lds[kTokFold / kWave];
    if (ways) sums_here<kSumCount>(a, ways);
    const int64_t chunks = ways ? ways : a.chunks;
    if (per_sequence) {
        fold_sequences<1>(a.part, a.n, chunks, [&](int64_t i, const double (&v)[1]) {
            share[i] = (float)(1.0 / (fmax(v[0], 1.0) * (double)a.n));
        });
        return;
    }
    double v[1] = {0.0};
    for (int64_t i = threadIdx.x; i < a.n * chunks; i += kTokFold) v[0] += a.part[i];
    block_sums<1>(v, lds, kTokFold);
    for (int64_t i = threadIdx.x; i < a.n; i += kTokFold) share[i] = (float)(1.0 / fmax(v[0], 1.0));
}

struct PreferenceEnd {
    double beta, smoothing;
    int ipo, average;
    float *total, *rewards, *weight;   // [1], [n], [n]: d total / d logp of every counted position of sequence n
    double *ratio;                     // [n, 2] scratch: a sequence's log ratio, and what its positions count
};

// softplus(-x) = -log sigmoid(x), and sigmoid, without overflow on either side.
__device__ __forceinline__ double minus_log_sigmoid(double x) { return log1p(exp(-fabs(x))) + fmax(-x, 0.0); }
__device__ __forceinline__ double sigmoid(double x) {
    const double e = exp(-fabs(x));
    return x >= 0.0 ? 1.0 / (1.0 + e) : e / (1.0 + e);
}

// The end of the preference loss: every sequence's log ratio from its partial sums, the pairs' losses, and what one position
// of each sequence weighs in the gradient.  One workgroup, latency: 5.1 us, with 37 or with 2^18 positions a sequence.
__global__ __launch_bounds__(kTokFold) void tok_preference_kernel(SumArgs a, int64_t ways, PreferenceEnd e) {
    __shared__ double lds[kTokFold / kWave];
    if (ways) sums_here<kSumPreference>(a, ways);
    fold_sequences<2>(a.part, a.n, ways ? ways : a.chunks, [&](int64_t i, const double (&v)[2]) {
        const double count = e.average ? fmax(v[1], 1.0) : 1.0;
        e.ratio[2 * i] = v[0] / count;
        e.ratio[2 * i + 1] = count;
    });
    __threadfence_block();
    __syncthreads();
    const int64_t half = a.n / 2;
    double v[1] = {0.0};
    for (int64_t i = threadIdx.x; i < half; i += kTokFold) {
        const double sa = e.ratio[2 * i], sb = e.ratio[2 * (half + i)];
        const double h = sa - sb, b = e.beta, eps = e.smoothing;
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
        e.weight[i] = (float)(dh / (double)half / e.ratio[2 * i + 1]);
        e.weight[half + i] = (float)(-dh / (double)half / e.ratio[2 * (half + i) + 1]);
    }
    block_sums<1>(v, lds, kTokFold);
    if (threadIdx.x == 0) *e.total = (float)(v[0] / (double)half);
}

// out4 = {total, surrogate, kl, share of the counted positions where the clipping holds}
__device__ __forceinline__ void policy_end(double surrogate, double far, double over, double count, double kl, float *out4) {
    out4[0] = (float)(kl != 0.0 ? surrogate + kl * far : surrogate);
    out4[1] = (float)surrogate;
    out4[2] = (float)far;
    out4[3] = (float)(over / fmax(count, 1.0));
}

// The end of the policy loss.  `each` [n, 4]: scratch.  One workgroup, latency: 6.0 us.  (By the last workgroup of the loss's
// pass, told by a ticket: 100 us for [8,21,512x512], 79 at that time with launches of their own.)
__global__ __launch_bounds__(kTokFold) void tok_policy_end_kernel(SumArgs a, int64_t ways, int per_sequence, double *each, double kl,
                                                                  float *out4) {
    __shared__ double lds[4 * kTokFold / kWave];
    if (ways) sums_here<kSumPolicy>(a, ways);
    const int64_t chunks = ways ? ways : a.chunks;
    double v[4] = {0.0, 0.0, 0.0, 0.0};
    if (per_sequence) {
        fold_sequences<4>(a.part, a.n, chunks, [&](int64_t i, const double (&u)[4]) {
            const double share = 1.0 / (fmax(u[3], 1.0) * (double)a.n);
            each[4 * i] = u[0] * share;
            each[4 * i + 1] = u[1] * share;
            each[4 * i + 2] = u[2];
            each[4 * i + 3] = u[3];
        });
        __threadfence_block();
        __syncthreads();
    }
    const double *from = per_sequence ? each : a.part;
    for (int64_t i = threadIdx.x; i < (per_sequence ? a.n : a.n * chunks); i += kTokFold)
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] += from[4 * i + k];
    block_sums<4>(v, lds, kTokFold);
    if (threadIdx.x == 0) {
        const double share = per_sequence ? 1.0 : 1.0 / fmax(v[3], 1.0);
        policy_end(v[0] * share, v[1] * share, v[2], v[3], kl, out4);
    }
}

// How many waves of the folding workgroup share a sequence where it takes the sums itself; 0: they are too many for it.
int64_t ways_of(int64_t n, int64_t l) {
    if (n == 0 || l > kTokHere / n) return 0;
    const int64_t ways = kTokFold / kWave / n, most = ceil_div(l, kWave);
    return ways < 1 ? 1 : ways > most ? (most ? most : 1) : ways;
}

int64_t chunks_of(int64_t l) { return l > kTokChunk ? ceil_div(l, kTokChunk) : 1; }
unsigned grid_of(int64_t blocks) { return (unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)); }

constexpr int64_t kThreadsMost = (int64_t)1 << 31;   // threads of a launch: a grid's are counted in 32 bits

// Every pointer on its element's bytes (a power of two); NULL passes.
bool on_bytes(const void *p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
template <typename... P>
bool on_floats(P... p) { return (on_bytes(p, 4) && ...); }

bool logits_ok(const spice_logits *x) {
    return x && x->n >= 0 && x->l >= 0 && x->c >= 1 && x->c <= 0x7fffffff - 65536 && x->dtype >= 0 && x->dtype <= 2 &&
           (x->data || x->n == 0 || x->l == 0) && on_bytes(x->data, x->dtype == 0 ? 4 : 2) &&
           (x->n == 0 || x->l <= ((int64_t)1 << 39) / x->n);
}

bool labels_ok(const spice_logits *x, const spice_labels *y) {
    return y && (y->data || x->n == 0 || x->l == 0) && aligned8(y->data) && (y->ignore_index < 0 || y->ignore_index >= x->c);
}

bool temperature_ok(double t) { return t > 0.0 && t <= 3.0e38 && 1.0 / t <= 3.0e38; }

TokArgs args_of(const spice_logits *x, const spice_labels *y, double t) {
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

template <typename T, int LANES, int NV, int MODE>
int launch_row(const TokArgs &a, hipStream_t stream) {
    constexpr int block = LANES < kTokThreads ? kTokThreads : LANES, rows = block / LANES;
    constexpr int64_t most = kThreadsMost / LANES;
    for (int64_t first = 0; first < a.x.n * a.x.l; first += most) {
        const int64_t left = a.x.n * a.x.l - first;
        tok_row_kernel<T, LANES, NV, MODE><<<(unsigned)ceil_div(left < most ? left : most, rows), block, 0, stream>>>(a, first);
        SPICE_LAUNCH_CHECK();
    }
    return SPICE_OK;
}

// Full vectors a lane of 4 and of 16 lanes a row: shorter rows share a wave.
constexpr int kShort4 = 8, kShort4Grad = 3, kShort16 = 6;

// How many lanes hold a row, by its full 16-byte vectors: as few as can keep them, so that a wave's fixed work (labels,
// fold, logarithm) is shared by many rows.  Forward / policy loss / gradient in us, bf16, 2^27 logits or 2^20 rows in all:
//   c = 64: 4 lanes 38 / 90 / 53, 16 lanes 102 / 176 / 98;   c = 256: 4 lanes 49 / 131 / 105, 16 lanes 75 / 156 / 102,
//   64 lanes 208 / 323 / 177;   c = 512: 16 lanes 53 / 129 / 96, 64 lanes 116 / 204 / 102;   c = 1000: 16 lanes
//   50 / 130 / 106, 64 lanes 67 / 129 / 83;   c = 4096: 64 lanes 46 / 109 / 84, 256 lanes 69 / 143 / 86;   c = 16384:
//   256 lanes 47 / 111, 512 lanes 55 / 123;   c = 32000: 512 lanes 49 / 113, 1024 lanes 55 / 149;   c = 131072: 16 vectors
//   of 1024 lanes 61 / 133, the long row kernel 56 / 135 (8 rows: 11.3 / 26.7 and 13.0 / 29.4).
// 4 lanes store a gradient in pieces of 64 bytes, which costs at odd widths (c = 200, gradient: 136, with 16 lanes 106): the
// gradient by itself leaves them earlier; the policy loss does not (161 against 166), so that its sums are the same with a
// gradient and without one.  The gradient by itself is also shared among workgroups sooner (kGradVecs vectors a lane;
// c = 2000: 84 with 64 lanes a row, 99 so; c = 4096: 84 and 77).
template <typename T, int MODE>
int launch_rows(const TokArgs &a, hipStream_t stream) {
    constexpr int short4 = MODE == kModeGrad ? kShort4Grad : kShort4;
    const auto whole = [&](int lanes) { return a.x.c / (lanes * vec_elements<T>()); };
    if (whole(4) <= short4) return launch_row<T, 4, short4, MODE>(a, stream);
    if (whole(16) <= kShort16) return launch_row<T, 16, kShort16, MODE>(a, stream);
    if constexpr (MODE == kModeGrad) {
        if (whole(64) <= 4) return launch_row<T, 64, 4, MODE>(a, stream);
        const int64_t pieces = ceil_div(a.x.c, (int64_t)kGradVecs * kTokThreads * vec_elements<T>());
        tok_row_grad_kernel<T><<<grid_of(a.x.n * a.x.l * pieces), kTokThreads, 0, stream>>>(a, pieces);
        SPICE_LAUNCH_CHECK();
        return SPICE_OK;
    } else {
        if (whole(64) <= 8) return launch_row<T, 64, 8, MODE>(a, stream);
        if (whole(256) <= 8) return launch_row<T, 256, 8, MODE>(a, stream);
        if (whole(512) <= 8) return launch_row<T, 512, 8, MODE>(a, stream);
        if (whole(1024) <= 8) return launch_row<T, 1024, 8, MODE>(a, stream);
        if (whole(1024) <= 16) return launch_row<T, 1024, 16, MODE>(a, stream);
        if (whole(1024) <= 20) return launch_row<T, 1024, 20, MODE>(a, stream);
        tok_long_row_kernel<T, MODE><<<grid_of(a.x.n * a.x.l), 1024, 0, stream>>>(a);
        SPICE_LAUNCH_CHECK();
        return SPICE_OK;
    }
}

// Neighbouring positions a lane of the planes kernels takes, and the most classes that one lane walks alone.
constexpr int kPlanesVec = 4, kPlanesClasses = 32;

bool next_to_each_other(const TokArgs &a) { return a.x.sl == 1 && (!a.grad || a.g_sl == 1); }

// Four positions a lane, at any alignment; the last group of a sequence reaches back into the one before, so there have to
// be as many positions as a lane (or, with many classes, a workgroup) takes, or a multiple of four.
bool planes_vec(const TokArgs &a) {
    const int64_t least = a.x.c > kPlanesClasses ? kSplitTile : kPlanesVec;
    return next_to_each_other(a) && (a.x.l >= least || a.x.l % kPlanesVec == 0);
}

int64_t planes_tiles(int64_t l, bool vec) { return ceil_div(l, (int64_t)kTokThreads * (vec ? kPlanesVec : 1)); }

template <typename T, int VEC, int MODE>
int launch_planes(const TokArgs &a, hipStream_t stream) {
    const bool split = a.x.c > kPlanesClasses;
    const int64_t tiles = split ? ceil_div(a.x.l, kSplitTile) : planes_tiles(a.x.l, VEC > 1);
    constexpr int groups = kTokThreads * VEC / kSplitTile;
    constexpr int64_t most = kThreadsMost / kTokThreads;
    for (int64_t first = 0; first < a.x.n * tiles; first += most) {
        const int64_t left = a.x.n * tiles - first;
        const unsigned grid = (unsigned)(left < most ? left : most);
        if (split) {
            if (a.x.c <= groups * 8)
                tok_split_kernel<T, VEC, 8, MODE><<<grid, kTokThreads, 0, stream>>>(a, tiles, first);
            else if (a.x.c <= groups * 16)
                tok_split_kernel<T, VEC, 16, MODE><<<grid, kTokThreads, 0, stream>>>(a, tiles, first);
            else
                tok_split_kernel<T, VEC, 0, MODE><<<grid, kTokThreads, 0, stream>>>(a, tiles, first);
        } else if constexpr (MODE == kModeGrad) {
            tok_planes_kernel<T, VEC, 0, MODE><<<grid, kTokThreads, 0, stream>>>(a, tiles, first);
        } else {
            if (a.x.c <= 8)
                tok_planes_kernel<T, VEC, 8, MODE><<<grid, kTokThreads, 0, stream>>>(a, tiles, first);
            else if (a.x.c <= 24)
                tok_planes_kernel<T, VEC, 24, MODE><<<grid, kTokThreads, 0, stream>>>(a, tiles, first);
            else
                tok_planes_kernel<T, VEC, 32, MODE><<<grid, kTokThreads, 0, stream>>>(a, tiles, first);
        }
        SPICE_LAUNCH_CHECK();
    }
    return SPICE_OK;
}

// Which kernel takes a call: rows where the classes are neighbours in memory, planes (where the positions are not
// neighbours, or the gradient's are not, one a lane), and a workgroup a position for few positions of many classes.
enum { kByRows, kByPlanes, kByAny };
int route_of(const TokArgs &a) {
    if (a.x.sc == 1 && (!a.grad || a.g_sc == 1)) return kByRows;   // (channels last: its gradient is in planes)
    // a workgroup a position fills more of the chip than 64 positions a workgroup (256 positions of 3001 classes: 6.5 against
    // 41 us, of 150 classes 6.3 both; 4096 of 1000: 22 against 17); strided, 512 of 150: 6 / 14 / 6 us forward / policy /
    // gradient against 8 / 18 / 8, 4096 of 150: 13 / 34 / 16 against 8 / 21 / 8, 65536 of 150: 117 / 219 / 159 against 16 / 43 / 22
    const bool few = a.x.n * a.x.l <= 512;
    return few && a.x.c > (next_to_each_other(a) ? 256 : kPlanesClasses) ? kByAny : kByPlanes;
}

// Rows of several sequences that share a wave: it cannot count each one's labels.
bool rows_share_waves(const TokArgs &a, int32_t dtype) {
    return route_of(a) == kByRows && a.per_sequence && a.x.n > 1 && a.x.c / (16 * (dtype == 0 ? 4 : 8)) <= kShort16;
}

template <typename T, int MODE>
int launch_typed(const TokArgs &a, hipStream_t stream) {
    const int64_t total = a.x.n * a.x.l;
    const int route = route_of(a);
    if (route == kByPlanes)
        return planes_vec(a) ? launch_planes<T, kPlanesVec, MODE>(a, stream) : launch_planes<T, 1, MODE>(a, stream);
    // rows and any strides: the sums over positions are a pass of their own over logp
    constexpr int mode = MODE == kModePreference || MODE == kModePolicy ? kModeLogp : MODE;
    if (route == kByRows) return launch_rows<T, mode>(a, stream);
    tok_any_kernel<T, mode><<<grid_of(total), kTokThreads, 0, stream>>>(a);
    SPICE_LAUNCH_CHECK();
    return SPICE_OK;
}

template <int MODE>
int launch_positions(const TokArgs &a, int32_t dtype, hipStream_t stream) {
    if (a.x.n * a.x.l == 0) return SPICE_OK;
    return dtype == 0 ? launch_typed<float, MODE>(a, stream)
           : dtype == 1 ? launch_typed<_Float16, MODE>(a, stream)
                        : launch_typed<__bf16, MODE>(a, stream);
}

// Items a sequence's partial sums come in: the planes kernel's tiles, or the chunks of the pass over logp.
int64_t items_of(const TokArgs &a) {
    if (route_of(a) != kByPlanes) return chunks_of(a.x.l);
    return !a.x.l ? 1 : a.x.c > kPlanesClasses ? ceil_div(a.x.l, kSplitTile) : planes_tiles(a.x.l, planes_vec(a));
}

// The losses' workspace: the partial sums, 4 n + 8 of the sequences', the preference loss's log ratios [n, l].
// Partial sums of a call at most: the workgroups' of the split planes kernel, or the waves' of the folding workgroup.
int64_t part_doubles(int64_t n, int64_t l) {
    const int64_t items = l > kSplitTile ? ceil_div(l, kSplitTile) : 1, waves = kTokFold / kWave;
    return (n * items > n + waves ? n * items : n + waves) * 4;
}

SumArgs sums_of(const TokArgs &a, double *part) {
    SumArgs s = {};
    s.logp = a.logp;
    s.ratio = a.ratio;
    s.y = a.y;
    s.n = a.x.n;
    s.l = a.x.l;
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
    return (size_t)(part_doubles(n, l) + 4 * n + 8 + n * l) * sizeof(double);
}

extern "C" int spice_token_logprobs(const spice_logits *x, const spice_labels *y, double temperature, float *logp, float *stats,
                                    void *stream) {
    if (!logits_ok(x) || !labels_ok(x, y) || !temperature_ok(temperature) || (!logp && x->n * x->l) || !aligned8(stats) ||
        !on_floats(logp))
        return SPICE_ERR_ARG;
    TokArgs a = args_of(x, y, temperature);
    a.logp = logp;
    a.stats = (float2 *)stats;
    return launch_positions<kModeLogp>(a, x->dtype, (hipStream_t)stream);
}

extern "C" int spice_token_logprobs_grad(const spice_logits *x, const spice_labels *y, double temperature, const float *stats,
                                         const float *weight, int64_t w_n_stride, int64_t w_l_stride, float scale,
                                         const float *device_scale, int32_t unless_one, int32_t class_last, void *grad,
                                         void *stream) {
    if (!logits_ok(x) || !labels_ok(x, y) || !temperature_ok(temperature) || !aligned8(stats) || (unless_one && !device_scale) ||
        ((!stats || !weight || !grad) && x->n * x->l) || !on_floats(weight, device_scale) || !on_bytes(grad, x->dtype == 0 ? 4 : 2))
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

extern "C" int spice_preference_loss_opts(const spice_logits *x, const spice_labels *y, const float *ref_logp,
                                          const spice_preference_options *p, float *total, float *rewards, float *weight,
                                          float *stats, void *workspace, size_t workspace_bytes, void *stream) {
    if (!logits_ok(x) || !labels_ok(x, y) || !p || x->n < 2 || x->n % 2 || !total || !rewards || !weight || !workspace ||
        !aligned8(workspace) || (!ref_logp && x->l) || !aligned8(stats) || !(p->beta > 0.0 && p->beta <= 3.0e38) ||
        !(p->smoothing >= 0.0 && p->smoothing < 0.5) || p->loss_type < 0 || p->loss_type > 1 ||
        (p->loss_type == SPICE_PREFERENCE_IPO && p->smoothing != 0.0) || !temperature_ok(p->temperature) ||
        !on_floats(ref_logp, total, rewards, weight))
        return SPICE_ERR_ARG;
    if (workspace_bytes < spice_token_loss_workspace_bytes(x->n, x->l)) return SPICE_ERR_WORKSPACE;
    hipStream_t s = (hipStream_t)stream;
    TokArgs a = args_of(x, y, p->temperature);
    a.stats = (float2 *)stats;
    a.ref = ref_logp;
    a.part = (double *)workspace;
    if (route_of(a) != kByPlanes) a.ratio = a.part + part_doubles(x->n, x->l) + 4 * x->n + 8;   // (the planes kernels sum it themselves)
    int rc = launch_positions<kModePreference>(a, x->dtype, s);
    if (rc) return rc;
    SumArgs sums = sums_of(a, a.part);
    int64_t ways = 0;
    if (route_of(a) == kByPlanes && x->l) {
        sums.chunks = items_of(a);
    } else if (!(ways = ways_of(x->n, x->l))) {
        rc = launch_sums<kSumPreference>(sums, s);
        if (rc) return rc;
    }
    PreferenceEnd e = {p->beta, p->smoothing, p->loss_type == SPICE_PREFERENCE_IPO, p->average != 0, total, rewards, weight,
                       a.part + part_doubles(x->n, x->l)};
    tok_preference_kernel<<<1, kTokFold, 0, s>>>(sums, ways, e);
    SPICE_LAUNCH_CHECK();
    return SPICE_OK;
}

extern "C" int spice_preference_loss(const spice_logits *x, const spice_labels *y, const float *ref_logp,
                                     const spice_preference_params *p, float *total, float *rewards, float *weight, float *,
                                     float *stats, void *workspace, size_t workspace_bytes, void *stream) {
    if (!p) return SPICE_ERR_ARG;
    const spice_preference_options o = {p->temperature, p->beta, p->smoothing, p->loss_type, p->average};
    return spice_preference_loss_opts(x, y, ref_logp, &o, total, rewards, weight, stats, workspace, workspace_bytes, stream);
}

extern "C" int spice_policy_loss_opts(const spice_logits *x, const spice_labels *y, const float *old_logp, const float *advantages,
                                      int64_t adv_n_stride, int64_t adv_l_stride, const float *ref_logp,
                                      const spice_policy_options *p, float *out4, float *logp, float *stats, float *weight,
                                      int32_t class_last, void *grad, void *workspace, size_t workspace_bytes, void *stream) {
    if (!logits_ok(x) || !labels_ok(x, y) || !p || !out4 || !workspace || !aligned8(workspace) ||
        ((!old_logp || !advantages || !logp) && x->n * x->l) || !(p->clip_low >= 0.0 && p->clip_low <= 1.0) ||
        !(p->clip_high >= 0.0) || !(p->kl_weight >= 0.0) || (p->kl_weight > 0.0 && !ref_logp && x->n * x->l) ||
        p->reduction < 0 || p->reduction > 1 || !aligned8(stats) || !temperature_ok(p->temperature) ||
        !on_floats(old_logp, advantages, ref_logp, out4, logp, weight) || !on_bytes(grad, x->dtype == 0 ? 4 : 2))
        return SPICE_ERR_ARG;
    if (workspace_bytes < spice_token_loss_workspace_bytes(x->n, x->l)) return SPICE_ERR_WORKSPACE;
    hipStream_t s = (hipStream_t)stream;
    TokArgs a = args_of(x, y, p->temperature);
    a.logp = logp;
    a.stats = (float2 *)stats;
    a.weight_out = weight;
    a.host_scale = (float)p->grad_scale;
    a.policy = Policy{old_logp, advantages, ref_logp, adv_n_stride, adv_l_stride, (float)(1.0 - p->clip_low),
                      (float)(1.0 + p->clip_high), (float)p->kl_weight};
    if (grad) grad_layout(a, grad, class_last);
    a.part = (double *)workspace;
    SumArgs sums = sums_of(a, a.part);
    double *scratch = a.part + part_doubles(x->n, x->l);
    float *share = (float *)scratch;
    a.share = share;
    a.per_sequence = p->reduction == SPICE_POLICY_SEQUENCE;
    const bool planes = route_of(a) == kByPlanes && x->l;
    int64_t ways = ways_of(x->n, x->l);
    int rc = SPICE_OK;
    if (!grad || (x->n * x->l <= kTokCount && !rows_share_waves(a, x->dtype))) {
        a.share = nullptr;
    } else {
        if (!ways) rc = launch_sums<kSumCount>(sums, s);
        if (rc) return rc;
        tok_share_kernel<<<1, kTokFold, 0, s>>>(sums, ways, a.per_sequence, share);
        SPICE_LAUNCH_CHECK();
    }
    rc = grad ? launch_positions<kModePolicyGrad>(a, x->dtype, s) : launch_positions<kModePolicy>(a, x->dtype, s);
    if (rc) return rc;
    if (planes) {
        sums.chunks = items_of(a);
        ways = 0;
    } else if (!ways) {
        rc = launch_sums<kSumPolicy>(sums, s);
        if (rc) return rc;
    }
    tok_policy_end_kernel<<<1, kTokFold, 0, s>>>(sums, ways, a.per_sequence, scratch, p->kl_weight, out4);
    SPICE_LAUNCH_CHECK();
    return SPICE_OK;
}

extern "C" int spice_policy_loss(const spice_logits *x, const spice_labels *y, const float *old_logp, const float *advantages,
                                 int64_t adv_n_stride, int64_t adv_l_stride, const float *ref_logp, const spice_policy_params *p,
                                 float *out4, float *logp, float *stats, float *weight, int32_t class_last, void *grad,
                                 void *workspace, size_t workspace_bytes, void *stream) {
    if (!p) return SPICE_ERR_ARG;
    const spice_policy_options o = {p->temperature, p->clip_low, p->clip_high, p->kl_weight, p->grad_scale, p->reduction, 0};
    return spice_policy_loss_opts(x, y, old_logp, advantages, adv_n_stride, adv_l_stride, ref_logp, &o, out4, logp, stats, weight,
                                  class_last, grad, workspace, workspace_bytes, stream);
}
