// The update end of a fine-tuning step over many tensors: global gradient norm, clipping, Adam.
//
//   norm = (sum over all tensors of g^2)^1/2 (or max |g|),   c = min(1, max_norm / (norm + 1e-6)),
//   clip:  out = c g
//   Adam:  g' = c g (+ decay p),  m += (1 - b1)(g' - m),  v += (1 - b2)(g'^2 - v),
//          p -= lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)     (decoupled decay: p *= 1 - lr decay first)
//
// The tensors of a call travel as kernel arguments: pointers, sizes and the first work item of each, as many as fit into
// 4 KB, so nothing is uploaded, nothing outlives the call and a captured launch holds all it needs.  A workgroup finds its
// tensor by bisection of the first-item table.  Squares are summed in fp64: a gradient of 1e20 or 1e-30 neither overflows
// nor vanishes, and the partial sums are folded in a fixed order by one workgroup, so the norm repeats bit for bit.
#include "common.h"

#include <math.h>

namespace spice {
namespace {

constexpr int kOptThreads = 256;
constexpr int kOptFold = 1024;
constexpr int64_t kOptItemLeast = 8192;            // elements of a work item at least
// Work items of the update and of clipping: 4 and 8 elements a lane, all of a workgroup's loads in flight at once and no
// loop.  Longer items were slower, the longest most: Adam, 808 M parameters with the norm, 4.61 ms at 1024 elements, 4.77 at
// 2048, 4.85 at 4096, 4.94 at 8192, 5.25 at 97 K; bf16 gradients clipped into fp32, 39.5 M: 55.8 us at 2048, 57.3 at 8192.
constexpr uint32_t kAdamItem = 1024, kClipItem = 2048;
constexpr int64_t kOptItems = 16384;                // work items of a call, about, at most
constexpr int64_t kOptEntryMost = (int64_t)1 << 30; // elements of one table entry: longer tensors take several

// A call's work items: `each` elements of one tensor.  Up to N table entries a launch.
template <int PTRS, int N>
struct Table {
    void *p[PTRS][N];
    uint32_t numel[N];
    uint32_t first[N];   // first work item of the entry, from the launch's first
    int32_t count;
    uint32_t each;
};

template <int PTRS>
constexpr int table_entries() { return PTRS == 1 ? 240 : PTRS == 2 ? 160 : 96; }
template <int PTRS>
using TableOf = Table<PTRS, table_entries<PTRS>()>;
static_assert(sizeof(TableOf<1>) <= 3900 && sizeof(TableOf<2>) <= 3900 && sizeof(TableOf<4>) <= 3900, "kernel arguments");

template <typename TB>
__device__ __forceinline__ int entry_of(const TB &t, uint32_t item) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= item) lo = mid; else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ float opt_f32(float v) { return v; }
__device__ __forceinline__ float opt_f32(_Float16 v) { return (float)v; }
__device__ __forceinline__ float opt_f32(__bf16 v) { return (float)v; }

__device__ __forceinline__ bool on16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T, int K>
struct __attribute__((aligned(sizeof(T) * K))) Vec { T v[K]; };

// Past the caches: what a step reads and writes once would leave its dirty lines in the memory-side cache, to be written
// back under the next call's reads (a 39.5 M parameter step with its norm: 266 us through the caches, 234 past them).
// The norm's own read goes through them: the update behind it finds part of the gradients there.
template <typename V>
__device__ __forceinline__ V take_once(const V *p) {
    if constexpr (sizeof(V) == 16) {
        return __builtin_bit_cast(V, __builtin_nontemporal_load((const u32x4_t *)p));
    } else {
        return __builtin_bit_cast(V, __builtin_nontemporal_load((const unsigned long long *)p));
    }
}
template <typename V>
__device__ __forceinline__ void put_once(V *p, const V &v) {
    if constexpr (sizeof(V) == 16) {
        __builtin_nontemporal_store(__builtin_bit_cast(u32x4_t, v), (u32x4_t *)p);
    } else {
        __builtin_nontemporal_store(__builtin_bit_cast(unsigned long long, v), (unsigned long long *)p);
    }
}

// NaN-keeping maximum
__device__ __forceinline__ double max_keep(double a, double b) { return (a > b || a != a) ? a : b; }

template <bool INF>
__device__ __forceinline__ double norm_join(double a, double b) { return INF ? max_keep(a, b) : a + b; }

template <bool INF>
__device__ __forceinline__ double norm_fold(double v, double *lds, int threads) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = norm_join<INF>(v, __shfl_xor(v, o, kWave));
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    v = lds[0];
    for (int w = 1; w < threads / kWave; ++w) v = norm_join<INF>(v, lds[w]);
    return v;
}

template <typename T, bool INF>
__device__ __forceinline__ double norm_take(double acc, T g) {
    const double d = (double)opt_f32(g);
    return INF ? max_keep(fabs(d), acc) : __builtin_fma(d, d, acc);
}

// Bound by the bytes read; eight 16-byte loads a lane in flight, since fp64 sums keep the loop from running ahead by itself
// (fp32, 39.5 M: 56 us with one load at a time, 29.7 so, 5.3 TB/s).  808 M: 542 us (6.0 TB/s); bf16, 39.5 M: 15.6 (5.1).
template <typename T, bool INF>
__global__ __launch_bounds__(kOptThreads) void grad_norm_kernel(TableOf<1> t, double *part) {
    __shared__ double lds[kOptThreads / kWave];
    const int e = entry_of(t, blockIdx.x);
    const uint32_t at = (blockIdx.x - t.first[e]) * t.each;
    const T *g = (const T *)t.p[0][e] + at;
    const uint32_t n = min(t.each, t.numel[e] - at);
    double acc = 0.0;
    uint32_t done = 0;
    if (on16(g)) {
        constexpr int K = 16 / sizeof(T);
        typedef Vec<T, K> VecTK;
        const Vec<T, K> *gv = (const Vec<T, K> *)g;
        const uint32_t nv = n / K;
        // UN loads in flight a lane; two chains of sums
        constexpr int UN = sizeof(T) == 4 ? 8 : 4;
        double two = 0.0;
        uint32_t i = threadIdx.x;
        for (; i + (UN - 1) * kOptThreads < nv; i += UN * kOptThreads) {
            u32x4_t x[UN];
#pragma unroll
            for (int j = 0; j < UN; ++j) x[j] = *(const u32x4_t *)(gv + i + j * kOptThreads);
#pragma unroll
            for (int j = 0; j < UN; ++j) {
                const Vec<T, K> v = __builtin_bit_cast(VecTK, x[j]);
#pragma unroll
                for (int k = 0; k < K; k += 2) {
                    acc = norm_take<T, INF>(acc, v.v[k]);
                    two = norm_take<T, INF>(two, v.v[k + 1]);
                }
            }
        }
        for (; i < nv; i += kOptThreads) {
            const Vec<T, K> x = gv[i];
#pragma unroll
            for (int k = 0; k < K; ++k) acc = norm_take<T, INF>(acc, x.v[k]);
        }
        acc = norm_join<INF>(acc, two);
        done = nv * K;
    }
    for (uint32_t i = done + threadIdx.x; i < n; i += kOptThreads) acc = norm_take<T, INF>(acc, g[i]);
    acc = norm_fold<INF>(acc, lds, kOptThreads);
    if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

// The call's record: {norm, clip factor, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)}.
struct RecordArgs {
    const double *part;
    int64_t parts;
    const float *norm_in;   // a norm taken before, or NULL
    int inf, clip, adam;
    double max_norm;
    double lr, beta1, beta2;
    int64_t host_step;
    int64_t *step;          // device step count, raised here; NULL: host_step
    float *record;
};

// The step's two factors, by a wave that does not wait for the norm.
__device__ __forceinline__ void record_step(const RecordArgs &a) {
    int64_t t = a.host_step;
    if (a.step) {
        t = *a.step + 1;
        *a.step = t;
    }
    a.record[2] = (float)(a.lr / (1.0 - pow(a.beta1, (double)t)));
    a.record[3] = (float)(1.0 / sqrt(1.0 - pow(a.beta2, (double)t)));
}

__device__ __forceinline__ float record_norm(const RecordArgs &a, double norm) {
    double c = 1.0;
    if (a.clip) {
        c = a.max_norm / (norm + 1e-6);
        if (c > 1.0) c = 1.0;
    }
    a.record[0] = (float)norm;
    a.record[1] = (float)c;
    return (float)c;
}

// One workgroup: a fixed order of the partial sums, 4.9 us with up to 16384 of them, mostly the launch.
__global__ __launch_bounds__(kOptFold) void grad_record_kernel(RecordArgs a) {
    __shared__ double lds[kOptFold / kWave];
    if (a.adam && threadIdx.x == kOptFold - 1) record_step(a);
    double norm = 0.0;
    if (a.norm_in) {
        norm = (double)*a.norm_in;
    } else if (a.inf) {
        for (int64_t i = threadIdx.x; i < a.parts; i += kOptFold) norm = norm_join<true>(norm, a.part[i]);
        norm = norm_fold<true>(norm, lds, kOptFold);
    } else {
        for (int64_t i = threadIdx.x; i < a.parts; i += kOptFold) norm += a.part[i];
        norm = sqrt(norm_fold<false>(norm, lds, kOptFold));
    }
    if (threadIdx.x == 0) record_norm(a, norm);
}

// Small calls: one workgroup takes the norm, leaves the record and, with outputs, clips; its waves share the items.  Bound by
// latency: 12 tensors of 5 to 2304 elements 6.9 us, where norm, record and clip as launches of their own took 18.8 in all.
template <typename T, typename O, bool INF, bool CLIP>
__global__ __launch_bounds__(kOptFold) void grad_here_kernel(TableOf<CLIP ? 2 : 1> t, int32_t items, RecordArgs a) {
    __shared__ double lds[kOptFold / kWave];
    __shared__ float factor;
    constexpr int kWaves = kOptFold / kWave;
    const uint32_t wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    if (a.adam && threadIdx.x == kOptFold - 1) record_step(a);
    double acc = 0.0;
    for (uint32_t item = wave; item < (uint32_t)items; item += kWaves) {
        const int e = entry_of(t, item);
        const uint32_t at = (item - t.first[e]) * t.each, n = min(t.each, t.numel[e] - at);
        const T *g = (const T *)t.p[0][e] + at;
#pragma unroll 8
        for (uint32_t i = lane; i < n; i += kWave) acc = norm_take<T, INF>(acc, g[i]);
    }
    acc = norm_fold<INF>(acc, lds, kOptFold);
    if (threadIdx.x == 0) factor = record_norm(a, INF ? acc : sqrt(acc));
    if constexpr (CLIP) {
        __syncthreads();
        const float c = factor;
        for (uint32_t item = wave; item < (uint32_t)items; item += kWaves) {
            const int e = entry_of(t, item);
            const uint32_t at = (item - t.first[e]) * t.each, n = min(t.each, t.numel[e] - at);
            const T *g = (const T *)t.p[0][e] + at;
            O *out = (O *)t.p[1][e] + at;
            if (c == 1.f && (const void *)g == (const void *)out) continue;
#pragma unroll 8
            for (uint32_t i = lane; i < n; i += kWave) out[i] = (O)(opt_f32(g[i]) * c);
        }
    }
}

// A stream: 39.5 M bf16 gradients into fp32 38 us in two launches (160 tensors, and the 30 largest: 237 MB, 6.2 TB/s, the
// gradients partly in the memory-side cache from the norm).
template <typename T, typename O>
__global__ __launch_bounds__(kOptThreads) void grad_clip_kernel(TableOf<2> t, const float *record) {
    const float c = record[1];
    const int e = entry_of(t, blockIdx.x);
    const uint32_t at = (blockIdx.x - t.first[e]) * t.each;
    const T *g = (const T *)t.p[0][e] + at;
    O *out = (O *)t.p[1][e] + at;
    if (c == 1.f && (const void *)g == (const void *)out) return;
    const uint32_t n = min(t.each, t.numel[e] - at);
    uint32_t done = 0;
    if (on16(g) && on16(out)) {
        constexpr int K = 16 / (sizeof(T) < sizeof(O) ? sizeof(O) : sizeof(T));
        const uint32_t nv = n / K;
        for (uint32_t i = threadIdx.x; i < nv; i += kOptThreads) {
            const Vec<T, K> x = ((const Vec<T, K> *)g)[i];
            Vec<O, K> y;
#pragma unroll
            for (int k = 0; k < K; ++k) y.v[k] = (O)(opt_f32(x.v[k]) * c);
            typedef Vec<O, K> VO;
            put_once((VO *)out + i, y);
        }
        done = nv * K;
    }
    for (uint32_t i = done + threadIdx.x; i < n; i += kOptThreads) out[i] = (O)(opt_f32(g[i]) * c);
}

struct AdamArgs {
    float rate, root;                 // record[2] and [3] where there is no record
    float a1, a2, eps, decay, keep;   // a = 1 - beta, taken in fp64 (1 - 0.999f is 1e-5 of itself off); keep = 1 - lr * decay with decoupled decay, else 1; decay = 0 then
};

template <typename T>
__device__ __forceinline__ void adam_take(T &p, T g, float &m, float &v, const AdamArgs &a, float c, float rate, float root) {
    float w = opt_f32(p), d = opt_f32(g) * c;
    w *= a.keep;
    d = __builtin_fmaf(a.decay, w, d);
    m = __builtin_fmaf(a.a1, d - m, m);
    v = __builtin_fmaf(a.a2, d * d - v, v);
    w -= rate * (m / __builtin_fmaf(sqrtf(v), root, a.eps));
    p = (T)w;
}

// A stream of seven arrays, four elements a lane: 28 bytes an element of fp32.  39.5 M 170 us (6.5 TB/s, the gradients partly
// in the memory-side cache from the norm), 808 M 4.11 ms (5.5 TB/s).
template <typename T>
__global__ __launch_bounds__(kOptThreads) void adam_kernel(TableOf<4> t, AdamArgs a, const float *record) {
    const float c = record ? record[1] : 1.f, rate = record ? record[2] : a.rate, root = record ? record[3] : a.root;
    const int e = entry_of(t, blockIdx.x);
    const uint32_t at = (blockIdx.x - t.first[e]) * t.each;
    T *p = (T *)t.p[0][e] + at;
    const T *g = (const T *)t.p[1][e] + at;
    float *m = (float *)t.p[2][e] + at, *v = (float *)t.p[3][e] + at;
    const uint32_t n = min(t.each, t.numel[e] - at);
    uint32_t done = 0;
    typedef Vec<T, 4> V4T;
    typedef Vec<float, 4> V4F;
    if (on16(p) && on16(g) && on16(m) && on16(v)) {
        const uint32_t nv = n / 4;
        for (uint32_t i = threadIdx.x; i < nv; i += kOptThreads) {
            V4T pv = take_once((const V4T *)p + i);
            const V4T gv = ((const V4T *)g)[i];
            V4F mv = take_once((const V4F *)m + i), vv = take_once((const V4F *)v + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) adam_take<T>(pv.v[j], gv.v[j], mv.v[j], vv.v[j], a, c, rate, root);
            put_once((V4T *)p + i, pv);
            put_once((V4F *)m + i, mv);
            put_once((V4F *)v + i, vv);
        }
        done = nv * 4;
    }
    for (uint32_t i = done + threadIdx.x; i < n; i += kOptThreads) adam_take<T>(p[i], g[i], m[i], v[i], a, c, rate, root);
}

// Elements of a work item: few items for large calls (their partial sums are folded by one workgroup), short ones for
// small calls (a workgroup's share of the chip).  A multiple of 1024 keeps every item's start on 16 bytes.
uint32_t item_elements(const int64_t *numel, int32_t count) {
    int64_t total = 0;
    for (int32_t i = 0; i < count; ++i) total += numel[i];
    const int64_t each = ceil_div(ceil_div(total, kOptItems), 1024) * 1024;
    return (uint32_t)(each < kOptItemLeast ? kOptItemLeast : each > ((int64_t)1 << 28) ? ((int64_t)1 << 28) : each);
}

bool counts_ok(const int64_t *numel, int32_t count) {
    if (count < 0 || (count && !numel)) return false;
    int64_t total = 0;
    for (int32_t i = 0; i < count; ++i) {
        if (numel[i] < 0 || numel[i] > ((int64_t)1 << 40)) return false;
        total += numel[i];
        if (total > ((int64_t)1 << 42)) return false;
    }
    return true;
}

// The tensors of one type among a call's: all of them without `dtypes`.
struct OfType {
    const int32_t *dtypes;
    int32_t dtype;
    bool operator()(int32_t i) const { return !dtypes || dtypes[i] == dtype; }
};

int64_t item_count(const int64_t *numel, int32_t count, uint32_t each, OfType of = {}) {
    int64_t items = 0;
    const int64_t most = kOptEntryMost / each * each;
    for (int32_t i = 0; i < count; ++i)
        for (int64_t at = 0; of(i) && at < numel[i]; at += most) items += ceil_div(numel[i] - at < most ? numel[i] - at : most, each);
    return items;
}

// Calls launch(table, first item, items) for as many tables as the tensors need.  ptrs: PTRS host arrays of device
// pointers; bytes: element size of each.
template <int PTRS, typename F>
int for_tables(void *const *const (&ptrs)[PTRS], const int64_t (&bytes)[PTRS], const int64_t *numel, int32_t count, uint32_t each, F launch,
               OfType of = {}) {
    TableOf<PTRS> t;
    t.count = 0;
    t.each = each;
    int64_t items = 0, before = 0;
    const int64_t most = kOptEntryMost / each * each;
    for (int32_t i = 0; i < count; ++i) {
        if (!of(i)) continue;
        for (int64_t at = 0; at < numel[i]; at += most) {
            const int64_t n = numel[i] - at < most ? numel[i] - at : most;
            for (int k = 0; k < PTRS; ++k) t.p[k][t.count] = (char *)ptrs[k][i] + at * bytes[k];
            t.numel[t.count] = (uint32_t)n;
            t.first[t.count] = (uint32_t)items;
            items += ceil_div(n, each);
            // (an entry has 2^30 / each items at most, and a launch's threads are counted in 32 bits)
            if (++t.count == table_entries<PTRS>() || items >= ((int64_t)1 << 22)) {
                const int rc = launch(t, before, items);
                if (rc) return rc;
                before += items;
                items = 0;
                t.count = 0;
            }
        }
    }
    return t.count ? launch(t, before, items) : SPICE_OK;
}

// Calls of few elements, whose latency counts: one workgroup's work.  Its 1024 threads read 32 elements each.
constexpr int64_t kOptHere = 32768;
constexpr uint32_t kOptHereItem = 512;

bool few(const int64_t *numel, int32_t count, int entries) {
    int64_t total = 0;
    if (count > entries) return false;
    for (int32_t i = 0; i < count; ++i)
        if ((total += numel[i]) > kOptHere) return false;
    return true;
}

bool pointers_ok(void *const *p, const int64_t *numel, int32_t count, int64_t bytes) {
    if (count && !p) return false;
    for (int32_t i = 0; i < count; ++i)
        if (numel[i] && (!p[i] || (reinterpret_cast<uintptr_t>(p[i]) & (uintptr_t)(bytes - 1)))) return false;
    return true;
}

bool on4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

int64_t type_bytes(int32_t dtype) { return dtype == 0 ? 4 : 2; }

template <typename T>
int launch_norm(void *const *grads, const int64_t *numel, int32_t count, int inf, double *part, hipStream_t s, OfType of = {}) {
    void *const *const p[1] = {grads};
    const int64_t b[1] = {(int64_t)sizeof(T)};
    const auto launch = [&](const TableOf<1> &t, int64_t before, int64_t items) {
        if (inf)
            grad_norm_kernel<T, true><<<(unsigned)items, kOptThreads, 0, s>>>(t, part + before);
        else
            grad_norm_kernel<T, false><<<(unsigned)items, kOptThreads, 0, s>>>(t, part + before);
        SPICE_LAUNCH_CHECK();
        return (int)SPICE_OK;
    };
    return for_tables<1>(p, b, numel, count, item_elements(numel, count), launch, of);
}

template <typename T>
int launch_norm_here(void *const *grads, const int64_t *numel, int32_t count, const RecordArgs &a, hipStream_t s) {
    void *const *const p[1] = {grads};
    const int64_t b[1] = {(int64_t)sizeof(T)};
    bool done = false;
    const auto launch = [&](const TableOf<1> &t, int64_t, int64_t items) {
        if (a.inf)
            grad_here_kernel<T, T, true, false><<<1, kOptFold, 0, s>>>(t, (int32_t)items, a);
        else
            grad_here_kernel<T, T, false, false><<<1, kOptFold, 0, s>>>(t, (int32_t)items, a);
        done = true;
        SPICE_LAUNCH_CHECK();
        return (int)SPICE_OK;
    };
    const int rc = for_tables<1>(p, b, numel, count, kOptHereItem, launch);
    if (rc || done) return rc;
    TableOf<1> none;      // (no elements at all: a norm of 0)
    none.count = 0;
    none.each = kOptHereItem;
    return launch(none, 0, 0);
}

template <typename T, typename O>
int launch_clip_here(void *const *grads, void *const *out, const int64_t *numel, int32_t count, const RecordArgs &a, hipStream_t s) {
    void *const *const p[2] = {grads, out};
    const int64_t b[2] = {(int64_t)sizeof(T), (int64_t)sizeof(O)};
    bool done = false;
    const auto launch = [&](const TableOf<2> &t, int64_t, int64_t items) {
        if (a.inf)
            grad_here_kernel<T, O, true, true><<<1, kOptFold, 0, s>>>(t, (int32_t)items, a);
        else
            grad_here_kernel<T, O, false, true><<<1, kOptFold, 0, s>>>(t, (int32_t)items, a);
        done = true;
        SPICE_LAUNCH_CHECK();
        return (int)SPICE_OK;
    };
    const int rc = for_tables<2>(p, b, numel, count, kOptHereItem, launch);
    if (rc || done) return rc;
    TableOf<2> none;
    none.count = 0;
    none.each = kOptHereItem;
    return launch(none, 0, 0);
}

template <typename T, typename O>
int launch_clip(void *const *grads, void *const *out, const int64_t *numel, int32_t count, const float *record, hipStream_t s) {
    void *const *const p[2] = {grads, out};
    const int64_t b[2] = {(int64_t)sizeof(T), (int64_t)sizeof(O)};
    return for_tables<2>(p, b, numel, count, kClipItem, [&](const TableOf<2> &t, int64_t, int64_t items) {
        grad_clip_kernel<T, O><<<(unsigned)items, kOptThreads, 0, s>>>(t, record);
        SPICE_LAUNCH_CHECK();
        return (int)SPICE_OK;
    });
}

template <typename T>
int launch_adam(void *const *params, void *const *grads, void *const *m, void *const *v, const int64_t *numel, int32_t count,
                const AdamArgs &a, const float *record, hipStream_t s) {
    void *const *const p[4] = {params, grads, m, v};
    const int64_t b[4] = {(int64_t)sizeof(T), (int64_t)sizeof(T), 4, 4};
    return for_tables<4>(p, b, numel, count, kAdamItem, [&](const TableOf<4> &t, int64_t, int64_t items) {
        adam_kernel<T><<<(unsigned)items, kOptThreads, 0, s>>>(t, a, record);
        SPICE_LAUNCH_CHECK();
        return (int)SPICE_OK;
    });
}

}  // namespace
}  // namespace spice

using namespace spice;

extern "C" size_t spice_grad_norm_workspace_bytes(const int64_t *numel, int32_t count) {
    if (!counts_ok(numel, count)) return 0;
    return (size_t)(item_count(numel, count, item_elements(numel, count)) * (int64_t)sizeof(double) + 64);
}

namespace spice {
namespace {

// The record from the items' sums.
int record_of(RecordArgs &a, const double *part, const int64_t *numel, int32_t count, hipStream_t s) {
    a.part = part;
    a.parts = item_count(numel, count, item_elements(numel, count));
    grad_record_kernel<<<1, kOptFold, 0, s>>>(a);
    SPICE_LAUNCH_CHECK();
    return SPICE_OK;
}

// The norm of the call's gradients and the record from it.
int norm_and_record(void *const *grads, const int64_t *numel, int32_t count, int32_t dtype, RecordArgs &a, double *part,
                    hipStream_t s) {
    if (few(numel, count, table_entries<1>()))
        return dtype == 0   ? launch_norm_here<float>(grads, numel, count, a, s)
               : dtype == 1 ? launch_norm_here<_Float16>(grads, numel, count, a, s)
                            : launch_norm_here<__bf16>(grads, numel, count, a, s);
    const int rc = dtype == 0   ? launch_norm<float>(grads, numel, count, a.inf, part, s)
                   : dtype == 1 ? launch_norm<_Float16>(grads, numel, count, a.inf, part, s)
                                : launch_norm<__bf16>(grads, numel, count, a.inf, part, s);
    if (rc) return rc;
    return record_of(a, part, numel, count, s);
}

// The same over tensors of several types: each type's launches leave their part of the items' sums, joined in fp64 like the
// rest.  (Norms per type, rounded to fp32 and joined there: squares of 3e19 overflow, and of 3e-25 vanish.)
int norm_of_types(void *const *grads, const int32_t *dtypes, const int64_t *numel, int32_t count, RecordArgs &a, double *part,
                  hipStream_t s) {
    const uint32_t each = item_elements(numel, count);
    for (int32_t dtype = 0; dtype <= 2; ++dtype) {
        const OfType of = {dtypes, dtype};
        const int rc = dtype == 0   ? launch_norm<float>(grads, numel, count, a.inf, part, s, of)
                       : dtype == 1 ? launch_norm<_Float16>(grads, numel, count, a.inf, part, s, of)
                                    : launch_norm<__bf16>(grads, numel, count, a.inf, part, s, of);
        if (rc) return rc;
        part += item_count(numel, count, each, of);
    }
    return record_of(a, part - item_count(numel, count, each), numel, count, s);
}
bool norm_ok(void *const *grads, const int64_t *numel, int32_t count, int32_t dtype, int32_t norm_type, double max_norm,
             const float *record, const void *workspace) {
    return dtype >= 0 && dtype <= 2 && counts_ok(numel, count) && pointers_ok(grads, numel, count, type_bytes(dtype)) && record && on4(record) &&
           workspace && aligned8(workspace) && norm_type >= 0 && norm_type <= 1 && max_norm >= 0.0;
}

RecordArgs norm_record(int32_t norm_type, double max_norm, float *record) {
    RecordArgs a = {};
    a.inf = norm_type == SPICE_NORM_INF;
    a.clip = 1;
    a.max_norm = max_norm;
    a.record = record;
    return a;
}

}  // namespace
}  // namespace spice

extern "C" int spice_grad_norm(void *const *grads, const int64_t *numel, int32_t count, int32_t dtype, int32_t norm_type,
                               double max_norm, float *record, void *workspace, size_t workspace_bytes, void *stream) {
    if (!norm_ok(grads, numel, count, dtype, norm_type, max_norm, record, workspace)) return SPICE_ERR_ARG;
    if (workspace_bytes < spice_grad_norm_workspace_bytes(numel, count)) return SPICE_ERR_WORKSPACE;
    RecordArgs a = norm_record(norm_type, max_norm, record);
    return norm_and_record(grads, numel, count, dtype, a, (double *)workspace, (hipStream_t)stream);
}

extern "C" int spice_grad_norm_of_types(void *const *grads, const int32_t *dtypes, const int64_t *numel, int32_t count,
                                        int32_t norm_type, double max_norm, float *record, void *workspace, size_t workspace_bytes,
                                        void *stream) {
    if (!norm_ok(grads, numel, count, 1, norm_type, max_norm, record, workspace) || (count && !dtypes)) return SPICE_ERR_ARG;
    for (int32_t i = 0; i < count; ++i)
        if (dtypes[i] < 0 || dtypes[i] > 2 || !pointers_ok(grads + i, numel + i, 1, type_bytes(dtypes[i]))) return SPICE_ERR_ARG;
    if (workspace_bytes < spice_grad_norm_workspace_bytes(numel, count)) return SPICE_ERR_WORKSPACE;
    RecordArgs a = norm_record(norm_type, max_norm, record);
    return norm_of_types(grads, dtypes, numel, count, a, (double *)workspace, (hipStream_t)stream);
}

extern "C" int spice_grad_norm_clip(void *const *grads, int32_t dtype, void *const *out, int32_t out_dtype, const int64_t *numel,
                                    int32_t count, int32_t norm_type, double max_norm, float *record, void *workspace,
                                    size_t workspace_bytes, void *stream) {
    if (!norm_ok(grads, numel, count, dtype, norm_type, max_norm, record, workspace) || !(out_dtype == dtype || out_dtype == 0) ||
        !pointers_ok(out, numel, count, type_bytes(out_dtype)))
        return SPICE_ERR_ARG;
    if (workspace_bytes < spice_grad_norm_workspace_bytes(numel, count)) return SPICE_ERR_WORKSPACE;
    RecordArgs a = norm_record(norm_type, max_norm, record);
    hipStream_t s = (hipStream_t)stream;
    if (few(numel, count, table_entries<2>())) {
        if (dtype == 0) return launch_clip_here<float, float>(grads, out, numel, count, a, s);
        if (dtype == 1)
            return out_dtype == 0 ? launch_clip_here<_Float16, float>(grads, out, numel, count, a, s)
                                  : launch_clip_here<_Float16, _Float16>(grads, out, numel, count, a, s);
        return out_dtype == 0 ? launch_clip_here<__bf16, float>(grads, out, numel, count, a, s)
                              : launch_clip_here<__bf16, __bf16>(grads, out, numel, count, a, s);
    }
    const int rc = norm_and_record(grads, numel, count, dtype, a, (double *)workspace, s);
    return rc ? rc : spice_grad_clip(grads, dtype, out, out_dtype, numel, count, record, stream);
}

extern "C" int spice_grad_clip(void *const *grads, int32_t dtype, void *const *out, int32_t out_dtype, const int64_t *numel,
                               int32_t count, const float *record, void *stream) {
    if (dtype < 0 || dtype > 2 || !(out_dtype == dtype || out_dtype == 0) || !counts_ok(numel, count) ||
        !pointers_ok(grads, numel, count, type_bytes(dtype)) || !pointers_ok(out, numel, count, type_bytes(out_dtype)) || !record ||
        !on4(record))
        return SPICE_ERR_ARG;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == 0) return launch_clip<float, float>(grads, out, numel, count, record, s);
    if (dtype == 1)
        return out_dtype == 0 ? launch_clip<_Float16, float>(grads, out, numel, count, record, s)
                              : launch_clip<_Float16, _Float16>(grads, out, numel, count, record, s);
    return out_dtype == 0 ? launch_clip<__bf16, float>(grads, out, numel, count, record, s)
                          : launch_clip<__bf16, __bf16>(grads, out, numel, count, record, s);
}

extern "C" int spice_adam_step_opts(void *const *params, void *const *grads, void *const *exp_avg, void *const *exp_avg_sq,
                                    const int64_t *numel, int32_t count, int32_t dtype, const spice_adam_options *p,
                                    const float *norm, int64_t *step, float *record, void *workspace, size_t workspace_bytes,
                                    void *stream) {
    if (dtype < 0 || dtype > 2 || !p || !counts_ok(numel, count) || !pointers_ok(params, numel, count, type_bytes(dtype)) ||
        !pointers_ok(grads, numel, count, type_bytes(dtype)) || !pointers_ok(exp_avg, numel, count, 4) ||
        !pointers_ok(exp_avg_sq, numel, count, 4) || !record || !(p->lr >= 0.0 && p->lr <= 1e30) ||
        !(p->beta1 >= 0.0 && p->beta1 < 1.0) || !(p->beta2 >= 0.0 && p->beta2 < 1.0) || !(p->eps >= 0.0) ||
        !(p->weight_decay >= 0.0) || (!step && p->step < 1) || p->max_norm != p->max_norm || !on4(record) ||
        !on4(norm) || !aligned8(step))
        return SPICE_ERR_ARG;
    const bool clip = p->max_norm >= 0.0, take = clip && !norm;
    if (take && (!workspace || !aligned8(workspace))) return SPICE_ERR_ARG;
    if (take && workspace_bytes < spice_grad_norm_workspace_bytes(numel, count)) return SPICE_ERR_WORKSPACE;
    hipStream_t s = (hipStream_t)stream;
    RecordArgs r = {};
    r.norm_in = clip ? norm : nullptr;
    r.clip = clip;
    r.adam = 1;
    r.max_norm = p->max_norm;
    r.lr = p->lr;
    r.beta1 = p->beta1;
    r.beta2 = p->beta2;
    r.host_step = p->step;
    r.step = step;
    r.record = record;
    AdamArgs a = {};
    a.a1 = (float)(1.0 - p->beta1);
    a.a2 = (float)(1.0 - p->beta2);
    a.eps = (float)p->eps;
    a.decay = p->decoupled ? 0.f : (float)p->weight_decay;
    a.keep = p->decoupled ? (float)(1.0 - p->lr * p->weight_decay) : 1.f;
    if (take) {
        const int rc = norm_and_record(grads, numel, count, dtype, r, (double *)workspace, s);
        if (rc) return rc;
    } else if (clip || step) {
        grad_record_kernel<<<1, kOptFold, 0, s>>>(r);
        SPICE_LAUNCH_CHECK();
    } else {    // nothing that only the device knows
        a.rate = (float)(p->lr / (1.0 - pow(p->beta1, (double)p->step)));
        a.root = (float)(1.0 / sqrt(1.0 - pow(p->beta2, (double)p->step)));
        record = nullptr;
    }
    return dtype == 0   ? launch_adam<float>(params, grads, exp_avg, exp_avg_sq, numel, count, a, record, s)
           : dtype == 1 ? launch_adam<_Float16>(params, grads, exp_avg, exp_avg_sq, numel, count, a, record, s)
                        : launch_adam<__bf16>(params, grads, exp_avg, exp_avg_sq, numel, count, a, record, s);
}

extern "C" int spice_adam_step(void *const *params, void *const *grads, void *const *exp_avg, void *const *exp_avg_sq,
                               const int64_t *numel, int32_t count, int32_t dtype, const spice_adam_params *p,
                               const float *norm, int64_t *step, float *record, void *workspace, size_t workspace_bytes,
                               void *stream) {
    if (!p) return SPICE_ERR_ARG;
    const spice_adam_options o = {p->lr, p->beta1, p->beta2, p->eps, p->weight_decay, p->max_norm, p->step, p->decoupled, 0};
    return spice_adam_step_opts(params, grads, exp_avg, exp_avg_sq, numel, count, dtype, &o, norm, step, record, workspace,
                                workspace_bytes, stream);
}
