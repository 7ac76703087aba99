// logits.cu -- operators on rows of class logits held on the device.
//
//   cbgpu_top_logits      a row's k largest logits and the log-sum-exp of the rest
//   cbgpu_distill         Kullback-Leibler loss of a student row against a teacher's top
//                         logits, and its derivative
//   cbgpu_sample_classes  a class drawn from a row under temperature / top-k / top-p / min-p
//
// Rows come from a booster (f64 approximants, few classes, stored class by
// class) or from a neural teacher or student (16 or 32 bits, up to kLgMaxClasses
// classes, stored row by row).  The three operators read each row once or
// twice and are bound by that traffic, so one launch does all of an operator.
//
// Two shapes of kernel:
//   narrow (<= kLgNarrow classes)  a block stages a tile of rows in shared memory, then 1, 8 or 32
//                                  lanes work on each row;
//   wide                           a block works on one row.
// Order of classes: larger logit first, equal logits by lower index, NaN last.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "../../include/cbgpu.h"
#include "cbgpu_common.cuh"

namespace cbgpu {
int record_error(int code, const char* msg);  // session.cu: sets cbgpu_last_error()
}

namespace {

constexpr int kLgMaxClasses = 262144;
constexpr int kLgMaxTop = 256;
constexpr int kLgNarrow = 1024;
constexpr int kLgThreads = 256;

int lfail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return cbgpu::record_error(code, buf);
}

// ---- number types ------------------------------------------------------------

typedef unsigned long long u64;

template <typename T>
struct Num {  // 16- and 32-bit logits: arithmetic in f32, 32-bit order keys
    typedef float C;
    typedef uint32_t Key;
};
template <>
struct Num<double> {
    typedef double C;
    typedef u64 Key;
};

__device__ __forceinline__ double to_c(double v) { return v; }
__device__ __forceinline__ float to_c(float v) { return v; }
__device__ __forceinline__ float to_c(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_c(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_c(typename Num<T>::C v);
template <>
__device__ __forceinline__ double from_c<double>(double v) { return v; }
template <>
__device__ __forceinline__ float from_c<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_c<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_c<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Order keys: larger logit, larger key; -0 and +0 share one; NaN is 0, below -inf.
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return v != v ? 0u : ((b >> 31) ? ~b : (b | 0x80000000u));
}
__device__ __forceinline__ u64 key_of(double v) {
    const u64 b = (u64)__double_as_longlong(v + 0.0);
    return v != v ? 0ull : ((b >> 63) ? ~b : (b | 0x8000000000000000ull));
}

__device__ __forceinline__ float lg_inf(float) { return __int_as_float(0x7f800000); }
__device__ __forceinline__ double lg_inf(double) { return __longlong_as_double(0x7ff0000000000000ll); }

// exp((a - m) / T).  f32: 2^((a - m) c) with c = log2(e) / T rounded to f32 (a relative change of the
// temperature by at most 2^-24, taken for teacher and student alike).
__device__ __forceinline__ float lg_exp(float d, float c) { return exp2f(d * c); }
__device__ __forceinline__ double lg_exp(double d, double c) { return exp(d * c); }
template <typename C>
struct Scale;
template <>
struct Scale<float> {
    float c;
    double inv_t;  // the 1 / T that c stands for
    __host__ explicit Scale(double t) : c((float)(1.4426950408889634 / t)), inv_t((double)c * 0.6931471805599453) {}
};
template <>
struct Scale<double> {
    double c, inv_t;
    __host__ explicit Scale(double t) : c(1.0 / t), inv_t(1.0 / t) {}
};

struct OpMax {
    template <typename V>
    __device__ V operator()(V a, V b) const { return a > b ? a : b; }
    __device__ float operator()(float a, float b) const { return fmaxf(a, b); }  // drops a NaN
    __device__ double operator()(double a, double b) const { return fmax(a, b); }
};
struct OpMin {
    template <typename V>
    __device__ V operator()(V a, V b) const { return a < b ? a : b; }
};
struct OpSum {
    template <typename V>
    __device__ V operator()(V a, V b) const { return a + b; }
};
struct OpOr {
    template <typename V>
    __device__ V operator()(V a, V b) const { return a | b; }
};

// ---- teams: the threads that share one row -----------------------------------

template <int G>  // G lanes of a warp
struct LaneTeam {
    static constexpr int size = G;
    int rank;
    unsigned mask;
    __device__ LaneTeam() {
        const int lane = threadIdx.x & 31;
        rank = lane & (G - 1);
        mask = G == 32 ? 0xffffffffu : (((1u << (G & 31)) - 1u) << (lane & ~(G - 1)));
    }
    __device__ void sync() const {
        if (G > 1) __syncwarp(mask);
    }
    template <typename V, typename Op>
    __device__ V reduce(V v, Op op) const {
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(mask, v, o));
        return v;
    }
    __device__ u64 exscan(u64 v) const {
        u64 inc = v;
#pragma unroll
        for (int o = 1; o < G; o <<= 1) {
            const u64 t = __shfl_up_sync(mask, inc, o, G);
            if (rank >= o) inc += t;
        }
        return inc - v;
    }
};

struct BlockTeam {  // a whole block of kLgThreads
    static constexpr int size = kLgThreads;
    int rank;
    u64* scratch;  // [kLgThreads / 32 + 1]
    __device__ explicit BlockTeam(u64* s) : rank(threadIdx.x), scratch(s) {}
    __device__ void sync() const { __syncthreads(); }
    template <typename V, typename Op>
    __device__ V reduce(V v, Op op) const {
        static_assert(sizeof(V) <= sizeof(u64), "scratch word");
        V* s = reinterpret_cast<V*>(scratch);
        for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
        if ((rank & 31) == 0) s[rank >> 5] = v;
        __syncthreads();
        V r = s[0];
        for (int w = 1; w < size / 32; ++w) r = op(r, s[w]);
        __syncthreads();
        return r;
    }
    __device__ u64 exscan(u64 v) const {
        u64 inc = v;
        for (int o = 1; o < 32; o <<= 1) {
            const u64 t = __shfl_up_sync(0xffffffffu, inc, o);
            if ((rank & 31) >= o) inc += t;
        }
        if ((rank & 31) == 31) scratch[rank >> 5] = inc;
        __syncthreads();
        u64 base = 0;
        for (int w = 0; w < (rank >> 5); ++w) base += scratch[w];
        __syncthreads();
        return base + inc - v;
    }
};

// ---- launch arguments ----------------------------------------------------------

template <typename T>
struct Rows {
    const T* data;
    int64_t n, row_stride, class_stride;
    int V;
};

// A logit of the teacher's lists, whatever its type.
__device__ __forceinline__ double load_any(const void* p, int dtype, int64_t i) {
    switch (dtype) {
        case CBGPU_F64: return ((const double*)p)[i];
        case CBGPU_F32: return (double)((const float*)p)[i];
        case CBGPU_F16: return (double)__half2float(((const __half*)p)[i]);
        default: return (double)__bfloat162float(((const __nv_bfloat16*)p)[i]);
    }
}

struct TeacherArgs {
    const void *index, *value;
    int index_bytes, value_dtype, k;
    __device__ int64_t idx(int64_t at) const {
        return index_bytes == 8 ? ((const int64_t*)index)[at] : (int64_t)((const int32_t*)index)[at];
    }
};

struct SampleArgs {
    const void* uniform;
    int uniform_dtype, top_k;
    double temperature, top_p, min_p;
    const float *temperature_rows, *top_p_rows, *min_p_rows;
    const int32_t* top_k_rows;
};

// Rows staged as [rows][V] in shared memory, `pitch` elements apart.  The
// loop runs along the axis that is closer in memory.
template <typename T, bool kStore>
__device__ __forceinline__ void tile_copy(T* s, int pitch, int rows, int V, T* g, int64_t rs, int64_t cs) {
    const uint32_t total = (uint32_t)rows * (uint32_t)V;
    if (cs <= rs) {
        for (uint32_t e = threadIdx.x; e < total; e += blockDim.x) {
            const uint32_t r = e / (uint32_t)V, c = e - r * (uint32_t)V;
            if (kStore) g[(int64_t)r * rs + (int64_t)c * cs] = s[r * pitch + c];
            else s[r * pitch + c] = g[(int64_t)r * rs + (int64_t)c * cs];
        }
    } else {
        for (uint32_t e = threadIdx.x; e < total; e += blockDim.x) {
            const uint32_t c = e / (uint32_t)rows, r = e - c * (uint32_t)rows;
            if (kStore) g[(int64_t)r * rs + (int64_t)c * cs] = s[r * pitch + c];
            else s[r * pitch + c] = g[(int64_t)r * rs + (int64_t)c * cs];
        }
    }
}

// ---- top logits ------------------------------------------------------------------

template <typename Key>
struct Ranked {  // a class in the operators' order
    Key key;
    uint32_t idx;
    __device__ bool before(const Ranked& o) const { return key > o.key || (key == o.key && idx < o.idx); }
};
template <typename Team, typename Key>
__device__ __forceinline__ Ranked<Key> team_first(const Team& t, Ranked<Key> v) {
    Ranked<Key> r;
    r.key = t.reduce(v.key, OpMax());
    r.idx = t.reduce(v.key == r.key ? v.idx : 0xffffffffu, OpMin());
    return r;
}

// k rounds, each taking the first class after the one before it; then the
// log-sum-exp of what is left, relative to its own largest.
template <typename T, typename Team, typename Get>
__device__ void top_row(const Team& t, Get get, int V, int k, Scale<typename Num<T>::C> sc, T* value, int32_t* index,
                        typename Num<T>::C* tail) {
    typedef typename Num<T>::C C;
    typedef typename Num<T>::Key Key;
    Ranked<Key> last{~(Key)0, 0u};  // before every class: no logit has the all-ones key
    for (int j = 0; j < k + (tail ? 1 : 0); ++j) {
        Ranked<Key> best{0, 0xffffffffu};
        for (int i = t.rank; i < V; i += t.size) {
            const Ranked<Key> r{key_of(to_c(get(i))), (uint32_t)i};
            if (last.before(r) && r.before(best)) best = r;
        }
        best = team_first(t, best);
        if (j == k) {  // the largest of the rest
            C sum = 0;
            const C top = best.idx < (uint32_t)V ? to_c(get((int)best.idx)) : -lg_inf(C());
            const bool some = top > -lg_inf(C());
            int bad = 0;
            double acc = 0.0;
            for (int i = t.rank; i < V; i += t.size) {
                const C a = to_c(get(i));
                bad |= a != a;
                const Ranked<Key> r{key_of(a), (uint32_t)i};
                if (last.before(r) && some) {
                    sum = lg_exp(a - top, sc.c);
                    acc += (double)sum;
                }
            }
            bad = t.reduce(bad, OpOr());
            acc = t.reduce(acc, OpSum());
            if (t.rank == 0) {
                const double v = bad ? (double)lg_inf(C()) - (double)lg_inf(C())
                                     : (some ? (double)top * sc.inv_t + log(acc) : -(double)lg_inf(C()));
                *tail = (C)v;
            }
            return;
        }
        if (t.rank == 0) {
            value[j] = get((int)best.idx);
            index[j] = (int32_t)best.idx;
        }
        last = best;
    }
}

template <typename T, int G>
__global__ void __launch_bounds__(kLgThreads)
lg_top_narrow_kernel(Rows<T> x, int k, Scale<typename Num<T>::C> sc, int tile, int pitch, T* __restrict__ value,
                     int32_t* __restrict__ index, typename Num<T>::C* __restrict__ tail) {
    extern __shared__ __align__(16) unsigned char lg_smem[];
    T* s = reinterpret_cast<T*>(lg_smem);
    const int64_t r0 = (int64_t)blockIdx.x * tile;
    const int rows = (int)(x.n - r0 < tile ? x.n - r0 : tile);
    tile_copy<T, false>(s, pitch, rows, x.V, const_cast<T*>(x.data) + r0 * x.row_stride, x.row_stride, x.class_stride);
    __syncthreads();
    const LaneTeam<G> t;
    for (int r = threadIdx.x / G; r < rows; r += kLgThreads / G) {
        const T* row = s + (size_t)r * pitch;
        top_row<T>(t, [&](int i) { return row[i]; }, x.V, k, sc, value + (r0 + r) * k, index + (r0 + r) * k,
                   tail ? tail + r0 + r : nullptr);
    }
}

template <typename T>
__global__ void __launch_bounds__(kLgThreads)
lg_top_wide_kernel(Rows<T> x, int k, Scale<typename Num<T>::C> sc, T* __restrict__ value, int32_t* __restrict__ index,
                   typename Num<T>::C* __restrict__ tail) {
    __shared__ u64 scratch[kLgThreads / 32 + 1];
    const BlockTeam t(scratch);
    const int64_t r = blockIdx.x;
    const T* row = x.data + r * x.row_stride;
    const int64_t cs = x.class_stride;
    top_row<T>(t, [&](int i) { return row[(int64_t)i * cs]; }, x.V, k, sc, value + r * k, index + r * k,
               tail ? tail + r : nullptr);
}

// ---- distillation ------------------------------------------------------------------
//
// Row a[V], temperature T, weight w; the teacher's buckets are its k top
// classes (their distinct valid indices S, the first entry of an index
// counting) and all others together (tail = their log-sum-exp at T):
//   q, Q  = softmax over (z_j / T, tail);  p = softmax(a / T);  P = sum of p outside S
//   loss  = w T^2 [ sum_S q ln(q / p) + Q ln(Q / P) ]
//   der1  = -d loss / d a = w T (q_i - p_i) in S,  -w T p_i (1 - Q / P) outside.
// With e_i = exp((a_i - m) / T), s their sum, s_t the sum outside S, r_j the
// teacher's exponentials and R their sum, the loss is
//   w T^2 [ (sum r_j (z_j - z_max - a_j + m) / T + r_t (tail - z_max / T - ln s_t)) / R - ln R + ln s ]:
// no difference of logarithms of rounded sums but ln s - ln R, both taken in 64 bits.

// A maximum that is subtracted: 0 where there is no class, so that the exponentials are 0 there.
template <typename C>
__device__ __forceinline__ C floor_max(C m) { return m == -lg_inf(C()) ? C(0) : m; }

template <typename C>
struct RowOut {  // what turns a row's logits into its loss and derivative
    double loss;
    C c_top, c_rest, q_scale;  // der1 = q_scale * r_i - c_top * e_i in S, -c_rest * e_i outside
    bool zero;
};

template <typename C>
__device__ __forceinline__ RowOut<C> distill_finish(double w, double t, double s_top, double s_rest, double r_sum,
                                                    double r_tail, double tail_rel, double cross) {
    RowOut<C> o{};
    const double s = s_top + s_rest;
    o.zero = s == 0.0 || r_sum == 0.0;  // every class masked (m is 0 then), or a teacher without an entry
    if (o.zero) return o;
    double kl = cross;
    if (r_tail > 0.0 || r_tail != r_tail) kl += r_tail * (tail_rel - log(s_rest));
    o.loss = w * t * t * (kl / r_sum - log(r_sum) + log(s));
    const double wt = w * t;
    o.q_scale = (C)(wt / r_sum);
    o.c_top = (C)(wt / s);
    const double q = r_tail / r_sum;
    o.c_rest = (C)(wt * (1.0 / s - (q != 0.0 && s_rest != 0.0 ? q / s_rest : (q != q ? q : 0.0))));
    return o;
}

constexpr uint32_t kAbsent32 = 0xffffffffu;  // a NaN no arithmetic gives
constexpr u64 kAbsent64 = ~0ull;
__device__ __forceinline__ bool is_absent(float v) { return __float_as_uint(v) == kAbsent32; }
__device__ __forceinline__ bool is_absent(double v) { return (u64)__double_as_longlong(v) == kAbsent64; }
__device__ __forceinline__ void set_absent(float* p) { *(uint32_t*)p = kAbsent32; }
__device__ __forceinline__ void set_absent(double* p) { *(u64*)p = kAbsent64; }
__device__ __forceinline__ float plain_nan(float v) { return v != v ? __int_as_float(0x7fc00000) : v; }
__device__ __forceinline__ double plain_nan(double v) {
    return v != v ? __longlong_as_double(0x7ff8000000000000ll) : v;
}

// tgt[i] = the teacher's logit of class i, or absent.
template <typename T, int G>
__global__ void __launch_bounds__(kLgThreads)
lg_distill_narrow_kernel(Rows<T> x, TeacherArgs tc, const typename Num<T>::C* __restrict__ tail,
                         const typename Num<T>::C* __restrict__ weight, double temp, Scale<typename Num<T>::C> sc,
                         int tile, int pitch, typename Num<T>::C* __restrict__ loss, T* der1, int64_t drs,
                         int64_t dcs) {
    typedef typename Num<T>::C C;
    extern __shared__ __align__(16) unsigned char lg_smem[];
    C* tgt_all = reinterpret_cast<C*>(lg_smem);
    T* s = reinterpret_cast<T*>(tgt_all + (size_t)tile * pitch);
    const int64_t r0 = (int64_t)blockIdx.x * tile;
    const int rows = (int)(x.n - r0 < tile ? x.n - r0 : tile);
    const int V = x.V;
    tile_copy<T, false>(s, pitch, rows, V, const_cast<T*>(x.data) + r0 * x.row_stride, x.row_stride, x.class_stride);
    __syncthreads();
    const LaneTeam<G> t;
    for (int r = threadIdx.x / G; r < rows; r += kLgThreads / G) {
        T* row = s + (size_t)r * pitch;
        C* tgt = tgt_all + (size_t)r * pitch;
        const double w = weight ? (double)weight[r0 + r] : 1.0;
        for (int i = t.rank; i < V; i += G) set_absent(&tgt[i]);
        t.sync();
        for (int j0 = 0; j0 < tc.k && w != 0.0; j0 += G) {
            const int j = j0 + t.rank;
            const int64_t at = (r0 + r) * tc.k + j;
            const int64_t idx = j < tc.k ? tc.idx(at) : -1;
            bool take = idx >= 0 && idx < V;
            if (G > 1) {  // of equal indices in this step the first counts
                const unsigned same = __match_any_sync(t.mask, take ? (int)idx : -1 - t.rank);
                take = take && (__ffs(same) - 1) == (int)(threadIdx.x & 31);
            }
            if (take && is_absent(tgt[idx])) tgt[idx] = plain_nan((C)load_any(tc.value, tc.value_dtype, at));
            t.sync();
        }
        C m = -lg_inf(C()), zm = -lg_inf(C());
        for (int i = t.rank; i < V; i += G) {
            m = OpMax()(m, to_c(row[i]));
            if (!is_absent(tgt[i])) zm = OpMax()(zm, tgt[i]);
        }
        m = floor_max(t.reduce(m, OpMax()));
        zm = t.reduce(zm, OpMax());
        const double tl = tail ? (double)tail[r0 + r] : -lg_inf(0.0);
        const double z_max = floor_max(fmax((double)zm * sc.inv_t, tl));
        double s_top = 0.0, s_rest = 0.0, r_sum = 0.0, cross = 0.0;
        for (int i = t.rank; i < V; i += G) {
            const C a = to_c(row[i]);
            const double e = (double)lg_exp(a - m, sc.c);
            const C z = tgt[i];
            if (is_absent(z)) {
                s_rest += e;
                continue;
            }
            s_top += e;
            const double d = (double)z * sc.inv_t - z_max;
            const double rj = exp(d);
            r_sum += rj;
            if (rj != 0.0) cross += rj * (d - ((double)a - (double)m) * sc.inv_t);
        }
        s_top = t.reduce(s_top, OpSum());
        s_rest = t.reduce(s_rest, OpSum());
        r_sum = t.reduce(r_sum, OpSum());
        cross = t.reduce(cross, OpSum());
        const double r_tail = exp(tl - z_max);
        RowOut<C> o = distill_finish<C>(w, temp, s_top, s_rest, r_sum + r_tail, r_tail, tl - z_max, cross);
        if (w == 0.0) {
            o = RowOut<C>{};
            o.zero = true;
        }
        if (t.rank == 0) loss[r0 + r] = (C)o.loss;
        if (der1)
            for (int i = t.rank; i < V; i += G) {
                C d = 0;
                if (!o.zero) {
                    const C e = lg_exp(to_c(row[i]) - m, sc.c);
                    const C z = tgt[i];
                    d = is_absent(z) ? -o.c_rest * e
                                     : o.q_scale * (C)exp((double)z * sc.inv_t - z_max) - o.c_top * e;
                }
                row[i] = from_c<T>(d);
            }
    }
    if (der1) {
        __syncthreads();
        tile_copy<T, true>(s, pitch, rows, V, der1 + r0 * drs, drs, dcs);
    }
}

template <typename T>
__global__ void __launch_bounds__(kLgThreads)
lg_distill_wide_kernel(Rows<T> x, TeacherArgs tc, const typename Num<T>::C* __restrict__ tail,
                       const typename Num<T>::C* __restrict__ weight, double temp, Scale<typename Num<T>::C> sc,
                       typename Num<T>::C* __restrict__ loss, T* der1, int64_t drs, int64_t dcs) {
    typedef typename Num<T>::C C;
    extern __shared__ __align__(16) unsigned char lg_smem[];
    __shared__ u64 scratch[kLgThreads / 32 + 1];
    __shared__ C s_a[kLgMaxTop];
    __shared__ int s_idx[kLgMaxTop];
    uint32_t* in_top = reinterpret_cast<uint32_t*>(lg_smem);  // a bit for each class
    const BlockTeam t(scratch);
    const int64_t r = blockIdx.x;
    const int V = x.V, k = tc.k, tid = threadIdx.x;
    const T* row = x.data + r * x.row_stride;
    T* out = der1 ? der1 + r * drs : nullptr;
    const int64_t cs = x.class_stride;
    const double w = weight ? (double)weight[r] : 1.0;
    if (w == 0.0) {
        if (tid == 0) loss[r] = 0;
        if (out)
            for (int i = tid; i < V; i += kLgThreads) out[(int64_t)i * dcs] = from_c<T>(C(0));
        return;
    }
    static_assert(kLgThreads >= kLgMaxTop, "one thread an entry");
    for (int i = tid; i < (V + 31) / 32; i += kLgThreads) in_top[i] = 0u;
    if (tid < k) {
        const int64_t idx = tc.idx(r * k + tid);
        s_idx[tid] = idx >= 0 && idx < V ? (int)idx : -1;
    }
    __syncthreads();
    const double tl = tail ? (double)tail[r] : -lg_inf(0.0);
    double z = -lg_inf(0.0), z_max;
    bool mine = tid < k && s_idx[tid] >= 0;
    for (int j = 0; mine && j < tid; ++j) mine = s_idx[j] != s_idx[tid];  // the first entry of an index counts
    if (mine) {
        atomicOr(&in_top[s_idx[tid] >> 5], 1u << (s_idx[tid] & 31));
        z = (double)(C)load_any(tc.value, tc.value_dtype, r * k + tid) * sc.inv_t;
        s_a[tid] = to_c(row[(int64_t)s_idx[tid] * cs]);
    }
    z_max = t.reduce(z, OpMax());
    z_max = floor_max(fmax(z_max, tl));
    __syncthreads();
    C m = -lg_inf(C());
    for (int i = tid; i < V; i += kLgThreads) m = OpMax()(m, to_c(row[(int64_t)i * cs]));
    m = floor_max(t.reduce(m, OpMax()));
    double s_rest = 0.0;
    for (int i = tid; i < V; i += kLgThreads)
        if (!((in_top[i >> 5] >> (i & 31)) & 1u)) s_rest += (double)lg_exp(to_c(row[(int64_t)i * cs]) - m, sc.c);
    s_rest = t.reduce(s_rest, OpSum());
    double s_top = 0.0, rj = 0.0, cross = 0.0;
    if (mine) {
        const C a = s_a[tid];
        s_top = (double)lg_exp(a - m, sc.c);
        rj = exp(z - z_max);
        if (rj != 0.0) cross = rj * (z - z_max - ((double)a - (double)m) * sc.inv_t);
    }
    const double e_own = s_top, r_own = rj;
    s_top = t.reduce(s_top, OpSum());
    const double r_tail = exp(tl - z_max);
    const double r_sum = t.reduce(rj, OpSum()) + r_tail;
    cross = t.reduce(cross, OpSum());
    const RowOut<C> o = distill_finish<C>(w, temp, s_top, s_rest, r_sum, r_tail, tl - z_max, cross);
    if (tid == 0) loss[r] = (C)o.loss;
    if (!out) return;
    // der1 may be the logits' own memory: every read of a class is by the thread that writes it,
    // but for the teacher's classes, which were read above
    for (int i = tid; i < V; i += kLgThreads)
        if (!((in_top[i >> 5] >> (i & 31)) & 1u))
            out[(int64_t)i * dcs] =
                from_c<T>(o.zero ? C(0) : -o.c_rest * lg_exp(to_c(row[(int64_t)i * cs]) - m, sc.c));
    if (mine) out[(int64_t)s_idx[tid] * dcs] = from_c<T>(o.zero ? C(0) : o.q_scale * (C)r_own - o.c_top * (C)e_own);
}

// ---- sampling ------------------------------------------------------------------------
//
// e_i = exp((a_i - max) / T) is taken in 64 bits and held as the integer
// w_i = rint(e_i 2^s), with 2^s V <= 2^62, so that every sum of weights is exact
// whatever its order: the draw does not depend on the launch's shape, and a
// class is drawn as the 64-bit definition draws it unless the drawn number lies
// within V 2^-s of a border.
//   top-k   the first k classes in order
//   top-p   a class stays while the mass before it is below p times the mass top-k left
//   min-p   a class stays while e_i >= min_p
//   draw    the first class by index whose running kept mass exceeds u times the kept mass

struct RowSampling {
    double inv_t, top_p, min_p, u;
    int top_k;
    bool greedy;
};
__device__ __forceinline__ RowSampling row_sampling(const SampleArgs& a, int64_t r, int V) {
    RowSampling s;
    const double t = a.temperature_rows ? (double)a.temperature_rows[r] : a.temperature;
    s.greedy = !(t > 0.0);
    s.inv_t = 1.0 / fmin(t, 1e6);
    s.top_p = a.top_p_rows ? (double)a.top_p_rows[r] : a.top_p;
    s.min_p = a.min_p_rows ? (double)a.min_p_rows[r] : a.min_p;
    s.min_p = s.min_p > 1.0 ? 1.0 : s.min_p;  // the first class always stays
    s.top_k = a.top_k_rows ? a.top_k_rows[r] : a.top_k;
    if (s.top_k <= 0 || s.top_k > V) s.top_k = V;
    s.u = a.uniform_dtype == CBGPU_F64 ? ((const double*)a.uniform)[r] : (double)((const float*)a.uniform)[r];
    return s;
}

// The least kept mass that holds top-p's prefix: max(1, ceil(p S)), the product in 64-bit floating
// point (0.9 of 1000 equal classes is 900 of them, although 0.9 is a little more than 9 / 10).
__device__ __forceinline__ u64 mass_part(double p, u64 total) {
    const double v = ceil(p * (double)total);
    const u64 t = v > 0.0 ? (v < 9.2e18 ? (u64)v : total) : 1ull;
    return t < 1ull ? 1ull : (t > total ? total : t);
}
// floor(u S) + 1, at most S: the running mass that exceeds u S.  The product is exact (53 x 62 bits):
// a number that equals a border goes to the class behind it.
__device__ __forceinline__ u64 draw_target(double u, u64 total) {
    if (!(u > 0.0)) return 1ull;
    if (u >= 1.0) return total;
    const u64 bits = (u64)__double_as_longlong(u);
    const int ex = (int)(bits >> 52);  // u = man 2^-down; a subnormal u is below 2^-62
    if (ex < 1023 - 64) return 1ull;
    const u64 man = (bits & 0xfffffffffffffull) | 0x10000000000000ull;
    const int down = 1075 - ex;  // 53 .. 116
    const u64 hi = __umul64hi(man, total), lo = man * total;
    return (down >= 64 ? hi >> (down - 64) : (hi << (64 - down)) | (lo >> down)) + 1ull;
}

// The last class of the shortest prefix (in order) whose metric reaches
// `target`: bit by bit the largest key that still reaches it, then the
// lowest index among that key's classes.  metric(i, key) is 0 for what is out already.
template <typename Key, typename Team, typename Met, typename KeyAt>
__device__ Ranked<Key> team_select(const Team& t, int V, u64 target, KeyAt key_at, Met metric) {
    Key key = 0;
    for (int b = (int)sizeof(Key) * 8 - 1; b >= 0; --b) {
        const Key cand = key | ((Key)1 << b);
        u64 f = 0;
        for (int i = t.rank; i < V; i += t.size) {
            const Key ki = key_at(i);
            if (ki >= cand) f += metric(i, ki);
        }
        if (t.reduce(f, OpSum()) >= target) key = cand;
    }
    u64 above = 0;
    for (int i = t.rank; i < V; i += t.size) {
        const Key ki = key_at(i);
        if (ki > key) above += metric(i, ki);
    }
    const u64 need = target - t.reduce(above, OpSum());
    int bits = 0;
    while ((1 << bits) < V) ++bits;
    uint32_t idx = (1u << bits) - 1u;
    for (int b = bits - 1; b >= 0; --b) {
        const uint32_t cand = idx & ~(1u << b);
        u64 f = 0;
        for (int i = t.rank; i < V; i += t.size) {
            const Key ki = key_at(i);
            if (ki == key && (uint32_t)i <= cand) f += metric(i, ki);
        }
        if (t.reduce(f, OpSum()) >= need) idx = cand;
    }
    return Ranked<Key>{key, idx};
}

template <typename T, typename Team, typename Get>
__device__ int sample_row(const Team& t, Get get, int V, int shift, const RowSampling& rs) {
    typedef typename Num<T>::C C;
    typedef typename Num<T>::Key Key;
    C m = -lg_inf(C());
    int bad = 0;
    for (int i = t.rank; i < V; i += t.size) {
        const C a = to_c(get(i));
        bad |= a != a;
        m = OpMax()(m, a);
    }
    m = t.reduce(m, OpMax());
    bad = t.reduce(bad, OpOr());
    if (bad || m == -lg_inf(C())) return -1;
    if (rs.greedy) {
        uint32_t at = 0xffffffffu;
        for (int i = t.rank; i < V; i += t.size)
            if (to_c(get(i)) == m && (uint32_t)i < at) at = (uint32_t)i;
        return (int)t.reduce(at, OpMin());
    }
    const double scale = __longlong_as_double((long long)(1023 + shift) << 52);
    auto share = [&](int i) {  // infinite logits share the mass among themselves
        const C a = to_c(get(i));
        return a == m ? 1.0 : exp(((double)a - (double)m) * rs.inv_t);
    };
    auto mass = [&](int i) { return (u64)__double2ull_rn(share(i) * scale); };
    auto key_at = [&](int i) { return key_of(to_c(get(i))); };
    Ranked<Key> last{0, 0xffffffffu};  // the last class that stays
    auto stays = [&](int i, Key k) { return k > last.key || (k == last.key && (uint32_t)i <= last.idx); };
    if (rs.top_k < V)
        last = team_select<Key>(t, V, (u64)rs.top_k, key_at, [&](int, Key) { return 1ull; });
    if (rs.top_p < 1.0) {
        u64 total = 0;
        for (int i = t.rank; i < V; i += t.size)
            if (stays(i, key_at(i))) total += mass(i);
        total = t.reduce(total, OpSum());
        const Ranked<Key> cut = team_select<Key>(t, V, mass_part(rs.top_p, total), key_at,
                                                 [&](int i, Key k) { return stays(i, k) ? mass(i) : 0ull; });
        last = cut;
    }
    auto kept = [&](int i) {
        if (!stays(i, key_at(i))) return 0ull;
        if (rs.min_p > 0.0 && share(i) < rs.min_p) return 0ull;
        return mass(i);
    };
    const int per = (V + t.size - 1) / t.size;  // runs of classes by index
    const int i0 = t.rank * per < V ? t.rank * per : V, i1 = i0 + per < V ? i0 + per : V;
    u64 own = 0;
    for (int i = i0; i < i1; ++i) own += kept(i);
    u64 upto = t.exscan(own);
    const u64 total = t.reduce(own, OpSum());
    const u64 target = draw_target(rs.u, total);
    uint32_t at = 0xffffffffu;
    if (upto < target && upto + own >= target)
        for (int i = i0; i < i1; ++i) {
            upto += kept(i);
            if (upto >= target) {
                at = (uint32_t)i;
                break;
            }
        }
    return (int)t.reduce(at, OpMin());
}

template <typename T, int G>
__global__ void __launch_bounds__(kLgThreads)
lg_sample_narrow_kernel(Rows<T> x, SampleArgs a, int shift, int tile, int pitch, int32_t* __restrict__ index) {
    extern __shared__ __align__(16) unsigned char lg_smem[];
    T* s = reinterpret_cast<T*>(lg_smem);
    const int64_t r0 = (int64_t)blockIdx.x * tile;
    const int rows = (int)(x.n - r0 < tile ? x.n - r0 : tile);
    tile_copy<T, false>(s, pitch, rows, x.V, const_cast<T*>(x.data) + r0 * x.row_stride, x.row_stride, x.class_stride);
    __syncthreads();
    const LaneTeam<G> t;
    for (int r = threadIdx.x / G; r < rows; r += kLgThreads / G) {
        const T* row = s + (size_t)r * pitch;
        const int got = sample_row<T>(t, [&](int i) { return row[i]; }, x.V, shift, row_sampling(a, r0 + r, x.V));
        if (t.rank == 0) index[r0 + r] = got;
    }
}

template <typename T>
__global__ void __launch_bounds__(kLgThreads)
lg_sample_wide_kernel(Rows<T> x, SampleArgs a, int shift, int32_t* __restrict__ index) {
    __shared__ u64 scratch[kLgThreads / 32 + 1];
    const BlockTeam t(scratch);
    const int64_t r = blockIdx.x;
    const T* row = x.data + r * x.row_stride;
    const int64_t cs = x.class_stride;
    const int got = sample_row<T>(t, [&](int i) { return row[(int64_t)i * cs]; }, x.V, shift, row_sampling(a, r, x.V));
    if (t.rank == 0) index[r] = got;
}

// ---- host ------------------------------------------------------------------------------

size_t dtype_size(int d) { return d == CBGPU_F64 ? 8 : (d == CBGPU_F32 ? 4 : 2); }

int check_logits(const char* who, const cbgpu_logits* x) {
    if (!x) return lfail(CBGPU_ERR_INVALID, "%s: logits is NULL", who);
    if (x->dtype < CBGPU_F64 || x->dtype > CBGPU_BF16)
        return lfail(CBGPU_ERR_INVALID, "%s: dtype %d is not one of the cbgpu_dtype values", who, x->dtype);
    if (x->n < 0 || x->n > 0x7fffffffll)
        return lfail(CBGPU_ERR_INVALID, "%s: n = %lld rows is outside 0..2^31 - 1", who, (long long)x->n);
    if (x->n_classes < 1 || x->n_classes > kLgMaxClasses)
        return lfail(CBGPU_ERR_INVALID, "%s: n_classes = %d is outside 1..%d", who, x->n_classes, kLgMaxClasses);
    if (x->row_stride < 0 || x->class_stride < 0)
        return lfail(CBGPU_ERR_INVALID, "%s: negative strides", who);
    if (x->n > 0 && !x->data) return lfail(CBGPU_ERR_INVALID, "%s: logits.data is NULL", who);
    if ((uintptr_t)x->data % dtype_size(x->dtype) != 0)
        return lfail(CBGPU_ERR_INVALID, "%s: logits.data is not aligned to its type", who);
    return CBGPU_OK;
}

int check_temperature(const char* who, double t, bool zero_ok) {
    if (!(t > 0.0 || (zero_ok && t == 0.0)) || !(t < INFINITY) || (t > 0.0 && (t < 1e-6 || t > 1e6)))
        return lfail(CBGPU_ERR_INVALID, "%s: temperature %g is outside %s1e-6..1e6", who, t, zero_ok ? "0 or " : "");
    return CBGPU_OK;
}

template <typename T>
Rows<T> rows_of(const cbgpu_logits* x) {
    return Rows<T>{(const T*)x->data, x->n, x->row_stride, x->class_stride, x->n_classes};
}

struct Tile {
    int rows, pitch;
    size_t smem;
};
// Rows a narrow block stages: about 32 KB, at least one for each lane team.
Tile narrow_tile(int V, size_t bytes_a_class, int teams, bool by_rows) {
    Tile t;
    t.pitch = by_rows ? V : (V | 1);  // an odd pitch for rows that are written class by class
    const size_t row = (size_t)t.pitch * bytes_a_class;
    size_t rows = 32768 / row;
    rows = rows < (size_t)teams ? (size_t)teams : rows / teams * teams;
    t.rows = (int)rows;
    t.smem = (rows * row + 15) / 16 * 16;
    return t;
}

template <typename K, typename... A>
int lg_launch(const char* who, K kernel, unsigned grid, size_t smem, cudaStream_t st, A... args) {
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return lfail(CBGPU_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    }
    kernel<<<grid, kLgThreads, smem, st>>>(args...);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return lfail(CBGPU_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
    return CBGPU_OK;
}

// Lanes a narrow row: 1 up to 12 classes, 8 up to 128, else a warp.
template <typename F1, typename F8, typename F32>
int by_lanes(int V, F1 f1, F8 f8, F32 f32) {
    return V <= 12 ? f1() : (V <= 128 ? f8() : f32());
}

unsigned tiles_of(int64_t n, int rows) { return (unsigned)((n + rows - 1) / rows); }

template <typename T>
int run_top(const cbgpu_logits* x, int k, double temp, void* value, int32_t* index, void* tail, cudaStream_t st) {
    typedef typename Num<T>::C C;
    const char* who = "top_logits";
    const Rows<T> rows = rows_of<T>(x);
    const Scale<C> sc(temp);
    if (rows.V > kLgNarrow)
        return lg_launch(who, lg_top_wide_kernel<T>, (unsigned)rows.n, 0, st, rows, k, sc, (T*)value, index, (C*)tail);
    auto narrow = [&](auto kernel, int lanes) {
        const Tile t = narrow_tile(rows.V, sizeof(T), kLgThreads / lanes, rows.class_stride <= rows.row_stride);
        return lg_launch(who, kernel, tiles_of(rows.n, t.rows), t.smem, st, rows, k, sc, t.rows, t.pitch, (T*)value,
                         index, (C*)tail);
    };
    return by_lanes(rows.V, [&] { return narrow(lg_top_narrow_kernel<T, 1>, 1); },
                    [&] { return narrow(lg_top_narrow_kernel<T, 8>, 8); },
                    [&] { return narrow(lg_top_narrow_kernel<T, 32>, 32); });
}

template <typename T>
int run_distill(const cbgpu_logits* x, const cbgpu_teacher* tc, const void* weight, double temp, void* loss, void* der1,
                int64_t drs, int64_t dcs, cudaStream_t st) {
    typedef typename Num<T>::C C;
    const char* who = "distill";
    const Rows<T> rows = rows_of<T>(x);
    const Scale<C> sc(temp);
    const TeacherArgs ta{tc->index, tc->value, tc->index_bytes, tc->value_dtype, tc->k};
    if (rows.V > kLgNarrow)
        return lg_launch(who, lg_distill_wide_kernel<T>, (unsigned)rows.n, sizeof(uint32_t) * ((rows.V + 31) / 32), st,
                         rows, ta, (const C*)tc->tail, (const C*)weight, temp, sc, (C*)loss, (T*)der1, drs, dcs);
    auto narrow = [&](auto kernel, int lanes) {
        const Tile t =
            narrow_tile(rows.V, sizeof(T) + sizeof(C), kLgThreads / lanes, rows.class_stride <= rows.row_stride);
        return lg_launch(who, kernel, tiles_of(rows.n, t.rows), t.smem, st, rows, ta, (const C*)tc->tail,
                         (const C*)weight, temp, sc, t.rows, t.pitch, (C*)loss, (T*)der1, drs, dcs);
    };
    return by_lanes(rows.V, [&] { return narrow(lg_distill_narrow_kernel<T, 1>, 1); },
                    [&] { return narrow(lg_distill_narrow_kernel<T, 8>, 8); },
                    [&] { return narrow(lg_distill_narrow_kernel<T, 32>, 32); });
}

template <typename T>
int run_sample(const cbgpu_logits* x, const cbgpu_sampling* s, int32_t* index, cudaStream_t st) {
    const char* who = "sample_classes";
    const Rows<T> rows = rows_of<T>(x);
    const SampleArgs a{s->uniform,          s->uniform_dtype, s->top_k,      s->temperature, s->top_p, s->min_p,
                       s->temperature_rows, s->top_p_rows,    s->min_p_rows, s->top_k_rows};
    int bits = 0;
    while ((1 << bits) < rows.V) ++bits;
    const int shift = bits < 10 ? 52 : 62 - bits;  // at most what a 64-bit exponential holds
    if (rows.V > kLgNarrow)
        return lg_launch(who, lg_sample_wide_kernel<T>, (unsigned)rows.n, 0, st, rows, a, shift, index);
    auto narrow = [&](auto kernel, int lanes) {
        const Tile t = narrow_tile(rows.V, sizeof(T), kLgThreads / lanes, rows.class_stride <= rows.row_stride);
        return lg_launch(who, kernel, tiles_of(rows.n, t.rows), t.smem, st, rows, a, shift, t.rows, t.pitch, index);
    };
    return by_lanes(rows.V, [&] { return narrow(lg_sample_narrow_kernel<T, 1>, 1); },
                    [&] { return narrow(lg_sample_narrow_kernel<T, 8>, 8); },
                    [&] { return narrow(lg_sample_narrow_kernel<T, 32>, 32); });
}

// [lo, hi) of the bytes behind a strided [n, V] array
struct Span {
    uintptr_t lo, hi;
    bool meets(const Span& o) const { return lo < o.hi && o.lo < hi; }
};
Span span_of(const void* p, size_t bytes) { return Span{(uintptr_t)p, p ? (uintptr_t)p + bytes : (uintptr_t)p}; }
Span span_of(const void* p, size_t es, int64_t n, int V, int64_t rs, int64_t cs) {
    return span_of(p, ((size_t)(n - 1) * (size_t)rs + (size_t)(V - 1) * (size_t)cs + 1) * es);
}

#define LG_BY_DTYPE(d, fn, ...)                              \
    ((d) == CBGPU_F64   ? fn<double>(__VA_ARGS__)            \
     : (d) == CBGPU_F32 ? fn<float>(__VA_ARGS__)             \
     : (d) == CBGPU_F16 ? fn<__half>(__VA_ARGS__)            \
                        : fn<__nv_bfloat16>(__VA_ARGS__))

}  // namespace

int cbgpu_top_logits(const cbgpu_logits* x, int32_t k, double temperature, void* value, int32_t* index, void* tail,
                     void* stream) {
    int rc = check_logits("top_logits", x);
    if (rc) return rc;
    if (k < 1 || k > kLgMaxTop || k > x->n_classes)
        return lfail(CBGPU_ERR_INVALID, "top_logits: k = %d is outside 1..min(%d, n_classes = %d)", k, kLgMaxTop,
                     x->n_classes);
    if ((rc = check_temperature("top_logits", temperature, false))) return rc;
    if (x->n > 0 && (!value || !index)) return lfail(CBGPU_ERR_INVALID, "top_logits: value or index is NULL");
    if (x->n == 0) return CBGPU_OK;
    return LG_BY_DTYPE(x->dtype, run_top, x, k, temperature, value, index, tail, (cudaStream_t)stream);
}

int cbgpu_distill(const cbgpu_logits* x, const cbgpu_teacher* t, const void* weight, double temperature, void* loss,
                  void* der1, int64_t der1_row_stride, int64_t der1_class_stride, void* stream) {
    int rc = check_logits("distill", x);
    if (rc) return rc;
    if (!t) return lfail(CBGPU_ERR_INVALID, "distill: teacher is NULL");
    if (t->k < 1 || t->k > kLgMaxTop)
        return lfail(CBGPU_ERR_INVALID, "distill: k = %d is outside 1..%d", t->k, kLgMaxTop);
    if (t->index_bytes != 4 && t->index_bytes != 8)
        return lfail(CBGPU_ERR_INVALID, "distill: index_bytes must be 4 or 8");
    if (t->value_dtype < CBGPU_F64 || t->value_dtype > CBGPU_BF16)
        return lfail(CBGPU_ERR_INVALID, "distill: value_dtype %d is not one of the cbgpu_dtype values", t->value_dtype);
    if ((rc = check_temperature("distill", temperature, false))) return rc;
    if (x->n == 0) return CBGPU_OK;
    if (!t->index || !t->value || !loss) return lfail(CBGPU_ERR_INVALID, "distill: index, value or loss is NULL");
    if (der1) {
        const int64_t n = x->n, V = x->n_classes, rs = der1_row_stride, cs = der1_class_stride;
        if (rs < 0 || cs < 0) return lfail(CBGPU_ERR_INVALID, "distill: negative strides");
        const bool apart = (n == 1 && V == 1) || (n == 1 && cs >= 1) || (V == 1 && rs >= 1) ||
                           (cs >= 1 && rs > cs * (V - 1)) || (rs >= 1 && cs > rs * (n - 1));
        if (!apart) return lfail(CBGPU_ERR_INVALID, "distill: elements of der1 share memory");
        const size_t es = dtype_size(x->dtype), wide = x->dtype == CBGPU_F64 ? 8 : 4;
        if ((uintptr_t)der1 % es != 0) return lfail(CBGPU_ERR_INVALID, "distill: der1 is not aligned to its type");
        const Span d = span_of(der1, es, n, (int)V, rs, cs);
        const bool same = der1 == x->data && (n == 1 || rs == x->row_stride) && (V == 1 || cs == x->class_stride);
        if (!same && d.meets(span_of(x->data, es, n, (int)V, x->row_stride, x->class_stride)))
            return lfail(CBGPU_ERR_INVALID, "distill: der1 overlaps the logits without being them");
        if (d.meets(span_of(t->index, (size_t)n * t->k * t->index_bytes)) ||
            d.meets(span_of(t->value, (size_t)n * t->k * dtype_size(t->value_dtype))) ||
            d.meets(span_of(t->tail, (size_t)n * wide)) || d.meets(span_of(weight, (size_t)n * wide)) ||
            d.meets(span_of(loss, (size_t)n * wide)))
            return lfail(CBGPU_ERR_INVALID, "distill: der1 overlaps the teacher, the weights or the loss");
    }
    return LG_BY_DTYPE(x->dtype, run_distill, x, t, weight, temperature, loss, der1, der1_row_stride,
                       der1_class_stride, (cudaStream_t)stream);
}

int cbgpu_sample_classes(const cbgpu_logits* x, const cbgpu_sampling* s, int32_t* index, void* stream) {
    int rc = check_logits("sample_classes", x);
    if (rc) return rc;
    if (!s) return lfail(CBGPU_ERR_INVALID, "sample_classes: sampling is NULL");
    if (s->uniform_dtype != CBGPU_F32 && s->uniform_dtype != CBGPU_F64)
        return lfail(CBGPU_ERR_INVALID, "sample_classes: uniform must be f32 or f64");
    if (!s->temperature_rows && (rc = check_temperature("sample_classes", s->temperature, true))) return rc;
    if (!s->top_k_rows && s->top_k < 0) return lfail(CBGPU_ERR_INVALID, "sample_classes: top_k %d < 0", s->top_k);
    if (!s->top_p_rows && !(s->top_p >= 0.0 && s->top_p <= 1.0))
        return lfail(CBGPU_ERR_INVALID, "sample_classes: top_p %g is outside 0..1", s->top_p);
    if (!s->min_p_rows && !(s->min_p >= 0.0 && s->min_p <= 1.0))
        return lfail(CBGPU_ERR_INVALID, "sample_classes: min_p %g is outside 0..1", s->min_p);
    if (x->n == 0) return CBGPU_OK;
    if (!s->uniform || !index) return lfail(CBGPU_ERR_INVALID, "sample_classes: uniform or index is NULL");
    return LG_BY_DTYPE(x->dtype, run_sample, x, s, index, (cudaStream_t)stream);
}
