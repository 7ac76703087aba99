// logits.cuh -- what the operators on class logits share (logits_top.cu, logits_distill.cu,
// logits_sample.cu): number types, teams of threads on one row, rows staged in
// shared memory, argument checks.
//
// Rows come from a booster (f64 approximants, few classes, stored class by
// class) or from a neural teacher or student (16 or 32 bits, up to kLgMaxClasses
// classes, stored row by row).  The operators read each row once or twice and
// are bound by that traffic, so one launch does all of an operator.
//
// Two shapes of kernel:
//   narrow  a block stages a tile of rows in shared memory, then 1, 8 or 32 lanes work on each row:
//           up to kLgNarrow classes, where there are few rows kLgFew (is_wide; the sampler has its own rule);
//   wide    a cluster of blocks holds one row in its shared memory.
// Order of classes: larger logit first, equal logits by lower index, NaN last.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cooperative_groups.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>

#include "../../include/cbgpu.h"
#include "cbgpu_common.cuh"

namespace cbgpu {
int record_error(int code, const char* msg);  // session.cu: sets cbgpu_last_error()
}

namespace {

constexpr int kLgMaxClasses = 262144;
constexpr int kLgMaxTop = 256;
constexpr int kLgNarrow = 512;
constexpr int kLgFew = 128;
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
    static constexpr int kKeyDrop = 0;  // low bits of a key that say nothing
};
template <>
struct Num<__half> {
    typedef float C;
    typedef uint32_t Key;
    static constexpr int kKeyDrop = 13;
};
template <>
struct Num<__nv_bfloat16> {
    typedef float C;
    typedef uint32_t Key;
    static constexpr int kKeyDrop = 16;
};
template <>
struct Num<double> {
    typedef double C;
    typedef u64 Key;
    static constexpr int kKeyDrop = 0;
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

// The logit of a key (0 for -0, some NaN for 0).
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k); }
__device__ __forceinline__ double of_key(u64 k) {
    return __longlong_as_double((long long)((k >> 63) ? k & 0x7fffffffffffffffull : ~k));
}

__device__ __forceinline__ float lg_inf(float) { return __int_as_float(0x7f800000); }
__device__ __forceinline__ double lg_inf(double) { return __longlong_as_double(0x7ff0000000000000ll); }
__device__ __forceinline__ float lowest(float) { return __int_as_float((int)0xff7fffffu); }  // of the finite numbers
__device__ __forceinline__ double lowest(double) { return __longlong_as_double((long long)0xffefffffffffffffull); }

// exp((a - m) / T).  f32: 2^((a - m) c) with c = log2(e) / T rounded to f32: a relative change of the
// temperature by at most 2^-24, taken for differences of logits, of teacher and student alike.  A maximum, which
// may be large beside T, meets a tail, which comes divided by T, in 64 bits and by T itself.
__device__ __forceinline__ float lg_exp(float d, float c) { return exp2f(d * c); }
__device__ __forceinline__ double lg_exp(double d, double c) { return exp(d * c); }
template <typename C>
struct Scale;
template <>
struct Scale<float> {
    float c;
    double inv_t;  // the 1 / T that c stands for
    double t, by_t;  // T and 1 / T
    __host__ explicit Scale(double t)
        : c((float)(1.4426950408889634 / t)), inv_t((double)c * 0.6931471805599453), t(t), by_t(1.0 / t) {}
};
template <>
struct Scale<double> {
    double c, inv_t, t, by_t;
    __host__ explicit Scale(double t) : c(1.0 / t), inv_t(c), t(t), by_t(c) {}
};

// A maximum that is subtracted: 0 where there is no class, so that the exponentials are 0 there.
template <typename C>
__device__ __forceinline__ C floor_max(C m) { return m == -lg_inf(C()) ? C(0) : m; }

struct OpMax {
    template <typename V>
    __device__ V operator()(V a, V b) const { return a > b ? a : b; }
    __device__ float operator()(float a, float b) const { return fmaxf(a, b); }  // drops a NaN
    __device__ double operator()(double a, double b) const { return fmax(a, b); }
};
// exp of a non-positive number by the table-driven method of P. T. P. Tang (ACM TOMS 15, 1989): with
// x log2(e) = (n + r) / 64, |r| <= 1/2, it is 2^(n / 64), from a table of 64 and an exponent, times a polynomial
// in r ln2 / 64 (below 0.0055), of which degree 5 leaves 4e-17 (degree 4 leaves 4e-14, some 180 units of a draw's
// last bit, for 1 to 2 % of the time of draws that are bound by it).  11 operations in 64
// bits, where exp() with its range checks takes two to three times as many instructions, and f64 rows and the
// sampler's masses are bound by them (draws 64 x 131071 f32: 55 us against 35).
struct ExpTable {
    static constexpr int kSize = 64;
    static constexpr double kPerUnit = kSize * 1.4426950408889634;  // y of exp<>() for x = 1
    double of[kSize];
    __device__ void fill() {  // by the block; a barrier follows
        if (threadIdx.x < kSize) of[threadIdx.x] = exp2((double)threadIdx.x / kSize);
    }
    // 2^(y / 64) for y <= 0.  Below 2^-1020, -inf included, it is 0, and a NaN stays one, with kExact;
    // else it is 2^-1020, for those who round it to 0 anyway.
    template <bool kExact>
    __device__ double exp(double y) const {
        const uint32_t hi = (uint32_t)__double2hiint(y);  // of negative numbers the larger is further down
        const bool none = kExact && hi > 0xc0efdfffu && hi <= 0xfff00000u;  // y <= -65280, -inf; not a NaN
        const double x = kExact ? (none ? -65280.0 : y)
                                : __hiloint2double((int)(hi < 0xc0efe000u ? hi : 0xc0efe000u), __double2loint(y));
        const double t = x + 6755399441055744.0;  // 1.5 2^52: the low word of t is n
        const int n = __double2loint(t);
        const double r = x - (t - 6755399441055744.0);
        constexpr double c = 0.6931471805599453 / kSize;
        double p = fma(r, c * c * c * c * c / 120.0, c * c * c * c / 24.0);
        p = fma(r, p, c * c * c / 6.0);
        p = fma(r, p, c * c / 2.0);
        p = fma(r, p, c);
        const double b = of[n & (kSize - 1)];
        const double e = fma(b * r, p, b);
        return kExact && none ? 0.0 : __hiloint2double(__double2hiint(e) + ((n >> 6) << 20), __double2loint(e));
    }
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
    __device__ V steps(V v, Op op) const {
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(mask, v, o));
        return v;
    }
    template <typename V, typename Op>
    __device__ V reduce(V v, Op op) const {
        return steps(v, op);
    }
    // a warp has these in one instruction
    __device__ uint32_t reduce(uint32_t v, OpMax) const { return G == 32 ? __reduce_max_sync(0xffffffffu, v) : steps(v, OpMax()); }
    __device__ uint32_t reduce(uint32_t v, OpMin) const { return G == 32 ? __reduce_min_sync(0xffffffffu, v) : steps(v, OpMin()); }
    __device__ int reduce(int v, OpMin) const { return G == 32 ? __reduce_min_sync(0xffffffffu, v) : steps(v, OpMin()); }
    __device__ int reduce(int v, OpOr) const { return G == 32 ? (int)__reduce_or_sync(0xffffffffu, (unsigned)v) : steps(v, OpOr()); }
    __device__ float reduce(float v, OpMax) const {  // a NaN is dropped
        if (G < 32) return steps(v, OpMax());
        float r;
        asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
        return r;
    }
    __device__ float reduce(float v, OpMin) const { return -reduce(-v, OpMax()); }
    // a sum of masses, below 2^62
    __device__ u64 sum(u64 v) const {
        if (G < 32) return reduce(v, OpSum());
        const uint32_t part = (1u << 26) - 1u;  // 32 of them fit 31 bits
        const u64 lo = __reduce_add_sync(0xffffffffu, (uint32_t)v & part);
        const u64 mid = __reduce_add_sync(0xffffffffu, (uint32_t)(v >> 26) & part);
        const u64 hi = __reduce_add_sync(0xffffffffu, (uint32_t)(v >> 52));
        return lo + (mid << 26) + (hi << 52);
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

template <int G>
__device__ __forceinline__ int team_count(const LaneTeam<G>& t, int v) {
    return G == 32 ? (int)__reduce_add_sync(0xffffffffu, (unsigned)v) : t.reduce(v, OpSum());
}

// ---- launch arguments ----------------------------------------------------------

template <typename T>
struct Rows {
    const T* data;
    int64_t n, row_stride, class_stride;
    int V;
};

// A logit of the teacher's lists, whatever its type: its bits, and the number they stand for.  Apart,
// so that a load can be under way while others are asked for.
__device__ __forceinline__ u64 load_bits(const void* p, int dtype, int64_t i) {
    if (dtype == CBGPU_F64) return ((const u64*)p)[i];
    return dtype == CBGPU_F32 ? ((const uint32_t*)p)[i] : ((const unsigned short*)p)[i];
}
__device__ __forceinline__ double of_bits(u64 b, int dtype) {
    if (dtype == CBGPU_F64) return __longlong_as_double((long long)b);
    if (dtype == CBGPU_F32) return (double)__uint_as_float((uint32_t)b);
    if (dtype == CBGPU_F16) return (double)__half2float(__ushort_as_half((unsigned short)b));
    return (double)__uint_as_float((uint32_t)b << 16);
}
__device__ __forceinline__ double load_any(const void* p, int dtype, int64_t i) {
    return of_bits(load_bits(p, dtype, i), dtype);
}

struct TeacherArgs {
    const void *index, *value;
    int index_bytes, value_dtype, k;
    __device__ u64 idx_bits(int64_t at) const {
        return index_bytes == 8 ? ((const u64*)index)[at] : (u64)((const uint32_t*)index)[at];
    }
    __device__ int64_t of_idx_bits(u64 b) const { return index_bytes == 8 ? (int64_t)b : (int64_t)(int32_t)(uint32_t)b; }
    __device__ int64_t idx(int64_t at) const { return of_idx_bits(idx_bits(at)); }
    __device__ void prefetch(int64_t at) const {  // hints: the lines of entry `at`
        asm volatile("prefetch.global.L2 [%0];" ::"l"((const char*)index + at * index_bytes));
        const int vb = value_dtype == CBGPU_F64 ? 8 : (value_dtype == CBGPU_F32 ? 4 : 2);
        asm volatile("prefetch.global.L2 [%0];" ::"l"((const char*)value + at * vb));
    }
};

struct SampleArgs {
    const void* uniform;
    int uniform_dtype, top_k;
    double temperature, top_p, min_p;
    const float *temperature_rows, *top_p_rows, *min_p_rows;
    const int32_t* top_k_rows;
};

// ---- narrow rows ------------------------------------------------------------------------------
//
// A block stages a tile of rows in shared memory, `pitch` elements apart, and
// gives each row to a team of G lanes; lane `rank` holds the classes
// [rank * per, rank * per + per), per <= ITEMS, in registers.  G = 1 for up to 16 classes
// (a booster's), 8 up to 128, 32 up to kLgNarrow: a lane then has work for each
// instruction of a reduction over its team.  Rows that a thread has to itself and that lie class
// by class in memory are read straight from there.
template <typename T>
struct TileIo {
    int64_t rs, cs;
    int V, rows, pitch;
    bool flat;  // the tile is one run of memory: copied by 16 bytes
    int shift;  // elements of shared memory before the first row, so that both sides lie alike to 16 bytes
    __device__ TileIo(const T* g, int64_t rs_, int64_t cs_, int V_, int rows_)
        : rs(rs_), cs(cs_), V(V_), rows(rows_) {
        flat = (cs == 1 || V == 1) && rs == V;
        pitch = flat ? V : (V | 1);
        shift = flat ? (int)(((uintptr_t)g & 15) / sizeof(T)) : 0;
    }
    template <bool kStore>
    __device__ void copy(T* s, T* g) const {
        const uint32_t total = (uint32_t)rows * (uint32_t)V;
        if (flat && (((uintptr_t)g ^ (uintptr_t)s) & 15) == 0) {
            constexpr uint32_t VE = 16 / sizeof(T);
            uint32_t head = (uint32_t)((16 - ((uintptr_t)g & 15)) & 15) / (uint32_t)sizeof(T);
            head = head < total ? head : total;
            const uint32_t vectors = (total - head) / VE, tail = head + vectors * VE;
            uint4* gv = reinterpret_cast<uint4*>(g + head);
            uint4* sv = reinterpret_cast<uint4*>(s + head);
#pragma unroll 4
            for (uint32_t v = threadIdx.x; v < vectors; v += kLgThreads) {
                if (kStore) __stcs(gv + v, sv[v]);
                else sv[v] = __ldcs(gv + v);
            }
            const uint32_t e = threadIdx.x < head ? threadIdx.x : tail + threadIdx.x - head;
            if (threadIdx.x < head || e < total) {
                if (kStore) g[e] = s[e];
                else s[e] = g[e];
            }
            return;
        }
        // along the axis that is closer in memory
        const uint32_t inner = cs <= rs ? (uint32_t)V : (uint32_t)rows;
        for (uint32_t e = threadIdx.x; e < total; e += kLgThreads) {
            const uint32_t o = e / inner, i = e - o * inner;
            const uint32_t r = cs <= rs ? o : i, c = cs <= rs ? i : o;
            T* at = g + (int64_t)r * rs + (int64_t)c * cs;
            if (kStore) *at = s[r * pitch + c];
            else s[r * pitch + c] = *at;
        }
    }
};

// A lane's classes.  Loops over them are unrolled to ITEMS and stop, by fours, at `per`, which all
// lanes share.
template <int G, int ITEMS>
struct Items {
    int first, count, per;
    template <typename Team>
    __device__ Items(const Team& t, int V) {
        per = (V + G - 1) / G;
        first = t.rank * per;
        count = V - first < per ? V - first : per;
    }
    __device__ bool has(int it) const { return it < count; }
};
#define LG_EACH(it)                                                      \
    _Pragma("unroll") for (int four_ = 0; four_ < ITEMS; four_ += 4)     \
        if (four_ < mine.per) _Pragma("unroll") for (int it = four_; it < four_ + 4; ++it)

template <typename Key>
struct Ranked {  // a class in the operators' order
    Key key;
    uint32_t idx;
    __device__ bool before(const Ranked& o) const {
        if (sizeof(Key) == 4) return ((u64)key << 32 | (uint32_t)~idx) > ((u64)o.key << 32 | (uint32_t)~o.idx);
        return key > o.key || (key == o.key && idx < o.idx);
    }
};
// ---- wide rows: a cluster of blocks holds a row in its shared memory --------------------------
//
// The row is cut into 16-byte vectors from the 16-byte boundary at or below
// its first class, `per` vectors a block, so that rows of any alignment are
// copied by 16 bytes; classes of the two vectors at the row's ends and rows
// whose classes are not neighbours in memory are loaded one by one, and
// what lies outside the row is held as -inf.

template <typename T>
struct WideRow {
    static constexpr int VE = 16 / (int)sizeof(T);
    const T* row;
    int64_t cs;
    int V, head, v0, nv;  // head: elements of the first vector before the row; this block's vectors [v0, v0 + nv)
    __device__ WideRow(const Rows<T>& x, int64_t r, int rank, int per)
        : row(x.data + r * x.row_stride), cs(x.class_stride), V(x.V) {
        head = cs == 1 ? (int)(((uintptr_t)row & 15) / sizeof(T)) : 0;
        v0 = rank * per;
        const int all = (head + V + VE - 1) / VE;
        nv = all - v0 < per ? all - v0 : per;
    }
    __device__ int first(int v) const { return (v0 + v) * VE - head; }  // class of vector v's first element
    __device__ bool valid(int i) const { return i >= 0 && i < V; }
    __device__ int slot(int i) const {  // where class i lies in this block's memory, or -1
        const int at = i + head - v0 * VE;
        return at >= 0 && at < nv * VE ? at : -1;
    }
    __device__ uint4 edge(int i) const {  // a vector from class i that is loaded class by class
        T e[VE];
        for (int j = 0; j < VE; ++j)
            e[j] = i + j >= 0 && i + j < V ? row[(int64_t)(i + j) * cs] : from_c<T>(-lg_inf(typename Num<T>::C()));
        uint4 q;
        memcpy(&q, e, sizeof q);
        return q;
    }
    // This block's vectors that lie inside the row whole: [lo, hi); the others are the row's ends.
    __device__ int whole_lo() const { return cs == 1 ? (v0 == 0 && head != 0 ? 1 : 0) : nv; }
    __device__ int whole_hi() const {
        const int inside = (head + V) / VE - v0;
        return cs == 1 ? (inside < nv ? inside : nv) : nv;
    }
    // Copies this block's part to s; see(vector) is called for each vector on
    // the way.  kAhead loads a thread are under way at a time.
    template <int NT = kLgThreads, int kAhead = 8, typename See>
    __device__ void load(uint4* s, See see) const {
        const int lo = whole_lo(), hi = whole_hi();
        const uint4* g = reinterpret_cast<const uint4*>(row + ((int64_t)v0 * VE - head));
        int v = lo + threadIdx.x;
        for (; v + (kAhead - 1) * NT < hi; v += kAhead * NT) {
            uint4 q[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) q[u] = __ldcs(g + v + u * NT);
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                see(q[u]);
                s[v + u * NT] = q[u];
            }
        }
        {
            uint4 q[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (v + u * NT < hi) q[u] = __ldcs(g + v + u * NT);
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (v + u * NT < hi) {
                    see(q[u]);
                    s[v + u * NT] = q[u];
                }
        }
        ends<NT>([&](int e) {
            const uint4 q = edge(first(e));
            see(q);
            s[e] = q;
        });
    }
    // Asks for this block's whole vectors in L2 (a hint; one thread).
    __device__ void prefetch() const {
        const int lo = whole_lo(), hi = whole_hi();
        if (hi <= lo) return;
        const T* g = row + ((int64_t)(v0 + lo) * VE - head);
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(g), "r"((hi - lo) * 16) : "memory");
    }
    // fn(v) for the vectors outside [whole_lo, whole_hi)
    template <int NT = kLgThreads, typename Fn>
    __device__ void ends(Fn fn) const {
        const int lo = whole_lo(), hi = whole_hi();
        if (cs != 1) {
            for (int v = threadIdx.x; v < nv; v += NT) fn(v);
            return;
        }
        if (threadIdx.x == 0 && lo == 1 && nv > 0) fn(0);
        if (threadIdx.x == 32 && hi < nv && hi >= lo) fn(nv - 1);
    }
};

__device__ __forceinline__ void unpack(const uint4& v, float (&o)[4], float) {
    o[0] = __uint_as_float(v.x), o[1] = __uint_as_float(v.y), o[2] = __uint_as_float(v.z), o[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void unpack(const uint4& v, double (&o)[2], double) {
    o[0] = __hiloint2double((int)v.y, (int)v.x), o[1] = __hiloint2double((int)v.w, (int)v.z);
}
__device__ __forceinline__ void unpack(const uint4& v, float (&o)[8], __nv_bfloat16) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) o[2 * j] = __uint_as_float(w[j] << 16), o[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
}
__device__ __forceinline__ void unpack(const uint4& v, float (&o)[8], __half) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        o[2 * j] = f.x, o[2 * j + 1] = f.y;
    }
}
__device__ __forceinline__ uint4 pack(const float (&o)[4], float) {
    return make_uint4(__float_as_uint(o[0]), __float_as_uint(o[1]), __float_as_uint(o[2]), __float_as_uint(o[3]));
}
__device__ __forceinline__ uint4 pack(const double (&o)[2], double) {
    return make_uint4((uint32_t)__double2loint(o[0]), (uint32_t)__double2hiint(o[0]), (uint32_t)__double2loint(o[1]),
                      (uint32_t)__double2hiint(o[1]));
}
__device__ __forceinline__ uint4 pack(const float (&o)[8], __nv_bfloat16) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(o[2 * j], o[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 pack(const float (&o)[8], __half) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const __half2 h = __floats2half2_rn(o[2 * j], o[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// The running maximum of vectors (a NaN is dropped), pairs of 16-bit logits at a time.
template <typename T>
struct VecMax {
    typename Num<T>::C m = -lg_inf(typename Num<T>::C());
    __device__ void operator()(const uint4& q) {
        typename Num<T>::C a[16 / sizeof(T)];
        unpack(q, a, T());
#pragma unroll
        for (int j = 0; j < 16 / (int)sizeof(T); ++j) m = OpMax()(m, a[j]);
    }
    __device__ typename Num<T>::C get() const { return m; }
};
template <typename H2>
struct PairMax {
    H2 m;
    __device__ void operator()(const uint4& q) {
        const H2* h = reinterpret_cast<const H2*>(&q);
        m = __hmax2(m, __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    }
};
template <>
struct VecMax<__half> : PairMax<__half2> {
    __device__ VecMax() { m = __float2half2_rn(-lg_inf(0.0f)); }
    __device__ float get() const { return fmaxf(__low2float(m), __high2float(m)); }
};
template <>
struct VecMax<__nv_bfloat16> : PairMax<__nv_bfloat162> {
    __device__ VecMax() { m = __float2bfloat162_rn(-lg_inf(0.0f)); }
    __device__ float get() const { return fmaxf(__low2float(m), __high2float(m)); }
};

// The same, but a NaN stays.
template <typename T>
struct VecMaxNan {
    typename Num<T>::C m = -lg_inf(typename Num<T>::C());
    __device__ static float both(float a, float b) {
        float r;
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
        return r;
    }
    __device__ static double both(double a, double b) { return a != a ? a : (b != b ? b : fmax(a, b)); }
    __device__ void operator()(const uint4& q) {
        typename Num<T>::C a[16 / sizeof(T)];
        unpack(q, a, T());
#pragma unroll
        for (int j = 0; j < 16 / (int)sizeof(T); ++j) m = both(m, a[j]);
    }
    __device__ typename Num<T>::C get() const { return m; }
};
template <typename H2>
struct PairMaxNan {
    H2 m;
    __device__ void operator()(const uint4& q) {
        const H2* h = reinterpret_cast<const H2*>(&q);
        m = __hmax2_nan(m, __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3])));
    }
    __device__ float get() const { return VecMaxNan<float>::both(__low2float(m), __high2float(m)); }
};
template <>
struct VecMaxNan<__half> : PairMaxNan<__half2> {
    __device__ VecMaxNan() { m = __float2half2_rn(-lg_inf(0.0f)); }
};
template <>
struct VecMaxNan<__nv_bfloat16> : PairMaxNan<__nv_bfloat162> {
    __device__ VecMaxNan() { m = __float2bfloat162_rn(-lg_inf(0.0f)); }
};

// Two f32 operations in one instruction.
__device__ __forceinline__ u64 f2(float a, float b) {
    u64 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void f2_split(u64 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ u64 f2_fma(u64 a, u64 b, u64 c) {
    u64 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ u64 f2_add(u64 a, u64 b) {
    u64 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ u64 f2_mul(u64 a, u64 b) {
    u64 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float ex2(float x) {  // within 2 ulp; a result below 2^-126 is 0
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x));
    return e;
}

// exp((a - m) / T) as 2^((a - m) c): the difference first, so that an exponential is at most 1 however far from 0
// the logits lie beside T (2^(a c - round(m c)) is one operation less, but its factor 2^(m c - round(m c)) is
// infinite from |m / T| of some 1e9 on: masks of -1e10, temperatures of 1e-6).
template <typename C>
struct Base;
template <>
struct Base<float> {
    float c, m;
    __device__ Base(float m_, const Scale<float>& sc) : c(sc.c), m(m_) {}
    __device__ float exp(float a) const { return ex2((a - m) * c); }
    // a vector: each class to its exponential
    template <int N>
    __device__ void exps(float (&a)[N]) const {
        const u64 c2 = f2(c, c), m2 = f2(-m, -m);
#pragma unroll
        for (int j = 0; j < N; j += 2) {
            f2_split(f2_mul(f2_add(f2(a[j], a[j + 1]), m2), c2), a[j], a[j + 1]);
            a[j] = ex2(a[j]), a[j + 1] = ex2(a[j + 1]);
        }
    }
    template <int N>
    __device__ static double total(const float (&e)[N]) {
        u64 s = f2(e[0], e[1]);
#pragma unroll
        for (int j = 2; j < N; j += 2) s = f2_add(s, f2(e[j], e[j + 1]));
        float lo, hi;
        f2_split(s, lo, hi);
        return (double)(lo + hi);
    }
    template <int N>
    __device__ static void times(float (&e)[N], float k) {
        const u64 k2 = f2(k, k);
#pragma unroll
        for (int j = 0; j < N; j += 2) f2_split(f2_mul(f2(e[j], e[j + 1]), k2), e[j], e[j + 1]);
    }
    __device__ double ln(float a) const { return ((double)a - (double)m) * (double)c * 0.6931471805599453; }
    __device__ float shift(const Base& to) const { return ex2((m - to.m) * c); }  // turns this base's sums into `to`'s
    __device__ double ln_shift(const Base& to) const { return to.ln(m); }  // the logarithm of that, in 64 bits
};
template <>
struct Base<double> {
    double c, m;
    __device__ Base(double m_, const Scale<double>& sc) : c(sc.c), m(m_) {}
    __device__ double exp(double a) const { return ::exp((a - m) * c); }
    template <int N>
    __device__ void exps(double (&a)[N]) const {
#pragma unroll
        for (int j = 0; j < N; ++j) a[j] = exp(a[j]);
    }
    template <int N>
    __device__ static double total(const double (&e)[N]) { return e[0] + e[1]; }
    template <int N>
    __device__ static void times(double (&e)[N], double k) { e[0] *= k, e[1] *= k; }
    __device__ double ln(double a) const { return (a - m) * c; }
    __device__ double shift(const Base& to) const { return ::exp(ln_shift(to)); }
    __device__ double ln_shift(const Base& to) const { return to.ln(m); }
};

constexpr int kLgWarps = kLgThreads / 32;

// The cluster's barrier in its two halves.  `kRelease` false: the thread has written nothing that
// another block reads.
template <bool kRelease>
__device__ __forceinline__ void cluster_arrive() {
    if (kRelease) asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    else asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// The largest of a warp's values (a NaN is dropped unless there is nothing else).
__device__ __forceinline__ float warp_max(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ double warp_max(double v) {
    for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
// Sum over the lanes below n (a power of two covers them), in all of them.
template <typename V>
__device__ __forceinline__ V warp_sum(V v, int n) {
    for (int o = 1; o < n; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// N values a thread -> their sums / maxima over the block, in every thread; two barriers.
template <int N, typename V, typename Op>
__device__ __forceinline__ void block_reduce(V (&v)[N], V (*scratch)[kLgWarps], Op op) {
#pragma unroll
    for (int i = 0; i < N; ++i)
        for (int o = 16; o > 0; o >>= 1) v[i] = op(v[i], __shfl_xor_sync(0xffffffffu, v[i], o));
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) scratch[i][threadIdx.x >> 5] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = scratch[i][0];
#pragma unroll
        for (int w = 1; w < kLgWarps; ++w) v[i] = op(v[i], scratch[i][w]);
    }
    __syncthreads();
}

// ---- the first k classes of a wide row ----------------------------------------------------------
//
// Every thread knows the largest of its own classes.  The k-th largest of a
// block's 256 such maxima is a lower bound of the row's k-th largest
// logit, and so is the least, over the cluster's blocks, of their ceil(k / blocks)-th
// largest; the classes at or above the larger of the two bounds are a few more than k, which the
// first block collects and sorts.  When ties or a lopsided row make that
// too many (or NaN too few), the exact bound (logit, index) is found bit by
// bit over the cluster instead, at some 50 passes over shared memory.  16-bit rows of 1025 to some 2050 classes have
// fewer vectors than threads: a k above their number (129 at least) leaves no bound, and the exact way is the only
// one (20000 x 1500 bf16, 188 vectors: 393 us at k 129, 1950 at k 200).

constexpr int kTopCap = 1024;  // classes the first block can collect

constexpr int kHits = 512;
constexpr int kSegments = 8192 / 32 + 1;  // a block holds up to 8193 vectors
constexpr int kGather = 3;
constexpr int kBins = 1024;    // of the sampler's histogram, which lies where the list comes to lie
struct SampleHist {
    uint32_t count[kBins];
};

template <typename Key>
struct TopShared {
    union __align__(16) {
        struct {
            Key key[kTopCap];
            uint32_t idx[kTopCap];
        };
        SampleHist hist;
        u64 segment[kSegments];  // the sampler's masses of 32 vectors each
    };
    uint32_t bound[16][2];  // of every block: its k-th and its ceil(k / blocks)-th largest thread maximum
    uint32_t flag[16];
    int base, vectors;
    uint16_t hit[kHits];    // places of the classes that the sampler collected from this block
    u64 part[2][16][kGather];  // values that go round the cluster
    u64 warp_part[kGather][kLgWarps];
    int count;
};

struct ClusterInfo {
    int rank, blocks;
    __device__ ClusterInfo() {
        auto c = cooperative_groups::this_cluster();
        rank = (int)c.block_rank(), blocks = (int)c.num_blocks();
    }
    template <typename V>
    __device__ V* of(V* mine, int b) const {
        return cooperative_groups::this_cluster().map_shared_rank(mine, b);
    }
    // All blocks' threads; what they wrote to each other's shared memory before is seen after.
    __device__ void sync() const {
        if (blocks > 1) {
            cluster_arrive<true>();
            cluster_wait();
        } else {
            __syncthreads();
        }
    }
};

// N values of each block's first warp (the same in its lanes), to sh.part[the turn before][block][0..N)
// of every block.  `turn` alternates between calls.
template <int N, typename Sh>
__device__ const u64 (*cluster_gather(const ClusterInfo& cl, Sh& sh, const u64 (&v)[N], int& turn))[kGather] {
    static_assert(N <= kGather, "words a block");
    if ((int)threadIdx.x < cl.blocks) {
        u64* to = cl.of(&sh.part[turn][cl.rank][0], (int)threadIdx.x);
#pragma unroll
        for (int i = 0; i < N; ++i) to[i] = v[i];
    }
    cl.sync();
    turn ^= 1;
    return sh.part[turn ^ 1];
}

// Sums over the cluster of N values a thread (each below 2^62 in all), in every thread.
template <int N, typename Sh>
__device__ void cluster_total(const ClusterInfo& cl, Sh& sh, u64 (&v)[N], int& turn) {
    const LaneTeam<32> warp;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = warp.sum(v[i]);
        if (warp.rank == 0) sh.warp_part[i][threadIdx.x >> 5] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = 0;
        for (int j = 0; j < kLgWarps; ++j) v[i] += sh.warp_part[i][j];
    }
    const u64(*of)[kGather] = cluster_gather<N>(cl, sh, v, turn);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = 0;
        for (int b = 0; b < cl.blocks; ++b) v[i] += of[b][i];
    }
}
template <typename Sh>
__device__ u64 cluster_total(const ClusterInfo& cl, Sh& sh, u64 v, int& turn) {
    u64 one[1] = {v};
    cluster_total<1>(cl, sh, one, turn);
    return one[0];
}

// fn(class, logit, place) for every place of this thread's vectors, also those outside the row (-inf; valid() tells)
template <typename T, typename Fn>
__device__ __forceinline__ void each_place(const WideRow<T>& w, const uint4* s, Fn fn) {
    constexpr int VE = WideRow<T>::VE;
    for (int v = threadIdx.x; v < w.nv; v += kLgThreads) {
        typename Num<T>::C a[VE];
        unpack(s[v], a, T());
        const int i = w.first(v);
#pragma unroll
        for (int j = 0; j < VE; ++j) fn(i + j, a[j], v * VE + j);
    }
}

// fn(class, logit) for this thread's classes
template <typename T, typename Fn>
__device__ __forceinline__ void each_class(const WideRow<T>& w, const uint4* s, Fn fn) {
    constexpr int VE = WideRow<T>::VE;
    for (int v = threadIdx.x; v < w.nv; v += kLgThreads) {
        typename Num<T>::C a[VE];
        unpack(s[v], a, T());
        const int i = w.first(v);
#pragma unroll
        for (int j = 0; j < VE; ++j)
            if (i + j >= 0 && i + j < w.V) fn(i + j, a[j], v * VE + j);
    }
}

// The last class of the shortest prefix (in order) whose metric over the cluster reaches `target`: bit by
// bit the largest key that still reaches it, then the lowest index among that key's classes.
template <typename T, typename Sh, typename Met>
__device__ Ranked<typename Num<T>::Key> cluster_select(const ClusterInfo& cl, Sh& sh, const WideRow<T>& w,
                                                       const uint4* s, u64 target, int& turn, Met metric) {
    typedef typename Num<T>::Key Key;
    typedef typename Num<T>::C C;
    Key key = 0;
    for (int b = (int)sizeof(Key) * 8 - 1; b >= 0; --b) {
        const Key cand = key | ((Key)1 << b);
        u64 f = 0;
        each_class(w, s, [&](int i, C a, int) {
            const Key k = key_of(a);
            if (k >= cand) f += metric(i, a, k);
        });
        if (cluster_total(cl, sh, f, turn) >= target) key = cand;
    }
    u64 above = 0;
    each_class(w, s, [&](int i, C a, int) {
        const Key k = key_of(a);
        if (k > key) above += metric(i, a, k);
    });
    const u64 need = target - cluster_total(cl, sh, above, turn);
    uint32_t idx = (1u << (32 - __clz(w.V))) - 1u;
    for (int b = 31 - __clz(w.V); b >= 0; --b) {
        const uint32_t cand = idx & ~(1u << b);
        u64 f = 0;
        each_class(w, s, [&](int i, C a, int) {
            const Key k = key_of(a);
            if (k == key && (uint32_t)i <= cand) f += metric(i, a, k);
        });
        if (cluster_total(cl, sh, f, turn) >= need) idx = cand;
    }
    return Ranked<Key>{key, idx};
}

// The first block's list in order; `n` entries, at most kTopCap.
template <typename Key>
__device__ void sort_list(TopShared<Key>& sh, int n) {
    static_assert(kTopCap >= 2 * kLgThreads, "room for the ranked entries behind the list");
    const int tid = threadIdx.x;
    if (n <= kLgThreads) {  // every entry counts those before it, some threads an entry
        int per = 1;
        while (n * per * 2 <= kLgThreads && per < 32) per *= 2;
        const int c = tid / per, part = tid & (per - 1);
        const Ranked<Key> own{sh.key[c < n ? c : 0], sh.idx[c < n ? c : 0]};
        int rank = 0;
        if (sizeof(Key) == 4) {  // key and index as one number, read by pairs
            u64* both = reinterpret_cast<u64*>(&sh.idx[kTopCap - 2 * kLgThreads]);
            if (tid < kLgThreads) both[tid] = tid < n ? (u64)sh.key[tid] << 32 | (uint32_t)~sh.idx[tid] : 0ull;
            __syncthreads();
            const u64 mine = (u64)own.key << 32 | (uint32_t)~own.idx;
#pragma unroll 4
            for (int i = 2 * part; i < n; i += 2 * per) {
                const ulonglong2 t = *reinterpret_cast<const ulonglong2*>(both + i);
                rank += (t.x > mine ? 1 : 0) + (t.y > mine ? 1 : 0);
            }
        } else {
#pragma unroll 4
            for (int i = part; i < n; i += per) rank += Ranked<Key>{sh.key[i], sh.idx[i]}.before(own) ? 1 : 0;
        }
        for (int o = 1; o < per; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
        __syncthreads();
        if (c < n && part == 0) sh.key[rank] = own.key, sh.idx[rank] = own.idx;
        __syncthreads();
        return;
    }
    int size = 1;
    while (size < n) size *= 2;
    for (int i = n + tid; i < size; i += kLgThreads) sh.key[i] = 0, sh.idx[i] = 0xffffffffu;
    __syncthreads();
    for (int len = 2; len <= size; len *= 2)
        for (int d = len / 2; d > 0; d /= 2) {
            for (int p = tid; p < size / 2; p += kLgThreads) {
                const int i = (p & (d - 1)) | ((p & ~(d - 1)) << 1), j = i | d;
                const Ranked<Key> a{sh.key[i], sh.idx[i]}, b{sh.key[j], sh.idx[j]};
                if ((i & len) == 0 ? b.before(a) : a.before(b))
                    sh.key[i] = b.key, sh.idx[i] = b.idx, sh.key[j] = a.key, sh.idx[j] = a.idx;
            }
            __syncthreads();
        }
}

// The largest bound that at least `target` of a block's kLgThreads values in shared memory reach, to
// 12 bits behind those that the values share; one warp.
__device__ __forceinline__ uint32_t warp_bound(const uint32_t* of, int target) {
    uint32_t v[kLgThreads / 32], most = 0, least = 0xffffffffu;
#pragma unroll
    for (int j = 0; j < kLgThreads / 32; ++j) {
        v[j] = of[((int)threadIdx.x & 31) + 32 * j];
        most = v[j] > most ? v[j] : most, least = v[j] < least ? v[j] : least;
    }
    most = __reduce_max_sync(0xffffffffu, most), least = __reduce_min_sync(0xffffffffu, least);
    const int bits = 32 - __clz((int)(most ^ least));
    uint32_t bound = bits < 32 ? most >> bits << bits : 0u;
    for (int b = bits - 1; b >= 0 && b >= bits - 12; --b) {
        const uint32_t cand = bound | (1u << b);
        int n = 0;
#pragma unroll
        for (int j = 0; j < kLgThreads / 32; ++j) n += v[j] >= cand;
        n = (int)__reduce_add_sync(0xffffffffu, (unsigned)n);
        if (n >= target) bound = cand;
        if (n == target) break;
    }
    return bound;
}

// Collects the row's first k classes, and perhaps some after them, in the
// first block's list (not sorted; returns how many, in every thread); they are
// replaced by -inf in the row, and `rest` gets the largest of this thread's classes
// that stay.  `mine`: the largest of this thread's classes.  Every block of the cluster runs.
// see(vector, least): this thread's vectors on the way, the collected classes as
// -inf and what stays below `least`; not for the exact bound (`exact`), which leaves that to the caller.
// `flag`: whether any thread of the cluster came with it set.
template <typename T, typename See>
__device__ int wide_top(const ClusterInfo& cl, TopShared<typename Num<T>::Key>& sh, const WideRow<T>& w, uint4* s,
                        typename Num<T>::C mine, int k, int& turn, typename Num<T>::C& rest, bool& exact, bool& flag,
                        See see) {
    typedef typename Num<T>::C C;
    typedef typename Num<T>::Key Key;
    constexpr int kDrop = (int)sizeof(Key) * 8 - 32;  // the bounds keep 32 bits of a key
    const int tid = threadIdx.x;
    const int share = (k + cl.blocks - 1) / cl.blocks;
    sh.idx[tid] = (uint32_t)(key_of(mine) >> kDrop);
    if (tid == 0) sh.count = 0;
    flag = __syncthreads_or(flag) != 0;
    if (tid < 64) {
        const uint32_t b = warp_bound(sh.idx, tid < 32 ? k : share);
        if ((tid & 31) < cl.blocks) {
            cl.of(&sh.bound[cl.rank][0], tid & 31)[tid >> 5] = b;
            if (tid < 32) *cl.of(&sh.flag[cl.rank], tid) = flag;
        }
    }
    cl.sync();
    uint32_t bk = 0, bs = 0xffffffffu;
    for (int b = 0; b < cl.blocks; ++b) {
        bk = bk > sh.bound[b][0] ? bk : sh.bound[b][0];
        bs = bs < sh.bound[b][1] ? bs : sh.bound[b][1];
        flag |= sh.flag[b] != 0;
    }
    const Key bound = (Key)(bk > bs ? bk : bs) << kDrop;
    const C least = bound <= key_of(-lg_inf(C())) ? -lg_inf(C()) : of_key(bound);
    T* se = reinterpret_cast<T*>(s);
    // a block collects in its own arrays; the first block's are the list
    auto take = [&](int i, C a, T* at) {
        const int p = atomicAdd(&sh.count, 1);
        if (p < kTopCap) sh.key[p] = key_of(a), sh.idx[p] = (uint32_t)i;
        *at = from_c<T>(-lg_inf(C()));
    };
    auto hand_over = [&] {
        __syncthreads();
        if (cl.rank != 0) {
            TopShared<Key>* first = cl.of(&sh, 0);
            const int n = sh.count < kTopCap ? sh.count : kTopCap;
            if (tid == 0 && n > 0) sh.base = atomicAdd(&first->count, sh.count);
            __syncthreads();
            for (int p = tid; p < n; p += kLgThreads)
                if (sh.base + p < kTopCap) first->key[sh.base + p] = sh.key[p], first->idx[sh.base + p] = sh.idx[p];
        }
        cl.sync();
    };
    constexpr int VE = WideRow<T>::VE;
    rest = -lg_inf(C());
    exact = false;
    // a thread's vectors that hold one are noted and gone through at the end, not one by one with the
    // warp waiting; each thread its own, so that its sums are in the same order always
    uint64_t hits = 0;
    int round = 0;
#pragma unroll 2
    for (int v = tid; v < w.nv; v += kLgThreads, ++round) {
        const uint4 q = s[v];
        VecMax<T> m;
        m(q);
        if (m.get() < least) {
            rest = OpMax()(rest, m.get());
            C a[VE];
            unpack(q, a, T());
            see(a, least);
        } else {
            hits |= 1ull << round;  // at most 33 rounds (8193 vectors)
        }
    }
    for (; hits; hits &= hits - 1) {
        const int v = tid + (__ffsll((long long)hits) - 1) * kLgThreads;
        C a[VE];
        unpack(s[v], a, T());
        const int i = w.first(v);
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            if (a[j] >= least && i + j >= 0 && i + j < w.V) {
                take(i + j, a[j], se + v * VE + j);
                a[j] = -lg_inf(C());
            } else {
                rest = OpMax()(rest, a[j]);
            }
        }
        see(a, least);
    }
    hand_over();
    const int n = cl.of(&sh, 0)->count;
    if (n >= k && n <= kTopCap) return n;
    // the exact bound, on the row as it was
    exact = true;
    cl.sync();
    if (tid == 0) sh.count = 0;
    w.load(s, [](const uint4&) {});
    __syncthreads();
    const Ranked<Key> last = cluster_select(cl, sh, w, s, (u64)k, turn, [](int, C, Key) { return 1ull; });
    rest = -lg_inf(C());
    __syncthreads();
    each_class(w, s, [&](int i, C a, int at) {
        if (last.before(Ranked<Key>{key_of(a), (uint32_t)i})) rest = OpMax()(rest, a);
        else take(i, a, se + at);
    });
    hand_over();
    return k;
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

// An array that a kernel reads or writes by elements of `size` bytes.
int check_aligned(const char* who, const char* name, const void* p, size_t size) {
    if ((uintptr_t)p % size != 0) return lfail(CBGPU_ERR_INVALID, "%s: %s is not aligned to its type", who, name);
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
    int rows;
    size_t smem;
};
// Rows a narrow block stages: about 24 KB (8 blocks an SM), but not so many that the SMs have less than
// four blocks each, and at least one for each lane team.
Tile narrow_tile(int64_t n, int V, size_t bytes_a_class, int teams) {
    const size_t row = (size_t)(V | 1) * bytes_a_class;
    size_t rows = 24576 / row;
    const size_t share = (size_t)((n + 148 * 4 - 1) / (148 * 4));
    rows = rows < share ? rows : share;
    rows = rows <= (size_t)teams ? (size_t)teams : (rows + teams - 1) / teams * teams;
    return Tile{(int)rows, rows * row + 32};
}

// What a kernel that needs asking is allowed: always the same, so that calls on several threads do not take
// it from each other.  The static arrays (up to 25 KB) fit beside it.
constexpr int kLgSmemMost = 200 * 1024;

template <typename K, typename... A>
int lg_launch_n(const char* who, K kernel, unsigned grid, int threads, size_t smem, cudaStream_t st, A... args) {
    cudaError_t e = cudaSuccess;
    if (smem > 20 * 1024)  // with the kernels' static arrays (up to 25 KB) above the 48 KB that need no asking
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kLgSmemMost);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    // (the launch's own error: the thread's last one may be another call's)
    if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e != cudaSuccess) return lfail(CBGPU_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
    return CBGPU_OK;
}
template <typename K, typename... A>
int lg_launch(const char* who, K kernel, unsigned grid, size_t smem, cudaStream_t st, A... args) {
    return lg_launch_n(who, kernel, grid, kLgThreads, smem, st, args...);
}

// Blocks of a wide row's cluster, vectors a block, shared memory.  About 64 KB a block (3 blocks an SM,
// so that one's copies run under another's arithmetic; 16 to 48 KB a block were slower, since each
// block pays for its barriers and sums: derivatives of 4096 x 64000 bf16 270 us at 64 KB, 320 at
// 43 KB); when there are few rows, up to 8 blocks of 6 KB or more, so that a row's bytes come
// through more SMs.  Clusters of 16 are for rows above 512 KB only: one of them is 10 us slower to
// start and to meet than one of 8.
struct Wide {
    int blocks, per;
    size_t smem;
    int64_t ahead;  // rows between one that is worked on and the one that takes its place
};
template <typename T>
Wide wide_shape(int64_t n, int V) {
    const int ve = 16 / (int)sizeof(T), vectors = (V + 2 * (ve - 1)) / ve;
    Wide w{1, 0, 0, 0};
    while (w.blocks < 16 && (size_t)V * sizeof(T) > (size_t)65536 * w.blocks) w.blocks *= 2;
    while (w.blocks < 8 && n * w.blocks <= 148 && (size_t)vectors * 16 >= (size_t)12288 * w.blocks)
        w.blocks *= 2;
    w.per = (vectors + w.blocks - 1) / w.blocks;
    w.smem = (size_t)w.per * 16;
    int resident = (int)((size_t)(220 * 1024) / (w.smem + 4096));
    resident = resident < 1 ? 1 : (resident > 8 ? 8 : resident);
    w.ahead = (148 * resident + w.blocks - 1) / w.blocks;
    return w;
}

// Launches `kernel` with clusters of w.blocks, w.blocks blocks a row, as many rows at a time as a grid holds.
template <typename K, typename... A>
int lg_launch_wide_n(const char* who, K kernel, int64_t n, const Wide& w, int threads, size_t smem, cudaStream_t st,
                     A... args) {
    cudaError_t e = cudaSuccess;
    if (smem > 32 * 1024)  // with the kernels' static arrays (less than 16 KB) above the 48 KB that need no asking
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kLgSmemMost);
    if (e == cudaSuccess && w.blocks > 8)
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)w.blocks;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const int64_t step = (int64_t)0x40000000 / w.blocks;
    for (int64_t r0 = 0; r0 < n && e == cudaSuccess; r0 += step) {
        cfg.gridDim = dim3((unsigned)((n - r0 < step ? n - r0 : step) * w.blocks));
        e = cudaLaunchKernelEx(&cfg, kernel, r0, w.per, args...);
    }
    if (e != cudaSuccess) return lfail(CBGPU_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
    return CBGPU_OK;
}
template <typename K, typename... A>
int lg_launch_wide(const char* who, K kernel, int64_t n, const Wide& w, size_t smem, cudaStream_t st, A... args) {
    return lg_launch_wide_n(who, kernel, n, w, kLgThreads, smem, st, args...);
}

// Rows above kLgFew classes are wide when there are few of them: a block of 256 threads a row instead of a
// warp (f32 rows of 256: 300 of them 10 us against 12 for derivatives and top 16; 4000 27 and 41 against 16
// and 23).
bool is_wide(int64_t n, int V) { return V > kLgNarrow || (V > kLgFew && n <= 148 * 2); }

unsigned tiles_of(int64_t n, int rows) { return (unsigned)((n + rows - 1) / rows); }

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
