// logits_distill.cu -- cbgpu_distill: the Kullback-Leibler loss of a student's rows against a teacher's
// top logits, and its derivative.
#include "logits.cuh"

namespace {

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
// no difference of logarithms of rounded sums but ln (s / R), taken in 64 bits.
// Where the others lie far below m (s_t < kFar), their exponentials and s_t are taken relative to the
// largest of the others instead: Q ln s_t and Q / s_t need s_t by itself, not beside s.
constexpr double kFar = 1e-20;

// The teacher's largest logit z_max and its tail: an entry's exponential is exp((z_j - z_max) / T - lift), the
// tail's exp(tail), both at most 1.  Differences are taken before they are scaled, so that their rounding does not
// grow with the logits.
struct TeacherBase {
    double z, tail, lift;
    template <typename C>
    __device__ TeacherBase(C z_max, double tl, const Scale<C>& sc) : z((double)floor_max(z_max)) {
        tail = fma(tl, sc.t, -z) * sc.by_t;  // beside z_max: tl - z / T
        if (tail == lg_inf(0.0) && tl < tail) tail = -lowest(0.0);  // out of range: the entries weigh nothing
        lift = floor_max(fmax(z_max == -lg_inf(C()) ? -lg_inf(0.0) : 0.0, tail));
        tail -= lift;
    }
    __device__ double entry(double zj, double inv_t) const { return fma(zj - z, inv_t, -lift); }
};

// A teacher's exponential r = exp(d) for the loss.  Where the 32-bit one is 0 (from -87 on) the 64-bit one is taken:
// the student's logarithm beside it may be as large as it is small, or infinite.  (64-bit ones end at -707.)
template <typename C>
__device__ __forceinline__ double loss_weight(C r, double d) {
    return sizeof(C) == 4 && r == C(0) && d > -745.0 ? exp(d) : (double)r;
}

template <typename C>
struct RowOut {  // what turns a row's logits into its loss and derivative
    double loss;
    C c_top, c_rest, q_scale;  // der1 = q_scale * r_i - c_top * e_i in S, -c_rest * e_i outside
    bool zero;
};

template <typename C>
__device__ __forceinline__ RowOut<C> distill_finish(double w, double t, double s_top, double s_rest, double r_sum,
                                                    double r_tail, double tail_rel, double cross, double rest_ln) {  // rest_ln: logarithm of s_rest's unit
    RowOut<C> o{};
    const double unit = rest_ln == 0.0 ? 1.0 : exp(rest_ln), s = s_top + s_rest * unit;
    o.zero = s == 0.0 || r_sum == 0.0;  // every class masked (m is 0 then), or a teacher without an entry
    if (o.zero) return o;
    double kl = cross;
    if (r_tail > 0.0 || r_tail != r_tail) kl += r_tail * (tail_rel - log(s_rest) - rest_ln);
    const double per_r = 1.0 / r_sum, per_s = 1.0 / s, wt = w * t;
    o.loss = wt * t * (kl * per_r + log(s * per_r));
    o.q_scale = (C)(wt * per_r);
    o.c_top = (C)(wt * per_s);
    const double q = r_tail * per_r;
    o.c_rest = (C)(wt * (per_s * unit - (q != 0.0 && s_rest != 0.0 ? q / s_rest : (q != q ? q : 0.0))));
    return o;
}

__device__ __forceinline__ float part_exp(float x) { return __expf(x); }
__device__ __forceinline__ double part_exp(double x) { return exp(x); }
// exp(x) for x <= 0 of a narrow row
__device__ __forceinline__ float row_exp(float x, const ExpTable&) { return __expf(x); }
__device__ __forceinline__ double row_exp(double x, const ExpTable& t) { return t.exp<true>(x * ExpTable::kPerUnit); }
__device__ __forceinline__ float row_exp(float d, const Scale<float>& sc, const ExpTable&) { return ex2(d * sc.c); }
__device__ __forceinline__ double row_exp(double d, const Scale<double>& sc, const ExpTable& t) {
    return t.exp<true>(d * sc.c * ExpTable::kPerUnit);
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

// Narrow rows: the student's exponentials stay in registers; tgt[i] = the
// teacher's logit of class i, or absent, and then its exponential.  32-bit rows take the teacher's by __expf, off
// by 2 ulp and one more for each unit of the argument: by 40 ulp where it weighs e^-34.  Bound by issue (1000003 x 10 f64, class by
// class, k 4: 94 us at 74 % of the slots; floor 36; 64-bit exponentials from a table, 165 us with exp()).
template <typename T, int G, int ITEMS>
__global__ void __launch_bounds__(kLgThreads, 4)
lg_distill_narrow_kernel(Rows<T> x, TeacherArgs tc, const typename Num<T>::C* __restrict__ tail,
                         const typename Num<T>::C* __restrict__ weight, double temp, Scale<typename Num<T>::C> sc,
                         int tile, int direct, typename Num<T>::C* __restrict__ loss, T* der1, int64_t drs,
                         int64_t dcs) {
    typedef typename Num<T>::C C;
    extern __shared__ __align__(16) unsigned char lg_smem[];
    const int64_t r0 = (int64_t)blockIdx.x * tile;
    const int rows = (int)(x.n - r0 < tile ? x.n - r0 : tile), V = x.V;
    const int tgt_pitch = V | 1;
    C* tgt_all = reinterpret_cast<C*>(lg_smem);
    T* g = const_cast<T*>(x.data) + r0 * x.row_stride;
    const TileIo<T> io(g, x.row_stride, x.class_stride, V, rows);
    T* s = reinterpret_cast<T*>(lg_smem + ((size_t)tile * tgt_pitch * sizeof(C) + 15) / 16 * 16) + io.shift;
    if (!direct) io.template copy<false>(s, g);
    __shared__ ExpTable table;  // of f64 rows
    if (sizeof(C) == 8) table.fill();
    __syncthreads();
    const LaneTeam<G> t;
    const Items<G, ITEMS> mine(t, V);
    for (int r = threadIdx.x / G; r < rows; r += kLgThreads / G) {
        T* row = s + (size_t)r * io.pitch;
        C* tgt = tgt_all + (size_t)r * tgt_pitch;
        C a[ITEMS] = {};
        if (direct) {
            const T* from = g + r * x.row_stride;
            LG_EACH(it)
                a[it] = mine.has(it) ? to_c(from[(int64_t)(mine.first + it) * x.class_stride]) : -lg_inf(C());
        } else {
            LG_EACH(it) a[it] = mine.has(it) ? to_c(row[mine.first + it]) : -lg_inf(C());
        }
        const double w = weight ? (double)weight[r0 + r] : 1.0;
        const double tl = tail ? (double)tail[r0 + r] : -lg_inf(0.0);
        for (int i = t.rank; i < V; i += G) set_absent(&tgt[i]);
        t.sync();
        u64 claimed = 0;  // which of this lane's entries count, a bit each
        static_assert(G == 1 || kLgMaxTop / G <= 64, "a bit an entry");
        const bool by_entry = G > 1 || 2 * tc.k <= V;  // (V <= 16 of them for a thread)
        for (int j0 = 0; j0 < tc.k; j0 += G) {
            const int j = j0 + t.rank;
            const int64_t at = (r0 + r) * tc.k + j;
            const int64_t idx = j < tc.k ? tc.idx(at) : -1;
            bool take = idx >= 0 && idx < V;
            if (G > 1) {  // of equal indices in this step the first counts
                const unsigned same = __match_any_sync(t.mask, take ? (int)idx : -1 - t.rank);
                take = take && (__ffs(same) - 1) == (int)(threadIdx.x & 31);
            }
            if (take && is_absent(tgt[idx])) {
                tgt[idx] = plain_nan((C)load_any(tc.value, tc.value_dtype, at));
                claimed |= 1ull << (by_entry ? j0 / G : 0);
            }
            t.sync();
        }
        C m = -lg_inf(C()), zm = -lg_inf(C());
        uint32_t top = 0;  // which of this lane's classes are entries
        LG_EACH(it) {
            m = OpMax()(m, a[it]);
            if (!mine.has(it)) continue;
            const C z = tgt[mine.first + it];
            if (!is_absent(z)) top |= 1u << it, zm = OpMax()(zm, z);
        }
        m = floor_max(t.reduce(m, OpMax()));
        zm = t.reduce(zm, OpMax());
        const TeacherBase z_base(zm, tl, sc);
        C sum_top = 0, sum_rest = 0;
        double r_sum = 0.0, cross = 0.0;
        constexpr bool kNone = sizeof(C) == 4;
        u64 none = 0;  // which of this lane's entries have a teacher's 32-bit exponential of 0
        auto logit = [&](int i) { return to_c(direct ? g[r * x.row_stride + (int64_t)i * x.class_stride] : row[i]); };
        // their part of `cross`, for which they keep their logit until here
        auto small = [&](int i) {
            const double d = z_base.entry((double)tgt[i], sc.inv_t), rj = loss_weight(C(0), d);
            if (rj != 0.0) cross += rj * (d - ((double)logit(i) - (double)m) * sc.inv_t);
            tgt[i] = C(0);
        };
        if (by_entry) {  // a lane an entry: fewer steps in 64 bits than by class (for which a warp's rows differ)
            for (int j0 = 0; j0 < tc.k; j0 += G) {
                if (!((claimed >> (j0 / G)) & 1)) continue;
                const int i = (int)tc.idx((r0 + r) * tc.k + j0 + t.rank);
                const C ai = logit(i);
                const double d = z_base.entry((double)tgt[i], sc.inv_t);
                const C rj = row_exp((C)d, table);
                r_sum += (double)rj;
                if (rj != C(0)) cross += (double)rj * (d - ((double)ai - (double)m) * sc.inv_t);
                if (kNone && rj == C(0)) none |= 1ull << (j0 / G);
                else tgt[i] = rj;
            }
            for (; none != 0; none &= none - 1)
                small((int)tc.idx((r0 + r) * tc.k + (__ffsll((long long)none) - 1) * G + t.rank));
            t.sync();
        }
        LG_EACH(it) {
            const C e = row_exp(a[it] - m, sc, table);
            if ((top >> it) & 1) {
                sum_top += e;
                if (by_entry) {
                    a[it] = e;
                    continue;
                }
                const double d = z_base.entry((double)tgt[mine.first + it], sc.inv_t);
                const double rj = (double)row_exp((C)d, table);
                r_sum += rj;
                if (rj != 0.0) cross += rj * (d - ((double)a[it] - (double)m) * sc.inv_t);
                if (kNone && rj == 0.0) none |= 1ull << it;
                else tgt[mine.first + it] = (C)rj;
            } else {
                sum_rest += e;
            }
            a[it] = e;
        }
        for (; none != 0; none &= none - 1) small(mine.first + __ffsll((long long)none) - 1);
        const double s_top = t.reduce((double)sum_top, OpSum());
        double s_rest = t.reduce((double)sum_rest, OpSum()), rest_ln = 0.0;
        r_sum = t.reduce(r_sum, OpSum());
        cross = t.reduce(cross, OpSum());
        const double r_tail = loss_weight(row_exp((C)z_base.tail, table), z_base.tail);
        if (s_rest < kFar && r_tail > 0.0) {  // the same for a row's lanes
            C mr = -lg_inf(C());
            LG_EACH(it) if (mine.has(it) && !((top >> it) & 1)) mr = OpMax()(mr, logit(mine.first + it));
            mr = t.reduce(mr, OpMax());
            if (mr != -lg_inf(C())) {
                C sum = 0;
                LG_EACH(it) if (mine.has(it) && !((top >> it) & 1)) {
                    a[it] = row_exp(logit(mine.first + it) - mr, sc, table);
                    sum += a[it];
                }
                s_rest = t.reduce((double)sum, OpSum());
                rest_ln = ((double)mr - (double)m) * sc.inv_t;
            }
        }
        RowOut<C> o = distill_finish<C>(w, temp, s_top, s_rest, r_sum + r_tail, r_tail, z_base.tail, cross, rest_ln);
        if (w == 0.0) {
            o = RowOut<C>{};
            o.zero = true;
        }
        if (t.rank == 0) loss[r0 + r] = (C)o.loss;
        if (!der1) continue;
        LG_EACH(it) {
            if (!mine.has(it)) continue;
            C d = C(0);
            if (!o.zero)
                d = (top >> it) & 1 ? o.q_scale * tgt[mine.first + it] - o.c_top * a[it] : -o.c_rest * a[it];
            if (direct) der1[(r0 + r) * drs + (int64_t)(mine.first + it) * dcs] = from_c<T>(d);
            else row[mine.first + it] = from_c<T>(d);
        }
    }
    if (der1 && !direct) {
        __syncthreads();
        TileIo<T> to = io;
        to.rs = drs, to.cs = dcs;
        to.flat = io.flat && (dcs == 1 || V == 1) && drs == V;
        to.template copy<true>(s, der1 + r0 * drs);
    }
}

// Wide: a block takes the entries whose classes lie in its part of the row (one
// thread an entry), puts -inf in their place and sums the rest; the blocks
// of the cluster exchange their maxima and sums once through each other's
// shared memory, then each writes its part of der1.  der1 may be the logits'
// own memory: all reads are before the exchange.
// Measured: derivatives of 4096 x 64000 bf16 266 us, 3.9 TB/s of a row's one read and one write (floor 163 us);
// losses of 512 x 131072 f32 92 us (floor 42).  No pipe is full: the exponentials', one a class and pass, is busy
// 51 % of the time (loss: 25 %), and the chain of a block, copy, maximum, sums, exchange, is what the rest waits
// for; three blocks an SM cover a part of it.  Rows held in registers instead were slower
// (the unrolled passes leave the instruction cache), and so were 512 threads a block.
// Roundings to fewer bits than 64 for 32- and 16-bit rows: exponentials (ex2.approx, within 2 ulp) and sums of up
// to 16 of them; a teacher's 64-bit logits, which become f32 as the student's are; the join for der1, whose
// per_e - q / s_rest cancels where the student agrees with the teacher, to 2^-24 of the probabilities.
template <typename C>
struct DistillPart {  // sums relative to the block's own maxima: m of its logits, z of its entries' logits
    double s_rest, s_top, r_sum, cross;
    C m, z, m_rest;  // m_rest: what s_rest is relative to, m or (far below it) the largest of the others
    __device__ C rest() const { return s_rest == 0.0 ? -lg_inf(C()) : m_rest; }
};

constexpr int kClaims = 1024;  // places where entries claim their index

template <typename C>
struct DistillJoin {  // for the second pass, from the joined parts
    C base, c_rest;     // the others: der1 = -c_rest * e, relative to base
    C q_scale, c_top;   // an entry: der1 = q_scale * r - c_top * e, both relative to this block's maxima
    bool zero;
};

// A warp joins the parts, a lane a part.  The second pass waits for this, so it is in C.
template <typename C>
__device__ DistillJoin<C> distill_join(const DistillPart<C>& p, int rank, int blocks, C w, C tl, const Scale<C>& sc) {
    const Base<C> base(floor_max(warp_max(p.m)), sc);
    const TeacherBase z_base(warp_max(p.z), (double)tl, sc);
    const C rest_max = warp_max(p.rest());
    const Base<C> rest(floor_max(rest_max), sc);
    // (a part of weight 0 may have no maximum: relative to 0 instead, its factor can be infinite)
    const C f = p.s_top == 0.0 ? C(0) : Base<C>(floor_max(p.m), sc).shift(base);
    const C h = p.s_rest == 0.0 ? C(0) : Base<C>(floor_max(p.m_rest), sc).shift(rest);
    const C unit = rest_max == -lg_inf(C()) ? C(0) : rest.shift(base);
    const C g = p.r_sum == 0.0 ? C(0) : part_exp((C)z_base.entry((double)floor_max(p.z), sc.inv_t));
    const C r_tail = part_exp((C)z_base.tail);
    const C s_rest = warp_sum((C)p.s_rest * h, blocks);
    const C s = s_rest * unit + warp_sum((C)p.s_top * f, blocks);
    const C r_sum = r_tail + warp_sum((C)p.r_sum * g, blocks);
    const C q = r_tail / r_sum, per_s = C(1) / s;
    DistillJoin<C> j;
    // Without a tail nothing needs the others' sum by itself, and blocks whose others lie far below have not looked
    // for their largest: the others are then relative to the row's maximum, beside which each is 1 at most.
    const bool apart = tl > -lg_inf(C());
    j.base = apart ? rest.m : base.m;
    j.zero = s == C(0) || r_sum == C(0);  // every class masked, or a teacher without an entry
    const C per_e = apart ? per_s * unit : per_s;
    j.c_rest = w * (q != q ? q : (q != C(0) && s_rest != C(0) ? per_e - q / s_rest : per_e));
    j.q_scale = __shfl_sync(0xffffffffu, w / r_sum * g, rank);
    j.c_top = __shfl_sync(0xffffffffu, w * per_s * f, rank);
    return j;
}

// The loss from the parts, in 64 bits; nothing waits for it.
template <typename C>
__device__ double distill_loss(const DistillPart<C>& p, int blocks, double w, double t, double tl, const Scale<C>& sc) {
    const Base<C> base(floor_max(warp_max(p.m)), sc);
    const TeacherBase z_base(warp_max(p.z), tl, sc);
    const double ln_f = Base<C>(floor_max(p.m), sc).ln_shift(base), f = exp(ln_f);
    const double ln_g = z_base.entry((double)floor_max(p.z), sc.inv_t), g = exp(ln_g);
    const C rest_max = warp_max(p.rest());
    const Base<C> rest(floor_max(rest_max), sc);
    const double s_rest =
        warp_sum(p.s_rest == 0.0 ? 0.0 : p.s_rest * exp(Base<C>(floor_max(p.m_rest), sc).ln_shift(rest)), blocks);
    const double rest_ln = rest_max == -lg_inf(C()) ? 0.0 : rest.ln_shift(base);
    const double s_top = warp_sum(p.s_top == 0.0 ? 0.0 : p.s_top * f, blocks);
    const double r_sum = warp_sum(p.r_sum == 0.0 ? 0.0 : p.r_sum * g, blocks);
    const double cross = warp_sum(p.r_sum == 0.0 || g == 0.0 ? 0.0 : g * (p.cross + p.r_sum * (ln_g - ln_f)), blocks);
    const double r_tail = exp(z_base.tail);
    return distill_finish<double>(w, t, s_top, s_rest, r_sum + r_tail, r_tail, z_base.tail, cross, rest_ln).loss;
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT)
lg_distill_wide_kernel(int64_t row0, int per, int64_t ahead, Rows<T> x, TeacherArgs tc, const typename Num<T>::C* __restrict__ tail,
                       const typename Num<T>::C* __restrict__ weight, double temp, Scale<typename Num<T>::C> sc,
                       typename Num<T>::C* __restrict__ loss, T* der1, int64_t drs, int64_t dcs) {
    typedef typename Num<T>::C C;
    constexpr int VE = WideRow<T>::VE, kWarps = NT / 32;
    extern __shared__ __align__(16) unsigned char lg_smem[];
    __shared__ __align__(16) C red_max[2][kWarps];
    __shared__ union {
        int claim[kClaims];
        double red[4][NT];  // s_rest, s_top, r_sum, cross of every thread
    } u;
    __shared__ int s_idx[kLgMaxTop];
    __shared__ DistillPart<C> parts[16];
    __shared__ DistillJoin<C> join;
    __shared__ int s_next;
    uint4* s = reinterpret_cast<uint4*>(lg_smem);
    T* se = reinterpret_cast<T*>(s);
    auto cluster = cooperative_groups::this_cluster();
    const int rank = (int)cluster.block_rank(), blocks = (int)cluster.num_blocks(), k = tc.k;
    const int tid = threadIdx.x, lane = tid & 31, warp_id = tid >> 5;
    const int64_t r = row0 + (int64_t)(blockIdx.x / (unsigned)blocks);
    const WideRow<T> w(x, r, rank, per);
    T* out = der1 ? der1 + r * drs : nullptr;
    // 16-byte stores where der1's row lies to the 16-byte boundaries as the logits' row does
    const bool vec_out = dcs == 1 && w.cs == 1 && (((uintptr_t)out - (uintptr_t)w.head * sizeof(T)) & 15) == 0;
    auto put = [&](int v, const C(&d)[VE]) {
        const int i = w.first(v);
        for (int j = 0; j < VE; ++j)
            if (i + j >= 0 && i + j < w.V) out[(int64_t)(i + j) * dcs] = from_c<T>(d[j]);
    };
    auto put_zeros = [&] {  // whatever the row holds
        const int end = w.first(w.nv) < w.V ? w.first(w.nv) : w.V;
        for (int i = (w.first(0) > 0 ? w.first(0) : 0) + tid; i < end; i += NT) out[(int64_t)i * dcs] = from_c<T>(C(0));
    };
    if (blocks > 1) cluster_arrive<false>();

    // the row's own numbers are asked for before its logits and used after them
    const C wt = weight ? weight[r] : C(1), tl = tail ? tail[r] : -lg_inf(C());
    u64 i_bits = 0, z_bits = 0;
    if (tid < k) {
        i_bits = tc.idx_bits(r * k + tid);
        z_bits = load_bits(tc.value, tc.value_dtype, r * k + tid);
    }
    if (r + ahead < x.n) {
        if (tid == NT - 1) WideRow<T>(x, r + ahead, rank, per).prefetch();
        if (tid < k && (tid & 15) == 0) tc.prefetch((r + ahead) * k + tid);
    }
    for (int i = tid; i < kClaims; i += NT) u.claim[i] = kLgMaxTop;
    if (tid == 0) s_next = 0;
    VecMax<T> most;
    w.template load<NT>(s, [&](const uint4& q) { most(q); });
    if (wt == C(0)) {  // the same for all blocks of the cluster
        if (tid == 0 && rank == 0) loss[r] = 0;
        if (out) put_zeros();
        if (blocks > 1) cluster_wait();
        return;
    }
    const int64_t idx = tid < k ? tc.of_idx_bits(i_bits) : -1;
    C z = tid < k ? (C)of_bits(z_bits, tc.value_dtype) : -lg_inf(C());
    const int own = idx >= 0 && idx < w.V ? (int)idx : -1;  // the class of this thread's entry
    if (tid < k) s_idx[tid] = own;
    __syncthreads();
    int at = own >= 0 ? w.slot(own) : -1;  // its place, if the class is in this block's part
    if (at >= 0) atomicMin(&u.claim[own % kClaims], tid);
    __syncthreads();
    if (warp_id * 32 < k) {
        // of equal indices the first counts: who holds its claim is the first of its index; for the
        // others (equal indices, or two that share a claim) the warp looks through the entries before
        unsigned late = __ballot_sync(0xffffffffu, at >= 0 && u.claim[own % kClaims] != tid);
        for (; late; late &= late - 1) {
            const int l = __ffs(late) - 1, who = warp_id * 32 + l;
            const int mine = __shfl_sync(0xffffffffu, own, l);
            bool again = false;
            for (int j = lane; j < who; j += 32) again |= s_idx[j] == mine;
            if (__any_sync(0xffffffffu, again) && lane == l) at = -1;
        }
    }
    C a_own = -lg_inf(C());
    if (at >= 0) {
        a_own = to_c(se[at]);
        se[at] = from_c<T>(-lg_inf(C()));
    } else {
        z = -lg_inf(C());
    }
    {
        const C m = warp_max(OpMax()(most.get(), a_own)), zm = warp_id * 32 < k ? warp_max(z) : -lg_inf(C());
        if (lane == 0) red_max[0][warp_id] = m, red_max[1][warp_id] = zm;
    }
    __syncthreads();
    C top[2] = {red_max[0][0], red_max[1][0]};
#pragma unroll
    for (int i = 1; i < kWarps; ++i) {
        top[0] = OpMax()(top[0], red_max[0][i]);
        top[1] = OpMax()(top[1], red_max[1][i]);
    }
    const Base<C> here(floor_max(top[0]), sc);
    const double z_here = (double)floor_max(top[1]);

    double sum[4] = {0.0, 0.0, 0.0, 0.0};  // s_rest, s_top, r_sum, cross
#pragma unroll 4
    for (int v = tid; v < w.nv; v += NT) {
        C a[VE];
        unpack(s[v], a, T());
        here.exps(a);
        sum[0] += Base<C>::total(a);
    }
    if (at >= 0) {
        sum[1] = (double)here.exp(a_own);
        const double d = ((double)z - z_here) * sc.inv_t;
        sum[2] = exp(d);
        if (sum[2] != 0.0) sum[3] = sum[2] * (d - here.ln(a_own));
    }
    const double e_own = sum[1], r_own = sum[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) u.red[i][tid] = sum[i];
    C m_rest = top[0];
    if (!__syncthreads_or(!(sum[0] < kFar)) && tl > -lg_inf(C())) {  // the block's others lie far below
        most = VecMax<T>();
        for (int v = tid; v < w.nv; v += NT) most(s[v]);
        const C m = warp_max(most.get());
        if (lane == 0) red_max[0][warp_id] = m;
        __syncthreads();
        m_rest = red_max[0][0];
#pragma unroll
        for (int i = 1; i < kWarps; ++i) m_rest = OpMax()(m_rest, red_max[0][i]);
        const Base<C> rest(floor_max(m_rest), sc);
        double own = 0.0;
        for (int v = tid; v < w.nv; v += NT) {
            C a[VE];
            unpack(s[v], a, T());
            rest.exps(a);
            own += Base<C>::total(a);
        }
        u.red[0][tid] = own;
        __syncthreads();
    }
    // a warp for each of the four sums, which it gives to all blocks of the cluster
    if (blocks > 1) cluster_wait();  // every block runs: its shared memory can be written
    if (warp_id < 4) {
        double v = 0.0;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) v += u.red[warp_id][lane + 32 * i];
        v = warp_sum(v, 32);
        if (lane < blocks) {
            DistillPart<C>* to = cluster.map_shared_rank(&parts[rank], lane);
            if (warp_id == 0) to->s_rest = v, to->m = top[0], to->z = top[1], to->m_rest = m_rest;
            else if (warp_id == 1) to->s_top = v;
            else if (warp_id == 2) to->r_sum = v;
            else to->cross = v;
        }
    }
    if (blocks > 1) {
        if (warp_id < 4) cluster_arrive<true>();
        else cluster_arrive<false>();
        cluster_wait();
    } else {
        __syncthreads();
    }
    DistillPart<C> p{0.0, 0.0, 0.0, 0.0, -lg_inf(C()), -lg_inf(C()), -lg_inf(C())};
    if (lane < blocks) p = parts[lane];
    if (out) {  // one warp works out what the second pass needs
        if (warp_id == 0) {
            const DistillJoin<C> j = distill_join<C>(p, rank, blocks, (C)((double)wt * temp), tl, sc);
            if (lane == 0) join = j;
        }
        __syncthreads();
    }
    if (warp_id == kWarps - 1 && rank == 0) {  // and another the loss, while the others are at the second pass
        const double v = distill_loss<C>(p, blocks, (double)wt, temp, (double)tl, sc);
        if (lane == 0) loss[r] = (C)v;
    }
    if (!out) return;
    if (join.zero) {
        put_zeros();
        return;
    }
    const Base<C> base(join.base, sc);
    const C c = -join.c_rest;
    auto der = [&](int v, C(&a)[VE]) {
        unpack(s[v], a, T());
        base.exps(a);
        Base<C>::times(a, c);
    };
    if (vec_out) {
        uint4* g = reinterpret_cast<uint4*>(out + ((int64_t)w.v0 * VE - w.head));
        const int lo = w.whole_lo(), hi = w.whole_hi();
        constexpr int kRun = 4;  // warps take runs of vectors as they come, since one is late by the loss
        for (;;) {
            int v = 0;
            if (lane == 0) v = atomicAdd(&s_next, kRun * 32);
            v = lo + __shfl_sync(0xffffffffu, v, 0);
            if (v >= hi) break;
            v += lane;
            if (v - lane + kRun * 32 <= hi) {
#pragma unroll
                for (int u = 0; u < kRun; ++u) {
                    C a[VE];
                    der(v + 32 * u, a);
                    __stcs(g + v + 32 * u, pack(a, T()));
                }
            } else {
                for (; v < hi; v += 32) {
                    C a[VE];
                    der(v, a);
                    __stcs(g + v, pack(a, T()));
                }
            }
        }
        w.template ends<NT>([&](int v) {
            C a[VE];
            der(v, a);
            put(v, a);
        });
    } else {
        for (int v = tid; v < w.nv; v += NT) {
            C a[VE];
            der(v, a);
            put(v, a);
        }
    }
    __syncthreads();  // the entries' classes over the zeros just written
    if (at >= 0)
        out[(int64_t)own * dcs] = from_c<T>(join.q_scale * (C)r_own - join.c_top * (C)e_own);
}

template <typename T>
int run_distill(const cbgpu_logits* x, const cbgpu_teacher* tc, const void* weight, double temp, void* loss, void* der1,
                int64_t drs, int64_t dcs, cudaStream_t st) {
    typedef typename Num<T>::C C;
    const char* who = "distill";
    const Rows<T> rows = rows_of<T>(x);
    const Scale<C> sc(temp);
    const TeacherArgs ta{tc->index, tc->value, tc->index_bytes, tc->value_dtype, tc->k};
    if (is_wide(rows.n, rows.V)) {
        auto wide = [&](auto kernel, int threads, const Wide& w) {
            return lg_launch_wide_n(who, kernel, rows.n, w, threads, w.smem, st, w.ahead, rows, ta, (const C*)tc->tail,
                                    (const C*)weight, temp, sc, (C*)loss, (T*)der1, drs, dcs);
        };
        // a thread an entry; small rows by small blocks (20000 x 1000 f32: 119 us against 192)
        if (tc->k <= 128 && (size_t)rows.V * sizeof(T) <= 16384)
            return wide(lg_distill_wide_kernel<T, 128>, 128, wide_shape<T>(rows.n, rows.V));
        return wide(lg_distill_wide_kernel<T, 256>, 256, wide_shape<T>(rows.n, rows.V));
    }
    auto narrow = [&](auto kernel, int lanes) {
        const bool direct = lanes == 1 && rows.class_stride > rows.row_stride && (!der1 || dcs > drs);
        Tile t = narrow_tile(rows.n, rows.V, sizeof(T) + sizeof(C), kLgThreads / lanes);
        if (direct) t = Tile{kLgThreads, (size_t)kLgThreads * (rows.V | 1) * sizeof(C) + 16};
        return lg_launch(who, kernel, tiles_of(rows.n, t.rows), t.smem, st, rows, ta, (const C*)tc->tail,
                         (const C*)weight, temp, sc, t.rows, (int)direct, (C*)loss, (T*)der1, drs, dcs);
    };
    if (rows.V <= 4) return narrow(lg_distill_narrow_kernel<T, 1, 4>, 1);
    if (rows.V <= 12) return narrow(lg_distill_narrow_kernel<T, 1, 12>, 1);
    if (rows.V <= 16) return narrow(lg_distill_narrow_kernel<T, 1, 16>, 1);
    if (rows.V <= 32) return narrow(lg_distill_narrow_kernel<T, 8, 4>, 8);
    if (rows.V <= 128) return narrow(lg_distill_narrow_kernel<T, 8, 16>, 8);
    return narrow(lg_distill_narrow_kernel<T, 32, 16>, 32);
}

}  // namespace

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
    const size_t wide = x->dtype == CBGPU_F64 ? 8 : 4;
    if ((rc = check_aligned("distill", "index", t->index, (size_t)t->index_bytes)) ||
        (rc = check_aligned("distill", "value", t->value, dtype_size(t->value_dtype))) ||
        (rc = check_aligned("distill", "tail", t->tail, wide)) ||
        (rc = check_aligned("distill", "weight", weight, wide)) || (rc = check_aligned("distill", "loss", loss, wide)))
        return rc;
    if (der1) {
        const int64_t n = x->n, V = x->n_classes, rs = der1_row_stride, cs = der1_class_stride;
        if (rs < 0 || cs < 0) return lfail(CBGPU_ERR_INVALID, "distill: negative strides");
        const bool apart = (n == 1 && V == 1) || (n == 1 && cs >= 1) || (V == 1 && rs >= 1) ||
                           (cs >= 1 && rs > cs * (V - 1)) || (rs >= 1 && cs > rs * (n - 1));
        if (!apart) return lfail(CBGPU_ERR_INVALID, "distill: elements of der1 share memory");
        const size_t es = dtype_size(x->dtype);
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

