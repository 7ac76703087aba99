// logits_sample.cu -- cbgpu_sample_classes: a class drawn from a row under temperature / top-k / top-p / min-p.
#include <type_traits>

#include "logits.cuh"

namespace {

// ---- sampling ------------------------------------------------------------------------
//
// e_i = exp((a_i - max) / T) is taken in 64 bits and held as the integer
// w_i = rint(e_i 2^s), with 2^s V <= 2^62, so that every sum of weights is exact
// whatever its order: the draw does not depend on the launch's shape.  A weight
// is off by less than 4 of its last bit (half of it by rint, the rest by the
// exponential and its argument), so a class is drawn as the definition draws it
// unless the drawn number lies within 8 V 2^-s of a border.
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

__device__ __forceinline__ double power_of_2(int e) { return __longlong_as_double((long long)(1023 + e) << 52); }

// rint(e 2^s) through the lowest bits of 2^52 + e 2^s
__device__ __forceinline__ u64 whole_mass(double e, double scale) {
    return (u64)__double_as_longlong(fma(e, scale, 4503599627370496.0)) - 0x4330000000000000ull;
}

// Narrow rows: logits and masses in registers, the classes that stay as bits.
// A thread that has a row to itself counts for each class what comes before
// it; a team finds the cut by halving an interval of logits.  Bound by issue: 100000 x 10 f64, top-k and
// top-p, 15 us at 60 % of the slots, of which 64-bit arithmetic is a fifth; with exp() instead of the
// table 37 us.
template <typename T, int G, int ITEMS>
__device__ int sample_row(const LaneTeam<G>& t, const Items<G, ITEMS>& mine, const typename Num<T>::C (&a)[ITEMS], int V,
                          int shift, const RowSampling& rs, const ExpTable& table) {
    typedef typename Num<T>::C C;
    const double scale = power_of_2(shift);
    const double reach = (double)(shift + 2) * 0.6931471805599453 / rs.inv_t;  // behind it a weight is 0
    const double per64 = rs.inv_t * ExpTable::kPerUnit;
    C m = -lg_inf(C());
    int bad = 0;
    LG_EACH(it) {
        if (!mine.has(it)) continue;
        bad |= a[it] != a[it];
        m = OpMax()(m, a[it]);
    }
    m = t.reduce(m, OpMax());
    bad = t.reduce(bad, OpOr());
    if (bad || m == -lg_inf(C())) return -1;
    if (rs.greedy) {
        int at = 0x7fffffff;
#pragma unroll
        for (int it = ITEMS - 1; it >= 0; --it)
            if (mine.has(it) && a[it] == m) at = mine.first + it;
        return t.reduce(at, OpMin());
    }
    u64 w[ITEMS] = {};
    uint32_t stay = 0, small = 0;  // small: below min-p
    LG_EACH(it) {
        w[it] = 0;
        if (!mine.has(it)) continue;
        const double e = a[it] == m ? 1.0 : table.exp<false>(((double)a[it] - (double)m) * per64);
        w[it] = whole_mass(e, scale);
        stay |= 1u << it;
        if (e < rs.min_p) small |= 1u << it;
    }
    // Keeps the shortest prefix (in order) of what stays whose metric, the
    // number or the mass of classes, reaches `target`.
    auto cut = [&](u64 target, auto by_mass) {
        constexpr bool kMass = decltype(by_mass)::value;
        // [lo, hi): where the last class that stays lies; it is halved until it holds one class or
        // one value
        u64 mass = 0;
        int n = 0;
        auto from = [&](C least) {
            mass = 0, n = 0;
            LG_EACH(it) if (((stay >> it) & 1) && a[it] >= least) {
                ++n;
                if (kMass) mass += w[it];
            }
            n = team_count(t, n);
            if (kMass) mass = t.sum(mass);
            return (kMass ? mass : (u64)n) >= target;
        };
        C lo = m, hi = lg_inf(C());
        if (!from(m)) {
            if (m == lg_inf(C())) return;  // beside infinite logits the others weigh nothing
            hi = m;
            int n_hi = n;
            C low = m;
            // (masked classes, -inf, weigh nothing, and towards them an interval of 16-bit logits cannot be halved)
            LG_EACH(it) if (((stay >> it) & 1) && a[it] > -lg_inf(C())) low = a[it] < low ? a[it] : low;
            low = t.reduce(low, OpMin());
            lo = (C)((double)m - reach);
            lo = low > lo ? low : lo;
            if (!from(lo)) return;  // what would be cut weighs nothing
            int n_lo = n;
            while (n_lo - n_hi > 1) {
                const C mid = to_c(from_c<T>(lo * C(0.5) + hi * C(0.5)));  // a logit there can be
                if (!(mid > lo && mid < hi)) break;
                if (from(mid)) lo = mid, n_lo = n;
                else hi = mid, n_hi = n;
            }
        }
        u64 above = 0, ties = 0;
        LG_EACH(it) if (((stay >> it) & 1) && a[it] >= lo) {
            (a[it] >= hi && hi > lo ? above : ties) += kMass ? w[it] : 1;
        }
        // of equal logits the lower indices: the lanes' classes are in the order of the lanes
        u64 before = t.sum(above) + t.exscan(ties);
        uint32_t keep = 0;
        LG_EACH(it) if (((stay >> it) & 1) && a[it] >= lo) {
            const bool sure = a[it] >= hi && hi > lo;
            if (sure || before < target) keep |= 1u << it;
            if (!sure) before += kMass ? w[it] : 1;
        }
        stay = keep;
    };
    auto sum_of = [&](uint32_t bits) {
        u64 f = 0;
        LG_EACH(it)
            if ((bits >> it) & 1) f += w[it];
        return f;
    };
    if (G == 1) {
        if (rs.top_k < V || rs.top_p < 1.0) {
            // what comes before each class, from one comparison a pair; before a class that top-k
            // keeps all stays, so the masses serve top-p too
            int rank[ITEMS] = {};
            u64 before[ITEMS] = {};
#pragma unroll
            for (int j = 1; j < ITEMS; ++j)
#pragma unroll
                for (int i = 0; i < j; ++i) {
                    const bool first = !(a[j] > a[i]);  // places without a class hold -inf
                    rank[j] += first, rank[i] += !first;
                    if (first) before[j] += w[i];
                    else before[i] += w[j];
                }
            u64 total = 0;
#pragma unroll
            for (int it = 0; it < ITEMS; ++it) {
                if (rank[it] >= rs.top_k) stay &= ~(1u << it);
                total += (stay >> it) & 1 ? w[it] : 0;
            }
            const u64 goal = rs.top_p < 1.0 ? mass_part(rs.top_p, total) : total + 1;
#pragma unroll
            for (int it = 0; it < ITEMS; ++it)
                if (before[it] >= goal) stay &= ~(1u << it);
        }
    } else if (rs.top_k <= 8 && rs.top_k < V) {
        // a few: one by one in order, as many as top-k asks for, then until top-p's mass is there
        uint32_t from = stay, got = 0;
        auto next = [&](u64& its) {
            C best = -lg_inf(C());
            LG_EACH(it) if ((from >> it) & 1) best = OpMax()(best, a[it]);
            const C top = t.reduce(best, OpMax());
            int at = ITEMS;
            its = 0;
#pragma unroll
            for (int it = ITEMS - 1; it >= 0; --it)
                if (((from >> it) & 1) && a[it] == top) at = it, its = w[it];
            const int i = at < ITEMS ? mine.first + at : 0x7fffffff, first = t.reduce(i, OpMin());
            if (i == first && at < ITEMS) from &= ~(1u << at), got |= 1u << at;
            its = i == first && at < ITEMS ? its : 0;
        };
        u64 its;
        for (int j = 0; j < rs.top_k; ++j) next(its);
        stay = got;
        if (rs.top_p < 1.0) {
            const u64 goal = mass_part(rs.top_p, t.sum(sum_of(stay)));
            from = stay, got = 0;
            u64 before = 0;
            for (int j = 0; j < rs.top_k && before < goal; ++j) {
                next(its);
                before += t.sum(its);
            }
            stay = got;
        }
    } else {
        if (rs.top_k < V) cut((u64)rs.top_k, std::false_type());
        if (rs.top_p < 1.0) cut(mass_part(rs.top_p, t.sum(sum_of(stay))), std::true_type());
    }
    stay &= ~small;
    const u64 own = sum_of(stay);
    u64 upto = t.exscan(own);
    const u64 target = draw_target(rs.u, t.sum(own));
    int at = 0x7fffffff;
    LG_EACH(it) {
        if (!((stay >> it) & 1)) continue;
        if (upto < target && upto + w[it] >= target) at = mine.first + it;
        upto += w[it];
    }
    return t.reduce(at, OpMin());
}

template <typename T, int G, int ITEMS>
__global__ void __launch_bounds__(kLgThreads, ITEMS == 32 ? (sizeof(T) == 8 ? 1 : 2) : (sizeof(T) == 8 ? 3 : 4))
lg_sample_narrow_kernel(Rows<T> x, SampleArgs a, int shift, int tile, int direct, int32_t* __restrict__ index) {
    typedef typename Num<T>::C C;
    extern __shared__ __align__(16) unsigned char lg_smem[];
    const int64_t r0 = (int64_t)blockIdx.x * tile;
    const int rows = (int)(x.n - r0 < tile ? x.n - r0 : tile), V = x.V;
    T* g = const_cast<T*>(x.data) + r0 * x.row_stride;
    const TileIo<T> io(g, x.row_stride, x.class_stride, V, rows);
    T* s = reinterpret_cast<T*>(lg_smem) + io.shift;
    if (!direct) io.template copy<false>(s, g);
    __shared__ ExpTable table;
    table.fill();
    __syncthreads();
    const LaneTeam<G> t;
    const Items<G, ITEMS> mine(t, V);
    for (int r = threadIdx.x / G; r < rows; r += kLgThreads / G) {
        C v[ITEMS];
#pragma unroll
        for (int it = 0; it < ITEMS; ++it) v[it] = -lg_inf(C());
        if (direct) {
            const T* row = g + r * x.row_stride;
            LG_EACH(it)
                v[it] = mine.has(it) ? to_c(row[(int64_t)(mine.first + it) * x.class_stride]) : -lg_inf(C());
        } else {
            const T* row = s + (size_t)r * io.pitch;
            LG_EACH(it) v[it] = mine.has(it) ? to_c(row[mine.first + it]) : -lg_inf(C());
        }
        const int got = sample_row<T, G, ITEMS>(t, mine, v, V, shift, row_sampling(a, r0 + r, V), table);
        if (t.rank == 0) index[r0 + r] = got;
    }
}

// ---- wide rows -------------------------------------------------------------------------------
//
// top-k up to kLgMaxTop: the first block collects the first k classes and does the rest alone.
// Else each class is weighed once, or again where the cut was not in the bin
// it was looked for in.  Where top-p or a larger top-k cuts, a
// histogram of the logits shows in which bin the cut lies (a bin's classes weigh nearly the same, so
// counts are enough: f32 masses added in shared memory took three times as long); the
// bin's classes and its neighbours' are collected and sorted, and the cut is then taken
// with exact masses, which also show whether the bin was the right one.
// Measured: 64 x 131071 f32 without cuts 32 us, where 64-bit exponentials take a fifth of their pipe and the
// rest is a block's chain of copy, maximum, masses and draw, three cluster barriers long; 256 x 128000
// bf16 with top-k 50 by row 37 us (1.8 TB/s); one row of 32000, top-p, 18 us on the device.  Cuts over many
// rows are far from their floor (256 x 128000 bf16, 10 us): top-k 1000 with top-p 0.95 186 us, through the four
// passes over shared memory; top-p 0.95 alone over normal logits 1300 us and more, where three bins hold more classes
// than the list (kTopCap) and the cut is found bit by bit.

template <typename T>
struct Weigh {
    typedef typename Num<T>::C C;
    typedef typename Num<T>::Key Key;
    C m;
    double inv_t, scale, min_p;
    Ranked<Key> last;  // the last class that stays
    bool cut, infinite;
    const ExpTable* table;
    double per64;  // 64 log2(e) / T
    __device__ Weigh(C m_, double inv_t_, int shift, const ExpTable* t)
        : m(m_), inv_t(inv_t_), scale(power_of_2(shift)), min_p(0.0), last{0, 0xffffffffu}, cut(false),
          infinite(m_ == lg_inf(C())), table(t), per64(inv_t_ * ExpTable::kPerUnit) {}
    __device__ double finite_share(C a) const { return table->template exp<false>(((double)a - (double)m) * per64); }
    // infinite logits share the mass among themselves
    __device__ double share(C a) const { return infinite ? (a == m ? 1.0 : 0.0) : finite_share(a); }
    __device__ u64 whole(double e) const { return whole_mass(e, scale); }
    __device__ u64 mass(C a) const { return whole(share(a)); }
    __device__ bool stays(int i, C a) const {
        const Key k = key_of(a);
        return !cut || k > last.key || (k == last.key && (uint32_t)i <= last.idx);
    }
    __device__ u64 operator()(int i, C a) const {
        if (!stays(i, a)) return 0;
        const double e = share(a);
        return e < min_p ? 0 : whole(e);
    }
    // no cut, no min-p, no infinite logits
    __device__ bool plain() const { return !(cut || infinite || min_p > 0.0); }
    // the mass of a vector whose first class is i
    template <int N>
    __device__ u64 vector(int i, const C (&a)[N]) const {
        u64 sum = 0;
        if (!plain()) {
#pragma unroll
            for (int j = 0; j < N; ++j) sum += (*this)(i + j, a[j]);
            return sum;
        }
#pragma unroll
        for (int j = 0; j < N; ++j) sum += whole(finite_share(a[j]));
        return sum;
    }
};

// Exclusive scan of a value a thread over the block, and the block's sum.
__device__ __forceinline__ u64 block_exscan(u64 v, u64 (&warp_part)[kLgWarps], u64& total) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    u64 inc = v;
    for (int o = 1; o < 32; o <<= 1) {
        const u64 t = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += t;
    }
    if (lane == 31) warp_part[wid] = inc;
    __syncthreads();
    u64 base = 0;
    total = 0;
    for (int i = 0; i < kLgWarps; ++i) {
        if (i == wid) base = total;
        total += warp_part[i];
    }
    __syncthreads();
    return base + inc - v;
}
__device__ __forceinline__ u64 block_total(u64 v, u64 (&warp_part)[kLgWarps]) {
    v = LaneTeam<32>().sum(v);
    if ((threadIdx.x & 31) == 0) warp_part[threadIdx.x >> 5] = v;
    __syncthreads();
    u64 t = 0;
    for (int i = 0; i < kLgWarps; ++i) t += warp_part[i];
    __syncthreads();
    return t;
}

// Draws from the classes that stay, given the mass that stays in each of the
// block's segments of 32 vectors (sh.segment, behind a barrier); every block of the cluster, one of
// them writes.
template <typename T, typename Sh>
__device__ void segment_draw(const ClusterInfo& cl, Sh& sh, const WideRow<T>& w, const uint4* s, const Weigh<T>& weigh,
                             int segs, double u, int& turn, int32_t* index) {
    constexpr int VE = WideRow<T>::VE;
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const u64* seg = sh.segment;
    // a run of segments a thread
    const int per = (segs + kLgThreads - 1) / kLgThreads, g0 = (int)threadIdx.x * per;
    u64 own = 0, block[1];
    for (int g = g0; g < g0 + per && g < segs; ++g) own += seg[g];
    u64 upto = block_exscan(own, sh.warp_part[0], block[0]);
    const u64(*of)[kGather] = cluster_gather<1>(cl, sh, block, turn);
    u64 total = 0, before = 0;
    for (int b = 0; b < cl.blocks; ++b) {
        if (b == cl.rank) before = total;
        total += of[b][0];
    }
    const u64 target = draw_target(u, total);
    if (!(before < target && before + block[0] >= target)) return;  // another block's
    __shared__ int s_seg;
    __shared__ u64 s_upto;
    upto += before;
    if (upto < target && upto + own >= target)
        for (int g = g0;; ++g) {
            if (upto + seg[g] >= target) {
                s_seg = g, s_upto = upto;
                break;
            }
            upto += seg[g];
        }
    __syncthreads();
    if (wid != 0) return;
    const int v = s_seg * 32 + lane;
    typename Num<T>::C a[VE];
    u64 mine = 0;
    if (v < w.nv) {
        unpack(s[v], a, T());
        mine = weigh.vector(w.first(v), a);
    }
    u64 sum = s_upto + LaneTeam<32>().exscan(mine);
    if (sum < target && sum + mine >= target) {
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            const u64 next = sum + weigh(w.first(v) + j, a[j]);
            if (sum < target && next >= target) *index = w.first(v) + j;
            sum = next;
        }
    }
}

// The segments' masses class by class, and the draw.
template <typename T, typename Sh>
__device__ void wide_draw(const ClusterInfo& cl, Sh& sh, const WideRow<T>& w, const uint4* s, const Weigh<T>& weigh,
                          double u, int& turn, int32_t* index) {
    const int lane = threadIdx.x & 31;
    const int segs = w.nv > 0 ? (w.nv + 31) / 32 : 0;
    const LaneTeam<32> warp;
    for (int g = threadIdx.x >> 5; g < segs; g += kLgWarps) {
        const int v = g * 32 + lane;
        u64 own = 0;
        if (v < w.nv) {
            typename Num<T>::C a[WideRow<T>::VE];
            unpack(s[v], a, T());
            own = weigh.vector(w.first(v), a);
        }
        own = warp.sum(own);
        if (lane == 0) sh.segment[g] = own;
    }
    __syncthreads();
    segment_draw(cl, sh, w, s, weigh, segs, u, turn, index);
}

// The draw from the first block's sorted list of k <= kLgThreads classes: a thread a class.
template <typename T, typename Sh>
__device__ void list_draw(Sh& sh, int k, const Weigh<T>& weigh, const RowSampling& rs, int32_t* index) {
    typedef typename Num<T>::C C;
    const int j = threadIdx.x;
    static_assert(kTopCap - 512 >= 2 * kLgThreads, "masses behind the list");
    u64* w_of = reinterpret_cast<u64*>(&sh.idx[512]);
    const double e = j < k ? weigh.share((C)of_key(sh.key[j])) : 0.0;
    u64 own = j < k ? weigh.whole(e) : 0;
    if (rs.top_p < 1.0) {
        u64 total;
        const u64 before = block_exscan(own, sh.warp_part[0], total);
        if (before >= mass_part(rs.top_p, total)) own = 0;
    }
    if (e < rs.min_p) own = 0;
    const u64 target = draw_target(rs.u, block_total(own, sh.warp_part[0]));
    w_of[j] = own;
    __syncthreads();
    if (own == 0) return;
    u64 upto = 0;  // of the kept classes before this one by index
#pragma unroll 8
    for (int i = 0; i < k; ++i) upto += sh.idx[i] < sh.idx[j] ? w_of[i] : 0;
    if (upto < target && upto + own >= target) *index = (int32_t)sh.idx[j];
}

// What a launch's rows can ask for, so that its kernel holds no registers for the rest: no cut at all,
// a top-k from the list alone, or anything (settings by rows).
enum WidePath { kPathPlain, kPathList, kPathAny };

template <typename T, WidePath kPath>
__global__ void __launch_bounds__(kLgThreads, 3)
lg_sample_wide_kernel(int64_t row0, int per, int64_t ahead, Rows<T> x, SampleArgs a, int shift,
                      int32_t* __restrict__ index) {
    typedef typename Num<T>::C C;
    typedef typename Num<T>::Key Key;
    extern __shared__ __align__(16) unsigned char lg_smem[];
    __shared__ TopShared<Key> sh;
    __shared__ C red_max[2][kLgWarps];
    __shared__ Ranked<Key> s_cut;
    __shared__ ExpTable table;
    uint4* s = reinterpret_cast<uint4*>(lg_smem);
    const ClusterInfo cl;
    const int tid = threadIdx.x;
    const int64_t r = row0 + (int64_t)(blockIdx.x / (unsigned)cl.blocks);
    const WideRow<T> w(x, r, cl.rank, per);
    if (cl.blocks > 1) cluster_arrive<false>();
    if (tid == 0 && r + ahead < x.n) WideRow<T>(x, r + ahead, cl.rank, per).prefetch();
    VecMaxNan<T> most;
    w.load(s, [&](const uint4& q) { most(q); });
    table.fill();
    const RowSampling rs = row_sampling(a, r, x.V);
    const C mine = most.get();
    int32_t* out = index + r;
    int turn = 0;
    if (cl.blocks > 1) cluster_wait();  // every block runs: its shared memory can be written
    if (kPath != kPathPlain && rs.top_k <= kLgMaxTop && !rs.greedy) {
        C rest;
        bool exact, bad = mine != mine;
        const int n = wide_top(cl, sh, w, s, bad ? -lg_inf(C()) : mine, rs.top_k, turn, rest, exact, bad,
                               [](C(&)[WideRow<T>::VE], C) {});
        if (cl.blocks > 1) cl.sync();  // no block leaves while another reads its shared memory
        if (cl.rank != 0) return;
        __syncthreads();
        sort_list(sh, n);
        const C m = (C)of_key(sh.key[0]);
        if (bad || m == -lg_inf(C())) {
            if (tid == 0) *out = -1;
            return;
        }
        list_draw<T>(sh, rs.top_k, Weigh<T>(m, rs.inv_t, shift, &table), rs, out);
        return;
    }
    // the largest logit, and the least that is not masked (negated)
    C low = -lg_inf(C());
    if (kPath == kPathAny && (rs.top_k < x.V || rs.top_p < 1.0))
        each_place(w, s, [&](int, C v, int) { low = v != -lg_inf(C()) ? OpMax()(low, -v) : low; });
    C ends[2] = {mine, low};
    block_reduce(ends, red_max, [](C p, C q) { return VecMaxNan<C>::both(p, q); });
    {
        const u64 v[2] = {(u64)__double_as_longlong((double)ends[0]), (u64)__double_as_longlong((double)ends[1])};
        const u64(*of)[kGather] = cluster_gather<2>(cl, sh, v, turn);
        for (int b = 0; b < cl.blocks; ++b) {
            ends[0] = VecMaxNan<C>::both(ends[0], (C)__longlong_as_double((long long)of[b][0]));
            ends[1] = OpMax()(ends[1], (C)__longlong_as_double((long long)of[b][1]));
        }
    }
    const C m = ends[0];
    if (m != m || m == -lg_inf(C())) {  // a NaN, or every class masked
        if (cl.rank == 0 && tid == 0) *out = -1;
        return;
    }
    if (rs.greedy) {
        uint32_t at = 0xffffffffu;
        each_class(w, s, [&](int i, C v, int) { at = v == m && (uint32_t)i < at ? (uint32_t)i : at; });
        at = __reduce_min_sync(0xffffffffu, at);
        if (tid == 0) sh.count = 0x7fffffff;
        __syncthreads();
        if ((tid & 31) == 0) atomicMin(&sh.count, (int)(at & 0x7fffffffu));
        __syncthreads();
        const u64 v[1] = {(u64)sh.count};
        const u64(*of)[kGather] = cluster_gather<1>(cl, sh, v, turn);
        u64 first = of[0][0];
        for (int b = 1; b < cl.blocks; ++b) first = first < of[b][0] ? first : of[b][0];
        if (cl.rank == 0 && tid == 0) *out = (int32_t)first;
        return;
    }
    Weigh<T> weigh(m, rs.inv_t, shift, &table);
    if (kPath == kPathAny && (rs.top_k < x.V || rs.top_p < 1.0)) {
        const bool by_count = rs.top_k < x.V, by_mass = rs.top_p < 1.0;
        // behind it a weight is below a quarter of the last bit: 0
        const float reach = (float)((double)(shift + 2) * 0.6931471805599453 / rs.inv_t);
        const float range = fminf((float)(m + ends[1]), reach);
        // (0: one bin for all that is not masked; a range of some 1e-36 has no reciprocal to scale by)
        const float per_bin = range > 3e-35f && range < lg_inf(0.0f) ? (float)(kBins - 1) / range : 0.0f;
        auto bin_of = [&](C v) {  // larger logits have lower bins
            if (weigh.infinite) return v == m ? 0 : kBins - 1;
            const float d = fminf((float)(m - v) * per_bin, (float)(kBins - 1));
            return __float_as_int(d + 8388608.0f) & (kBins - 1);
        };
        for (int i = tid; i < kBins; i += kLgThreads) sh.hist.count[i] = 0u;
        __syncthreads();
        // (places outside the row, -inf, weigh nothing and are counted in the last bin, behind any cut)
        each_place(w, s, [&](int, C v, int) { atomicAdd(&sh.hist.count[bin_of(v)], 1u); });
        __shared__ struct {
            int bin, count_bin;  // top-p's and top-k's
            u64 above;           // classes before top-k's bin
        } found;
        // the first block adds the histograms up and gives the bins to all
        if (cl.blocks > 1) {
            cl.sync();
            if (cl.rank != 0) {
                SampleHist* to = cl.of(&sh.hist, 0);
                for (int i = tid; i < kBins; i += kLgThreads)
                    if (sh.hist.count[i] != 0u) atomicAdd(&to->count[i], sh.hist.count[i]);
            }
        }
        cl.sync();
        if (cl.rank == 0) {
            constexpr int kPer = kBins / kLgThreads;
            // masses in 2^-20: a bin weighs its count times its middle's weight
            const float c = per_bin > 0.0f ? (float)(rs.inv_t * 1.4426950408889634) / per_bin : 0.0f;
            u64 mass_bin[kPer], mass_own = 0, count_own = 0, mass_all, count_all;
            for (int j = 0; j < kPer; ++j) {
                const int bin = tid * kPer + j;
                mass_bin[j] = (u64)((double)sh.hist.count[bin] * (double)ex2(-(float)bin * c) * 1048576.0);
                mass_own += mass_bin[j];
                count_own += sh.hist.count[bin];
            }
            const u64 mass_upto = block_exscan(mass_own, sh.warp_part[0], mass_all);
            const u64 count_upto = block_exscan(count_own, sh.warp_part[1], count_all);
            __shared__ u64 s_mass;  // of what top-k leaves, to a bin
            if (tid == 0) found.bin = 0, found.count_bin = 0, found.above = 0, s_mass = mass_all;
            __syncthreads();
            const u64 k = (u64)rs.top_k;
            if (by_count && count_upto < k && count_upto + count_own >= k) {
                u64 above = count_upto, mass = mass_upto;
                int j = 0;
                for (; above + sh.hist.count[tid * kPer + j] < k; ++j) above += sh.hist.count[tid * kPer + j], mass += mass_bin[j];
                found.count_bin = tid * kPer + j, found.above = above;
                s_mass = mass + mass_bin[j];
            }
            __syncthreads();
            const u64 goal = (u64)(rs.top_p * (double)s_mass);
            if (by_mass && mass_upto < goal && mass_upto + mass_own >= goal) {
                u64 upto = mass_upto;
                int j = 0;
                for (; j + 1 < kPer; ++j) {
                    upto += mass_bin[j];
                    if (upto >= goal) break;
                }
                found.bin = tid * kPer + j;
            }
            if (tid == 0) sh.count = 0;
            __syncthreads();
            if (tid > 0 && tid < cl.blocks) *cl.of(&found, tid) = found;
        }
        cl.sync();  // the bins are known, and the list can take the histogram's place
        auto push = [&](int i, C v) {
            TopShared<Key>* first = cl.of(&sh, 0);
            const int p = atomicAdd(&first->count, 1);
            if (p < kTopCap) first->key[p] = key_of(v), first->idx[p] = (uint32_t)i;
        };
        auto restart = [&] {  // an empty list; also ends what read the last one
            cl.sync();
            if (cl.rank == 0 && tid == 0) sh.count = 0;
            cl.sync();
        };
        auto give_cut = [&](const Ranked<Key>& cut) {  // by one thread of the first block
            for (int b = 0; b < cl.blocks; ++b) *cl.of(&s_cut, b) = cut;
        };
        if (by_count) {
            const u64 k = (u64)rs.top_k;
            const int bin = found.count_bin;
            const u64 above = found.above;
            weigh.cut = bin < kBins - 1 || range < reach;  // else what is cut weighs nothing
            if (weigh.cut)
                each_place(w, s, [&](int i, C v, int) {
                    if (bin_of(v) == bin && w.valid(i)) push(i, v);
                });
            cl.sync();
            const int n = cl.of(&sh, 0)->count;
            if (!weigh.cut) {
            } else if (n <= kTopCap) {
                if (cl.rank == 0) {
                    sort_list(sh, n);
                    const int j = (int)(k - above) - 1;
                    if (tid == 0) give_cut(Ranked<Key>{sh.key[j], sh.idx[j]});
                }
                cl.sync();
                weigh.last = s_cut;
            } else {
                weigh.last = cluster_select(cl, sh, w, s, k, turn, [](int, C, Key) { return 1ull; });
            }
        }
        if (by_mass) {
            // The masses above the bin are kept by segments on the way (lane r of a warp has the r-th of its
            // segments), so that the draw has only the bin's own classes to add.
            const int lane = tid & 31, wid = tid >> 5, segs = w.nv > 0 ? (w.nv + 31) / 32 : 0;
            constexpr int VE = WideRow<T>::VE;
            u64 kept = 0;
            int bin = found.bin, lo = -1, hi = kBins, step = 1;  // the cut's bin is in (lo, hi)
            for (bool first = !by_count;; first = false) {
                if (!first) restart();
                // logits above `high` are before the bin's neighbours, those from `low` on are in one of the three
                const C high = per_bin > 0.0f && bin >= 2 ? m - (C)(((float)bin - 1.5f) / per_bin) : lg_inf(C());
                C low = per_bin > 0.0f && bin + 2 < kBins ? m - (C)(((float)bin + 1.5f) / per_bin) : -lg_inf(C());
                low = OpMax()(low, lowest(C()));  // not the masked classes
                u64 sums[3] = {0, 0, 0};          // of all that stays; above; collected
                if (tid == 0) sh.vectors = 0;
                __syncthreads();
                auto weigh_all = [&](auto plain) {
                    int round = 0;
                    for (int g = wid; g < segs; g += kLgWarps, ++round) {
                        const int v = g * 32 + lane;
                        u64 own = 0;  // above, and not too small for min-p
                        if (v < w.nv) {
                            C a[VE];
                            unpack(s[v], a, T());
                            const int i = w.first(v);
#pragma unroll
                            for (int j = 0; j < VE; ++j) {
                                u64 f;
                                if (decltype(plain)::value) {
                                    f = weigh.whole(weigh.finite_share(a[j]));
                                    if (a[j] > high) own += f;
                                } else {
                                    if (!weigh.stays(i + j, a[j])) continue;
                                    const double e = weigh.share(a[j]);
                                    f = weigh.whole(e);
                                    if (a[j] > high) {
                                        sums[1] += f;
                                        own += e < rs.min_p ? 0 : f;
                                    }
                                }
                                sums[0] += f;
                                if (a[j] <= high && a[j] >= low && w.valid(i + j)) {
                                    sums[2] += f;
                                    push(i + j, a[j]);
                                    const int p = atomicAdd(&sh.vectors, 1);
                                    if (p < kHits) sh.hit[p] = (uint16_t)(v * VE + j);
                                }
                            }
                        }
                        if (decltype(plain)::value) sums[1] += own;
                        own = LaneTeam<32>().sum(own);
                        if (lane == round) kept = own;
                    }
                };
                if (weigh.plain() && !(rs.min_p > 0.0)) weigh_all(std::true_type());
                else weigh_all(std::false_type());
                cluster_total<3>(cl, sh, sums, turn);
                const u64 above = sums[1], within = sums[2], goal = mass_part(rs.top_p, sums[0]);
                const bool before = above >= goal, behind = above + within < goal;
                if ((before || behind) && hi - lo > 2) {  // the bins' weights were a little off: bins near
                    if (before) hi = bin - 1 > lo ? bin - 1 : lo + 1, bin = bin - 1 - step;
                    else lo = bin + 1 < hi ? bin + 1 : hi - 1, bin = bin + 1 + step;
                    bin = bin > lo ? (bin < hi ? bin : hi - 1) : lo + 1;
                    bin = bin < 0 ? 0 : (bin < kBins ? bin : kBins - 1);
                    step *= 2;
                    continue;
                }
                const int n = cl.of(&sh, 0)->count;
                Ranked<Key> last;
                if (n <= kTopCap && !before && !behind) {
                    if (cl.rank == 0) {
                        sort_list(sh, n);
                        // a run of the list a thread
                        const int run = (n + kLgThreads - 1) / kLgThreads, j0 = tid * run;
                        u64 own = 0;
                        for (int j = j0; j < j0 + run && j < n; ++j) own += weigh.mass((C)of_key(sh.key[j]));
                        u64 all;
                        u64 upto = above + block_exscan(own, sh.warp_part[0], all);
                        if (upto < goal && upto + own >= goal)
                            for (int j = j0;; ++j) {
                                upto += weigh.mass((C)of_key(sh.key[j]));
                                if (upto >= goal) {
                                    give_cut(Ranked<Key>{sh.key[j], sh.idx[j]});
                                    break;
                                }
                            }
                    }
                    cl.sync();
                    last = s_cut;
                } else {
                    last = cluster_select(cl, sh, w, s, goal, turn, [&](int i, C v, Key) {
                        return weigh.stays(i, v) ? weigh.mass(v) : 0ull;
                    });
                }
                weigh.last = last;
                weigh.cut = true;
                weigh.min_p = rs.min_p;
                // (the list is read: cl.sync or cluster_select came after)
                // (of the block alone: what follows goes round the cluster once either way)
                if (before || behind || segs > 32 * kLgWarps || sh.vectors > kHits) break;  // weighed anew below
                const int g = wid + kLgWarps * lane;
                if (g < segs) sh.segment[g] = kept;
                __syncthreads();
                for (int p = tid; p < sh.vectors; p += kLgThreads) {
                    const int at = sh.hit[p];
                    const C a = to_c(reinterpret_cast<const T*>(s)[at]);
                    atomicAdd(&sh.segment[at / (VE * 32)], weigh(w.first(0) + at, a));
                }
                __syncthreads();
                segment_draw(cl, sh, w, s, weigh, segs, rs.u, turn, out);
                return;
            }
        }
    }
    weigh.min_p = rs.min_p;
    __syncthreads();
    wide_draw(cl, sh, w, s, weigh, rs.u, turn, out);
}

// A warp draws from up to kLgNarrow classes in less time than a block (f32 rows of 512, top-p: 8 of them 21 us
// against 23, 20000 156 against 522), and from twice as many when the rows fill the SMs (f32 rows of 700, top-p: 8
// of them 27 against 25, 1184 29 against 47, 20000 242 against 532).
constexpr int kSampleNarrow = 1024;
constexpr int64_t kSampleMany = 148 * 8;

template <typename T>
int run_sample(const cbgpu_logits* x, const cbgpu_sampling* s, int32_t* index, cudaStream_t st) {
    const char* who = "sample_classes";
    const Rows<T> rows = rows_of<T>(x);
    const SampleArgs a{s->uniform,          s->uniform_dtype, s->top_k,      s->temperature, s->top_p, s->min_p,
                       s->temperature_rows, s->top_p_rows,    s->min_p_rows, s->top_k_rows};
    int bits = 0;
    while ((1 << bits) < rows.V) ++bits;
    const int shift = bits < 10 ? 52 : 62 - bits;  // at most what a 64-bit exponential holds
    if (rows.V > kSampleNarrow || (rows.V > kLgNarrow && rows.n < kSampleMany)) {
        const Wide w = wide_shape<T>(rows.n, rows.V);
        auto wide = [&](auto kernel) {
            return lg_launch_wide(who, kernel, rows.n, w, w.smem, st, w.ahead, rows, a, shift, index);
        };
        const bool by_rows = a.top_k_rows || a.top_p_rows;
        const int k = a.top_k > 0 && a.top_k < rows.V ? a.top_k : rows.V;
        if (!by_rows && k <= kLgMaxTop) return wide(lg_sample_wide_kernel<T, kPathList>);
        if (!by_rows && k == rows.V && a.top_p >= 1.0) return wide(lg_sample_wide_kernel<T, kPathPlain>);
        return wide(lg_sample_wide_kernel<T, kPathAny>);
    }
    auto narrow = [&](auto kernel, int lanes) {
        const bool direct = lanes == 1 && rows.class_stride > rows.row_stride;
        Tile t = narrow_tile(rows.n, rows.V, sizeof(T), kLgThreads / lanes);
        if (direct) t = Tile{kLgThreads, 0};
        return lg_launch(who, kernel, tiles_of(rows.n, t.rows), t.smem, st, rows, a, shift, t.rows, (int)direct, index);
    };
    if (rows.V <= 4) return narrow(lg_sample_narrow_kernel<T, 1, 4>, 1);
    if (rows.V <= 12) return narrow(lg_sample_narrow_kernel<T, 1, 12>, 1);
    if (rows.V <= 16) return narrow(lg_sample_narrow_kernel<T, 1, 16>, 1);
    if (rows.V <= 32) return narrow(lg_sample_narrow_kernel<T, 8, 4>, 8);
    if (rows.V <= 128) return narrow(lg_sample_narrow_kernel<T, 8, 16>, 8);
    if (rows.V <= kLgNarrow) return narrow(lg_sample_narrow_kernel<T, 32, 16>, 32);
    return narrow(lg_sample_narrow_kernel<T, 32, 32>, 32);
}

}  // namespace

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
    if ((rc = check_aligned("sample_classes", "uniform", s->uniform, dtype_size(s->uniform_dtype))) ||
        (rc = check_aligned("sample_classes", "index", index, 4)) ||
        (rc = check_aligned("sample_classes", "temperature_rows", s->temperature_rows, 4)) ||
        (rc = check_aligned("sample_classes", "top_p_rows", s->top_p_rows, 4)) ||
        (rc = check_aligned("sample_classes", "min_p_rows", s->min_p_rows, 4)) ||
        (rc = check_aligned("sample_classes", "top_k_rows", s->top_k_rows, 4)))
        return rc;
    return LG_BY_DTYPE(x->dtype, run_sample, x, s, index, (cudaStream_t)stream);
}
