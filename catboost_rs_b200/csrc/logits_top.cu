// logits_top.cu -- cbgpu_top_logits: a row's k largest logits and the log-sum-exp of the rest.
#include <type_traits>

#include "logits.cuh"

namespace {

// Narrow rows.  A lane's classes are keys in registers (0: none, or taken; 1: NaN).
// Up to kRounds of them are taken one by one, each lane offering its best;
// above that (a warp a row) the k-th key is found bit by bit, and the keys
// from it on are listed and sorted.
constexpr int kRounds = 16;

template <typename Key>
struct TopList {
    Key key[kLgMaxTop];
    uint32_t idx[kLgMaxTop];
};

template <typename Key>
__device__ void warp_sort(TopList<Key>& l, int n) {
    const int lane = threadIdx.x & 31;
    int size = 1;
    while (size < n) size *= 2;
    for (int i = n + lane; i < size; i += 32) l.key[i] = 0, l.idx[i] = 0xffffffffu;
    __syncwarp();
    for (int len = 2; len <= size; len *= 2)
        for (int d = len / 2; d > 0; d /= 2) {
            for (int p = lane; p < size / 2; p += 32) {
                const int i = (p & (d - 1)) | ((p & ~(d - 1)) << 1), j = i | d;
                const Ranked<Key> a{l.key[i], l.idx[i]}, b{l.key[j], l.idx[j]};
                if ((i & len) == 0 ? b.before(a) : a.before(b))
                    l.key[i] = b.key, l.idx[i] = b.idx, l.key[j] = a.key, l.idx[j] = a.idx;
            }
            __syncwarp();
        }
}

template <typename T, int G, int ITEMS>
__global__ void __launch_bounds__(kLgThreads)
lg_top_narrow_kernel(Rows<T> x, int k, Scale<typename Num<T>::C> sc, int tile, T* __restrict__ value,
                     int32_t* __restrict__ index, typename Num<T>::C* __restrict__ tail) {
    typedef typename Num<T>::C C;
    typedef typename Num<T>::Key Key;
    constexpr int kBits = (int)sizeof(Key) * 8 - Num<T>::kKeyDrop;
    constexpr bool kLists = G == 32;
    extern __shared__ __align__(16) unsigned char lg_smem[];
    __shared__ TopList<Key> lists[kLists ? kLgWarps : 1];
    const int64_t r0 = (int64_t)blockIdx.x * tile;
    const int rows = (int)(x.n - r0 < tile ? x.n - r0 : tile), V = x.V;
    T* g = const_cast<T*>(x.data) + r0 * x.row_stride;
    const TileIo<T> io(g, x.row_stride, x.class_stride, V, rows);
    T* s = reinterpret_cast<T*>(lg_smem) + io.shift;
    io.template copy<false>(s, g);
    __syncthreads();
    const LaneTeam<G> t;
    const Items<G, ITEMS> mine(t, V);
    for (int r = threadIdx.x / G; r < rows; r += kLgThreads / G) {
        const T* row = s + (size_t)r * io.pitch;
        T* val = value + (r0 + r) * k;
        int32_t* idx = index + (r0 + r) * k;
        Key key[ITEMS] = {};
        LG_EACH(it)
            key[it] = mine.has(it) ? (key_of(to_c(row[mine.first + it])) >> Num<T>::kKeyDrop) + 1 : 0;
        bool nan = false;  // among the first k
        if (!kLists || k <= kRounds) {
            Key best = 0;
            int at = 0;
            auto look = [&] {
                best = 0;
                LG_EACH(it) best = key[it] > best ? key[it] : best;
                at = 0;
#pragma unroll
                for (int it = ITEMS - 1; it >= 0; --it)
                    at = key[it] == best ? it : at;
            };
            look();
            for (int j = 0; j < k; ++j) {
                const Key top = t.reduce(best, OpMax());
                const int i = t.reduce(best == top ? mine.first + at : 0x7fffffff, OpMin());
                nan = top == 1;
                if (best == top && i == mine.first + at) {
                    val[j] = row[i];
                    idx[j] = i;
                    LG_EACH(it) key[it] = it == at ? 0 : key[it];
                    look();
                }
            }
        } else {
            TopList<Key>& list = lists[kLists ? threadIdx.x >> 5 : 0];
            // the bits that all keys share come first
            Key most = 0, least = ~(Key)0;
            LG_EACH(it) if (mine.has(it)) most = key[it] > most ? key[it] : most, least = key[it] < least ? key[it] : least;
            most = t.reduce(most, OpMax()), least = t.reduce(least, OpMin());
            const int bits = most == least ? 0 : 64 - __clzll((long long)(u64)(most ^ least));
            Key bound = bits < kBits ? most >> bits << bits : 0;
            int above = 0;
            bool exact = false;
            for (int b = bits - 1; b >= 0 && !exact; --b) {
                const Key cand = bound | ((Key)1 << b);
                int n = 0;
                LG_EACH(it) n += key[it] >= cand;
                n = team_count(t, n);
                if (n >= k) bound = cand;
                exact = n == k;
            }
            int own = 0, ties = 0;
            LG_EACH(it) own += key[it] > bound, ties += key[it] == bound;
            above = team_count(t, own);
            // of equal keys the lower indices: the lanes' classes are in the order of the lanes
            int spare = k - above - (int)t.exscan((u64)ties);
            spare = spare < 0 ? 0 : (spare < ties ? spare : ties);
            int to = (int)t.exscan((u64)(own + spare));
            LG_EACH(it) {
                const bool take = key[it] > bound || (key[it] == bound && spare > 0);
                if (take && key[it] == bound) --spare;
                if (take) {
                    list.key[to] = key[it], list.idx[to] = (uint32_t)(mine.first + it);
                    ++to;
                    key[it] = 0;
                }
            }
            __syncwarp();
            warp_sort(list, k);
            for (int j = t.rank; j < k; j += G) {
                const int i = (int)list.idx[j];
                val[j] = row[i];
                idx[j] = i;
            }
            nan = list.key[k - 1] == 1;
            __syncwarp();
        }
        if (!tail) continue;
        C m = -lg_inf(C());
        LG_EACH(it)
            if (key[it] != 0) m = OpMax()(m, to_c(row[mine.first + it]));
        m = floor_max(t.reduce(m, OpMax()));
        C part = 0;
        LG_EACH(it)
            if (key[it] != 0) part += lg_exp(to_c(row[mine.first + it]) - m, sc.c);
        const double sum = t.reduce((double)part, OpSum());
        if (t.rank == 0) {
            const double none = sum == 0.0 ? -lg_inf(0.0) : log(sum) + (double)m * sc.inv_t;
            tail[r0 + r] = (C)(nan ? lg_inf(0.0) - lg_inf(0.0) : none);
        }
    }
}

// Many rows of up to kThreadMost classes and a small k: a thread a row, which keeps the first LIST
// classes in order in registers (a class sinks through them; of equal ones the earlier stays ahead) and
// adds what falls out to the tail, relative to the last of the list.  No shuffles and no second look
// (200000 x 100 f32, k 8: 127 us with 8 lanes a row).  The rows are read by 16 bytes where they lie to
// it; a warp's 32 rows share no lines, but the lines stay in L1 until they are used up.
constexpr int kThreadMost = 128;
constexpr int kTopThreads = 64;  // small blocks: the last of them leave less of an SM idle

template <typename T, int LIST>
__global__ void __launch_bounds__(kTopThreads)
lg_top_thread_kernel(Rows<T> x, int k, Scale<float> sc, int by16, T* __restrict__ value, int32_t* __restrict__ index,
                     float* __restrict__ tail) {
    const int64_t r = blockIdx.x * (int64_t)kTopThreads + threadIdx.x;
    if (r >= x.n) return;
    const T* row = x.data + r * x.row_stride;
    uint32_t key[LIST];
    int idx[LIST];
#pragma unroll
    for (int j = 0; j < LIST; ++j) key[j] = 0, idx[j] = 0x7fffffff;  // keys are one more, as NaN is 0
    float sum = 0.0f, last = 0.0f;  // `last`: the logit that sum is relative to
    bool nan = false;
    auto add = [&](float v, int i) {
        nan |= v != v;
        const uint32_t own = key_of(v) + 1, end = key[LIST - 1];
        uint32_t c = own;
        int ci = i;
#pragma unroll
        for (int j = 0; j < LIST; ++j) {  // from its place on all move down by one
            const bool up = own > key[j];
            const uint32_t t = key[j];
            const int ti = idx[j];
            key[j] = up ? c : t, idx[j] = up ? ci : ti;
            c = up ? t : c, ci = up ? ti : ci;
        }
        if (tail && c != 0) {  // a class fell out: the list is full
            const float now = of_key(key[LIST - 1] - 1);
            if (end != key[LIST - 1]) sum *= ex2((last - now) * sc.c);
            last = now;
            sum += now == -lg_inf(0.0f) ? 0.0f : ex2((of_key(c - 1) - now) * sc.c);
        }
    };
    int i = 0;
    if (by16) {
        constexpr int VE = 16 / (int)sizeof(T);
        for (; i + VE <= x.V; i += VE) {
            float a[VE];
            unpack(*reinterpret_cast<const uint4*>(row + i), a, T());
#pragma unroll
            for (int j = 0; j < VE; ++j) add(a[j], i + j);
        }
    }
    for (; i < x.V; ++i) add(to_c(row[(int64_t)i * x.class_stride]), i);
    float m = -lg_inf(0.0f);
#pragma unroll
    for (int j = 0; j < LIST; ++j) {
        if (j < k) {
            value[r * k + j] = row[(int64_t)idx[j] * x.class_stride];
            index[r * k + j] = idx[j];
        } else if (key[j] > 1 && m == -lg_inf(0.0f)) {
            m = of_key(key[j] - 1);  // the largest of the rest
        }
    }
    if (!tail) return;
    double rest = 0.0;
    if (m != -lg_inf(0.0f)) {
        rest = sum > 0.0f ? (double)sum * (double)ex2((last - m) * sc.c) : 0.0;
#pragma unroll
        for (int j = 0; j < LIST; ++j)
            if (j >= k && key[j] > 1) rest += (double)ex2((of_key(key[j] - 1) - m) * sc.c);
    }
    const double none = rest == 0.0 ? -lg_inf(0.0) : log(rest) + (double)m * sc.inv_t;
    tail[r] = (float)(nan ? lg_inf(0.0) - lg_inf(0.0) : none);
}

template <typename T>
__global__ void __launch_bounds__(kLgThreads)
lg_top_wide_kernel(int64_t row0, int per, int64_t ahead, Rows<T> x, int k, Scale<typename Num<T>::C> sc,
                   T* __restrict__ value, int32_t* __restrict__ index, typename Num<T>::C* __restrict__ tail) {
    typedef typename Num<T>::C C;
    typedef typename Num<T>::Key Key;
    constexpr int VE = WideRow<T>::VE;
    extern __shared__ __align__(16) unsigned char lg_smem[];
    __shared__ TopShared<Key> sh;
    __shared__ C red_max[kLgWarps];
    __shared__ double red[kLgWarps];
    __shared__ struct {
        double sum;
        C max;
    } parts[16];
    uint4* s = reinterpret_cast<uint4*>(lg_smem);
    const ClusterInfo cl;
    const int tid = threadIdx.x, lane = tid & 31, warp_id = tid >> 5;
    const int64_t r = row0 + (int64_t)(blockIdx.x / (unsigned)cl.blocks);
    const WideRow<T> w(x, r, cl.rank, per);
    if (cl.blocks > 1) cluster_arrive<false>();
    if (tid == 0 && r + ahead < x.n) WideRow<T>(x, r + ahead, cl.rank, per).prefetch();
    VecMax<T> most;
    w.load(s, [&](const uint4& q) { most(q); });
    if (cl.blocks > 1) cluster_wait();  // every block runs
    int turn = 0;
    C rest, ref = C(0);
    bool exact, flag = false;
    double sum = 0.0;
    // the tail's sum is taken on the way, relative to the least class that is collected
    const int n = wide_top(cl, sh, w, s, most.get(), k, turn, rest, exact, flag, [&](C(&a)[VE], C least) {
        if (!tail) return;
        ref = floor_max(least);
        const Base<C> at(ref, sc);
        if (at.huge) at.template exps<true>(a);
        else at.template exps<false>(a);
        sum += Base<C>::total(a);
    });
    if (tail) {
        sum = warp_sum(sum, 32);
        rest = warp_max(rest);
        if (lane == 0) red[warp_id] = sum, red_max[warp_id] = rest;
        __syncthreads();
        sum = red[0], rest = red_max[0];
#pragma unroll
        for (int i = 1; i < kLgWarps; ++i) sum += red[i], rest = OpMax()(rest, red_max[i]);
        if (exact || (sum < 1e-20 && rest > -lg_inf(C()))) {  // the rest lies far below: relative to its own largest
            __syncthreads();
            ref = floor_max(rest);
            const Base<C> at(ref, sc);
            double part = 0.0;
            for (int v = tid; v < w.nv; v += kLgThreads) {
                C a[VE];
                unpack(s[v], a, T());
                if (at.huge) at.template exps<true>(a);
                else at.template exps<false>(a);
                part += Base<C>::total(a);
            }
            part = warp_sum(part, 32);
            if (lane == 0) red[warp_id] = part;
            __syncthreads();
            sum = red[0];
            for (int i = 1; i < kLgWarps; ++i) sum += red[i];
        }
        if (tid == 0) {
            auto* to = cl.of(&parts[cl.rank], 0);
            to->max = ref, to->sum = sum;
        }
    }
    if (cl.blocks > 1) cl.sync();  // also: no block leaves while another reads its shared memory
    if (cl.rank != 0) return;
    __syncthreads();
    sort_list(sh, n);
    for (int j = tid; j < k; j += kLgThreads) {
        value[r * k + j] = from_c<T>(of_key(sh.key[j]));
        index[r * k + j] = (int32_t)sh.idx[j];
    }
    if (!tail || tid >= 32) return;
    // only parts that hold something have a say in the base; the list behind its first k is below it
    const bool has = tid < cl.blocks && parts[tid].sum != 0.0;
    C m = has ? parts[tid].max : -lg_inf(C());
    if (tid == 0 && n > k) m = OpMax()(m, of_key(sh.key[k]));
    m = warp_max(m);
    const Base<C> base(floor_max(m), sc);
    sum = has ? parts[tid].sum * exp(Base<C>(parts[tid].max, sc).ln_shift(base)) : 0.0;
    for (int j = k + tid; j < n; j += 32) sum += (double)base.exp(of_key(sh.key[j]));
    sum = warp_sum(sum, 32);
    if (tid == 0) {
        const double nan = (double)lg_inf(C()) - (double)lg_inf(C());
        // ln sum + the logarithm of the base's 1; a NaN among the first k (its key is 0) counts as one anywhere
        tail[r] = sh.key[k - 1] == 0 ? (C)nan : (C)(sum == 0.0 ? -lg_inf(0.0) : log(sum) - base.ln(C(0)));
    }
}

template <typename T>
int run_top(const cbgpu_logits* x, int k, double temp, void* value, int32_t* index, void* tail, cudaStream_t st) {
    typedef typename Num<T>::C C;
    const char* who = "top_logits";
    const Rows<T> rows = rows_of<T>(x);
    const Scale<C> sc(temp);
    if (is_wide(rows.n, rows.V)) {
        const Wide w = wide_shape<T>(rows.n, rows.V);
        return lg_launch_wide(who, lg_top_wide_kernel<T>, rows.n, w, w.smem, st, w.ahead, rows, k, sc, (T*)value, index,
                              (C*)tail);
    }
    auto narrow = [&](auto kernel, int lanes) {
        const Tile t = narrow_tile(rows.n, rows.V, sizeof(T), kLgThreads / lanes);
        return lg_launch(who, kernel, tiles_of(rows.n, t.rows), t.smem, st, rows, k, sc, t.rows, (T*)value, index,
                         (C*)tail);
    };
    if constexpr (sizeof(C) == 4) {
        // enough rows that a thread a row fills the SMs, and enough classes that the list is worth it
        if (rows.V > 16 && rows.V <= kThreadMost && k <= 8 && rows.n >= 148 * kLgThreads) {
            const int by16 = rows.class_stride == 1 && ((uintptr_t)rows.data & 15) == 0 &&
                             (rows.row_stride * sizeof(T)) % 16 == 0;
            auto threads = [&](auto kernel) {
                return lg_launch_n(who, kernel, tiles_of(rows.n, kTopThreads), kTopThreads, 0, st, rows, k, sc, by16,
                                   (T*)value, index, (C*)tail);
            };
            if (k == 1) return threads(lg_top_thread_kernel<T, 2>);
            return k <= 4 ? threads(lg_top_thread_kernel<T, 5>) : threads(lg_top_thread_kernel<T, 9>);
        }
    }
    if (rows.V <= 4) return narrow(lg_top_narrow_kernel<T, 1, 4>, 1);
    if (rows.V <= 12) return narrow(lg_top_narrow_kernel<T, 1, 12>, 1);
    if (rows.V <= 16) return narrow(lg_top_narrow_kernel<T, 1, 16>, 1);
    if (rows.V <= 32 && k <= kRounds) return narrow(lg_top_narrow_kernel<T, 8, 4>, 8);
    if (rows.V <= 128 && k <= kRounds) return narrow(lg_top_narrow_kernel<T, 8, 16>, 8);
    if (rows.V <= 128) return narrow(lg_top_narrow_kernel<T, 32, 4>, 32);
    return narrow(lg_top_narrow_kernel<T, 32, 16>, 32);
}

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
    const size_t wide = x->dtype == CBGPU_F64 ? 8 : 4;
    if ((rc = check_aligned("top_logits", "value", value, dtype_size(x->dtype))) ||
        (rc = check_aligned("top_logits", "index", index, 4)) || (rc = check_aligned("top_logits", "tail", tail, wide)))
        return rc;
    if (x->n == 0) return CBGPU_OK;
    return LG_BY_DTYPE(x->dtype, run_top, x, k, temperature, value, index, tail, (cudaStream_t)stream);
}

