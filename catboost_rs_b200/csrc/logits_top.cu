// logits_top.cu -- cbgpu_top_logits: a row's k largest logits and the log-sum-exp of the rest.
#include <type_traits>

#include "logits.cuh"

namespace {

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
lg_top_wide_kernel(int64_t row0, int per, int64_t ahead, Rows<T> x, int k, Scale<typename Num<T>::C> sc,
                   T* __restrict__ value, int32_t* __restrict__ index, typename Num<T>::C* __restrict__ tail) {
    typedef typename Num<T>::C C;
    typedef typename Num<T>::Key Key;
    constexpr int VE = WideRow<T>::VE;
    extern __shared__ __align__(16) unsigned char lg_smem[];
    __shared__ TopShared<Key> sh;
    __shared__ C red_max[1][kLgWarps];
    __shared__ double red[1][kLgWarps];
    __shared__ struct {
        double sum;
        C max;
    } parts[16];
    uint4* s = reinterpret_cast<uint4*>(lg_smem);
    const ClusterInfo cl;
    const int tid = threadIdx.x;
    const int64_t r = row0 + (int64_t)(blockIdx.x / (unsigned)cl.blocks);
    const WideRow<T> w(x, r, cl.rank, per);
    if (cl.blocks > 1) cluster_arrive<false>();
    if (tid == 0 && r + ahead < x.n) WideRow<T>(x, r + ahead, cl.rank, per).prefetch();
    VecMax<T> most;
    w.load(s, [&](const uint4& q) { most(q); });
    if (cl.blocks > 1) cluster_wait();  // every block runs
    int turn = 0;
    C rest;
    const int n = wide_top(cl, sh, w, s, most.get(), k, turn, rest);
    if (tail) {  // the log-sum-exp of what stayed in the row, and of the list behind its first k
        C m[1] = {rest};
        block_reduce(m, red_max, OpMax());
        const Base<C> here(floor_max(m[0]), sc);
        double sum[1] = {0.0};
        auto add = [&](auto huge) {
#pragma unroll 4
            for (int v = tid; v < w.nv; v += kLgThreads) {
                C a[VE];
                unpack(s[v], a, T());
                here.template exps<decltype(huge)::value>(a);
                sum[0] += Base<C>::total(a);
            }
        };
        if (here.huge) add(std::true_type());
        else add(std::false_type());
        block_reduce(sum, red, OpSum());
        if (tid == 0) {
            auto* to = cl.of(&parts[cl.rank], 0);
            to->max = m[0], to->sum = sum[0];
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
    C m = tid < cl.blocks ? parts[tid].max : -lg_inf(C());
    if (tid == 0 && n > k) m = OpMax()(m, of_key(sh.key[k]));
    m = warp_max(m);
    const Base<C> base(floor_max(m), sc);
    double sum = 0.0;
    if (tid < cl.blocks && parts[tid].sum != 0.0)
        sum = parts[tid].sum * exp(Base<C>(floor_max(parts[tid].max), sc).ln_shift(base));
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
    if (rows.V > kLgNarrow) {
        const Wide w = wide_shape<T>(rows.n, rows.V);
        return lg_launch_wide(who, lg_top_wide_kernel<T>, rows.n, w, w.smem, st, w.ahead, rows, k, sc, (T*)value, index,
                              (C*)tail);
    }
    auto narrow = [&](auto kernel, int lanes) {
        const Tile t = narrow_tile(rows.V, sizeof(T), kLgThreads / lanes, rows.class_stride <= rows.row_stride);
        return lg_launch(who, kernel, tiles_of(rows.n, t.rows), t.smem, st, rows, k, sc, t.rows, t.pitch, (T*)value,
                         index, (C*)tail);
    };
    return by_lanes(rows.V, [&] { return narrow(lg_top_narrow_kernel<T, 1>, 1); },
                    [&] { return narrow(lg_top_narrow_kernel<T, 8>, 8); },
                    [&] { return narrow(lg_top_narrow_kernel<T, 32>, 32); });
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
    if (x->n == 0) return CBGPU_OK;
    return LG_BY_DTYPE(x->dtype, run_top, x, k, temperature, value, index, tail, (cudaStream_t)stream);
}

