// logits_sample.cu -- cbgpu_sample_classes: a class drawn from a row under temperature / top-k / top-p / min-p.
#include "logits.cuh"

namespace {

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
    return LG_BY_DTYPE(x->dtype, run_sample, x, s, index, (cudaStream_t)stream);
}
