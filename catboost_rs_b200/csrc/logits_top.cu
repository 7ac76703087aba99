// logits_top.cu -- cbgpu_top_logits: a row's k largest logits and the log-sum-exp of the rest.
#include <type_traits>

#include "logits.cuh"

namespace {

// Narrow rows.  A lane's classes are keys in registers (0: none, or taken; 1: NaN).
// Up to kRounds of them are taken one by one, each lane offering its best;
// above that (a warp a row) the k-th key is found bit by bit, and the keys
// from it on are listed and sorted.  Bound by issue and shuffles (20000 x 512 f32, k 16: 100 us; a block
// a row 180).
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
            const double none = sum == 0.0 ? -lg_inf(0.0) : log(sum) + (double)m * sc.by_t;
            tail[r0 + r] = (C)(nan ? lg_inf(0.0) - lg_inf(0.0) : none);
        }
    }
}

// Many rows of up to kThreadMost classes and a small k: a thread a row, without shuffles, from a stage in
// shared memory that each warp fills by asynchronous copies.  The LIST largest logits are found first,
// without their classes: eight at a time go through a sorting network (Batcher 1968) and a bitonic merge
// with the list, 9 minima and maxima a class for a list of 8.  The row is read once more for the classes
// at or above the k-th (bits, one a class) and the others' sum.  A row with a NaN, which shows in that
// sum, is gone through k times instead.  Bound by issue and the copies, which blocks overlap: 200000 x
// 100 f32, k 8: 41 us, where 8 lanes a row take 129; read from global memory instead of a stage 68,
// and with keys and classes that sink through a list of 9, five selections a place, 92.  There is no list above 8
// and none of 64-bit logits: k 9 takes 137 us by 8 lanes a row, k 16 203, and 200000 x 32 f64, k 8, 94.
constexpr int kThreadMost = 128;
constexpr int kTopThreads = 64;  // small blocks: the last of them leave less of an SM idle

// Elements a row of the stage takes: whole eights, an odd number of 16-byte vectors, so that eight threads'
// vectors of one place lie in all the banks.
template <typename T>
__host__ __device__ int top_pitch(int V) {
    constexpr int VE = 16 / (int)sizeof(T);
    return ((V + 7) / 8 * 8 / VE | 1) * VE;
}

__device__ __forceinline__ void in_order(float& a, float& b) {
    const float hi = fmaxf(a, b), lo = fminf(a, b);
    a = hi, b = lo;
}
template <int LIST>
struct Firsts {  // the LIST largest, in order
    float of[LIST];
    __device__ Firsts() {
#pragma unroll
        for (int j = 0; j < LIST; ++j) of[j] = -lg_inf(0.0f);
    }
    __device__ void merge(const float* b) {  // with LIST more, in order
#pragma unroll
        for (int j = 0; j < LIST; ++j) of[j] = fmaxf(of[j], b[LIST - 1 - j]);
#pragma unroll
        for (int d = LIST / 2; d > 0; d /= 2)
#pragma unroll
            for (int j = 0; j < LIST; ++j)
                if ((j & d) == 0) in_order(of[j], of[j + d]);
    }
    __device__ void add(float (&a)[8]) {
        if constexpr (LIST == 1) {
#pragma unroll
            for (int j = 0; j < 8; ++j) of[0] = fmaxf(of[0], a[j]);
        } else {
#pragma unroll
            for (int h = 0; h < 8; h += 4) {
                in_order(a[h], a[h + 1]), in_order(a[h + 2], a[h + 3]);
                in_order(a[h], a[h + 2]), in_order(a[h + 1], a[h + 3]);
                in_order(a[h + 1], a[h + 2]);
            }
            if constexpr (LIST == 8) {
#pragma unroll
                for (int j = 0; j < 4; ++j) in_order(a[j], a[j + 4]);
                in_order(a[2], a[4]), in_order(a[3], a[5]);
                in_order(a[1], a[2]), in_order(a[3], a[4]), in_order(a[5], a[6]);
            } else {
                merge(a + 4);
            }
            merge(a);
        }
    }
};

// A warp's rows to its stage by BYTES at a time, all under way at once.
template <int BYTES, typename T>
__device__ __forceinline__ void copy_rows(T* stage, int pitch, const T* from, int64_t stride, int rows, int V) {
    constexpr int PER = BYTES / (int)sizeof(T);
    const int lane = threadIdx.x & 31, whole = V / PER;
    for (int o = 0; o < rows; ++o)
        for (int c = lane; c < whole; c += 32) {
            const uint32_t to = (uint32_t)__cvta_generic_to_shared(stage + (size_t)o * pitch + c * PER);
            const T* g = from + o * stride + c * PER;
            if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(g) : "memory");
            else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(g), "n"(BYTES) : "memory");
        }
    if (lane < rows)
        for (int i = whole * PER; i < V; ++i) stage[(size_t)lane * pitch + i] = from[lane * stride + i];
}

template <typename T, int LIST>
__global__ void __launch_bounds__(kTopThreads)
lg_top_thread_kernel(Rows<T> x, int k, Scale<float> sc, int unit, T* __restrict__ value, int32_t* __restrict__ index,
                     float* __restrict__ tail) {
    constexpr int VE = 16 / (int)sizeof(T), kWords = kThreadMost / 32;
    extern __shared__ __align__(16) unsigned char lg_smem[];
    const int V = x.V, lane = threadIdx.x & 31;
    const int64_t r0 = blockIdx.x * (int64_t)kTopThreads + (threadIdx.x & ~31u), r = r0 + lane;
    if (r0 >= x.n) return;
    const int rows = (int)(x.n - r0 < 32 ? x.n - r0 : 32);
    // a warp stages its rows
    const int pitch = top_pitch<T>(V);
    T* stage = reinterpret_cast<T*>(lg_smem) + (size_t)(threadIdx.x & ~31u) * pitch;
    T* row = stage + (size_t)lane * pitch;
    const T* from = x.data + r0 * x.row_stride;
    if (unit >= 4) {
        if (unit == 16) copy_rows<16>(stage, pitch, from, x.row_stride, rows, V);
        else if (unit == 8) copy_rows<8>(stage, pitch, from, x.row_stride, rows, V);
        else copy_rows<4>(stage, pitch, from, x.row_stride, rows, V);
        asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
    } else if (x.class_stride > x.row_stride) {  // neighbours in memory are rows
        for (int i = 0; lane < rows && i < V; i += 8) {
            T v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (i + j < V) v[j] = from[lane * x.row_stride + (i + j) * x.class_stride];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (i + j < V) row[i + j] = v[j];
        }
    } else {
        for (int o = 0; o < rows; o += 8)
            for (int i = lane; i < V; i += 32) {
                T v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (o + j < rows) v[j] = from[(o + j) * x.row_stride + i * x.class_stride];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (o + j < rows) stage[(size_t)(o + j) * pitch + i] = v[j];
            }
    }
    for (int i = V; i < (V + 7) / 8 * 8; ++i) row[i] = from_c<T>(-lg_inf(0.0f));
    __syncwarp();
    if (lane >= rows) return;
    auto logit = [&](int i) { return to_c(row[i]); };
    auto eight = [&](int i, float(&a)[8]) {  // classes from i on; -inf behind the last
#pragma unroll
        for (int h = 0; h < 8; h += VE) {
            float part[VE];
            unpack(*reinterpret_cast<const uint4*>(row + i + h), part, T());
#pragma unroll
            for (int j = 0; j < VE; ++j) a[h + j] = part[j];
        }
    };
    Firsts<LIST> first;
    for (int i = 0; i < V; i += 8) {
        float a[8];
        eight(i, a);
        first.add(a);
    }
    float last = first.of[0];  // the k-th
#pragma unroll
    for (int j = 1; j < LIST; ++j) last = j < k ? first.of[j] : last;
    uint32_t in[kWords];  // the classes at or above it
    double sum = 0.0;     // of the others, relative to it
    int spare = -k;       // of those equal to it, the last ones are not among the first k
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
        in[w] = 0;
        for (int i = w * 32; i < w * 32 + 32 && i < V; i += 8) {
            float a[8];
            eight(i, a);
            uint32_t bits = 0;
            float part[2] = {0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float e = ex2((a[j] - last) * sc.c);
                if (a[j] >= last) bits |= 1u << j;
                else part[j & 1] += e;
            }
            bits = i + 8 <= V ? bits : bits & ((1u << (V - i)) - 1u);  // none behind the last class
            in[w] |= bits << (i - w * 32);
            sum += (double)(part[0] + part[1]);
        }
        spare += __popc(in[w]);
    }
    const double nan = (double)(lg_inf(0.0f) - lg_inf(0.0f));
    if (sum != sum) {
        uint32_t key = 0xffffffffu;  // above all keys
        int at = -1;
        for (int j = 0; j < k; ++j) {
            uint32_t best = 0;
            int next = -1;
            for (int i = 0; i < V; ++i) {
                const uint32_t c = key_of(logit(i));
                if ((c < key || (c == key && i > at)) && (next < 0 || c > best)) best = c, next = i;
            }
            key = best, at = next;
            value[r * k + j] = row[at];
            index[r * k + j] = at;
        }
        if (tail) tail[r] = (float)nan;
        return;
    }
    const int ties = spare;
#pragma unroll
    for (int w = kWords - 1; w >= 0; --w)
        for (uint32_t look = in[w]; spare > 0 && look != 0;) {
            const int b = 31 - __clz((int)look);
            look ^= 1u << b;
            if (logit(w * 32 + b) == last) in[w] ^= 1u << b, --spare;
        }
    uint32_t used = 0;  // places that are taken: of equal logits the lower class comes first
#pragma unroll
    for (int j = 0; j < LIST; ++j) {
        if (j >= k) break;
        int i = 0;
        bool got = false;
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
            if (!got && in[w] != 0) i = w * 32 + __ffs((int)in[w]) - 1, in[w] &= in[w] - 1u, got = true;
        }
        const T v = row[i];
        int to = 0;
#pragma unroll
        for (int o = 0; o < LIST - 1; ++o) to += first.of[o] > to_c(v) ? 1 : 0;
        to += __ffs((int)~(used >> to)) - 1;
        used |= 1u << to;
        value[r * k + to] = v;
        index[r * k + to] = i;
    }
    if (!tail) return;
    if (ties > 0 && last != -lg_inf(0.0f)) sum += (double)ties;
    float base = last;
    if (sum < 1e-20) {  // the others lie far below (or are masked): relative to the largest of them
        base = -lg_inf(0.0f);
        for (int i = 0; i < V; ++i) {
            const float v = logit(i);
            base = v < last ? fmaxf(base, v) : base;
        }
        sum = 0.0;
        if (base != -lg_inf(0.0f))
            for (int i = 0; i < V; ++i) {
                const float v = logit(i);
                sum += v < last ? (double)ex2((v - base) * sc.c) : 0.0;
            }
    }
    const double none = sum == 0.0 ? -lg_inf(0.0) : log(sum) + (double)base * sc.by_t;
    tail[r] = (float)(ties > 0 && last == lg_inf(0.0f) ? nan : none);
}

// Wide rows: the maxima that the threads keep while they copy their part give a bound that a few more
// than k classes reach (logits.cuh, wide_top); those go to the first block, which sorts them, and the tail's
// sum is taken in the same second look.  2048 x 64000 bf16, k 64: 138 us (floor 41), with the
// exponentials' pipe 29 % busy and 41 % of the issue slots; the rest is a block's chain of copy, bound,
// collection, hand-over and sort with their barriers.  8 x 131071 f32, k 128: 12 us on the device.
// kBlocks: what an SM holds at least.  Five, of 48 registers, for rows of up to 16 KB (20000 x 700 f32, k 16: 184 us
// against 207 with 62 registers; bf16 203 against 225); above, where shared memory leaves three, registers count
// (512 x 131072 f32: 131 us against 143; 2048 x 64000 bf16 143 against 147).
template <typename T, int kBlocks>
__global__ void __launch_bounds__(kLgThreads, kBlocks)
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
    w.template load<kLgThreads, kBlocks == 5 && sizeof(T) == 4 ? 4 : 8>(s, [&](const uint4& q) { most(q); });
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
        at.exps(a);
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
                at.exps(a);
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
        // ln sum + the base's logit scaled; a NaN among the first k (its key is 0) counts as one anywhere
        tail[r] = sh.key[k - 1] == 0 ? (C)nan : (C)(sum == 0.0 ? -lg_inf(0.0) : log(sum) + (double)base.m * sc.by_t);
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
        auto wide = [&](auto kernel) {
            return lg_launch_wide(who, kernel, rows.n, w, w.smem, st, w.ahead, rows, k, sc, (T*)value, index, (C*)tail);
        };
        if constexpr (sizeof(T) < 8)
            if (w.smem <= 16384) return wide(lg_top_wide_kernel<T, 5>);
        return wide(lg_top_wide_kernel<T, 4>);
    }
    auto narrow = [&](auto kernel, int lanes) {
        const Tile t = narrow_tile(rows.n, rows.V, sizeof(T), kLgThreads / lanes);
        return lg_launch(who, kernel, tiles_of(rows.n, t.rows), t.smem, st, rows, k, sc, t.rows, (T*)value, index,
                         (C*)tail);
    };
    if constexpr (sizeof(C) == 4) {
        // a block an SM or more (9600 rows of 100, k 8: 14 us against 18 with 8 lanes a row; 4800: the same)
        if (rows.V > 16 && rows.V <= kThreadMost && k <= 8 && rows.n >= 148 * kTopThreads) {
            // the bytes that rows are copied by: what their starts have in common
            int unit = 16;
            const uintptr_t starts = (uintptr_t)rows.data | (uintptr_t)(rows.row_stride * (int64_t)sizeof(T));
            while (starts % (uintptr_t)unit != 0) unit /= 2;
            if (rows.class_stride != 1) unit = 0;
            auto threads = [&](auto kernel) {
                const size_t smem = (size_t)kTopThreads * top_pitch<T>(rows.V) * sizeof(T);
                return lg_launch_n(who, kernel, tiles_of(rows.n, kTopThreads), kTopThreads, smem, st, rows, k, sc, unit,
                                   (T*)value, index, (C*)tail);
            };
            if (k == 1) return threads(lg_top_thread_kernel<T, 1>);
            return k <= 4 ? threads(lg_top_thread_kernel<T, 4>) : threads(lg_top_thread_kernel<T, 8>);
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

