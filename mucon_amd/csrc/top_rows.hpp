// The largest elements of a row, in order, and the row's log-sum-exp.
//
// One workgroup a row, the row in registers where it fits (read once).  Each thread's largest element gives a lower bound of the k-th largest of all without a count of the
// row: in every one of the NT / 64 waves at least j = ceil(64 k / NT) threads hold an element at least as large as the wave's j-th largest thread maximum, so at least k
// elements are at least as large as the smallest of these numbers.  The elements from the bound up are collected into an LDS list -- k to 3 k of them where the row
// is in no particular order -- and the list is sorted.  Where they do not fit it (few distinct values, k near the number of threads) the k-th largest value is found bit by bit,
// and the list holds exactly the k.  Rows with a NaN, which compares with nothing, go by their keys instead.
#pragma once
#include "row_common.hpp"

namespace rows {

constexpr int LIST = 4096;          // most entries of the LDS list: 32 KB
constexpr int SHORT_LIST = 2048;    // of workgroups of 512 and fewer: four of them share a CU

// bitonic, descending; m a power of two
template <int NT>
__device__ void sort_bitonic(u64 *list, int m) {
    for (int size = 2; size <= m; size <<= 1) {
        for (int stride = size >> 1; stride >= 1; stride >>= 1) {
            for (int t = threadIdx.x; t < (m >> 1); t += NT) {
                const int lo = ((t & ~(stride - 1)) << 1) | (t & (stride - 1));
                const int hi = lo + stride;
                const u64 a = list[lo], b = list[hi];
                const bool down = (lo & size) == 0;
                if (down ? a < b : a > b) {
                    list[lo] = b;
                    list[hi] = a;
                }
            }
            __syncthreads();
        }
    }
}

struct SortShared {
    uint32_t bin[2048];
    uint32_t w[16];
    uint32_t low, high, most;
};

// Descending, by 2,048 buckets over the range of the keys: an entry's place is its bucket's start and how many of the bucket are larger.  false: some bucket holds more
// than 64 (nothing is changed).  A bitonic sort of 2,048 entries is 66 exchanges of all of them through LDS, 25 us of a 1,024-thread workgroup; this is six passes.
template <int NT, int L>
__device__ bool sort_buckets(u64 *list, int n, SortShared &sh) {
    constexpr int E = L / NT, B = 2048 / NT;
    const int tid = threadIdx.x;
    u64 c[E];
    uint32_t low = ~0u, high = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int i = e * NT + tid;
        c[e] = i < n ? list[i] : 0;
        if (i < n) {
            low = min(low, key_of(c[e]));
            high = max(high, key_of(c[e]));
        }
    }
#pragma unroll
    for (int b = 0; b < B; ++b) sh.bin[b * NT + tid] = 0;
    if (tid == 0) {
        sh.low = ~0u;
        sh.high = sh.most = 0;
    }
    __syncthreads();
    low = wave_reduce<MinU>(low);
    high = wave_reduce<MaxU>(high);
    if ((tid & 63) == 0) {
        atomicMin(&sh.low, low);
        atomicMax(&sh.high, high);
    }
    __syncthreads();
    high = sh.high;
    const float scale = 2047.f / (float)max(high - sh.low, 1u);
    auto bucket = [&](u64 v) { return min((int)((float)(high - key_of(v)) * scale), 2047); };      // (grows as the key falls)
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (e * NT + tid < n) atomicAdd(&sh.bin[bucket(c[e])], 1u);
    __syncthreads();
    uint32_t count[B], sum = 0, most = 0;
#pragma unroll
    for (int b = 0; b < B; ++b) {
        count[b] = sh.bin[tid * B + b];
        sum += count[b];
        most = max(most, count[b]);
    }
    most = wave_reduce<MaxU>(most);
    if ((tid & 63) == 0) atomicMax(&sh.most, most);
    uint32_t all, start = block_scan<NT>(sum, sh.w, &all);
    __syncthreads();
    if (sh.most > 64) return false;
#pragma unroll
    for (int b = 0; b < B; ++b) {      // from here on: where the bucket's next entry goes
        sh.bin[tid * B + b] = start;
        start += count[b];
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (e * NT + tid < n) list[atomicAdd(&sh.bin[bucket(c[e])], 1u)] = c[e];
    __syncthreads();
    int place[E];      // now a bucket's word is its end
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (e * NT + tid >= n) continue;
        const int b = bucket(c[e]), end = (int)sh.bin[b], from = b ? (int)sh.bin[b - 1] : 0;
        int larger = 0;
        for (int i = from; i < end; ++i) larger += list[i] > c[e];
        place[e] = from + larger;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (e * NT + tid < n) list[place[e]] = c[e];
    __syncthreads();
    return true;
}

// Descending.  Up to 256 entries: each thread counts how many are larger than its own (two barriers); more: buckets; many alike: a bitonic sort, filled up with 0, which
// no composite is.
template <int NT, int L>
__device__ void sort_list(u64 *list, int n, SortShared &sh) {
    if (n <= 256 && n <= NT) {
        int width = 1;
        while (width < n) width <<= 1;
        const int parts = min(64, NT / width), i = threadIdx.x / parts, part = threadIdx.x & (parts - 1);
        const u64 c = i < n ? list[i] : ~0ull;
        int place = 0;
        for (int j = part; j < n; j += parts) place += list[j] > c;
        for (int s = 1; s < parts; s <<= 1) place += __shfl_xor(place, s);
        __syncthreads();
        if (i < n && part == 0) list[place] = c;
        __syncthreads();
        return;
    }
    if (sort_buckets<NT, L>(list, n, sh)) return;
    int m = 64;
    while (m < n) m <<= 1;
    for (int i = n + threadIdx.x; i < m; i += NT) list[i] = 0;
    __syncthreads();
    sort_bitonic<NT>(list, m);
}

// j-th largest (1-based) of the wave's 64 keys: bit by bit, counted by ballots
template <int BITS>
__device__ __forceinline__ uint32_t wave_nth(uint32_t key, int j) {
    uint32_t t = 0;
#pragma unroll
    for (int b = BITS - 1; b >= 0; --b) {
        const uint32_t mid = t | (1u << b);
        if (__popcll(__ballot(key >= mid)) >= j) t = mid;
    }
    return t;
}

template <int L>
struct SelectShared {
    u64 list[L];
    u64 u[16];
    double d[16];
    float f[16];
    uint32_t w[16];
    int n;
    SortShared sort;
};

// Elements equal to key `t` (by `is`) in index order behind the `have` that lie in the list, until it holds k
template <int TY, int NT, class IS, int L>
__device__ void add_equals(const char *row, int vocab, uint32_t t, int have, int k, SelectShared<L> &sh, IS is) {
    constexpr int N = El<TY>::N;
    const int nvec = (vocab + N - 1) / N;
    for (int base = 0; base < nvec && have < k; base += NT) {
        const int i = base + (int)threadIdx.x;
        uint32_t hits = 0;
        if (i < nvec) {
            const Vec v = load_vec<TY>(row, i, vocab);
#pragma unroll
            for (int e = 0; e < N; ++e) hits |= (uint32_t)(is(v, e) && i * N + e < vocab) << e;
        }
        uint32_t all;
        int at = have + (int)block_scan<NT>((uint32_t)__popc(hits), sh.w, &all);
        while (hits && at < k) {
            const int e = __ffs(hits) - 1;
            hits &= hits - 1;
            sh.list[at++] = composite(t, i * N + e);
        }
        have += (int)all;
    }
    __syncthreads();
}

// The first k of a row with NaN: the k-th largest key bit by bit, the larger ones, the equal ones by index
template <int TY, int NT, int L>
__device__ void select_by_keys(const char *row, int vocab, int k, SelectShared<L> &sh) {
    constexpr int N = El<TY>::N, BITS = key_bits<TY>();
    RowIn<TY, NT, 0> in(row, vocab);
    uint32_t t = 0;
    for (int b = BITS - 1; b >= 0; --b) {
        const uint32_t mid = t | (1u << b);
        uint32_t c = 0;
        in.each([&](const Vec &v, int i) {
#pragma unroll
            for (int e = 0; e < N; ++e) c += key_of<TY>(v, e) >= mid && i * N + e < vocab;
        });
        if (block_reduce<NT, Sum>(c, sh.w) >= (uint32_t)k) t = mid;
    }
    __syncthreads();
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    in.each([&](const Vec &v, int i) {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (key_of<TY>(v, e) > t && i * N + e < vocab) sh.list[atomicAdd(&sh.n, 1)] = composite(key_of<TY>(v, e), i * N + e);   // fewer than k of them
    });
    __syncthreads();
    add_equals<TY, NT>(row, vocab, t, sh.n, k, sh, [&](const Vec &v, int e) { return key_of<TY>(v, e) == t; });
}

// Puts the first k elements of the row's order (and possibly some behind them) into sh.list, sorted; returns how many lie there (>= k).  The row has no NaN;
// mine: the thread's largest element.
template <int TY, int NT, class ROW, int L>
__device__ int select_first(ROW &in, int k, float mine, SelectShared<L> &sh) {
    constexpr int N = El<TY>::N, BITS = key_bits<TY>(), NW = NT / 64;
    const int tid = threadIdx.x, vocab = in.vocab;
    float bound = -INFINITY;
    if (k <= NT && k < vocab) {
        const uint32_t nth = wave_nth<BITS>(key_of_bits<TY>(to_bits<TY>(mine)), (k + NW - 1) / NW);
        __syncthreads();
        if ((tid & 63) == 0) sh.w[tid >> 6] = nth;
        __syncthreads();
        uint32_t low = sh.w[0];
        for (int w = 1; w < NW; ++w) low = min(low, sh.w[w]);
        bound = low <= key_ninf<TY>() ? -INFINITY : value_of_key<TY>(low);
    }
    if (tid == 0) sh.n = 0;
    __syncthreads();
    in.each([&](const Vec &v, int i) {
        if (!(largest<TY>(v) >= bound)) return;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            if (value_of<TY>(v, e) >= bound && i * N + e < vocab) {
                const int at = atomicAdd(&sh.n, 1);
                if (at < L) sh.list[at] = composite(key_of<TY>(v, e), i * N + e);
            }
        }
    });
    __syncthreads();
    const int n = sh.n;
    if (n <= L) {
        sort_list<NT, L>(sh.list, n, sh.sort);
        return n;
    }
    // the k-th largest value, bit by bit of its key
    uint32_t t = 0;
    for (int b = BITS - 1; b >= 0; --b) {
        const uint32_t mid = t | (1u << b);
        bool enough = mid <= key_ninf<TY>();      // (below are the keys of NaNs, which compare with nothing)
        if (!enough) {
            const float x = value_of_key<TY>(mid);
            uint32_t c = 0;
            in.each([&](const Vec &v, int i) {
#pragma unroll
                for (int e = 0; e < N; ++e) c += value_of<TY>(v, e) >= x && i * N + e < vocab;
            });
            enough = block_reduce<NT, Sum>(c, sh.w) >= (uint32_t)k;
        }
        if (enough) t = mid;
    }
    const float x = value_of_key<TY>(t);
    __syncthreads();
    if (tid == 0) sh.n = 0;
    __syncthreads();
    in.each([&](const Vec &v, int i) {
        if (!(largest<TY>(v) > x)) return;
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (value_of<TY>(v, e) > x && i * N + e < vocab) sh.list[atomicAdd(&sh.n, 1)] = composite(key_of<TY>(v, e), i * N + e);   // fewer than k of them
    });
    __syncthreads();
    add_equals<TY, NT>(in.row, vocab, t, sh.n, k, sh, [&](const Vec &v, int e) { return value_of<TY>(v, e) == x; });
    sort_list<NT, L>(sh.list, k, sh.sort);
    return k;
}

struct TopArgs {
    const void *x;
    long long stride;
    int vocab, k;
    double temperature;
    Exponent c;
    void *values;
    int32_t *index;
    float *lse;
};

template <int TY, int NT, int NV>
__global__ __launch_bounds__(NT, NT == 512 ? 8 : 1) void top_rows_kernel(TopArgs a) {
    constexpr int L = NT > 512 ? LIST : SHORT_LIST;
    __shared__ SelectShared<L> sh;
    const long long r = blockIdx.x;
    RowIn<TY, NT, NV> in(row_at<TY>(a.x, r, a.stride), a.vocab);
    float mine = -INFINITY;
    in.each([&](const Vec &v, int) { mine = maximum(mine, largest<TY>(v)); });
    const float m = block_reduce<NT, MaxNan>(mine, sh.f);
    double s = 0.0;
    if (isfinite(m)) {
        in.each([&](const Vec &v, int) { s += weights_of<TY>(v, m, a.c); });
        s = block_reduce<NT, Sum>(s, sh.d);
    }
    if (threadIdx.x == 0) a.lse[r] = isfinite(m) ? (float)((double)m / a.temperature + log(s)) : m;
    if (isnan(m)) {
        select_by_keys<TY, NT>(in.row, a.vocab, a.k, sh);
        sort_list<NT, L>(sh.list, a.k, sh.sort);
    } else {
        select_first<TY, NT>(in, a.k, mine, sh);
    }
    typedef typename El<TY>::type T;
    for (int i = threadIdx.x; i < a.k; i += NT) {
        const int at = index_of(sh.list[i]);
        a.index[r * a.k + i] = at;
        static_cast<T *>(a.values)[r * a.k + i] = reinterpret_cast<const T *>(in.row)[at];
    }
}

// ---- few long rows: `slices` workgroups a row, then one that joins them ----
// Each slice gives its own first k (the row's first k are among them) and its part of the log-sum-exp.
constexpr int CUT = 8;      // vectors a thread holds of a slice
struct Slices {
    int count;      // of a row
    int length;     // elements of one, a multiple of 256, at most CUT vectors a thread
    int keep;       // most composites of one: LIST / count
    struct Part {
        float m;
        double s;       // (the slice kept min(k, its length) composites)
    } *part;        // [rows][count]
    u64 *kept;      // [rows][count][keep]
};

// The first k of slice `s` of row r, its largest element m and its sum of exp((x - m) / T)
template <int TY, int NT>
__device__ void cut_slice(const char *row, int vocab, long long r, int s, int k, const Exponent &c, const Slices &sl, SelectShared<LIST> &sh) {
    const int first = s * sl.length, length = min(sl.length, vocab - first);
    Slices::Part &part = sl.part[r * sl.count + s];
    RowIn<TY, NT, CUT, true> in(row + (long long)first * sizeof(typename El<TY>::type), length);
    float mine = -INFINITY;
    in.each([&](const Vec &v, int) { mine = maximum(mine, largest<TY>(v)); });
    const float m = block_reduce<NT, MaxNan>(mine, sh.f);
    double sum = 0.0;
    if (isfinite(m)) {
        in.each([&](const Vec &v, int) { sum += weights_of<TY>(v, m, c); });
        sum = block_reduce<NT, Sum>(sum, sh.d);
    }
    k = min(k, length);
    if (isnan(m))
        select_by_keys<TY, NT>(in.row, length, k, sh);
    else
        select_first<TY, NT>(in, k, mine, sh);
    for (int i = threadIdx.x; i < k; i += NT) {
        const u64 v = sh.list[i];
        sl.kept[(r * sl.count + s) * sl.keep + i] = composite(key_of(v), index_of(v) + first);
    }
    if (threadIdx.x == 0) part = Slices::Part{m, sum};
}

// The row's slices in the list, sorted; *m the row's largest element.  (What a slice kept follows from its length: no address waits for a load.)
template <int NT>
__device__ void join_slices(long long r, int vocab, int k, const Slices &sl, SelectShared<LIST> &sh, float *m) {
    const int each = min(k, sl.length), last = min(k, vocab - (sl.count - 1) * sl.length), n = (sl.count - 1) * each + last, lane = threadIdx.x & 63;
    float top = -INFINITY;
    for (int s = lane; s < sl.count; s += 64) top = maximum(top, sl.part[r * sl.count + s].m);
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += NT) sh.list[i] = sl.kept[(r * sl.count + i / each) * sl.keep + i % each];
    __syncthreads();
    sort_list<NT, LIST>(sh.list, n, sh.sort);
    *m = wave_reduce<MaxNan>(top);
}

template <int TY, int NT>
__global__ __launch_bounds__(NT) void top_cut_kernel(TopArgs a, Slices sl) {
    __shared__ SelectShared<LIST> sh;
    const long long r = blockIdx.x / sl.count;
    cut_slice<TY, NT>(row_at<TY>(a.x, r, a.stride), a.vocab, r, (int)(blockIdx.x % sl.count), a.k, a.c, sl, sh);
}
template <int TY, int NT>
__global__ __launch_bounds__(NT) void top_join_kernel(TopArgs a, Slices sl) {
    __shared__ SelectShared<LIST> sh;
    const long long r = blockIdx.x;
    float m;
    join_slices<NT>(r, a.vocab, a.k, sl, sh, &m);
    typedef typename El<TY>::type T;
    const T *row = reinterpret_cast<const T *>(row_at<TY>(a.x, r, a.stride));
    for (int i = threadIdx.x; i < a.k; i += NT) {
        const int at = index_of(sh.list[i]);
        a.index[r * a.k + i] = at;
        static_cast<T *>(a.values)[r * a.k + i] = row[at];
    }
    if (threadIdx.x < 64) {
        double s = 0.0;
        for (int i = threadIdx.x; i < sl.count; i += 64) {
            const Slices::Part p = sl.part[r * sl.count + i];
            if (p.s > 0.0) s += p.s * exp(((double)p.m - (double)m) / a.temperature);
        }
        s = wave_reduce<Sum>(s);
        if (threadIdx.x == 0) a.lse[r] = isfinite(m) ? (float)((double)m / a.temperature + log(s)) : m;
    }
}

// ---- rows of up to 256 tokens: a wave a row, four a workgroup ----
// A bitonic sort of 64 E composites in registers, E consecutive places a lane: exchanges between lanes and within one, no LDS and no barrier.
template <int E, int SIZE, int STRIDE>
__device__ __forceinline__ void exchange_held(u64 (&c)[E]) {
    const int lane = threadIdx.x & 63;
    if constexpr (STRIDE >= E) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int place = lane * E + e;
            const u64 o = lane_xor<STRIDE / E>(c[e]);
            const bool larger = ((place & STRIDE) == 0) == ((place & SIZE) == 0);
            c[e] = (c[e] > o) == larger ? c[e] : o;
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (e & STRIDE) continue;
            const bool down = ((lane * E + e) & SIZE) == 0;
            const u64 a = c[e], b = c[e | STRIDE];
            c[e] = (a > b) == down ? a : b;
            c[e | STRIDE] = (a > b) == down ? b : a;
        }
    }
    if constexpr (STRIDE > 1) exchange_held<E, SIZE, STRIDE / 2>(c);
}
template <int E, int SIZE = 2>
__device__ __forceinline__ void sort_held(u64 (&c)[E]) {
    exchange_held<E, SIZE, SIZE / 2>(c);
    if constexpr (SIZE < 64 * E) sort_held<E, SIZE * 2>(c);
}
// the row's composites in order, lane l places E l and following; 0 behind the end
template <int TY, int E>
__device__ __forceinline__ void sorted_row(const char *row, int vocab, u64 (&c)[E]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int i = e * 64 + lane;
        c[e] = i < vocab ? composite(key_of_bits<TY>(load_bits<TY>(row, i)), i) : 0;
    }
    sort_held(c);
}

template <int TY, int E>
__global__ __launch_bounds__(256) void top_small_kernel(TopArgs a, long long rows) {
    const int lane = threadIdx.x & 63;
    const long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= rows) return;
    const char *row = row_at<TY>(a.x, r, a.stride);
    u64 c[E];
    sorted_row<TY, E>(row, a.vocab, c);
    const uint32_t top = __shfl(key_of(c[0]), 0);
    const float m = value_of_key<TY>(top);
    typedef typename El<TY>::type T;
    double s = 0.0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int place = lane * E + e;
        if (place < a.k) {
            const int at = index_of(c[e]);
            a.index[r * a.k + place] = at;
            static_cast<T *>(a.values)[r * a.k + place] = reinterpret_cast<const T *>(row)[at];
        }
        if (place < a.vocab) s += (double)weight_of(value_of_key<TY>(key_of(c[e])) - m, a.c);
    }
    s = wave_reduce<Sum>(s);
    if (lane == 0) a.lse[r] = top == key_top<TY>() ? NAN : isinf(m) ? m : (float)((double)m / a.temperature + log(s));
}

}  // namespace rows
