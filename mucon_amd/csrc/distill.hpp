// The distillation loss of a student's rows on a teacher's top logits, and its gradient.
//
// Per row, T the temperature, a_k = t_k / T the listed teacher logits, q = softmax(s / T) the student:
//   p_k = softmax over the listed (no teacher log-sum-exp given), or exp(a_k - lse) with the rest p_r = max(0, 1 - sum p_k) on the tokens that are not listed, together;
//   L   = T^2 [ sum_k p_k (log p_k - log q_k) + p_r (log p_r - log q_r) ],   q_r = sum of q over the tokens that are not listed;
//   dL / ds_j = T [ q_j (P - [j not listed] p_r / q_r) - sum_{k: i_k = j} p_k ],   P = sum p_k + p_r.
// With a rest, the unlisted tokens (those whose bit is not set in an LDS bitmap) are summed against their own maximum m_o and the listed ones against theirs: q_r is never
// taken as 1 - sum q_k, which cancels, and is as good where it is e^-1000 of the row, as where a student is certain of what its teacher doubts.  Their part of the gradient,
//   T exp((s_j - m_o) / T) [P exp((m_o - m) / T) / Z - p_r / Zo],   Z the row's sum against its maximum m, Zo = sum_unlisted exp((s - m_o) / T) >= 1,
// has no large factor.  Only where no unlisted token is above -inf is there no rest term.  Sums over the vocabulary and the logarithms of the listed entries, which are
// subtracted from each other, are held in 64 bits, as are the gradient's factors and its listed tokens; the exponentials of a row are fp32 (row_common.hpp, weight_of).
#pragma once
#include "row_common.hpp"
#include "top_rows.hpp"

namespace rows {

struct DistillRow {   // what the gradient of a row needs
    double in, out;   // dL / ds_j = T in exp((s_j - m) / T) - T p for the listed tokens, T out exp((s_j - mo) / T) for the others
    double lp0;       // log p_k = (t_k - t0) / T - lp0
    float t0;         // the largest listed logit (with a rest: 0)
    float m, mo;      // the row's maximum, that of the unlisted tokens (no rest: the row's)
};

struct DistillArgs {
    const void *s;
    long long stride;
    const void *t;            // [rows][k], of type `tt`
    const int32_t *index;     // [rows][k]
    const float *lse;         // [rows], or NULL: the listed entries are all
    const float *weight;      // [rows], or NULL
    int vocab, k;
    int tt;
    double temperature, it;   // it: 1 / temperature
    Exponent c;
    float *losses;            // [rows]: weight * L
    DistillRow *stat;         // [rows]
    // backward
    void *grad;
    const float *upstream;    // [rows] (each) or [1]; NULL: 1
    int each;
    const double *norm;       // 1 / sum of the weights (mean), or NULL: `scale` alone
    double scale;
};

__device__ __forceinline__ float teacher_value(const void *t, int type, long long at) {
    if (type == F32) return static_cast<const float *>(t)[at];
    const uint32_t b = static_cast<const uint16_t *>(t)[at];
    return type == BF16 ? value_of_bits<BF16>(b) : value_of_bits<F16>(b);
}
// e_k = exp(d_k) of the listed entries, d_k = (t_k - t0) / T - lse (no rest: without lse), and what a row's loss and gradient need of them
struct ListSums {
    double S, A, B;    // sum e_k, sum e_k d_k, sum e_k s_k / T
};
__device__ __forceinline__ double below_of(float t, float t0, double it, double lse) { return ((double)t - (double)t0) * it - lse; }

// What the tokens of a row add up to.  Without a rest every token counts as unlisted.
struct TokenSums {
    double Zo, Zl;     // of exp((s - mo) / T) over the unlisted tokens, of exp((s - m) / T) over the listed ones
    float mo, m;       // the unlisted tokens' maximum, the row's; 0 where it is -inf
};
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }

// The end of a row, by one wave.  The three logarithms side by side in three lanes: one after the other they are a third of a short row's time.
__device__ __forceinline__ DistillRow finish_row(const ListSums &l, const TokenSums &z, float t0, double lse, double it, bool rest, double *loss) {
    const int lane = threadIdx.x & 63;
    const double above = rest ? ((double)z.m - (double)z.mo) * it : 0.0;
    const double wo = above <= 0.0 ? 1.0 : exp_of(-above);      // (below 0: none is unlisted)
    const double Z = rest ? z.Zo * wo + z.Zl : z.Zo;
    double pr = 1.0 - l.S;
    pr = pr < 0.0 || z.Zo == 0.0 ? 0.0 : pr;      // (NaN stays)
    const double logs = log(lane == 0 ? Z : lane == 1 ? z.Zo : rest ? pr : l.S);
    const double logZ = __shfl(logs, 0), log_out = __shfl(logs, 1), log_last = __shfl(logs, 2);
    const double B = l.B - l.S * ((double)z.m * it + logZ);      // sum e_k log q_k
    DistillRow st;
    st.m = z.m;
    st.mo = z.mo;
    st.t0 = t0;
    if (rest) {
        const double log_qr = log_out - above - logZ;
        *loss = l.A - B + (pr > 0.0 ? pr * (log_last - log_qr) : pr);
        const double P = l.S + pr;
        st.in = P / Z;
        st.out = st.in * wo - (pr > 0.0 ? pr / z.Zo : pr);
        st.lp0 = lse;
    } else {
        *loss = l.S == 0.0 ? 0.0 : (l.A - B) / l.S - log_last;
        st.in = st.out = l.S == 0.0 ? 0.0 : 1.0 / Z;
        st.lp0 = l.S == 0.0 ? 0.0 : log_last;
    }
    return st;
}

// what multiplies a row's gradient
__device__ __forceinline__ double grad_factor(const DistillArgs &a, long long r) {
    double g = a.scale * a.temperature * (a.weight ? (double)a.weight[r] : 1.0);
    if (a.norm) g *= a.norm[0];
    if (a.upstream) g *= (double)a.upstream[a.each ? r : 0];
    return g;
}

template <int TY>
__device__ __forceinline__ char *grad_row(const DistillArgs &a, long long r) {
    return static_cast<char *>(a.grad) + r * a.vocab * (long long)sizeof(typename El<TY>::type);
}
template <int TY>
__device__ __forceinline__ void store_one(char *row, int j, float x) {
    if (TY == F32)
        reinterpret_cast<float *>(row)[j] = x;
    else
        reinterpret_cast<uint16_t *>(row)[j] = (uint16_t)to_bits<TY>(x);
}

// ---- rows of up to 64 tokens and 64 listed entries: a wave a row, lane j its token j and its entry j ----
// MODE 0: losses and row records;  1: losses and gradient;  2: gradient from the records
template <int TY, int MODE>
__global__ __launch_bounds__(256) void distill_small_kernel(DistillArgs a, long long rows) {
    const int lane = threadIdx.x & 63;
    const long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= rows) return;
    const bool rest = a.lse != nullptr, mine = lane < a.vocab;
    const float weight = a.weight ? a.weight[r] : 1.f;
    char *out = MODE ? grad_row<TY>(a, r) : nullptr;
    if (!(weight > 0.f)) {
        if (MODE && mine) store_one<TY>(out, lane, 0.f);
        if (MODE != 2 && lane == 0) a.losses[r] = 0.f;      // (no record: the gradient looks at the weight too)
        return;
    }
    const char *row = row_at<TY>(a.s, r, a.stride);
    int index = lane < a.k ? a.index[r * a.k + lane] : -1;
    if (index >= a.vocab) index = -1;
    const float t = index >= 0 ? teacher_value(a.t, a.tt, r * a.k + lane) : -INFINITY;
    const float x = mine ? value_of_bits<TY>(load_bits<TY>(row, lane)) : -INFINITY;
    DistillRow st;
    if (MODE == 2) {
        st = a.stat[r];
    } else {
        bool in = false;
        float t0 = 0.f;
        double lse = 0.0;
        TokenSums z;
        z.m = z.mo = base_of(wave_reduce<MaxF>(x));
        if (rest) {
            for (int k = 0; k < a.k; ++k) in |= __shfl(index, k) == lane;
            z.mo = base_of(wave_reduce<MaxF>(in ? -INFINITY : x));
            lse = (double)a.lse[r];
        }
        const double e = mine ? exp_of(((double)x - (double)(in ? z.m : z.mo)) * a.it) : 0.0;
        z.Zo = wave_reduce<Sum>(in ? 0.0 : e);
        if (rest) {
            z.Zl = wave_reduce<Sum>(in ? e : 0.0);
        } else {
            t0 = base_of(wave_reduce<MaxF>(t));
        }
        const float xi = __shfl(x, index < 0 ? 0 : index);
        ListSums l{0.0, 0.0, 0.0};
        if (index >= 0) {
            const double d = below_of(t, t0, a.it, lse), w = exp_of(d);
            if (w != 0.0) l = ListSums{w, w * d, w * ((double)xi * a.it)};
        }
        l.S = wave_reduce<Sum>(l.S);
        l.A = wave_reduce<Sum>(l.A);
        l.B = wave_reduce<Sum>(l.B);
        double loss;
        st = finish_row(l, z, t0, lse, a.it, rest, &loss);
        if (lane == 0) {
            a.losses[r] = (float)(loss * a.temperature * a.temperature * (double)weight);
            if (MODE == 0) a.stat[r] = st;
        }
    }
    if (MODE == 0) return;
    const double g = grad_factor(a, r);
    const double p = index >= 0 ? g * exp_of(below_of(t, st.t0, a.it, st.lp0)) : 0.0;
    bool in = false;
    double take = 0.0;
    for (int k = 0; k < a.k; ++k) {
        const bool here = __shfl(index, k) == lane;
        const double pk = __shfl(p, k);
        in |= here;
        take += here ? pk : 0.0;
    }
    const double e = exp_of(((double)x - (double)(in ? st.m : st.mo)) * a.it);
    if (mine) store_one<TY>(out, lane, (float)(g * (in ? st.in : st.out) * e - take));
}

// ---- a workgroup a row ----
struct RowList {      // the list in LDS
    double *e;        // t_k, later e_k
    double *w;        // the student's logit s_k, later exp((s_k - m) / T)
    int *index;       // -1: empty
    uint32_t *bits;   // of the tokens that are listed
    float t0;
    double lse;
    ListSums own;     // this thread's entries
};
struct ListShared {
    int again;        // whether a token is listed twice
    uint32_t top;     // key of the largest listed logit
    uint32_t high;    // key of the largest student logit of a listed token
};
__host__ __device__ __forceinline__ int list_words(int vocab, int k) { return 5 * k + ((vocab + 31) >> 5); }

// The list and its sums.  They need nothing of the row's maximum, so all of this runs while the row's loads are on their way.  The bits stand when it returns; the caller's
// next barrier stands before the first use of e and of sh.high.
template <int TY, int NT>
__device__ __forceinline__ RowList load_list(const DistillArgs &a, long long r, const char *row, double *lds, ListShared &sh) {
    RowList l;
    l.e = lds;
    l.w = lds + a.k;
    l.index = reinterpret_cast<int *>(l.w + a.k);
    l.bits = reinterpret_cast<uint32_t *>(l.index + a.k);
    for (int i = threadIdx.x; i < (a.vocab + 31) >> 5; i += NT) l.bits[i] = 0;
    if (threadIdx.x == 0) {
        sh.again = 0;
        sh.top = sh.high = 0;
    }
    __syncthreads();
    uint32_t top = 0, first = 0;      // first: the student's logit of the thread's first entry, on its way over the barrier
    for (int k = threadIdx.x; k < a.k; k += NT) {
        const float t = teacher_value(a.t, a.tt, r * a.k + k);
        const int j = a.index[r * a.k + k];
        const bool ok = j >= 0 && j < a.vocab;
        if (ok && k == (int)threadIdx.x) first = load_bits<TY>(row, j);
        l.index[k] = ok ? j : -1;
        l.e[k] = (double)t;
        if (ok && (atomicOr(&l.bits[j >> 5], 1u << (j & 31)) >> (j & 31) & 1)) sh.again = 1;
        if (ok) top = max(top, key_of_bits<F32>(__float_as_uint(t)));
    }
    if (!a.lse && top) atomicMax(&sh.top, top);
    __syncthreads();
    l.t0 = a.lse || !sh.top ? 0.f : base_of(value_of_key<F32>(sh.top));
    l.lse = a.lse ? (double)a.lse[r] : 0.0;
    l.own = ListSums{0.0, 0.0, 0.0};
    uint32_t high = 0;
    for (int k = threadIdx.x; k < a.k; k += NT) {
        const int j = l.index[k];
        double e = 0.0;
        if (j >= 0) {
            const double d = below_of((float)l.e[k], l.t0, a.it, l.lse);
            e = exp_of(d);
            const uint32_t b = k == (int)threadIdx.x ? first : load_bits<TY>(row, j);
            const float x = value_of_bits<TY>(b);
            if (e != 0.0) {
                l.own.S += e;
                l.own.A += e * d;
                l.own.B += e * ((double)x * a.it);
            }
            l.w[k] = (double)x;
            high = max(high, key_of_bits<TY>(b));
        }
        l.e[k] = e;
    }
    if (a.lse && high) atomicMax(&sh.high, high);
    return l;
}
// The listed tokens' weights against the row's maximum m, by the threads that hold their entries; the sum over this thread's tokens, each token once: by its first entry, so
// that the sum's order does not change
template <int NT>
__device__ __forceinline__ double list_weights(const DistillArgs &a, const RowList &l, int again, float m) {
    double sum = 0.0;
    for (int k = threadIdx.x; k < a.k; k += NT) {
        const int j = l.index[k];
        if (j < 0) continue;
        const double w = exp_of((l.w[k] - (double)m) * a.it);
        l.w[k] = w;
        bool first = true;
        if (again)
            for (int q = 0; q < k; ++q) first &= l.index[q] != j;
        if (first) sum += w;
    }
    return sum;
}
// the row's maximum, of that of its unlisted tokens and the listed ones' key (no rest: 0; NaN counts in the sums)
template <int TY>
__device__ __forceinline__ float row_maximum(float mo, uint32_t high) { return base_of(high ? fmaxf(mo, value_of_key<TY>(high)) : mo); }

// A gradient row was written as if nothing were listed; its listed tokens get their own values, the probabilities of all entries that name one together and in the list's
// order.  A barrier stands between the two stores of an element.  gp: what turns e_k into the gradient's p_k.  q and p cancel where the student has learnt: in 64 bits.
template <int TY, int NT>
__device__ __forceinline__ void fix_listed(const DistillArgs &a, const RowList &l, int again, char *out, const DistillRow &st, double g, double gp) {
    const double fin = g * st.in;
    for (int k = threadIdx.x; k < a.k; k += NT) {
        const int j = l.index[k];
        if (j < 0) continue;
        double take = gp * l.e[k];
        if (again) {
            take = 0.0;
            for (int q = 0; q < a.k; ++q)
                if (l.index[q] == j) take += gp * l.e[q];
        }
        store_one<TY>(out, j, (float)(fin * l.w[k] - take));
    }
}

// sums of C doubles over the block, in one round; the first wave gets them
template <int NT, int C>
__device__ __forceinline__ void block_sums(double (&v)[C], double (*scratch)[16]) {
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] = wave_reduce<Sum>(v[i]);
    if (NT == 64) return;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int i = 0; i < C; ++i) scratch[i][threadIdx.x >> 6] = v[i];
    __syncthreads();
    if (threadIdx.x >= 64) return;
#pragma unroll
    for (int i = 0; i < C; ++i) {
        v[i] = scratch[i][threadIdx.x & (NT / 64 - 1)];
#pragma unroll
        for (int q = 1; q < NT / 64; q <<= 1) v[i] += __shfl_xor(v[i], q);
    }
}

// A vector without the listed tokens (in: their bits; few vectors have any)
template <int TY>
__device__ __forceinline__ void hide_listed(Vec &v, uint32_t in) {
    constexpr int N = El<TY>::N;
    if (!(in & ((1u << N) - 1))) return;
    auto all = [&](int e) { return (uint32_t)((int)(in << (31 - e)) >> 31); };      // bit e in every bit
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const uint32_t mask = TY == F32 ? all(q) : (all(2 * q) & 0xffffu) | (all(2 * q + 1) & 0xffff0000u);
        v.d[q] = (v.d[q] & ~mask) | (El<TY>::LOWEST & mask);
    }
}
// the bits of vector i (behind the row's end: of the last)
template <int TY>
__device__ __forceinline__ uint32_t bits_at(const RowList &l, int i, int nvec) {
    const int at = min(i, nvec - 1) * El<TY>::N;
    return l.bits[at >> 5] >> (at & 31);
}
// What an unlisted token's exponential is multiplied with, for fp32 gradients in two parts.
struct Factor {
    float hi, lo;
};
__device__ __forceinline__ Factor factor_of(double f) {
    const float hi = (float)f;
    return Factor{hi, isfinite(hi) ? (float)(f - (double)hi) : 0.f};
}
// A vector of a gradient row in which nothing is listed
template <int TY>
__device__ __forceinline__ void grad_vector(const Vec &v, float base, const Exponent &c, const Factor &f, float *x) {
#pragma unroll
    for (int e = 0; e < El<TY>::N; ++e) {
        const float d = value_of<TY>(v, e) - base;
        if (TY == F32) {
            const float w = weight_of(d, c);
            x[e] = fmaf(w, f.hi, w * f.lo);
        } else {      // (rounded to 2^-9 or 2^-12 of itself: an exponent off by 2^-25 of its 60 or so does not reach it)
            x[e] = f.hi * __builtin_amdgcn_exp2f(d * c.one);
        }
    }
}

// A row without weight: zeros
template <int TY, int NT>
__device__ void empty_row(const DistillArgs &a, long long r, bool grad) {
    if (threadIdx.x == 0) a.losses[r] = 0.f;
    if (!grad) return;
    float x[El<TY>::N];
#pragma unroll
    for (int e = 0; e < El<TY>::N; ++e) x[e] = 0.f;
    char *out = grad_row<TY>(a, r);
    for (int i = threadIdx.x; i * El<TY>::N < a.vocab; i += NT) store_vec<TY>(out, i, a.vocab, x);
}

// The first wave, with the row's sums (Zo, Zl and the list's): its loss, and its record -- for the gradient of a later call, or (GRAD) of this workgroup, with what turns e_k into the gradient's p_k
template <bool GRAD>
__device__ __forceinline__ void end_row(const DistillArgs &a, long long r, const double (&all)[5], float mo, float m, const RowList &list, bool rest, float weight, double g, DistillRow *row, double *gp) {
    double loss;
    const DistillRow st = finish_row(ListSums{all[2], all[3], all[4]}, TokenSums{all[0], all[1], mo, m}, list.t0, list.lse, a.it, rest, &loss);
    if (threadIdx.x) return;
    a.losses[r] = (float)(loss * a.temperature * a.temperature * (double)weight);
    if (GRAD) {
        *row = st;
        *gp = rest ? g : all[2] == 0.0 ? 0.0 : g / all[2];
    } else {
        a.stat[r] = st;
    }
}

// The row in registers, NV vectors a thread: read once; GRAD: its gradient written in the same pass.  Dynamic LDS: the list.
// (64 registers for up to four vectors a thread, eight waves a SIMD: 4,096 x 4,096 bf16 forward 22.9 -> 22.0 us)
template <int TY, int NT, int NV, bool GRAD>
__global__ __launch_bounds__(NT, NV <= 4 ? 8 : 1) void distill_row_kernel(DistillArgs a) {
    constexpr int N = El<TY>::N;
    extern __shared__ double lds[];
    __shared__ double sd[5][16];
    __shared__ float sf[16];
    __shared__ DistillRow shared_row;
    __shared__ double shared_gp;
    __shared__ ListShared sh;
    const long long r = blockIdx.x;
    const int tid = threadIdx.x;
    const float weight = a.weight ? a.weight[r] : 1.f;
    if (!(weight > 0.f)) return empty_row<TY, NT>(a, r, GRAD);
    const char *row = row_at<TY>(a.s, r, a.stride);
    const int nvec = (a.vocab + N - 1) / N;
    Vec v[NV];
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        const int i = q * NT + tid;
        if (i < nvec)
            v[q] = load_vec<TY>(row, i, a.vocab);
        else
            v[q] = Vec{{El<TY>::LOWEST, El<TY>::LOWEST, El<TY>::LOWEST, El<TY>::LOWEST}};
    }
    const RowList list = load_list<TY, NT>(a, r, row, lds, sh);
    const bool rest = a.lse != nullptr;
    float m = -INFINITY;
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        if (rest) hide_listed<TY>(v[q], bits_at<TY>(list, q * NT + tid, nvec));
#pragma unroll
        for (int e = 0; e < N; ++e) m = fmaxf(m, value_of<TY>(v[q], e));
    }
    m = wave_reduce<MaxF>(m);
    if ((tid & 63) == 0) sf[tid >> 6] = m;
    __syncthreads();
    for (int w = 0; w < NT / 64; ++w) m = fmaxf(m, sf[w]);
    const float base = base_of(m), M = row_maximum<TY>(m, sh.high);
    double s = 0.0;
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        forget(v[q]);
        s += weights_of<TY>(v[q], base, a.c);
    }
    double all[5] = {s, rest || GRAD ? list_weights<NT>(a, list, sh.again, M) : 0.0, list.own.S, list.own.A, list.own.B};
    block_sums<NT, 5>(all, sd);
    const double g = GRAD ? grad_factor(a, r) : 0.0;
    if (tid < 64) end_row<GRAD>(a, r, all, base, M, list, rest, weight, g, &shared_row, &shared_gp);
    if (!GRAD) return;
    __syncthreads();
    const DistillRow st = shared_row;
    const Factor fout = factor_of(g * st.out);
    char *out = grad_row<TY>(a, r);
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        const int i = q * NT + tid;
        forget(v[q]);
        float x[N];
        grad_vector<TY>(v[q], st.mo, a.c, fout, x);
        if (i < nvec) store_vec<TY>(out, i, a.vocab, x);
    }
    __syncthreads();
    fix_listed<TY, NT>(a, list, sh.again, out, st, g, shared_gp);
}

// Longer rows: streamed, with a running maximum; GRAD: the row once more, from a cache, for its gradient.  Several such workgroups share a CU, so that one loads while
// another adds up; a row held in the registers of one workgroup of 1,024 leaves the memory idle meanwhile (2,048 rows of 131,072 bf16: 345 us, so 254).
template <int TY, int NT, bool GRAD>
__global__ __launch_bounds__(NT) void distill_stream_kernel(DistillArgs a) {
    constexpr int N = El<TY>::N, AHEAD = 4;
    extern __shared__ double lds[];
    __shared__ double sd[5][16];
    __shared__ float sf[16];
    __shared__ DistillRow shared_row;
    __shared__ double shared_gp;
    __shared__ ListShared sh;
    const long long r = blockIdx.x;
    const int tid = threadIdx.x;
    const float weight = a.weight ? a.weight[r] : 1.f;
    if (!(weight > 0.f)) return empty_row<TY, NT>(a, r, GRAD);
    const char *row = row_at<TY>(a.s, r, a.stride);
    const int nvec = (a.vocab + N - 1) / N;
    const RowList list = load_list<TY, NT>(a, r, row, lds, sh);
    __syncthreads();
    const bool rest = a.lse != nullptr;
    float m = -INFINITY;
    double s = 0.0;
    for (int first = tid; first < nvec; first += NT * AHEAD) {
        Vec v[AHEAD];
        float top = -INFINITY;
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
            const int i = first + q * NT;
            if (i < nvec)
                v[q] = load_vec<TY>(row, i, a.vocab);
            else
                v[q] = Vec{{El<TY>::LOWEST, El<TY>::LOWEST, El<TY>::LOWEST, El<TY>::LOWEST}};
        }
        uint32_t in[AHEAD];      // (read behind the loads, not between them)
        if (rest)
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) in[q] = bits_at<TY>(list, first + q * NT, nvec);
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
            if (rest) hide_listed<TY>(v[q], in[q]);
#pragma unroll
            for (int e = 0; e < N; ++e) top = fmaxf(top, value_of<TY>(v[q], e));
        }
        if (top > m) {
            s *= (double)weight_of(m - top, a.c);
            m = top;
        }
        const float base = base_of(m);
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) s += weights_of<TY>(v[q], base, a.c);
    }
    const float mo = block_reduce<NT, MaxF>(m, sf), base = base_of(mo), M = row_maximum<TY>(mo, sh.high);
    if (m != mo && s != 0.0) s *= (double)weight_of(m - base, a.c);   // (s is NaN where the thread met one)
    double all[5] = {s, rest || GRAD ? list_weights<NT>(a, list, sh.again, M) : 0.0, list.own.S, list.own.A, list.own.B};
    block_sums<NT, 5>(all, sd);
    const double g = GRAD ? grad_factor(a, r) : 0.0;
    if (tid < 64) end_row<GRAD>(a, r, all, base, M, list, rest, weight, g, &shared_row, &shared_gp);
    if (!GRAD) return;
    __syncthreads();
    const DistillRow st = shared_row;
    const Factor fout = factor_of(g * st.out);
    char *out = grad_row<TY>(a, r);
    for (int first = tid; first < nvec; first += NT * AHEAD) {
        Vec v[AHEAD];
#pragma unroll
        for (int q = 0; q < AHEAD; ++q)
            if (first + q * NT < nvec) v[q] = load_vec<TY, true>(row, first + q * NT, a.vocab);
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
            float x[N];
            grad_vector<TY>(v[q], st.mo, a.c, fout, x);
            if (first + q * NT < nvec) store_vec<TY>(out, first + q * NT, a.vocab, x);
        }
    }
    __syncthreads();
    fix_listed<TY, NT>(a, list, sh.again, out, st, g, shared_gp);
}

// sum of the rows' losses over the sum of their weights (mean), or the sum; norm[0] = what the gradient multiplies with
__global__ __launch_bounds__(1024) void distill_join_kernel(const float *losses, const float *weight, long long n, int mean, float *out, double *norm) {
    __shared__ double sd[16];
    double l = 0.0, w = 0.0;
    for (long long i = threadIdx.x; i < n; i += 1024) {
        if (losses) l += (double)losses[i];
        const float wi = weight ? weight[i] : 1.f;
        if (wi > 0.f) w += (double)wi;
    }
    l = block_reduce<1024, Sum>(l, sd);
    w = block_reduce<1024, Sum>(w, sd);
    if (threadIdx.x) return;
    const double f = mean ? (w > 0.0 ? 1.0 / w : 0.0) : 1.0;
    if (out) out[0] = (float)(l * f);
    if (norm) norm[0] = f;
}

// The gradient from the row records: `chunks` workgroups a row, each PER elements of it; the last rows first, which the forward read last
template <int TY, int NT>
__global__ __launch_bounds__(NT) void distill_bwd_kernel(DistillArgs a, int chunks, long long rows) {
    constexpr int N = El<TY>::N, NV = 4, PER = NT * NV * N;
    __shared__ uint32_t bits[PER / 32];
    __shared__ int again, found;
    const long long r = rows - 1 - blockIdx.x / chunks;
    const int first = (int)(blockIdx.x % chunks) * PER, tid = threadIdx.x;
    const char *row = row_at<TY>(a.s, r, a.stride);
    char *out = grad_row<TY>(a, r);
    const int nvec = (a.vocab + N - 1) / N, from = first / N + tid;
    const DistillRow st = a.stat[r];      // (in front of every store: scalar loads; a row without weight has none, and does not look at it)
    const double g = grad_factor(a, r);
    float x[N];
    if (a.weight && !(a.weight[r] > 0.f)) {
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = 0.f;
#pragma unroll
        for (int q = 0; q < NV; ++q)
            if (from + q * NT < nvec) store_vec<TY>(out, from + q * NT, a.vocab, x);
        return;
    }
    Vec v[NV];
#pragma unroll
    for (int q = 0; q < NV; ++q)
        if (from + q * NT < nvec) v[q] = load_vec<TY, true>(row, from + q * NT, a.vocab);
    for (int i = tid; i < PER / 32; i += NT) bits[i] = 0;
    if (tid == 0) again = found = 0;
    __syncthreads();
    // (a listed token's store waits for the others' at the barrier; which tokens are listed twice is looked for meanwhile.  Its entry's logits read here too, ahead of the barrier:
    // 16,384 x 1,000 bf16 28 -> 32 us, the wave with the list holds up the others' stores)
    for (int k = tid; k < a.k; k += NT) {
        const int j = a.index[r * a.k + k];
        if (j < first || j - first >= PER || j >= a.vocab) continue;
        if (atomicOr(&bits[(j - first) >> 5], 1u << (j & 31)) >> (j & 31) & 1) again = 1;
        found = 1;
    }
    const Factor fout = factor_of(g * st.out);
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        grad_vector<TY>(v[q], st.mo, a.c, fout, x);
        if (from + q * NT < nvec) store_vec<TY>(out, from + q * NT, a.vocab, x);
    }
    __syncthreads();
    if (!found) return;
    for (int k = tid; k < a.k; k += NT) {
        const int at = a.index[r * a.k + k];
        if (at < first || at - first >= PER || at >= a.vocab) continue;
        const float t = teacher_value(a.t, a.tt, r * a.k + k), listed = value_of_bits<TY>(load_bits<TY>(row, at));
        double p = 0.0;
        if (again) {      // all entries of the token, in the list's order
            for (int q = 0; q < a.k; ++q)
                if (a.index[r * a.k + q] == at) p += exp_of(below_of(teacher_value(a.t, a.tt, r * a.k + q), st.t0, a.it, st.lp0));
        } else {
            p = exp_of(below_of(t, st.t0, a.it, st.lp0));
        }
        store_one<TY>(out, at, (float)(g * (st.in * exp_of(((double)listed - (double)st.m) * a.it) - p)));
    }
}

}  // namespace rows
