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
// subtracted from each other, are held in 64 bits; the exponentials of a row are fp32.
#pragma once
#include "row_common.hpp"
#include "top_rows.hpp"

namespace rows {

struct DistillRow {   // what the gradient of a row needs
    float m, mo;      // the row's maximum, that of the unlisted tokens (no rest: the row's)
    float in, out;    // dL / ds_j = T in exp((s_j - m) / T) - T p for the listed tokens, T out exp((s_j - mo) / T) for the others
    float used;       // 0: a row without weight
    double lp0;       // log p_k = a_k - lp0
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
    double temperature;
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
// e_k = exp(a_k - shift) of the listed entries and what a row's loss and gradient need of them
struct ListSums {
    double S, A, B;    // sum e_k, sum e_k (a_k - shift), sum e_k s_k / T
};

// What the tokens of a row add up to.  Without a rest every token counts as unlisted.
struct TokenSums {
    double Zo, Zl;     // of exp((s - mo) / T) over the unlisted tokens, of exp((s - ml) / T) over the listed ones
    float mo, ml;      // their maxima, -inf where there is none
};
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }

// The end of a row, by one wave.  The two exponentials and then the three logarithms side by side in a lane each: one after the other they are a third of a short row's
// time.
__device__ __forceinline__ DistillRow finish_row(const ListSums &l, const TokenSums &z, double shift, double temperature, bool rest, double *loss) {
    const int lane = threadIdx.x & 63;
    const float m = base_of(fmaxf(z.mo, z.ml));
    const double below = exp(((double)(lane == 0 ? z.mo : z.ml) - (double)m) / temperature);
    const double wo = __shfl(below, 0), wl = __shfl(below, 1);
    const double Z = z.Zo * wo + (rest ? z.Zl * wl : 0.0);
    double pr = 1.0 - l.S;
    pr = pr < 0.0 || z.Zo == 0.0 ? 0.0 : pr;      // (NaN stays)
    const double logs = log(lane == 0 ? Z : lane == 1 ? z.Zo : rest ? pr : l.S);
    const double logZ = __shfl(logs, 0), log_out = __shfl(logs, 1), log_last = __shfl(logs, 2);
    const double B = l.B - l.S * ((double)m / temperature + logZ);      // sum e_k log q_k
    DistillRow st;
    st.m = m;
    st.mo = rest ? base_of(z.mo) : m;
    st.used = 1.f;
    if (rest) {
        const double log_qr = log_out + ((double)st.mo - (double)m) / temperature - logZ;
        *loss = l.A - B + (pr > 0.0 ? pr * (log_last - log_qr) : pr);
        const double P = l.S + pr;
        st.in = (float)(P / Z);
        st.out = (float)(P * wo / Z - (pr > 0.0 ? pr / z.Zo : pr));
        st.lp0 = shift;
    } else {
        *loss = l.S == 0.0 ? 0.0 : (l.A - B) / l.S - log_last;
        st.in = st.out = l.S == 0.0 ? 0.f : (float)(1.0 / Z);
        st.lp0 = l.S == 0.0 ? 0.0 : shift + log_last;
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
        if (MODE != 2 && lane == 0) {
            a.losses[r] = 0.f;
            if (MODE == 0) a.stat[r] = DistillRow{0.f, 0.f, 0.f, 0.f, 0.f, 0.0};
        }
        return;
    }
    const char *row = row_at<TY>(a.s, r, a.stride);
    int index = lane < a.k ? a.index[r * a.k + lane] : -1;
    if (index >= a.vocab) index = -1;
    const float t = index >= 0 ? teacher_value(a.t, a.tt, r * a.k + lane) : -INFINITY;
    const float x = mine ? value_of_bits<TY>(load_bits<TY>(row, lane)) : -INFINITY;
    const float c = (float)(1.4426950408889634 / a.temperature);
    DistillRow st;
    if (MODE == 2) {
        st = a.stat[r];
    } else {
        bool in = false;
        double shift;
        TokenSums z{0.0, 0.0, 0.f, -INFINITY};
        if (rest) {
            for (int k = 0; k < a.k; ++k) in |= __shfl(index, k) == lane;
            z.ml = wave_reduce<MaxF>(in ? x : -INFINITY);
            shift = (double)a.lse[r];
        }
        z.mo = wave_reduce<MaxF>(in ? -INFINITY : x);
        const float e = mine ? __builtin_amdgcn_exp2f((x - base_of(in ? z.ml : z.mo)) * c) : 0.f;
        z.Zo = wave_reduce<Sum>(in ? 0.0 : (double)e);
        if (rest) {
            z.Zl = wave_reduce<Sum>(in ? (double)e : 0.0);
        } else {
            const float amax = wave_reduce<MaxF>(t);
            shift = amax == -INFINITY ? 0.0 : (double)amax / a.temperature;
        }
        const float xi = __shfl(x, index < 0 ? 0 : index);
        ListSums l{0.0, 0.0, 0.0};
        if (index >= 0) {
            const double d = (double)t / a.temperature - shift, w = exp(d);
            if (w != 0.0) l = ListSums{w, w * d, w * ((double)xi / a.temperature)};
        }
        l.S = wave_reduce<Sum>(l.S);
        l.A = wave_reduce<Sum>(l.A);
        l.B = wave_reduce<Sum>(l.B);
        double loss;
        st = finish_row(l, z, shift, a.temperature, rest, &loss);
        if (lane == 0) {
            a.losses[r] = (float)(loss * a.temperature * a.temperature * (double)weight);
            if (MODE == 0) a.stat[r] = st;
        }
    }
    if (MODE == 0) return;
    const double g = grad_factor(a, r);
    const float p = index >= 0 ? (float)(g * exp((double)t / a.temperature - st.lp0)) : 0.f;
    bool in = false;
    float take = 0.f;
    for (int k = 0; k < a.k; ++k) {
        const bool here = __shfl(index, k) == lane;
        const float pk = __shfl(p, k);
        in |= here;
        take += here ? pk : 0.f;
    }
    const float e = __builtin_amdgcn_exp2f((x - (in ? st.m : st.mo)) * c);
    if (mine) store_one<TY>(out, lane, (float)(g * (double)(in ? st.in : st.out)) * e - take);
}

// ---- a workgroup a row ----
struct RowList {      // the list in LDS
    int *index;       // -1: empty
    float *e;         // e_k
    uint32_t *bits;   // of the tokens that are listed
    double shift;
    ListSums own;     // this thread's entries
    double Zl;        // ... and their tokens, each once, of exp((s - ml) / T) (with a rest)
    float ml;         // the largest student logit of a listed token (with a rest)
};
struct ListShared {
    int again;        // whether a token is listed twice
    uint32_t top;     // key of the largest listed logit (no rest), of the largest student logit of a listed token (with one)
};
__host__ __device__ __forceinline__ int list_words(int vocab, int k) { return 2 * k + ((vocab + 31) >> 5); }

// The list and its sums.  They need nothing of the row's maximum, so all of this runs while the row's loads are on their way.  The bits stand when it returns; the caller's
// next barrier stands before the first use of e.
template <int TY, int NT>
__device__ __forceinline__ RowList load_list(const DistillArgs &a, long long r, const char *row, uint32_t *lds, ListShared &sh) {
    RowList l;
    l.index = reinterpret_cast<int *>(lds);
    l.e = reinterpret_cast<float *>(lds + a.k);
    l.bits = lds + 2 * a.k;
    for (int i = threadIdx.x; i < (a.vocab + 31) >> 5; i += NT) l.bits[i] = 0;
    if (threadIdx.x == 0) {
        sh.again = 0;
        sh.top = 0;
    }
    __syncthreads();
    uint32_t top = 0;
    for (int k = threadIdx.x; k < a.k; k += NT) {
        const int j = a.index[r * a.k + k];
        const bool ok = j >= 0 && j < a.vocab;
        const float t = ok ? teacher_value(a.t, a.tt, r * a.k + k) : -INFINITY;
        l.index[k] = ok ? j : -1;
        l.e[k] = t;
        if (ok && (atomicOr(&l.bits[j >> 5], 1u << (j & 31)) >> (j & 31) & 1)) sh.again = 1;
        if (ok) top = max(top, a.lse ? key_of_bits<TY>(load_bits<TY>(row, j)) : key_of_bits<F32>(__float_as_uint(t)));
    }
    if (top) atomicMax(&sh.top, top);
    __syncthreads();
    l.ml = -INFINITY;
    if (a.lse) {
        l.shift = (double)a.lse[r];
        if (sh.top) l.ml = value_of_key<TY>(sh.top);
    } else {
        l.shift = sh.top <= key_ninf<F32>() ? 0.0 : (double)value_of_key<F32>(sh.top) / a.temperature;
    }
    l.own = ListSums{0.0, 0.0, 0.0};
    l.Zl = 0.0;
    for (int k = threadIdx.x; k < a.k; k += NT) {
        const int j = l.index[k];
        double e = 0.0;
        if (j >= 0) {
            const double d = (double)l.e[k] / a.temperature - l.shift;
            e = exp(d);
            const double x = (double)value_of_bits<TY>(load_bits<TY>(row, j));
            if (e != 0.0) {
                l.own.S += e;
                l.own.A += e * d;
                l.own.B += e * (x / a.temperature);
            }
            if (a.lse && x != -INFINITY) {
                bool first = true;      // (the token's first entry, so that the sum's order does not change)
                if (sh.again)
                    for (int q = 0; q < k; ++q) first &= l.index[q] != j;
                if (first) l.Zl += exp((x - (double)l.ml) / a.temperature);
            }
        }
        l.e[k] = (float)e;
    }
    return l;
}

// A gradient row was written as if nothing were listed; its listed tokens get their own values, the probabilities of all entries that name one together and in the list's
// order.  A barrier stands between the two stores of an element.  gp: what turns e_k into the gradient's p_k
template <int TY, int NT>
__device__ __forceinline__ void fix_listed(const DistillArgs &a, const RowList &l, int again, const char *row, char *out, const DistillRow &st, double g, float gp, float c) {
    const float fin = (float)(g * (double)st.in);
    for (int k = threadIdx.x; k < a.k; k += NT) {
        const int j = l.index[k];
        if (j < 0) continue;
        float take = gp * l.e[k];
        if (again) {
            take = 0.f;
            for (int q = 0; q < a.k; ++q)
                if (l.index[q] == j) take += gp * l.e[q];
        }
        const float x = value_of_bits<TY>(load_bits<TY>(row, j));
        store_one<TY>(out, j, fin * __builtin_amdgcn_exp2f((x - st.m) * c) - take);
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
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const uint32_t mask = TY == F32 ? ~0u : (e & 1) ? 0xffff0000u : 0xffffu;
        uint32_t &d = v.d[TY == F32 ? e : e >> 1];
        if ((in >> e) & 1) d = (d & ~mask) | (El<TY>::LOWEST & mask);
    }
}
// A vector's exponentials of (x - base) c, added up
template <int TY>
__device__ __forceinline__ void add_vector(const Vec &v, float base, float c, double &s) {
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < El<TY>::N; ++e) sum += __builtin_amdgcn_exp2f((value_of<TY>(v, e) - base) * c);
    s += (double)sum;
}
// A vector of a gradient row in which nothing is listed
template <int TY>
__device__ __forceinline__ void grad_vector(const Vec &v, float base, float c, float scale, float *x) {
#pragma unroll
    for (int e = 0; e < El<TY>::N; ++e) x[e] = scale * __builtin_amdgcn_exp2f((value_of<TY>(v, e) - base) * c);
}

// A row without weight: zeros
template <int TY, int NT>
__device__ void empty_row(const DistillArgs &a, long long r, bool grad) {
    if (threadIdx.x == 0) {
        a.losses[r] = 0.f;
        a.stat[r] = DistillRow{0.f, 0.f, 0.f, 0.f, 0.f, 0.0};
    }
    if (!grad) return;
    float x[El<TY>::N];
#pragma unroll
    for (int e = 0; e < El<TY>::N; ++e) x[e] = 0.f;
    char *out = grad_row<TY>(a, r);
    for (int i = threadIdx.x; i * El<TY>::N < a.vocab; i += NT) store_vec<TY>(out, i, a.vocab, x);
}

// The first wave, with the row's sums (Zo, Zl and the list's): its loss, and its record -- for the gradient of a later call, or (GRAD) of this workgroup, with what turns e_k into the gradient's p_k
template <bool GRAD>
__device__ __forceinline__ void end_row(const DistillArgs &a, long long r, const double (&all)[5], float mo, float ml, double shift, bool rest, float weight, double g, DistillRow *row, float *gp) {
    double loss;
    const DistillRow st = finish_row(ListSums{all[2], all[3], all[4]}, TokenSums{all[0], all[1], mo, ml}, shift, a.temperature, rest, &loss);
    if (threadIdx.x) return;
    a.losses[r] = (float)(loss * a.temperature * a.temperature * (double)weight);
    if (GRAD) {
        *row = st;
        *gp = (float)(rest ? g : all[2] == 0.0 ? 0.0 : g / all[2]);
    } else {
        a.stat[r] = st;
    }
}

// The row in registers, NV vectors a thread: read once; GRAD: its gradient written in the same pass.  Dynamic LDS: the list.
template <int TY, int NT, int NV, bool GRAD>
__global__ __launch_bounds__(NT) void distill_row_kernel(DistillArgs a) {
    constexpr int N = El<TY>::N;
    extern __shared__ uint32_t lds[];
    __shared__ double sd[5][16];
    __shared__ float sf[16];
    __shared__ DistillRow shared_row;
    __shared__ float shared_gp;
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
    const float c = (float)(1.4426950408889634 / a.temperature);
    const bool rest = a.lse != nullptr;
    float m = -INFINITY;
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        const int i = q * NT + tid;
        if (rest && i < nvec) hide_listed<TY>(v[q], list.bits[(i * N) >> 5] >> ((i * N) & 31));
#pragma unroll
        for (int e = 0; e < N; ++e) m = fmaxf(m, value_of<TY>(v[q], e));
    }
    m = wave_reduce<MaxF>(m);
    if ((tid & 63) == 0) sf[tid >> 6] = m;
    __syncthreads();
    for (int w = 0; w < NT / 64; ++w) m = fmaxf(m, sf[w]);
    const float base = base_of(m);
    double s = 0.0;
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        forget(v[q]);
        add_vector<TY>(v[q], base, c, s);
    }
    double all[5] = {s, list.Zl, list.own.S, list.own.A, list.own.B};
    block_sums<NT, 5>(all, sd);
    const double g = GRAD ? grad_factor(a, r) : 0.0;
    if (tid < 64) end_row<GRAD>(a, r, all, m, list.ml, list.shift, rest, weight, g, &shared_row, &shared_gp);
    if (!GRAD) return;
    __syncthreads();
    const DistillRow st = shared_row;
    const float fout = (float)(g * (double)st.out);
    char *out = grad_row<TY>(a, r);
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        const int i = q * NT + tid;
        forget(v[q]);
        float x[N];
        grad_vector<TY>(v[q], st.mo, c, fout, x);
        if (i < nvec) store_vec<TY>(out, i, a.vocab, x);
    }
    __syncthreads();
    fix_listed<TY, NT>(a, list, sh.again, row, out, st, g, shared_gp, c);
}

// Longer rows: streamed, with a running maximum; GRAD: the row once more, from a cache, for its gradient.  Several such workgroups share a CU, so that one loads while
// another adds up; a row held in the registers of one workgroup of 1,024 leaves the memory idle meanwhile (2,048 rows of 131,072 bf16: 345 us, so 263).
template <int TY, int NT, bool GRAD>
__global__ __launch_bounds__(NT) void distill_stream_kernel(DistillArgs a) {
    constexpr int N = El<TY>::N, AHEAD = 4;
    extern __shared__ uint32_t lds[];
    __shared__ double sd[5][16];
    __shared__ float sf[16];
    __shared__ DistillRow shared_row;
    __shared__ float shared_gp;
    __shared__ ListShared sh;
    const long long r = blockIdx.x;
    const int tid = threadIdx.x;
    const float weight = a.weight ? a.weight[r] : 1.f;
    if (!(weight > 0.f)) return empty_row<TY, NT>(a, r, GRAD);
    const char *row = row_at<TY>(a.s, r, a.stride);
    const int nvec = (a.vocab + N - 1) / N;
    const RowList list = load_list<TY, NT>(a, r, row, lds, sh);
    __syncthreads();
    const float c = (float)(1.4426950408889634 / a.temperature);
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
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
            const int i = first + q * NT;
            if (rest && i < nvec) hide_listed<TY>(v[q], list.bits[(i * N) >> 5] >> ((i * N) & 31));
#pragma unroll
            for (int e = 0; e < N; ++e) top = fmaxf(top, value_of<TY>(v[q], e));
        }
        if (top > m) {
            s *= (double)__builtin_amdgcn_exp2f((m - top) * c);
            m = top;
        }
        const float base = base_of(m);
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) add_vector<TY>(v[q], base, c, s);
    }
    const float M = block_reduce<NT, MaxF>(m, sf);
    const float base = base_of(M);
    if (m != M && s != 0.0) s *= (double)__builtin_amdgcn_exp2f((m - base) * c);   // (s is NaN where the thread met one)
    double all[5] = {s, list.Zl, list.own.S, list.own.A, list.own.B};
    block_sums<NT, 5>(all, sd);
    const double g = GRAD ? grad_factor(a, r) : 0.0;
    if (tid < 64) end_row<GRAD>(a, r, all, M, list.ml, list.shift, rest, weight, g, &shared_row, &shared_gp);
    if (!GRAD) return;
    __syncthreads();
    const DistillRow st = shared_row;
    const float fout = (float)(g * (double)st.out);
    char *out = grad_row<TY>(a, r);
    for (int first = tid; first < nvec; first += NT * AHEAD) {
        Vec v[AHEAD];
#pragma unroll
        for (int q = 0; q < AHEAD; ++q)
            if (first + q * NT < nvec) v[q] = load_vec<TY, true>(row, first + q * NT, a.vocab);
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
            float x[N];
            grad_vector<TY>(v[q], st.mo, c, fout, x);
            if (first + q * NT < nvec) store_vec<TY>(out, first + q * NT, a.vocab, x);
        }
    }
    __syncthreads();
    fix_listed<TY, NT>(a, list, sh.again, row, out, st, g, shared_gp, c);
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
    const DistillRow st = a.stat[r];
    float x[N];
    if (st.used == 0.f) {
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
    // (a listed token's store waits for the others' at the barrier; which tokens are listed twice is looked for meanwhile)
    for (int i = tid; i < PER / 32; i += NT) bits[i] = 0;
    if (tid == 0) again = found = 0;
    __syncthreads();
    for (int k = tid; k < a.k; k += NT) {
        const int j = a.index[r * a.k + k] - first;
        if (j >= 0 && j < PER && j + first < a.vocab) {
            found = 1;
            if (atomicOr(&bits[j >> 5], 1u << (j & 31)) >> (j & 31) & 1) again = 1;
        }
    }
    const double g = grad_factor(a, r);
    const float c = (float)(1.4426950408889634 / a.temperature);
    const float fout = (float)(g * (double)st.out), fin = (float)(g * (double)st.in);
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        grad_vector<TY>(v[q], st.mo, c, fout, x);
        if (from + q * NT < nvec) store_vec<TY>(out, from + q * NT, a.vocab, x);
    }
    __syncthreads();
    if (!found) return;
    auto taken = [&](int k) { return (float)(g * exp((double)teacher_value(a.t, a.tt, r * a.k + k) / a.temperature - st.lp0)); };
    for (int k = tid; k < a.k; k += NT) {
        const int j = a.index[r * a.k + k];
        if (j < first || j - first >= PER || j >= a.vocab) continue;
        float take = 0.f;
        if (again) {
            for (int q = 0; q < a.k; ++q)
                if (a.index[r * a.k + q] == j) take += taken(q);
        } else {
            take = taken(k);
        }
        store_one<TY>(out, j, fin * __builtin_amdgcn_exp2f((value_of_bits<TY>(load_bits<TY>(row, j)) - st.m) * c) - take);
    }
}

}  // namespace rows
