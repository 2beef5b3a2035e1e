// One token a row, drawn with a given number u in [0, 1).
//
// w_j = exp((x_j - max x) / T), the order of a row: larger first, equal ones by index.  Each filter keeps a prefix of that order: top_k its first k; top_p, of these, the
// shortest prefix that holds at least top_p of their sum; min_p those with w >= min_p.  The token is the first of the kept whose inclusive sum exceeds u times their sum.
// So every step is one question about the sorted row -- "where does its running sum (or count) cross this number" -- and no row of a large vocabulary is sorted:
//   up to 256 tokens: a wave holds the row sorted in its registers (16,384 x 48 fp32: 15 us; 14,769 x 106: 239 us by way of the list below);
//   few candidates (top_k up to 512, or a vocabulary that fits the list): the candidates are collected and sorted in LDS (top_rows.hpp), the sums are a scan over them;
//   16-bit logits: there are only 65,536 values.  How often each occurs is counted in LDS (128 KB of 16-bit counters), a weight is computed once a value instead of once a
//   token, and a crossing lies in a page of 1,024 values, then at a value, then at one of the tokens that have it;
//   fp32 logits: a histogram of the weights over T log2 w (88 bins an octave down to 2^-46, where a weight ends) finds the bin of a crossing, the bin's elements are collected
//   and sorted, and the crossing lies among them.
// The borders are 64-bit: sums over values or bins are integers of 2^-44 (LDS atomics fill them: their order does not matter), the list's are doubles.  With fp32 sums of a
// nucleus of 30,000 tokens one row in some thousand would draw another token than the definition gives.
#pragma once
#include "row_common.hpp"
#include "top_rows.hpp"

namespace rows {

constexpr int LISTED_K = 512;                     // top_k up to here: half the threads, whose maxima bound the list well
constexpr int BINS = 4096;
constexpr double BINS_PER_OCTAVE = 88.0;         // 46.5 octaves in 4,096 bins
constexpr double UNIT = 17592186044416.0;        // 2^44: 2^18 weights of 1 sum to 2^62
constexpr int PAGE = 1024, PAGES = 64;           // the 65,536 values of a 16-bit type

struct SampleArgs {
    const void *x;
    long long stride;
    int vocab;
    const float *uniform;
    float temperature, top_p, min_p;             // where the pointer below is NULL
    int top_k;
    const float *temperatures, *top_ps, *min_ps;
    const int32_t *top_ks;
    long long *token;
    float *logp;
};

struct SampleShared {
    SelectShared<LIST> sel;
    union {
        double sum[LIST];    // inclusive sums of the sorted list
        struct {
            u64 mass[BINS];
            uint32_t count[BINS];
        };
    };
    u64 found[5];
};
struct CountShared {
    uint32_t times[PAGES * PAGE / 2];            // two 16-bit counters a word
    u64 mass[PAGES];
    uint32_t count[PAGES];
    u64 pages;                                   // those that have something
    u64 u[16];
    uint32_t w[16];
    uint32_t at[PAGE];                           // equals by (group of vectors, wave)
    u64 found[4];
};

// a row's parameters
struct Drawing {
    double it, u;       // 1 / temperature (0: the first of the order), the uniform within [0, 1)
    float top_p, min_p;
    int k;              // 0: all
    __device__ __forceinline__ Drawing(const SampleArgs &a, long long r) {
        const float T = a.temperatures ? a.temperatures[r] : a.temperature;
        it = T > 0.f ? 1.0 / (double)fminf(T, 3.402823466e38f) : 0.0;      // (inf: the largest finite one, all weights 1)
        k = a.top_ks ? a.top_ks[r] : a.top_k;
        if (k >= a.vocab || k < 0) k = 0;
        top_p = a.top_ps ? a.top_ps[r] : a.top_p;
        min_p = a.min_ps ? a.min_ps[r] : a.min_p;
        min_p = min_p > 1.f ? 1.f : min_p > 0.f ? min_p : 0.f;
        const float v = a.uniform[r];
        u = !(v > 0.f) ? 0.0 : v >= 1.f ? 0.99999994039535522 : (double)v;
    }
    // (a top_p of nothing keeps the first of the order: no running sum is asked where it reaches a number that it has from the start)
    __device__ __forceinline__ bool greedy() const { return !(it > 0.0) || k == 1 || top_p <= 0.f; }
};
template <int TY>
__device__ __forceinline__ bool no_distribution(uint32_t top) { return top >= key_inf<TY>() || top <= key_ninf<TY>(); }

// ---- rows of up to 256 tokens: a wave a row, four a workgroup, the row sorted in registers ----
template <int TY, int E>
__global__ __launch_bounds__(256) void sample_small_kernel(SampleArgs a, long long rows) {
    const int lane = threadIdx.x & 63;
    const long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= rows) return;
    const Drawing d(a, r);
    u64 c[E];
    sorted_row<TY, E>(row_at<TY>(a.x, r, a.stride), a.vocab, c);
    const uint32_t top = __shfl(key_of(c[0]), 0);
    if (no_distribution<TY>(top) || d.greedy()) {
        if (lane == 0) {
            const bool none = no_distribution<TY>(top);
            a.token[r] = none ? -1 : index_of(c[0]);
            a.logp[r] = none ? NAN : 0.f;
        }
        return;
    }
    int n = d.k ? d.k : a.vocab;
    double w[E], upto[E], part = 0.0;
    uint32_t in_p = 0, in_m = 0, passed = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        w[e] = lane * E + e < n ? exp(((double)value_of_key<TY>(key_of(c[e])) - (double)value_of_key<TY>(top)) * d.it) : 0.0;
        part += w[e];
        in_m += lane * E + e < n && w[e] >= (double)d.min_p;
    }
    double run = part;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const double o = __shfl_up(run, s);
        if (lane >= s) run += o;
    }
    const double total = __shfl(run, 63), up = __shfl_up(run, 1);
    run = lane ? up : 0.0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        in_p += lane * E + e < n && run < (double)d.top_p * total;
        run += w[e];
        upto[e] = run;
    }
    if (d.top_p < 1.f) n = min(n, (int)wave_reduce<Sum>(in_p));
    if (d.min_p > 0.f) n = min(n, (int)wave_reduce<Sum>(in_m));
    n = max(n, 1);
    double last = upto[0];
#pragma unroll
    for (int e = 1; e < E; ++e) last = (n - 1) % E == e ? upto[e] : last;
    const double W = __shfl(last, (n - 1) / E), target = d.u * W;
#pragma unroll
    for (int e = 0; e < E; ++e) passed += lane * E + e < n && upto[e] <= target;
    const int at = min((int)wave_reduce<Sum>(passed), n - 1);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (lane * E + e != at) continue;
        a.token[r] = index_of(c[e]);
        a.logp[r] = (float)log(w[e] / W);
    }
}

// ---- the list's way: sorted candidates in sel.list ----
template <int TY, int NT, int L>
__device__ void draw_from_list(SelectShared<L> &sel, double *sum, int n, int k, double it, float top_p, float min_p, double u, long long *token, float *logp) {
    const int tid = threadIdx.x;
    n = k > 0 && k < n ? k : n;
    const double top = (double)value_of_key<TY>(key_of(sel.list[0]));
    const int per = (n + NT - 1) / NT;           // consecutive entries a thread
    auto weight = [&](int i) { return exp(((double)value_of_key<TY>(key_of(sel.list[i])) - top) * it); };
    double part = 0.0;
    int above = 0;
    for (int i = tid * per; i < min(n, (tid + 1) * per); ++i) {
        const double w = weight(i);
        part += w;
        above += w >= (double)min_p;
    }
    double total;
    const double before = block_scan<NT>(part, sel.d, &total);
    double run = before;
    int in_p = 0;
    for (int i = tid * per; i < min(n, (tid + 1) * per); ++i) {
        in_p += run < (double)top_p * total;
        run += weight(i);
        sum[i] = run;
    }
    if (min_p > 0.f) {
        const int c = (int)block_reduce<NT, Sum>((uint32_t)above, sel.w);
        n = min(n, c);
    }
    if (top_p < 1.f) {
        const int c = (int)block_reduce<NT, Sum>((uint32_t)in_p, sel.w);
        n = min(n, c);
    }
    n = max(n, 1);
    __syncthreads();
    const double W = sum[n - 1], target = u * W;
    uint32_t passed = 0;
    for (int i = tid; i < n; i += NT) passed += sum[i] <= target;
    passed = block_reduce<NT, Sum>(passed, sel.w);
    if (tid == 0) {
        const int i = min((int)passed, n - 1);
        *token = index_of(sel.list[i]);
        *logp = (float)log(weight(i) / W);
    }
}

// ---- weights in units of 2^-44 ----
struct Weigh {
    double top, octaves;      // the largest logit; log2(e) / T
    __device__ __forceinline__ Weigh(float top_, double it) : top((double)top_), octaves(it * 1.4426950408889634) {}
    __device__ __forceinline__ double below(float x) const { return fmax(((double)x - top) * octaves, -100.0); }     // log2 of the weight, down to where nothing is left
    __device__ __forceinline__ double weight(float x) const { return exp2_of(below(x)); }
    __device__ static __forceinline__ u64 to_units(double w) { return (u64)(w * UNIT + 0.5); }
    __device__ __forceinline__ u64 units(float x) const { return to_units(weight(x)); }
    __device__ __forceinline__ int bin(float x) const { return min((int)(below(x) * -BINS_PER_OCTAVE), BINS - 1); }     // grows as x falls
};

// "At which token of the order does the running sum (the running count) reach -- strict: exceed -- this number?"  The three filters' ends are three such questions, asked in
// a loop, so that the code that answers them is there once.
struct Question {
    bool count, strict;      // (the last question, the draw, is the strict one: it alone wants the token's index)
    double target;
    __device__ __forceinline__ bool past(u64 v) const { return strict ? (double)v > target : (double)v >= target; }
};
struct Crossing {
    u64 mass;      // sum up to and with the crossing token
    int index;     // the token
    float x;
};

// over: the units of all tokens with at least min_p, total: of all; answer(question) -> Crossing
template <class ANSWER>
__device__ __forceinline__ Crossing ask_all(const Drawing &d, bool limit_k, u64 over, u64 total, u64 *W, ANSWER answer) {
    Crossing c{0, 0, 0.f};
    *W = over;
#pragma unroll 1
    for (int step = limit_k ? 0 : 1; step < 3; ++step) {
        if (step == 1 && !(d.top_p < 1.f)) continue;
        const Question q{step == 0, step == 2, step == 0 ? (double)d.k : step == 1 ? (double)d.top_p * (double)total : d.u * (double)*W};
        c = answer(q);
        if (step == 0) total = c.mass;
        if (step < 2) *W = min(*W, c.mass);
    }
    return c;
}

// index of the `nth` (1-based) element equal to x (not -inf), in index order.  A first pass counts the equals of every group of NT vectors by wave -- `at`: up to NT numbers --,
// the wave that has the nth looks at its vectors again.
template <int TY, int NT>
__device__ int nth_equal(RowIn<TY, NT, 0> &in, float x, uint32_t nth, uint32_t *at, uint32_t *scratch, u64 *found) {
    constexpr int N = El<TY>::N, NW = NT / 64;
    static_assert(MAX_VOCAB / N / 64 <= NT, "a number a thread");
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (tid == 0) found[0] = found[1] = found[2] = 0;
    in.each([&](const Vec &v, int i) {
        uint32_t c = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) c += __popcll(__ballot(value_of<TY>(v, e) == x));
        if (lane == 0 && i < in.nvec) at[i / NT * NW + wave] = c;
    });
    __syncthreads();
    const int waves = (in.nvec + 63) / 64;      // that had a vector
    const uint32_t mine = tid < waves ? at[tid] : 0;
    uint32_t all;
    const uint32_t pre = block_scan<NT>(mine, scratch, &all);
    if (pre < nth && nth <= pre + mine) {
        found[0] = tid;
        found[1] = pre;
    }
    __syncthreads();
    const int group = (int)found[0] / NW;
    if (wave == (int)found[0] % NW) {
        const int i = group * NT + tid;
        const Vec v = in.get(i);
        uint32_t hits = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) hits |= (uint32_t)(value_of<TY>(v, e) == x) << e;
        uint32_t upto = __popc(hits);
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const uint32_t o = __shfl_up(upto, s);
            if (lane >= s) upto += o;
        }
        uint32_t run = (uint32_t)found[1] + upto - __popc(hits);
        while (hits) {
            const int e = __ffs(hits) - 1;
            hits &= hits - 1;
            if (++run == nth) found[2] = (u64)(i * N + e);
        }
    }
    __syncthreads();
    return (int)found[2];
}

// the smallest j >= 1 of `n` equal tokens of weight w at which the running sum (count) is past the target
template <class PAST>
__device__ __forceinline__ uint32_t equals_needed(bool COUNT, u64 above, uint32_t above_count, u64 w, uint32_t n, PAST past) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (COUNT ? past(above_count + mid) : past(above + (u64)mid * w))
            hi = mid;
        else
            lo = mid;
    }
    return hi;
}

// ---- 16-bit logits: by value ----
// The first token of the order at which the running sum crosses
template <int TY, int NT>
__device__ __forceinline__ Crossing cross_values(RowIn<TY, NT, 0> &in, const Weigh &wg, Question ask, CountShared &sh) {
    const int tid = threadIdx.x, lane = tid & 63;
    const bool COUNT = ask.count;
    auto past = [&](u64 v) { return ask.past(v); };
    // the page: page 63 holds the largest values
    __syncthreads();
    if (tid < 64) {
        const int page = PAGES - 1 - lane;
        const u64 m = sh.mass[page];
        const uint32_t c = sh.count[page];
        u64 um = m;
        uint32_t uc = c;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const u64 om = __shfl_up(um, s);
            const uint32_t oc = __shfl_up(uc, s);
            if (lane >= s) {
                um += om;
                uc += oc;
            }
        }
        const u64 hits = __ballot(c > 0 && (COUNT ? past(uc) : past(um)));      // (there is one: a target is at most the sum of everything)
        if (lane == (hits ? __ffsll(hits) - 1 : 0)) {
            sh.found[0] = page;
            sh.found[1] = um - m;
            sh.found[2] = uc - c;
        }
    }
    __syncthreads();
    const int page = (int)sh.found[0];
    const u64 base = sh.found[1];
    const uint32_t cbase = (uint32_t)sh.found[2];
    // the value: a value a thread, the largest first
    const uint32_t key = page * PAGE + (PAGE - 1 - tid);
    const uint32_t c = (sh.times[key >> 1] >> (16 * (key & 1))) & 0xffff;
    const float x = value_of_key<TY>(key);
    const u64 w = c ? wg.units(x) : 0;
    u64 all;
    uint32_t call = 0, cpre = cbase;
    const u64 pre = base + block_scan<NT>((u64)c * w, sh.u, &all);
    if (COUNT) cpre = cbase + block_scan<NT>(c, sh.w, &call);
    const u64 hits = __ballot(c > 0 && (COUNT ? past(cpre + c) : past(pre + c * w)));
    __syncthreads();
    if (lane == 0) sh.w[tid >> 6] = hits ? tid + __ffsll(hits) - 1 : NT;
    __syncthreads();
    uint32_t first = NT;
    for (int i = 0; i < NT / 64; ++i) first = min(first, sh.w[i]);
    if ((uint32_t)tid == min(first, (uint32_t)NT - 1)) {
        const uint32_t j = equals_needed(COUNT, pre, cpre, w, max(c, 1u), past);
        sh.found[0] = pre + (u64)j * w;
        sh.found[1] = j;
        sh.found[2] = key;
        sh.found[3] = c;
    }
    __syncthreads();
    Crossing out{sh.found[0], 0, value_of_key<TY>((uint32_t)sh.found[2])};
    if (ask.strict) {
        const uint32_t j = (uint32_t)sh.found[1];
        __syncthreads();
        out.index = nth_equal<TY, NT>(in, out.x, j, sh.at, sh.w, sh.found);
    }
    return out;
}

// The row's counts alone say everything: one pass over it, and one for the token's index.  false: a counter ran over (a value that 65,536 tokens have)
template <int TY, int NT>
__device__ bool draw_by_value(RowIn<TY, NT, 0> &in, const Drawing &d, CountShared &sh, long long *token, float *logp) {
    static_assert(NT == PAGE && (key_ninf<TY>() & 1) == 1, "a value a thread; -inf in the upper half of its word");
    const int tid = threadIdx.x;
    for (int i = tid; i < PAGES * PAGE / 8; i += NT) reinterpret_cast<uint4 *>(sh.times)[i] = uint4{0, 0, 0, 0};
    if (tid < PAGES) {
        sh.mass[tid] = 0;
        sh.count[tid] = 0;
    }
    if (tid == 0) sh.pages = 0;
    __syncthreads();
    // Two elements a word: key = bits ^ (negative: all ones, else the sign bit), -0 at its own key until the row is through.  -inf, that of a masked vocabulary and of
    // what is behind the row's end, is counted with an odd key: its counter is the upper half of a word, where running over harms no other; it has no weight and is left
    // out of everything below.
    uint32_t counted = 0;
    in.each([&](const Vec &v, int) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            typedef short s16x2 __attribute__((ext_vector_type(2)));
            const uint32_t w = v.d[q], negative = __builtin_bit_cast(uint32_t, __builtin_bit_cast(s16x2, w) >> (s16x2){15, 15});
            const uint32_t keys = w ^ (negative | 0x80008000u);
            const uint32_t lo = keys & 0xffffu, hi = keys >> 16;
            atomicAdd(&sh.times[lo >> 1], (lo & 1) ? 65536u : 1u);
            atomicAdd(&sh.times[hi >> 1], (hi & 1) ? 65536u : 1u);
            counted += (lo != key_ninf<TY>()) + (hi != key_ninf<TY>());
        }
    });
    counted = block_reduce<NT, Sum>(counted, sh.w);
    __syncthreads();
    if (tid == 0) {
        sh.times[key_ninf<TY>() >> 1] &= 0xffffu;
        // -0 is +0 (the upper half of one word, the lower of the next)
        const uint32_t minus = sh.times[0x7fffu >> 1] >> 16;
        sh.times[0x7fffu >> 1] &= 0xffffu;
        sh.times[0x8000u >> 1] += minus;
    }
    __syncthreads();
    // the largest value, the smallest key (below -inf are NaNs of negative sign), the pages that have something
    uint32_t high = 0, low = ~0u;
    u64 some = 0;
#pragma unroll 8
    for (int i = 0; i < PAGES / 2; ++i) {
        const uint32_t at = i * PAGE + tid, w = sh.times[at];
        if (w) {
            high = 2 * at + (w >> 16 ? 1 : 0);
            low = min(low, 2 * at + (w & 0xffffu ? 0 : 1));
            some |= 1ull << (at >> 9);
        }
    }
    some = wave_reduce<Or>(some);
    if ((tid & 63) == 0 && some) atomicOr(&sh.pages, some);
    high = block_reduce<NT, MaxU>(high, sh.w);
    low = block_reduce<NT, MinU>(low, sh.w);
    if (counted == 0 || high >= key_inf<TY>() || low < key_ninf<TY>()) {      // nothing above -inf, +inf or NaN
        if (tid == 0) {
            *token = -1;
            *logp = NAN;
        }
        return true;
    }
    const float top = value_of_key<TY>(high);
    const Weigh wg(top, d.it);
    // the pages' sums; what has at least min_p; all counters together
    u64 over = 0;
    uint32_t seen = 0;
    for (u64 left = sh.pages; left; left &= left - 1) {
        const int page = __ffsll(left) - 1;
        const uint32_t key = page * PAGE + tid;
        const uint32_t c = (sh.times[key >> 1] >> (16 * (key & 1))) & 0xffff;
        if (!__ballot(c > 0)) continue;
        const double w = wg.weight(value_of_key<TY>(key));
        const u64 m = c ? c * Weigh::to_units(w) : 0;
        seen += c;
        if (c && w >= (double)d.min_p) over += m;
        const u64 wave_mass = wave_reduce<Sum>(m);
        const uint32_t wave_count = wave_reduce<Sum>(c);
        if ((tid & 63) == 0) {
            atomicAdd(&sh.mass[page], wave_mass);
            atomicAdd(&sh.count[page], wave_count);
        }
    }
    if (block_reduce<NT, Sum>(seen, sh.w) != counted) return false;
    over = block_reduce<NT, Sum>(over, sh.u);      // (min_p <= 0: everything)
    u64 W;
    const u64 total = wave_reduce<Sum>(sh.mass[tid & 63]);
    const Crossing c = ask_all(d, d.k > 0 && (uint32_t)d.k < counted, over, total, &W, [&](Question q) { return cross_values<TY, NT>(in, wg, q, sh); });
    if (tid == 0) {
        *token = c.index;
        *logp = (float)log(exp(((double)c.x - (double)top) * d.it) / ((double)W / UNIT));
    }
    return true;
}

// ---- fp32 logits, and 16-bit ones that ran over a counter: by bins of the weights' logarithm ----
template <int TY, int NT>
__device__ __forceinline__ Crossing cross_bins(RowIn<TY, NT, 0> &in, const Weigh &wg, Question ask, SampleShared &sh) {
    constexpr int N = El<TY>::N, PER = BINS / NT;
    const int tid = threadIdx.x;
    const bool COUNT = ask.count;
    auto past = [&](u64 v) { return ask.past(v); };
    // the bin: consecutive bins a thread
    u64 m = 0;
    uint32_t c = 0;
    for (int b = 0; b < PER; ++b) {
        m += sh.mass[tid * PER + b];
        if (COUNT) c += sh.count[tid * PER + b];
    }
    u64 all;
    uint32_t call = 0, cbefore = 0;
    const u64 before = block_scan<NT>(m, sh.sel.u, &all);
    if (COUNT) cbefore = block_scan<NT>(c, sh.sel.w, &call);
    __syncthreads();
    if (tid == 0) sh.found[0] = ~0ull;
    __syncthreads();
    {
        const bool mine = COUNT ? past(cbefore + c) && !past(cbefore) : past(before + m) && !past(before);
        const bool first = tid == 0 && past(0ull);      // (target <= 0: the first bin that has something)
        if (mine || first) {
            u64 pm = before;
            uint32_t pc = cbefore;
            for (int b = tid * PER; b < BINS; ++b) {
                const u64 im = sh.mass[b];
                const uint32_t ic = COUNT ? sh.count[b] : 0;
                if (COUNT ? ic > 0 && past(pc + ic) : im > 0 && past(pm + im)) {
                    sh.found[0] = b;
                    sh.found[1] = pm;
                    sh.found[2] = pc;
                    break;
                }
                pm += im;
                pc += ic;
            }
        }
    }
    __syncthreads();
    const int bin = (int)sh.found[0];      // (there is one: a target is at most the sum of everything)
    const u64 base = sh.found[1];
    const uint32_t cbase = (uint32_t)sh.found[2];
    // its elements: few of the row, told apart by fp32 values a little wider than the bin before the bin itself is computed
    const float far_x = (float)(wg.top - (double)(bin + 1) / (BINS_PER_OCTAVE * wg.octaves)), near_x = (float)(wg.top - (double)bin / (BINS_PER_OCTAVE * wg.octaves));
    const float slack = 1e-6f * (fabsf(far_x) + fabsf(near_x) + fabsf((float)wg.top));
    const bool told = slack < INFINITY;      // (at temperatures near the largest fp32 a border lies behind every number: the bin itself tells all of them apart)
    const float low = bin == BINS - 1 || !told ? -INFINITY : far_x - slack, high = told ? near_x + slack : INFINITY;
    if (tid == 0) sh.sel.n = 0;
    __syncthreads();
    in.each([&](const Vec &v, int i) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float x = value_of<TY>(v, e);
            if (x >= low && x <= high && i * N + e < in.vocab && wg.bin(x) == bin) {
                const int at = atomicAdd(&sh.sel.n, 1);
                if (at < LIST) sh.sel.list[at] = composite(key_of<TY>(v, e), i * N + e);
            }
        }
    });
    __syncthreads();
    const int n = sh.sel.n;
    if (n <= LIST) {
        sort_list<NT, LIST>(sh.sel.list, n, sh.sel.sort);
        const int per = (n + NT - 1) / NT;
        u64 part = 0;
        for (int i = tid * per; i < min(n, (tid + 1) * per); ++i) part += wg.units(value_of_key<TY>(key_of(sh.sel.list[i])));
        u64 total;
        u64 run = base + block_scan<NT>(part, sh.sel.u, &total);
        if (tid == 0) sh.found[3] = ~0ull;
        __syncthreads();
        for (int i = tid * per; i < min(n, (tid + 1) * per); ++i) {
            const u64 had = run;
            run += wg.units(value_of_key<TY>(key_of(sh.sel.list[i])));
            const bool at = COUNT ? past(cbase + i + 1) && (i == 0 || !past(cbase + i)) : past(run) && (i == 0 || !past(had));
            if (at) {      // (one thread: the sums do not fall)
                sh.found[3] = i;
                sh.found[4] = run;
            }
        }
        __syncthreads();
        const u64 c0 = sh.sel.list[min(sh.found[3], (u64)max(n - 1, 0))];
        return Crossing{sh.found[4], index_of(c0), value_of_key<TY>(key_of(c0))};
    }
    // too many alike: the crossing value bit by bit of its key within the bin, then the place among its equals
    uint32_t t = 0;
    u64 above = base;
    uint32_t cabove = cbase;
    for (int b = key_bits<TY>() - 1; b >= -1; --b) {
        // b >= 0: the sum of the keys from `mid` up; b == -1: of the keys above t
        const uint32_t mid = b >= 0 ? t | (1u << b) : t;
        u64 pm = 0;
        uint32_t pc = 0;
        in.each([&](const Vec &v, int i) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float x = value_of<TY>(v, e);
                const uint32_t key = key_of<TY>(v, e);
                if (i * N + e < in.vocab && (b >= 0 ? key >= mid : key > t) && wg.bin(x) == bin) {
                    pm += wg.units(x);
                    pc += 1;
                }
            }
        });
        pm = base + block_reduce<NT, Sum>(pm, sh.sel.u);
        pc = cbase + block_reduce<NT, Sum>(pc, sh.sel.w);
        if (b < 0) {
            above = pm;
            cabove = pc;
        } else if (COUNT ? past(pc) : past(pm)) {
            t = mid;
        }
    }
    const float x = value_of_key<TY>(t);
    const u64 w = wg.units(x);
    const uint32_t j = equals_needed(COUNT, above, cabove, w, (uint32_t)in.vocab, past);
    Crossing out{above + (u64)j * w, 0, x};
    __syncthreads();
    if (ask.strict) out.index = nth_equal<TY, NT>(in, x, j, reinterpret_cast<uint32_t *>(sh.sel.list), sh.sel.w, sh.found);
    return out;
}

template <int TY, int NT>
__device__ void draw_by_bins(RowIn<TY, NT, 0> &in, const Drawing &d, float top, SampleShared &sh, long long *token, float *logp) {
    constexpr int N = El<TY>::N;
    const int tid = threadIdx.x;
    const Weigh wg(top, d.it);
    __syncthreads();
    for (int b = tid; b < BINS; b += NT) {
        sh.mass[b] = 0;
        sh.count[b] = 0;
    }
    __syncthreads();
    u64 over = 0;       // weights of at least min_p
    in.each([&](const Vec &v, int i) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const double t = wg.below(value_of<TY>(v, e)), w = exp2_of(t);
            const u64 q = Weigh::to_units(w);
            const int b = min((int)(t * -BINS_PER_OCTAVE), BINS - 1);
            if (i * N + e < in.vocab) {
                if (q) atomicAdd(&sh.mass[b], q);
                if (d.k > 0) atomicAdd(&sh.count[b], 1u);
                if (w >= (double)d.min_p) over += q;
            }
        }
    });
    over = block_reduce<NT, Sum>(over, sh.sel.u);     // (min_p <= 0: everything)
    u64 total = 0, W;
    for (int b = tid; b < BINS; b += NT) total += sh.mass[b];
    total = block_reduce<NT, Sum>(total, sh.sel.u);
    const Crossing c = ask_all(d, d.k > 0, over, total, &W, [&](Question q) {
        __syncthreads();
        return cross_bins<TY, NT>(in, wg, q, sh);
    });
    if (tid == 0) {
        *token = c.index;
        *logp = (float)log(exp(((double)c.x - (double)top) * d.it) / ((double)W / UNIT));
    }
}

// The largest element in order, or that there is no distribution; false: go on with `m`, the row's largest
template <int TY, int NT, int NV>
__device__ bool first_or_none(RowIn<TY, NT, NV> &in, const Drawing &d, float m, uint32_t *scratch, long long *token, float *logp) {
    constexpr int N = El<TY>::N;
    if (!(m < INFINITY) || m == -INFINITY) {      // NaN or +inf, or nothing above -inf
        if (threadIdx.x == 0) {
            *token = -1;
            *logp = NAN;
        }
        return true;
    }
    if (!d.greedy()) return false;
    uint32_t at = ~0u;
    in.each([&](const Vec &v, int i) {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (value_of<TY>(v, e) == m) at = min(at, (uint32_t)(i * N + e));
    });
    at = block_reduce<NT, MinU>(at, scratch);
    if (threadIdx.x == 0) {
        *token = (long long)at;
        *logp = 0.f;
    }
    return true;
}

// rows that fit a list of L
template <int TY, int NT, int NV, int L>
__global__ __launch_bounds__(NT) void sample_listed_kernel(SampleArgs a) {
    __shared__ SelectShared<L> sel;
    __shared__ double sum[L];
    const long long r = blockIdx.x;
    const Drawing d(a, r);
    RowIn<TY, NT, NV> in(row_at<TY>(a.x, r, a.stride), a.vocab);
    float mine = -INFINITY;
    in.each([&](const Vec &v, int) { mine = maximum(mine, largest<TY>(v)); });
    const float m = block_reduce<NT, MaxNan>(mine, sel.f);
    if (first_or_none<TY, NT, NV>(in, d, m, sel.w, a.token + r, a.logp + r)) return;
    const int n = select_first<TY, NT>(in, d.k > 0 ? d.k : a.vocab, mine, sel);
    draw_from_list<TY, NT>(sel, sum, n, d.k, d.it, d.top_p, d.min_p, d.u, a.token + r, a.logp + r);
}

// longer ones
template <int TY, int NT>
__global__ __launch_bounds__(NT) void sample_rows_kernel(SampleArgs a) {
    __shared__ union alignas(16) {
        SampleShared s;
        char by_value[TY == F32 ? 1 : sizeof(CountShared)];
    } sh;
    const long long r = blockIdx.x;
    const Drawing d(a, r);
    RowIn<TY, NT, 0> in(row_at<TY>(a.x, r, a.stride), a.vocab);
    const bool listed = d.k > 0 && d.k <= LISTED_K;
    if constexpr (TY != F32)
        if (!listed && !d.greedy() && draw_by_value<TY, NT>(in, d, *reinterpret_cast<CountShared *>(sh.by_value), a.token + r, a.logp + r)) return;
    float mine = -INFINITY;
    in.each([&](const Vec &v, int) { mine = maximum(mine, largest<TY>(v)); });
    __syncthreads();
    const float m = block_reduce<NT, MaxNan>(mine, sh.s.sel.f);
    if (first_or_none<TY, NT, 0>(in, d, m, sh.s.sel.w, a.token + r, a.logp + r)) return;
    if (listed) {
        const int n = select_first<TY, NT>(in, d.k, mine, sh.s.sel);
        draw_from_list<TY, NT>(sh.s.sel, sh.s.sum, n, d.k, d.it, d.top_p, d.min_p, d.u, a.token + r, a.logp + r);
        return;
    }
    draw_by_bins<TY, NT>(in, d, m, sh.s, a.token + r, a.logp + r);
}

}  // namespace rows
