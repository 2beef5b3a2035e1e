// Rows of logits: loads, the order of a row's elements and the reductions that the row operators (top_rows.hpp, distill.hpp, sample.hpp) share.
//
// A row is `vocab` elements of fp32, bf16 or fp16, contiguous, at any alignment its type has (a vocabulary of 50,001 leaves every other row of a 16-bit tensor off a
// 4-byte border): 16-byte loads through a type of the element's alignment, which gfx950 takes in one global_load_dwordx4 at any address.  Only whole vectors inside the row
// are loaded that way; the last, partial one goes element by element.
#pragma once
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace rows {

enum { F32 = 0, BF16 = 1, F16 = 2 };
constexpr int MAX_VOCAB = 1 << 18;   // a listed token's bit lies in LDS (32 KB), sums of 2^44-fold weights stay below 2^62
constexpr int MAX_K = 1024;

typedef unsigned long long u64;
typedef uint32_t u32v4_1 __attribute__((ext_vector_type(4), aligned(2)));   // a 16-byte vector at a 2-byte border

template <int TY> struct El;
template <> struct El<F32> {
    typedef float type;
    static constexpr int N = 4;                     // elements of a 16-byte vector
    static constexpr uint32_t LOWEST = 0xff800000u; // -inf in every element of a word
};
template <> struct El<BF16> {
    typedef uint16_t type;
    static constexpr int N = 8;
    static constexpr uint32_t LOWEST = 0xff80ff80u;
};
template <> struct El<F16> {
    typedef uint16_t type;
    static constexpr int N = 8;
    static constexpr uint32_t LOWEST = 0xfc00fc00u;
};

struct Vec {
    uint32_t d[4];
};

// The raw vector as if it were new: keeps the compiler from carrying every element's unpacked value from one pass over a register-held row to the next (two to
// four times the row's registers: spills)
__device__ __forceinline__ void forget(Vec &v) { asm volatile("" : "+v"(v.d[0]), "+v"(v.d[1]), "+v"(v.d[2]), "+v"(v.d[3])); }

__device__ __forceinline__ float half_value(uint32_t bits) { return __half2float(__ushort_as_half((unsigned short)bits)); }

// raw bits of element e / its value
template <int TY>
__device__ __forceinline__ uint32_t bits_of(const Vec &v, int e) {
    if (TY == F32) return v.d[e];
    return (e & 1) ? v.d[e >> 1] >> 16 : v.d[e >> 1] & 0xffffu;
}
template <int TY>
__device__ __forceinline__ float value_of_bits(uint32_t b) {
    if (TY == F32) return __uint_as_float(b);
    if (TY == BF16) return __uint_as_float(b << 16);
    return half_value(b);
}
template <int TY>
__device__ __forceinline__ float value_of(const Vec &v, int e) {
    if (TY == BF16) return (e & 1) ? __uint_as_float(v.d[e >> 1] & 0xffff0000u) : __uint_as_float(v.d[e >> 1] << 16);
    return value_of_bits<TY>(bits_of<TY>(v, e));
}

// fp32 -> the type's bits, round to nearest even
template <int TY>
__device__ __forceinline__ uint32_t to_bits(float x) {
    if (TY == F32) return __float_as_uint(x);
    if (TY == BF16) {
        const __bf16 r = (__bf16)x;
        return (uint32_t)__builtin_bit_cast(uint16_t, r);
    }
    return (uint32_t)__half_as_ushort(__float2half_rn(x));
}

// The order of a row: a key that grows with the value as an unsigned number; -0 and +0 the same, every NaN above +inf.  16 bits for the 16-bit types.
template <int TY>
__device__ __forceinline__ uint32_t key_of_bits(uint32_t b) {
    if (TY == F32) {
        if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
        if (b == 0x80000000u) b = 0;
        return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
    }
    const uint32_t inf = TY == BF16 ? 0x7f80u : 0x7c00u;
    if ((b & 0x7fffu) > inf) return 0xffffu;
    if (b == 0x8000u) b = 0;
    return b ^ ((b >> 15) ? 0xffffu : 0x8000u);
}
template <int TY>
__device__ __forceinline__ uint32_t key_of(const Vec &v, int e) { return key_of_bits<TY>(bits_of<TY>(v, e)); }
template <int TY>
__device__ __forceinline__ float value_of_key(uint32_t k) {   // (the NaN key gives a NaN)
    if (TY == F32) return __uint_as_float((k >> 31) ? k ^ 0x80000000u : ~k);
    return value_of_bits<TY>(((k >> 15) ? k ^ 0x8000u : ~k) & 0xffffu);
}
template <int TY> __device__ __forceinline__ uint32_t key_top() { return TY == F32 ? 0xffffffffu : 0xffffu; }
template <int TY> __device__ __forceinline__ uint32_t key_inf() { return TY == F32 ? 0xff800000u : TY == BF16 ? 0xff80u : 0xfc00u; }
template <int TY> __host__ __device__ constexpr uint32_t key_ninf() { return TY == F32 ? 0x007fffffu : TY == BF16 ? 0x007fu : 0x03ffu; }
template <int TY> constexpr int key_bits() { return TY == F32 ? 32 : 16; }

// larger composite = earlier in the order: by key, then by the lower index
__device__ __forceinline__ u64 composite(uint32_t key, int index) { return ((u64)key << 32) | (uint32_t)~(uint32_t)index; }
__device__ __forceinline__ int index_of(u64 c) { return (int)~(uint32_t)c; }
__device__ __forceinline__ uint32_t key_of(u64 c) { return (uint32_t)(c >> 32); }

template <int TY>
__device__ __forceinline__ const char *row_at(const void *base, long long row, long long stride) {
    return static_cast<const char *>(base) + row * stride * (long long)sizeof(typename El<TY>::type);
}
template <int TY>
__device__ __forceinline__ uint32_t load_bits(const char *row, int i) {
    return (uint32_t)reinterpret_cast<const typename El<TY>::type *>(row)[i];
}
template <>
__device__ __forceinline__ uint32_t load_bits<F32>(const char *row, int i) {
    return reinterpret_cast<const uint32_t *>(row)[i];
}

// vector i of a row: elements behind the row's end are -inf.  LAST: nobody reads the row again
template <int TY, bool LAST = false>
__device__ __forceinline__ Vec load_vec(const char *row, int i, int vocab) {
    Vec v;
    constexpr int N = El<TY>::N;
    if ((i + 1) * N <= vocab) {
        const u32v4_1 *at = reinterpret_cast<const u32v4_1 *>(row + 16ll * i), r = LAST ? __builtin_nontemporal_load(at) : *at;
        v.d[0] = r[0];
        v.d[1] = r[1];
        v.d[2] = r[2];
        v.d[3] = r[3];
        return v;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) v.d[q] = El<TY>::LOWEST;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        if (i * N + e < vocab) {
            const uint32_t b = load_bits<TY>(row, i * N + e);
            if (TY == F32)
                v.d[e] = b;
            else
                v.d[e >> 1] = (e & 1) ? (v.d[e >> 1] & 0xffffu) | (b << 16) : (v.d[e >> 1] & 0xffff0000u) | b;
        }
    }
    return v;
}

// The elements of a workgroup's row: NV > 0 vectors a thread in registers (vector q NT + tid of the row; those behind the row's end are -inf), read once; NV = 0: read
// again by every pass, four vectors ahead.  SHORT: the row may be much shorter than NV vectors a thread.
template <int TY, int NT, int NV, bool SHORT = false>
struct RowIn {
    Vec v[NV > 0 ? NV : 1];
    const char *row;
    int vocab, nvec;
    __device__ __forceinline__ RowIn(const char *row_, int vocab_) : row(row_), vocab(vocab_), nvec((vocab_ + El<TY>::N - 1) / El<TY>::N) {
#pragma unroll
        for (int q = 0; q < NV; ++q) v[q] = get(q * NT + (int)threadIdx.x);
    }
    __device__ __forceinline__ Vec get(int i) const {
        return i < nvec ? load_vec<TY>(row, i, vocab) : Vec{{El<TY>::LOWEST, El<TY>::LOWEST, El<TY>::LOWEST, El<TY>::LOWEST}};
    }
    template <class F>
    __device__ __forceinline__ void each(F f) {       // f(vector, its number)
        if (NV > 0) {
#pragma unroll
            for (int q = 0; q < NV; ++q) {
                if (SHORT && q * NT >= nvec) continue;
                forget(v[q]);
                f(v[q], q * NT + (int)threadIdx.x);
            }
        } else {
            for (int first = threadIdx.x; first < nvec; first += 4 * NT) {
                Vec w[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) w[q] = get(first + q * NT);
#pragma unroll
                for (int q = 0; q < 4; ++q) f(w[q], first + q * NT);
            }
        }
    }
};

// NaN if either is
__device__ __forceinline__ float maximum(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// ---- exp(d / T) of d = x - m <= 0 (or -inf, or NaN): 2^(d c), c = log2(e) / T ----
// c in one fp32 number is off by the same share for every element of a row -- 1.3e-8 at T = 1, 3e-8 at most --, which moves the row's sum by that share of its mean exponent
// (5e-8 over 50,000 tokens, three times what the sum's rounding leaves).  So c = hi + lo, hi rounded towards 0: lo > 0 keeps -inf times both -inf.  d c is rounded once: a weight
// is off by |d c| / 2 steps of 2^-24, of either sign from element to element (a second fp32 number for the rounding, eight instructions instead of four, left the losses' errors at
// 2.1e-8 of themselves and brought the gradients' from 3.3e-8 to 3.0e-8, 50,001 fp32 tokens at T = 1; a forward of 2,048 x 50,001 went from 77 to 80 us).
struct Exponent {
    float hi, lo;
    float one;      // the nearest, where the weight itself is rounded to 16 bits
};
inline Exponent exponent_of(double temperature) {
    const double c = 1.4426950408889634 / temperature;
    float hi = (float)c;
    if ((double)hi > c) hi = nextafterf(hi, 0.f);
    return Exponent{hi, fmaxf((float)(c - (double)hi), 1.17549435e-38f), (float)c};
}
__device__ __forceinline__ float weight_of(float d, const Exponent &c) { return __builtin_amdgcn_exp2f(fmaf(d, c.hi, d * c.lo)); }
// The weights of a vector's elements against m, added up: two or three fp32 roundings of half a step, of either sign; the vectors are summed in 64 bits
template <int TY>
__device__ __forceinline__ double weights_of(const Vec &v, float m, const Exponent &c) {
    constexpr int N = El<TY>::N;
    float w[N];
#pragma unroll
    for (int e = 0; e < N; ++e) w[e] = weight_of(value_of<TY>(v, e) - m, c);
#pragma unroll
    for (int n = N / 2; n >= 1; n >>= 1)
#pragma unroll
        for (int e = 0; e < n; ++e) w[e] += w[e + n];
    return (double)w[0];
}

// 2^t in 64 bits, |t| up to 1100: the nearest power of two times the exponential's series to the 11th power, off by 6e-15 of itself at most
__device__ __forceinline__ double exp2_of(double t) {
    const double n = rint(t), f = (t - n) * 0.69314718055994530942;
    double p = 2.505210838544172e-8;
    p = fma(p, f, 2.755731922398589e-7);
    p = fma(p, f, 2.7557319223985893e-6);
    p = fma(p, f, 2.48015873015873e-5);
    p = fma(p, f, 1.984126984126984e-4);
    p = fma(p, f, 1.3888888888888889e-3);
    p = fma(p, f, 8.333333333333333e-3);
    p = fma(p, f, 4.1666666666666664e-2);
    p = fma(p, f, 0.16666666666666666);
    p = fma(p, f, 0.5);
    p = fma(p, f, 1.0);
    p = fma(p, f, 1.0);
    return ldexp(p, (int)n);
}
__device__ __forceinline__ double exp_of(double d) {      // e^d
    const double t = d * 1.4426950408889634;
    return exp2_of(t < -1100.0 ? -1100.0 : t > 1100.0 ? 1100.0 : t);      // (NaN stays)
}

// the largest element of a vector, NaN if there is one
template <int TY>
__device__ __forceinline__ float largest(const Vec &v) {
    float m = value_of<TY>(v, 0);
#pragma unroll
    for (int e = 1; e < El<TY>::N; ++e) m = maximum(m, value_of<TY>(v, e));
    return m;
}
struct MaxNan {
    __device__ static float of(float a, float b) { return maximum(a, b); }
};

// vector i of a gradient row from fp32 values; past the caches, which hold the rows that are still to be read (2,048 rows of 131,072 bf16, loss and gradient: 315 -> 279 us,
// 263 with the second read of a row as its last, 254 with its listed tokens' weights taken once)
template <int TY>
__device__ __forceinline__ void store_vec(char *row, int i, int vocab, const float *x) {
    constexpr int N = El<TY>::N;
    if ((i + 1) * N <= vocab) {
        u32v4_1 r;
        if (TY == F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e) r[e] = __float_as_uint(x[e]);
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) r[q] = to_bits<TY>(x[2 * q]) | (to_bits<TY>(x[2 * q + 1]) << 16);
        }
        __builtin_nontemporal_store(r, reinterpret_cast<u32v4_1 *>(row + 16ll * i));
        return;
    }
#pragma unroll
    for (int e = 0; e < N; ++e)
        if (i * N + e < vocab) reinterpret_cast<typename El<TY>::type *>(row)[i * N + e] = __builtin_bit_cast(typename El<TY>::type, (typename El<TY>::type)to_bits<TY>(x[e]));
}
template <>
__device__ __forceinline__ void store_vec<F32>(char *row, int i, int vocab, const float *x) {
    if ((i + 1) * 4 <= vocab) {
        u32v4_1 r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = __float_as_uint(x[e]);
        __builtin_nontemporal_store(r, reinterpret_cast<u32v4_1 *>(row + 16ll * i));
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (i * 4 + e < vocab) reinterpret_cast<float *>(row)[i * 4 + e] = x[e];
}

// ---- reductions: over a wave by butterflies, over a block through LDS; every lane gets the result, sums in one fixed order ----
struct MaxF {
    __device__ static float of(float a, float b) { return fmaxf(a, b); }
};
struct MaxU {
    template <class T> __device__ static T of(T a, T b) { return a > b ? a : b; }
};
struct MinU {
    template <class T> __device__ static T of(T a, T b) { return a < b ? a : b; }
};
struct Or {
    template <class T> __device__ static T of(T a, T b) { return a | b; }
};
struct Sum {
    template <class T> __device__ static T of(T a, T b) { return a + b; }
};
// The value of lane ^ S.  Within a row of 16 lanes by DPP moves, which cost a vector instruction and no trip through the LDS pipe that a CU's waves share (16,384 rows of 48:
// top_logits 14.4 -> 12.9 us, sample_logits 16.6 -> 16.0 us); across rows by __shfl_xor.
template <int S>
__device__ __forceinline__ uint32_t lane_xor_word(uint32_t v) {
#define MUCON_DPP(x, ctrl) (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(x), ctrl, 0xf, 0xf, true)
    if constexpr (S == 1) return MUCON_DPP(v, 0xB1);                          // quad_perm [1,0,3,2]
    else if constexpr (S == 2) return MUCON_DPP(v, 0x4E);                     // quad_perm [2,3,0,1]
    else if constexpr (S == 4) return MUCON_DPP(MUCON_DPP(v, 0x141), 0x1B);   // row_half_mirror (^ 7), quad_perm [3,2,1,0] (^ 3)
    else if constexpr (S == 8) return MUCON_DPP(v, 0x128);                    // row_ror:8
    else return (uint32_t)__shfl_xor((int)v, S);
#undef MUCON_DPP
}
template <int S, class T>
__device__ __forceinline__ T lane_xor(T v) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, lane_xor_word<S>(__builtin_bit_cast(uint32_t, v)));
    } else {
        const u64 b = __builtin_bit_cast(u64, v);
        return __builtin_bit_cast(T, (u64)lane_xor_word<S>((uint32_t)b) | (u64)lane_xor_word<S>((uint32_t)(b >> 32)) << 32);
    }
}
template <class OP, class T>
__device__ __forceinline__ T wave_reduce(T v) {
    v = OP::of(v, lane_xor<32>(v));
    v = OP::of(v, lane_xor<16>(v));
    v = OP::of(v, lane_xor<8>(v));
    v = OP::of(v, lane_xor<4>(v));
    v = OP::of(v, lane_xor<2>(v));
    return OP::of(v, lane_xor<1>(v));
}
// scratch: one value a wave; two barriers, the first frees scratch of an earlier use
template <int NT, class OP, class T>
__device__ __forceinline__ T block_reduce(T v, T *scratch) {
    v = wave_reduce<OP>(v);
    if (NT == 64) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    T r = scratch[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) r = OP::of(r, scratch[w]);
    return r;
}
// exclusive prefix sum over the block's threads, and the total
template <int NT, class T>
__device__ __forceinline__ T block_scan(T v, T *scratch, T *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    T inc = v;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const T o = __shfl_up(inc, s);
        if (lane >= s) inc = inc + o;
    }
    __syncthreads();
    if (lane == 63) scratch[wave] = inc;
    __syncthreads();
    T before = T(0), all = T(0);
    for (int w = 0; w < NT / 64; ++w) {
        if (w < wave) before = before + scratch[w];
        all = all + scratch[w];
    }
    *total = all;
    const T up = __shfl_up(inc, 1);
    return lane ? before + up : before;
}

}  // namespace rows
