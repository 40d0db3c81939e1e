// Shared by the kernels of a model's head and training step (layer_norm.hip, log_probs.hip, fp8_matmul.hip, adamw.hip): element types,
// 16-byte accesses at any element alignment, wave reductions, power-of-two block scales.
#pragma once
#include "w2c_common.h"
#include <type_traits>

// element types of the C ABI
enum { W2C_F32 = 0, W2C_BF16 = 1, W2C_F16 = 2 };

namespace {

struct bf16_t { uint16_t b; };
struct f16_t { _Float16 h; };
template <typename T> struct ElemOf;
template <> struct ElemOf<float> { static constexpr int VEC = 4; };
template <> struct ElemOf<bf16_t> { static constexpr int VEC = 8; };
template <> struct ElemOf<f16_t> { static constexpr int VEC = 8; };

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16_t x) { return bf16_to_f32(x.b); }
__device__ __forceinline__ float to_f32(f16_t x) { return (float)x.h; }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ bf16_t from_f32<bf16_t>(float x) { return bf16_t{f32_to_bf16(x)}; }
template <> __device__ __forceinline__ f16_t from_f32<f16_t>(float x) { return f16_t{(_Float16)x}; }

// N consecutive elements with the alignment of ONE element: rows of odd length and views into a row start anywhere, and this part's
// global accesses of 16 bytes need no more than that.  (Split over two cache lines such an access costs one more request, no more.)
template <typename T, int N> struct __attribute__((packed)) Pack { T v[N]; };
template <typename T, int N> using PackAt = Pack<T, N> __attribute__((aligned(sizeof(T))));

template <typename T, int N>
__device__ __forceinline__ void load_n(const T* __restrict__ p, float (&v)[N]) {
    PackAt<T, N> t;
    __builtin_memcpy(&t, p, sizeof(t));
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = to_f32(t.v[i]);
}
template <typename T, int N>
__device__ __forceinline__ void store_n(T* __restrict__ p, const float (&v)[N]) {
    PackAt<T, N> t;
#pragma unroll
    for (int i = 0; i < N; ++i) t.v[i] = from_f32<T>(v[i]);
    __builtin_memcpy(p, &t, sizeof(t));
}
// the same, of which only the first `n` elements exist (n <= 0: none; absent ones read as `fill`)
template <typename T, int N>
__device__ __forceinline__ void load_part(const T* __restrict__ p, long long n, float (&v)[N], float fill = 0.f) {
    if (n >= N) load_n<T, N>(p, v);
    else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < n ? to_f32(p[i]) : fill;
    }
}
template <typename T, int N>
__device__ __forceinline__ void store_part(T* __restrict__ p, long long n, const float (&v)[N]) {
    if (n >= N) store_n<T, N>(p, v);
    else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < n) p[i] = from_f32<T>(v[i]);
    }
}

// the same for the elements [lo, hi) of an access that starts at c, before, in or behind them
template <typename T, int N>
__device__ __forceinline__ void load_range(const T* __restrict__ p, int c, int lo, int hi, float (&v)[N], float fill) {
    if (c >= lo && c + N <= hi) load_n<T, N>(p + c, v);
    else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = c + i >= lo && c + i < hi ? to_f32(p[c + i]) : fill;
    }
}
template <typename T, int N>
__device__ __forceinline__ void store_range(T* __restrict__ p, int c, int lo, int hi, const float (&v)[N]) {
    if (c >= lo && c + N <= hi) store_n<T, N>(p + c, v);
    else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (c + i >= lo && c + i < hi) p[c + i] = from_f32<T>(v[i]);
    }
}
// elements from the 16-byte boundary at or below p to p: accesses that start that much earlier are aligned (a row of odd length starts anywhere,
// and an access across two cache lines costs a second request: 4 096 rows of 50 257 bf16 read at 4.3 TB/s as they lie, 5.0 aligned)
template <typename T>
__device__ __forceinline__ int misaligned(const T* p) {
    return (int)(reinterpret_cast<uintptr_t>(p) & 15) / (int)sizeof(T);
}

// a 16-byte access kept as it came, so that several can be in flight before the first is widened
template <typename T>
__device__ __forceinline__ u32x4_t load_raw(const T* __restrict__ p) {
    PackAt<T, ElemOf<T>::VEC> t;
    __builtin_memcpy(&t, p, sizeof(t));
    return __builtin_bit_cast(u32x4_t, t);
}
// ... of which only the first n elements exist; the absent ones are `fill`
template <typename T>
__device__ __forceinline__ u32x4_t load_raw_part(const T* __restrict__ p, long long n, float fill = 0.f) {
    constexpr int VEC = ElemOf<T>::VEC;
    if (n >= VEC) return load_raw<T>(p);
    Pack<T, VEC> t;
#pragma unroll
    for (int i = 0; i < VEC; ++i) t.v[i] = i < n ? p[i] : from_f32<T>(fill);
    return __builtin_bit_cast(u32x4_t, t);
}
// ... the elements [lo, hi) of an access that starts at c, before, in or behind them
template <typename T>
__device__ __forceinline__ u32x4_t load_raw_range(const T* __restrict__ p, int c, int lo, int hi, float fill) {
    constexpr int VEC = ElemOf<T>::VEC;
    if (c >= lo && c + VEC <= hi) return load_raw<T>(p + c);
    Pack<T, VEC> t;
#pragma unroll
    for (int i = 0; i < VEC; ++i) t.v[i] = c + i >= lo && c + i < hi ? p[c + i] : from_f32<T>(fill);
    return __builtin_bit_cast(u32x4_t, t);
}
template <typename T>
__device__ __forceinline__ void widen(u32x4_t r, float (&v)[ElemOf<T>::VEC]) {
    const Pack<T, ElemOf<T>::VEC> t = __builtin_bit_cast(Pack<T, ElemOf<T>::VEC>, r);
#pragma unroll
    for (int i = 0; i < ElemOf<T>::VEC; ++i) v[i] = to_f32(t.v[i]);
}

// Reductions over a wave whose 64 lanes are all active, by DPP moves in the vector unit (a shuffle is a trip through the LDS crossbar, some 60 cycles a
// step): four row shifts, then the rows' last lanes handed on to the next rows.  Lane 63 has the result; every lane gets it.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp(uint32_t absent, uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)absent, (int)v, CTRL, ROWS, 0xF, false);
}
template <typename F>
__device__ __forceinline__ uint32_t wave_reduce(uint32_t v, F step) {
    v = step(v, std::integral_constant<int, 0x111>(), std::integral_constant<int, 0xF>());       // row_shr 1, 2, 4, 8
    v = step(v, std::integral_constant<int, 0x112>(), std::integral_constant<int, 0xF>());
    v = step(v, std::integral_constant<int, 0x114>(), std::integral_constant<int, 0xF>());
    v = step(v, std::integral_constant<int, 0x118>(), std::integral_constant<int, 0xF>());
    v = step(v, std::integral_constant<int, 0x142>(), std::integral_constant<int, 0xA>());       // lane 15 of a row to rows 1 and 3
    v = step(v, std::integral_constant<int, 0x143>(), std::integral_constant<int, 0xC>());       // lane 31 to rows 2 and 3
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ float wave_sum(float v) {
    return __uint_as_float(wave_reduce(__float_as_uint(v), [](uint32_t a, auto ctrl, auto rows) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(dpp<decltype(ctrl)::value, decltype(rows)::value>(0u, a)));
    }));
}
__device__ __forceinline__ float wave_max(float v) {
    return __uint_as_float(wave_reduce(__float_as_uint(v), [](uint32_t a, auto ctrl, auto rows) {
        return __float_as_uint(__builtin_fmaxf(__uint_as_float(a), __uint_as_float(dpp<decltype(ctrl)::value, decltype(rows)::value>(a, a))));
    }));
}

// A launch counts the work-items of a dimension in 32 bits: the most blocks of so many threads.
constexpr long long most_blocks(int threads) { return 0xFFFFFFFFll / threads; }

// Block scales are powers of two, held as a biased exponent byte (e8m0: value 2^(b - 127), 255 = NaN): the matrix instructions take them as
// they are, and scaling by one is exact.  The scale of a block is the smallest 2^e with amax <= TOP * 2^e, by the fields of the two
// floats; a block of zeros has 2^0.  amax has to be finite and >= 0.
constexpr float FP8_TOP = 448.f;                    // largest e4m3 value, 1.75 * 2^8
__device__ __forceinline__ int scale_exponent(float amax) {
    const uint32_t b = __float_as_uint(amax), t = __float_as_uint(FP8_TOP);
    const int e = (int)(b >> 23) - (int)(t >> 23) + ((b & 0x7FFFFFu) > (t & 0x7FFFFFu) ? 1 : 0);
    return amax > 0.f ? (e < -127 ? -127 : e) : 0;
}
__device__ __forceinline__ float pow2f(int e) {      // 2^e for -149 <= e <= 127 (e = -127 and below are subnormal)
    return e >= -126 ? __uint_as_float((uint32_t)(e + 127) << 23) : __uint_as_float(1u << (e + 149));
}

}  // namespace
