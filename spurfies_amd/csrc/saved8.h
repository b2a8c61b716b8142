// Device helpers of the training operators that keep their saved activations in 8 bits: element types, unaligned 16-byte row accesses, the 8-bit block
// format, and sums over the lanes of a row.
//
// Block format (include/spurfies_hip.h: spf_saved8_*): 32 consecutive columns share a step 2^s, kept as the byte s + 127; an element is a magnitude in
// steps (7 bits, round to nearest even) and a top bit that is set where the element is not greater than zero.  Powers of two keep both directions
// exact but for the one rounding, so the bytes do not depend on who computes them.  Sign and magnitude instead of two's complement: a derivative
// that depends on the element's sign alone (LeakyReLU) stays exact for elements that round to zero steps.
#pragma once
#include "common.h"

namespace spf {

constexpr int S8_BLOCK = 32;

template <int TYPE> struct elem_of;
template <> struct elem_of<SPF_TYPE_F32> { using type = float; };
template <> struct elem_of<SPF_TYPE_BF16> { using type = __bf16; };
template <> struct elem_of<SPF_TYPE_F16> { using type = _Float16; };

// 16 bytes of a row, from any address that an element may have (the hardware takes unaligned vector accesses; as copies, so that the compiler knows the
// alignment is the element's — an `aligned` attribute of a dependent vector type is dropped, and a scalar load then ignores the address's low bits)
template <typename T> constexpr int VEC = 16 / (int)sizeof(T);
template <typename T> using vec_t = T __attribute__((ext_vector_type(16 / sizeof(T))));
template <typename T> __device__ __forceinline__ vec_t<T> load_any(const T* p) {
    vec_t<T> v;
    __builtin_memcpy(&v, p, sizeof v);
    return v;
}
template <typename T> __device__ __forceinline__ void store_any(T* p, vec_t<T> v) { __builtin_memcpy(p, &v, sizeof v); }

// n valid elements from p on (n >= VEC: all), the others zero.  before: there is a vector's worth of the row in front of p.  Then a cut vector of a 16-bit type is
// one load that ends where the row does, shifted: up to seven single elements would each wait for the one before, in every row (layer norm of 20000 x 2500 bf16,
// forward and backward: 199 us by elements, 166 so; with a single element left, 200000 x 257, it is 215 against 220).  In fp32 the at most three elements are the
// cheaper way (7000 x 8191: 229 us, 259 shifted).
template <typename T> __device__ __forceinline__ vec_t<T> load_vec(const T* p, long long n, bool before = false) {
    vec_t<T> v = {};
    if (n >= VEC<T>) {
        v = load_any(p);
    } else if (sizeof(T) == 2 && before) {
        if (n > 0) {
            const vec_t<T> w = load_any(p + n - VEC<T>);
            v = __builtin_bit_cast(vec_t<T>, __builtin_bit_cast(unsigned __int128, w) >> (8 * (int)sizeof(T) * (VEC<T> - (int)n)));
        }
    } else {
#pragma unroll
        for (int i = 0; i < VEC<T>; ++i)
            if (i < n) v[i] = p[i];
    }
    return v;
}
template <typename T> __device__ __forceinline__ void store_vec(T* p, vec_t<T> v, long long n) {
    if (n >= VEC<T>) {
        store_any(p, v);
    } else {
#pragma unroll
        for (int i = 0; i < VEC<T>; ++i)
            if (i < n) p[i] = v[i];
    }
}
template <typename T, int N> __device__ __forceinline__ void to_f32(vec_t<T> v, float (&f)[N]) {
    static_assert(N == VEC<T>, "one vector");
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = (float)v[i];
}
template <typename T, int N> __device__ __forceinline__ vec_t<T> from_f32(const float (&f)[N]) {
    static_assert(N == VEC<T>, "one vector");
    vec_t<T> v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (T)f[i];          // round to nearest even
    return v;
}

// ---- lanes ------------------------------------------------------------------------------------------------------------------------------
// Cross-lane moves of the vector pipe (no LDS): partner lane ^ 1, ^ 2, the other quad of 8, the other half of 16.  All 64 lanes must be active.
template <int CTRL> __device__ __forceinline__ uint32_t dpp(uint32_t v) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true); }
constexpr int DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E, DPP_HALF_MIRROR = 0x141, DPP_MIRROR = 0x140;

// largest value over the G = 4 or 8 lanes of a 32-column block
template <int G> __device__ __forceinline__ uint32_t block_max(uint32_t v) {
    v = max(v, dpp<DPP_XOR1>(v));
    v = max(v, dpp<DPP_XOR2>(v));
    if (G == 8) v = max(v, dpp<DPP_HALF_MIRROR>(v));
    return v;
}
// sum over groups of L = 8 .. 64 lanes, the same in every lane of a group
template <int L> __device__ __forceinline__ float lane_sum(float v) {
    v += __uint_as_float(dpp<DPP_XOR1>(__float_as_uint(v)));
    v += __uint_as_float(dpp<DPP_XOR2>(__float_as_uint(v)));
    v += __uint_as_float(dpp<DPP_HALF_MIRROR>(__float_as_uint(v)));
    if (L >= 16) v += __uint_as_float(dpp<DPP_MIRROR>(__float_as_uint(v)));
    if (L >= 32) {
        const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
    }
    if (L >= 64) {
        const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
    }
    return v;
}

// ---- 8-bit blocks -----------------------------------------------------------------------------------------------------------------------
// f: this lane's N = 4 or 8 elements of a block whose other elements are in the 32 / N - 1 neighbouring lanes (columns behind the row's end: 0).
// -> w: the bytes, four a word; the return value is the block's step byte (the same in all of its lanes).
template <int N> __device__ __forceinline__ uint32_t s8_pack(const float (&f)[N], uint32_t (&w)[N / 4]) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);         // as integers: NaN > infinity > every finite magnitude
    top = block_max<S8_BLOCK / N>(top);
    // The least s with round(top / 2^s) <= 127: top's exponent - 6, one more if its mantissa is 127.5 / 64 or larger — the carry of adding
    // 2^-7 of the leading bit.  The last 2^-7 of the fp32 range would need s = 122 and stand for infinity: it keeps s = 121 and 127 steps.
    int e = (int)((top + 0x10000u) >> 23) - 6;
    e = min(max(e, 1), 248);
    const bool bad = top >= 0x7f800000u;
    const float inv = __uint_as_float((uint32_t)(254 - e) << 23);                             // 2^-s, exact
#pragma unroll
    for (int q = 0; q < N / 4; ++q) {
        uint32_t m[4], n[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float v = f[4 * q + i];
            // 2^23 + |v| / 2^s rounds to a whole number, ties to even, in the low bits (the product is exact)
            m[i] = __float_as_uint(fminf(__builtin_fmaf(fabsf(v), inv, 8388608.0f), 8388608.0f + 127.0f));
            n[i] = v > 0.f ? 0u : 0x80000000u;                                                // top bit: not greater than zero (as a NaN is not)
        }
        const uint32_t mag = __builtin_amdgcn_perm(__builtin_amdgcn_perm(m[3], m[2], 0x0c0c0400u), __builtin_amdgcn_perm(m[1], m[0], 0x0c0c0400u), 0x05040100u);
        const uint32_t sgn = __builtin_amdgcn_perm(__builtin_amdgcn_perm(n[3], n[2], 0x0c0c0703u), __builtin_amdgcn_perm(n[1], n[0], 0x0c0c0703u), 0x05040100u);
        // a block with an infinity or a NaN: zero magnitudes (what it stands for is NaN)
        w[q] = ((bad ? 0u : mag) & 0x7f7f7f7fu) | (sgn & 0x80808080u);
    }
    return bad ? 255u : (uint32_t)e;
}
// columns behind the row's end are zero bytes
template <int N> __device__ __forceinline__ void s8_mask(uint32_t (&w)[N / 4], long long n) {
    if (n >= N) return;
#pragma unroll
    for (int q = 0; q < N / 4; ++q) {
        const int k = (int)(n < 0 ? 0 : n) - 4 * q;
        w[q] &= k >= 4 ? 0xffffffffu : k <= 0 ? 0u : (1u << (8 * k)) - 1u;
    }
}
__device__ __forceinline__ float s8_step(uint32_t byte) { return byte == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23); }
// The magnitudes of a word's bytes.  The conversions take any byte of a register, if the compiler is kept from folding the mask into a bit-field extract for each.
__device__ __forceinline__ void s8_magnitudes(uint32_t w, float (&m)[4]) {
    uint32_t mag = w & 0x7f7f7f7fu;
    asm("" : "+v"(mag));
    m[0] = (float)(mag & 0xffu);
    m[1] = (float)((mag >> 8) & 0xffu);
    m[2] = (float)((mag >> 16) & 0xffu);
    m[3] = (float)(mag >> 24);
}
template <int N> __device__ __forceinline__ void s8_unpack(const uint32_t (&w)[N / 4], float step, float (&f)[N]) {
#pragma unroll
    for (int q = 0; q < N / 4; ++q) {
        float m[4];
        s8_magnitudes(w[q], m);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[4 * q + i] = __uint_as_float(__float_as_uint(m[i] * step) | ((w[q] << (24 - 8 * i)) & 0x80000000u));
    }
}
template <int N> __device__ __forceinline__ void s8_store(uint8_t* codes, size_t at, const uint32_t (&w)[N / 4]) {
    if (N == 4) {
        *reinterpret_cast<uint32_t*>(codes + at) = w[0];
    } else {
        *reinterpret_cast<uint2*>(codes + at) = make_uint2(w[0], w[N / 4 - 1]);
    }
}
template <int N> __device__ __forceinline__ void s8_load(const uint8_t* codes, size_t at, uint32_t (&w)[N / 4]) {
    if (N == 4) {
        w[0] = *reinterpret_cast<const uint32_t*>(codes + at);
    } else {
        const uint2 v = *reinterpret_cast<const uint2*>(codes + at);
        w[0] = v.x, w[N / 4 - 1] = v.y;
    }
}

// row = n / d for 0 <= n < 2^31 by one multiplication (d fixed for a launch): n / d = (mulhi(n, mul) + n) >> shift (Granlund & Montgomery, Division by invariant
// integers using multiplication, 1994)
struct fast_div {
    uint32_t d, mul, shift;
    fast_div() = default;
    explicit fast_div(uint32_t div) : d(div), mul(0), shift(0) {
        while ((1ull << shift) < d) ++shift;
        mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
};

inline int type_size(int type) { return type == SPF_TYPE_F32 ? 4 : 2; }
inline bool type_ok(int type) { return type == SPF_TYPE_F32 || type == SPF_TYPE_BF16 || type == SPF_TYPE_F16; }

}  // namespace spf
