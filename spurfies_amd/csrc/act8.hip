// Saved activations in 8 bits: written, restored, and read by the backward pass of an activation function.
//
//   spf_saved8_pack / spf_saved8_restore     x <-> {bytes, step bytes}                                  (format: saved8.h)
//   spf_act8_forward                         y = f(x) and, in the same pass, the bytes of x (the smooth functions) and of y (the next layer's input)
//   spf_act8_backward                        dx = dy * f'(restored)
//
// One kernel each way: a pass over rows of 32-column blocks, 16 bytes of x a lane, so 8 (fp32) or 4 (16-bit types) lanes share a block and find its
// largest magnitude with two or three moves of the vector pipe — no LDS, no second read.  Bound by HBM; the arithmetic (about 8 vector instructions
// an element for the bytes, 17 for GELU in 16 bits, 40 in fp32) stays under the loads of other waves, but for softplus' logarithm.  Each thread has four blocks in flight.
// Measured on MI355X (medians): 389017 x 256 fp32, LeakyReLU, 152 us forward and 168 back (5.9 and 5.4 TB/s); 16384 x 8192 bf16, GELU, 119 and 150 (5.7 and 4.5 TB/s; 139 and
// 192 with the library's erf and exp), fp32 211 and 220 (5.8 and 5.5 TB/s), softplus fp32 383 and 218; 389017 x 104 fp32 packed in 47 us and restored in 32.
#include <math.h>

#include "saved8.h"

namespace {
using namespace spf;

constexpr int KIND_NONE = -1;                // pack / restore only
constexpr int UNROLL = 4;

struct rows8 {                               // the blocks of a matrix, numbered along its rows
    uint32_t n_blocks;
    fast_div per_row;
    long long cols;
};

// What follows comes in two forms.  FINE, for fp32: errors of a few units of 2^-24 relative to the result, wherever that lies (such passes are bound by HBM with room
// for it).  The other, for 16-bit results: short, with relative errors of 2^-16 and less where half a step of the result is 2^-12 or more.

// e^-(x + lo) for x >= 0 and a small lo.  The hardware's 2^t takes a rounded t = -x log2 e, off by up to x / 2^24; FINE puts that back: e^-x = 2^t (1 + r ln 2) with
// t + r = -x log2 e.  Beyond x = 200 all of it is zero (the bound keeps infinities out of r).
template <bool FINE> __device__ __forceinline__ float exp_neg(float x, float lo) {
    constexpr float L = 1.44269504088896341f, L_LOW = 1.92596299e-8f, LN2 = 0.693147180559945309f;         // log2 e = L + L_LOW
    if (!FINE) return __builtin_amdgcn_exp2f(x * -L);
    lo = x < 200.f ? lo : 0.f;
    x = fminf(x, 200.f);
    const float t = x * -L;
    float r = __builtin_fmaf(x, -L, -t);
    r = __builtin_fmaf(x, -L_LOW, r);
    r = __builtin_fmaf(lo, -L, r);
    const float e = __builtin_amdgcn_exp2f(t);
    return __builtin_fmaf(e * LN2, r, e);
}
// 1 / d; FINE: with a step of Newton's
template <bool FINE> __device__ __forceinline__ float inverse(float d) {
    const float r = __builtin_amdgcn_rcpf(d);
    return FINE ? __builtin_fmaf(__builtin_fmaf(-d, r, 1.f), r, r) : r;
}
// 1 / (1 + e^-v), and 1 minus that.  FINE: from e^-|v|, which neither overflows nor cancels; lo: v's rounding.  (In 16 bits that form costs 3 - 4 % of SiLU's passes.)
template <bool FINE> __device__ __forceinline__ float sigmoid(float v, float lo, float& other) {
    if (!FINE) {
        const float s = inverse<false>(1.f + __builtin_amdgcn_exp2f(v * -1.44269504088896341f));
        other = 1.f - s;
        return s;
    }
    const float a = exp_neg<true>(fabsf(v), v > 0.f ? lo : -lo), r = inverse<true>(1.f + a), q = a * r;
    other = v > 0.f ? q : r;
    return v > 0.f ? r : q;
}
template <int N> __device__ __forceinline__ float polynomial(const float (&c)[N], float t) {
    float p = c[N - 1];
#pragma unroll
    for (int i = N - 2; i >= 0; --i) p = __builtin_fmaf(p, t, c[i]);
    return p;
}
// The normal distribution's P(Z < v), and e^(-v^2 / 2) beside it, which both GELU and its derivative need.  P(Z > x) = e^(-x^2 / 2) t P(t) for x >= 0, t = 1 / (1 + k x), P
// a polynomial fitted to least relative error over 0 .. 14, so that the far tail keeps its digits (an absolute error of 10^-7 is all of the result at -5): degree 8,
// 0.4 / 2^24, for fp32, degree 6, 15 / 2^24, for 16 bits.  fp32 within one of zero: 1/2 + v Q(v^2), where the tail's own roundings would show.
template <bool FINE> __device__ __forceinline__ float normal_cdf(float v, float& bell) {
    const float square = v * v;
    if (!FINE) {
        constexpr float P[] = {0.143713042f, 0.141772494f, 0.139719039f, 0.0265500005f, 0.180952981f, -0.179763913f, 0.0470560566f};
        bell = __builtin_amdgcn_exp2f(square * (-0.5f * 1.44269504088896341f));
        const float t = inverse<false>(__builtin_fmaf(fabsf(v), 0.36f, 1.f)), tail = t * polynomial(P, t) * bell;
        return v > 0.f ? 1.f - tail : tail;
    }
    constexpr float P[] = {0.103759058f, 0.103016756f, 0.103030212f, 0.0510278642f, 0.160947382f, -0.150948197f, 0.251490533f, -0.152828425f, 0.0305047948f};
    constexpr float Q[] = {0.398942292f, -0.0664903596f, 0.00997333135f, -0.00118635304f, 0.000113512659f, -7.66467929e-06f};
    bell = exp_neg<true>(0.5f * square, 0.5f * __builtin_fmaf(v, v, -square));
    const float t = inverse<true>(__builtin_fmaf(fminf(fabsf(v), 64.f), 0.26f, 1.f)), tail = t * polynomial(P, t) * bell;       // (64: infinities stay out of the inverse)
    const float far = v > 0.f ? 1.f - tail : tail;
    return square < 1.f ? __builtin_fmaf(v, polynomial(Q, square), 0.5f) : far;
}

template <int KIND, bool FINE> __device__ __forceinline__ float act(float v, float p, float ip) {
    if (KIND == SPF_ACT_LEAKY_RELU) return v > 0.f ? v : v * p;
    if (KIND == SPF_ACT_SOFTPLUS) {                                                // log(1 + e^z) / p = max(v, 0) + log(1 + e^-|z|) / p, z = p v
        const float z = v * p, lo = __builtin_fmaf(v, p, -z);
        return v != v ? v : fmaxf(v, 0.f) + log1pf(exp_neg<FINE>(fabsf(z), z > 0.f ? lo : -lo)) * ip;     // (fmaxf drops a NaN)
    }
    if (KIND == SPF_ACT_SILU) {
        float other;
        return v * sigmoid<FINE>(v, 0.f, other);
    }
    float bell;
    return v * normal_cdf<FINE>(v, bell);
}
// f'(v); LeakyReLU: from the sign of the restored value, which is the sign of the element (a restored NaN stays one)
template <int KIND, bool FINE> __device__ __forceinline__ float act_slope(float v, float p) {
    if (KIND == SPF_ACT_LEAKY_RELU) return v != v ? v : ((int)__float_as_uint(v) < 0 ? p : 1.f);
    float other;
    if (KIND == SPF_ACT_SOFTPLUS) {
        const float z = v * p, s = sigmoid<FINE>(z, __builtin_fmaf(v, p, -z), other);
        return v != v ? v : s;
    }
    if (KIND == SPF_ACT_SILU) {
        const float s = sigmoid<FINE>(v, 0.f, other);
        return s * (1.f + v * other);
    }
    float bell;
    const float cdf = normal_cdf<FINE>(v, bell);
    return cdf + v * bell * 0.39894228040143268f;
}

template <typename T, int KIND>
__global__ void __launch_bounds__(256)
act8_forward_kernel(const T* __restrict__ x, long long ldx, T* __restrict__ y, long long ldy, uint8_t* __restrict__ in_codes, uint8_t* __restrict__ in_steps,
                    uint8_t* __restrict__ out_codes, uint8_t* __restrict__ out_steps, rows8 m, float p, float ip) {
    constexpr int V = VEC<T>, G = S8_BLOCK / V, SWEEP = 256 / G;
    const int c = ((int)threadIdx.x % G) * V;
    const uint32_t first = blockIdx.x * (uint32_t)(SWEEP * UNROLL) + threadIdx.x / G;
    vec_t<T> raw[UNROLL];
    uint32_t row[UNROLL];
    long long col[UNROLL], left[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const uint32_t b = first + u * SWEEP;
        row[u] = m.per_row(b);
        col[u] = (long long)(b - row[u] * m.per_row.d) * S8_BLOCK + c;
        left[u] = b < m.n_blocks ? m.cols - col[u] : 0;
        raw[u] = load_vec(x + (long long)row[u] * ldx + col[u], left[u], col[u] > 0);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const uint32_t b = first + u * SWEEP;
        const bool ok = b < m.n_blocks;
        float f[V];
        uint32_t w[V / 4];
        to_f32<T>(raw[u], f);
        if (in_codes) {
            const uint32_t e = s8_pack(f, w);
            s8_mask<V>(w, left[u]);
            if (ok) s8_store<V>(in_codes, (size_t)b * S8_BLOCK + c, w);
            if (ok && c == 0) in_steps[b] = (uint8_t)e;
        }
        if (KIND != KIND_NONE) {
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = act<KIND, sizeof(T) == 4>(f[i], p, ip);
            const vec_t<T> out = from_f32<T>(f);
            store_vec(y + (long long)row[u] * ldy + col[u], out, left[u]);
            if (out_codes) {                                       // the bytes of y as the next layer sees it
                to_f32<T>(out, f);
#pragma unroll
                for (int i = 0; i < V; ++i) f[i] = i < left[u] ? f[i] : 0.f;
                const uint32_t e = s8_pack(f, w);
                s8_mask<V>(w, left[u]);
                if (ok) s8_store<V>(out_codes, (size_t)b * S8_BLOCK + c, w);
                if (ok && c == 0) out_steps[b] = (uint8_t)e;
            }
        }
    }
}

template <typename T, int KIND>
__global__ void __launch_bounds__(256)
act8_backward_kernel(const T* __restrict__ dy, long long ldy, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ steps, T* __restrict__ dx,
                     long long ldx, rows8 m, float p) {
    constexpr int V = VEC<T>, G = S8_BLOCK / V, SWEEP = 256 / G;
    const int c = ((int)threadIdx.x % G) * V;
    const uint32_t first = blockIdx.x * (uint32_t)(SWEEP * UNROLL) + threadIdx.x / G;
    vec_t<T> raw[UNROLL];
    uint32_t row[UNROLL], w[UNROLL][V / 4], e[UNROLL];
    long long col[UNROLL], left[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const uint32_t b = first + u * SWEEP;
        row[u] = m.per_row(b);
        col[u] = (long long)(b - row[u] * m.per_row.d) * S8_BLOCK + c;
        left[u] = b < m.n_blocks ? m.cols - col[u] : 0;
        if (left[u] > 0) {
            s8_load<V>(codes, (size_t)b * S8_BLOCK + c, w[u]);
            e[u] = steps[b];
            if (KIND != KIND_NONE) raw[u] = load_vec(dy + (long long)row[u] * ldy + col[u], left[u], col[u] > 0);
        }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        if (left[u] <= 0) continue;
        float f[V], g[V];
        s8_unpack<V>(w[u], s8_step(e[u]), f);
        if (KIND != KIND_NONE) {
            to_f32<T>(raw[u], g);
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = g[i] * act_slope<KIND, sizeof(T) == 4>(f[i], p);
        } else if (sizeof(T) == 2 && (float)(T)65504.f == 65504.f) {
            // fp16's largest numbers round up to 65536: the largest finite one stands for them (and for anything larger from a wider type)
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = fabsf(f[i]) > 65504.f ? copysignf(65504.f, f[i]) : f[i];
        }
        store_vec(dx + (long long)row[u] * ldx + col[u], from_f32<T>(f), left[u]);
    }
}

// rows of whole blocks that follow each other without a gap are one long row
rows8 blocks_of(int64_t rows, int64_t cols, bool dense) {
    const int64_t per_row = (cols + S8_BLOCK - 1) / S8_BLOCK;
    rows8 m;
    m.n_blocks = (uint32_t)(rows * per_row);
    m.per_row = fast_div(dense && cols % S8_BLOCK == 0 ? m.n_blocks : (uint32_t)per_row);
    m.cols = dense && cols % S8_BLOCK == 0 ? rows * cols : cols;
    return m;
}
// blocks are numbered in 31 bits, with room for a launch's overhang
const char* size_problem(int64_t rows, int64_t cols) {
    if (rows < 0 || cols < 0) return "negative size";
    if (rows > 0 && (cols + S8_BLOCK - 1) / S8_BLOCK > ((1ll << 31) - 1024) / rows) return "more than 2^31 - 1024 blocks of 32 columns";
    return nullptr;
}
bool misaligned(const void* p, int size) { return ((uintptr_t)p & (uintptr_t)(size - 1)) != 0; }

template <typename T, int KIND>
void launch_forward(const void* x, int64_t ldx, void* y, int64_t ldy, uint8_t* ic, uint8_t* is, uint8_t* oc, uint8_t* os, const rows8& m, float p, hipStream_t s) {
    const int sweep = 256 / (S8_BLOCK / VEC<T>) * UNROLL;
    act8_forward_kernel<T, KIND><<<div_up(m.n_blocks, sweep), 256, 0, s>>>((const T*)x, ldx, (T*)y, ldy, ic, is, oc, os, m, p, (float)(1.0 / (double)p));
}
template <typename T, int KIND>
void launch_backward(const void* dy, int64_t ldy, const uint8_t* c, const uint8_t* st, void* dx, int64_t ldx, const rows8& m, float p, hipStream_t s) {
    const int sweep = 256 / (S8_BLOCK / VEC<T>) * UNROLL;
    act8_backward_kernel<T, KIND><<<div_up(m.n_blocks, sweep), 256, 0, s>>>((const T*)dy, ldy, c, st, (T*)dx, ldx, m, p);
}

#define BY_KIND(FN, T, ...)                                                    \
    switch (kind) {                                                            \
        case SPF_ACT_LEAKY_RELU: FN<T, SPF_ACT_LEAKY_RELU>(__VA_ARGS__); break; \
        case SPF_ACT_SOFTPLUS: FN<T, SPF_ACT_SOFTPLUS>(__VA_ARGS__); break;    \
        case SPF_ACT_SILU: FN<T, SPF_ACT_SILU>(__VA_ARGS__); break;            \
        case SPF_ACT_GELU: FN<T, SPF_ACT_GELU>(__VA_ARGS__); break;            \
        default: FN<T, KIND_NONE>(__VA_ARGS__); break;                         \
    }
#define BY_TYPE(FN, ...)                                                       \
    if (type == SPF_TYPE_F32) {                                                \
        BY_KIND(FN, float, __VA_ARGS__)                                        \
    } else if (type == SPF_TYPE_BF16) {                                        \
        BY_KIND(FN, __bf16, __VA_ARGS__)                                       \
    } else {                                                                   \
        BY_KIND(FN, _Float16, __VA_ARGS__)                                     \
    }

int forward(const char* who, const void* x, int type, int64_t ldx, int64_t rows, int64_t cols, int kind, float p, void* y, int64_t ldy, uint8_t* ic, uint8_t* is,
            uint8_t* oc, uint8_t* os, void* stream) {
    if (!type_ok(type)) return fail(SPF_EINVAL, "%s: unknown element type %d", who, type);
    if (const char* why = size_problem(rows, cols)) return fail(SPF_EINVAL, "%s: %s", who, why);
    if (rows == 0 || cols == 0) return SPF_OK;
    if (!x || (kind != KIND_NONE && !y) || (!ic != !is) || (!oc != !os)) return fail(SPF_EINVAL, "%s: null pointer", who);
    if (ldx < 0 || (kind != KIND_NONE && ldy < cols)) return fail(SPF_EINVAL, "%s: row stride", who);
    if (misaligned(x, type_size(type)) || misaligned(y, type_size(type)) || misaligned(ic, 16) || misaligned(oc, 16)) return fail(SPF_EINVAL, "%s: misaligned pointer", who);
    const rows8 m = blocks_of(rows, cols, ldx == cols && (kind == KIND_NONE || ldy == cols));
    BY_TYPE(launch_forward, x, ldx, y, ldy, ic, is, oc, os, m, p, (hipStream_t)stream)
    SPF_LAUNCH_CHECK(who);
    return SPF_OK;
}
int backward(const char* who, const void* dy, int type, int64_t ldy, int64_t rows, int64_t cols, int kind, float p, const uint8_t* c, const uint8_t* st, void* dx,
             int64_t ldx, void* stream) {
    if (!type_ok(type)) return fail(SPF_EINVAL, "%s: unknown element type %d", who, type);
    if (const char* why = size_problem(rows, cols)) return fail(SPF_EINVAL, "%s: %s", who, why);
    if (rows == 0 || cols == 0) return SPF_OK;
    if (!c || !st || !dx || (kind != KIND_NONE && !dy)) return fail(SPF_EINVAL, "%s: null pointer", who);
    if (ldy < 0 || ldx < cols) return fail(SPF_EINVAL, "%s: row stride", who);
    if (misaligned(dy, type_size(type)) || misaligned(dx, type_size(type)) || misaligned(c, 16)) return fail(SPF_EINVAL, "%s: misaligned pointer", who);
    const rows8 m = blocks_of(rows, cols, ldx == cols && (kind == KIND_NONE || ldy == cols));
    BY_TYPE(launch_backward, dy, ldy, c, st, dx, ldx, m, p, (hipStream_t)stream)
    SPF_LAUNCH_CHECK(who);
    return SPF_OK;
}
int kind_problem(const char* who, int kind, float p) {
    if (kind < SPF_ACT_LEAKY_RELU || kind > SPF_ACT_GELU) return fail(SPF_EINVAL, "%s: unknown activation %d", who, kind);
    if (kind == SPF_ACT_LEAKY_RELU && !(p >= 0.f && p < INFINITY)) return fail(SPF_EINVAL, "%s: LeakyReLU needs a slope >= 0 (the sign of y is the sign of x)", who);
    if (kind == SPF_ACT_SOFTPLUS && !(p > 0.f && p < INFINITY)) return fail(SPF_EINVAL, "%s: softplus needs beta > 0", who);
    return SPF_OK;
}

}  // namespace

extern "C" {

int spf_saved8_pack(const void* x, int32_t type, int64_t ldx, int64_t rows, int64_t cols, uint8_t* codes, uint8_t* steps, void* stream) {
    if (rows > 0 && cols > 0 && (!codes || !steps)) return spf::fail(SPF_EINVAL, "spf_saved8_pack: null pointer");
    return forward("spf_saved8_pack", x, type, ldx, rows, cols, KIND_NONE, 1.f, nullptr, 0, codes, steps, nullptr, nullptr, stream);
}

int spf_saved8_restore(const uint8_t* codes, const uint8_t* steps, int64_t rows, int64_t cols, void* out, int32_t type, int64_t ldo, void* stream) {
    return backward("spf_saved8_restore", nullptr, type, 0, rows, cols, KIND_NONE, 1.f, codes, steps, out, ldo, stream);
}

int spf_act8_forward(const void* x, int32_t type, int64_t ldx, int64_t rows, int64_t cols, int32_t kind, float param, void* y, int64_t ldy, uint8_t* in_codes,
                     uint8_t* in_steps, uint8_t* out_codes, uint8_t* out_steps, void* stream) {
    if (int rc = kind_problem("spf_act8_forward", kind, param)) return rc;
    return forward("spf_act8_forward", x, type, ldx, rows, cols, kind, param, y, ldy, in_codes, in_steps, out_codes, out_steps, stream);
}

int spf_act8_backward(const void* dy, int32_t type, int64_t ldy, int64_t rows, int64_t cols, int32_t kind, float param, const uint8_t* codes, const uint8_t* steps,
                      void* dx, int64_t ldx, void* stream) {
    if (int rc = kind_problem("spf_act8_backward", kind, param)) return rc;
    return backward("spf_act8_backward", dy, type, ldy, rows, cols, kind, param, codes, steps, dx, ldx, stream);
}

}  // extern "C"
