// Layer norm over the last dimension, forward and backward, with the input saved whole or in 8 bits.
//
//   y  = n w + b,  n = (x - mean) rstd,  rstd = 1 / sqrt(var + eps)            per row of `cols` elements, var over cols (not cols - 1)
//   dx = rstd (t - mean(t) - n mean(t n)),  t = dy w;     dw = sum over rows of dy n;     db = sum over rows of dy
//
// A row stays in registers from its one read to its one write: up to 16 elements a thread, so the threads a row gets follow from its width — 8 to 64
// lanes of a wave (several rows share a wave below 256 fp32 / 512 16-bit columns), then 256, then 1024 threads.  The mean is taken before the squares (two
// sums over the registers), so rows that sit far from zero lose no more than the mean's own rounding.  Workgroups walk over the rows with the next row's loads in flight.
// The weight gradients need every row: each thread keeps its columns' sums in registers over all the rows of its workgroup, the workgroup's rows
// are added through LDS, and one line per workgroup goes to the workspace; a second launch adds the lines in a fixed order.  No atomics: the same
// call gives the same bits.  Rows too wide for that (forward 16384, backward 8192 columns) are read again for each
// step — they stay in the caches — with the column sums in a kernel of their own.
// Measured on MI355X (medians), HBM-bound: 389017 x 256 fp32 148 us forward (5.4 TB/s) and 239 + 7 back (5.0 TB/s); 16384 x 4096 bf16 saved in 8 bits 68 (5.0 TB/s) and
// 86 + 6 (3.9 TB/s: there the barrier that every row ends in shows, at three workgroups a compute unit); 8192 x 12288 bf16 93 (4.3 TB/s) and, read again, 331 back (1.8 TB/s).
#include <math.h>

#include "saved8.h"

namespace {
using namespace spf;

constexpr int NORM_MAX_FORWARD = 16384;          // columns that stay in a workgroup's registers; the backward pass holds twice as much for each
constexpr int NORM_MAX_BACKWARD = 8192;
constexpr int NORM_GROUPS = 1024;                // lines of column sums, at most

struct norm_args {
    const void *x, *dy;
    void *y, *dx;
    long long ldx, ldy, ldd, rows;               // row strides of x, y or dx, dy
    int cols;
    const void *w, *b;
    float eps;
    float *mean, *rstd;
    uint8_t *in_codes, *in_steps, *out_codes, *out_steps;
    float* lines;                                // [groups][2][line] column sums, or null
    int line;
};

// weight or bias of V columns from c on (`none` where there is no such parameter; behind the row's end: its last one).  The parameter's type is a template
// argument and the loads are unconditional: a switch over the type inside the columns' conditions was compiled into a use of an unset register.
template <typename W, int V> __device__ __forceinline__ void load_weights(const void* w, long long c, int cols, float none, float (&f)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = none;
    if (w) {
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = (float)reinterpret_cast<const W*>(w)[min(c + i, (long long)cols - 1)];
    }
}

// the sum over a row's ROWT threads, in all of them; `red`: LDS of one call, two floats a wave
template <int ROWT> __device__ __forceinline__ float row_sum(float v, float* red) {
    v = lane_sum<(ROWT < 64 ? ROWT : 64)>(v);
    if (ROWT <= 64) return v;
    constexpr int WAVES = ROWT / 64;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) s += red[i];
    return s;
}
template <int ROWT> __device__ __forceinline__ void row_sum2(float& a, float& b, float* red) {
    a = lane_sum<(ROWT < 64 ? ROWT : 64)>(a);
    b = lane_sum<(ROWT < 64 ? ROWT : 64)>(b);
    if (ROWT <= 64) return;
    constexpr int WAVES = ROWT / 64;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a, red[WAVES + (threadIdx.x >> 6)] = b;
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) a += red[i], b += red[WAVES + i];
}

template <typename T, typename W, int ROWT, int NV>
__global__ void __launch_bounds__(ROWT < 256 ? 256 : ROWT)
norm_forward_kernel(norm_args a) {
    constexpr int V = VEC<T>, WG = ROWT < 256 ? 256 : ROWT, RPW = WG / ROWT;
    __shared__ float red[2][2][WG / 64];         // two sums a row, two rows in turn
    const int t = threadIdx.x % ROWT, slot = threadIdx.x / ROWT;
    const int nb = (a.cols + S8_BLOCK - 1) / S8_BLOCK;
    float w[NV][V], b[NV][V];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        load_weights<W>(a.w, (v * ROWT + t) * V, a.cols, 1.f, w[v]);
        load_weights<W>(a.b, (v * ROWT + t) * V, a.cols, 0.f, b[v]);
    }
    const T* x = (const T*)a.x;
    vec_t<T> next[NV];
    auto load = [&](long long row) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * ROWT + t) * V;
            next[v] = load_vec(x + row * a.ldx + c, row < a.rows ? a.cols - c : 0, c > 0);
        }
    };
    const float inv_cols = 1.f / (float)a.cols;
    load((long long)blockIdx.x * RPW + slot);
    int turn = 0;
    for (long long base = (long long)blockIdx.x * RPW; base < a.rows; base += (long long)gridDim.x * RPW, turn ^= 1) {
        const long long row = base + slot;
        const bool ok = row < a.rows;
        float f[NV][V], s = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) to_f32<T>(next[v], f[v]);
        if (a.in_codes) {                        // the bytes of x, before x is gone
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int c = (v * ROWT + t) * V;
                uint32_t k[V / 4];
                const uint32_t e = s8_pack(f[v], k);
                s8_mask<V>(k, a.cols - c);
                if (ok && c < nb * S8_BLOCK) {
                    s8_store<V>(a.in_codes, (size_t)row * nb * S8_BLOCK + c, k);
                    if (c % S8_BLOCK == 0) a.in_steps[(size_t)row * nb + c / S8_BLOCK] = (uint8_t)e;
                }
            }
        }
        load(row + (long long)gridDim.x * RPW);
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < V; ++i) s += f[v][i];
        const float mean = row_sum<ROWT>(s, red[turn][0]) * inv_cols;
        float q = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                f[v][i] = (v * ROWT + t) * V + i < a.cols ? f[v][i] - mean : 0.f;
                q += f[v][i] * f[v][i];
            }
        const float rstd = 1.f / sqrtf(row_sum<ROWT>(q, red[turn][1]) * inv_cols + a.eps);
        if (a.mean && ok && t == 0) a.mean[row] = mean, a.rstd[row] = rstd;
        T* y = (T*)a.y + row * a.ldy;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * ROWT + t) * V;
#pragma unroll
            for (int i = 0; i < V; ++i) f[v][i] = f[v][i] * rstd * w[v][i] + b[v][i];
            const vec_t<T> out = from_f32<T>(f[v]);
            store_vec(y + c, out, ok ? a.cols - c : 0);
            if (a.out_codes) {                   // the bytes of y as the next layer sees it
                to_f32<T>(out, f[v]);
#pragma unroll
                for (int i = 0; i < V; ++i) f[v][i] = c + i < a.cols ? f[v][i] : 0.f;
                uint32_t k[V / 4];
                const uint32_t e = s8_pack(f[v], k);
                s8_mask<V>(k, a.cols - c);
                if (ok && c < nb * S8_BLOCK) {
                    s8_store<V>(a.out_codes, (size_t)row * nb * S8_BLOCK + c, k);
                    if (c % S8_BLOCK == 0) a.out_steps[(size_t)row * nb + c / S8_BLOCK] = (uint8_t)e;
                }
            }
        }
    }
}

template <typename T, typename W, int ROWT, int NV, bool SAVED8>
__global__ void __launch_bounds__(ROWT < 256 ? 256 : ROWT)
norm_backward_kernel(norm_args a) {
    constexpr int V = VEC<T>, WG = ROWT < 256 ? 256 : ROWT, RPW = WG / ROWT, WIDTH = ROWT * NV * V;
    __shared__ float red[2][2 * (WG / 64)];      // two rows in turn
    __shared__ float fold[RPW > 1 ? RPW * WIDTH : 1];
    const int t = threadIdx.x % ROWT, slot = threadIdx.x / ROWT;
    const int nb = (a.cols + S8_BLOCK - 1) / S8_BLOCK;
    float w[NV][V], dw[NV][V] = {}, db[NV][V] = {};
#pragma unroll
    for (int v = 0; v < NV; ++v) load_weights<W>(a.w, (v * ROWT + t) * V, a.cols, 1.f, w[v]);
    vec_t<T> next_x[SAVED8 ? 1 : NV], next_g[NV];
    uint32_t next_k[SAVED8 ? NV : 1][V / 4], next_e[SAVED8 ? NV : 1];
    float next_mean = 0.f, next_rstd = 0.f;
    auto load = [&](long long row) {
        const bool ok = row < a.rows;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * ROWT + t) * V;
            const long long n = ok ? a.cols - c : 0;
            next_g[v] = load_vec((const T*)a.dy + row * a.ldd + c, n, c > 0);
            if constexpr (SAVED8) {
                next_e[v] = 0;
#pragma unroll
                for (int q = 0; q < V / 4; ++q) next_k[v][q] = 0;
                if (n > 0) {
                    s8_load<V>(a.in_codes, (size_t)row * nb * S8_BLOCK + c, next_k[v]);
                    next_e[v] = a.in_steps[(size_t)row * nb + c / S8_BLOCK];
                }
            } else {
                next_x[v] = load_vec((const T*)a.x + row * a.ldx + c, n, c > 0);
            }
        }
        next_mean = ok ? a.mean[row] : 0.f;
        next_rstd = ok ? a.rstd[row] : 0.f;
    };
    const float inv_cols = 1.f / (float)a.cols;
    load((long long)blockIdx.x * RPW + slot);
    int turn = 0;
    for (long long base = (long long)blockIdx.x * RPW; base < a.rows; base += (long long)gridDim.x * RPW, turn ^= 1) {
        const long long row = base + slot;
        float n[NV][V], g[NV][V];
        const float mean = next_mean, rstd = next_rstd;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            to_f32<T>(next_g[v], g[v]);
            if constexpr (SAVED8) {
                s8_unpack<V>(next_k[v], s8_step(next_e[v]), n[v]);
            } else {
                to_f32<T>(next_x[v], n[v]);
            }
        }
        load(row + (long long)gridDim.x * RPW);
        float c1 = 0.f, c2 = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                n[v][i] = (v * ROWT + t) * V + i < a.cols ? (n[v][i] - mean) * rstd : 0.f;
                dw[v][i] += g[v][i] * n[v][i];
                db[v][i] += g[v][i];
                g[v][i] *= w[v][i];
                c1 += g[v][i];
                c2 += g[v][i] * n[v][i];
            }
        if (!a.dx) continue;
        row_sum2<ROWT>(c1, c2, red[turn]);
        c1 *= inv_cols, c2 *= inv_cols;
        T* dx = (T*)a.dx + row * a.ldy;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * ROWT + t) * V;
#pragma unroll
            for (int i = 0; i < V; ++i) g[v][i] = rstd * (g[v][i] - c1 - n[v][i] * c2);
            store_vec(dx + c, from_f32<T>(g[v]), row < a.rows ? a.cols - c : 0);
        }
    }
    if (!a.lines) return;
    float* line = a.lines + (size_t)blockIdx.x * 2 * a.line;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        if constexpr (RPW > 1) {
            __syncthreads();
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < V; ++i) fold[slot * WIDTH + (v * ROWT + t) * V + i] = which ? db[v][i] : dw[v][i];
            __syncthreads();
            for (int c = threadIdx.x; c < a.cols; c += WG) {
                float s = 0.f;
#pragma unroll
                for (int r = 0; r < RPW; ++r) s += fold[r * WIDTH + c];
                line[which * a.line + c] = s;
            }
        } else {
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const int c = (v * ROWT + t) * V + i;
                    if (c < a.cols) line[which * a.line + c] = which ? db[v][i] : dw[v][i];
                }
        }
    }
}

// ---- rows that do not fit into a workgroup's registers ---------------------------------------------------------------------------------------------
template <typename T, typename W>
__global__ void __launch_bounds__(1024)
norm_wide_forward_kernel(norm_args a) {
    constexpr int V = VEC<T>, STEP = 1024 * V;
    __shared__ float red[2][16];
    const int nb = (a.cols + S8_BLOCK - 1) / S8_BLOCK;
    const long long row = (long long)blockIdx.y * gridDim.x + blockIdx.x;
    if (row >= a.rows) return;                   // the same for the whole workgroup
    const T* x = (const T*)a.x + row * a.ldx;
    T* y = (T*)a.y + row * a.ldy;
    const float inv_cols = 1.f / (float)a.cols;
    float f[V], s = 0.f;
    for (long long c = threadIdx.x * V; c < a.cols; c += STEP) {
        to_f32<T>(load_vec(x + c, a.cols - c, c > 0), f);
#pragma unroll
        for (int i = 0; i < V; ++i) s += f[i];
    }
    const float mean = row_sum<1024>(s, red[0]) * inv_cols;
    float q = 0.f;
    for (long long c = threadIdx.x * V; c < a.cols; c += STEP) {
        to_f32<T>(load_vec(x + c, a.cols - c, c > 0), f);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float d = c + i < a.cols ? f[i] - mean : 0.f;
            q += d * d;
        }
    }
    const float rstd = 1.f / sqrtf(row_sum<1024>(q, red[1]) * inv_cols + a.eps);
    if (a.mean && threadIdx.x == 0) a.mean[row] = mean, a.rstd[row] = rstd;
    for (long long at = 0; at < a.cols; at += STEP) {                   // whole waves (a block's lanes work together)
        const long long c = at + threadIdx.x * V, left = a.cols - c;
        uint32_t k[V / 4];
        to_f32<T>(load_vec(x + c, left, c > 0), f);
        if (a.in_codes) {
            const uint32_t e = s8_pack(f, k);
            s8_mask<V>(k, left);
            if (c < (long long)nb * S8_BLOCK) {
                s8_store<V>(a.in_codes, (size_t)row * nb * S8_BLOCK + c, k);
                if (c % S8_BLOCK == 0) a.in_steps[(size_t)row * nb + c / S8_BLOCK] = (uint8_t)e;
            }
        }
        float w[V], b[V];
        load_weights<W>(a.w, c, a.cols, 1.f, w);
        load_weights<W>(a.b, c, a.cols, 0.f, b);
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = i < left ? (f[i] - mean) * rstd * w[i] + b[i] : 0.f;
        const vec_t<T> out = from_f32<T>(f);
        store_vec(y + c, out, left);
        if (a.out_codes) {
            to_f32<T>(out, f);
            const uint32_t e = s8_pack(f, k);
            s8_mask<V>(k, left);
            if (c < (long long)nb * S8_BLOCK) {
                s8_store<V>(a.out_codes, (size_t)row * nb * S8_BLOCK + c, k);
                if (c % S8_BLOCK == 0) a.out_steps[(size_t)row * nb + c / S8_BLOCK] = (uint8_t)e;
            }
        }
    }
}

// n = (x - mean) rstd of V columns from c on, zero behind the row's end
template <typename T, bool SAVED8> __device__ __forceinline__ void normalised(const norm_args& a, long long row, long long c, int nb, float mean, float rstd, float (&n)[VEC<T>]) {
    constexpr int V = VEC<T>;
    if constexpr (SAVED8) {
        uint32_t k[V / 4];
        s8_load<V>(a.in_codes, (size_t)row * nb * S8_BLOCK + c, k);
        s8_unpack<V>(k, s8_step(a.in_steps[(size_t)row * nb + c / S8_BLOCK]), n);
    } else {
        to_f32<T>(load_vec((const T*)a.x + row * a.ldx + c, a.cols - c, c > 0), n);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) n[i] = c + i < a.cols ? (n[i] - mean) * rstd : 0.f;
}

template <typename T, typename W, bool SAVED8>
__global__ void __launch_bounds__(1024)
norm_wide_backward_kernel(norm_args a) {
    constexpr int V = VEC<T>, STEP = 1024 * V;
    __shared__ float red[32];
    const int nb = (a.cols + S8_BLOCK - 1) / S8_BLOCK;
    const long long row = (long long)blockIdx.y * gridDim.x + blockIdx.x;
    if (row >= a.rows) return;                   // the same for the whole workgroup
    const T* dy = (const T*)a.dy + row * a.ldd;
    T* dx = (T*)a.dx + row * a.ldy;
    const float mean = a.mean[row], rstd = a.rstd[row], inv_cols = 1.f / (float)a.cols;
    float n[V], g[V], w[V], c1 = 0.f, c2 = 0.f;
    for (long long c = threadIdx.x * V; c < a.cols; c += STEP) {
        to_f32<T>(load_vec(dy + c, a.cols - c, c > 0), g);
        normalised<T, SAVED8>(a, row, c, nb, mean, rstd, n);
        load_weights<W>(a.w, c, a.cols, 1.f, w);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float t = g[i] * w[i];
            c1 += t;
            c2 += t * n[i];
        }
    }
    row_sum2<1024>(c1, c2, red);
    c1 *= inv_cols, c2 *= inv_cols;
    for (long long c = threadIdx.x * V; c < a.cols; c += STEP) {
        to_f32<T>(load_vec(dy + c, a.cols - c, c > 0), g);
        normalised<T, SAVED8>(a, row, c, nb, mean, rstd, n);
        load_weights<W>(a.w, c, a.cols, 1.f, w);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float t = g[i] * w[i];
            g[i] = rstd * (t - c1 - n[i] * c2);
        }
        store_vec(dx + c, from_f32<T>(g), a.cols - c);
    }
}
// a workgroup's 256 threads take 256 V columns of every gridDim.y-th row
template <typename T, bool SAVED8>
__global__ void __launch_bounds__(256)
norm_wide_columns_kernel(norm_args a) {
    constexpr int V = VEC<T>;
    const int nb = (a.cols + S8_BLOCK - 1) / S8_BLOCK;
    const long long c = ((long long)blockIdx.x * 256 + threadIdx.x) * V;
    if (c >= a.cols) return;
    float dw[V] = {}, db[V] = {}, n[V], g[V];
    for (long long row = blockIdx.y; row < a.rows; row += gridDim.y) {
        to_f32<T>(load_vec((const T*)a.dy + row * a.ldd + c, a.cols - c, c > 0), g);
        normalised<T, SAVED8>(a, row, c, nb, a.mean[row], a.rstd[row], n);
#pragma unroll
        for (int i = 0; i < V; ++i) dw[i] += g[i] * n[i], db[i] += g[i];
    }
    float* line = a.lines + (size_t)blockIdx.y * 2 * a.line;
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (c + i < a.cols) line[c + i] = dw[i], line[a.line + c + i] = db[i];
}

// out[0 / 1][c] (+)= sum over the lines, in order: 16 threads a column, each every 16th line
template <typename W>
__global__ void __launch_bounds__(1024)
norm_columns_kernel(const float* __restrict__ lines, int groups, int line, int cols, W* dw, W* db, int add) {
    __shared__ float part[16][64];
    const int lane = threadIdx.x & 63, k = threadIdx.x >> 6, which = blockIdx.y;
    const int c = (blockIdx.z * gridDim.x + blockIdx.x) * 64 + lane;
    W* out = which ? db : dw;
    if (!out) return;                              // the same for the whole workgroup
    float s = 0.f;
    if (c < cols) {
        const float* p = lines + (size_t)which * line + c;
#pragma unroll 8
        for (int g = k; g < groups; g += 16) s += p[(size_t)g * 2 * line];
    }
    part[k][lane] = s;
    __syncthreads();
    if (k != 0 || c >= cols) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) s += part[i][lane];
    out[c] = (W)(add ? (float)out[c] + s : s);
}

// ---- launches ---------------------------------------------------------------------------------------------------------------------------------
// Workgroups of 1024 threads in two dimensions of the grid: a launch has less than 2^32 threads in each, which are 2^22 workgroups.  (Workgroups that walk over the rows instead
// take 8 - 13 % longer.)
constexpr int64_t ACROSS = 1 << 20;
dim3 wide_grid(int64_t rows) { return dim3((unsigned)(rows < ACROSS ? rows : ACROSS), (unsigned)((rows + ACROSS - 1) / ACROSS)); }
dim3 columns_grid(int64_t cols) { const dim3 d = wide_grid((cols + 63) / 64); return dim3(d.x, 2, d.y); }
// f(threads a row, vectors a thread): the smallest shape whose registers hold the row
template <typename T, bool BACKWARD, typename F> void by_width(int cols, F f) {
    constexpr int V = VEC<T>;
#define SHAPE(ROWT, NV) if (cols <= ROWT * NV * V) return f(std::integral_constant<int, ROWT>(), std::integral_constant<int, NV>());
    SHAPE(8, 1) SHAPE(16, 1) SHAPE(32, 1) SHAPE(64, 1) SHAPE(64, 2)
    if constexpr (V == 4) {
        SHAPE(64, 4) SHAPE(256, 2) SHAPE(256, 4) SHAPE(1024, 2)
        if constexpr (!BACKWARD) { SHAPE(1024, 4) }
    } else {
        SHAPE(256, 1) SHAPE(256, 2) SHAPE(1024, 1)
        if constexpr (!BACKWARD) { SHAPE(1024, 2) }
    }
#undef SHAPE
}
// Workgroups for `steps` row steps: as many as the chip holds at once (they walk over the rows), and all with the same number of steps.  More than that run
// in rounds, the last of which is mostly empty: 1024 of the backward pass at 4096 bf16 columns, of which 768 fit, took 98 us; 745 take 86.
template <auto KERNEL> int groups_for(int64_t steps, int threads, int64_t most) {
    static const int resident = [&] {
        int n = 0;
        return hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, KERNEL, threads, 0) == hipSuccess && n > 0 ? n : 1;
    }();
    int64_t slots = 256ll * resident;
    slots = slots < most ? slots : most;
    const int64_t rounds = (steps + slots - 1) / slots;
    return (int)((steps + rounds - 1) / rounds);
}
int line_of(int64_t cols) { return (int)((cols + 7) / 8 * 8); }

const char* bad_sizes(int64_t rows, int64_t cols) {
    if (rows < 0 || cols < 0) return "negative size";
    if (rows >= (1ll << 31) || cols >= (1ll << 30)) return "rows < 2^31 and columns < 2^30 are supported";
    return nullptr;
}
bool misaligned(const void* p, int size) { return ((uintptr_t)p & (uintptr_t)(size - 1)) != 0; }

template <typename T, typename W> void forward(const norm_args& a, hipStream_t s) {
    if (a.cols > NORM_MAX_FORWARD) {
        norm_wide_forward_kernel<T, W><<<wide_grid(a.rows), 1024, 0, s>>>(a);
        return;
    }
    by_width<T, false>(a.cols, [&](auto rowt, auto nv) {
        constexpr int ROWT = decltype(rowt)::value, NV = decltype(nv)::value, WG = ROWT < 256 ? 256 : ROWT, RPW = WG / ROWT;
        const int groups = groups_for<norm_forward_kernel<T, W, ROWT, NV>>((a.rows + RPW - 1) / RPW, WG, 2048);
        norm_forward_kernel<T, W, ROWT, NV><<<groups, WG, 0, s>>>(a);
    });
}
template <typename T, typename W, bool SAVED8> int backward_groups(const norm_args& a, hipStream_t s) {
    int groups = 0;
    if (a.cols > NORM_MAX_BACKWARD) {
        if (a.dx) norm_wide_backward_kernel<T, W, SAVED8><<<wide_grid(a.rows), 1024, 0, s>>>(a);
        if (a.lines) {
            const unsigned across = (unsigned)((a.cols + 256 * VEC<T> - 1) / (256 * VEC<T>));
            groups = (int)(a.rows < 64 ? a.rows : 64);
            norm_wide_columns_kernel<T, SAVED8><<<dim3(across, groups), 256, 0, s>>>(a);
        }
        return groups;
    }
    by_width<T, true>(a.cols, [&](auto rowt, auto nv) {
        constexpr int ROWT = decltype(rowt)::value, NV = decltype(nv)::value, WG = ROWT < 256 ? 256 : ROWT, RPW = WG / ROWT;
        groups = groups_for<norm_backward_kernel<T, W, ROWT, NV, SAVED8>>((a.rows + RPW - 1) / RPW, WG, NORM_GROUPS);
        norm_backward_kernel<T, W, ROWT, NV, SAVED8><<<groups, WG, 0, s>>>(a);
    });
    return groups;
}
template <typename T, typename W> void backward(const norm_args& a, void* dweight, void* dbias, int add, hipStream_t s) {
    const int groups = a.in_codes ? backward_groups<T, W, true>(a, s) : backward_groups<T, W, false>(a, s);
    if (a.lines)
        norm_columns_kernel<W><<<columns_grid(a.cols), 1024, 0, s>>>(a.lines, groups, a.line, a.cols, (W*)dweight, (W*)dbias, add);
}

// the parameters have the rows' type or fp32
#define BY_TYPES(FN, ...)                                                                     \
    if (type == SPF_TYPE_F32) FN<float, float>(__VA_ARGS__);                                  \
    else if (type == SPF_TYPE_BF16 && wtype == SPF_TYPE_F32) FN<__bf16, float>(__VA_ARGS__);   \
    else if (type == SPF_TYPE_BF16) FN<__bf16, __bf16>(__VA_ARGS__);                           \
    else if (wtype == SPF_TYPE_F32) FN<_Float16, float>(__VA_ARGS__);                          \
    else FN<_Float16, _Float16>(__VA_ARGS__);

}  // namespace

extern "C" {

int spf_layer_norm_forward(const void* x, int32_t type, int64_t ldx, int64_t rows, int64_t cols, const void* weight, const void* bias, int32_t wtype, float eps,
                           void* y, int64_t ldy, float* mean, float* rstd, uint8_t* in_codes, uint8_t* in_steps, uint8_t* out_codes, uint8_t* out_steps, void* stream) {
    const char* who = "spf_layer_norm_forward";
    if (!type_ok(type) || (wtype != type && wtype != SPF_TYPE_F32)) return fail(SPF_EINVAL, "%s: unknown element type, or parameters neither of the rows' type nor fp32", who);
    if (const char* why = bad_sizes(rows, cols)) return fail(SPF_EINVAL, "%s: %s", who, why);
    if (!(eps >= 0.f && eps < INFINITY)) return fail(SPF_EINVAL, "%s: eps must be finite and not negative", who);
    if (rows == 0 || cols == 0) return SPF_OK;
    if (!x || !y || (!mean != !rstd) || (!in_codes != !in_steps) || (!out_codes != !out_steps)) return fail(SPF_EINVAL, "%s: null pointer", who);
    if (ldx < 0 || ldy < cols) return fail(SPF_EINVAL, "%s: row stride", who);
    if (misaligned(x, type_size(type)) || misaligned(y, type_size(type)) || misaligned(weight, type_size(wtype)) || misaligned(bias, type_size(wtype)) || misaligned(in_codes, 16) ||
        misaligned(out_codes, 16))
        return fail(SPF_EINVAL, "%s: misaligned pointer", who);
    norm_args a = {};
    a.x = x, a.y = y, a.ldx = ldx, a.ldy = ldy, a.rows = rows, a.cols = (int)cols, a.w = weight, a.b = bias, a.eps = eps;
    a.mean = mean, a.rstd = rstd, a.in_codes = in_codes, a.in_steps = in_steps, a.out_codes = out_codes, a.out_steps = out_steps;
    BY_TYPES(forward, a, (hipStream_t)stream)
    SPF_LAUNCH_CHECK(who);
    return SPF_OK;
}

int64_t spf_layer_norm_workspace_floats(int64_t rows, int64_t cols) {
    if (bad_sizes(rows, cols) || rows == 0 || cols == 0) return 0;
    // a workgroup takes up to 32 rows side by side; one line each, at most NORM_GROUPS
    return 2ll * line_of(cols) * (cols > NORM_MAX_BACKWARD ? (rows < 64 ? rows : 64) : (rows < NORM_GROUPS ? rows : NORM_GROUPS));
}

int spf_layer_norm_backward(const void* dy, int32_t type, int64_t ldd, int64_t rows, int64_t cols, const void* x, int64_t ldx, const uint8_t* codes, const uint8_t* steps,
                            const float* mean, const float* rstd, const void* weight, int32_t wtype, void* dx, int64_t lddx, void* dweight, void* dbias,
                            int32_t accumulate, float* workspace, void* stream) {
    const char* who = "spf_layer_norm_backward";
    if (!type_ok(type) || (wtype != type && wtype != SPF_TYPE_F32)) return fail(SPF_EINVAL, "%s: unknown element type, or parameters neither of the rows' type nor fp32", who);
    if (const char* why = bad_sizes(rows, cols)) return fail(SPF_EINVAL, "%s: %s", who, why);
    if (rows == 0 || cols == 0) return SPF_OK;
    if (!dy || !mean || !rstd || (!x == !codes) || (!codes != !steps)) return fail(SPF_EINVAL, "%s: needs dy, mean, rstd and one of x and its 8-bit form", who);
    if ((dweight || dbias) && !workspace) return fail(SPF_EINVAL, "%s: the weight gradients need the workspace", who);
    if (ldd < 0 || ldx < 0 || (dx && lddx < cols)) return fail(SPF_EINVAL, "%s: row stride", who);
    if (misaligned(x, type_size(type)) || misaligned(dy, type_size(type)) || misaligned(dx, type_size(type)) || misaligned(weight, type_size(wtype)) ||
        misaligned(dweight, type_size(wtype)) || misaligned(dbias, type_size(wtype)) || misaligned(codes, 16) || misaligned(workspace, 4))
        return fail(SPF_EINVAL, "%s: misaligned pointer", who);
    if (dweight && dweight == dbias) return fail(SPF_EINVAL, "%s: dweight and dbias are one address", who);
    if (!dx && !dweight && !dbias) return SPF_OK;
    norm_args a = {};
    a.dy = dy, a.ldd = ldd, a.rows = rows, a.cols = (int)cols, a.x = x, a.ldx = ldx, a.in_codes = (uint8_t*)codes, a.in_steps = (uint8_t*)steps;
    a.mean = (float*)mean, a.rstd = (float*)rstd, a.w = weight, a.dx = dx, a.ldy = lddx;
    a.lines = dweight || dbias ? workspace : nullptr, a.line = line_of(cols);
    BY_TYPES(backward, a, dweight, dbias, accumulate, (hipStream_t)stream)
    SPF_LAUNCH_CHECK(who);
    return SPF_OK;
}

}  // extern "C"
