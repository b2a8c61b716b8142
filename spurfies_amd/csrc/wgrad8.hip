// Weight gradient of a linear layer whose input was saved in 8 bits:  dW[n][k] = sum over rows m of G[m][n] A[m][k],  db[n] = sum of G[m][n].
//
// A is read as the bytes it was saved in (1 + 1/32 bytes an element instead of 4 or 2) and becomes bf16 on its way into LDS: at most 7 bits times a power
// of two, so that conversion is exact.  G goes to the matrix pipe in bf16 pieces that add up to it exactly — one for bf16, two for fp16, three for fp32
// (8 bits each, by truncation) — so every product is exact and the only rounding is the fp32 accumulation.
//
// A workgroup owns a TN x TK tile of dW over a contiguous share of the rows: a stage of MS rows is loaded to registers while the stage before it is
// multiplied, written to LDS row by row (its natural order), and read back transposed: v_mfma_f32_32x32x16_bf16 wants eight consecutive rows of one column
// in a lane, which is what ds_read_b64_tr_b16 delivers (each group of 16 lanes transposes a 4 x 16 block).  Two LDS buffers, one barrier a stage; the
// row pitch is 64 bytes longer than the tile, so that the four rows of a transposed read lie in different banks.
// The rows are shared out over enough workgroups to fill the chip.  Each leaves an fp32 tile in the workspace, and a second launch adds them in a
// fixed order (no atomics: the same call gives the same bits).  db rides along: a loading thread always holds the same eight columns of G.
#include "saved8.h"

namespace {
using namespace spf;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T> constexpr int PIECES = 1;
template <> constexpr int PIECES<_Float16> = 2;
template <> constexpr int PIECES<float> = 3;

struct wgrad8_args {
    const void* g;
    long long ldg;
    const uint8_t *codes, *steps;
    long long rows, share;           // rows in all, and of one split (a multiple of the stage)
    int n, k, nb;                    // columns of G, columns of A, 32-column blocks of a row of A
    int tiles_n, tiles_k, splits;
    float *dw, *db;                  // fp32 tiles: [split][n][k], [split][n] (db: null or)
};

// the high halves of two floats as one word: two bf16 by truncation
__device__ __forceinline__ uint32_t high_halves(float a, float b) { return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u); }
__device__ __forceinline__ float high_part(float a) { return __uint_as_float(__float_as_uint(a) & 0xffff0000u); }

__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// eight rows of column (lane & 31) of a 32-column strip, from row 8 (lane / 32) on: an operand of the matrix instruction
__device__ __forceinline__ bf16x8 read_columns(const __bf16* p, int pitch) {
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    union { s16x4 h[2]; bf16x8 v; } r;
    r.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
    r.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * pitch));
    return r.v;
}

template <typename T, int TN, int TK, int WN, int WK, int MS>
__global__ void __launch_bounds__(64 * WN * WK)
wgrad8_kernel(wgrad8_args a) {
    constexpr int THREADS = 64 * WN * WK, NP = PIECES<T>, FN = TN / WN / 32, FK = TK / WK / 32;
    constexpr int PN = TN + 32, PK = TK + 32;                              // row pitches in LDS, elements
    constexpr int GC = MS * TN / 8 / THREADS, GROW = THREADS / (TN / 8);     // 8-element pieces of G a thread loads, and the rows between them
    constexpr int AC = MS * TK / 16 / THREADS, AROW = THREADS / (TK / 16);   // 16-byte pieces of A
    static_assert(GC >= 1 && AC >= 1 && GC * GROW == MS && AC * AROW == MS, "the loads cover a stage");
    __shared__ __attribute__((aligned(16))) __bf16 sg[2][NP][MS * PN];
    __shared__ __attribute__((aligned(16))) __bf16 sa[2][MS * PK];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int split = blockIdx.x / (a.tiles_n * a.tiles_k), tile = blockIdx.x % (a.tiles_n * a.tiles_k);
    const int n0 = (tile / a.tiles_k) * TN, k0 = (tile % a.tiles_k) * TK;
    const long long m_begin = split * a.share, m_end = min(m_begin + a.share, a.rows);

    // this thread's pieces of a stage
    const int gcol = (tid % (TN / 8)) * 8, grow = tid / (TN / 8), acol = (tid % (TK / 16)) * 16, arow = tid / (TK / 16);
    const T* gp = (const T*)a.g + n0 + gcol;
    const int g_left = a.n - n0 - gcol;
    const bool a_in = k0 + acol < a.nb * S8_BLOCK;
    const uint8_t* ap = a.codes + k0 + acol;
    const uint8_t* ep = a.steps + (k0 + acol) / S8_BLOCK;
    vec_t<T> rg[GC][8 / VEC<T>];
    u32x4 ra[AC];
    uint32_t re[AC];
    auto load = [&](long long m0) {
#pragma unroll
        for (int i = 0; i < GC; ++i) {
            const long long m = m0 + grow + i * GROW;
            const int left = m < m_end ? g_left : 0;
#pragma unroll
            for (int q = 0; q < 8 / VEC<T>; ++q) rg[i][q] = load_vec(gp + m * a.ldg + q * VEC<T>, left - q * VEC<T>);
        }
#pragma unroll
        for (int i = 0; i < AC; ++i) {
            const long long m = m0 + arow + i * AROW;
            ra[i] = u32x4{0, 0, 0, 0};
            re[i] = 0;
            if (a_in && m < m_end) {
                ra[i] = *reinterpret_cast<const u32x4*>(ap + m * a.nb * S8_BLOCK);
                re[i] = ep[m * a.nb];
            }
        }
    };
    float bias[8] = {};
    const bool with_bias = a.db && k0 == 0;
    auto store = [&](int buf) {
#pragma unroll
        for (int i = 0; i < GC; ++i) {
            float f[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = (float)rg[i][j / VEC<T>][j % VEC<T>];
            if (with_bias)
#pragma unroll
                for (int j = 0; j < 8; ++j) bias[j] += f[j];
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                u32x4 w;
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = high_halves(f[2 * j], f[2 * j + 1]);
                *reinterpret_cast<u32x4*>(&sg[buf][p][(grow + i * GROW) * PN + gcol]) = w;
                if (p + 1 < NP)
#pragma unroll
                    for (int j = 0; j < 8; ++j) f[j] -= high_part(f[j]);
            }
        }
#pragma unroll
        for (int i = 0; i < AC; ++i) {
            const float step = s8_step(re[i]);
            u32x4 w[2];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t c = ra[i][j], mag = c & 0x7f7f7f7fu;
                const float m0 = (float)(mag & 0xffu) * step, m1 = (float)((mag >> 8) & 0xffu) * step, m2 = (float)((mag >> 16) & 0xffu) * step, m3 = (float)(mag >> 24) * step;
                // the signs: bytes 0, 1 and 2, 3 moved to the tops of two bf16 pairs
                w[j / 2][2 * (j % 2)] = high_halves(m0, m1) | (__builtin_amdgcn_perm(0u, c, 0x010c000cu) & 0x80008000u);
                w[j / 2][2 * (j % 2) + 1] = high_halves(m2, m3) | (__builtin_amdgcn_perm(0u, c, 0x030c020cu) & 0x80008000u);
            }
            __bf16* d = &sa[buf][(arow + i * AROW) * PK + acol];
            *reinterpret_cast<u32x4*>(d) = w[0];
            *reinterpret_cast<u32x4*>(d + 8) = w[1];
        }
    };

    f32x16 acc[FN][FK] = {};
    const int wn = (wave / WK) * (TN / WN), wk = (wave % WK) * (TK / WK);
    const int at_row = (lane >> 5) * 8 + ((lane >> 2) & 3), at_col = ((lane >> 4) & 1) * 16 + (lane & 3) * 4;

    if (m_begin < m_end) load(m_begin);
    int buf = 0;
    for (long long m0 = m_begin; m0 < m_end; m0 += MS, buf ^= 1) {
        store(buf);
        if (m0 + MS < m_end) load(m0 + MS);
        lds_barrier();
#pragma unroll
        for (int s = 0; s < MS / 16; ++s) {
            bf16x8 fa[FK];
#pragma unroll
            for (int j = 0; j < FK; ++j) fa[j] = read_columns(&sa[buf][(16 * s + at_row) * PK + wk + 32 * j + at_col], PK);
#pragma unroll
            for (int p = 0; p < NP; ++p)
#pragma unroll
                for (int i = 0; i < FN; ++i) {
                    const bf16x8 fg = read_columns(&sg[buf][p][(16 * s + at_row) * PN + wn + 32 * i + at_col], PN);
#pragma unroll
                    for (int j = 0; j < FK; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fg, fa[j], acc[i][j], 0, 0, 0);
                }
        }
    }

    // the tile: a lane holds column (lane & 31) and rows 8 (q / 4) + 4 (lane / 32) + q % 4 of each 32 x 32 block
    float* dw = a.dw + (size_t)split * a.n * a.k;
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FK; ++j) {
            const int col = k0 + wk + 32 * j + (lane & 31);
#pragma unroll
            for (int q = 0; q < 16; ++q) {
                const int row = n0 + wn + 32 * i + 8 * (q / 4) + 4 * (lane >> 5) + q % 4;
                if (row < a.n && col < a.k) dw[(size_t)row * a.k + col] = acc[i][j][q];
            }
        }
    if (with_bias) {                                                        // the same for the whole workgroup
        __syncthreads();
        float* fold = reinterpret_cast<float*>(&sg[0][0][0]);               // [GROW][TN]
        static_assert(GROW * TN * 4 <= (int)sizeof(sg), "the column sums fit");
#pragma unroll
        for (int j = 0; j < 8; ++j) fold[grow * TN + gcol + j] = bias[j];
        __syncthreads();
        for (int c = tid; c < TN; c += THREADS) {
            float s = 0.f;
            for (int r = 0; r < GROW; ++r) s += fold[r * TN + c];
            if (n0 + c < a.n) a.db[(size_t)split * a.n + n0 + c] = s;
        }
    }
}

// out[i] (+)= sum over the splits, in order; eight threads an element group share the splits
template <typename W>
__global__ void __launch_bounds__(256)
wgrad8_reduce_kernel(const float* __restrict__ tiles, int splits, long long count, W* dw, const float* __restrict__ bias_tiles, int n, W* db, int add) {
    __shared__ float part[8][33];
    const int lane = threadIdx.x & 31, k = threadIdx.x >> 5;
    const long long groups = (count + 31) / 32;
    const bool is_bias = blockIdx.x >= groups;                              // the last workgroups add db
    const long long c = (is_bias ? (long long)blockIdx.x - groups : (long long)blockIdx.x) * 32 + lane;
    const long long len = is_bias ? n : count;
    const float* src = is_bias ? bias_tiles : tiles;
    float s = 0.f;
    if (c < len) {
#pragma unroll 8
        for (int i = k; i < splits; i += 8) s += src[(size_t)i * len + c];
    }
    part[k][lane] = s;
    __syncthreads();
    if (k != 0 || c >= len) return;
#pragma unroll
    for (int i = 1; i < 8; ++i) s += part[i][lane];
    W* out = is_bias ? db : dw;
    out[c] = (W)(add ? (float)out[c] + s : s);
}

struct plan {
    int tn, tk, ms, tiles_n, tiles_k, splits;
    int64_t share;
};
// A 256 x 256 tile reads each operand least often and keeps the matrix pipe fed; a layer that does not fill one takes 64 x 64.  The rows are split until
// there is a workgroup for each of the 256 compute units, as long as a share is worth its fp32 tile (eight stages).
plan plan_of(int64_t rows, int64_t n, int64_t k) {
    plan p;
    const bool big = n > 128 && k > 128;
    p.tn = p.tk = big ? 256 : 64;
    p.ms = big ? 32 : 64;
    p.tiles_n = (int)((n + p.tn - 1) / p.tn);
    p.tiles_k = (int)((k + p.tk - 1) / p.tk);
    const int64_t stages = (rows + p.ms - 1) / p.ms, tiles = (int64_t)p.tiles_n * p.tiles_k;
    int64_t s = (big ? 256 : 1024) / tiles;
    s = s < stages / 8 ? s : stages / 8;
    s = s < 1 ? 1 : s;
    const int64_t per = (stages + s - 1) / s;
    p.splits = (int)((stages + per - 1) / per);
    p.share = per * p.ms;
    return p;
}

template <typename T> void launch(const wgrad8_args& a, const plan& p, hipStream_t s) {
    const unsigned wgs = (unsigned)(p.tiles_n * p.tiles_k * p.splits);
    if (p.tn == 256)
        wgrad8_kernel<T, 256, 256, 2, 4, 32><<<wgs, 512, 0, s>>>(a);
    else
        wgrad8_kernel<T, 64, 64, 2, 2, 64><<<wgs, 256, 0, s>>>(a);
}

const char* bad_sizes(int64_t rows, int64_t n, int64_t k) {
    if (rows < 0 || n < 0 || k < 0) return "negative size";
    if (rows >= (1ll << 31) || n > (1 << 20) || k > (1 << 20) || n * k > (1ll << 34)) return "rows < 2^31, widths <= 2^20 and a product <= 2^34 are supported";
    return nullptr;
}
bool misaligned(const void* p, int size) { return ((uintptr_t)p & (uintptr_t)(size - 1)) != 0; }

}  // namespace

extern "C" {

int64_t spf_wgrad8_workspace_floats(int64_t rows, int64_t n, int64_t cols) {
    if (bad_sizes(rows, n, cols) || rows == 0 || n == 0 || cols == 0) return 0;
    return (int64_t)plan_of(rows, n, cols).splits * n * (cols + 1);
}

int spf_wgrad8(const void* g, int32_t type, int64_t ldg, const uint8_t* codes, const uint8_t* steps, int64_t rows, int64_t n, int64_t cols, void* dw, void* db,
               int32_t wtype, int32_t accumulate, float* workspace, void* stream) {
    const char* who = "spf_wgrad8";
    if (!type_ok(type) || !type_ok(wtype)) return fail(SPF_EINVAL, "%s: unknown element type", who);
    if (const char* why = bad_sizes(rows, n, cols)) return fail(SPF_EINVAL, "%s: %s", who, why);
    if (rows == 0 || n == 0 || cols == 0) return SPF_OK;
    if (!g || !codes || !steps || !dw || !workspace) return fail(SPF_EINVAL, "%s: null pointer", who);
    if (ldg < 0) return fail(SPF_EINVAL, "%s: row stride", who);
    if (misaligned(g, type_size(type)) || misaligned(codes, 16) || misaligned(dw, type_size(wtype)) || misaligned(db, type_size(wtype)) || misaligned(workspace, 4))
        return fail(SPF_EINVAL, "%s: misaligned pointer", who);
    const plan p = plan_of(rows, n, cols);
    wgrad8_args a = {g, ldg, codes, steps, rows, p.share, (int)n, (int)cols, (int)((cols + S8_BLOCK - 1) / S8_BLOCK), p.tiles_n, p.tiles_k, p.splits, workspace,
                     db ? workspace + (int64_t)p.splits * n * cols : nullptr};
    hipStream_t s = (hipStream_t)stream;
    if (type == SPF_TYPE_F32) launch<float>(a, p, s);
    else if (type == SPF_TYPE_BF16) launch<__bf16>(a, p, s);
    else launch<_Float16>(a, p, s);
    const int64_t groups = (n * cols + 31) / 32 + (db ? (n + 31) / 32 : 0);
    const auto reduce = [&](auto* w, auto* b) { wgrad8_reduce_kernel<<<(unsigned)groups, 256, 0, s>>>(workspace, p.splits, n * cols, w, a.db, (int)n, b, accumulate); };
    if (wtype == SPF_TYPE_F32) reduce((float*)dw, (float*)db);
    else if (wtype == SPF_TYPE_BF16) reduce((__bf16*)dw, (__bf16*)db);
    else reduce((_Float16*)dw, (_Float16*)db);
    SPF_LAUNCH_CHECK(who);
    return SPF_OK;
}

}  // extern "C"
