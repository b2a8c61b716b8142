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
    void *dw, *db;                   // splits == 1: the results; else fp32 tiles [split][n][k], [split][n].  db: null or
    int type, add;                   // of the results (splits == 1)
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

template <typename W> __device__ __forceinline__ void put(void* out, size_t i, float v, bool add) {
    W* p = reinterpret_cast<W*>(out) + i;
    *p = (W)(add ? (float)*p + v : v);
}

template <typename T, int TN, int TK, int WN, int WK, int MS>
__global__ void __launch_bounds__(64 * WN * WK)
wgrad8_kernel(wgrad8_args a) {
    constexpr int THREADS = 64 * WN * WK, NP = PIECES<T>, FN = TN / WN / 32, FK = TK / WK / 32;
    constexpr int PN = TN + 32, PK = TK + 32;                              // row pitches in LDS, elements
    constexpr int GC = MS * TN / 8 / THREADS, GROW = THREADS / (TN / 8);     // 8-element pieces of G a thread loads, and the rows between them
    constexpr int AB = MS * TK / 16 >= THREADS ? 16 : 8;                    // bytes of A in a piece
    constexpr int AC = MS * TK / AB / THREADS, AROW = THREADS / (TK / AB);
    static_assert(GC >= 1 && AC >= 1 && GC * GROW == MS && AC * AROW == MS, "the loads cover a stage");
    __shared__ __attribute__((aligned(16))) __bf16 sg[2][NP][MS * PN];
    __shared__ __attribute__((aligned(16))) __bf16 sa[2][MS * PK];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // Workgroups go to the eight XCDs in turn; each XCD gets a run of tiles, so that the ones that share rows and columns meet in its L2: split by split, and
    // within a split strips of eight tiles of G's columns.
    const int tiles = a.tiles_n * a.tiles_k, total = tiles * a.splits;
    const int wg = total % 8 == 0 ? (int)(blockIdx.x % 8) * (total / 8) + (int)(blockIdx.x / 8) : (int)blockIdx.x;
    const int split = wg / tiles, tile = wg % tiles, strip = tile / (8 * a.tiles_k);
    const int height = min(8, a.tiles_n - 8 * strip), in_strip = tile - strip * 8 * a.tiles_k;
    const int n0 = (8 * strip + in_strip % height) * TN, k0 = (in_strip / height) * TK;
    const long long m_begin = split * a.share, m_end = min(m_begin + a.share, a.rows);

    // this thread's pieces of a stage
    const int gcol = (tid % (TN / 8)) * 8, grow = tid / (TN / 8), acol = (tid % (TK / AB)) * AB, arow = tid / (TK / AB);
    const T* gp = (const T*)a.g + n0 + gcol;
    const int g_left = a.n - n0 - gcol;
    const bool a_in = k0 + acol < a.nb * S8_BLOCK;
    const uint8_t* ap = a.codes + k0 + acol;
    const uint8_t* ep = a.steps + (k0 + acol) / S8_BLOCK;
    vec_t<T> rg[GC][8 / VEC<T>];
    uint32_t ra[AC][AB / 4], re[AC];
    auto load_g = [&](long long m0, int i) {                              // rows behind the share's end are zeros
        const long long m = m0 + grow + i * GROW;
        const int left = m < m_end ? g_left : 0;
#pragma unroll
        for (int q = 0; q < 8 / VEC<T>; ++q) rg[i][q] = load_vec(gp + m * a.ldg + q * VEC<T>, left - q * VEC<T>);
    };
    auto load_a = [&](long long m0, int i) {
        const long long m = m0 + arow + i * AROW;
#pragma unroll
        for (int j = 0; j < AB / 4; ++j) ra[i][j] = 0;
        re[i] = 0;
        if (a_in && m < m_end) {
            const uint8_t* p = ap + m * a.nb * S8_BLOCK;
            if constexpr (AB == 16) {
                const u32x4 v = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
                for (int j = 0; j < 4; ++j) ra[i][j] = v[j];
            } else {
                const uint2 v = *reinterpret_cast<const uint2*>(p);
                ra[i][0] = v.x, ra[i][1] = v.y;
            }
            re[i] = ep[m * a.nb];
        }
    };
    float bias[8] = {};
    const bool with_bias = a.db && k0 == 0;
    auto store_g = [&](int buf, int i) {
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = (float)rg[i][j / VEC<T>][j % VEC<T>];
        if (with_bias)
#pragma unroll
            for (int j = 0; j < 8; ++j) bias[j] += f[j];
        __bf16* d = &sg[buf][0][(grow + i * GROW) * PN + gcol];
        if constexpr (NP == 1) {
            *reinterpret_cast<vec_t<T>*>(d) = rg[i][0];
        } else {
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                u32x4 w;
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = high_halves(f[2 * j], f[2 * j + 1]);
                *reinterpret_cast<u32x4*>(d + p * MS * PN) = w;
                if (p + 1 < NP)
#pragma unroll
                    for (int j = 0; j < 8; ++j) f[j] -= high_part(f[j]);
            }
        }
    };
    auto store_a = [&](int buf, int i) {
        const float step = s8_step(re[i]);
        __bf16* d = &sa[buf][(arow + i * AROW) * PK + acol];
#pragma unroll
        for (int h = 0; h < AB / 8; ++h) {
            u32x4 w;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t c = ra[i][2 * h + j], mag = c & 0x7f7f7f7fu;
                const float m0 = (float)(mag & 0xffu) * step, m1 = (float)((mag >> 8) & 0xffu) * step, m2 = (float)((mag >> 16) & 0xffu) * step, m3 = (float)(mag >> 24) * step;
                // the signs: bytes 0, 1 and 2, 3 moved to the tops of two bf16 pairs
                w[2 * j] = high_halves(m0, m1) | (__builtin_amdgcn_perm(0u, c, 0x010c000cu) & 0x80008000u);
                w[2 * j + 1] = high_halves(m2, m3) | (__builtin_amdgcn_perm(0u, c, 0x030c020cu) & 0x80008000u);
            }
            *reinterpret_cast<u32x4*>(d + 8 * h) = w;
        }
    };

    f32x16 acc[FN][FK] = {};
    const int wn = (wave / WK) * (TN / WN), wk = (wave % WK) * (TK / WK);
    const int at_row = (lane >> 5) * 8 + ((lane >> 2) & 3), at_col = ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
    auto multiply = [&](int buf, int s) {
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
    };

    // Stage i is multiplied while stage i + 1 goes from registers to the other LDS buffer, a piece behind each 16 rows, and each piece of stage i + 2 is under
    // way from memory as soon as its registers are free: for a whole stage's time.
    if (m_begin < m_end) {
#pragma unroll
        for (int i = 0; i < GC; ++i) load_g(m_begin, i);
#pragma unroll
        for (int i = 0; i < AC; ++i) load_a(m_begin, i);
#pragma unroll
        for (int i = 0; i < GC; ++i) store_g(0, i), load_g(m_begin + MS, i);
#pragma unroll
        for (int i = 0; i < AC; ++i) store_a(0, i), load_a(m_begin + MS, i);
        lds_barrier();
    }
    int buf = 0;
    for (long long m0 = m_begin; m0 < m_end; m0 += MS, buf ^= 1) {
        constexpr int PARTS = MS / 16;
#pragma unroll
        for (int s = 0; s < PARTS; ++s) {
            multiply(buf, s);
#pragma unroll
            for (int i = 0; i < GC; ++i)
                if (i * PARTS / GC == s) store_g(buf ^ 1, i), load_g(m0 + 2 * MS, i);
#pragma unroll
            for (int i = 0; i < AC; ++i)
                if ((AC - 1 - i) * PARTS / AC == PARTS - 1 - s) store_a(buf ^ 1, i), load_a(m0 + 2 * MS, i);
        }
        lds_barrier();
    }

    // the tile: a lane holds column (lane & 31) and rows 8 (q / 4) + 4 (lane / 32) + q % 4 of each 32 x 32 block
    auto write = [&](auto one, void* dw, void* db, bool add) {
        using W = decltype(one);
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int j = 0; j < FK; ++j) {
                const int col = k0 + wk + 32 * j + (lane & 31);
#pragma unroll
                for (int q = 0; q < 16; ++q) {
                    const int row = n0 + wn + 32 * i + 8 * (q / 4) + 4 * (lane >> 5) + q % 4;
                    if (row < a.n && col < a.k) put<W>(dw, (size_t)row * a.k + col, acc[i][j][q], add);
                }
            }
        if (with_bias) {                                                    // the same for the whole workgroup
            __syncthreads();
            float* fold = reinterpret_cast<float*>(&sg[0][0][0]);           // [GROW][TN]
            static_assert(GROW * TN * 4 <= (int)sizeof(sg), "the column sums fit");
#pragma unroll
            for (int j = 0; j < 8; ++j) fold[grow * TN + gcol + j] = bias[j];
            __syncthreads();
            for (int c = tid; c < TN; c += THREADS) {
                float s = 0.f;
                for (int r = 0; r < GROW; ++r) s += fold[r * TN + c];
                if (n0 + c < a.n) put<W>(db, n0 + c, s, add);
            }
        }
    };
    if (a.splits > 1)
        write(float(), (float*)a.dw + (size_t)split * a.n * a.k, (float*)a.db + (size_t)split * a.n, false);
    else if (a.type == SPF_TYPE_F32)
        write(float(), a.dw, a.db, a.add != 0);
    else if (a.type == SPF_TYPE_BF16)
        write(__bf16(), a.dw, a.db, a.add != 0);
    else
        write(_Float16(), a.dw, a.db, a.add != 0);
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
    int tn, tk, tiles_n, tiles_k, splits;
    int64_t share;
};
constexpr int STAGE = 32;
// A 256 x 256 tile reads each operand least often and keeps the matrix pipe fed, but a workgroup has a compute unit to itself and leaves 256 KB behind:
// it is taken where every compute unit gets eight stages of rows or more.  Smaller work takes 64 x 64 tiles, several to a compute unit, and shares as short
// as two stages, since what counts there is the chain of loads.
plan plan_of(int64_t rows, int64_t n, int64_t k) {
    plan p;
    const int64_t stages = (rows + STAGE - 1) / STAGE;
    const bool big = n > 128 && k > 128 && ((n + 255) / 256) * ((k + 255) / 256) * stages >= 256 * 8;
    p.tn = p.tk = big ? 256 : 64;
    p.tiles_n = (int)((n + p.tn - 1) / p.tn);
    p.tiles_k = (int)((k + p.tk - 1) / p.tk);
    const int64_t tiles = (int64_t)p.tiles_n * p.tiles_k, most = big ? 256 : 1024, least = big ? 8 : 2;
    int64_t s = most / tiles;
    s = s < stages / least ? s : stages / least;
    s = s < 1 ? 1 : s;
    const int64_t per = (stages + s - 1) / s;
    p.splits = (int)((stages + per - 1) / per);
    p.share = per * STAGE;
    return p;
}

template <typename T> void launch(const wgrad8_args& a, const plan& p, hipStream_t s) {
    const unsigned wgs = (unsigned)(p.tiles_n * p.tiles_k * p.splits);
    if (p.tn == 256)
        wgrad8_kernel<T, 256, 256, 2, 4, STAGE><<<wgs, 512, 0, s>>>(a);
    else
        wgrad8_kernel<T, 64, 64, 2, 2, STAGE><<<wgs, 256, 0, s>>>(a);
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
    const int64_t splits = plan_of(rows, n, cols).splits;
    return splits > 1 ? splits * n * (cols + 1) : 0;
}

int spf_wgrad8(const void* g, int32_t type, int64_t ldg, const uint8_t* codes, const uint8_t* steps, int64_t rows, int64_t n, int64_t cols, void* dw, void* db,
               int32_t wtype, int32_t accumulate, float* workspace, void* stream) {
    const char* who = "spf_wgrad8";
    if (!type_ok(type) || !type_ok(wtype)) return fail(SPF_EINVAL, "%s: unknown element type", who);
    if (const char* why = bad_sizes(rows, n, cols)) return fail(SPF_EINVAL, "%s: %s", who, why);
    if (rows == 0 || n == 0 || cols == 0) return SPF_OK;
    const plan p = plan_of(rows, n, cols);
    if (!g || !codes || !steps || !dw || (p.splits > 1 && !workspace)) return fail(SPF_EINVAL, "%s: null pointer", who);
    if (ldg < 0) return fail(SPF_EINVAL, "%s: row stride", who);
    if (misaligned(g, type_size(type)) || misaligned(codes, 16) || misaligned(dw, type_size(wtype)) || misaligned(db, type_size(wtype)) || misaligned(workspace, 4))
        return fail(SPF_EINVAL, "%s: misaligned pointer", who);
    float* bias_tiles = db ? workspace + (int64_t)p.splits * n * cols : nullptr;
    wgrad8_args a = {g, ldg, codes, steps, rows, p.share, (int)n, (int)cols, (int)((cols + S8_BLOCK - 1) / S8_BLOCK), p.tiles_n, p.tiles_k, p.splits, dw, db, wtype, accumulate};
    if (p.splits > 1) a.dw = workspace, a.db = bias_tiles;
    hipStream_t s = (hipStream_t)stream;
    if (type == SPF_TYPE_F32) launch<float>(a, p, s);
    else if (type == SPF_TYPE_BF16) launch<__bf16>(a, p, s);
    else launch<_Float16>(a, p, s);
    if (p.splits > 1) {
        const int64_t groups = (n * cols + 31) / 32 + (db ? (n + 31) / 32 : 0);
        const auto reduce = [&](auto* w, auto* b) { wgrad8_reduce_kernel<<<(unsigned)groups, 256, 0, s>>>(workspace, p.splits, n * cols, w, bias_tiles, (int)n, b, accumulate); };
        if (wtype == SPF_TYPE_F32) reduce((float*)dw, (float*)db);
        else if (wtype == SPF_TYPE_BF16) reduce((__bf16*)dw, (__bf16*)db);
        else reduce((_Float16*)dw, (_Float16*)db);
    }
    SPF_LAUNCH_CHECK(who);
    return SPF_OK;
}

}  // extern "C"
