// Weight gradient of a linear layer whose input was saved in 8 bits:  dW[n][k] = sum over rows m of G[m][n] A[m][k],  db[n] = sum of G[m][n].
//
// A is read as the bytes it was saved in (1 + 1/32 bytes an element instead of 4 or 2) and becomes bf16 on its way into LDS: at most 7 bits times a power
// of two, so that conversion is exact.  G goes to the matrix pipe in bf16 pieces that add up to it exactly — one for bf16, two for fp16, three for fp32
// (8 bits each, by truncation) — so every product is exact and the only rounding is the fp32 accumulation.
//
// A workgroup owns a TN x TK tile of dW (256, 128 or 64 square) over a contiguous share of the rows: a stage of MS rows is loaded to registers while the stage before it is
// multiplied, written to LDS row by row (its natural order), and read back transposed: v_mfma_f32_32x32x16_bf16 wants eight consecutive rows of one column
// in a lane, which is what ds_read_b64_tr_b16 delivers (each group of 16 lanes transposes a 4 x 16 block).  Two LDS buffers, one barrier a stage; the
// row pitch is 64 bytes longer than the tile, so that the four rows of a transposed read lie in different banks.
// The rows are shared out over enough workgroups to fill the chip.  Each leaves an fp32 tile in the workspace, and a second launch adds them in a
// fixed order (no atomics: the same call gives the same bits).  db rides along: a loading thread always holds the same eight columns of G.
//
// Measured on MI355X: 8192 rows, 4096 x 4096, bf16: 251 - 272 us from box to box = 1010 - 1095 TFLOP/s (a plain bf16 product of that shape by the library, where this took
// 251: 221 - 227 us); 389017 rows, 256 x 256, fp32: 154 us, of which this kernel 135 (3.7 TB/s of operands; three piece products keep the matrix pipe half busy) and
// the sum of the splits 12; 1237 rows, 131 x 515, fp16: 9 + 3 us.
#include <math.h>

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
    void *dw, *db;                   // of type `type`: the results [n][k], [n], or the splits' fp32 tiles [split][n][k], [split][n].  db: null or
    int type;
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

template <typename T, int TN, int TK, int WN, int WK, int MS, bool PLAIN>
__global__ void __launch_bounds__(64 * WN * WK)
wgrad8_kernel(wgrad8_args a) {
    constexpr int THREADS = 64 * WN * WK, NP = PIECES<T>, FN = TN / WN / 32, FK = TK / WK / 32;
    constexpr int PN = TN + 32, PK = TK + 32;                              // row pitches in LDS, elements
    constexpr int GC = MS * TN / 8 / THREADS, GROW = THREADS / (TN / 8);     // 8-element pieces of G a thread loads, and the rows between them
    constexpr int AB = MS * TK / 16 >= THREADS ? 16 : 8;                    // bytes of A in a piece
    constexpr int AC = MS * TK / AB / THREADS, AROW = THREADS / (TK / AB);
    static_assert(GC >= 1 && AC >= 1 && GC * GROW == MS && AC * AROW == MS, "the loads cover a stage");
    // the two buffers are objects of their own, and every access names its own at compile time: reads of one may pass writes of the other
    __shared__ __attribute__((aligned(16))) __bf16 sg0[NP][MS * PN], sg1[NP][MS * PN], sa0[MS * PK], sa1[MS * PK];
    auto g_of = [&](auto buf, int p) -> __bf16* { return decltype(buf)::value ? sg1[p] : sg0[p]; };
    auto a_of = [&](auto buf) -> __bf16* { return decltype(buf)::value ? sa1 : sa0; };

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // Workgroups go to the eight XCDs in turn; each XCD gets a run of tiles, so that the ones that share rows and columns meet in its L2: split by split, and
    // within a split strips of eight tiles of G's columns.
    const int tiles = a.tiles_n * a.tiles_k, total = tiles * a.splits;
    const int wg = total % 8 == 0 ? (int)(blockIdx.x % 8) * (total / 8) + (int)(blockIdx.x / 8) : (int)blockIdx.x;
    const int split = wg / tiles, tile = wg % tiles, strip = tile / (8 * a.tiles_k);
    const int height = min(8, a.tiles_n - 8 * strip), in_strip = tile - strip * 8 * a.tiles_k;
    const int n0 = (8 * strip + in_strip % height) * TN, k0 = (in_strip / height) * TK;
    const long long m_begin = split * a.share, m_end = min(m_begin + a.share, a.rows);

    // This thread's pieces of a stage.  PLAIN: loads without conditions, so that the loop has no branches but the column sums' and its parts can be interleaved.  The rows
    // behind the share's end read its last row again: their part of A counts as zero in the product, and the column sums leave them out (a product with zero would turn an
    // infinity into a NaN; as a branch, 389017 x 256 x 256 fp32 in 159 us against 162 by a product and 163 by selects).  Columns behind the end read other elements of
    // the row and only reach outputs that do not exist; a piece that the end cuts holds the last eight columns instead.
    const int gcol = (tid % (TN / 8)) * 8, grow = tid / (TN / 8), acol = (tid % (TK / AB)) * AB, arow = tid / (TK / AB);
    const int g_left = a.n - n0 - gcol;
    const bool a_in = k0 + acol < a.nb * S8_BLOCK;
    const int g_at = PLAIN ? min(n0 + gcol, a.n - 8) : n0 + gcol, a_at = PLAIN && !a_in ? 0 : k0 + acol;
    const long long g_row = a.ldg * (long long)sizeof(T), a_row = (long long)a.nb * S8_BLOCK;      // bytes
    vec_t<T> rg[GC][8 / VEC<T>];
    uint32_t ra[AC][AB / 4], re[AC];
    const long long m_last = (m_end - 1) / MS * MS;                         // the share's last stage (shares start at multiples of MS)
    auto load_g = [&](long long m0, int i) {
        if constexpr (PLAIN) {
            const long long m = min(m0, m_last);
            const uint32_t at = min((uint32_t)(grow + i * GROW), (uint32_t)(m_end - 1 - m)) * (uint32_t)g_row + (uint32_t)g_at * (uint32_t)sizeof(T);
            const T* p = reinterpret_cast<const T*>((const uint8_t*)a.g + m * g_row + at);
#pragma unroll
            for (int q = 0; q < 8 / VEC<T>; ++q) rg[i][q] = load_any(p + q * VEC<T>);
        } else {
            const long long m = m0 + grow + i * GROW;
            const int left = m < m_end ? g_left : 0;
#pragma unroll
            for (int q = 0; q < 8 / VEC<T>; ++q) rg[i][q] = load_vec((const T*)a.g + m * a.ldg + g_at + q * VEC<T>, left - q * VEC<T>);
        }
    };
    auto load_a = [&](long long m0, int i) {
        long long m = m0 + arow + i * AROW;
        const bool in = m < m_end;
        const uint8_t *p, *e;
        if constexpr (PLAIN) {
            m = min(m0, m_last);
            const uint32_t r = min((uint32_t)(arow + i * AROW), (uint32_t)(m_end - 1 - m));
            p = a.codes + m * a_row + (r * (uint32_t)a_row + (uint32_t)a_at);
            e = a.steps + m * a.nb + (r * (uint32_t)a.nb + (uint32_t)a_at / S8_BLOCK);
        } else {
            p = a.codes + m * a_row + a_at;
            e = a.steps + m * a.nb + a_at / S8_BLOCK;
#pragma unroll
            for (int j = 0; j < AB / 4; ++j) ra[i][j] = 0;
            re[i] = 0;
        }
        if (PLAIN || (a_in && in)) {
            if constexpr (AB == 16) {
                const u32x4 v = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
                for (int j = 0; j < 4; ++j) ra[i][j] = v[j];
            } else {
                const uint2 v = *reinterpret_cast<const uint2*>(p);
                ra[i][0] = v.x, ra[i][1] = v.y;
            }
            re[i] = *e;
        }
    };
    float bias[8] = {};
    const bool with_bias = a.db && k0 == 0;
    // The conversion of the stage from row m0 on into buffer buf, in units of one 16-byte store each: piece p of G's loads i, and eight bytes h of A's loads i
    float rest[8];                                                          // of G: what the pieces so far leave
    auto convert_g = [&](auto buf, int i, int p, long long m0, auto sums) {
        if (p == 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) rest[j] = (float)rg[i][j / VEC<T>][j % VEC<T>];
            if constexpr (decltype(sums)::value) {
                const bool there = m0 + grow + i * GROW < m_end;
                if (there) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) bias[j] += rest[j];
                }
            }
        }
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = high_halves(rest[2 * j], rest[2 * j + 1]);
        if constexpr (NP == 1) w = __builtin_bit_cast(u32x4, rg[i][0]);
        *reinterpret_cast<u32x4*>(g_of(buf, p) + (grow + i * GROW) * PN + gcol) = w;
#pragma unroll
        for (int j = 0; j < 8; ++j) rest[j] -= high_part(rest[j]);
    };
    auto convert_a = [&](auto buf, int i, int h, long long m0) {
        const float step = m0 + arow + i * AROW < m_end ? s8_step(re[i]) : 0.f;
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t c = ra[i][2 * h + j];
            float v[4];
            s8_magnitudes(c, v);
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] *= step;
            // the signs: bytes 0, 1 and 2, 3 moved to the tops of two bf16 pairs
            w[2 * j] = high_halves(v[0], v[1]) | (__builtin_amdgcn_perm(0u, c, 0x010c000cu) & 0x80008000u);
            w[2 * j + 1] = high_halves(v[2], v[3]) | (__builtin_amdgcn_perm(0u, c, 0x030c020cu) & 0x80008000u);
        }
        *reinterpret_cast<u32x4*>(a_of(buf) + (arow + i * AROW) * PK + acol + 8 * h) = w;
    };
    // unit u of them, and the load of the stage from row next on as soon as the registers are free
    constexpr int G_UNITS = GC * NP, UNITS = G_UNITS + AC * (AB / 8);
    auto convert = [&](auto buf, int u, long long m0, long long next, auto sums) {
        if (u < G_UNITS) {
            convert_g(buf, u / NP, u % NP, m0, sums);
            if (u % NP == 0) load_g(next, u / NP);
        } else {
            const int i = (u - G_UNITS) / (AB / 8), h = (u - G_UNITS) % (AB / 8);
            convert_a(buf, i, h, m0);
            if (h == AB / 8 - 1) load_a(next, i);
        }
    };

    f32x16 acc[FN][FK] = {};
    const int wn = (wave / WK) * (TN / WN), wk = (wave % WK) * (TK / WK);
    const int at_row = (lane >> 5) * 8 + ((lane >> 2) & 3), at_col = ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
    auto read_a = [&](auto buf, int s, bf16x8 (&fa)[FK]) {
#pragma unroll
        for (int j = 0; j < FK; ++j) fa[j] = read_columns(a_of(buf) + (16 * s + at_row) * PK + wk + 32 * j + at_col, PK);
    };
    auto read_g = [&](auto buf, int f) {
        const int s = f / (NP * FN), p = f / FN % NP, i = f % FN;
        return read_columns(g_of(buf, p) + (16 * s + at_row) * PN + wn + 32 * i + at_col, PN);
    };

    // Stage i is multiplied while stage i + 1 goes from registers to the other LDS buffer and stage i + 2 is under way from memory: each load has a whole
    // stage's time.  The products of each fragment of G stand between the read of the next fragment and a unit of the conversion, and stay there: left
    // to itself the compiler puts all products first, both waves of a SIMD do so at the same time, and either the matrix or the vector pipe rests.
    using first = std::integral_constant<int, 0>;
    using second = std::integral_constant<int, 1>;
    auto work = [&](auto sums) {
#pragma unroll
        for (int i = 0; i < GC; ++i) load_g(m_begin, i);
#pragma unroll
        for (int i = 0; i < AC; ++i) load_a(m_begin, i);
#pragma unroll
        for (int u = 0; u < UNITS; ++u) convert(first(), u, m_begin, m_begin + MS, sums);
        lds_barrier();
        auto stage = [&](auto here, auto there, long long m0) {
            constexpr int STEPS = MS / 16, PER_STEP = NP * FN, FRAGMENTS = STEPS * PER_STEP;
            bf16x8 fa[2][FK], fg[2];
            read_a(here, 0, fa[0]);
            fg[0] = read_g(here, 0);
#pragma unroll
            for (int f = 0; f < FRAGMENTS; ++f) {
                if (f + 1 < FRAGMENTS) fg[(f + 1) % 2] = read_g(here, f + 1);
                if (f % PER_STEP == PER_STEP - 1 && f + 1 < FRAGMENTS) read_a(here, f / PER_STEP + 1, fa[(f / PER_STEP + 1) % 2]);
#pragma unroll
                for (int j = 0; j < FK; ++j)
                    acc[f % FN][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fg[f % 2], fa[f / PER_STEP % 2][j], acc[f % FN][j], 0, 0, 0);
#pragma unroll
                for (int u = 0; u < UNITS; ++u)
                    if (u * FRAGMENTS / UNITS == f) convert(there, u, m0 + MS, m0 + 2 * MS, sums);
                if constexpr (PLAIN) __builtin_amdgcn_sched_barrier(0);
            }
            lds_barrier();
        };
        for (long long m0 = m_begin; m0 < m_end; m0 += 2 * MS) {             // (a stage behind the end adds nothing)
            stage(first(), second(), m0);
            stage(second(), first(), m0 + MS);
        }
    };
    if (with_bias)                                                          // (shares are never empty)
        work(std::true_type());
    else
        work(std::false_type());

    // the column of G at a place of the tile; a.n where there is none.  A piece that the end cuts holds the last eight columns: the first of them belong to
    // the piece before it
    auto output = [&](int at) {
        const int left = a.n - n0 - (at & ~7);
        if (!PLAIN || left >= 8 || left <= 0) return n0 + at;
        const int c = n0 + at - (8 - left);
        return c >= n0 + (at & ~7) ? c : a.n;
    };
    // the tile: a lane holds column (lane & 31) and rows 8 (q / 4) + 4 (lane / 32) + q % 4 of each 32 x 32 block
    auto write = [&](auto* dw, auto* db) {
        using W = std::remove_pointer_t<decltype(dw)>;
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int j = 0; j < FK; ++j) {
                const int col = k0 + wk + 32 * j + (lane & 31);
#pragma unroll
                for (int q = 0; q < 16; ++q) {
                    const int row = output(wn + 32 * i + 8 * (q / 4) + 4 * (lane >> 5) + q % 4);
                    if (row < a.n && col < a.k) dw[(size_t)row * a.k + col] = (W)acc[i][j][q];
                }
            }
        if (with_bias) {                                                    // the same for the whole workgroup
            __syncthreads();
            float* fold = reinterpret_cast<float*>(&sg0[0][0]);             // [waves][TN]
            static_assert(WN * WK * TN * 4 <= (int)sizeof(sg0), "the column sums fit");
#pragma unroll
            for (int j = 0; j < 8; ++j) {
#pragma unroll
                for (int off = TN / 8; off < 64; off *= 2) bias[j] += __shfl_xor(bias[j], off);
                if (lane < TN / 8) fold[wave * TN + gcol + j] = bias[j];
            }
            __syncthreads();
            for (int c = tid; c < TN; c += THREADS) {
                float s = 0.f;
                for (int r = 0; r < WN * WK; ++r) s += fold[r * TN + c];
                if (output(c) < a.n) db[output(c)] = (W)s;
            }
        }
    };
    if (a.type == SPF_TYPE_F32)
        write((float*)a.dw + (size_t)split * a.n * a.k, (float*)a.db + (size_t)split * a.n);
    else if (a.type == SPF_TYPE_BF16)
        write((__bf16*)a.dw, (__bf16*)a.db);
    else
        write((_Float16*)a.dw, (_Float16*)a.db);
}

// out[i] (+)= sum over the splits: eight threads share them, each takes every eighth in order.  A workgroup adds 128 outputs at a time; it walks over them, as a grid with
// one for each would pass a launch's 2^32 threads at 2^31 outputs.
constexpr long long REDUCE_GROUPS = 1 << 22;
template <typename W>
__global__ void __launch_bounds__(256)
wgrad8_reduce_kernel(const float* __restrict__ tiles, int splits, long long count, W* dw, const float* __restrict__ bias_tiles, int n, W* db, int add) {
    __shared__ float part[8][128];
    const int lane = threadIdx.x & 31, k = threadIdx.x >> 5, at = threadIdx.x;
    const long long groups = (count + 127) / 128, all = groups + (db ? (n + 127) / 128 : 0);       // the last ones add db
    for (long long group = blockIdx.x; group < all; group += gridDim.x) {
        const bool is_bias = group >= groups;
        const long long first = (is_bias ? group - groups : group) * 128, c = first + 4 * lane, len = is_bias ? n : count;
        const float* src = is_bias ? bias_tiles : tiles;
        float s[4] = {};
#pragma unroll 8
        for (int i = k; i < splits; i += 8) {
            const vec_t<float> v = load_vec(src + (size_t)i * len + c, len - c);
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] += v[j];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) part[k][4 * lane + j] = s[j];
        __syncthreads();
        if (at < 128 && first + at < len) {
            float t = part[0][at];
#pragma unroll
            for (int i = 1; i < 8; ++i) t += part[i][at];
            W* out = (is_bias ? db : dw) + first + at;
            *out = (W)(add ? (float)*out + t : t);
        }
        __syncthreads();
    }
}

constexpr int STAGE = 32;
// The loads without conditions need eight columns of G and 32-bit offsets within a stage
bool plain(int64_t n, int64_t ldg, int type) { return n >= 8 && ldg * type_size(type) < (1ll << 31) / STAGE; }

struct plan {
    int side, tiles_n, tiles_k, splits;
    int64_t share;
};
// The tile and the number of row splits with the least estimated time.  A large tile reads its operands least often, but a layer that does not fill it wastes it,
// and a workgroup with a large tile has a compute unit to itself; splits fill the chip and shorten the chain of stages, but each leaves an fp32 tile that is written
// and read again.  The constants are microseconds on MI355X: a stage with all its compute unit's workgroups at work, a stage of a workgroup that is alone there,
// and 5 MB of split tiles.  Measured with the tile set by hand, 256 / 128 / 64 wide: 8192 rows, 4096 x 4096: fp32 621, 783, 1282 us, bf16 261, 437, 652;
// 389017 rows, 256 x 256, fp32: 154, 180, 259; 400000 rows, 128 x 256, fp32: 137, 101, 157; 1000 rows, 2000 x 2000, bf16: 47, 25, 25.
struct tile_kind {
    int side, resident[3];           // workgroups of a compute unit; by SPF_TYPE_*
    float busy[3], alone[3];
};
const tile_kind TILES[] = {{256, {1, 1, 1}, {2.5f, 1.13f, 1.8f}, {1.1f, 1.1f, 1.1f}}, {128, {2, 3, 2}, {1.56f, 1.08f, 1.25f}, {1.0f, 0.75f, 0.85f}},
                           {64, {3, 5, 4}, {0.88f, 0.73f, 0.8f}, {0.6f, 0.6f, 0.6f}}};

plan plan_of(int64_t rows, int64_t n, int64_t k, int type) {
    const int64_t stages = (rows + STAGE - 1) / STAGE;
    plan best = {};
    float least = INFINITY;
    for (const tile_kind& t : TILES) {
        if (t.side > 64 && n < 8) continue;                       // (only the 64-wide kernel has a form with conditions)
        const int64_t tiles_n = (n + t.side - 1) / t.side, tiles_k = (k + t.side - 1) / t.side, tiles = tiles_n * tiles_k, slots = 256 * t.resident[type];
        for (int64_t want = 1; want <= stages && want <= 1024; want = want < slots / tiles && 2 * want > slots / tiles ? slots / tiles : 2 * want) {
            const int64_t per = (stages + want - 1) / want, splits = (stages + per - 1) / per, wgs = tiles * splits;
            const int64_t rounds = (wgs + slots - 1) / slots, beside = wgs >= slots ? t.resident[type] : (wgs + 255) / 256;
            const float full = t.busy[type] * (float)beside / (float)t.resident[type], stage = full > t.alone[type] ? full : t.alone[type];
            // (three stages' time to fill and to leave)
            const float us = (float)rounds * (float)(per + 3) * stage + (splits > 1 ? 3.f + (float)splits * (float)n * (float)k * (8.f / 5e6f) : 0.f);
            if (us < least) {
                least = us;
                best = {t.side, (int)tiles_n, (int)tiles_k, (int)splits, per * STAGE};
            }
        }
    }
    return best;
}

// db alone, for a layer whose weight is not trained: the bits of wgrad8_kernel's, in whose order the rows are added.  There a row of a stage belongs to one of 16 threads (32
// with 64-wide tiles) that hold a column; the `fold` of them that share a wave are added as a tree, the waves one after the other.  Here a workgroup takes those threads of a
// share side by side for 128 (64) columns, eight a thread, and wgrad8_reduce_kernel adds the shares.  389017 x 256 fp32 (254 shares): 75 us,
// 5.3 TB/s; 8192 x 4096 bf16, which a 4096-wide layer does not share out: 59 us, a chain of loads.
template <typename T>
__global__ void __launch_bounds__(256)
bias_sums_kernel(const T* __restrict__ g, long long ldg, long long rows, long long share, int n, int slots, int fold, float* __restrict__ lines) {
    constexpr int V = VEC<T>;
    __shared__ float part[256 * 8];
    const int across = 256 / slots, t = threadIdx.x % across, slot = threadIdx.x / across, width = across * 8;
    const int first = blockIdx.x * width, c = first + t * 8;
    const long long begin = blockIdx.y * share, end = min(begin + share, rows);
    float s[8] = {}, f[V];
#pragma unroll 8
    for (long long row = begin + slot; row < end; row += slots) {
#pragma unroll
        for (int q = 0; q < 8 / V; ++q) {
            to_f32<T>(load_vec(g + row * ldg + c + q * V, n - c - q * V, c + q * V > 0), f);
#pragma unroll
            for (int i = 0; i < V; ++i) s[q * V + i] += f[i];
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) part[slot * width + t * 8 + i] = s[i];
    for (int off = 1; off < fold; off *= 2) {                               // part[d] += part[d + off] for d = 0, 2 off, 4 off ...
        __syncthreads();
        for (int i = threadIdx.x; i < slots / (2 * off) * width; i += 256) {
            const int at = i / width * 2 * off * width + i % width;
            part[at] += part[at + off * width];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < width && first + i < n; i += 256) {
        float sum = 0.f;
        for (int d = 0; d < slots; d += fold) sum += part[d * width + i];
        lines[(size_t)blockIdx.y * n + first + i] = sum;
    }
}

template <typename T> void launch(const wgrad8_args& a, const plan& p, bool is_plain, hipStream_t s) {
    const unsigned wgs = (unsigned)(p.tiles_n * p.tiles_k * p.splits);
    if (p.side == 256) {
        // eight waves; the more pieces G has, the fewer of its fragments a wave should read: 64 x 128 outputs a wave take 10 fragments from LDS for 24
        // products of fp32, 128 x 64 would take 14
        constexpr int WN = PIECES<T> > 1 ? 4 : 2;
        wgrad8_kernel<T, 256, 256, WN, 8 / WN, STAGE, true><<<wgs, 512, 0, s>>>(a);
    } else if (p.side == 128)
        wgrad8_kernel<T, 128, 128, 2, 2, STAGE, true><<<wgs, 256, 0, s>>>(a);
    else if (is_plain)
        wgrad8_kernel<T, 64, 64, 2, 2, STAGE, true><<<wgs, 256, 0, s>>>(a);
    else
        wgrad8_kernel<T, 64, 64, 2, 2, STAGE, false><<<wgs, 256, 0, s>>>(a);
}

const char* bad_sizes(int64_t rows, int64_t n, int64_t k) {
    if (rows < 0 || n < 0 || k < 0) return "negative size";
    if (rows >= (1ll << 31) || n > (1 << 20) || k > (1 << 20) || n * k > (1ll << 34)) return "rows < 2^31, widths <= 2^20 and a product <= 2^34 are supported";
    return nullptr;
}
bool misaligned(const void* p, int size) { return ((uintptr_t)p & (uintptr_t)(size - 1)) != 0; }

}  // namespace

extern "C" {

int64_t spf_wgrad8_workspace_floats(int64_t rows, int64_t n, int64_t cols, int32_t type, int32_t accumulate) {
    if (bad_sizes(rows, n, cols) || !type_ok(type) || rows == 0 || n == 0 || cols == 0) return 0;
    const int64_t splits = plan_of(rows, n, cols, type).splits;
    return splits > 1 || accumulate ? splits * n * (cols + 1) : 0;
}

int32_t spf_wgrad8_tile(int64_t rows, int64_t n, int64_t cols, int32_t type) {
    if (bad_sizes(rows, n, cols) || !type_ok(type) || rows == 0 || n == 0 || cols == 0) return 0;
    return plan_of(rows, n, cols, type).side;
}

int spf_wgrad8(const void* g, int32_t type, int64_t ldg, const uint8_t* codes, const uint8_t* steps, int64_t rows, int64_t n, int64_t cols, void* dw, void* db,
               int32_t wtype, int32_t accumulate, float* workspace, void* stream) {
    const char* who = "spf_wgrad8";
    if (!type_ok(type) || !type_ok(wtype)) return fail(SPF_EINVAL, "%s: unknown element type", who);
    if (const char* why = bad_sizes(rows, n, cols)) return fail(SPF_EINVAL, "%s: %s", who, why);
    if (rows == 0 || n == 0 || cols == 0) return SPF_OK;
    const plan p = plan_of(rows, n, cols, type);
    const bool direct = p.splits == 1 && !accumulate, is_plain = plain(n, ldg, type);
    if (!g || !codes || !steps || !dw || (!direct && !workspace)) return fail(SPF_EINVAL, "%s: null pointer", who);
    if (ldg < 0 || (p.side > 64 && !is_plain)) return fail(SPF_EINVAL, "%s: a row stride below 0, or of 64 MB or more in a large product", who);
    if (misaligned(g, type_size(type)) || misaligned(codes, 16) || misaligned(dw, type_size(wtype)) || misaligned(db, type_size(wtype)) || misaligned(workspace, 4))
        return fail(SPF_EINVAL, "%s: misaligned pointer", who);
    wgrad8_args a = {g, ldg, codes, steps, rows, p.share, (int)n, (int)cols, (int)((cols + S8_BLOCK - 1) / S8_BLOCK), p.tiles_n, p.tiles_k, p.splits, dw, db, wtype};
    float* bias_tiles = db && !direct ? workspace + (int64_t)p.splits * n * cols : nullptr;
    if (!direct) a.dw = workspace, a.db = bias_tiles, a.type = SPF_TYPE_F32;
    hipStream_t s = (hipStream_t)stream;
    if (type == SPF_TYPE_F32) launch<float>(a, p, is_plain, s);
    else if (type == SPF_TYPE_BF16) launch<__bf16>(a, p, is_plain, s);
    else launch<_Float16>(a, p, is_plain, s);
    if (!direct) {
        const int64_t all = (n * cols + 127) / 128 + (db ? (n + 127) / 128 : 0), groups = all < REDUCE_GROUPS ? all : REDUCE_GROUPS;
        const auto reduce = [&](auto* w, auto* b) { wgrad8_reduce_kernel<<<(unsigned)groups, 256, 0, s>>>(workspace, p.splits, n * cols, w, bias_tiles, (int)n, b, accumulate); };
        if (wtype == SPF_TYPE_F32) reduce((float*)dw, (float*)db);
        else if (wtype == SPF_TYPE_BF16) reduce((__bf16*)dw, (__bf16*)db);
        else reduce((_Float16*)dw, (_Float16*)db);
    }
    SPF_LAUNCH_CHECK(who);
    return SPF_OK;
}

int64_t spf_wgrad8_bias_workspace_floats(int64_t rows, int64_t n, int64_t cols, int32_t type) {
    if (bad_sizes(rows, n, cols) || !type_ok(type) || rows == 0 || n == 0 || cols == 0) return 0;
    return plan_of(rows, n, cols, type).splits * n;
}

int spf_wgrad8_bias(const void* g, int32_t type, int64_t ldg, int64_t rows, int64_t n, int64_t cols, void* db, int32_t wtype, int32_t accumulate, float* workspace, void* stream) {
    const char* who = "spf_wgrad8_bias";
    if (!type_ok(type) || !type_ok(wtype)) return fail(SPF_EINVAL, "%s: unknown element type", who);
    if (const char* why = bad_sizes(rows, n, cols)) return fail(SPF_EINVAL, "%s: %s", who, why);
    if (rows == 0 || n == 0 || cols == 0) return SPF_OK;
    if (!g || !db || !workspace) return fail(SPF_EINVAL, "%s: null pointer", who);
    if (ldg < 0) return fail(SPF_EINVAL, "%s: row stride", who);
    if (misaligned(g, type_size(type)) || misaligned(db, type_size(wtype)) || misaligned(workspace, 4)) return fail(SPF_EINVAL, "%s: misaligned pointer", who);
    const plan p = plan_of(rows, n, cols, type);
    const int slots = p.side == 64 ? 32 : 16, fold = 512 / p.side, width = 256 / slots * 8;
    const dim3 grid((unsigned)((n + width - 1) / width), p.splits);
    hipStream_t s = (hipStream_t)stream;
    const auto sums = [&](auto* x) { bias_sums_kernel<<<grid, 256, 0, s>>>(x, ldg, rows, p.share, (int)n, slots, fold, workspace); };
    if (type == SPF_TYPE_F32) sums((const float*)g);
    else if (type == SPF_TYPE_BF16) sums((const __bf16*)g);
    else sums((const _Float16*)g);
    const auto reduce = [&](auto* b) { wgrad8_reduce_kernel<<<(unsigned)((n + 127) / 128), 256, 0, s>>>(nullptr, p.splits, 0, (decltype(b))nullptr, workspace, (int)n, b, accumulate); };
    if (wtype == SPF_TYPE_F32) reduce((float*)db);
    else if (wtype == SPF_TYPE_BF16) reduce((__bf16*)db);
    else reduce((_Float16*)db);
    SPF_LAUNCH_CHECK(who);
    return SPF_OK;
}

}  // extern "C"
