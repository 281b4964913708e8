// skm_fp8.hip -- matrix products of 8-bit floats with a scale for each block of 128 (gfx950 only).
//
// A block of 128 numbers is stored as 8-bit floats (e4m3 or e5m2) times 2^e, e the smallest integer with
// max |x| <= top * 2^e (top 448 / 57344, the format's largest number).  A power of two costs nothing against any other
// scale -- the 8-bit number has the same significand either way -- and buys two things: x * 2^-e is exact, so the
// rounding to 8 bits is the only one, and the matrix cores apply 2^e themselves (v_mfma_scale_f32_*_f8f6f4 takes one
// E8M0 byte per row and 32 k), so the product of blocks needs no vector-ALU work on the accumulators.
//
// Storage: q [rows][Kp] bytes, Kp = K rounded up to 128, zeros behind K; one scale byte (e + 127) per row and block of
// 128 k, [rows][S] with S = Kp / 128 rounded up to 4 -- also where 128 rows share their scale (tiles of weights): the
// kernels then have one operand layout, at 0.8 % more bytes.
#include "skm_ops.h"

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

#define FP8_BLOCK 128
// least e: the smallest number of either format (2^-16 in e5m2) times 2^e is still a normal float32 and bf16 number; only a
// block whose largest number is below 57344 * 2^-110 (4e-29) loses digits to this
#define FP8_MIN_EXP (-110)

static inline long fp8_kpad(long K) { return (K + FP8_BLOCK - 1) / FP8_BLOCK * FP8_BLOCK; }
static inline long fp8_sstride(long K) { return (fp8_kpad(K) / FP8_BLOCK + 3) / 4 * 4; }

extern "C" long skm_fp8_row_bytes(long K) { return K < 1 ? 0 : fp8_kpad(K); }
extern "C" long skm_fp8_scale_bytes(long K) { return K < 1 ? 0 : fp8_sstride(K); }

// ------------------------------------------------------------------ quantization ------

// e of a block whose largest finite magnitude is `top` (>= 0): 448 = 1.75 * 2^8, 57344 = 1.75 * 2^15
__device__ __forceinline__ int fp8_exponent(float top, int fmt)
{
    const unsigned u = __float_as_uint(top);
    if (u == 0) return 0;
    const int e = (int)(u >> 23) - 127 - (fmt == SKM_FP8_E4M3 ? 8 : 15) + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return e < FP8_MIN_EXP ? FP8_MIN_EXP : e;
}

__device__ __forceinline__ float fp8_pow2(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }

__device__ __forceinline__ float fp8_finite_abs(float x)
{
    const float a = fabsf(x);
    return a < __builtin_inff() ? a : 0.f;      // NaN and infinities do not set the scale
}

// four scaled numbers -> four bytes, to nearest even.  The scale keeps finite numbers inside the format; the instruction
// makes NaN of an infinity in e4m3, which has none.
template <int FMT>
__device__ __forceinline__ unsigned fp8_pack4(float a, float b, float c, float d)
{
    if (FMT == SKM_FP8_E4M3) {
        const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
    }
    const int lo = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_bf8_f32(c, d, lo, true);
}

// n numbers from p on, 8 at most, zeros behind them
template <typename T>
__device__ __forceinline__ void load8(const T *p, int n, float (&v)[8])
{
    typedef T v8 __attribute__((ext_vector_type(8)));
    if (n >= 8) {
        const v8 x = load_any<v8>(p);
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = (float)x[q];
    } else {
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = q < n ? (float)p[q] : 0.f;
    }
}

struct RowsArgs {
    const void *x;
    long M, ldx;
    int K, KB, S;           // blocks of a row, scale bytes of a row
    uint8_t *q, *s;
};

// a lane's value from another lane of its 16 (CTRL 0x120 + n: n lanes on)
template <int CTRL>
__device__ __forceinline__ float lanes16_ror(float v)
{
    const int i = __float_as_int(v);
    return __int_as_float(__builtin_amdgcn_update_dpp(i, i, CTRL, 0xF, 0xF, false));
}

// Blocks of 1 x 128: 16 lanes per block, 8 numbers a lane, the block's largest by four DPP steps; no LDS, no barrier.
// Bound by memory: 8192 x 4096 bf16 in 19.4 us, 5.2 TB/s (a large copy: 5.0); rows at odd addresses (4095) 22.8 us.
template <typename T, int FMT>
__global__ __launch_bounds__(256) void k_fp8_rows(RowsArgs a)
{
    const long b = ((long)blockIdx.x * 256 + threadIdx.x) >> 4;
    const int l = threadIdx.x & 15;
    const long row = b / a.KB;
    const int kb = (int)(b - row * a.KB);
    if (row >= a.M) return;                 // whole blocks of 16 lanes
    const int k = kb * FP8_BLOCK + l * 8;
    float v[8];
    load8(static_cast<const T *>(a.x) + row * a.ldx + k, a.K - k, v);
    float top = 0.f;
#pragma unroll
    for (int q = 0; q < 8; ++q) top = fmaxf(top, fp8_finite_abs(v[q]));
    top = fmaxf(top, lanes16_ror<0x128>(top));
    top = fmaxf(top, lanes16_ror<0x124>(top));
    top = fmaxf(top, lanes16_ror<0x122>(top));
    top = fmaxf(top, lanes16_ror<0x121>(top));
    const int e = fp8_exponent(top, FMT);
    const float f = fp8_pow2(-e);
    uint2 o;
    o.x = fp8_pack4<FMT>(v[0] * f, v[1] * f, v[2] * f, v[3] * f);
    o.y = fp8_pack4<FMT>(v[4] * f, v[5] * f, v[6] * f, v[7] * f);
    *reinterpret_cast<uint2 *>(a.q + row * (long)a.KB * FP8_BLOCK + k) = o;
    if (l == 0) a.s[row * a.S + kb] = (uint8_t)(e + 127);
    if (kb == a.KB - 1 && l < a.S - a.KB) a.s[row * a.S + a.KB + l] = 127;
}

struct TileArgs {
    const void *x;
    long R, ldx, sx;        // rows, their stride, distance between matrices
    int C;                  // columns
    uint8_t *q, *s;         // [z][R][Cp], [z][R][Sc]              (tiles only)
    uint8_t *qt, *st;       // [z][C][Rp], [z][C][Sr]              NULL: not wanted
    long Cp, Rp;
    int Sc, Sr;
    // columns by plan: rows in the plan's order, every expert from a new tile
    const int32_t *tiles, *count, *pair;    // count[0] tiles of (expert, row, rows, 0)
    int slots;
    const float *w;         // weight of a pair or NULL
};

// blocks of 128 x 128 (COLS = 0) or 128 x 1 (COLS = 1): one workgroup per 128 x 128; a thread holds 8 columns of 8
// consecutive rows, so that a transposed block goes through LDS in 8-byte pieces.  One read of x serves both results of
// weights.  Bound by memory: 8192 x 4096 bf16 tiles 21.9 us (4.6 TB/s), tiles and their transpose 26.5 us (5.1), columns
// 21.9 us (4.6); rows at odd addresses (4095) 41-46 us, an 8-byte piece then lies in two cache lines more often.
template <typename T, int FMT, int COLS>
__global__ __launch_bounds__(256) void k_fp8_tiles(TileArgs a)
{
    __shared__ float red[16][FP8_BLOCK];
    __shared__ __align__(16) uint8_t lt[FP8_BLOCK][FP8_BLOCK];
    const int tid = threadIdx.x, cg = tid & 15, rg = tid >> 4;
    const int c0 = blockIdx.x * FP8_BLOCK, c = c0 + cg * 8;
    const long rb = blockIdx.y, z = blockIdx.z;
    long r0 = rb * FP8_BLOCK;
    int rows = (int)(a.R - r0 < FP8_BLOCK ? a.R - r0 : FP8_BLOCK);
    if (COLS && a.tiles) {
        if (rb >= a.count[0]) return;
        r0 = a.tiles[rb * 4 + 1];
        rows = a.tiles[rb * 4 + 2];
    }
    const T *x = static_cast<const T *>(a.x) + z * a.sx;
    float v[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = rg * 8 + i;
        if (r < rows && c < a.C) {
            long src = r0 + r;
            float w = 1.f;
            if (COLS && a.pair) {
                const int pr = a.pair[src];
                src = pr / a.slots;
                if (a.w) w = a.w[pr];
            }
            load8(x + src * a.ldx + c, a.C - c, v[i]);
            if (COLS && a.w)
#pragma unroll
                for (int q = 0; q < 8; ++q) v[i][q] *= w;
        } else {
#pragma unroll
            for (int q = 0; q < 8; ++q) v[i][q] = 0.f;
        }
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, fp8_finite_abs(v[i][q]));
        red[rg][cg * 8 + q] = m;
    }
    __syncthreads();
    if (tid < FP8_BLOCK) {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) m = fmaxf(m, red[i][tid]);
        red[0][tid] = m;
    }
    __syncthreads();
    int e[8];
    if (COLS) {
#pragma unroll
        for (int q = 0; q < 8; ++q) e[q] = fp8_exponent(red[0][cg * 8 + q], FMT);
    } else {
        float m = fmaxf(red[0][tid & 63], red[0][64 + (tid & 63)]);
        m = wave_max(m);
#pragma unroll
        for (int q = 0; q < 8; ++q) e[q] = fp8_exponent(m, FMT);
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        const float f = fp8_pow2(-e[q]);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i][q] *= f;
    }
    if (!COLS && a.q) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = rg * 8 + i;
            if (r < rows) {
                uint2 o;
                o.x = fp8_pack4<FMT>(v[i][0], v[i][1], v[i][2], v[i][3]);
                o.y = fp8_pack4<FMT>(v[i][4], v[i][5], v[i][6], v[i][7]);
                *reinterpret_cast<uint2 *>(a.q + (z * a.R + r0 + r) * a.Cp + c) = o;
            }
        }
        if (tid < rows) {
            uint8_t *s = a.s + (z * a.R + r0 + tid) * a.Sc;
            s[blockIdx.x] = (uint8_t)(e[0] + 127);
            if (blockIdx.x == gridDim.x - 1)
                for (int b = gridDim.x; b < a.Sc; ++b) s[b] = 127;
        }
    }
    if (!a.qt) return;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        uint2 o;
        o.x = fp8_pack4<FMT>(v[0][q], v[1][q], v[2][q], v[3][q]);
        o.y = fp8_pack4<FMT>(v[4][q], v[5][q], v[6][q], v[7][q]);
        *reinterpret_cast<uint2 *>(&lt[cg * 8 + q][(rg ^ cg) * 8]) = o;     // 16 lanes meet different banks
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int col = i * 32 + (tid >> 3), piece = tid & 7;
        if (c0 + col < a.C) {
            const int x = col >> 3;         // rows 16 piece .. + 7 and + 8 .. + 15: a pair of 8-byte pieces, in order or not
            const i32x4 v = *reinterpret_cast<const i32x4 *>(&lt[col][((2 * piece) ^ (x & 14)) * 8]);
            *reinterpret_cast<i32x4 *>(a.qt + (z * a.C + c0 + col) * a.Rp + rb * FP8_BLOCK + piece * 16) =
                x & 1 ? __builtin_shufflevector(v, v, 2, 3, 0, 1) : v;
        }
    }
    if (tid < FP8_BLOCK && c0 + tid < a.C) {
        const float m = red[0][tid];
        uint8_t *s = a.st + (z * a.C + c0 + tid) * a.Sr;
        s[rb] = (uint8_t)((COLS ? fp8_exponent(m, FMT) : e[0]) + 127);
        if (rb == gridDim.y - 1)
            for (int b = gridDim.y; b < a.Sr; ++b) s[b] = 127;
    }
}

#define FP8_IN_TYPES(F, ...)                                                             \
    switch (dtype * 2 + fmt) {                                                           \
    case SKM_DT_F32 * 2 + SKM_FP8_E4M3: F(float, SKM_FP8_E4M3, ##__VA_ARGS__); break;    \
    case SKM_DT_F32 * 2 + SKM_FP8_E5M2: F(float, SKM_FP8_E5M2, ##__VA_ARGS__); break;    \
    case SKM_DT_BF16 * 2 + SKM_FP8_E4M3: F(bf16_t, SKM_FP8_E4M3, ##__VA_ARGS__); break;  \
    case SKM_DT_BF16 * 2 + SKM_FP8_E5M2: F(bf16_t, SKM_FP8_E5M2, ##__VA_ARGS__); break;  \
    case SKM_DT_F16 * 2 + SKM_FP8_E4M3: F(f16_t, SKM_FP8_E4M3, ##__VA_ARGS__); break;    \
    default: F(f16_t, SKM_FP8_E5M2, ##__VA_ARGS__); break;                               \
    }

static int fp8_check_types(const char *who, int dtype, int fmt)
{
    SKM_REQUIRE(dtype == SKM_DT_F32 || dtype == SKM_DT_BF16 || dtype == SKM_DT_F16, "%s: element type %d", who, dtype);
    SKM_REQUIRE(fmt == SKM_FP8_E4M3 || fmt == SKM_FP8_E5M2, "%s: 8-bit format %d", who, fmt);
    return SKM_OK;
}

extern "C" int skm_fp8_rows(void *ctx_, const void *x, int dtype, long M, int K, long ldx, int fmt, void *q, void *s,
                            void *stream)
{
    SkmCtx *ctx = static_cast<SkmCtx *>(ctx_);
    SKM_REQUIRE(ctx && M >= 0 && K >= 1 && ldx >= K && (M == 0 || (x && q && s)), "skm_fp8_rows: bad argument");
    if (int rc = fp8_check_types("skm_fp8_rows", dtype, fmt)) return rc;
    if (M == 0) return SKM_OK;
    RowsArgs a{x, M, ldx, K, (int)(fp8_kpad(K) / FP8_BLOCK), (int)fp8_sstride(K), static_cast<uint8_t *>(q),
               static_cast<uint8_t *>(s)};
    SkmDeviceGuard guard(ctx);
    hipStream_t st = (hipStream_t)stream;
    SkmProfScope ps(ctx, "k_fp8_rows", st);
    const long most = SKM_MAX_GROUPS * 16 / a.KB;       // rows of a launch
    for (long m = 0; m < M; m += most) {
        a.M = M - m < most ? M - m : most;
        a.x = static_cast<const char *>(x) + m * ldx * skm_dt_size(dtype);
        a.q = static_cast<uint8_t *>(q) + m * a.KB * FP8_BLOCK;
        a.s = static_cast<uint8_t *>(s) + m * a.S;
        const unsigned grid = (unsigned)((a.M * a.KB + 15) / 16);
#define ROWS_LAUNCH(T, FMT) hipLaunchKernelGGL((k_fp8_rows<T, FMT>), dim3(grid), dim3(256), 0, st, a)
        FP8_IN_TYPES(ROWS_LAUNCH)
        SKM_HIP(hipGetLastError());
    }
    return SKM_OK;
}

extern "C" int skm_fp8_tiles(void *ctx_, const void *w, int dtype, int batch, int N, int K, long ldw, long sw, int fmt,
                             void *q, void *s, void *qt, void *st_, void *stream)
{
    SkmCtx *ctx = static_cast<SkmCtx *>(ctx_);
    SKM_REQUIRE(ctx && batch >= 0 && N >= 1 && K >= 1 && ldw >= K && (batch == 0 || (w && q && s)) && !qt == !st_,
                "skm_fp8_tiles: bad argument");
    if (int rc = fp8_check_types("skm_fp8_tiles", dtype, fmt)) return rc;
    if (batch == 0) return SKM_OK;
    SKM_REQUIRE(batch <= 65535 && fp8_kpad(N) / FP8_BLOCK <= 65535 && fp8_kpad(K) / FP8_BLOCK <= SKM_MAX_GROUPS,
                "skm_fp8_tiles: too large");
    TileArgs a{};
    a.x = w; a.R = N; a.ldx = ldw; a.sx = sw; a.C = K;
    a.q = static_cast<uint8_t *>(q); a.s = static_cast<uint8_t *>(s);
    a.qt = static_cast<uint8_t *>(qt); a.st = static_cast<uint8_t *>(st_);
    a.Cp = fp8_kpad(K); a.Rp = fp8_kpad(N); a.Sc = (int)fp8_sstride(K); a.Sr = (int)fp8_sstride(N);
    SkmDeviceGuard guard(ctx);
    hipStream_t st = (hipStream_t)stream;
    SkmProfScope ps(ctx, "k_fp8_tiles", st);
    const dim3 grid((unsigned)(a.Cp / FP8_BLOCK), (unsigned)(a.Rp / FP8_BLOCK), (unsigned)batch);
#define TILES_LAUNCH(T, FMT, COLS) hipLaunchKernelGGL((k_fp8_tiles<T, FMT, COLS>), grid, dim3(256), 0, st, a)
    FP8_IN_TYPES(TILES_LAUNCH, 0)
    SKM_HIP(hipGetLastError());
    return SKM_OK;
}

extern "C" int skm_fp8_columns(void *ctx_, const void *x, int dtype, long R, int C, long ldx, int fmt,
                               const int32_t *tiles, const int32_t *tile_count, long max_tiles, const int32_t *pair,
                               int slots, const float *weights, void *qt, void *st_, void *stream)
{
    SkmCtx *ctx = static_cast<SkmCtx *>(ctx_);
    SKM_REQUIRE(ctx && R >= 0 && C >= 1 && ldx >= C, "skm_fp8_columns: bad argument");
    SKM_REQUIRE(!tiles || (tile_count && pair && slots >= 1 && max_tiles >= 0), "skm_fp8_columns: incomplete plan");
    SKM_REQUIRE(tiles || !weights, "skm_fp8_columns: weights go with a plan");
    if (int rc = fp8_check_types("skm_fp8_columns", dtype, fmt)) return rc;
    const long blocks = tiles ? max_tiles : fp8_kpad(R) / FP8_BLOCK;
    if (blocks == 0) return SKM_OK;
    SKM_REQUIRE(x && qt && st_, "skm_fp8_columns: bad argument");
    SKM_REQUIRE(blocks <= 65535 && fp8_kpad(C) / FP8_BLOCK <= SKM_MAX_GROUPS,
                "skm_fp8_columns: more than 65535 blocks of rows or 2^31 - 128 columns");
    TileArgs a{};
    a.x = x; a.R = R; a.ldx = ldx; a.C = C;
    a.qt = static_cast<uint8_t *>(qt); a.st = static_cast<uint8_t *>(st_);
    a.Rp = blocks * FP8_BLOCK; a.Sr = (int)fp8_sstride(a.Rp);
    a.tiles = tiles; a.count = tile_count; a.pair = tiles ? pair : nullptr; a.slots = slots; a.w = weights;
    SkmDeviceGuard guard(ctx);
    hipStream_t st = (hipStream_t)stream;
    SkmProfScope ps(ctx, "k_fp8_columns", st);
    const dim3 grid((unsigned)(fp8_kpad(C) / FP8_BLOCK), (unsigned)blocks, 1);
    FP8_IN_TYPES(TILES_LAUNCH, 1)
    SKM_HIP(hipGetLastError());
    return SKM_OK;
}

// ------------------------------------------------------------------ product ------
struct Fp8Args {
    const uint8_t *A, *B;   // [M][lda], [N][ldb] bytes
    const uint8_t *sA, *sB; // [M][SA], [N][SB]
    long lda, ldb;
    int SA, SB;
    int M, N;
    long rowsA;             // rows that A has (by plan: tokens or pairs)
    int kb0, kb1;           // blocks of 128 k
    void *C;
    long ldc;
    int accumulate;
    int c_bf16;             // (host) C's type
    int tile_rows;          // (host) rows of a plan's tile
    long mean_blocks;       // (host) blocks of an expert on average
    int tiles_m, tiles_n;
    long zC;                // split over k: slab z holds the partial sums of its blocks, zC elements apart
    int slabs;
    // experts: row tiles from a table, the B operand by expert
    const int32_t *tiles, *tile_count, *pair;
    int slots;              // A row of a pair: pair / slots; 0: the plan's own order
    long eB, esB;           // B, sB of the next expert
    // weight gradient: blockIdx.y = expert, its blocks first[e] .. first[e + 1]
    const int32_t *first;
    long eC;
};

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// eight 8-bit floats times a power of two as bf16: exact (4 significant bits, normal numbers: FP8_MIN_EXP)
template <int FMT>
__device__ __forceinline__ bf16x8 fp8_to_bf16(int lo, int hi, float scale)
{
    bf16x2 v[4];
    if (FMT == SKM_FP8_E4M3) {
        v[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)lo, scale, false);
        v[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)lo, scale, true);
        v[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)hi, scale, false);
        v[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)hi, scale, true);
    } else {
        v[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8((unsigned)lo, scale, false);
        v[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8((unsigned)lo, scale, true);
        v[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8((unsigned)hi, scale, false);
        v[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8((unsigned)hi, scale, true);
    }
    bf16x8 o;
#pragma unroll
    for (int q = 0; q < 8; ++q) o[q] = v[q >> 1][q & 1];
    return o;
}

typedef __attribute__((address_space(3))) void *lds_ptr;
typedef __attribute__((address_space(1))) const void *glb_ptr;

// C = A B'.  Workgroup: 4 waves as 2 x 2, a wave MT x NT tiles of 32 x 32 (v_mfma_scale_f32_32x32x64_f8f6f4), one block
// of 128 k a stage, DEPTH (2, 3) stages in LDS filled by global loads that go there directly.
//   LDS: a row's 128 bytes of a stage are one line; its 16-byte pieces are stored at piece ^ ((row >> 1) & 7), so that the
//   lanes of a read phase (16 rows, the same piece) meet different bank groups (row & 7 costs 4 cycles more per read,
//   measured).  The loads put consecutive lanes'
//   pieces at consecutive addresses, so the exchange is made on the global side, within the line.
//   The scales come the same way, a dword (four blocks) of every row in every fourth stage.
//   The 8-bit matrix instructions add 8 products at a time in a window of 13 bits below the largest of the 8 (a product
//   2^-14 of it is lost, measured), the sums of 8 in float32.  Of each 8, up to 7 lose less than 2^-13 of the largest: at
//   worst 2^-10 of the sum of the products' magnitudes, 1.4e-5 (2^-16) of the result's norm with random operands.  A
//   bf16 result's own rounding is 2^-8 of it, an f16 one's 2^-11; where the products cancel, what is cut off can exceed
//   either.  That is the price of twice the rate, taken for results of 16 bits.  A float32 result is wanted for its digits
//   (weight gradients that are added up, rows that a gradient is formed with), so there the operands become bf16 --
//   exactly, scale included -- and the products are exact and the sums float32, at half the rate.
//   Which of the 64 k of a product lies where in the operand registers does not matter as long as A and B agree and a
//   scale covers all of them: a lane's 32 bytes are 32 consecutive k of its row here.
// A stage is two halves of 64 k in two sets of fragments: while one set is multiplied, the other is read.  Stage s:
//   read half 1 of s; multiply half 0 (all but the last row of tiles)
//   wait for the own reads and for the own loads of stage s + 1; barrier: nobody reads stage s any more, stage s + 1 is
//   complete
//   issue the loads of stage s + DEPTH into the buffer that is free; multiply the rest of half 0
//   read half 0 of s + 1; multiply half 1
// so a load has DEPTH - 1/2 stages to arrive, an LDS read half a stage, and the barrier stands among multiplications
// that are under way already.
// Why 256 x 256: a stage's 64 KB of LDS reads (128 x 128: 32 KB a quarter of the products) fit under its multiplications,
// and every operand byte is loaded half as often.
// Measured: 8192 x 8192 x 8192 to bf16 436 to 477 us by the run, 2300 to 2520 TFLOP/s (matrix pipe busy 63 % of the cycles at
// 1.93 GHz: the engine clock gives way to power on random operands); 4096 x 8192 x 4096 at 2600.  To float32 880 us, 1250
// TFLOP/s (63 %, 1.88 GHz), as fast as a plain bf16 product of the size on this GPU (1241).
template <int MT, int NT> struct Fp8Lds {
    // [DEPTH stages of (BM + BN) rows of 128 bytes][two groups of four blocks of (BM + BN) scale dwords]
    // 256 x 128 has room for three stages, and a load then has two and a half to arrive.
    static constexpr int BM = MT * 64, BN = NT * 64, DEPTH = MT == 4 && NT == 2 ? 3 : 2;
    static constexpr int STAGE = (BM + BN) * FP8_BLOCK, GROUP = (BM + BN) * 4, BYTES = DEPTH * STAGE + 2 * GROUP;
};

// one tile: `rows` rows from row0 on, the columns from col0 on, blocks kb0 .. kb1
template <int MT, int NT, int FA, int FB, typename TO>
__device__ __forceinline__ void fp8_tile(const Fp8Args &g, uint8_t *sh, int rows, long row0, int col0, int kb0, int kb1,
                                         const uint8_t *B, const uint8_t *sB, TO *C)
{
    typedef Fp8Lds<MT, NT> Lds;
    constexpr int BM = Lds::BM, BN = Lds::BN, DEPTH = Lds::DEPTH, STAGE = Lds::STAGE, GROUP = Lds::GROUP, LOADS = (MT + NT) * 2;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1, r = lane & 31, h = lane >> 5;
    const int cols = g.N - col0;

    // From this tile's first row (A by plan: from A's first), so that a lane's offset is 32 bits wide.
    const bool by_pair = g.tiles && g.slots;
    const long a0 = by_pair ? 0 : row0;
    const uint8_t *ba = g.A + a0 * g.lda + (long)kb0 * FP8_BLOCK, *bb = B + col0 * g.ldb + (long)kb0 * FP8_BLOCK;
    const uint8_t *bsa = g.sA + a0 * g.SA, *bsb = sB + (long)col0 * g.SB;
    // one row of A (B) per 8 lanes and load: rows behind the last repeat it
    const int lr = lane >> 3;
#define FP8_PIECE(I) (((lane & 7) ^ ((((I) & 1) << 2) | (lr >> 1))) * 16)   // rows 8 I + lr: exchanged by (row >> 1) & 7
    unsigned oa[MT * 2], ob[NT * 2];
#pragma unroll
    for (int i = 0; i < MT * 2; ++i) {
        int rr = (wave * MT * 2 + i) * 8 + lr;
        rr = rr < rows ? rr : rows - 1;
        if (by_pair) rr = g.pair[row0 + rr] / g.slots;
        oa[i] = (unsigned)rr * (unsigned)g.lda + FP8_PIECE(i);
    }
#pragma unroll
    for (int i = 0; i < NT * 2; ++i) {
        int cc = (wave * NT * 2 + i) * 8 + lr;
        cc = cc < cols ? cc : cols - 1;
        ob[i] = (unsigned)cc * (unsigned)g.ldb + FP8_PIECE(i);
    }
#undef FP8_PIECE
    // scales: 64 rows a load, the rows of A, then the columns of B; waves take turns (one too many repeats the last)
    constexpr int CHUNKS = (BM + BN) / 64, MINE = (CHUNKS + 3) / 4;
    unsigned os[MINE];
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        int rr = (wave + 4 * i < CHUNKS ? wave + 4 * i : CHUNKS - 1) * 64 + lane;
        if (rr < BM) {
            rr = rr < rows ? rr : rows - 1;
            if (by_pair) rr = g.pair[row0 + rr] / g.slots;
            os[i] = (unsigned)rr * (unsigned)g.SA;
        } else {
            rr = rr - BM < cols ? rr - BM : cols - 1;
            os[i] = (unsigned)rr * (unsigned)g.SB;
        }
    }

    // loads of the stage S (blocks from kb0) into buffer ST; scales of the blocks 4 G .. 4 G + 3
#define FP8_ISSUE1(S, L, BUF)                                                                                          \
    {                                                                                                                  \
        const uint8_t *p_ = ((L) < MT * 2 ? ba : bb) + (long)(S) * FP8_BLOCK;                                          \
        const unsigned o_ = (L) < MT * 2 ? oa[(L) < MT * 2 ? (L) : 0] : ob[(L) < MT * 2 ? 0 : (L) - MT * 2];            \
        const int row8_ = (L) < MT * 2 ? wave * MT * 2 + (L) : BM / 8 + wave * NT * 2 + (L) - MT * 2;                   \
        __builtin_amdgcn_global_load_lds((glb_ptr)(p_ + o_), (lds_ptr)((BUF) + row8_ * 8 * FP8_BLOCK), 16, 0, 0);      \
    }
#define FP8_ISSUE(S, BUF)                                                                                              \
    _Pragma("unroll") for (int l_ = 0; l_ < LOADS; ++l_) FP8_ISSUE1(S, l_, BUF)
#define FP8_SCALES(G, BUF)                                                                                             \
    _Pragma("unroll") for (int i = 0; i < MINE; ++i) {                                                                 \
        const int c = wave + 4 * i < CHUNKS ? wave + 4 * i : CHUNKS - 1;                                               \
        const uint8_t *l = (c * 64 < BM ? bsa : bsb) + (long)(G) * 4;                                                  \
        __builtin_amdgcn_global_load_lds((glb_ptr)(l + os[i]), (lds_ptr)((BUF) + c * 256), 4, 0, 0);                   \
    }

    f32x16 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.f;

    // this lane's pieces of a half H: 4 H + 2 h and the next, exchanged by (row >> 1) & 7 = (r >> 1) & 7
    const int x7 = (r >> 1) & 7;
    int at[2][2];
#pragma unroll
    for (int H = 0; H < 2; ++H)
#pragma unroll
        for (int u = 0; u < 2; ++u) at[H][u] = r * FP8_BLOCK + ((H * 4 + h * 2 + u) ^ x7) * 16;
    i32x8 fa[2][MT], fb[2][NT];
    int sa[MT], sb[NT], na[MT], nb[NT];
    // fragment F of half H: rows of A, then columns of B
#define FP8_READ1(H, F, BUF)                                                                                           \
    {                                                                                                                  \
        const uint8_t *p_ = (BUF) + ((F) < MT ? wm * MT + (F) : MT + wn * NT + (F)) * 32 * FP8_BLOCK;                  \
        const i32x4 lo_ = *reinterpret_cast<const i32x4 *>(p_ + at[H][0]), hi_ = *reinterpret_cast<const i32x4 *>(p_ + at[H][1]); \
        const i32x8 v_ = __builtin_shufflevector(lo_, hi_, 0, 1, 2, 3, 4, 5, 6, 7);                                    \
        if ((F) < MT) fa[H][(F) < MT ? (F) : 0] = v_;                                                                  \
        else fb[H][(F) < MT ? 0 : (F) - MT] = v_;                                                                      \
    }
#define FP8_READ(H, BUF)                                                                                               \
    _Pragma("unroll") for (int f = 0; f < MT + NT; ++f) FP8_READ1(H, f, BUF)
#define FP8_READ_SCALES(KB, BUF)                                                                                           \
    {                                                                                                                  \
        const uint8_t *l = (BUF) + r * 4 + ((KB) & 3);                                                                 \
        _Pragma("unroll") for (int i = 0; i < MT; ++i) na[i] = l[(wm * MT + i) * 128];                                 \
        _Pragma("unroll") for (int j = 0; j < NT; ++j) nb[j] = l[(BM + (wn * NT + j) * 32) * 4];                       \
    }
#define FP8_TILE(H, I, J)                                                                                              \
    acc[I][J] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[H][J], fa[H][I], acc[I][J], FB, FA, 0, sb[J], 0, sa[I]);
    // Float32 results, a half in U units: unit u multiplies eight k of every lane of row u / 4 of the wave's tiles with its
    // NT columns and converts for later: the next unit's row, and in the second half of the units the columns of the next
    // half.  So the conversions (one instruction per two numbers) stand beside multiplications that do not need them.
    constexpr int U = MT * 4;
    bf16x8 xa[2], xb[2][NT][4];
#define FP8_SCALE(S) __uint_as_float((unsigned)(S) << 23)
#define FP8_XA(V, T, S) fp8_to_bf16<FA>((V)[2 * (T)], (V)[2 * (T) + 1], FP8_SCALE(S))
#define FP8_XB(V, T, S) fp8_to_bf16<FB>((V)[2 * (T)], (V)[2 * (T) + 1], FP8_SCALE(S))
#define FP8_UNIT(H, Q, SNA, SNB)                                                                                       \
    {                                                                                                                  \
        _Pragma("unroll") for (int j_ = 0; j_ < NT; ++j_) acc[(Q) / 4][j_] =                                           \
            __builtin_amdgcn_mfma_f32_32x32x16_bf16(xb[H][j_][(Q) & 3], xa[(Q) & 1], acc[(Q) / 4][j_], 0, 0, 0);       \
        if ((Q) + 1 < U) xa[((Q) + 1) & 1] = FP8_XA(fa[H][((Q) + 1) / 4 < MT ? ((Q) + 1) / 4 : 0], ((Q) + 1) & 3, sa[((Q) + 1) / 4 < MT ? ((Q) + 1) / 4 : 0]); \
        else xa[((Q) + 1) & 1] = FP8_XA(fa[(H) ^ 1][0], 0, SNA[0]);                                                    \
        constexpr int EACH_ = NT * 8 / U;                                                                              \
        if ((Q) >= U / 2) {                                                                                            \
            _Pragma("unroll") for (int c_ = 0; c_ < EACH_; ++c_) {                                                     \
                const int n_ = ((Q) - U / 2) * EACH_ + c_;                                                             \
                xb[(H) ^ 1][n_ / 4 < NT ? n_ / 4 : 0][n_ & 3] =                                                        \
                    FP8_XB(fb[(H) ^ 1][n_ / 4 < NT ? n_ / 4 : 0], n_ & 3, SNB[n_ / 4 < NT ? n_ / 4 : 0]);              \
                asm volatile("" : "+v"(xb[(H) ^ 1][n_ / 4 < NT ? n_ / 4 : 0][n_ & 3]));         /* not later */        \
            }                                                                                                          \
        }                                                                                                              \
    }
    // the columns first
#define FP8_READ1B(H, F, BUF) FP8_READ1(H, ((F) < NT ? MT + (F) : (F) - NT), BUF)
#define FP8_SCALE_GROUP(KB) (sh + DEPTH * STAGE + (((KB) >> 2) & 1) * GROUP)
    const int n = kb1 - kb0;
    if (n > 0) {
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) {   // behind the last stage the last one again: every stage has as many loads
            const int si = i < n ? i : n - 1;
            FP8_SCALES((kb0 + si) >> 2, FP8_SCALE_GROUP(kb0 + si))
            FP8_ISSUE(si, sh + i * STAGE)
        }
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((DEPTH - 1) * (LOADS + MINE)) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        FP8_READ(0, sh)
        FP8_READ_SCALES(kb0, FP8_SCALE_GROUP(kb0))
#pragma unroll
        for (int i = 0; i < MT; ++i) sa[i] = na[i];
#pragma unroll
        for (int j = 0; j < NT; ++j) sb[j] = nb[j];
        if (sizeof(TO) == 4) {
            xa[0] = FP8_XA(fa[0][0], 0, sa[0]);
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int t = 0; t < 4; ++t) xb[0][j][t] = FP8_XB(fb[0][j], t, sb[j]);
        }
    }
    // Behind the barrier of a stage: the loads of stage s2 fill the buffer that it frees while the next stage is read.  The
    // two buffers (and the two groups of scales, or the same group with the same bytes) do not overlap: restrict lets the
    // compiler mix the instructions.
    auto late = [&](int s2, int kb, uint8_t *__restrict__ fill, const uint8_t *__restrict__ next,
                    uint8_t *__restrict__ fill_scales, const uint8_t *__restrict__ next_scales) __attribute__((always_inline)) {
        FP8_SCALES((kb0 + s2) >> 2, fill_scales)
        if (sizeof(TO) == 4) {
            FP8_READ_SCALES(kb + 1, next_scales)
            constexpr int POST = 4 + U, EACH = (LOADS + POST - 1) / POST;
#pragma unroll
            for (int u = 0; u < POST; ++u) {
                if (u < 4) {
                    FP8_UNIT(0, U - 4 + u, sa, sb)
                } else {
                    FP8_UNIT(1, u - 4, na, nb)
                }
#pragma unroll
                for (int l = u * EACH; l < (u + 1) * EACH; ++l)
                    if (l < LOADS) FP8_ISSUE1(s2, l, fill)
                if (u >= 4 && u < 4 + MT + NT) {
                    FP8_READ1B(0, u - 4, next)
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
            // In this order: the four waves' loads take 16 cycles each on the way to the cache, a wave that waits to issue
            // one multiplies nothing, so there is one beside every multiplication (64 cycles).
            constexpr int EACH = (LOADS + (MT + 1) * NT - 1) / ((MT + 1) * NT);
#pragma unroll
            for (int u = 0; u < (MT + 1) * NT; ++u) {
                if (u < NT) {
                    FP8_TILE(0, MT - 1, u)
                } else {
                    FP8_TILE(1, (u - NT) / NT, (u - NT) % NT)
                }
#pragma unroll
                for (int l = u * EACH; l < (u + 1) * EACH; ++l)
                    if (l < LOADS) FP8_ISSUE1(s2, l, fill)
                if (u >= NT && u < NT + MT + NT) {
                    FP8_READ1(0, u - NT, next)
                }
                if (u == (MT + 2 * NT < (MT + 1) * NT ? MT + 2 * NT : (MT + 1) * NT - 1)) {
                    FP8_READ_SCALES(kb + 1, next_scales)
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    // One straight block per stage, without a branch: behind the last stage the last one is loaded again into the free
    // buffer, and what is read of it is not used; a group's scales are loaded again with each of its stages.
    int cur = 0, nxt = STAGE;               // where stages s and s + 1 are
    for (int s = 0; s < n; ++s) {
        const int kb = kb0 + s, s2 = s + DEPTH < n ? s + DEPTH : n - 1;
        if (sizeof(TO) == 4) {
#pragma unroll
            for (int u = 0; u < U - 4; ++u) {
                FP8_UNIT(0, u, sa, sb)
                constexpr int EACH = (MT + NT + U - 5) / (U - 4);
#pragma unroll
                for (int f = u * EACH; f < (u + 1) * EACH; ++f)
                    if (f < MT + NT) FP8_READ1B(1, f, sh + cur)
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
            constexpr int EACH = (MT + NT + (MT - 1) * NT - 1) / ((MT - 1) * NT);
#pragma unroll
            for (int u = 0; u < (MT - 1) * NT; ++u) {
                FP8_TILE(0, u / NT, u % NT)
#pragma unroll
                for (int f = u * EACH; f < (u + 1) * EACH; ++f)
                    if (f < MT + NT) FP8_READ1(1, f, sh + cur)
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        // the multiplications stand in front of the barrier (an empty statement that takes their results; it reads nothing)
#pragma unroll
        for (int i = 0; i < MT - 1; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) asm volatile("" : "+a"(acc[i][j]));
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((DEPTH - 2) * (LOADS + MINE)) : "memory");
        __builtin_amdgcn_sched_barrier(0);
        late(s2, kb, sh + cur, sh + nxt, FP8_SCALE_GROUP(kb0 + s2), FP8_SCALE_GROUP(kb + 1));
        cur = nxt;
        nxt = nxt + STAGE == DEPTH * STAGE ? 0 : nxt + STAGE;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < MT; ++i) sa[i] = na[i];
#pragma unroll
        for (int j = 0; j < NT; ++j) sb[j] = nb[j];
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // nothing lands in LDS behind the loop
#undef FP8_SCALE_GROUP
#undef FP8_READ1
#undef FP8_ISSUE1
#undef FP8_TILE
#undef FP8_ISSUE
#undef FP8_SCALES
#undef FP8_READ
#undef FP8_READ_SCALES
#undef FP8_SCALE
#undef FP8_XA
#undef FP8_XB
#undef FP8_UNIT
#undef FP8_READ1B
    // Result of a 32 x 32 tile (B's columns are the rows of the instruction): lane: row lane & 31 of C; register q: column
    // (q & 3) + 8 (q >> 2) + 4 (lane >> 5).  32 rows at a time go through the wave's own part of LDS, so that 16 bytes of a
    // row are stored by one lane and a row's bytes by neighbouring ones.
    constexpr int CW = NT * 32, PITCH = CW + 4, VE = 16 / sizeof(TO), PER = CW / VE, RSTEP = 64 / PER;
    static_assert(Lds::BYTES >= 4 * 32 * PITCH * sizeof(float), "the result's rows fit where the stages were");
    float *lw = reinterpret_cast<float *>(sh) + wave * 32 * PITCH;
    typedef TO vo __attribute__((ext_vector_type(VE)));
    __syncthreads();                        // the other waves have read their last stage
    const int sr = lane / PER, scol = (lane % PER) * VE, gc = wn * CW + scol;
    // cols - gc columns from here on: VE of them or fewer
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 v = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                *reinterpret_cast<f32x4 *>(lw + r * PITCH + j * 32 + 8 * q + 4 * h) = v;
            }
        wave_sync();
#pragma unroll
        for (int t = 0; t < 32 / RSTEP; ++t) {
            const int lrow = t * RSTEP + sr, rr = (wm * MT + i) * 32 + lrow;
            float v[VE];
#pragma unroll
            for (int q = 0; q < VE; q += 4) {
                const f32x4 x = *reinterpret_cast<const f32x4 *>(lw + lrow * PITCH + scol + q);
                v[q] = x[0]; v[q + 1] = x[1]; v[q + 2] = x[2]; v[q + 3] = x[3];
            }
            if (rr < rows && gc < cols) {
                TO *d = C + (row0 + rr) * g.ldc + col0 + gc;
                if (gc + VE <= cols) {
                    vo o;
                    if (g.accumulate) {
                        o = load_any<vo>(d);
#pragma unroll
                        for (int q = 0; q < VE; ++q) v[q] += (float)o[q];
                    }
#pragma unroll
                    for (int q = 0; q < VE; ++q) o[q] = (TO)v[q];
                    store_any(d, o);
                } else {
#pragma unroll
                    for (int q = 0; q < VE; ++q)
                        if (gc + q < cols) d[q] = (TO)(g.accumulate ? (float)d[q] + v[q] : v[q]);
                }
            }
        }
        wave_sync();
    }
}

template <int MT, int NT, int FA, int FB, typename TO>
__global__ __launch_bounds__(256, (MT * NT > 4) ? 1 : 2) void k_gemm_fp8(Fp8Args g)
{
    constexpr int BM = MT * 64, BN = NT * 64;
    // One array: with two of them hipcc waits for the loads in flight in front of every read of LDS.
    __shared__ __align__(16) uint8_t sh[Fp8Lds<MT, NT>::BYTES];

    int tm, tn;
    {   // workgroups w, w + 8, ... share an XCD: an XCD takes a run of consecutive tiles, columns of 8 row tiles at a time
        const int tiles_m = g.tiles ? g.tile_count[0] : g.tiles_m;     // by plan: of the grid's, those that there are
        const int total = tiles_m * g.tiles_n;
        const int q = total / 8, rem = total % 8, x = blockIdx.x % 8, i = blockIdx.x / 8;
        if (i >= q + (x < rem ? 1 : 0)) return;
        int t = x * q + (x < rem ? x : rem) + i;
        const int group = 8 * g.tiles_n, gi = t / group, m0 = gi * 8;
        const int gm = tiles_m - m0 < 8 ? tiles_m - m0 : 8;
        t -= gi * group;
        tm = m0 + t % gm;
        tn = t / gm;
    }
    int kb0 = g.kb0, kb1 = g.kb1;
    int rows = g.M - tm * BM;               // rows of this tile
    long row0 = (long)tm * BM;
    const uint8_t *B = g.B, *sB = g.sB;
    TO *C = static_cast<TO *>(g.C);
    if (g.tiles) {
        const int32_t *t = g.tiles + (long)tm * 4;
        B += t[0] * g.eB;
        sB += t[0] * g.esB;
        row0 = t[1];
        rows = t[2];
    } else if (g.first) {
        const int e = blockIdx.y;
        kb0 = g.first[e];
        kb1 = g.first[e + 1];
        C += e * g.eC;
    } else if (g.slabs > 1) {
        const int z = blockIdx.y, n = kb1 - kb0;
        kb1 = kb0 + (int)((long)n * (z + 1) / g.slabs);
        kb0 += (int)((long)n * z / g.slabs);
        C += z * g.zC;
    }
    // A last tile of half the rows or less is half the work: experts of about 1000 rows often have one.  Little comes of
    // it while the tiles are dealt in the table's order and the last round over the CUs is nearly empty (8191 tokens, 4 of
    // 32 experts, 2048 x 4096, the whole chain in four runs of either: 377 against 383 us, runs 5 us apart; 8192 tokens, 2 of
    // 16, a training step: 663 and 664)
    if constexpr (MT == 4)
        if (rows <= BM / 2) {
            fp8_tile<MT / 2, NT, FA, FB, TO>(g, sh, rows, row0, tn * BN, kb0, kb1, B, sB, C);
            return;
        }
    fp8_tile<MT, NT, FA, FB, TO>(g, sh, rows, row0, tn * BN, kb0, kb1, B, sB, C);
}

template <int MT, int NT, typename TO>
static void fp8_launch(const Fp8Args &g, int fa, int fb, unsigned gx, unsigned gy, hipStream_t st)
{
    const dim3 grid(gx, gy), block(256);
    switch (fa * 2 + fb) {
    case 0: hipLaunchKernelGGL((k_gemm_fp8<MT, NT, 0, 0, TO>), grid, block, 0, st, g); break;
    case 1: hipLaunchKernelGGL((k_gemm_fp8<MT, NT, 0, 1, TO>), grid, block, 0, st, g); break;
    case 2: hipLaunchKernelGGL((k_gemm_fp8<MT, NT, 1, 0, TO>), grid, block, 0, st, g); break;
    default: hipLaunchKernelGGL((k_gemm_fp8<MT, NT, 1, 1, TO>), grid, block, 0, st, g); break;
    }
}

// ------------------------------------------------------------------ few rows ------
// What A may be where it is quantized on the way: a float matrix in rows of ldx.
struct Fp8Float {
    const void *x;
    long ldx;
    int K;
};

// C = A B' for up to 16 MT rows of A (or tiles of up to 16 rows of an expert): the bytes of B are what counts, each is
// read once, straight into registers.  A workgroup holds 16 NT columns, its waves share the k blocks in groups of four
// (one scale dword per row and group) and add their parts through LDS in a fixed order.  v_mfma_scale_f32_16x16x128:
// B's columns are the rows of the instruction, so a lane ends with 4 consecutive columns of one row of C.
// A lane (row r of 16, quarter g) holds bytes 16 g .. and 64 + 16 g .. of a block's 128: a load covers 64 consecutive
// bytes of 16 rows.
// XT = uint8_t: A is quantized already.  Otherwise a float type: every wave quantizes the blocks of its four k blocks, as
// k_fp8_rows does it (16 lanes a block, so one row's four blocks at a time), into LDS -- the same work in every workgroup,
// under the latency of B's bytes, costs less than a launch before this one.  LDS: a row's 512 bytes, the 16-byte pieces of
// each 256 exchanged by the row, so that the 16 rows that read the same piece meet different banks.
// Bound by the bytes of B and, for one row, by the launch: 1 x 4096 x 4096 6.7 us, 64 x 8192 x 4096 18.5 us (two waves a
// SIMD, half of their time without an instruction to issue: too little of B is in flight), 8 tokens of 4
// places over 64 experts of 2048 x 2048 24 us (about 105 MB, 4.4 TB/s).
// By plan every tile of 16 rows reads its expert's weights again and every workgroup quantizes the tile's float rows again:
// 64 experts of 2048 x 4096 with 16 rows each 183 us from 8-bit rows and 276 from float ones (128-row tiles: 141 and 145).
template <int MT, int NT, int FA, int FB, typename TO, typename XT>
__global__ __launch_bounds__(512, 2) void k_gemm_fp8_rows16(Fp8Args g, Fp8Float fx)
{
    constexpr bool FLOAT = sizeof(XT) > 1;
    static_assert(!FLOAT || MT == 1, "float rows are quantized for one row tile");
    // a wave's part of the sums; with float rows also 8 KB + 64 bytes of them.  As many as there are waves: a fixed eight
    // would leave room for two workgroups on a CU where four waves are enough for k
    constexpr int PART = (FLOAT && MT * NT * 4 < 33 ? 33 : MT * NT * 4) * 64;
    extern __shared__ __align__(16) float lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int r = lane & 15, q4 = lane >> 4;
    int rows = g.M;
    long row0 = 0;
    const uint8_t *B = g.B, *sB = g.sB;
    if (g.tiles) {
        if ((int)blockIdx.y >= g.tile_count[0]) return;
        const int32_t *t = g.tiles + (long)blockIdx.y * 4;
        B += t[0] * g.eB;
        sB += t[0] * g.esB;
        row0 = t[1];
        rows = t[2];
    }
    const int col0 = blockIdx.x * 16 * NT;
    const uint8_t *pb[NT], *qb[NT], *pa[MT], *qa[MT];
    int src_row = 0;                        // of row r of the tile
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int n = col0 + j * 16 + r < g.N ? col0 + j * 16 + r : g.N - 1;
        pb[j] = B + n * g.ldb + q4 * 16;
        qb[j] = sB + (long)n * g.SB;
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int m = i * 16 + r < rows ? i * 16 + r : rows - 1;
        long src = row0 + m;
        if (g.tiles && g.slots) src = g.pair[src] / g.slots;
        src_row = (int)src;
        if (!FLOAT) {
            pa[i] = g.A + src * g.lda + q4 * 16;
            qa[i] = g.sA + src * g.SA;
        }
    }
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[i][j][q] = 0.f;
    uint8_t *lw = reinterpret_cast<uint8_t *>(lds + wave * PART);
    uint8_t *ls = lw + 16 * 512;            // scales [16][4]

    const int groups = (g.kb1 + 3) / 4;
    for (int gr = wave; gr < groups; gr += waves) {
        const int nb = g.kb1 - gr * 4 < 4 ? g.kb1 - gr * 4 : 4;
        i32x8 w[NT][4], a[MT][4];
        int sw[NT], sx[MT];
        // a short group repeats its first block, unused
#define ROWS16_LOAD(DST, PTR)                                                                                          \
    _Pragma("unroll") for (int b = 0; b < 4; ++b) {                                                                    \
        const uint8_t *p_ = (PTR) + (long)(gr * 4 + (b < nb ? b : 0)) * FP8_BLOCK;                                     \
        const i32x4 lo_ = *reinterpret_cast<const i32x4 *>(p_), hi_ = *reinterpret_cast<const i32x4 *>(p_ + 64);       \
        (DST)[b] = __builtin_shufflevector(lo_, hi_, 0, 1, 2, 3, 4, 5, 6, 7);                                          \
    }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            sw[j] = *reinterpret_cast<const int *>(qb[j] + gr * 4);
            ROWS16_LOAD(w[j], pb[j])
        }
        if (!FLOAT) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                sx[i] = *reinterpret_cast<const int *>(qa[i] + gr * 4);
                ROWS16_LOAD(a[i], pa[i])
            }
        } else {
            // lane: block q4 of the group, numbers 8 r .. 8 r + 7 of it
            const int k = (gr * 4 + q4) * FP8_BLOCK + r * 8;
            const int piece = (q4 & 1) * 8 + (r >> 1), line = (q4 >> 1) * 256;
            for (int m = 0; m < rows; ++m) {
                const XT *x = static_cast<const XT *>(fx.x) + (long)__builtin_amdgcn_readlane(src_row, m) * fx.ldx;
                float v[8];
                load8(x + k, fx.K - k, v);
                float top = 0.f;
#pragma unroll
                for (int q = 0; q < 8; ++q) top = fmaxf(top, fp8_finite_abs(v[q]));
                top = fmaxf(top, lanes16_ror<0x128>(top));
                top = fmaxf(top, lanes16_ror<0x124>(top));
                top = fmaxf(top, lanes16_ror<0x122>(top));
                top = fmaxf(top, lanes16_ror<0x121>(top));
                const int e = fp8_exponent(top, FA);
                const float f = fp8_pow2(-e);
                uint2 o;
                o.x = fp8_pack4<FA>(v[0] * f, v[1] * f, v[2] * f, v[3] * f);
                o.y = fp8_pack4<FA>(v[4] * f, v[5] * f, v[6] * f, v[7] * f);
                *reinterpret_cast<uint2 *>(lw + m * 512 + line + (piece ^ m) * 16 + (r & 1) * 8) = o;
                if (r == 0) ls[m * 4 + q4] = (uint8_t)(e + 127);
            }
            wave_sync();
            sx[0] = *reinterpret_cast<const int *>(ls + r * 4);
#pragma unroll
            for (int b = 0; b < 4; ++b) {               // rows behind the last: whatever is there, for columns not stored
                const uint8_t *p = lw + r * 512 + (b >> 1) * 256;
                const i32x4 lo = *reinterpret_cast<const i32x4 *>(p + (((b & 1) * 8 + q4) ^ r) * 16);
                const i32x4 hi = *reinterpret_cast<const i32x4 *>(p + (((b & 1) * 8 + 4 + q4) ^ r) * 16);
                a[0][b] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            }
            wave_sync();
        }
#undef ROWS16_LOAD
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            if (b < nb) {
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        const int sa = (sx[i] >> (8 * b)) & 255, sb = (sw[j] >> (8 * b)) & 255;
                        if (sizeof(TO) == 4) {
#pragma unroll
                            for (int t = 0; t < 4; ++t) {
                                const bf16x8 xa = fp8_to_bf16<FA>(a[i][b][2 * t], a[i][b][2 * t + 1], fp8_pow2(sa - 127));
                                const bf16x8 xb = fp8_to_bf16<FB>(w[j][b][2 * t], w[j][b][2 * t + 1], fp8_pow2(sb - 127));
                                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xb, xa, acc[i][j], 0, 0, 0);
                            }
                        } else {
                            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[j][b], a[i][b], acc[i][j], FB, FA,
                                                                                         0, sb, 0, sa);
                        }
                    }
            }
        }
    }
    if (FLOAT) __syncthreads();             // the parts of the sums go where the rows were (a wave's own: others' are read)
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) lds[wave * PART + ((i * NT + j) * 4 + q) * 64 + lane] = acc[i][j][q];
    __syncthreads();
    // one wave per 16 x 16 tile of the result, in turn
    for (int t = wave; t < MT * NT; t += waves) {
        float v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = lds[(t * 4 + q) * 64 + lane];
        for (int w = 1; w < waves; ++w)
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] += lds[w * PART + (t * 4 + q) * 64 + lane];
        const int m = t / NT * 16 + r, n = col0 + t % NT * 16 + 4 * q4;
        if (m >= rows) continue;
        TO *c = static_cast<TO *>(g.C) + (row0 + m) * g.ldc + n;
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (n + q < g.N) c[q] = (TO)(g.accumulate ? (float)c[q] + v[q] : v[q]);
    }
}

template <int MT, int NT, typename TO, typename XT>
static void rows16_launch(const Fp8Args &g, const Fp8Float &fx, int fa, int fb, unsigned gy, hipStream_t st)
{
    const int groups = (g.kb1 + 3) / 4;
    const dim3 grid((unsigned)((g.N + 16 * NT - 1) / (16 * NT)), gy), block(64u * (groups < 8 ? groups : 8));
    const size_t lds = (block.x / 64) * (sizeof(XT) > 1 && MT * NT * 4 < 33 ? 33 : MT * NT * 4) * 256;
    switch (fa * 2 + fb) {
    case 0: hipLaunchKernelGGL((k_gemm_fp8_rows16<MT, NT, 0, 0, TO, XT>), grid, block, lds, st, g, fx); break;
    case 1: hipLaunchKernelGGL((k_gemm_fp8_rows16<MT, NT, 0, 1, TO, XT>), grid, block, lds, st, g, fx); break;
    case 2: hipLaunchKernelGGL((k_gemm_fp8_rows16<MT, NT, 1, 0, TO, XT>), grid, block, lds, st, g, fx); break;
    default: hipLaunchKernelGGL((k_gemm_fp8_rows16<MT, NT, 1, 1, TO, XT>), grid, block, lds, st, g, fx); break;
    }
}

template <int MT, int NT, typename XT>
static int rows16_types(const Fp8Args &g, const Fp8Float &fx, int fa, int fb, int dtype, unsigned gy, hipStream_t st)
{
    switch (dtype) {
    case SKM_DT_F32: rows16_launch<MT, NT, float, XT>(g, fx, fa, fb, gy, st); break;
    case SKM_DT_BF16: rows16_launch<MT, NT, bf16_t, XT>(g, fx, fa, fb, gy, st); break;
    default: rows16_launch<MT, NT, f16_t, XT>(g, fx, fa, fb, gy, st); break;
    }
    SKM_HIP(hipGetLastError());
    return SKM_OK;
}

// rows of A: up to 16 (one row tile, quantized on the way if it is a float matrix)
static int rows16_run(SkmCtx *ctx, const Fp8Args &g, const Fp8Float &fx, int x_dtype, int fa, int fb, int dtype, unsigned gy,
                      hipStream_t st)
{
    // threads along x of the narrowest column tiles (a launch has fewer than 2^32)
    const int groups = (g.kb1 + 3) / 4;
    if ((((long)g.N + 15) / 16) * 64 * (groups < 8 ? groups : 8) > 0xFFFFFFFFL) {
        skm_set_error("product of few rows: %d columns of %d blocks are too many for one launch", g.N, g.kb1);
        return SKM_ERR_UNSUPPORTED;
    }
    SkmProfScope ps(ctx, "k_gemm_fp8_rows16", st);
    if (g.A) {
        // two column tiles a workgroup (A's rows are read once per workgroup) where they are enough for every CU:
        // 64 x 8192 x 4096 18.5 us against 27.8, 64 x 4096 x 4096 16.7 against 14.5
        const bool two = (g.N + 31) / 32 >= ctx->cu_count;
        if (g.M > 32 && !g.tiles)
            return two ? rows16_types<4, 2, uint8_t>(g, fx, fa, fb, dtype, gy, st) : rows16_types<4, 1, uint8_t>(g, fx, fa, fb, dtype, gy, st);
        if (g.M > 16 && !g.tiles)
            return two ? rows16_types<2, 2, uint8_t>(g, fx, fa, fb, dtype, gy, st) : rows16_types<2, 1, uint8_t>(g, fx, fa, fb, dtype, gy, st);
        return rows16_types<1, 1, uint8_t>(g, fx, fa, fb, dtype, gy, st);
    }
    switch (x_dtype) {
    case SKM_DT_F32: return rows16_types<1, 1, float>(g, fx, fa, fb, dtype, gy, st);
    case SKM_DT_BF16: return rows16_types<1, 1, bf16_t>(g, fx, fa, fb, dtype, gy, st);
    default: return rows16_types<1, 1, f16_t>(g, fx, fa, fb, dtype, gy, st);
    }
}

// the sum of the slabs, in their order, to the result's type
template <typename TO>
__global__ __launch_bounds__(256) void k_fp8_slabs(const float *__restrict__ part, int slabs, long zC, int M, int N,
                                                   TO *__restrict__ C, long ldc, int accumulate)
{
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long)M * N) return;
    const long m = i / N;
    TO *c = C + m * ldc + (i - m * N);
    float v = 0.f;
    for (int z = 0; z < slabs; ++z) v += part[z * zC + i];
    *c = (TO)(accumulate ? (float)*c + v : v);
}

// Few tiles and a long k: slabs of k blocks, so that there are two workgroups per CU, four blocks a slab at least.
// 1000 x 400 x 30720, float32: 394 us in one slab, 41.5 us (and 7 for their sum) in 16.
static int fp8_slabs(const SkmCtx *ctx, long M, long N, long K)
{
    const long tiles = ((M + 127) / 128) * ((N + 127) / 128), kb = fp8_kpad(K) / FP8_BLOCK;
    if (tiles > ctx->cu_count) return 1;
    long z = 2L * ctx->cu_count / tiles;
    if (z > kb / 4) z = kb / 4;
    return z < 2 ? 1 : (int)z;
}

static int fp8_run(SkmCtx *ctx, Fp8Args g, int fa, int fb, int dtype, unsigned gy, hipStream_t st, const char *tag,
                   void *ws = nullptr)
{
    // 256 x 256 tiles (float32 results: 256 x 128, the converted operands need the registers) where they fill half of the
    // GPU, 128 x 128 else (8200 x 4096 x 4096: 157 against 250 us).  Float32 results of up to 10 blocks are written more than
    // multiplied: two small workgroups on a CU, one writes while the other multiplies (8192 x 8192 x 512: 93 against 108 us).  Experts: as the plan's tiles are.
    const int wn = dtype != SKM_DT_F32 ? 256 : 128;
    const long wide = (long)((g.M + 255) / 256) * ((g.N + wn - 1) / wn) * gy;
    const bool brief = dtype == SKM_DT_F32 && !g.tiles && (g.first ? g.mean_blocks : g.kb1) <= 10;
    const bool big = g.tiles ? g.tile_rows == 256 : wide >= ctx->cu_count / 2 && g.slabs == 1 && !brief;
    const int bm = big ? 256 : 128, bn = big ? wn : 128;
    const int csize = skm_dt_size(dtype);
    const Fp8Args whole = g;
    if (g.slabs > 1) {                      // partial sums
        g.C = ws;
        g.ldc = g.N;
        g.zC = (long)g.M * g.N;
        g.accumulate = 0;
        dtype = SKM_DT_F32;
    }
    if (!g.tiles) g.tiles_m = (g.M + bm - 1) / bm;
    g.tiles_n = (g.N + bn - 1) / bn;
    // a lane's offset inside a tile (by plan: inside A) is 32 bits wide
    const long reach = g.tiles && g.slots ? g.rowsA : 256;
    if (reach * g.lda > 0xFFFFFFFFL || reach * g.SA > 0x7FFFFFFFL || 256 * g.ldb > 0xFFFFFFFFL) {
        skm_set_error("%s: %ld rows of %ld bytes are more than 4 GB", tag, reach, g.lda > g.ldb ? g.lda : g.ldb);
        return SKM_ERR_UNSUPPORTED;
    }
    const long total = (long)g.tiles_m * g.tiles_n;
    SKM_REQUIRE(total <= SKM_MAX_GROUPS && gy <= 65535, "%s: too many tiles", tag);
    if (total == 0 || gy == 0) return SKM_OK;
    {
        SkmProfScope ps(ctx, tag, st);
        switch (dtype * 2 + big) {
        case SKM_DT_F32 * 2: fp8_launch<2, 2, float>(g, fa, fb, (unsigned)total, gy, st); break;
        case SKM_DT_F32 * 2 + 1: fp8_launch<4, 2, float>(g, fa, fb, (unsigned)total, gy, st); break;
        case SKM_DT_BF16 * 2: fp8_launch<2, 2, bf16_t>(g, fa, fb, (unsigned)total, gy, st); break;
        case SKM_DT_BF16 * 2 + 1: fp8_launch<4, 4, bf16_t>(g, fa, fb, (unsigned)total, gy, st); break;
        case SKM_DT_F16 * 2: fp8_launch<2, 2, f16_t>(g, fa, fb, (unsigned)total, gy, st); break;
        default: fp8_launch<4, 4, f16_t>(g, fa, fb, (unsigned)total, gy, st); break;
        }
        SKM_HIP(hipGetLastError());
    }
    if (g.slabs > 1) {
        SkmProfScope ps(ctx, "k_fp8_slabs", st);
        const dim3 grid((unsigned)((g.zC + 255) / 256)), block(256);
        const float *part = static_cast<const float *>(ws);
        if (csize == 4)
            hipLaunchKernelGGL(k_fp8_slabs<float>, grid, block, 0, st, part, g.slabs, g.zC, g.M, g.N,
                               static_cast<float *>(whole.C), whole.ldc, whole.accumulate);
        else if (whole.c_bf16)
            hipLaunchKernelGGL(k_fp8_slabs<bf16_t>, grid, block, 0, st, part, g.slabs, g.zC, g.M, g.N,
                               static_cast<bf16_t *>(whole.C), whole.ldc, whole.accumulate);
        else
            hipLaunchKernelGGL(k_fp8_slabs<f16_t>, grid, block, 0, st, part, g.slabs, g.zC, g.M, g.N,
                               static_cast<f16_t *>(whole.C), whole.ldc, whole.accumulate);
        SKM_HIP(hipGetLastError());
    }
    return SKM_OK;
}

static int fp8_check_product(const char *who, int fa, int fb, int dtype, int M, int N, int K)
{
    SKM_REQUIRE((fa == 0 || fa == 1) && (fb == 0 || fb == 1), "%s: 8-bit formats %d, %d", who, fa, fb);
    SKM_REQUIRE(dtype == SKM_DT_F32 || dtype == SKM_DT_BF16 || dtype == SKM_DT_F16, "%s: result type %d", who, dtype);
    SKM_REQUIRE(M >= 0 && N >= 0 && K >= 0 && M < 0x7FFFFF00 && N < 0x7FFFFF00 && K < 0x7FFFFF00, "%s: bad shape", who);
    return SKM_OK;
}

// Up to this many rows the weights are read straight into registers, a workgroup's waves splitting k ...
#define FP8_FEW_ROWS 64
// ... with more than 32 rows only where the columns make a workgroup for every CU (64 x 2048 x 8192: 24 us against 14 in
// slabs, 64 x 4096 x 4096: 14.5 against 17)
static bool fp8_few(const SkmCtx *ctx, long M, long N) { return M <= 32 || (M <= FP8_FEW_ROWS && (N + 15) / 16 >= ctx->cu_count); }

// a float A is quantized on the way (no memory for it) up to one row tile
static bool fp8_on_the_way(long rows) { return rows <= 16; }

static size_t fp8_operand_bytes(long rows, long K)
{
    return skm_align_up((size_t)rows * fp8_kpad(K), 256) + skm_align_up((size_t)rows * fp8_sstride(K), 256);
}

static size_t fp8_slab_bytes(const SkmCtx *ctx, long M, long N, long K)
{
    if (fp8_few(ctx, M, N)) return 0;
    const int z = fp8_slabs(ctx, M, N, K);
    return z > 1 ? skm_align_up((size_t)z * M * N * 4, 256) : 0;
}

extern "C" size_t skm_gemm_fp8_workspace_bytes(void *ctx, int M, int N, int K, int a_float)
{
    if (!ctx || M <= 0 || N <= 0 || K <= 0) return 0;
    return (a_float && !fp8_on_the_way(M) ? fp8_operand_bytes(M, K) : 0) + fp8_slab_bytes(static_cast<SkmCtx *>(ctx), M, N, K);
}

// A: q, s in 8-bit floats (a_dtype < 0), or a float matrix in rows of lda that goes through 8-bit floats of format fmt_a;
// in the second case with more than 16 rows it is quantized into ws, q and s set to that
static int fp8_take_a(SkmCtx *ctx, const char *who, const void *&q, const void *&s, int a_dtype, long lda, int fmt_a, long rows,
                      int K, bool on_the_way, void *ws, size_t ws_bytes, Fp8Float *fx, void *stream)
{
    if (a_dtype < 0) {
        SKM_REQUIRE(q && s && ((uintptr_t)q & 15) == 0 && ((uintptr_t)s & 3) == 0, "%s: A is missing or not aligned", who);
        return SKM_OK;
    }
    if (int rc = fp8_check_types(who, a_dtype, fmt_a)) return rc;
    SKM_REQUIRE(q && lda >= K, "%s: A is missing or its rows overlap", who);
    if (on_the_way) {
        *fx = Fp8Float{q, lda, K};
        q = s = nullptr;
        return SKM_OK;
    }
    if (!ws || ws_bytes < fp8_operand_bytes(rows, K) || ((uintptr_t)ws & 15)) {
        skm_set_error("%s: workspace too small or not aligned", who);
        return SKM_ERR_WORKSPACE;
    }
    uint8_t *wq = static_cast<uint8_t *>(ws), *wss = wq + skm_align_up((size_t)rows * fp8_kpad(K), 256);
    if (int rc = skm_fp8_rows(ctx, q, a_dtype, rows, K, lda, fmt_a, wq, wss, stream)) return rc;
    q = wq;
    s = wss;
    return SKM_OK;
}

extern "C" int skm_gemm_fp8(void *ctx_, const void *A, const void *sA, int fmt_a, int a_dtype, long lda, const void *B,
                            const void *sB, int fmt_b, int M, int N, int K, void *C, int c_dtype, long ldc, int accumulate,
                            void *ws, size_t ws_bytes, void *stream)
{
    SkmCtx *ctx = static_cast<SkmCtx *>(ctx_);
    SKM_REQUIRE(ctx, "skm_gemm_fp8: bad argument");
    if (int rc = fp8_check_product("skm_gemm_fp8", fmt_a, fmt_b, c_dtype, M, N, K)) return rc;
    if (M == 0 || N == 0) return SKM_OK;
    SKM_REQUIRE(K >= 1 && B && sB && C && ldc >= N && ((uintptr_t)B & 15) == 0 && ((uintptr_t)sB & 3) == 0,
                "skm_gemm_fp8: bad argument");
    Fp8Float fx{};
    if (int rc = fp8_take_a(ctx, "skm_gemm_fp8", A, sA, a_dtype, lda, fmt_a, M, K, fp8_on_the_way(M), ws, ws_bytes, &fx, stream))
        return rc;
    SkmDeviceGuard guard(ctx);
    Fp8Args g{};
    g.A = static_cast<const uint8_t *>(A); g.B = static_cast<const uint8_t *>(B);
    g.sA = static_cast<const uint8_t *>(sA); g.sB = static_cast<const uint8_t *>(sB);
    g.lda = g.ldb = fp8_kpad(K);
    g.SA = g.SB = (int)fp8_sstride(K);
    g.M = M; g.N = N; g.rowsA = M; g.kb1 = (int)(fp8_kpad(K) / FP8_BLOCK);
    g.C = C; g.ldc = ldc; g.accumulate = accumulate != 0; g.slabs = 1;
    hipStream_t st = (hipStream_t)stream;
    if (fp8_few(ctx, M, N)) return rows16_run(ctx, g, fx, a_dtype, fmt_a, fmt_b, c_dtype, 1, st);
    g.c_bf16 = c_dtype == SKM_DT_BF16;
    g.slabs = fp8_slabs(ctx, M, N, K);
    if (g.slabs > 1) {
        if (!ws || ws_bytes < skm_gemm_fp8_workspace_bytes(ctx, M, N, K, a_dtype >= 0) || ((uintptr_t)ws & 15)) {
            skm_set_error("skm_gemm_fp8: workspace too small or not aligned");
            return SKM_ERR_WORKSPACE;
        }
        // behind the quantized A
        char *part = static_cast<char *>(ws) + (a_dtype >= 0 ? fp8_operand_bytes(M, K) : 0);
        return fp8_run(ctx, g, fmt_a, fmt_b, c_dtype, (unsigned)g.slabs, st, "k_gemm_fp8", part);
    }
    // A last row tile of up to 64 rows that would put a few workgroups behind all the others goes to the kernel for few rows
    // (8200 x 4096 x 4096: 157 -> 122 us)
    const int wn = c_dtype != SKM_DT_F32 ? 256 : 128, rest = M % 256;
    const long tn = (N + wn - 1) / wn, cu = ctx->cu_count;
    if (rest && rest <= FP8_FEW_ROWS && M > 256 && (M / 256) * tn >= cu / 2 &&
        ((M / 256 + 1) * tn + cu - 1) / cu > ((M / 256) * tn + cu - 1) / cu) {
        Fp8Args tail = g;
        g.M = g.rowsA = M - rest;
        tail.M = tail.rowsA = rest;
        tail.A += (long)g.M * g.lda;
        tail.sA += (long)g.M * g.SA;
        tail.C = static_cast<char *>(C) + (long)g.M * ldc * skm_dt_size(c_dtype);
        if (int rc = rows16_run(ctx, tail, fx, a_dtype, fmt_a, fmt_b, c_dtype, 1, st)) return rc;
    }
    return fp8_run(ctx, g, fmt_a, fmt_b, c_dtype, 1, st, "k_gemm_fp8");
}

extern "C" size_t skm_gemm_fp8_experts_workspace_bytes(void *ctx, long rows, int K, int a_float, int more_rows)
{
    (void)ctx;
    return a_float && more_rows != 16 && rows > 0 && K > 0 ? fp8_operand_bytes(rows, K) : 0;
}

extern "C" int skm_gemm_fp8_experts(void *ctx_, const void *A, const void *sA, int fmt_a, int a_dtype, long lda, long rows,
                                    const void *W, const void *sW, int fmt_w, int E, int N, int K, const int32_t *pair,
                                    int slots, long n, const int32_t *first, const int32_t *tiles, int more_rows,
                                    const int32_t *more_tiles, const int32_t *more_count, void *C, int c_dtype, void *ws,
                                    size_t ws_bytes, void *stream)
{
    SkmCtx *ctx = static_cast<SkmCtx *>(ctx_);
    SKM_REQUIRE(ctx && E >= 1 && n >= 0 && n <= 0x3FFFFFFF && slots >= 0, "skm_gemm_fp8_experts: bad argument");
    SKM_REQUIRE(more_rows == 0 || ((more_rows == 16 || more_rows == 256) && more_tiles && more_count),
                "skm_gemm_fp8_experts: a second table has tiles of 16 or 256 rows");
    if (int rc = fp8_check_product("skm_gemm_fp8_experts", fmt_a, fmt_w, c_dtype, (int)n, N, K)) return rc;
    if (n == 0 || N == 0) return SKM_OK;
    SKM_REQUIRE(K >= 1 && W && sW && C && pair && first && tiles && ((uintptr_t)W & 15) == 0 && ((uintptr_t)sW & 3) == 0,
                "skm_gemm_fp8_experts: bad argument");
    SKM_REQUIRE(slots ? rows * slots == n : rows == n, "skm_gemm_fp8_experts: %ld rows of A for %ld pairs", rows, n);
    const long most = skm_route_plan_tiles(n, E, more_rows ? more_rows : 128);
    SKM_REQUIRE(more_rows != 16 || most <= 65535, "skm_gemm_fp8_experts: more than 65535 tiles of 16 rows");
    Fp8Float fx{};
    if (int rc = fp8_take_a(ctx, "skm_gemm_fp8_experts", A, sA, a_dtype, lda, fmt_a, rows, K, more_rows == 16, ws, ws_bytes,
                            &fx, stream))
        return rc;
    SkmDeviceGuard guard(ctx);
    Fp8Args g{};
    g.A = static_cast<const uint8_t *>(A); g.B = static_cast<const uint8_t *>(W);
    g.sA = static_cast<const uint8_t *>(sA); g.sB = static_cast<const uint8_t *>(sW);
    g.lda = g.ldb = fp8_kpad(K);
    g.SA = g.SB = (int)fp8_sstride(K);
    g.M = (int)n; g.N = N; g.rowsA = rows; g.kb1 = (int)(fp8_kpad(K) / FP8_BLOCK);
    g.C = C; g.ldc = N; g.slabs = 1;
    g.tiles = more_rows ? more_tiles : tiles;
    g.tile_count = more_rows ? more_count : first + E;
    g.tile_rows = more_rows ? more_rows : 128;
    g.pair = pair; g.slots = slots;
    g.eB = (long)N * g.ldb; g.esB = (long)N * g.SB;
    if (more_rows == 16)
        return rows16_run(ctx, g, fx, a_dtype, fmt_a, fmt_w, c_dtype, (unsigned)most, (hipStream_t)stream);
    g.tiles_m = (int)most;
    return fp8_run(ctx, g, fmt_a, fmt_w, c_dtype, 1, (hipStream_t)stream, "k_gemm_fp8_experts");
}

extern "C" int skm_gemm_fp8_experts_wgrad(void *ctx_, const void *A, const void *sA, int fmt_a, const void *B,
                                          const void *sB, int fmt_b, int E, int M, int N, const int32_t *first,
                                          long max_tiles, float *C, int accumulate, void *stream)
{
    SkmCtx *ctx = static_cast<SkmCtx *>(ctx_);
    SKM_REQUIRE(ctx && E >= 1 && E <= 65535 && max_tiles >= 0 && max_tiles < 0x7FFFFFFF / FP8_BLOCK,
                "skm_gemm_fp8_experts_wgrad: bad argument");
    if (int rc = fp8_check_product("skm_gemm_fp8_experts_wgrad", fmt_a, fmt_b, SKM_DT_F32, M, N, 1)) return rc;
    if (M == 0 || N == 0) return SKM_OK;
    SKM_REQUIRE(C && first && (max_tiles == 0 || (A && sA && B && sB)) &&
                    (((uintptr_t)A | (uintptr_t)B) & 15) == 0 && (((uintptr_t)sA | (uintptr_t)sB) & 3) == 0,
                "skm_gemm_fp8_experts_wgrad: bad argument");
    SkmDeviceGuard guard(ctx);
    Fp8Args g{};
    g.A = static_cast<const uint8_t *>(A); g.B = static_cast<const uint8_t *>(B);
    g.sA = static_cast<const uint8_t *>(sA); g.sB = static_cast<const uint8_t *>(sB);
    g.lda = g.ldb = max_tiles * FP8_BLOCK;
    g.SA = g.SB = (int)fp8_sstride(g.lda);
    g.M = M; g.N = N; g.rowsA = M;
    g.C = C; g.ldc = N; g.accumulate = accumulate != 0; g.slabs = 1;
    g.first = first; g.eC = (long)M * N; g.mean_blocks = max_tiles / E;
    return fp8_run(ctx, g, fmt_a, fmt_b, SKM_DT_F32, (unsigned)E, (hipStream_t)stream, "k_gemm_fp8_wgrad");
}
