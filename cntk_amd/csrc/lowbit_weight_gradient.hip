// The weight gradient of a linear layer whose input was kept in 8 bits: dw[n, k] = sum over m of dy[m, n] x8[m, k], and the
// column sums of dy. x8's values are bfloat16 numbers as they are; dy of a wider type is a sum of bfloat16 numbers (half precision: two,
// single: three), each multiplied in turn, so every product is exact and the sums are in 32 bits. (bfloat16 ends at 2^-133: what a single-precision dy has below
// that, of numbers under 2^-110, is not multiplied. Half precision's numbers are nowhere near.)
//
// Both factors run along memory in the axis that is not summed over, and the matrix unit wants the other. For many results a first launch turns
// them over into tiles in the workspace (dy: 2 bytes an element and term, x8: 2), reading each once; the second multiplies tiles. Turning
// them inside the product would repeat the work in every block of output rows, but for two cases: LDS turns 16-bit numbers over as
// it reads them, so a bfloat16 dy goes into a large product as it lies; and for few results, or where one factor is read once all the same, both are
// turned over in registers, in one launch or one for every part of the depth at once.
//
// Measured with bias, m x n x k: 4096 x 9304 x 2048 in bfloat16 25.6 + 147 us, 1.06 PFLOP/s in the second launch (a copy's rate and the largest
// library product's: 20 and 123 us); 2048^3 8.1 + 27.4; 257 x 2048 x 429 in single precision 8.7 in one launch.
#include "lowbit_product.h"

#include <algorithm>

namespace cntkq {
namespace lowbit {

namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kDepth = 32; // rows of dy and x8 in a tile
constexpr uint32_t kMostRunTiles = 8; // tiles of depth that a workgroup of the first launch goes through
constexpr uint32_t kMostParts = 16; // of the depth, each with results of its own
constexpr size_t kMostRows = (size_t) 1 << 21; // of a pair of launches: more rows come in several, each added to the one before
constexpr uint32_t kXCols = 256, kYCols = 128, kSumCols = 512; // columns of a workgroup

constexpr int terms_of(int dtype)
{
    return dtype == kBF16 ? 1 : (dtype == kF16 ? 2 : 3);
}

struct Pack
{
    const void* dy;
    int64_t dy_stride;
    const int8_t* saved;
    const uint8_t* scales;
    uint32_t m, n, k, pitch, m_tiles, x_chunks, y_chunks, runs, run_tiles;
    char* x_tiles;
    char* y_tiles;
    float* sums; // [runs][n], or null
};

// two numbers' upper halves, the first in the lower one
__device__ __forceinline__ uint32_t upper_halves(float a, float b)
{
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}

// Eight rows of four columns of x8 as they lie in memory; rows and columns beyond the end are the last ones.
struct RawX
{
    uint32_t codes[8], scale[8];
};
__device__ __forceinline__ void fetch_x(const Pack& a, uint32_t row, uint32_t col, RawX& r)
{
    col = min(col, a.pitch - 4);
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
        const size_t at = min(row + i, a.m - 1);
        r.codes[i] = *reinterpret_cast<const uint32_t*>(a.saved + at * a.pitch + col);
        r.scale[i] = a.scales[at * (a.pitch / kBlock) + col / kBlock];
    }
}
// Eight rows of two columns of dy.
template <int DT, bool EVEN>
struct RawY;
template <int DT>
struct RawY<DT, true>
{
    uint32_t pair[8];
};
template <>
struct RawY<kF32, true>
{
    f32x2 pair[8];
};
template <int DT>
struct RawY<DT, false>
{
    typename Type<DT>::T v[8][2];
};
template <int DT, bool EVEN>
__device__ __forceinline__ void fetch_y(const Pack& a, uint32_t row, uint32_t col, RawY<DT, EVEN>& r)
{
    typedef typename Type<DT>::T T;
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
        const T* p = static_cast<const T*>(a.dy) + (int64_t) min(row + i, a.m - 1) * a.dy_stride;
        if constexpr (!EVEN)
        {
            r.v[i][0] = p[min(col, a.n - 1)];
            r.v[i][1] = p[min(col + 1, a.n - 1)];
        }
        else if constexpr (DT == kF32)
            r.pair[i] = *reinterpret_cast<const f32x2_at4*>(p + min(col, a.n - 2));
        else
            r.pair[i] = *reinterpret_cast<const u32_at2*>(p + min(col, a.n - 2));
    }
}
// (zeros beyond the last row and column; INSIDE: they are all there, or of no interest)
template <int DT, bool EVEN, bool INSIDE = false>
__device__ __forceinline__ void up_y(const Pack& a, uint32_t row, uint32_t col, const RawY<DT, EVEN>& r, float (&v)[8][2])
{
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
        float x, y;
        if constexpr (!EVEN)
        {
            x = Type<DT>::up(r.v[i][0]);
            y = Type<DT>::up(r.v[i][1]);
        }
        else if constexpr (DT == kF32)
        {
            x = r.pair[i][0];
            y = r.pair[i][1];
        }
        else if constexpr (DT == kBF16)
        {
            x = __uint_as_float(r.pair[i] << 16);
            y = __uint_as_float(r.pair[i] & 0xffff0000u);
        }
        else
        {
            const uint32_t w = r.pair[i];
            const f16x2 h = __builtin_bit_cast(f16x2, w);
            x = (float) h[0];
            y = (float) h[1];
        }
        if constexpr (DT == kF32) // (a NaN's upper half is one too if it is a quiet one)
        {
            x = __builtin_canonicalizef(x);
            y = __builtin_canonicalizef(y);
        }
        const bool in = row + i < a.m;
        v[i][0] = INSIDE || (in && col < a.n) ? x : 0.0f;
        v[i][1] = INSIDE || (in && col + 1 < a.n) ? y : 0.0f;
    }
}
__device__ __forceinline__ u32x4 eight_upper_halves(float a, float b, float c, float d, float e, float f, float g, float h)
{
    return u32x4{upper_halves(a, b), upper_halves(c, d), upper_halves(e, f), upper_halves(g, h)};
}

// What the upper halves leave, exactly down to 2^-133; FIRST: and nothing of an infinity or a NaN.
template <bool FIRST>
__device__ __forceinline__ void take_upper_halves(float (&v)[8][2])
{
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
        {
            const float up = __uint_as_float(__float_as_uint(v[i][j]) & 0xffff0000u);
            v[i][j] = !FIRST || magnitude(v[i][j]) < 0x7f800000u ? v[i][j] - up : 0.0f;
        }
}

// Wavefront w of a workgroup has eight rows of a tile's 32; a lane has four columns of x8 or two of dy, and writes for each the
// eight values that one lane of the matrix instruction takes. The next tile's loads are on their way while one is turned over. Bound by memory:
// 4096 rows of 9304 and 2048 columns in half precision, 254 MB, 66 to 69 us, in single precision, 407 MB, 89 to 91; of 9303 in bfloat16, value by value, 54.
__device__ __forceinline__ void turn_x(const Pack& a, uint32_t chunk, uint32_t first, uint32_t last)
{
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, col = chunk * kXCols + lane * 4;
    if (col / 16 * 16 >= a.k)
        return;
    RawX raw;
    fetch_x(a, first * kDepth + wave * 8, col, raw);
    for (uint32_t mt = first; mt < last; ++mt)
    {
        const RawX now = raw;
        const uint32_t row = mt * kDepth + wave * 8;
        fetch_x(a, row + kDepth, col, raw);
        float v[8][4];
#pragma unroll
        for (int i = 0; i < 8; ++i)
        {
            const float f = save8_factor(now.scale[i]);
            const uint32_t codes = row + i < a.m && col < a.pitch ? now.codes[i] : 0;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[i][j] = row + i < a.m && col < a.pitch ? (float) (int) (int8_t) (codes >> (8 * j)) * f : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            *reinterpret_cast<u32x4*>(a.x_tiles + ((size_t) ((col + j) / 16) * a.m_tiles + mt) * kTileBytes + (wave * 16 + (col + j) % 16) * 16) =
                eight_upper_halves(v[0][j], v[1][j], v[2][j], v[3][j], v[4][j], v[5][j], v[6][j], v[7][j]);
    }
}
// The wavefronts' sums of the workgroup's COLS columns, added up and written.
template <uint32_t COLS>
__device__ __forceinline__ void write_sums(const Pack& a, const float (&part)[4][COLS], uint32_t run, uint32_t first_col)
{
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < COLS; i += kThreads)
        if (first_col + i < a.n)
            a.sums[(size_t) run * a.n + first_col + i] = part[0][i] + part[1][i] + part[2][i] + part[3][i];
}

template <int DT, bool EVEN>
__global__ __launch_bounds__(kThreads) void weight_gradient_pack_kernel(Pack a)
{
    constexpr int TERMS = terms_of(DT);
    __shared__ float part[4][kYCols];
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const uint32_t run = blockIdx.x % a.runs, chunk = blockIdx.x / a.runs;
    const uint32_t first = run * a.run_tiles, last = min(first + a.run_tiles, a.m_tiles);
    if (chunk < a.x_chunks)
        return turn_x(a, chunk, first, last);
    const uint32_t col = (chunk - a.x_chunks) * kYCols + lane * 2;
    const uint32_t n_tiles = (a.n + 15) / 16;
    float sum[2] = {0.0f, 0.0f};
    RawY<DT, EVEN> raw;
    fetch_y<DT, EVEN>(a, first * kDepth + wave * 8, col, raw);
    for (uint32_t mt = first; mt < last; ++mt)
    {
        const RawY<DT, EVEN> now = raw;
        const uint32_t row = mt * kDepth + wave * 8;
        fetch_y<DT, EVEN>(a, row + kDepth, col, raw);
        float v[8][2];
        up_y<DT, EVEN>(a, row, col, now, v);
#pragma unroll
        for (int i = 0; i < 8; ++i)
        {
            sum[0] += v[i][0];
            sum[1] += v[i][1];
        }
        if (col / 16 < n_tiles)
        {
            each<TERMS>([&](auto t) {
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    *reinterpret_cast<u32x4*>(a.y_tiles + ((size_t) ((col + j) / 16) * (TERMS * a.m_tiles) + t * a.m_tiles + mt) * kTileBytes +
                                              (wave * 16 + (col + j) % 16) * 16) =
                        eight_upper_halves(v[0][j], v[1][j], v[2][j], v[3][j], v[4][j], v[5][j], v[6][j], v[7][j]);
                take_upper_halves<t == 0>(v);
            });
        }
    }
    if (a.sums != nullptr)
    {
        part[wave][lane * 2] = sum[0];
        part[wave][lane * 2 + 1] = sum[1];
        write_sums(a, part, run, (chunk - a.x_chunks) * kYCols);
    }
}

// The same where the product takes dy as it lies in memory (Columns): x8 is turned over, dy's columns are added up, eight to a lane, in the
// order of the kernel above. The same matrices, 101 MB: 25.6 us. (Adding up inside the product, from the operand in registers, cost its blocks more:
// 11.3 + 214 us, 2048^3 6.4 + 34.2.)
__global__ __launch_bounds__(kThreads) void weight_gradient_pack_x_kernel(Pack a)
{
    __shared__ float part[4][kSumCols];
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const uint32_t run = blockIdx.x % a.runs, chunk = blockIdx.x / a.runs;
    const uint32_t first = run * a.run_tiles, last = min(first + a.run_tiles, a.m_tiles);
    if (chunk < a.x_chunks)
        return turn_x(a, chunk, first, last);
    const uint32_t first_col = (chunk - a.x_chunks) * kSumCols, col = min(first_col + lane * 8, a.n - 8);
    const auto fetch = [&](uint32_t row, u32x4(&w)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            w[i] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.dy) + (int64_t) min(row + i, a.m - 1) * a.dy_stride + col);
    };
    float sum[8] = {};
    u32x4 ahead[8], now[8];
    fetch(first * kDepth + wave * 8, ahead);
    for (uint32_t mt = first; mt < last; ++mt)
    {
        const uint32_t row = mt * kDepth + wave * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            now[i] = ahead[i];
        fetch(row + kDepth, ahead);
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
            {
                const uint32_t w = row + i < a.m ? now[i][j] : 0;
                sum[2 * j] += __uint_as_float(w << 16);
                sum[2 * j + 1] += __uint_as_float(w & 0xffff0000u);
            }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        part[wave][lane * 8 + j] = sum[j];
    write_sums(a, part, run, first_col);
}

struct Sums
{
    const float* sums;
    float* db;
    uint32_t runs, n, first_block; // the workgroups below first_block multiply, the others add the column sums up
};

template <bool ACCUMULATE>
__device__ __forceinline__ float column_sum(const Sums& b, uint32_t at)
{
    float v = ACCUMULATE ? b.db[at] : 0.0f;
#pragma unroll 4
    for (uint32_t r = 0; r < b.runs; ++r)
        v += b.sums[(size_t) r * b.n + at];
    return v;
}

template <int TQ, int TP, int NB, bool ACCUMULATE, typename DY>
__global__ __launch_bounds__(256, (TileKernel<Bf16Op, TQ, TP, NB>::kPerUnit)) void weight_gradient_kernel(Tiles x, DY dy, Output o, uint32_t depth, uint32_t y_blocks, uint32_t x_blocks, Sums b)
{
    typedef TileKernel<Bf16Op, TQ, TP, NB, ACCUMULATE, DY> K;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    if (blockIdx.x >= b.first_block)
    {
        const uint32_t at = (blockIdx.x - b.first_block) * K::kThreads + threadIdx.x;
        if (at < b.n)
            b.db[at] = column_sum<ACCUMULATE>(b, at);
        return;
    }
    K kernel;
    kernel.template run<kF32>(lds, x, dy, o, depth, y_blocks, x_blocks, blockIdx.x, b.first_block);
}

// tiles of depth: an even number, as the product takes them
size_t depth_tiles(size_t m)
{
    return 2 * ceil_div(m, 2 * kDepth);
}

// Few results: a workgroup has 32 rows of dw and 16 XW columns; its wavefronts share the depth out among them, take
// both factors as they lie in memory, and turn them over in registers: a lane has XW neighbouring columns of eight rows of x8 and two of dy's,
// each in an operand of the matrix unit of its own, so that its results are 4 XW neighbouring columns of two rows. Bound by the latency of a
// launch and of a wavefront's loads, larger ones by the arithmetic of turning dy over for every 16 XW columns: 257 x 2048 x 429 in single precision, 9 MB, 8.7 us.
template <int XW>
struct RawColumns;
template <>
struct RawColumns<2>
{
    uint32_t codes[8], scale[8];
};
template <>
struct RawColumns<4> : RawX
{
};
__device__ __forceinline__ void fetch_columns(const Pack& a, uint32_t row, uint32_t col, RawColumns<2>& r)
{
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
        const size_t at = min(row + i, a.m - 1);
        r.codes[i] = *reinterpret_cast<const uint16_t*>(a.saved + at * a.pitch + col);
        r.scale[i] = a.scales[at * (a.pitch / kBlock) + col / kBlock];
    }
}
__device__ __forceinline__ void fetch_columns(const Pack& a, uint32_t row, uint32_t col, RawColumns<4>& r)
{
    fetch_x(a, row, col, r);
}

// INSIDE: none of the 32 rows is beyond the last one. (What is beyond the last column goes into results that are not written.)
template <int DT, bool EVEN, int XW, bool INSIDE>
__device__ __forceinline__ void direct_tile(const Pack& a, uint32_t row, uint32_t x_col, uint32_t y_col, f32x4 (&acc)[XW][2], float (&column)[2])
{
    RawColumns<XW> raw_x;
    RawY<DT, EVEN> raw_y;
    fetch_columns(a, row, x_col, raw_x);
    fetch_y<DT, EVEN>(a, row, y_col, raw_y);
    float v[8][2], x[8][XW];
    up_y<DT, EVEN, INSIDE>(a, row, y_col, raw_y, v);
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
        const float f = save8_factor(raw_x.scale[i]);
#pragma unroll
        for (int j = 0; j < XW; ++j)
            x[i][j] = INSIDE || row + i < a.m ? (float) (int) (int8_t) (raw_x.codes[i] >> (8 * j)) * f : 0.0f;
#pragma unroll
        for (int j = 0; j < 2; ++j)
            column[j] += v[i][j];
    }
    u32x4 fx[XW];
#pragma unroll
    for (int j = 0; j < XW; ++j)
        fx[j] = eight_upper_halves(x[0][j], x[1][j], x[2][j], x[3][j], x[4][j], x[5][j], x[6][j], x[7][j]);
    each<terms_of(DT)>([&](auto term) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
        {
            const u32x4 fy = eight_upper_halves(v[0][j], v[1][j], v[2][j], v[3][j], v[4][j], v[5][j], v[6][j], v[7][j]);
#pragma unroll
            for (int i = 0; i < XW; ++i)
                acc[i][j] = Bf16Op::mma<0, 0>(fx[i], fy, acc[i][j], 0, 0);
        }
        take_upper_halves<term == 0>(v);
    });
}

template <int DT, bool EVEN, bool ACCUMULATE, int XW>
__global__ __launch_bounds__(512) void weight_gradient_direct_kernel(Pack a, Output o, float* db, size_t part)
{
    extern __shared__ __attribute__((aligned(16))) f32x4 sums[];
    const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), waves = blockDim.x / 64;
    const uint32_t x_col = (blockIdx.x * 16 + lane % 16) * XW, y_col = (blockIdx.y * 16 + lane % 16) * 2;
    f32x4 acc[XW][2] = {};
    float column[2] = {0.0f, 0.0f};
    // the workgroup's part of the depth
    const uint32_t end = min((blockIdx.z + 1) * a.run_tiles, a.m_tiles), whole = min(end, a.m / kDepth);
    uint32_t t = blockIdx.z * a.run_tiles + wave;
    for (; t < whole; t += waves)
        direct_tile<DT, EVEN, XW, true>(a, t * kDepth + lane / 16 * 8, x_col, y_col, acc, column);
    if (t < end)
        direct_tile<DT, EVEN, XW, false>(a, t * kDepth + lane / 16 * 8, x_col, y_col, acc, column);
    // sums[row of the two][column of the XW][wavefront][lane], then the column sums: [wavefront][group of lanes][column]
#pragma unroll
    for (int i = 0; i < XW; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
            sums[((j * XW + i) * waves + wave) * 64 + lane] = acc[i][j];
    float* columns = reinterpret_cast<float*>(sums + 2 * XW * waves * 64);
#pragma unroll
    for (int j = 0; j < 2; ++j)
        columns[wave * 128 + lane / 16 * 32 + lane % 16 * 2 + j] = column[j];
    __syncthreads();
    if (wave < 2)
    {
        f32x4 v[XW];
#pragma unroll
        for (int i = 0; i < XW; ++i)
        {
            v[i] = sums[(wave * XW + i) * waves * 64 + lane];
            for (uint32_t w = 1; w < waves; ++w)
                v[i] += sums[((wave * XW + i) * waves + w) * 64 + lane];
        }
        const uint32_t col = (blockIdx.x * 16 + lane / 16 * 4) * XW;
        o.out = static_cast<float*>(o.out) + blockIdx.z * part;
#pragma unroll
        for (int i = 0; i < XW; ++i) // the results 4 i to 4 i + 3 of the lane's 4 XW in a row
            write4<kF32, ACCUMULATE>(o, y_col + wave, col + i * 4,
                                     f32x4{v[4 * i % XW][4 * i / XW], v[(4 * i + 1) % XW][(4 * i + 1) / XW], v[(4 * i + 2) % XW][(4 * i + 2) / XW],
                                           v[(4 * i + 3) % XW][(4 * i + 3) / XW]});
    }
    else if (wave == 2 && db != nullptr && blockIdx.x == 0)
    {
        db += blockIdx.z * part;
        const uint32_t at = blockIdx.y * 32 + lane;
        if (lane < 32 && at < a.n)
        {
            float v = ACCUMULATE ? db[at] : 0.0f;
            for (uint32_t w = 0; w < waves * 4; ++w)
                v += columns[w * 32 + lane];
            db[at] = v;
        }
    }
}

// How a weight gradient is made. kDirect: in one launch, few results of few rows, or a narrow one: one factor is read once then. kParts: few results of
// many rows, the same launch for parts of the depth and another that adds the parts' results up. kTiles: many results, factors in tiles.
//
// m x n x k, us in one launch and with tiles. Up to 1024 rows, in single precision: 1 x 2048 x 429 4.7 / 7.7, 257 x 2048 x 429 8.7 / 15.0, 512^3 5.9 / 10.1,
// 1024 x 128 x 128 8.1 / 8.6; in bfloat16 512^3 4.8 / 7.2, 1024^3 12.4 / 14.0, but 1 x 4096 x 4096 36 / 19. More rows, in single precision:
// 4096 x 1024 x 1024 52 / 64, 16384 x 1024 x 512 110 / 165, 16384 x 2048 x 1024 379 / 538, 4096 x 4096 x 512 109 / 116; in bfloat16 4096 x 1024 x 1024 36 / 40,
// 16384 x 1024 x 512 77 / 83, but 2048 x 2048 x 1024 34 / 27. Narrow, in bfloat16: 4096 x 65536 x 64 189 / 198, 4096 x 64 x 65536 211 / 403,
// 300 x 1000000 x 40 238 / 296 (single precision 317 / 1402), but 4096 x 65536 x 128 345 / 212. In parts and with tiles, in single precision:
// 1500 x 128 x 128 9.0 / 10.4, 6886 x 1024 x 128 19 / 43, 65536 x 128 x 128 33 / 185, 1000000 x 64 x 64 418 / 4184; in bfloat16 1500 x 128 x 128 7.7 / 7.6,
// 4096 x 512 x 512 17 / 24, 65536 x 512 x 512 152 / 155, 1000000 x 64 x 64 304 / 2043. Just above 2^18 results nothing cuts the depth, and a deep one has
// few workgroups for it; in one launch and with tiles: 16384 x 520 x 512 in bfloat16 86 / 127, in single precision 103 / 352, 65536 x 520 x 512 316 / 474 and 426 / 1872.
enum class Way
{
    kDirect,
    kParts,
    kTiles
};
Way way_of(size_t m, size_t n, size_t k, int dtype)
{
    const size_t results = n * k, few = (size_t) 1 << 18;
    const bool high = n > (size_t) 65535 * 32; // a grid's second side ends there
    const bool narrow = n <= 64 || k <= 64;
    if (k == 0 || high)
        return Way::kTiles;
    if (m > 1024 && results <= few)
        return Way::kParts;
    return narrow || results <= (dtype == kF32 ? 8 * few : 4 * few) ? Way::kDirect : Way::kTiles;
}

// Into how many parts the depth is cut: two workgroups on every compute unit, or sixteen parts, and sixteen tiles in each at least.
uint32_t depth_parts(size_t m, size_t n, size_t k)
{
    const size_t groups = ceil_div(n, 32) * ceil_div(k, 64);
    return (uint32_t) std::max<size_t>(1, std::min(std::min<size_t>(kMostParts, ceil_div(2 * kComputeUnits, groups)), ceil_div(m, kDepth) / 16));
}

// Results of several parts of the depth, in a row in `parts`: added up in their order. The column sums follow each part's results.
template <bool ACCUMULATE>
__global__ __launch_bounds__(kThreads) void weight_gradient_join_kernel(const float* parts, uint32_t count, uint32_t part, Output o, float* db)
{
    const uint32_t at = blockIdx.x * kThreads + threadIdx.x, results = o.rows * o.cols;
    if (at >= results + (db != nullptr ? o.rows : 0))
        return;
    float* to = at < results ? static_cast<float*>(o.out) + (int64_t) (at / o.cols) * o.stride + at % o.cols : db + (at - results);
    float v = ACCUMULATE ? *to : 0.0f;
#pragma unroll 4
    for (uint32_t i = 0; i < count; ++i)
        v += parts[(size_t) i * part + at];
    *to = v;
}

struct Workspace
{
    size_t x, y, sums; // bytes
};
// As few tiles of depth for a workgroup of the first launch as it takes for eight workgroups on every compute unit.
uint32_t run_tiles(size_t m_tiles, size_t n, size_t k)
{
    const size_t chunks = ceil_div(k, kXCols) + ceil_div(n, kYCols);
    uint32_t run = kMostRunTiles;
    while (run > 1 && ceil_div(m_tiles, run) * chunks < 8 * kComputeUnits)
        run /= 2;
    return run;
}
Workspace workspace_of(size_t m, size_t n, size_t k, int dtype)
{
    if (n == 0) // nothing to make, and no workgroups to deal the depth to
        return {0, 0, 0};
    if (way_of(m, n, k, dtype) == Way::kDirect)
        return {0, 0, 0};
    if (way_of(m, n, k, dtype) == Way::kParts)
        return {0, 0, depth_parts(m, n, k) * (n * k + n) * sizeof(float)};
    const size_t m_tiles = depth_tiles(std::min(m, kMostRows));
    return {ceil_div(k, 16) * m_tiles * kTileBytes, ceil_div(n, 16) * m_tiles * terms_of(dtype) * kTileBytes,
            ceil_div(m_tiles, run_tiles(m_tiles, n, k)) * n * sizeof(float)};
}

template <int TQ, int TP, int NB, bool ACCUMULATE, typename DY>
hipError_t multiply(hipStream_t s, const Tiles& x, const DY& y, uint32_t depth, const Output& o, Sums b)
{
    typedef TileKernel<Bf16Op, TQ, TP, NB> K;
    const uint32_t x_blocks = (uint32_t) ceil_div(o.cols, K::kQTiles * 16), y_blocks = (uint32_t) ceil_div(o.rows, K::kPTiles * 16);
    const auto kernel = &weight_gradient_kernel<TQ, TP, NB, ACCUMULATE, DY>;
    static std::atomic<uint64_t> known{0};
    const hipError_t allowed = allow_lds(reinterpret_cast<const void*>(kernel), K::kLds, known);
    if (allowed != hipSuccess)
        return allowed;
    b.first_block = tile_workgroups(x_blocks * y_blocks, K::kPerUnit);
    const uint32_t blocks = b.first_block + (b.db != nullptr ? (uint32_t) ceil_div(b.n, K::kThreads) : 0);
    kernel<<<blocks, K::kThreads, K::kLds, s>>>(x, y, o, depth, y_blocks, x_blocks, b);
    return hipGetLastError();
}

// Blocks of 160 x 256, 128 x 256, 128 x 128 or 64 x 128 (rows of dw first): as for the 4-bit products, and with two heights of the large ones, of
// which one may need a round less. Stage times from products of 8192^3 (1050, 970, 1068 and 1429 us); m x n x k, us in the same order:
// 4096 x 9304 x 2048 146 / 184 / 158 / 223 (dy in tiles; as it lies 147; of 160 x 256 the kernel keeps 15 to 18 registers too many, 64 to 76 bytes a lane,
// which go through memory at the change of blocks but not in the stages between), 2048^3 51 / 45 / 25.1 / 27.5, 257 x 2048 x 429 12.5 / 10.1 / 7.6 / 6.3.
template <bool ACCUMULATE, typename DY>
hipError_t multiply_best(hipStream_t s, const Tiles& x, const DY& y, uint32_t depth, const Output& o, const Sums& b)
{
    const size_t n = o.rows, k = o.cols;
    const double tall = tile_cost(ceil_div(n, 160) * ceil_div(k, 256), 21.0), large = tile_cost(ceil_div(n, 128) * ceil_div(k, 256), 19.0),
                 medium = tile_cost(ceil_div(n, 128) * ceil_div(k, 128), 10.5), small = tile_cost(ceil_div(n, 64) * ceil_div(k, 128), 7.5);
    const double best = std::min(std::min(tall, large), std::min(medium, small));
    if (medium == best)
        return multiply<4, 4, 4, ACCUMULATE>(s, x, y, depth, o, b);
    if (small == best)
        return multiply<4, 2, 4, ACCUMULATE>(s, x, y, depth, o, b);
    return large == best ? multiply<8, 4, 3, ACCUMULATE>(s, x, y, depth, o, b) : multiply<8, 5, 3, ACCUMULATE>(s, x, y, depth, o, b);
}

// Whether the product of many results takes dy as it lies in memory: in whole copies of 16 bytes, every offset in 32 bits (whole stages reach up to four tiles of
// depth beyond the last row). The two launches so and with dy's tiles, m x n x k, us: 64 x 4096 x 4096 19.4 / 19.6, 512 x 2048 x 2048 17.5 / 18.5,
// 2048 x 4096 x 1024 32.6 / 35.0, 4096 x 9304 x 2048 155 / 173, 8192^3 1039 / 1093.
bool reads_columns(const WeightGradient& w, size_t m)
{
    return w.dtype == kBF16 && w.n % 8 == 0 && w.dy_stride % 8 == 0 && reinterpret_cast<uintptr_t>(w.dy) % 16 == 0 &&
           w.dy_stride >= (int64_t) w.n && (uint64_t) w.dy_stride < (uint64_t) 1 << 31 && (m + 4 * kDepth) * (uint64_t) w.dy_stride * 2 < 0xffffffffu;
}

template <int DT>
struct PackLauncher
{
    static hipError_t run(hipStream_t s, const Pack& a)
    {
        const uint32_t blocks = (a.x_chunks + a.y_chunks) * a.runs;
        if (a.n % 2 == 0)
            weight_gradient_pack_kernel<DT, true><<<blocks, kThreads, 0, s>>>(a);
        else
            weight_gradient_pack_kernel<DT, false><<<blocks, kThreads, 0, s>>>(a);
        return hipGetLastError();
    }
};

template <bool EVEN, bool ACCUMULATE, int XW>
struct Direct
{
    template <int DT>
    struct ForType
    {
        static hipError_t run(hipStream_t s, const Pack& a, const Output& o, float* db, size_t part)
        {
            const auto kernel = &weight_gradient_direct_kernel<DT, EVEN, ACCUMULATE, XW>;
            const dim3 grid((uint32_t) ceil_div(a.k, 16 * XW), (uint32_t) ceil_div(a.n, 32), a.runs);
            // (512^3 in single precision with 4 / 8 wavefronts 7.4 / 6.1, but 64 x 1024 x 1024 5.0 / 6.7)
            const uint32_t waves = a.m_tiles >= 8 && grid.x * grid.y <= 2 * kComputeUnits ? 8 : 4, bytes = waves * (2 * XW * 1024 + 512);
            static std::atomic<uint64_t> known{0};
            const hipError_t allowed = allow_lds(reinterpret_cast<const void*>(kernel), 8 * (2 * XW * 1024 + 512), known);
            if (allowed != hipSuccess)
                return allowed;
            kernel<<<grid, waves * 64, bytes, s>>>(a, o, db, part);
            return hipGetLastError();
        }
    };
};
template <bool EVEN, bool ACCUMULATE>
hipError_t direct(hipStream_t s, int dtype, const Pack& a, const Output& o, float* db, size_t part = 0)
{
    // Four columns of x8 a lane, where there is work for it, share what becomes of dy; m x n x k, us with four and two: 257 x 2048 x 429 in single precision
    // 8.5 / 9.5, 512 x 1024 x 1024 11.0 / 13.4, in bfloat16 7.1 / 7.5 and 8.7 / 9.8, but 512^3 7.0 / 5.7 and 128 x 1024 x 1024 6.1 / 5.9.
    if (ceil_div(a.k, 32) * ceil_div(a.n, 32) * a.m_tiles >= 28 * kComputeUnits)
        return by_dtype<Direct<EVEN, ACCUMULATE, 4>::template ForType>(dtype, s, a, o, db, part);
    return by_dtype<Direct<EVEN, ACCUMULATE, 2>::template ForType>(dtype, s, a, o, db, part);
}

} // namespace

size_t weight_gradient_workspace_bytes(size_t m, size_t n, size_t k, int dtype)
{
    const Workspace w = workspace_of(m, n, k, dtype);
    return w.x + w.y + w.sums;
}

size_t weight_gradient_workgroups(size_t m, size_t n, size_t k)
{
    const size_t m_tiles = depth_tiles(std::min(m, kMostRows)), pack = (ceil_div(k, kXCols) + ceil_div(n, kYCols)) * ceil_div(m_tiles, run_tiles(m_tiles, n, k));
    return std::max(std::max(pack, 2 * ceil_div(k, 32)), 2 * kComputeUnits + ceil_div(n, kThreads)); // (one launch has up to twice the threads)
}

hipError_t launch_weight_gradient(hipStream_t s, const WeightGradient& w)
{
    const Workspace ws = workspace_of(w.m, w.n, w.k, w.dtype);
    char* base = static_cast<char*>(w.workspace);
    Pack a;
    a.dy_stride = w.dy_stride;
    a.n = (uint32_t) w.n;
    a.k = (uint32_t) w.k;
    a.pitch = (uint32_t) save8_pitch(w.k);
    a.x_chunks = (uint32_t) ceil_div(w.k, kXCols);
    a.y_chunks = (uint32_t) ceil_div(w.n, kYCols);
    a.x_tiles = base;
    a.y_tiles = base + ws.x;
    a.sums = w.db != nullptr ? reinterpret_cast<float*>(base + ws.x + ws.y) : nullptr;
    const uint8_t* scales = static_cast<const uint8_t*>(w.saved) + w.m * a.pitch;
    Output o = {};
    o.out = w.dw;
    o.stride = w.dw_stride;
    o.rows = (uint32_t) w.n;
    o.cols = (uint32_t) w.k;
    const Way way = way_of(w.m, w.n, w.k, w.dtype);
    if (way == Way::kDirect || way == Way::kParts)
    {
        a.dy = w.dy;
        a.saved = static_cast<const int8_t*>(w.saved);
        a.scales = scales;
        a.m = (uint32_t) w.m;
        a.m_tiles = (uint32_t) ceil_div(w.m, kDepth);
        a.run_tiles = a.m_tiles;
        a.runs = 1;
        if (way == Way::kParts)
        {
            const size_t part = w.n * w.k + w.n;
            a.run_tiles = (uint32_t) ceil_div(a.m_tiles, depth_parts(w.m, w.n, w.k));
            a.runs = (uint32_t) ceil_div(a.m_tiles, a.run_tiles);
            Output parts = o;
            parts.out = base;
            parts.stride = (int64_t) w.k;
            float* sums = w.db != nullptr ? reinterpret_cast<float*>(base) + w.n * w.k : nullptr;
            const hipError_t rc = w.n % 2 == 0 ? direct<true, false>(s, w.dtype, a, parts, sums, part) : direct<false, false>(s, w.dtype, a, parts, sums, part);
            if (rc != hipSuccess)
                return rc;
            const auto join = w.accumulate ? &weight_gradient_join_kernel<true> : &weight_gradient_join_kernel<false>;
            join<<<(uint32_t) ceil_div(part, kThreads), kThreads, 0, s>>>(reinterpret_cast<const float*>(base), a.runs, (uint32_t) part, o, w.db);
            return hipGetLastError();
        }
        if (w.n % 2 == 0)
            return w.accumulate ? direct<true, true>(s, w.dtype, a, o, w.db) : direct<true, false>(s, w.dtype, a, o, w.db);
        return w.accumulate ? direct<false, true>(s, w.dtype, a, o, w.db) : direct<false, false>(s, w.dtype, a, o, w.db);
    }
    size_t row = 0;
    do
    {
        const size_t m = std::min(w.m - row, kMostRows);
        const bool columns = reads_columns(w, m);
        a.dy = static_cast<const char*>(w.dy) + (int64_t) row * w.dy_stride * (w.dtype == kF32 ? 4 : 2);
        a.saved = static_cast<const int8_t*>(w.saved) + row * a.pitch;
        a.scales = scales + row * (a.pitch / kBlock);
        a.m = (uint32_t) m;
        a.m_tiles = (uint32_t) depth_tiles(m);
        a.run_tiles = run_tiles(depth_tiles(std::min(w.m, kMostRows)), w.n, w.k);
        a.runs = (uint32_t) ceil_div(a.m_tiles, a.run_tiles);
        hipError_t rc = hipSuccess;
        if (m != 0 && columns)
        {
            weight_gradient_pack_x_kernel<<<(a.x_chunks + (w.db != nullptr ? (uint32_t) ceil_div(w.n, kSumCols) : 0)) * a.runs, kThreads, 0, s>>>(a);
            rc = hipGetLastError();
        }
        else if (m != 0)
            rc = by_dtype<PackLauncher>(w.dtype, s, a);
        if (rc != hipSuccess)
            return rc;
        const Tiles x = {a.x_tiles, nullptr, (uint32_t) ceil_div(w.k, 16), a.m_tiles};
        const Tiles y = {a.y_tiles, nullptr, (uint32_t) ceil_div(w.n, 16), a.m_tiles * (uint32_t) terms_of(w.dtype)};
        const Sums b = {a.sums, w.db, a.runs, (uint32_t) w.n, 0};
        const bool accumulate = w.accumulate || row != 0;
        if (columns)
        {
            const Columns c = {static_cast<const char*>(a.dy), (uint32_t) (w.dy_stride * 2), a.m, a.n};
            rc = accumulate ? multiply_best<true>(s, x, c, a.m_tiles, o, b) : multiply_best<false>(s, x, c, a.m_tiles, o, b);
        }
        else
            rc = accumulate ? multiply_best<true>(s, x, y, y.k_tiles, o, b) : multiply_best<false>(s, x, y, y.k_tiles, o, b);
        if (rc != hipSuccess)
            return rc;
        row += m;
    } while (row < w.m);
    return hipSuccess;
}

} // namespace lowbit
} // namespace cntkq
