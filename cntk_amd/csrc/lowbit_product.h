// The matrix products of the low-bit operators: out[i, j] = sum over k of P[i, k] Q[j, k], both operands in tiles of 1 KB that hold
// a matrix instruction's operand lane by lane (lowbit_formats.h for the 4-bit ones; in bfloat16 a tile is 16 rows x 32, lane l holding
// row l % 16, columns (l / 16) * 8 to + 7).
//
// Q's rows go through the instruction's first operand: a lane's four results are then four neighbouring columns of one output row.
// One pair of tiles is one matrix instruction of 16 cycles whichever the format, so one kernel serves both.
#pragma once

#include "lowbit_internal.h"

#include <atomic>
#include <type_traits>

namespace cntkq {
namespace lowbit {

// An operand in tiles. Tile (t, k) lies at tiles + (t * k_tiles + k) * 1 KB, its scale group at scales + ((t / 4) * k_tiles + k) * 256.
struct Tiles
{
    const char* tiles;
    const char* scales;
    uint32_t row_tiles;
    uint32_t k_tiles; // an even number, in memory: the other operand may have a multiple of them, over which this one's repeat
};

// A bfloat16 operand as a matrix in memory whose columns are the operand's rows: column j of row k at base + k * pitch + 2 j. Multiples of 16
// bytes all of them: base, pitch and 2 cols; no offset that a product of whole stages reaches is above 32 bits.
struct Columns
{
    const char* base;
    uint32_t pitch, rows, cols;
};

struct Output
{
    const void* bias;
    int bias_dtype;
    void* out;
    int64_t stride;
    uint32_t rows, cols;
};

constexpr uint32_t kComputeUnits = 256; // of an MI355X, with 160 KB of LDS each

// Workgroups for `blocks` blocks of results: as many as the device holds at a time, a multiple of its eight dies.
inline uint32_t tile_workgroups(uint32_t blocks, int per_unit)
{
    const uint32_t most = kComputeUnits * (uint32_t) per_unit;
    return blocks < most ? blocks : most;
}

// What a kernel of `c` (the time of a stage of two workgroups on a compute unit, in any unit) takes for `blocks` blocks: whole rounds of two
// workgroups on every compute unit, and the rest, for which a unit with one workgroup needs 0.7 of the time.
inline double tile_cost(size_t blocks, double c)
{
    const size_t round = 2 * kComputeUnits, rest = blocks % round;
    return (double) (blocks / round) * c + (rest == 0 ? 0.0 : (rest <= kComputeUnits ? 0.7 * c : c));
}

// How many wavefronts share the depth of a workgroup where there are `groups` of them: at least two tiles of depth for each, and not more
// in all than the device holds at a time; 4 to 16. (512 x 2048 x 2048 in 4 bits, us with 4 / 8 / 16: 6.1 / 5.5 / 6.9; 64 x 9304 x 2048: 11.3 / 7.8 / 6.7.)
inline uint32_t depth_waves(size_t groups, uint32_t depth)
{
    uint32_t waves = 4;
    while (waves < 16 && waves * 4 <= depth && groups * waves * 2 <= 32 * kComputeUnits)
        waves *= 2;
    return waves;
}

// Lets a kernel be launched with `bytes` of LDS on the current device, asked for once on each (bits of `known`).
inline hipError_t allow_lds(const void* kernel, int bytes, std::atomic<uint64_t>& known)
{
    int device = 0;
    const hipError_t rc = hipGetDevice(&device);
    if (rc != hipSuccess || (device < 64 && (known.load(std::memory_order_relaxed) >> device & 1) != 0))
        return rc;
    const hipError_t set = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (set == hipSuccess && device < 64)
        known.fetch_or((uint64_t) 1 << device, std::memory_order_relaxed);
    return set;
}

#ifdef __HIPCC__

template <int N, int I = 0, typename F>
__device__ __forceinline__ void each(F&& f)
{
    if constexpr (I < N)
    {
        f(std::integral_constant<int, I>());
        each<N, I + 1>(f);
    }
}

// The matrix instructions of the two formats. SQ, SP: which byte of the scale words is meant.
struct Mx4Op
{
    static constexpr bool kScaled = true;
    template <int SQ, int SP>
    static __device__ __forceinline__ f32x4 mma(u32x4 q, u32x4 p, f32x4 c, uint32_t sq, uint32_t sp)
    {
        const i32x8 a = {(int) q[0], (int) q[1], (int) q[2], (int) q[3], 0, 0, 0, 0};
        const i32x8 b = {(int) p[0], (int) p[1], (int) p[2], (int) p[3], 0, 0, 0, 0};
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 4, SQ, (int) sq, SP, (int) sp); // 4: the 4-bit format
    }
};
struct Bf16Op
{
    static constexpr bool kScaled = false;
    template <int SQ, int SP>
    static __device__ __forceinline__ f32x4 mma(u32x4 q, u32x4 p, f32x4 c, uint32_t, uint32_t)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, q), __builtin_bit_cast(bf16x8, p), c, 0, 0, 0);
    }
};

// A run of memory that the lanes of a wavefront copy from: a lane whose own offset lies at its end or beyond reads nothing and gets zeros. The offset
// that all lanes share takes no part in that check.
struct Span
{
    const char* base;
    uint32_t bytes;
};
__device__ __forceinline__ Span span(const char* base, uint64_t bytes)
{
    return {base, bytes < 0xffffffffu ? (uint32_t) bytes : 0xffffffffu};
}
// One lane's copy of 16 (4) bytes straight to LDS: `lane_at` + `at` is the place in the span, `to` the wavefront's place in LDS, where the
// lanes follow one another. Whether a lane reads is a matter of `lane_at` alone: with any `at` that is used, a lane below the span's end stays below it.
template <int BYTES>
__device__ __forceinline__ void copy_to_lds(const Span& from, uint32_t lane_at, uint32_t at, char* to)
{
    // (the span is the same for all lanes; said so, since 64-bit comparisons leave their results in vector registers)
    const uint64_t p = reinterpret_cast<uint64_t>(from.base);
    const uint32_t low = __builtin_amdgcn_readfirstlane((uint32_t) p), high = __builtin_amdgcn_readfirstlane((uint32_t) (p >> 32));
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>((uint64_t) high << 32 | low), 0, __builtin_amdgcn_readfirstlane(from.bytes), 0x00027000);
    auto* l = (__attribute__((address_space(3))) void*) to;
    if constexpr (BYTES == 16)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, l, 16, lane_at, at, 0, 0);
    else
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, l, 4, lane_at, at, 0, 0);
}

// Waits for all but the last N of the wavefront's accesses to memory, copies to LDS among them. The compiler takes no part in the order of
// those copies with the reads of LDS behind a barrier; it does count this wait among its own, which spares it waits for registers
// that were loaded long ago.
template <int N>
__device__ __forceinline__ void wait_copies()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 7 << 4 | 15 << 8); // the other two counters at their ends
    asm volatile("" ::: "memory");
}
// Every wavefront of the workgroup is here.
__device__ __forceinline__ void meet()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
// What was read from and written to LDS is over.
__device__ __forceinline__ void wait_lds()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(15 | 3 << 14 | 7 << 4 | 0 << 8);
    asm volatile("" ::: "memory");
}

// The bias of a column (zero without any; beyond the last column the last one's).
__device__ __forceinline__ float bias_of(const Output& o, uint32_t col)
{
    if (o.bias == nullptr)
        return 0.0f;
    col = min(col, o.cols - 1);
    if (o.bias_dtype == kF32)
        return static_cast<const float*>(o.bias)[col];
    if (o.bias_dtype == kF16)
        return (float) static_cast<const _Float16*>(o.bias)[col];
    return (float) static_cast<const __bf16*>(o.bias)[col];
}

// Four neighbouring values of an output row, from column `col` on, as far as they are inside; ACCUMULATE: added to what is there.
template <int DT, bool ACCUMULATE>
__device__ __forceinline__ void write4(const Output& o, uint32_t row, uint32_t col, f32x4 v)
{
    typedef typename Type<DT>::T T;
    T* p = static_cast<T*>(o.out) + (int64_t) row * o.stride + col;
    const bool there = row < o.rows;
    if (there && col + 4 <= o.cols)
    {
        if constexpr (DT == kF32)
        {
            if constexpr (ACCUMULATE)
                v += *reinterpret_cast<const f32x4_at4*>(p);
            *reinterpret_cast<f32x4_at4*>(p) = v;
        }
        else
            *reinterpret_cast<u32x2_at2*>(p) = u32x2{pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3])};
    }
    else if (there)
    {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (col + i < o.cols)
                p[i] = Type<DT>::down(v[i] + (ACCUMULATE ? (float) p[i] : 0.0f));
    }
}
// Two tiles side by side: 16-bit results change lanes so that a lane has eight neighbouring columns, 16 bytes, of its row. Groups of 16 lanes
// hold columns 4 g .. 4 g + 3 of both tiles; the first swap brings the second tile's lower half to the first's upper lanes and the other
// way round, the second one pairs neighbouring groups.
template <int DT>
__device__ __forceinline__ void write_pair(const Output& o, uint32_t row, uint32_t first_col, uint32_t lane, f32x4 a, f32x4 b)
{
    static_assert(DT != kF32, "32-bit results are 16 bytes as they are");
    typedef typename Type<DT>::T T;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
    {
        const auto halves = __builtin_amdgcn_permlane32_swap(pack2<DT>(a[2 * i], a[2 * i + 1]), pack2<DT>(b[2 * i], b[2 * i + 1]), false, false);
        const auto quarters = __builtin_amdgcn_permlane16_swap(halves[0], halves[1], false, false);
        w[i] = quarters[0];
        w[i + 2] = quarters[1];
    }
    const uint32_t col = first_col + lane / 16 * 8;
    T* p = static_cast<T*>(o.out) + (int64_t) row * o.stride + col;
    const bool there = row < o.rows;
    if (there && col + 8 <= o.cols)
        *reinterpret_cast<u32x4_at2*>(p) = u32x4{w[0], w[1], w[2], w[3]};
    else if (there)
    {
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (col + i < o.cols)
                reinterpret_cast<uint16_t*>(p)[i] = (uint16_t) (w[i / 2] >> (16 * (i % 2)));
    }
}

// The block of output tiles that has number `index`. Workgroups are dealt to the eight dies in turn, each with a second-level cache
// of its own: every die gets a run of blocks, walked in bands of four block rows, so that the blocks a die works on at a time share
// rows and columns.
__device__ __forceinline__ void block_of(uint32_t index, uint32_t p_blocks, uint32_t q_blocks, uint32_t& bp, uint32_t& bq)
{
    const uint32_t total = p_blocks * q_blocks, die = index % 8, at = index / 8;
    const uint32_t each_die = total / 8, more = total % 8;
    const uint32_t t = die * each_die + min(die, more) + at;
    const uint32_t band = t / (4 * q_blocks), high = min(4u, p_blocks - band * 4), in = t - band * 4 * q_blocks;
    bp = band * 4 + in % high;
    bq = in / high;
}

// Four numbers of a row that lies along memory's other axis, from LDS: a group of 16 lanes reads four rows of 16 numbers, four to a lane,
// and lane i of it gets column i. (Nothing else writes there meanwhile: not said, the compiler lets every such read wait for all copies to LDS.)
typedef short i16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x2 read_turned(__attribute__((address_space(3))) i16x4* __restrict at)
{
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(at));
}

// A workgroup of 2 x 2 wavefronts, each with TQ x TP tiles of results, goes through blocks first, first + step, ..., one tile of
// depth at a time. What it reads is one stream over all its blocks: tiles are copied to LDS NB - 1 stages ahead, into one of NB buffers,
// across the change of blocks too. A stage is worked off row of tiles by row of tiles (of Q); three rows ahead of its use a row's Q
// fragment is read from LDS, and P fragments of the next stage with it. So the matrix unit waits neither for memory nor for LDS, and the first
// stages of a block arrive while the results of the one before are written.
//
// PT: Tiles, or Columns for a P that is turned over on its way from LDS to registers. Of such a one a stage is 32 rows of memory as long as
// the block is high, in chunks of 16 bytes that the copies share out, so a copy takes a few runs of a row. Reading a tile, 16 lanes read
// 32 bytes of each of four rows, the next 16 lanes of the four rows 8 further on, which lie at the same banks; the tiles of a row of LDS have
// changed places by a pattern that sets them apart. (Without it 28 % of LDS's cycles were conflicts, and 4096 x 9304 x 2048 took 149.5 us instead of 147.)
template <typename Op, int TQ, int TP, int NB, bool ACCUMULATE = false, typename PT = Tiles>
struct TileKernel
{
    static constexpr int WQ = 2, WP = 2, kWaves = WQ * WP, kThreads = kWaves * 64;
    static constexpr int kQTiles = WQ * TQ, kPTiles = WP * TP;
    static_assert(TQ % 4 == 0 && (!Op::kScaled || TP % 2 == 0), "Q's scale words are whole for a wavefront, P's for the workgroup");
    static constexpr int kQGroups = kQTiles / 4, kPGroups = kPTiles / 4;
    // copies of a wavefront for a stage: of Q's tiles, of P's, and of the scale groups (where there are fewer than wavefronts, some are
    // copied twice, by wavefronts that would otherwise have one copy less to wait for than the others)
    static constexpr int kQCopies = (kQTiles + kWaves - 1) / kWaves, kPCopies = (kPTiles + kWaves - 1) / kWaves;
    static_assert(kQCopies * kWaves == kQTiles, "Q's tiles are shared out evenly");
    static constexpr int kPerStage = kQCopies + kPCopies + (Op::kScaled ? 2 : 0);
    static_assert(!Op::kScaled || (kQGroups <= kWaves && kPGroups <= kWaves), "a scale group a wavefront");
    static constexpr int kTileLds = (kQTiles + kPTiles) * (int) kTileBytes;
    static constexpr int kStage = kTileLds + (Op::kScaled ? (kQGroups + kPGroups) * (int) kScaleGroupBytes : 0);
    static constexpr int kBuffers = NB;
    static constexpr int kBiasLds = Op::kScaled ? kQTiles * 16 * 4 : 0; // the biases of a block's columns
    static constexpr int kLds = kBuffers * kStage + kBiasLds;
    static constexpr int kPerUnit = kLds <= 80 * 1024 ? 2 : 1; // workgroups on a compute unit
    static constexpr int kPWords = (TP + 3 + (TP % 4 != 0 ? 2 : 0)) / 4; // scale words that a wavefront's P tiles touch

    static constexpr int kRing = 4, kAhead = 3; // Q fragments held, and how many rows ahead they are read
    // what a wavefront holds of a stage throughout: its P fragments and scales
    struct Fragments
    {
        u32x4 p[TP];
        uint32_t q_scales[TQ / 4], p_scales[(TP + 3) / 4];
    };

    static constexpr bool kTurned = std::is_same<PT, Columns>::value;
    static_assert(!kTurned || !Op::kScaled, "bfloat16 only");
    static constexpr uint32_t kChunks = 2 * kPTiles; // of a row of a stage of Columns

    Tiles q;
    PT p;
    uint32_t p_turn[2]; // where the lane's rows of a stage of Columns are, for the even tiles and the odd ones of the wavefront
    uint32_t depth, p_blocks, q_blocks;
    char* lds;
    uint32_t lane, wave, step;
    // the block whose stages are copied, where the wavefront's tiles and scales of it lie, and the same of the block after it
    uint32_t fill_block, fill_k, q_at, p_at, scale_at;
    struct Spans
    {
        Span q, p, q_scales, p_scales;
    };
    Spans spans, next_spans;
    uint32_t q_lane_at[kQCopies], p_lane_at[kPCopies];
    uint32_t fill_buffer, read_buffer;

    __device__ __forceinline__ uint32_t blocks() const { return p_blocks * q_blocks; }

    // The tiles of t from `first` on, and the scale group that is the wavefront's, `group` of t, or the last one.
    // A lane's offset is a whole number of rows of tiles and a place in a tile, the shared one is less than a row.
    static __device__ __forceinline__ Span tiles_from(const Tiles& t, uint32_t first)
    {
        const uint64_t row_bytes = (uint64_t) t.k_tiles * kTileBytes;
        return span(t.tiles + first * row_bytes, first < t.row_tiles ? (t.row_tiles - first) * row_bytes : 0);
    }
    // All rows from column 16 * first on. (Whole stages end beyond the last row: the stage's offset is added to the lanes' own, which are checked.)
    static __device__ __forceinline__ Span tiles_from(const Columns& t, uint32_t first)
    {
        return span(t.base + first * 32, (uint64_t) (t.rows - 1) * t.pitch + (t.cols - first * 16) * 2);
    }
    // tile t of a row of a stage lies where tile t ^ exchange(row) would
    static __device__ __forceinline__ uint32_t exchange(uint32_t row)
    {
        if constexpr (kPTiles % 8 == 0) // rows of 256 bytes
            return (row & 3) | (row >> 1 & 4);
        else if constexpr (kPTiles % 4 == 0) // 128 bytes
            return (row >> 1 & 1) | (row >> 2 & 2);
        else // an odd multiple of 64 bytes
            return row >> 3 & 1;
    }
    static __device__ __forceinline__ Span scales_of(const Tiles& t, uint32_t group)
    {
        const uint64_t group_bytes = (uint64_t) t.k_tiles * kScaleGroupBytes;
        return span(t.scales + min(group, (t.row_tiles - 1) / 4) * group_bytes, group_bytes);
    }
    __device__ __forceinline__ void aim(uint32_t block, Spans& s) const
    {
        uint32_t bp, bq;
        block_of(block, p_blocks, q_blocks, bp, bq);
        // (beyond the last tile it is that one, whose results are not written: an empty span would leave it to the shared offset what is read)
        s.q = tiles_from(q, min(bq * kQTiles + wave * kQCopies, q.row_tiles - 1));
        s.p = tiles_from(p, bp * kPTiles);
        if constexpr (Op::kScaled)
        {
            s.q_scales = scales_of(q, bq * kQGroups + min(wave, (uint32_t) kQGroups - 1));
            s.p_scales = scales_of(p, bp * kPGroups + min(wave, (uint32_t) kPGroups - 1));
        }
        else
            s.q_scales = s.p_scales = {nullptr, 0};
    }
    // which of P's tiles the wavefront copies
    __device__ __forceinline__ uint32_t p_tile(int i) const { return min(wave * kPCopies + i, (uint32_t) kPTiles - 1); }

    // the part of copying one stage that belongs to row I of the stage that is multiplied meanwhile
    template <int I>
    __device__ __forceinline__ void fill_row()
    {
        char* to = lds + fill_buffer * kStage;
#pragma unroll
        for (int i = I; i < kQCopies; i += TQ)
            copy_to_lds<16>(spans.q, q_lane_at[i], q_at, to + (wave * kQCopies + i) * kTileBytes);
#pragma unroll
        for (int i = (I + 2) % TQ; i < kPCopies; i += TQ)
            copy_to_lds<16>(spans.p, p_lane_at[i] + (kTurned ? p_at : 0), kTurned ? 0 : p_at, to + (kQTiles + p_tile(i)) * kTileBytes);
        if constexpr (Op::kScaled && I == 1)
            copy_to_lds<4>(spans.q_scales, lane * 4, scale_at, to + kTileLds + min(wave, (uint32_t) kQGroups - 1) * kScaleGroupBytes);
        if constexpr (Op::kScaled && I == 3)
            copy_to_lds<4>(spans.p_scales, lane * 4, scale_at, to + kTileLds + (kQGroups + min(wave, (uint32_t) kPGroups - 1)) * kScaleGroupBytes);
    }
    // b for `second`, a otherwise. (Each value on its way through readfirstlane, which costs nothing: a choice between two members becomes one
    // between their addresses else, and the object that they belong to then stays in memory.)
    static __device__ __forceinline__ uint32_t pick(bool second, uint32_t a, uint32_t b)
    {
        const uint32_t x = __builtin_amdgcn_readfirstlane(a), y = __builtin_amdgcn_readfirstlane(b);
        return second ? y : x;
    }
    static __device__ __forceinline__ Span pick(bool second, const Span& a, const Span& b)
    {
        const uint64_t x = reinterpret_cast<uint64_t>(a.base), y = reinterpret_cast<uint64_t>(b.base);
        const uint32_t low = pick(second, (uint32_t) x, (uint32_t) y), high = pick(second, (uint32_t) (x >> 32), (uint32_t) (y >> 32));
        return {reinterpret_cast<const char*>((uint64_t) high << 32 | low), pick(second, a.bytes, b.bytes)};
    }
    // On to the next stage, without a branch; after the last stage of all it is copied again, and nobody reads it.
    __device__ __forceinline__ void fill_next()
    {
        fill_buffer = fill_buffer + 1 == kBuffers ? 0 : fill_buffer + 1;
        fill_k = __builtin_amdgcn_readfirstlane(fill_k + 1);
        const bool over = fill_k == depth;
        fill_k = over ? 0 : fill_k;
        q_at += kTileBytes;
        if constexpr (kTurned)
            p_at += 32 * p.pitch;
        else
            p_at += kTileBytes;
        // (an operand may have fewer tiles of depth than the other, over which it repeats)
        q_at = over || (!Op::kScaled && q_at == q.k_tiles * kTileBytes) ? 0 : q_at;
        if constexpr (kTurned)
            p_at = over ? 0 : p_at;
        else
            p_at = over || (!Op::kScaled && p_at == p.k_tiles * kTileBytes) ? 0 : p_at;
        scale_at = over ? 0 : scale_at + kScaleGroupBytes;
        spans.q = pick(over, spans.q, next_spans.q);
        spans.p = pick(over, spans.p, next_spans.p);
        spans.q_scales = pick(over, spans.q_scales, next_spans.q_scales);
        spans.p_scales = pick(over, spans.p_scales, next_spans.p_scales);
        fill_block = over ? min(fill_block + step, blocks()) : fill_block;
    }
    // where the stages after the present block's come from; called once for each block before the copies get there
    __device__ __forceinline__ void look_ahead()
    {
        const uint32_t block = fill_block + step;
        aim(block < blocks() ? block : min(fill_block, blocks() - 1), next_spans);
    }
    __device__ __forceinline__ void fill()
    {
        each<TQ>([&](auto i) { fill_row<i>(); });
        fill_next();
    }
    __device__ __forceinline__ u32x4 read_q(uint32_t buffer, int i) const
    {
        return *reinterpret_cast<const u32x4*>(lds + buffer * kStage + (wave % WQ * TQ + i) * kTileBytes + lane * 16);
    }
    __device__ __forceinline__ u32x4 read_p(uint32_t buffer, int i) const
    {
        if constexpr (kTurned)
        {
            const uint32_t tile = (wave / WQ * TP + i) * 32;
            auto* at = (__attribute__((address_space(3))) i16x4*) (lds + buffer * kStage + kQTiles * kTileBytes + (kPTiles % 4 == 0 ? p_turn[0] ^ tile : p_turn[i % 2] + tile));
            const u32x2 a = read_turned(at), b = read_turned(at + 4 * kChunks * 16 / sizeof(i16x4));
            return u32x4{a[0], a[1], b[0], b[1]};
        }
        else
            return *reinterpret_cast<const u32x4*>(lds + buffer * kStage + (kQTiles + wave / WQ * TP + i) * kTileBytes + lane * 16);
    }
    __device__ __forceinline__ void read_scales(uint32_t buffer, Fragments& f) const
    {
        const char* at = lds + buffer * kStage + kTileLds + lane * 4;
        if constexpr (Op::kScaled)
        {
#pragma unroll
            for (int i = 0; i < TQ / 4; ++i)
                f.q_scales[i] = *reinterpret_cast<const uint32_t*>(at + (wave % WQ * (TQ / 4) + i) * kScaleGroupBytes);
            if constexpr (TP % 4 == 0)
            {
#pragma unroll
                for (int i = 0; i < TP / 4; ++i)
                    f.p_scales[i] = *reinterpret_cast<const uint32_t*>(at + (kQGroups + wave / WQ * (TP / 4) + i) * kScaleGroupBytes);
            }
            else
            {
                // the second wavefront's tiles begin within a word
                const uint32_t first = wave / WQ * TP;
                uint32_t w[kPWords];
#pragma unroll
                for (int i = 0; i < kPWords; ++i)
                    w[i] = *reinterpret_cast<const uint32_t*>(at + (kQGroups + min(first / 4 + i, (uint32_t) kPGroups - 1)) * kScaleGroupBytes);
#pragma unroll
                for (int i = 0; i < (TP + 3) / 4; ++i)
                    f.p_scales[i] = (uint32_t) ((((uint64_t) w[i + 1 < kPWords ? i + 1 : i] << 32) | w[i]) >> (8 * (first % 4)));
            }
        }
    }

    // One stage: `now` and the first kAhead of ring are there, the next stage's are read meanwhile. OUTSTANDING accesses may be on their way at
    // its beginning. (No branch: behind one, the compiler would put the multiplications that it has the choice to.)
    template <int OUTSTANDING>
    __device__ __forceinline__ void stage(Fragments& now, Fragments& next, u32x4 (&ring)[kRing], f32x4 (&acc)[TQ][TP])
    {
        // The next stage is in LDS, and everyone has read the one before this one, whose buffer is filled again: what was read from there has been
        // multiplied.
        wait_copies<OUTSTANDING>();
        meet();
        const uint32_t buffer = read_buffer, after = read_buffer + 1 == kBuffers ? 0 : read_buffer + 1;
        read_buffer = after;
        each<TQ>([&](auto i) {
            __builtin_amdgcn_sched_barrier(0); // the rows stay apart: hoisting every read to the front takes more registers than there are
            ring[(i + kAhead) % kRing] = i + kAhead < TQ ? read_q(buffer, i + kAhead) : read_q(after, i + kAhead - TQ);
#pragma unroll
            for (int j = i; j < TP; j += TQ)
                next.p[j] = read_p(after, j);
            if constexpr (i == 0)
                read_scales(after, next);
            fill_row<i>();
            each<TP>([&](auto j) {
                acc[i][j] = Op::template mma<i % 4, j % 4>(ring[i % kRing], now.p[j], acc[i][j], Op::kScaled ? now.q_scales[i / 4] : 0,
                                                           Op::kScaled ? now.p_scales[j / 4] : 0);
            });
        });
        __builtin_amdgcn_sched_barrier(0);
        fill_next();
    }

    // What a block's results are written with, at least, where it lies inside the output: stores that need not be over before the
    // next block goes on.
    template <int DT>
    static constexpr int kStores = DT == kF32 ? TQ * TP : TQ * TP / 2;

    // `bias`: of the thread's column of the block (4-bit products only)
    template <int DT>
    __device__ __forceinline__ void write(const Output& o, uint32_t block, const f32x4 (&acc)[TQ][TP], float bias) const
    {
        uint32_t bp, bq;
        block_of(block, p_blocks, q_blocks, bp, bq);
        const uint32_t q0 = (bq * kQTiles + wave % WQ * TQ) * 16, p0 = (bp * kPTiles + wave / WQ * TP) * 16;
        const uint32_t col = q0 + lane / 16 * 4, row = p0 + lane % 16;
        float* shared = reinterpret_cast<float*>(lds + kBuffers * kStage);
        if constexpr (Op::kScaled)
        {
            if (depth == 0)
            {
                wait_lds(); // (between two blocks' biases there is otherwise a stage, whose multiplications have waited for them)
                meet();
            }
            if (wave * 64 + lane < kQTiles * 16)
                shared[wave * 64 + lane] = bias;
            wait_lds();
            meet();
        }
        const float* biases = shared + wave % WQ * TQ * 16 + lane / 16 * 4;
        const auto result = [&](auto i, auto j) {
            if constexpr (Op::kScaled)
                return acc[i][j] + *reinterpret_cast<const f32x4*>(biases + i * 16);
            else
                return acc[i][j];
        };
        each<TP>([&](auto j) {
            __builtin_amdgcn_sched_barrier(0); // (as in a stage: row by row, for the registers)
            if constexpr (DT == kF32)
                each<TQ>([&](auto i) { write4<DT, ACCUMULATE>(o, row + j * 16, col + i * 16, result(i, j)); });
            else
                each<TQ / 2>([&](auto i) {
                    write_pair<DT>(o, row + j * 16, q0 + i * 32, lane, result(std::integral_constant<int, 2 * i>(), j),
                                   result(std::integral_constant<int, 2 * i + 1>(), j));
                });
        });
        if (q0 + TQ * 16 > o.cols || p0 + TP * 16 > o.rows)
            wait_copies<0>(); // fewer stores than a block inside has
    }

    template <int DT>
    __device__ __forceinline__ void run(char* memory, const Tiles& q_, const PT& p_, const Output& o, uint32_t depth_, uint32_t p_blocks_,
                                        uint32_t q_blocks_, uint32_t first, uint32_t step_)
    {
        static_assert(TQ % kRing == 0, "a stage leaves the ring where it found it");
        // At a stage's beginning the next one has to be there; of the copies after it all may still be on their way. In the first
        // stages of a block what is waited for was asked for before the stores of the block before: they may be too, where there were as many
        // (a block that ends at the output's edge waits for everything itself).
        constexpr int kOne = (kBuffers - 3) * kPerStage;
        constexpr int kAfterStores = kOne + kStores<DT> < 63 ? kOne + kStores<DT> : 63;
        static_assert((kBuffers == 3 || kBuffers == 4) && kOne <= 63, "as many first stages as are told apart; the counter ends at 63");
        q = q_;
        p = p_;
        depth = depth_;
        p_blocks = p_blocks_;
        q_blocks = q_blocks_;
        lds = memory;
        lane = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0));
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
        step = step_;
        fill_buffer = read_buffer = 0;
        Fragments a, b;
        u32x4 ring[kRing];
        if (depth != 0)
        {
#pragma unroll
            for (int i = 0; i < kQCopies; ++i)
                q_lane_at[i] = i * q.k_tiles * kTileBytes + lane * 16;
#pragma unroll
            for (int i = 0; i < kPCopies; ++i)
            {
                if constexpr (kTurned)
                {
                    const uint32_t chunk = p_tile(i) * 64 + lane, row = chunk / kChunks;
                    p_lane_at[i] = row * p.pitch + (chunk % kChunks ^ 2 * exchange(row)) * 16;
                }
                else
                    p_lane_at[i] = p_tile(i) * p.k_tiles * kTileBytes + lane * 16;
            }
            if constexpr (kTurned)
            {
                const uint32_t row = lane / 16 * 8 + lane % 16 / 4; // and the row four further on, whose tiles are exchanged alike
                const uint32_t at = row * kChunks * 16 + lane % 4 * 8, odd = wave / WQ * TP % 2;
                if constexpr (kPTiles % 4 == 0)
                    p_turn[0] = at + exchange(row) * 32;
                else
                {
                    p_turn[0] = odd ? at - exchange(row) * 32 : at + exchange(row) * 32;
                    p_turn[1] = odd ? at + exchange(row) * 32 : at - exchange(row) * 32;
                }
            }
            fill_block = first;
            fill_k = q_at = p_at = scale_at = 0;
            aim(first, spans);
            look_ahead();
            for (int i = 0; i < kBuffers - 1; ++i)
            {
                fill();
                if (fill_k == 0)
                    look_ahead();
            }
            wait_copies<0>();
            meet();
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                ring[i] = read_q(0, i);
#pragma unroll
            for (int i = 0; i < TP; ++i)
                a.p[i] = read_p(0, i);
            read_scales(0, a);
        }
        for (uint32_t block = first; block < blocks(); block += step)
        {
            f32x4 acc[TQ][TP] = {};
            float bias = 0.0f;
            if constexpr (Op::kScaled)
            {
                uint32_t bp, bq;
                block_of(block, p_blocks, q_blocks, bp, bq);
                bias = bias_of(o, bq * kQTiles * 16 + (wave * 64 + lane) % (kQTiles * 16));
            }
            look_ahead();
            if (depth != 0)
            {
                stage<kAfterStores>(a, b, ring, acc);
                stage<kBuffers == 3 ? kOne : kAfterStores>(b, a, ring, acc);
#pragma nounroll
                for (uint32_t k = 2; k < depth; k += 2)
                {
                    stage<kOne>(a, b, ring, acc);
                    stage<kOne>(b, a, ring, acc);
                }
            }
            write<DT>(o, block, acc, bias);
        }
        wait_copies<0>(); // nothing may be on its way to the LDS of a workgroup that is gone
    }
};

#endif // __HIPCC__

} // namespace lowbit
} // namespace cntkq
