// Product of e4m3 matrices with an fp32 scale per block of 128:
//
//   out[m, n] = residual[m, n] + sum_g sx[m, g] sw[n / 128, g] sum_{k in block g} x[m, k] w[n, k]
//
// x [M, K] has a scale per row and 128 columns, w [N, K] one per 128 rows and
// 128 columns.  The tensor cores form each 128-deep block product in fp32 tensor
// memory; the epilogue warps scale it and add it to fp32 registers while the next
// blocks' products run into other parts of the tensor memory.  One rounding, of
// the finished sum with the residual.
//
// Many rows (tile_kernel): tensor memory lanes are rows of x, columns are rows
// of w, so a thread's scale is one number a block.  Persistent CTAs of 128 x TN
// tiles, the block products in 2 to 4 parts of the tensor memory.  What bounds it
// short of the power limit are the products with their barriers, 500 ns of a 620 ns
// block of 128 x 256 (512 clocks of tensor pipe), and then, each as much, the
// operands' way from L2 beside them and the epilogue's reads, which hold them up:
// at 4096 x 8256 x 5120, 198 us, copies alone take 144, products alone 162, reads
// alone 149, products with either of the others 190 (at 512 x 5120 x 4096, 18.6:
// 14.2, 16.6, 15.5, with reads 18.4, with copies 17.2).  In a loop of seconds the GPU
// runs at its 1000 W limit, 1.53 GHz.  Measured on the way at 16384 x 8256 x 5120:
// packed fp32 pairs in the epilogue 811 us, single ones, a part released as soon as
// it is in registers, scales loaded four blocks ahead and two product warps in turn
// 685 to 700 us (2.0 PFLOP/s; 794 to 814 us at the power limit).  Pairs of CTAs
// (256 x 256 tiles, 32 KB a block and SM) measured 705 and 827 us.
// Few rows (split_kernel): the weights' bytes bound the call.  Lanes are 128
// rows of w (one scale a block), columns the rows of x; the CTAs of a cluster
// split K and add their sums in rank order through distributed shared memory.
// Weights from memory (several sets in turn): 8 x 16384 x 8192 25.6 us (5.2 TB/s),
// 8 to 32 x 8256 x 5120 12.1 to 12.5 us (3.5 TB/s, start and end of ten blocks a CTA
// the rest), 64 rows 14.0, 128 rows 20.7, of 5120 x 4096 9.9, 12.1 and 17.6 us at 32,
// 64 and 128; with one set of 42 MB in L2 8 rows take 9.0 us.
//
// Operands arrive by TMA (128-byte swizzle; zeros past K, M and N), one warp
// issues the copies, one or two the products.  Every wait is bounded: outputs whose
// sums a wait gave up on are NaN, and status says so.  No warp leaves before the
// copies and products it issued have ended.
#include <cooperative_groups.h>
#include <cudaTypedefs.h>

#include <mutex>

#include <type_traits>

#include "sq_tc.cuh"
#include "sq_vec.cuh"

namespace sq {
namespace {

constexpr int kBlock = 128;                // depth of a scale block and of a pipeline stage
constexpr int kEpilogueWarps = 8;
constexpr int kMostParts = 4;              // blocks in tensor memory at a time
constexpr int kRowTile = 128 * kBlock;     // bytes of a 128-row operand tile
constexpr int kScaleGroup = 4;             // blocks whose scales are loaded together
constexpr int kMostRows = 0x7fff0000;      // of either operand: the end of a tile is an int too

struct Sync {
    uint64_t full[8], empty[8];  // operand stages
    uint64_t ready[kMostParts], free_[kMostParts];  // parts of the tensor memory
    uint64_t done[2];                               // all products of a product warp
    uint32_t tmem;
    int abort;
};

// Position in a ring (of operand stages, of parts of the tensor memory) and the parity of its use.
template <int STAGES>
struct Ring {
    int stage = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void next() {
        if (++stage == STAGES) stage = 0, parity ^= 1;
    }
    __device__ __forceinline__ void back() {
        if (--stage < 0) stage = STAGES - 1, parity ^= 1;
    }
};

// A copy warp leaves once the copies it issued have landed (with a limit again), also where another
// warp gave up on them: those of the last `count` <= STAGES stages before `at`.
template <int STAGES>
__device__ __forceinline__ void drain_copies(Sync &s, Ring<STAGES> at, int64_t count) {
    int never = 0;
    for (int i = 0; i < STAGES && i < count; ++i) {
        at.back();
        tc::bar_wait(&s.full[at.stage], at.parity, &never, tc::kWaitClocks);
    }
}

__device__ __forceinline__ void set_up(Sync &s, int stages, uint32_t columns, int warp) {
    if (threadIdx.x == 0) {
        for (int i = 0; i < stages; ++i) {
            tc::bar_init(&s.full[i], 1);
            tc::bar_init(&s.empty[i], 1);
        }
        for (int i = 0; i < kMostParts; ++i) {
            tc::bar_init(&s.ready[i], 1);
            tc::bar_init(&s.free_[i], kEpilogueWarps);
        }
        for (int i = 0; i < 2; ++i) tc::bar_init(&s.done[i], 1);
        s.abort = 0;
        tc::bar_init_fence();
    }
    if (warp == kEpilogueWarps + 1) tc::tmem_alloc(&s.tmem, columns);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
}

// Waits (with a limit again) until the products that product warp w issued have ended, once.
__device__ __forceinline__ void end_products(Sync &s, int w) {
    if (tc::elected()) tc::mma_commit(&s.done[w]);
    __syncwarp();
    int never = 0;
    tc::bar_wait(&s.done[w], 0, &never, tc::kWaitClocks);
    __syncwarp();
}

// Product warp: blocks w, w + W, ... of `count`, each four steps of 32 along K into
// N columns of the tensor memory, its PARTS parts in turn.  The whole warp takes
// the waits and one elected lane issues, which keeps the descriptors in uniform
// registers; two waits, four products and two commits took a warp about 900 clocks,
// so two warps alternate (W = 2) where there are registers for them.  base: shared
// address of the first stage, its two operand tiles kRowTile apart.  False: it gave up,
// and its products have ended; else they have when the epilogue has read them.
template <int N, int W, int PARTS, int STAGES, int STAGE_BYTES>
__device__ __forceinline__ bool issue_blocks(Sync &s, int w, int64_t count, uint32_t tmem, uint32_t base, int64_t limit) {
    // A wait knows its phase from the one before by parity alone, so it may only begin when the phase two
    // before has ended.  Copies land in any order: with the stages even each warp has its own, and waits
    // for every use of them.  Parts are released in order, so the other warp's are no trouble; free_ first,
    // so that a block's stage is asked about only when the blocks before it are.
    static_assert(STAGES % W == 0, "two product warps must not share a stage");
    Ring<STAGES> at;
    Ring<PARTS> part;
    int64_t it = w;
    bool ok = true;
    if (w) at.next(), part.next();
    for (; it < count; it += W) {
        ok = tc::bar_wait(&s.free_[part.stage], part.parity ^ 1, &s.abort, limit) &&
             tc::bar_wait(&s.full[at.stage], at.parity, &s.abort, limit);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        tc::fence_after();
        if (tc::elected()) {
            const uint32_t a = base + at.stage * STAGE_BYTES, b = a + kRowTile;
#pragma unroll
            for (int k = 0; k < kBlock / 32; ++k)
                tc::mma_e4m3(tmem + part.stage * N, tc::operand(a + 32 * k), tc::operand(b + 32 * k), tc::e4m3_product(N), k > 0);
            tc::mma_commit(&s.ready[part.stage]);
            tc::mma_commit(&s.empty[at.stage]);
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < W; ++i) at.next(), part.next();
    }
    if (!ok) end_products(s, w);
    return ok;
}

// ---------------------------------------------------------------------------
// many rows
// ---------------------------------------------------------------------------
// A third warpgroup (copy warp, two product warps and an idle one) hands registers to the two of the epilogue.
constexpr int kTileThreads = 384, kEpilogueRegisters = 216, kIssueRegisters = 56;  // 2 x 216 + 56 <= 3 x 168
constexpr int kGroupRows = 8;  // row tiles that share a sweep over the columns (operands stay in L2)

template <int TN>
struct TileShape {
    static constexpr int kStage = kRowTile + TN * kBlock;
    static constexpr int kStaging = kEpilogueWarps * 32 * 16 * 4;
    static constexpr int kRoom = (226 * 1024 - kStaging - 1024 - int(sizeof(Sync))) / kStage;
    static constexpr int kStages = kRoom > 8 ? 8 : kRoom & ~1;  // even, for the two product warps
    static constexpr int kBytes = kStages * kStage + kStaging + 1024 + int(sizeof(Sync));
    static constexpr int kParts = 512 / TN < kMostParts ? 512 / TN : kMostParts;
    static constexpr int kColumns = kParts * TN <= 256 ? 256 : 512;
};

// Tile `i` of the sweep: groups of kGroupRows row tiles, rows fastest within a group.
__device__ __forceinline__ int2 tile_at(int64_t i, int row_tiles, int column_tiles) {
    const int64_t group = i / (int64_t(kGroupRows) * column_tiles);
    const int first = int(group) * kGroupRows, rows = min(kGroupRows, row_tiles - first);
    const int64_t in = i - group * kGroupRows * column_tiles;
    return make_int2(first + int(in % rows), int(in / rows));
}

// Four consecutive values of a row of out or residual: one access where `wide`, else the first n singly.
template <class T>
struct Four {
    alignas(4 * sizeof(T)) T v[4];
    __device__ __forceinline__ void load(const T *p, bool wide, int n) {
        if (wide) {
            if (sizeof(T) == 2) *reinterpret_cast<uint2 *>(v) = *reinterpret_cast<const uint2 *>(p);
            else *reinterpret_cast<uint4 *>(v) = *reinterpret_cast<const uint4 *>(p);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = i < n ? p[i] : from_float<T>(0.f);
        }
    }
    __device__ __forceinline__ void store(T *p, bool wide, int n) const {
        if (wide) {
            if (sizeof(T) == 2) *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(v);
            else *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(v);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < n) p[i] = v[i];
        }
    }
};

template <class T, int TN>
__global__ void __launch_bounds__(kTileThreads, 1)
    tile_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap, sq_matmul_args a,
                bool wide) {
    using S = TileShape<TN>;
    extern __shared__ unsigned char raw[];
    unsigned char *base = raw + ((1024u - (tc::smem_u32(raw) & 1023u)) & 1023u);
    float *staging = reinterpret_cast<float *>(base + S::kStages * S::kStage);
    Sync &s = *reinterpret_cast<Sync *>(staging + S::kStaging / 4);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int blocks = (a.hidden + kBlock - 1) / kBlock;
    const int row_tiles = (a.rows + 127) / 128, column_tiles = (a.width + TN - 1) / TN;
    const int64_t tiles = int64_t(row_tiles) * column_tiles, first = blockIdx.x, step = gridDim.x;
    set_up(s, S::kStages, S::kColumns, warp);
    const uint32_t tmem = s.tmem;
    bool issued = false;

    if (warp >= kEpilogueWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kIssueRegisters));
        if (warp == kEpilogueWarps) {  // copies
            if (lane == 0) {
                Ring<S::kStages> at;
                int64_t count = 0;
                bool ok = true;
                for (int64_t i = first; i < tiles && ok; i += step) {
                    const int2 tile = tile_at(i, row_tiles, column_tiles);
                    const int x_row = tile.x * 128, w_row = tile.y * TN;
                    for (int g = 0; g < blocks; ++g, ++count, at.next()) {
                        if (!(ok = tc::bar_wait(&s.empty[at.stage], at.parity ^ 1, &s.abort, a.wait_clocks))) break;
                        unsigned char *to = base + at.stage * S::kStage;
                        tc::bar_expect(&s.full[at.stage], S::kStage);
                        tc::tma_load(to, &xmap, g * kBlock, x_row, &s.full[at.stage]);
                        tc::tma_load(to + kRowTile, &wmap, g * kBlock, w_row, &s.full[at.stage]);
                    }
                }
                drain_copies(s, at, count);
            }
            __syncwarp();
        } else if (warp < kEpilogueWarps + 3) {  // products
            const int64_t mine = first < tiles ? (tiles - first + step - 1) / step : 0;
            issued = issue_blocks<TN, 2, S::kParts, S::kStages, S::kStage>(s, warp - kEpilogueWarps - 1, mine * blocks, tmem, tc::smem_u32(base),
                                                                       a.wait_clocks);
        }
    } else {  // scales and sums: warp w holds lanes 32 (w % 4) .. + 31, half q = w / 4 of the columns
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kEpilogueRegisters));
        constexpr int C = TN / 2, CHUNKS = C / 16;
        const int q = warp >> 2;  // the half of the columns
        const uint32_t mine = tmem + (uint32_t(32 * (warp & 3)) << 16) + q * C;
        float *stage = staging + warp * 32 * 16;
        // Scales of kScaleGroup blocks from g on, loaded that many blocks before their use (a load's way
        // from L2 is longer than a block): the lane's row of x, and the two 128-row blocks of w that the
        // C <= 128 columns can meet.
        const int last = (a.width - 1) / kBlock;
        const float *sx = nullptr, *sw0 = nullptr, *sw1 = nullptr;
        float next_x[kScaleGroup], next_0[kScaleGroup], next_1[kScaleGroup];
        auto aim = [&](int64_t i) {
            const int2 at = tile_at(i, row_tiles, column_tiles);
            const int n0 = at.y * TN + q * C;
            sx = a.x_scale + int64_t(min(at.x * 128 + 32 * (warp & 3) + lane, a.rows - 1)) * blocks;
            sw0 = a.w_scale + int64_t(min(n0 / kBlock, last)) * blocks;
            sw1 = a.w_scale + int64_t(min((n0 + C - 1) / kBlock, last)) * blocks;
        };
        auto fetch_scales = [&](int g) {
#pragma unroll
            for (int q = 0; q < kScaleGroup; ++q) {
                const int at = min(g + q, blocks - 1);
                next_x[q] = sx[at], next_0[q] = sw0[at], next_1[q] = sw1[at];
            }
        };
        if (first < tiles) {
            aim(first);
            fetch_scales(0);
        }
        Ring<S::kParts> part;
        bool ok = true;
        int64_t i = first;
        for (; i < tiles; i += step) {
            const int2 at = tile_at(i, row_tiles, column_tiles);
            const int m0 = at.x * 128 + 32 * (warp & 3), n0 = at.y * TN + q * C;
            const int cross = (kBlock - n0 % kBlock) / 16;  // first chunk of the second block of w
            float acc[C];
#pragma unroll
            for (int j = 0; j < C; ++j) acc[j] = 0.f;
            float s0[kScaleGroup], s1[kScaleGroup];
            for (int g = 0; g < blocks; ++g, part.next()) {
                if (g % kScaleGroup == 0) {
#pragma unroll
                    for (int q = 0; q < kScaleGroup; ++q) s0[q] = next_x[q] * next_0[q], s1[q] = next_x[q] * next_1[q];
                    fetch_scales(g + kScaleGroup);
                }
                const float f0 = s0[0], f1 = s1[0];
#pragma unroll
                for (int q = 0; q + 1 < kScaleGroup; ++q) s0[q] = s0[q + 1], s1[q] = s1[q + 1];
                ok = __all_sync(0xffffffffu, tc::bar_wait(&s.ready[part.stage], part.parity, &s.abort, a.wait_clocks));
                if (!ok) break;
                tc::fence_after();
                const uint32_t from = mine + part.stage * TN;
                // The next 16 columns are on their way while 16 are added; the part is free once all are in registers.
                uint32_t r[2][16];
                tc::tmem_load(from, r[0]);
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) {
                    tc::tmem_wait(r[c & 1]);
                    if (c + 1 < CHUNKS) {
                        tc::tmem_load(from + 16 * (c + 1), r[(c + 1) & 1]);
                    } else {
                        tc::fence_before();
                        __syncwarp();
                        if (lane == 0) tc::bar_arrive(&s.free_[part.stage]);
                    }
                    const float f = c < cross ? f0 : f1;
#pragma unroll
                    for (int j = 0; j < 16; ++j) acc[16 * c + j] = fmaf(__uint_as_float(r[c & 1][j]), f, acc[16 * c + j]);
                }
            }
            if (!ok) break;
            if (i + step < tiles) {
                aim(i + step);
                fetch_scales(0);
            }
            // Out through shared memory, 16 columns at a time, the residual's next 16 columns on their way
            // meanwhile: a row's 16 values leave by four lanes (four rows of eight per access), or singly
            // where rows are not aligned for that (two rows per access, every value in a register of its
            // own: packed on arrival, as fours would be, each load was waited for, 4096 x 8255 x 5120 with
            // residual in 336 us for 232).  16-byte pieces of row r are rotated by r / 2 so that neither side
            // meets bank conflicts.
            auto put = [&](auto four) {
                constexpr bool kFour = decltype(four)::value;
                using Value = std::conditional_t<kFour, Four<T>, T>;
                constexpr int kEach = kFour ? 4 : 1, kAccesses = 16 / kEach, kLanes = 16 / kEach;
                const int r0 = lane / kLanes, c0 = lane % kLanes * kEach;  // within the rows of an access
                constexpr int kRows = 32 / kLanes;
                const int rows = a.rows - m0 - r0, columns = a.width - n0 - c0;  // that exist from the lane's first on
                const int64_t out_step = int64_t(kRows) * a.width, residual_step = int64_t(kRows) * a.residual_stride;
                const T *residual = a.residual ? static_cast<const T *>(a.residual) + int64_t(m0 + r0) * a.residual_stride + n0 + c0 : nullptr;
                T *out = static_cast<T *>(a.out) + int64_t(m0 + r0) * a.width + n0 + c0;
                Value old[kAccesses];
                auto fetch = [&](int c) {
                    if (!residual || 16 * c >= columns) return;
                    const T *from = residual + 16 * c;
#pragma unroll
                    for (int i = 0; i < kAccesses; ++i, from += residual_step)
                        if (i * kRows < rows) old[i] = *reinterpret_cast<const Value *>(from);
                };
                if (kFour) fetch(0);
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) {
                    if (!kFour) fetch(c);
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float *v = acc + 16 * c + 4 * j;
                        *reinterpret_cast<float4 *>(stage + lane * 16 + ((j + (lane >> 1)) & 3) * 4) = make_float4(v[0], v[1], v[2], v[3]);
                    }
                    __syncwarp();
                    Value add[kAccesses];
#pragma unroll
                    for (int i = 0; i < kAccesses; ++i) add[i] = old[i];
                    if (kFour && c + 1 < CHUNKS) fetch(c + 1);
                    T *to = out + 16 * c;
#pragma unroll
                    for (int i = 0; i < kAccesses; ++i, to += out_step) {
                        const int row = i * kRows + r0;
                        const float *from = stage + row * 16 + (((c0 >> 2) + (row >> 1)) & 3) * 4 + (c0 & 3);
                        Value y;
                        if constexpr (kFour) {
                            const float4 v = *reinterpret_cast<const float4 *>(from);
                            const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                            for (int j = 0; j < 4; ++j) y.v[j] = from_float<T>(residual ? x[j] + to_float(add[i].v[j]) : x[j]);
                        } else {
                            y = from_float<T>(residual ? *from + to_float(add[i]) : *from);
                        }
                        if (i * kRows < rows && 16 * c < columns) *reinterpret_cast<Value *>(to) = y;
                    }
                }
            };
            if (wide) put(std::true_type());
            else put(std::false_type());
        }
        for (; i < tiles; i += step) {  // given up
            const int2 at = tile_at(i, row_tiles, column_tiles);
            const int m0 = at.x * 128 + 32 * (warp & 3), n0 = at.y * TN + q * C;
            for (int m = m0; m < min(m0 + 32, a.rows); ++m)
                for (int n = n0 + lane; n < min(n0 + C, a.width); n += 32)
                    static_cast<T *>(a.out)[int64_t(m) * a.width + n] = from_float<T>(NAN);
        }
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    if (s.abort) {  // by all or none
        if (threadIdx.x == 0) flag(a.status, SQ_STATUS_TIMEOUT);
        if (issued) end_products(s, warp - kEpilogueWarps - 1);
        __syncthreads();
    }
    if (warp == kEpilogueWarps + 1) tc::tmem_free(tmem, S::kColumns);
}

// ---------------------------------------------------------------------------
// few rows
// ---------------------------------------------------------------------------
template <int TM>
struct SplitShape {
    static constexpr int kStage = kRowTile + TM * kBlock;
    static constexpr int kProductWarps = TM <= 32 ? 2 : 1;  // more rows have no registers for a second
    static constexpr int kStages = 112640 / kStage / kProductWarps * kProductWarps;  // 6, 4, 4, 3: two CTAs an SM
    static constexpr int kScales = 2 * kScaleGroup * TM * 4;  // of two groups of blocks
    static constexpr int kBytes = kStages * kStage + kScales + 1024 + int(sizeof(Sync));
    static constexpr int kParts = 256 / TM < kMostParts ? 256 / TM : kMostParts;  // 256 columns: two CTAs an SM
    static constexpr int kColumns = kParts * TM;
    static constexpr int kThreads = 32 * (kEpilogueWarps + 1 + kProductWarps);
};

template <class T, int TM>
__global__ void __launch_bounds__(SplitShape<TM>::kThreads, 2)
    split_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap, sq_matmul_args a,
                 bool wide) {
    using S = SplitShape<TM>;
    namespace cg = cooperative_groups;
    extern __shared__ unsigned char raw[];
    unsigned char *base = raw + ((1024u - (tc::smem_u32(raw) & 1023u)) & 1023u);
    float *ring = reinterpret_cast<float *>(base + S::kStages * S::kStage);  // [2][kScaleGroup][TM]
    Sync &s = *reinterpret_cast<Sync *>(ring + S::kScales / 4);
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = int(cluster.num_blocks()), rank = int(cluster.block_rank());
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int blocks = (a.hidden + kBlock - 1) / kBlock;
    const int g0 = int(int64_t(blocks) * rank / ranks), g1 = int(int64_t(blocks) * (rank + 1) / ranks);
    const int n0 = int(blockIdx.x) / ranks * 128;  // and all rows of x: TM or fewer
    set_up(s, S::kStages, S::kColumns, warp);
    const uint32_t tmem = s.tmem;
    float *sums = reinterpret_cast<float *>(base);  // [TM][128], once the operands are consumed
    bool issued = false;

    if (warp == kEpilogueWarps) {
        if (lane == 0) {
            Ring<S::kStages> at;
            bool ok = true;
            int g = g0;
            for (; g < g1; ++g, at.next()) {
                if (!(ok = tc::bar_wait(&s.empty[at.stage], at.parity ^ 1, &s.abort, a.wait_clocks))) break;
                unsigned char *to = base + at.stage * S::kStage;
                tc::bar_expect(&s.full[at.stage], S::kStage);
                tc::tma_load(to, &wmap, g * kBlock, n0, &s.full[at.stage]);
                tc::tma_load(to + kRowTile, &xmap, g * kBlock, 0, &s.full[at.stage]);
            }
            drain_copies(s, at, g - g0);
        }
        __syncwarp();
    } else if (warp > kEpilogueWarps) {
        issued = issue_blocks<TM, S::kProductWarps, S::kParts, S::kStages, S::kStage>(s, warp - kEpilogueWarps - 1, g1 - g0, tmem, tc::smem_u32(base),
                                                                                 a.wait_clocks);
    } else {
        constexpr int C = TM / 2, W = C < 16 ? C : 16, CHUNKS = C / W;
        const int tid = threadIdx.x, half = warp >> 2;
        const uint32_t mine = tmem + (uint32_t(32 * (warp & 3)) << 16) + half * C;
        // Scales of kScaleGroup blocks, a column of a block each: loaded while the group before is worked on.
        constexpr int EACH = (kScaleGroup * TM + 32 * kEpilogueWarps - 1) / (32 * kEpilogueWarps);
        const float *sw = a.w_scale + int64_t(n0 / kBlock) * blocks;
        float next[EACH];
        auto fetch_scales = [&](int g) {
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                const int i = e * 32 * kEpilogueWarps + tid, at = min(g + i / TM, blocks - 1);
                if (i < kScaleGroup * TM) next[e] = a.x_scale[int64_t(min(i % TM, a.rows - 1)) * blocks + at] * sw[at];
            }
        };
        fetch_scales(g0);
        float acc[C];
#pragma unroll
        for (int j = 0; j < C; ++j) acc[j] = 0.f;
        Ring<S::kParts> part;
        for (int it = 0; it < g1 - g0; ++it, part.next()) {
            const float *group = ring + (it / kScaleGroup & 1) * kScaleGroup * TM;
            if (it % kScaleGroup == 0) {
#pragma unroll
                for (int e = 0; e < EACH; ++e) {
                    const int i = e * 32 * kEpilogueWarps + tid;
                    if (i < kScaleGroup * TM) const_cast<float *>(group)[i] = next[e];
                }
                fetch_scales(g0 + it + kScaleGroup);
                // The group's scales are there for all, and all are done with those of two groups ago.
                asm volatile("bar.sync 1, %0;\n" ::"n"(32 * kEpilogueWarps) : "memory");
            }
            tc::bar_wait(&s.ready[part.stage], part.parity, &s.abort, a.wait_clocks);  // giving up: the sums are not used
            __syncwarp();
            tc::fence_after();
            const uint32_t from = mine + part.stage * TM;
            const float *f = group + it % kScaleGroup * TM + half * C;
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) {
                uint32_t r[W];
                tc::tmem_load(from + W * c, r);
                tc::tmem_wait(r);
#pragma unroll
                for (int j = 0; j < W; j += 4) {
                    const float4 v = *reinterpret_cast<const float4 *>(f + W * c + j);
                    float *sum = acc + W * c + j;
                    sum[0] = fmaf(__uint_as_float(r[j]), v.x, sum[0]);
                    sum[1] = fmaf(__uint_as_float(r[j + 1]), v.y, sum[1]);
                    sum[2] = fmaf(__uint_as_float(r[j + 2]), v.z, sum[2]);
                    sum[3] = fmaf(__uint_as_float(r[j + 3]), v.w, sum[3]);
                }
            }
            tc::fence_before();
            __syncwarp();
            if (lane == 0) tc::bar_arrive(&s.free_[part.stage]);
        }
        // Every product has been read from tensor memory, hence every operand by the tensor cores.
        if (!s.abort) {
#pragma unroll
            for (int j = 0; j < C; ++j) sums[(half * C + j) * 128 + 32 * (warp & 3) + lane] = acc[j];
        }
    }
    tc::fence_before();
    cluster.sync();
    tc::fence_after();
    if (s.abort) {  // by all or none of the CTA
        if (threadIdx.x == 0) flag(a.status, SQ_STATUS_TIMEOUT);
        if (issued) end_products(s, warp - kEpilogueWarps - 1);
        __syncthreads();
    }
    if (warp == kEpilogueWarps + 1) tc::tmem_free(tmem, S::kColumns);
    // The sums of the ranks (NaN where one gave up), in their order; each rank finishes its share of the rows of x, four columns a thread.
    const int share = TM * rank / ranks, count = TM * (rank + 1) / ranks - share;
#pragma unroll 4
    for (int i = threadIdx.x; i < count * 32; i += S::kThreads) {
        const int m = share + i / 32, n = n0 + i % 32 * 4;
        if (m >= a.rows || n >= a.width) continue;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        int gone = 0;
        for (int q = 0; q < ranks; ++q) {
            const float4 part = reinterpret_cast<const float4 *>(cluster.map_shared_rank(sums, q))[share * 32 + i];
            gone |= *cluster.map_shared_rank(&s.abort, q);
            v.x += part.x, v.y += part.y, v.z += part.z, v.w += part.w;
        }
        if (gone) v = make_float4(NAN, NAN, NAN, NAN);
        const float x[4] = {v.x, v.y, v.z, v.w};
        Four<T> old, y;
        if (a.residual) old.load(static_cast<const T *>(a.residual) + int64_t(m) * a.residual_stride + n, wide, a.width - n);
#pragma unroll
        for (int j = 0; j < 4; ++j) y.v[j] = from_float<T>(a.residual ? x[j] + to_float(old.v[j]) : x[j]);
        y.store(static_cast<T *>(a.out) + int64_t(m) * a.width + n, wide, a.width - n);
    }
    cluster.sync();
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
PFN_cuTensorMapEncodeTiled_v12000 encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
        else
            (void)cudaGetLastError();
    });
    return fn;
}

// Bytes [rows, hidden] in boxes of 128 columns and `box` rows, zeros outside.
bool byte_map(CUtensorMap *map, const void *p, int hidden, int rows, int64_t stride, int box) {
    const cuuint64_t size[2] = {cuuint64_t(hidden), cuuint64_t(rows)}, strides[1] = {cuuint64_t(stride)};
    const cuuint32_t boxes[2] = {cuuint32_t(kBlock), cuuint32_t(box)}, steps[2] = {1, 1};
    return encoder() && encoder()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(p), size, strides, boxes, steps,
                                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class T, int TN>
int32_t launch_tile(const sq_matmul_args &a, bool wide, int sms, cudaStream_t s) {
    using S = TileShape<TN>;
    CUtensorMap x, w;
    if (!byte_map(&x, a.x, a.hidden, a.rows, a.x_stride, 128) || !byte_map(&w, a.w, a.hidden, a.width, a.w_stride, TN))
        return SQ_ERR_CUDA;
    if (cudaFuncSetAttribute(tile_kernel<T, TN>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes) != cudaSuccess)
        return SQ_ERR_CUDA;
    const int64_t tiles = int64_t((a.rows + 127) / 128) * ((a.width + TN - 1) / TN);
    tile_kernel<T, TN><<<unsigned(tiles < sms ? tiles : sms), kTileThreads, S::kBytes, s>>>(x, w, a, wide);
    return cudaGetLastError() == cudaSuccess ? SQ_OK : SQ_ERR_CUDA;
}

template <class T, int TM>
int32_t launch_split(const sq_matmul_args &a, bool wide, int sms, cudaStream_t s) {
    using S = SplitShape<TM>;
    CUtensorMap x, w;
    if (!byte_map(&x, a.x, a.hidden, a.rows, a.x_stride, TM) || !byte_map(&w, a.w, a.hidden, a.width, a.w_stride, 128))
        return SQ_ERR_CUDA;
    if (cudaFuncSetAttribute(split_kernel<T, TM>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes) != cudaSuccess)
        return SQ_ERR_CUDA;
    const int columns = (a.width + 127) / 128, blocks = (a.hidden + kBlock - 1) / kBlock;
    // K is split while two CTAs an SM are not in use and each keeps two blocks.
    int split = 8;
    while (split > 1 && (int64_t(columns) * split > 2 * sms || blocks < 2 * split)) split /= 2;
    cudaLaunchConfig_t c{};
    c.gridDim = dim3(unsigned(columns * split));
    c.blockDim = dim3(unsigned(S::kThreads));
    c.dynamicSmemBytes = S::kBytes;
    c.stream = s;
    cudaLaunchAttribute cluster;
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = unsigned(split);
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    c.attrs = &cluster;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, split_kernel<T, TM>, x, w, a, wide) == cudaSuccess ? SQ_OK : SQ_ERR_CUDA;
}

template <class T>
int32_t launch_matmul(const sq_matmul_args &a, int sms, cudaStream_t s) {
    const int64_t size = sizeof(T);
    auto rows4 = [&](const void *p, int64_t stride) { return reinterpret_cast<uintptr_t>(p) % (4 * size) == 0 && stride % 4 == 0; };
    const bool wide = a.width % 4 == 0 && rows4(a.out, a.width) && (!a.residual || rows4(a.residual, a.residual_stride));
    if (a.rows <= 16) return launch_split<T, 16>(a, wide, sms, s);
    if (a.rows <= 32) return launch_split<T, 32>(a, wide, sms, s);
    if (a.rows <= 64) return launch_split<T, 64>(a, wide, sms, s);
    if (a.rows <= 128) return launch_split<T, 128>(a, wide, sms, s);
    // The tile whose waves take least; ns of a block of 128 x TN with every SM at it, measured (start and
    // end of a call, about 6 us, are the same for all).
    constexpr int kTile[5] = {256, 192, 160, 128, 64}, kTime[5] = {590, 470, 410, 330, 270};
    int best = 0;
    int64_t least = INT64_MAX;
    for (int i = 0; i < 5; ++i) {
        const int64_t tiles = int64_t((a.rows + 127) / 128) * ((a.width + kTile[i] - 1) / kTile[i]);
        const int64_t time = (tiles + sms - 1) / sms * kTime[i];
        if (time < least) least = time, best = kTile[i];
    }
    switch (best) {
        case 256: return launch_tile<T, 256>(a, wide, sms, s);
        case 192: return launch_tile<T, 192>(a, wide, sms, s);
        case 160: return launch_tile<T, 160>(a, wide, sms, s);
        case 128: return launch_tile<T, 128>(a, wide, sms, s);
        default: return launch_tile<T, 64>(a, wide, sms, s);
    }
}

}  // namespace
}  // namespace sq

extern "C" int32_t sq_matmul_fp8(const sq_matmul_args *args, sq_stream_t stream) {
    if (!args) return SQ_ERR_ARGUMENT;
    sq_matmul_args a = *args;
    if (a.rows < 0 || a.width < 1 || a.hidden < 1) return SQ_ERR_ARGUMENT;
    if (a.dtype < SQ_F32 || a.dtype > SQ_F16) return SQ_ERR_ARGUMENT;
    if (a.hidden % 16 || a.rows > sq::kMostRows || a.width > sq::kMostRows || a.hidden > sq::kMostRows) return SQ_ERR_UNSUPPORTED;
    if (a.rows == 0) return SQ_OK;
    if (!a.x || !a.x_scale || !a.w || !a.w_scale || !a.out) return SQ_ERR_ARGUMENT;
    if (!sq::aligned16(a.x) || !sq::aligned16(a.w) || a.x_stride < a.hidden || a.w_stride < a.hidden || a.x_stride % 16 ||
        a.w_stride % 16 || a.residual_stride < 0)
        return SQ_ERR_SHAPE;
    if (a.wait_clocks == 0) a.wait_clocks = sq::tc::kWaitClocks;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const int sms = sq::sms_of(s);
    if (sms < 1) return SQ_ERR_CUDA;
    return a.dtype == SQ_F32    ? sq::launch_matmul<float>(a, sms, s)
           : a.dtype == SQ_BF16 ? sq::launch_matmul<__nv_bfloat16>(a, sms, s)
                                : sq::launch_matmul<__half>(a, sms, s);
}
