// Product of e4m3 matrices with an fp32 scale per block of 128:
//
//   out[m, n] = residual[m, n] + sum_g sx[m, g] sw[n / 128, g] sum_{k in block g} x[m, k] w[n, k]
//
// x [M, K] has a scale per row and 128 columns, w [N, K] one per 128 rows and
// 128 columns.  The tensor cores form each 128-deep block product exactly as
// fp32 sums in tensor memory; the epilogue warps scale it and add it to fp32
// registers while the next block's product runs into the other half of the
// tensor memory.  One rounding, of the finished sum with the residual.
//
// Many rows (tile_kernel): tensor memory lanes are rows of x, columns are rows
// of w, so a thread's scale is one number a block.  Persistent CTAs, one per SM.
// Few rows (split_kernel): the weights' bytes bound the call.  Lanes are 128
// rows of w (one scale a block), columns the rows of x; the CTAs of a cluster
// split K and add their sums in rank order through distributed shared memory.
//
// Operands arrive by TMA (128-byte swizzle; zeros past K, M and N), one warp
// issues the copies, one the products; every wait is bounded.
#include <cooperative_groups.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "sq_tc.cuh"
#include "sq_vec.cuh"

namespace sq {
int sms_of(cudaStream_t stream);  // sq_fast.cu
namespace {

constexpr int kBlock = 128;                // depth of a scale block and of a pipeline stage
constexpr int kEpilogueWarps = 8;
constexpr int kCtaThreads = 32 * (kEpilogueWarps + 2);  // + copy warp, product warp
constexpr int kRowTile = 128 * kBlock;     // bytes of a 128-row operand tile

struct Sync {
    uint64_t full[8], empty[8];  // operand stages
    uint64_t ready[2], free_[2]; // halves of the tensor memory
    uint32_t tmem;
    int abort;
};

// A CTA that gives up leaves once what it issued has ended (again with a limit):
// the copies of its last stages, the products of its last two blocks.
__device__ __forceinline__ void drain_copies(Sync &s, int stages, int64_t count) {
    int never = 0;
    for (int64_t i = max(int64_t(0), count - stages); i < count; ++i)
        tc::bar_wait(&s.full[i % stages], uint32_t(i / stages) & 1, &never);
}
__device__ __forceinline__ void drain_products(Sync &s, int64_t count) {
    int never = 0;
    for (int64_t i = max(int64_t(0), count - 2); i < count; ++i) tc::bar_wait(&s.ready[i & 1], uint32_t(i >> 1) & 1, &never);
}

__device__ __forceinline__ void set_up(Sync &s, int stages, uint32_t columns, int warp) {
    if (threadIdx.x == 0) {
        for (int i = 0; i < stages; ++i) {
            tc::bar_init(&s.full[i], 1);
            tc::bar_init(&s.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            tc::bar_init(&s.ready[i], 1);
            tc::bar_init(&s.free_[i], kEpilogueWarps);
        }
        s.abort = 0;
        tc::bar_init_fence();
    }
    if (warp == kEpilogueWarps + 1) tc::tmem_alloc(&s.tmem, columns);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
}

// The product warp's part of one block: 4 steps of 32 along K into buffer `half`.
template <int N>
__device__ __forceinline__ bool issue_block(Sync &s, int stages, int64_t it, uint32_t a, uint32_t b, uint32_t tmem) {
    const int stage = int(it % stages), half = int(it & 1);
    if (!tc::bar_wait(&s.full[stage], uint32_t(it / stages) & 1, &s.abort)) return false;
    if (!tc::bar_wait(&s.free_[half], (uint32_t(it >> 1) & 1) ^ 1, &s.abort)) return false;
    tc::fence_after();
#pragma unroll
    for (int k = 0; k < kBlock / 32; ++k)
        tc::mma_e4m3(tmem + half * N, tc::operand(a + 32 * k), tc::operand(b + 32 * k), tc::e4m3_product(N), k > 0);
    tc::mma_commit(&s.empty[stage]);
    tc::mma_commit(&s.ready[half]);
    return true;
}

// ---------------------------------------------------------------------------
// many rows
// ---------------------------------------------------------------------------
constexpr int kGroupRows = 16;  // row tiles that share a sweep over the columns (operands stay in L2)

template <int TN>
struct TileShape {
    static constexpr int kStage = kRowTile + TN * kBlock;
    static constexpr int kStaging = kEpilogueWarps * 32 * 16 * 4;
    static constexpr int kStages = (226 * 1024 - kStaging - 1024 - int(sizeof(Sync))) / kStage > 8
                                       ? 8 : (226 * 1024 - kStaging - 1024 - int(sizeof(Sync))) / kStage;
    static constexpr int kBytes = kStages * kStage + kStaging + 1024 + int(sizeof(Sync));
    static constexpr int kColumns = 2 * TN <= 64 ? 64 : 2 * TN <= 128 ? 128 : 2 * TN <= 256 ? 256 : 512;
};

// Tile `i` of the sweep: groups of kGroupRows row tiles, rows fastest within a group.
__device__ __forceinline__ int2 tile_at(int64_t i, int row_tiles, int column_tiles) {
    const int64_t group = i / (int64_t(kGroupRows) * column_tiles);
    const int first = int(group) * kGroupRows, rows = min(kGroupRows, row_tiles - first);
    const int64_t in = i - group * kGroupRows * column_tiles;
    return make_int2(first + int(in % rows), int(in / rows));
}

template <class T, int TN>
__global__ void __launch_bounds__(kCtaThreads, 1)
    tile_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap, sq_matmul_args a,
                bool wide) {
    using S = TileShape<TN>;
    extern __shared__ unsigned char raw[];
    unsigned char *base = raw + ((1024u - (tc::smem_u32(raw) & 1023u)) & 1023u);
    float *staging = reinterpret_cast<float *>(base + S::kStages * S::kStage);
    Sync &s = *reinterpret_cast<Sync *>(base + S::kStages * S::kStage + S::kStaging);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int blocks = (a.hidden + kBlock - 1) / kBlock;
    const int row_tiles = (a.rows + 127) / 128, column_tiles = (a.width + TN - 1) / TN;
    const int64_t tiles = int64_t(row_tiles) * column_tiles;
    set_up(s, S::kStages, S::kColumns, warp);
    const uint32_t tmem = s.tmem;

    if (warp == kEpilogueWarps) {  // copies
        if (lane == 0) {
            int64_t it = 0;
            bool ok = true;
            for (int64_t i = blockIdx.x; i < tiles && ok; i += gridDim.x) {
                const int2 at = tile_at(i, row_tiles, column_tiles);
                for (int g = 0; g < blocks; ++g, ++it) {
                    const int stage = int(it % S::kStages);
                    if (!(ok = tc::bar_wait(&s.empty[stage], (uint32_t(it / S::kStages) & 1) ^ 1, &s.abort))) break;
                    unsigned char *to = base + stage * S::kStage;
                    tc::bar_expect(&s.full[stage], S::kStage);
                    tc::tma_load(to, &xmap, g * kBlock, at.x * 128, &s.full[stage]);
                    tc::tma_load(to + kRowTile, &wmap, g * kBlock, at.y * TN, &s.full[stage]);
                }
            }
            if (!ok) drain_copies(s, S::kStages, it);
        }
        __syncwarp();
    } else if (warp == kEpilogueWarps + 1) {  // products
        if (lane == 0) {
            int64_t it = 0;
            bool ok = true;
            for (int64_t i = blockIdx.x; i < tiles && ok; i += gridDim.x)
                for (int g = 0; g < blocks; ++g, ++it) {
                    const uint32_t to = tc::smem_u32(base + int(it % S::kStages) * S::kStage);
                    if (!(ok = issue_block<TN>(s, S::kStages, it, to, to + kRowTile, tmem))) break;
                }
            if (!ok) drain_products(s, it);
        }
        __syncwarp();
    } else {  // scales and sums: warp w holds lanes 32 (w % 4) .. + 31, half w / 4 of the columns
        constexpr int C = TN / 2, CHUNKS = C / 16;
        const uint32_t mine = tmem + (uint32_t(32 * (warp & 3)) << 16) + (warp >> 2) * C;
        float *stage = staging + warp * 32 * 16;
        int64_t it = 0;
        bool ok = true;
        for (int64_t i = blockIdx.x; i < tiles && ok; i += gridDim.x) {
            const int2 at = tile_at(i, row_tiles, column_tiles);
            const int m0 = at.x * 128 + 32 * (warp & 3), n0 = at.y * TN + (warp >> 2) * C;
            const float *sx = a.x_scale + int64_t(min(m0 + lane, a.rows - 1)) * blocks;
            // The C <= 128 columns cross at most one boundary of 128-row weight blocks.
            const int last = (a.width - 1) / kBlock;
            const float *sw0 = a.w_scale + int64_t(min(n0 / kBlock, last)) * blocks;
            const float *sw1 = a.w_scale + int64_t(min((n0 + C - 1) / kBlock, last)) * blocks;
            const int cross = (kBlock - n0 % kBlock) / 16;  // first chunk of the second block
            uint64_t acc[C / 2];
#pragma unroll
            for (int j = 0; j < C / 2; ++j) acc[j] = 0;
            float fx = sx[0], f0 = sw0[0], f1 = sw1[0];
            for (int g = 0; g < blocks; ++g, ++it) {
                const float s0 = fx * f0, s1 = fx * f1;
                if (g + 1 < blocks) fx = sx[g + 1], f0 = sw0[g + 1], f1 = sw1[g + 1];
                ok = __all_sync(0xffffffffu, tc::bar_wait(&s.ready[it & 1], uint32_t(it >> 1) & 1, &s.abort));
                if (!ok) break;
                tc::fence_after();
                const uint32_t from = mine + int(it & 1) * TN;
                uint32_t r[2][16];
                tc::tmem_load(from, r[0]);
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) {
                    tc::tmem_wait(r[c & 1]);
                    if (c + 1 < CHUNKS) tc::tmem_load(from + 16 * (c + 1), r[(c + 1) & 1]);
                    const float f = c < cross ? s0 : s1;
                    const uint64_t ff = tc::pair(f, f);
#pragma unroll
                    for (int j = 0; j < 8; ++j) tc::fma2(acc[8 * c + j], r[c & 1][2 * j], r[c & 1][2 * j + 1], ff);
                }
                tc::fence_before();
                __syncwarp();
                if (lane == 0) tc::bar_arrive(&s.free_[it & 1]);
            }
            if (!ok) break;
            // Out through shared memory, 16 columns at a time: a row's 16 values leave by four lanes.
            // 16-byte pieces of row r are rotated by r / 2 so that neither side meets bank conflicts.
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) {
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 lo = tc::unpair(acc[8 * c + 2 * j]), hi = tc::unpair(acc[8 * c + 2 * j + 1]);
                    *reinterpret_cast<float4 *>(stage + lane * 16 + ((j + (lane >> 1)) & 3) * 4) = make_float4(lo.x, lo.y, hi.x, hi.y);
                }
                __syncwarp();
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int row = q * 8 + (lane >> 2), m = m0 + row, n = n0 + 16 * c + 4 * (lane & 3);
                    const float4 v = *reinterpret_cast<const float4 *>(stage + row * 16 + (((lane & 3) + (row >> 1)) & 3) * 4);
                    float x[4] = {v.x, v.y, v.z, v.w};
                    if (m >= a.rows || n >= a.width) continue;
                    const T *res = a.residual ? static_cast<const T *>(a.residual) + int64_t(m) * a.residual_stride + n : nullptr;
                    T *out = static_cast<T *>(a.out) + int64_t(m) * a.width + n;
                    if (wide) {
                        T y[4];
                        if (res) {
                            T old[4];
                            if (sizeof(T) == 2) *reinterpret_cast<uint2 *>(old) = *reinterpret_cast<const uint2 *>(res);
                            else *reinterpret_cast<uint4 *>(old) = *reinterpret_cast<const uint4 *>(res);
#pragma unroll
                            for (int j = 0; j < 4; ++j) x[j] += to_float(old[j]);
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j) y[j] = from_float<T>(x[j]);
                        if (sizeof(T) == 2) *reinterpret_cast<uint2 *>(out) = *reinterpret_cast<const uint2 *>(y);
                        else *reinterpret_cast<uint4 *>(out) = *reinterpret_cast<const uint4 *>(y);
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (n + j < a.width) out[j] = from_float<T>(res ? x[j] + to_float(res[j]) : x[j]);
                    }
                }
            }
        }
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    if (s.abort && threadIdx.x == 0) flag(a.status, SQ_STATUS_TIMEOUT);
    if (warp == kEpilogueWarps + 1) tc::tmem_free(tmem, S::kColumns);
}

// ---------------------------------------------------------------------------
// few rows
// ---------------------------------------------------------------------------
template <int TM>
struct SplitShape {
    static constexpr int kStage = kRowTile + TM * kBlock;
    static constexpr int kStages = 98304 / kStage;  // 5, 4, 4, 3: two CTAs an SM
    static constexpr int kBytes = kStages * kStage + 2 * TM * 4 + 1024 + int(sizeof(Sync));
    static constexpr int kColumns = 2 * TM;
};

template <class T, int TM>
__global__ void __launch_bounds__(kCtaThreads, 2)
    split_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap, sq_matmul_args a) {
    using S = SplitShape<TM>;
    namespace cg = cooperative_groups;
    extern __shared__ unsigned char raw[];
    unsigned char *base = raw + ((1024u - (tc::smem_u32(raw) & 1023u)) & 1023u);
    float *factor = reinterpret_cast<float *>(base + S::kStages * S::kStage);  // [2][TM]
    Sync &s = *reinterpret_cast<Sync *>(factor + 2 * TM);
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = int(cluster.num_blocks()), rank = int(cluster.block_rank());
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int blocks = (a.hidden + kBlock - 1) / kBlock;
    const int g0 = int(int64_t(blocks) * rank / ranks), g1 = int(int64_t(blocks) * (rank + 1) / ranks);
    const int n0 = int(blockIdx.x) / ranks * 128, m0 = blockIdx.y * TM;
    set_up(s, S::kStages, S::kColumns, warp);
    const uint32_t tmem = s.tmem;
    float *sums = reinterpret_cast<float *>(base);  // [TM][128], once the operands are consumed

    if (warp == kEpilogueWarps) {
        if (lane == 0) {
            bool ok = true;
            int it = 0;
            for (; it < g1 - g0; ++it) {
                const int stage = it % S::kStages;
                if (!(ok = tc::bar_wait(&s.empty[stage], (uint32_t(it / S::kStages) & 1) ^ 1, &s.abort))) break;
                unsigned char *to = base + stage * S::kStage;
                tc::bar_expect(&s.full[stage], S::kStage);
                tc::tma_load(to, &wmap, (g0 + it) * kBlock, n0, &s.full[stage]);
                tc::tma_load(to + kRowTile, &xmap, (g0 + it) * kBlock, m0, &s.full[stage]);
            }
            if (!ok) drain_copies(s, S::kStages, it);
        }
        __syncwarp();
    } else if (warp == kEpilogueWarps + 1) {
        if (lane == 0) {
            bool ok = true;
            int it = 0;
            for (; it < g1 - g0; ++it) {
                const uint32_t to = tc::smem_u32(base + it % S::kStages * S::kStage);
                if (!(ok = issue_block<TM>(s, S::kStages, it, to, to + kRowTile, tmem))) break;
            }
            if (!ok) drain_products(s, it);
        }
        __syncwarp();
    } else {
        constexpr int C = TM / 2, W = C < 16 ? C : 16, CHUNKS = C / W;
        const int tid = threadIdx.x, half = warp >> 2;
        const uint32_t mine = tmem + (uint32_t(32 * (warp & 3)) << 16) + half * C;
        const float *sw = a.w_scale + int64_t(n0 / kBlock) * blocks;
        const float *sx = a.x_scale + int64_t(min(m0 + tid % TM, a.rows - 1)) * blocks;
        uint64_t acc[C / 2];
#pragma unroll
        for (int j = 0; j < C / 2; ++j) acc[j] = 0;
        float next = tid < TM && g0 < g1 ? sx[g0] * sw[g0] : 0.f;
        for (int it = 0; it < g1 - g0; ++it) {
            // Scales of the block's columns, one thread each; the barrier also says that every warp
            // has left the buffer of two blocks ago.
            if (tid < TM) {
                factor[(it & 1) * TM + tid] = next;
                if (g0 + it + 1 < g1) next = sx[g0 + it + 1] * sw[g0 + it + 1];
            }
            asm volatile("bar.sync 1, %0;\n" ::"n"(32 * kEpilogueWarps) : "memory");
            tc::bar_wait(&s.ready[it & 1], uint32_t(it >> 1) & 1, &s.abort);  // giving up: the sums are not used
            __syncwarp();
            tc::fence_after();
            const uint32_t from = mine + (it & 1) * TM;
            const float *f = factor + (it & 1) * TM + half * C;
            uint32_t r[2][W];
            tc::tmem_load(from, r[0]);
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) {
                tc::tmem_wait(r[c & 1]);
                if (c + 1 < CHUNKS) tc::tmem_load(from + W * (c + 1), r[(c + 1) & 1]);
#pragma unroll
                for (int j = 0; j < W / 4; ++j) {
                    const float4 v = *reinterpret_cast<const float4 *>(f + W * c + 4 * j);
                    tc::fma2(acc[W / 2 * c + 2 * j], r[c & 1][4 * j], r[c & 1][4 * j + 1], tc::pair(v.x, v.y));
                    tc::fma2(acc[W / 2 * c + 2 * j + 1], r[c & 1][4 * j + 2], r[c & 1][4 * j + 3], tc::pair(v.z, v.w));
                }
            }
            tc::fence_before();
            __syncwarp();
            if (lane == 0) tc::bar_arrive(&s.free_[it & 1]);
        }
        // Every product has been read from tensor memory, hence every operand by the tensor cores.
        if (!s.abort) {
#pragma unroll
            for (int j = 0; j < C / 2; ++j) {
                const float2 v = tc::unpair(acc[j]);
                sums[(half * C + 2 * j) * 128 + 32 * (warp & 3) + lane] = v.x;
                sums[(half * C + 2 * j + 1) * 128 + 32 * (warp & 3) + lane] = v.y;
            }
        }
    }
    tc::fence_before();
    cluster.sync();
    tc::fence_after();
    if (warp == kEpilogueWarps + 1) tc::tmem_free(tmem, S::kColumns);
    // The sums of the ranks, in their order; each rank finishes its share of the rows of x.
    const int first = TM * rank / ranks, count = TM * (rank + 1) / ranks - first;
    for (int i = threadIdx.x; i < count * 128; i += kCtaThreads) {
        const int m = m0 + first + i / 128, n = n0 + i % 128;
        if (m >= a.rows || n >= a.width) continue;
        float v = 0.f;
        for (int q = 0; q < ranks; ++q) v += cluster.map_shared_rank(sums, q)[first * 128 + i];
        if (a.residual) v += to_float(static_cast<const T *>(a.residual)[int64_t(m) * a.residual_stride + n]);
        static_cast<T *>(a.out)[int64_t(m) * a.width + n] = from_float<T>(v);
    }
    if (s.abort && threadIdx.x == 0) flag(a.status, SQ_STATUS_TIMEOUT);
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
    tile_kernel<T, TN><<<unsigned(tiles < sms ? tiles : sms), kCtaThreads, S::kBytes, s>>>(x, w, a, wide);
    return cudaGetLastError() == cudaSuccess ? SQ_OK : SQ_ERR_CUDA;
}

template <class T, int TM>
int32_t launch_split(const sq_matmul_args &a, int sms, cudaStream_t s) {
    using S = SplitShape<TM>;
    CUtensorMap x, w;
    if (!byte_map(&x, a.x, a.hidden, a.rows, a.x_stride, TM) || !byte_map(&w, a.w, a.hidden, a.width, a.w_stride, 128))
        return SQ_ERR_CUDA;
    if (cudaFuncSetAttribute(split_kernel<T, TM>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes) != cudaSuccess)
        return SQ_ERR_CUDA;
    const int columns = (a.width + 127) / 128, rows = (a.rows + TM - 1) / TM, blocks = (a.hidden + kBlock - 1) / kBlock;
    // K is split while two CTAs an SM are not in use and each keeps two blocks.
    int split = 8;
    while (split > 1 && (int64_t(columns) * rows * split > 2 * sms || blocks < 2 * split)) split /= 2;
    cudaLaunchConfig_t c{};
    c.gridDim = dim3(unsigned(columns * split), unsigned(rows));
    c.blockDim = dim3(kCtaThreads);
    c.dynamicSmemBytes = S::kBytes;
    c.stream = s;
    cudaLaunchAttribute cluster;
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = unsigned(split);
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    c.attrs = &cluster;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, split_kernel<T, TM>, x, w, a) == cudaSuccess ? SQ_OK : SQ_ERR_CUDA;
}

template <class T>
int32_t launch_matmul(const sq_matmul_args &a, int sms, cudaStream_t s) {
    const int64_t size = sizeof(T);
    auto rows4 = [&](const void *p, int64_t stride) { return reinterpret_cast<uintptr_t>(p) % (4 * size) == 0 && stride % 4 == 0; };
    const bool wide = a.width % 4 == 0 && rows4(a.out, a.width) && (!a.residual || rows4(a.residual, a.residual_stride));
    if (a.rows <= 16) return launch_split<T, 16>(a, sms, s);
    if (a.rows <= 32) return launch_split<T, 32>(a, sms, s);
    if (a.rows <= 64) return launch_split<T, 64>(a, sms, s);
    if (a.rows <= 128) return launch_split<T, 128>(a, sms, s);
    // The column tile whose waves of tiles cost least, a tile costing its operand bytes.
    int best = 256;
    int64_t least = INT64_MAX;
    for (int tn : {256, 192, 160, 128, 96, 64}) {
        const int64_t tiles = int64_t((a.rows + 127) / 128) * ((a.width + tn - 1) / tn), cost = (tiles + sms - 1) / sms * (128 + tn);
        if (cost < least) least = cost, best = tn;
    }
    switch (best) {
        case 256: return launch_tile<T, 256>(a, wide, sms, s);
        case 192: return launch_tile<T, 192>(a, wide, sms, s);
        case 160: return launch_tile<T, 160>(a, wide, sms, s);
        case 128: return launch_tile<T, 128>(a, wide, sms, s);
        case 96: return launch_tile<T, 96>(a, wide, sms, s);
        default: return launch_tile<T, 64>(a, wide, sms, s);
    }
}

}  // namespace
}  // namespace sq

extern "C" int32_t sq_matmul_fp8(const sq_matmul_args *args, sq_stream_t stream) {
    if (!args) return SQ_ERR_ARGUMENT;
    const sq_matmul_args &a = *args;
    if (a.rows < 0 || a.width < 1 || a.hidden < 1) return SQ_ERR_ARGUMENT;
    if (a.dtype < SQ_F32 || a.dtype > SQ_F16) return SQ_ERR_ARGUMENT;
    if (a.hidden % 16) return SQ_ERR_UNSUPPORTED;
    if (a.rows == 0) return SQ_OK;
    if (!a.x || !a.x_scale || !a.w || !a.w_scale || !a.out) return SQ_ERR_ARGUMENT;
    if (!sq::aligned16(a.x) || !sq::aligned16(a.w) || a.x_stride < a.hidden || a.w_stride < a.hidden || a.x_stride % 16 ||
        a.w_stride % 16 || a.residual_stride < 0)
        return SQ_ERR_SHAPE;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const int sms = sq::sms_of(s);
    if (sms < 1) return SQ_ERR_CUDA;
    return a.dtype == SQ_F32    ? sq::launch_matmul<float>(a, sms, s)
           : a.dtype == SQ_BF16 ? sq::launch_matmul<__nv_bfloat16>(a, sms, s)
                                : sq::launch_matmul<__half>(a, sms, s);
}
