// Products of 4-bit weights (q4.cuh) for few activation rows: y[t][o] = sum_k x[t][k] code[o][k] scale[o][k / group] (+ bias[o]).
//
// What it cannot do without is reading the weights (half a byte each and two bytes a group); it comes to 0.64 of the copy rate (65536 x 4096, one row
// 33.5 us), where four warps a scheduler keep 59 % of the issue slots busy and no unit full.  Every warp streams them through a ring of its own in shared memory:
// TMA copies of the 128 or 256 columns (a unit) of RT row tiles, 1 or 2 KB each, and their scales, some units ahead, across rows and
// experts: some 70 KB under way per SM, which the bandwidth times the latency wants (loads to registers two units ahead in 16 warps an
// SM were 16 KB, and 65536 x 4096 with 8 tokens took 69 us).  A warp waits for and refills its own stages only.
// A lane's 16 bytes of a tile are the A fragments of four mma.sync m16n8k16, the codes as exact numbers -8 .. 7, and its eight columns of an
// activation row are the B fragments of two of them, read where the row lies (L1 holds the few rows that an SM's warps share).
// Sums of a group are scaled and added in fp32.  Beside bf16, whose numbers reach as far as fp32's, the codes are 2^-10 of what they are up to
// the last step: 128 times 8 times the largest number stays finite, and so does a result that should be.  A block's warps take the units of
// its rows in turn and their sums meet in shared memory, in warp order: results do not depend on the schedule.
//
// float32 activations come as three bf16 planes (all 24 bits, stage_planes), each multiplied exactly; the first has sums of its own, since the
// tensor core cuts small terms beside large ones off.
//
// The same kernel multiplies rows sorted by expert (`offsets`): blocks go through the experts that have rows; rows of none, ahead
// of the first one's or behind the last one's, become zero.
#include "common.cuh"
#include "launch_order.cuh"
#include "q4.cuh"
#include "tma.cuh"
#include "umma.cuh"

#include <atomic>
#include <cmath>
#include <cstring>
#include <type_traits>

namespace t81b200 {

// gemm_q4_tc.cu
int gemm_q4_tc_launch(const uint8_t *codes, const void *scales, const float *bias, void *C, int64_t M, const void *x, bool f16, int planes, int64_t ldx, int c_dtype, int64_t ldc, int64_t N,
                      int64_t K, int group, const int32_t *offsets, int n_experts, cudaStream_t st);
double gemm_q4_tc_estimate_us(int64_t M, int64_t N, int64_t K, int planes, int n_experts, double reached);

namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32, kMostExperts = 1024, kOwners = 1024, kBlocksPerSm = 2;
enum { STATUS_CONSUMER = 6 };

__device__ int g_gemv_q4_status = 0;

struct Q4Params {
    const uint8_t *codes;
    const __nv_bfloat16 *scales;
    const float *bias;
    const void *x;
    void *y;
    int64_t ldx, ldy, plane_elems;  // elements
    int M, kx;                      // kx: columns of x that may be read, a multiple of 8 (zeros past K)
    int rows;                       // of x
    int y_dtype;
    int64_t bias_stride;            // from one expert to the next
    const int32_t *offsets;         // n_experts + 1, or null: one matrix for all rows
    int n_experts;
    int col_tiles, groups, units;   // of a row
    int row_tiles, row_items;       // 16-row tiles, and blocks' shares of them (RT * k_split-wise rows)
    int k_warps;                    // warps that share a row tile's units
};

template <typename T> constexpr int kDown = std::is_same<T, __nv_bfloat16>::value ? 10 : 0;

// Where a warp is: a block's share of the row tiles (of an expert), and a piece of at most TOK rows of x.  Items go through the shares of one
// piece before those of the next, and a block takes every gridDim.x-th.
template <int TOK> struct Walk {
    int share, piece, expert, tile0, tok, end;
    // `owner`: the experts of the first kOwners pieces; items of one unit or two leave no time to look for them.
    __device__ __forceinline__ void open(const Q4Params &p, const ExpertList &list, const int16_t *owner, int tiles_per_item, int tile_of_item, int steps) {
        share += steps;
        if (steps == 0 || share >= p.row_items) {
            const int more = share / p.row_items;
            piece += more;
            share -= more * p.row_items;
            tok = piece * TOK;
            end = p.rows;
            if (p.offsets) {
                expert = piece < kOwners ? owner[piece] : list.expert_of(piece, p.n_experts);
                tok = list.first(expert) + (piece - list.before(expert)) * TOK;
                end = list.first(expert + 1);
            }
            end = min(end, tok + TOK);
        }
        tile0 = share * tiles_per_item + tile_of_item;
    }
};

// A unit is W x 128 columns; four stages of 128 or two of 256.
template <int RT, int W, int GROUP> struct Stage {
    static constexpr int kCodes = RT * W * 1024, kScales = W * (128 / GROUP) * 32, kBytes = kCodes + (RT * kScales + 127) / 128 * 128, kCount = W == 1 ? 4 : 2;
};

// acc = (FIRST) or += the fragment's product with 16 of the 32 columns of x at hand, the second ones with `second`.
template <typename T, int PLANES, int NT, bool FIRST>
__device__ __forceinline__ void products(float (&acc)[NT][PLANES == 1 ? 1 : 2][4], const uint32_t (&a)[4], const uint4 (&x)[PLANES][NT], int second) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        mma_16816<T, !FIRST>(acc[n][0], a, second ? x[0][n].z : x[0][n].x, second ? x[0][n].w : x[0][n].y);
        if constexpr (PLANES == 3) {
            mma_16816<T, !FIRST>(acc[n][1], a, second ? x[1][n].z : x[1][n].x, second ? x[1][n].w : x[1][n].y);
            mma_16816<T, true>(acc[n][1], a, second ? x[2][n].z : x[2][n].x, second ? x[2][n].w : x[2][n].y);
        }
    }
}

__device__ __forceinline__ void store(void *y, int64_t at, float v, int dtype) {
    if (dtype == T81B200_F32) static_cast<float *>(y)[at] = v;
    else if (dtype == T81B200_BF16) static_cast<__nv_bfloat16 *>(y)[at] = __float2bfloat16_rn(v);
    else static_cast<__half *>(y)[at] = __float2half_rn(v);
}

// T: type of the operands; PLANES: 1, or 3 of float32 activations; RT: row tiles a warp; NT: blocks of 8 rows of x at a time; W: 128
// columns of a unit.
template <typename T, int PLANES, int RT, int NT, int W, int GROUP>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
gemv_q4_kernel(const __grid_constant__ CUtensorMap map_codes, const __grid_constant__ CUtensorMap map_scales, const __grid_constant__ Q4Params p) {
    using S = Stage<RT, W, GROUP>;
    constexpr int PER = 128 / GROUP, SUMS = PLANES == 1 ? 1 : 2, TOK = 8 * NT;
    // Rows of x are fetched a unit at a time before the wait for its codes, or 128 columns at a time, as registers hold them.
    constexpr bool EARLY = PLANES * NT == 1;
    extern __shared__ __align__(128) uint8_t ring[];  // [warps][stages][RT units of codes, RT of scales], then part
    __shared__ __align__(8) uint64_t full[kWarps][S::kCount];
    __shared__ int failed;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int kw = warp % p.k_warps, row_warps = kWarps / p.k_warps, rw = warp / p.k_warps;
    constexpr int WIDTH = RT * 16 + 1, PART = kWarps * TOK * WIDTH;
    float *part = reinterpret_cast<float *>(ring + kWarps * S::kCount * S::kBytes);  // two of [warps][TOK][WIDTH] in turn, so that one barrier a pass is enough
    if (lane < S::kCount) mbar_init(smem_u32(&full[warp][lane]), 1);
    if (threadIdx.x == 0) {
        failed = 0;
        prefetch_map(&map_codes);
        prefetch_map(&map_scales);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    wait_for_kernel_ahead();
    ExpertList list;
    int16_t *const owner = reinterpret_cast<int16_t *>(reinterpret_cast<uint8_t *>(part + 2 * PART) + ExpertList::bytes(p.n_experts));
    int items = (p.rows + TOK - 1) / TOK * p.row_items;
    if (p.offsets) {
        items = list.build(reinterpret_cast<int32_t *>(part + 2 * PART), p.offsets, p.n_experts, p.rows, TOK) * p.row_items;
        for (int e = threadIdx.x; e < p.n_experts; e += kThreads)
            for (int q = list.before(e); q < min(list.before(e + 1), kOwners); ++q) owner[q] = (int16_t)e;
        const int ahead = list.first(0), taken = list.first(p.n_experts) - ahead;
        for (int64_t at = (int64_t)blockIdx.x * kWarps + warp; at < (int64_t)p.rows - taken; at += (int64_t)gridDim.x * kWarps) {  // rows of no expert: a warp each
            const int64_t row = at < ahead ? at : at + taken;
            for (int i = lane; i < p.M; i += 32) store(p.y, row * p.ldy + i, 0.0f, p.y_dtype);
        }
    }
    __syncthreads();

    const uint32_t my_ring = smem_u32(ring) + (uint32_t)(warp * S::kCount * S::kBytes), my_full = smem_u32(&full[warp][0]);
    const int per_item = row_warps * RT;
    Walk<TOK> fill, use;
    fill.share = use.share = (int)blockIdx.x;
    fill.piece = use.piece = fill.expert = use.expert = 0;
    int fill_item = (int)blockIdx.x, item = fill_item;
    if (item < items) {
        fill.open(p, list, owner, per_item, rw * RT, 0);
        use.open(p, list, owner, per_item, rw * RT, 0);
    }
    // ---- copies (what lies past the matrix arrives as zeros, or is the next expert's rows) ----
    int fill_unit = kw, fill_row = fill.expert * p.row_tiles + fill.tile0;
    uint32_t slot = 0;
    auto issue = [&]() {
        if (fill_item >= items) return;
        if (elect_one()) {
            const uint32_t bar = my_full + 8u * slot, dst = my_ring + slot * S::kBytes;
            mbar_arrive_expect_tx(bar, (uint32_t)(S::kCodes + RT * S::kScales));
            tma_load_3d(dst, &map_codes, 0, fill_unit * (2 * W), fill_row, bar);
            tma_load_2d(dst + S::kCodes, &map_scales, fill_unit * (W * PER * 16), fill_row, bar);
        }
        __syncwarp();
        slot = slot + 1 == S::kCount ? 0 : slot + 1;
        fill_unit += p.k_warps;
        if (fill_unit >= p.units) {
            fill_unit = kw;
            fill_item += (int)gridDim.x;
            if (fill_item < items) fill.open(p, list, owner, per_item, rw * RT, (int)gridDim.x);
            fill_row = fill.expert * p.row_tiles + fill.tile0;
        }
    };
    if (p.units > 0)
        for (int i = 0; i < S::kCount; ++i) issue();
    const Q4Decode<T, kDown<T>> decode;
    const uint32_t zero = unknown_zero();
    Ring at;
    bool ok = true, buffer = false;
    for (; item < items; item += (int)gridDim.x) {
        const int tile0 = use.tile0;
        float sum[RT][NT][SUMS][4] = {};
        // this lane's eight columns of a row of x for the B fragments; rows past the last are some other row's, and not stored
        const T *src_x[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) src_x[n] = static_cast<const T *>(p.x) + (int64_t)min(use.tok + 8 * n + g, use.end - 1) * p.ldx + kw * (W * 128) + 8 * t;
        for (int unit = kw; unit < p.units; unit += p.k_warps) {
            const int columns = p.kx - unit * (W * 128);  // from here on
            const bool whole = columns >= W * 128;
            uint4 b[EARLY ? 4 * W : 4][PLANES][NT];       // 32 columns each
            auto load_x = [&](int i, int into) {
#pragma unroll
                for (int pl = 0; pl < PLANES; ++pl)
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const T *src = src_x[n] + pl * p.plane_elems + 32 * i;
                        if (whole) b[into][pl][n] = __ldg(reinterpret_cast<const uint4 *>(src));
                        else b[into][pl][n] = 32 * i + 8 * t < columns ? __ldg(reinterpret_cast<const uint4 *>(src)) : make_uint4(0u, 0u, 0u, 0u);
                    }
            };
            if constexpr (EARLY)
#pragma unroll
                for (int i = 0; i < 4 * W; ++i) load_x(i, i);
            ok = __all_sync(0xffffffffu, mbar_wait(my_full + 8u * at.stage, at.phase));
            if (!ok) break;
            const uint8_t *src = ring + (warp * S::kCount + at.stage) * S::kBytes;
#pragma unroll
            for (int h = 0; h < W; ++h) {
                if constexpr (!EARLY)
#pragma unroll
                    for (int i = 0; i < 4; ++i) load_x(4 * h + i, i);
                uint32_t word[RT][8], scale[RT][PER];
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const uint8_t *at_r = src + (r * W + h) * 1024 + lane * 16;
                    const uint4 q0 = *reinterpret_cast<const uint4 *>(at_r), q1 = *reinterpret_cast<const uint4 *>(at_r + 512);
                    word[r][0] = q0.x; word[r][1] = q0.y; word[r][2] = q0.z; word[r][3] = q0.w;
                    word[r][4] = q1.x; word[r][5] = q1.y; word[r][6] = q1.z; word[r][7] = q1.w;
#pragma unroll
                    for (int i = 0; i < PER; ++i) scale[r][i] = *reinterpret_cast<const uint32_t *>(src + S::kCodes + r * S::kScales + (h * PER + i) * 32 + 4 * g);
                }
                // 128 columns: sum += scale * sums over the columns of a group, group after group.
                // (What lies past the last column meets zeros of x, rows past the last are not stored.)
                float c[RT][NT][SUMS][4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {  // 32 columns
                    const auto &x = b[EARLY ? 4 * h + i : i];
#pragma unroll
                    for (int j = 2 * i; j < 2 * i + 2; ++j)
#pragma unroll
                        for (int r = 0; r < RT; ++r) {
                            uint32_t a[4];
                            q4_fragments(decode, word[r][j], a);
                            if (j % (GROUP / 16) == 0) products<T, PLANES, NT, true>(c[r], a, x, j & 1);
                            else products<T, PLANES, NT, false>(c[r], a, x, j & 1);
                        }
                    if ((i + 1) % (GROUP / 32) != 0) continue;
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        const uint32_t s = scale[r][i / (GROUP / 32)];
                        const float lo = __uint_as_float(s << 16), hi = __uint_as_float(s & 0xFFFF0000u);
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int u = 0; u < SUMS; ++u)
#pragma unroll
                                for (int k = 0; k < 4; ++k) sum[r][n][u][k] = fmaf(c[r][n][u][k], k < 2 ? lo : hi, sum[r][n][u][k]);
                    }
                }
            }
            // Into the stage just read, once what was read has been used: a copy does not wait for loads of shared memory still on their way.
            uint32_t used = 0;
#pragma unroll
            for (int r = 0; r < RT; ++r) used |= __float_as_uint(sum[r][0][0][0]);
            if (all_loaded(used, zero)) issue();
            at.advance(S::kCount);
#pragma unroll
            for (int n = 0; n < NT; ++n) src_x[n] += p.k_warps * (W * 128);
        }
        if (!ok && lane == 0) failed = 1;
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float v = SUMS == 2 ? sum[r][n][0][i] + sum[r][n][SUMS - 1][i] : sum[r][n][0][i];
                    part[(warp * TOK + 8 * n + 2 * t + (i & 1)) * WIDTH + r * 16 + g + 8 * (i >> 1)] = v;
                }
        __syncthreads();
        if (failed) break;  // whoever reads it late finds it, too, at the next barrier: it is never taken back
        for (int i = threadIdx.x; i < (use.end - use.tok) * row_warps * RT * 16; i += kThreads) {
            const int r = i % (RT * 16), share = i / (RT * 16) % row_warps, tok = i / (RT * 16 * row_warps);
            const int row = (tile0 - rw * RT + share * RT) * 16 + r;
            if (row >= p.M) continue;
            float v = 0.0f;
            for (int w = 0; w < p.k_warps; ++w) v += part[((share * p.k_warps + w) * TOK + tok) * WIDTH + r];
            v *= (float)(1 << kDown<T>);
            if (p.bias) v += p.bias[use.expert * p.bias_stride + row];
            store(p.y, (int64_t)(use.tok + tok) * p.ldy + row, v, p.y_dtype);
        }
        part = buffer ? part - PART : part + PART;
        buffer = !buffer;
        if (item + (int)gridDim.x < items) use.open(p, list, owner, per_item, rw * RT, (int)gridDim.x);
    }
    if (failed) give_up(&g_gemv_q4_status, STATUS_CONSUMER);
}

template <typename T, int PLANES, int RT, int NT, int W, int GROUP>
int launch(Q4Params &p, cudaStream_t st) {
    using S = Stage<RT, W, GROUP>;
    const int row_warps = kWarps / p.k_warps;
    p.row_items = (p.row_tiles + RT * row_warps - 1) / (RT * row_warps);
    const int64_t pieces = p.offsets ? (p.rows + 8 * NT - 1) / (8 * NT) + (p.rows < p.n_experts ? p.rows : p.n_experts) : (p.rows + 8 * NT - 1) / (8 * NT);
    const int64_t items = (int64_t)p.row_items * pieces, most = (int64_t)sm_count() * kBlocksPerSm;
    if (items >= 1ll << 31) return fail(T81B200_ELIMIT, "linear_q4: too many rows for a matrix of this size");
    constexpr size_t fixed = (size_t)kWarps * (S::kCount * S::kBytes + 2 * 8 * NT * (RT * 16 + 1) * sizeof(float)), limit = fixed + ExpertList::bytes(kMostExperts) + kOwners * 2;
    const size_t smem = fixed + (p.offsets ? ExpertList::bytes(p.n_experts) + kOwners * 2 : 0);
    CUtensorMap mc, ms;
    memset(&mc, 0, sizeof mc);
    memset(&ms, 0, sizeof ms);
    if (p.units > 0) {
        const cuuint64_t tiles = (cuuint64_t)p.row_tiles * (p.offsets ? p.n_experts : 1), scale_row = (cuuint64_t)(p.groups + 1) * 16;
        const cuuint64_t dims[3] = {kQ4TileBytes / 4, (cuuint64_t)p.col_tiles, tiles}, strides[2] = {kQ4TileBytes, (cuuint64_t)p.col_tiles * kQ4TileBytes};
        const cuuint32_t box[3] = {kQ4TileBytes / 4, 2 * W, RT};
        if (int rc = make_map(&mc, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, p.codes, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE)) return rc;
        if (int rc = make_map_2d(&ms, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p.scales, scale_row, tiles, scale_row * 2, W * (128 / GROUP) * 16, RT, CU_TENSOR_MAP_SWIZZLE_NONE)) return rc;
    }
    auto kernel = gemv_q4_kernel<T, PLANES, RT, NT, W, GROUP>;
    static std::atomic<bool> configured[64];  // the shared-memory limit is an attribute of the function on a device
    int dev = 0;
    T81_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
        T81_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)limit));
        if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
    }
    T81_CUDA_TRY(launch_behind(kernel, dim3((unsigned)(items < most ? items : most)), dim3(kThreads), smem, st, mc, ms, p));
    return T81B200_OK;
}

template <typename T, int PLANES, int RT, int NT, int W>
int launch_group(Q4Params &p, int group, cudaStream_t st) {
    p.units = (p.units + W - 1) / W;
    // As many warps share a row tile's units as find one: a block then has row tiles enough for the SMs, and folds the more sums behind its barrier.
    // Where there are row tiles and pieces of x for all blocks anyway, fewer can do as well or better (us, eight, four, two, one: 1024 x 4096, one row
    // 3.6, 5.2, 8.6, 15.0; 4096 x 14336 11.0, 14.4, 25.7, 48.9; 14336 x 4096 12.0, 11.4, 13.3, 22.0; 65536 x 4096, 8 rows 40.7, 43.4, 42.0, 40.7; 64 experts of 2816 x 2048,
    // 8 tokens 26.2, 23.3, 22.6, 22.8, one token 8.5, 7.6, 9.2, 13.1); the rule has no term for that.
    p.k_warps = p.units >= 8 ? 8 : (p.units >= 4 ? 4 : (p.units >= 2 ? 2 : 1));
    if (group == 32) return launch<T, PLANES, RT, NT, W, 32>(p, st);
    if (group == 64) return launch<T, PLANES, RT, NT, W, 64>(p, st);
    return launch<T, PLANES, RT, NT, W, 128>(p, st);
}

template <typename T, int PLANES, int RT, int NT>
int launch_width(Q4Params &p, int group, cudaStream_t st) {
    if constexpr (PLANES == 1)
        if (p.units >= 16) return launch_group<T, PLANES, RT, NT, 2>(p, group, st);
    return launch_group<T, PLANES, RT, NT, 1>(p, group, st);
}

// p.units: of 128 columns.
template <typename T, int PLANES>
int launch_shape(Q4Params &p, int group, cudaStream_t st) {
    // Sixteen rows of x at a time beyond eight: 16 tokens of 4096 x 14336, bf16, 16.3 us, in two passes of eight 21.4.  Not for experts, most of
    // which have a few rows (64 of 2816 x 2048, 8 tokens in 6 each: 28 and 36 us), and not in three planes, which the registers do not hold.
    const bool two = PLANES == 1 && p.rows > 8 && !p.offsets;
    const int64_t pieces = p.offsets ? (p.rows < p.n_experts ? p.rows : p.n_experts) : (two ? (p.rows + 15) / 16 : (p.rows + 7) / 8);
    // Two row tiles a warp read each piece of an activation row once for both, where that leaves every block its shares (us, one and two: 65536 x
    // 4096, 8 tokens 47.7 and 39.7, 4096 x 14336 11.4 and 12.0, 1024 x 4096 3.3 and 4.1).
    const bool wide = p.row_tiles * pieces >= 4 * (int64_t)sm_count();
    if constexpr (PLANES == 1)
        if (two) return wide ? launch_width<T, PLANES, 2, 2>(p, group, st) : launch_width<T, PLANES, 1, 2>(p, group, st);
    return wide ? launch_width<T, PLANES, 2, 1>(p, group, st) : launch_width<T, PLANES, 1, 1>(p, group, st);
}

// Rows that the kernels read where they are: 16-bit, on 16-byte boundaries, whole pieces of eight columns.
bool in_place(const void *B, int b_dtype, int64_t ldb, int64_t K) {
    return b_dtype != T81B200_F32 && reinterpret_cast<uintptr_t>(B) % 16 == 0 && ldb % 8 == 0 && K % 8 == 0;
}
int64_t staged_row(int64_t K) { return (K + 7) & ~(int64_t)7; }

// Whether the tensor-core kernel's tiles take less time than this kernel's pieces of 16 rows of x (8 of experts' rows), by both estimates.  Ours:
// fitted to 9 to 128 rows of 512 x 512 to 32768 x 4096 and 32 to 1024 rows of 8 to 64 experts (us, tiles and pieces: 32 rows of 1024 x 4096 10.9
// and 5.6, of 4096 x 4096 12.6 and 12.2, of 14336 x 4096 20.4 and 29.8, 64 of 2048 x 2048 9.8 and 7.9; 256 rows in 64 experts of 2816 x
// 2048 58 and 52, 512 67 and 84).  float32, pieces of 8: 77 rows of 1999 x 3001 15.3 and 24.0, 256 of 14336 x 4096 69 and 406.
bool tiles_are_faster(int64_t M, int64_t N, int64_t K, int planes, int n_experts) {
    if (N <= (planes == 3 ? 8 : 16) && n_experts == 0) return false;
    const double tiles = (double)q4_row_tiles(M) * (double)q4_col_tiles(K);
    const double reached = n_experts == 0 ? 1.0 : n_experts * (1.0 - pow(1.0 - 1.0 / n_experts, (double)N));
    const double pieces = n_experts != 0 ? reached + (double)N / 8.0 : (double)(planes == 3 ? (N + 7) / 8 : (N + 15) / 16);
    const double ours = 3.5 + pieces * (planes == 3 ? 0.05 + 3.2e-4 * tiles : (n_experts == 0 ? 1.95e-4 * tiles : 0.05 + 1.15e-4 * tiles));
    return gemm_q4_tc_estimate_us(M, N, K, planes, n_experts, reached) < ours;
}

int product_q4(const char *name, const uint8_t *codes, const void *scales, const float *bias, void *C, int64_t M, const void *B, int b_dtype, int64_t ldb, int c_dtype, int64_t ldc,
               int64_t N, int64_t K, int group, const int32_t *offsets, int n_experts, void *workspace, size_t workspace_bytes, cudaStream_t st) {
    if (M < 0 || N < 0 || K < 0 || ldb < K || ldc < M || n_experts < 0) return fail(T81B200_EINVAL, "%s: bad dimensions", name);
    if (!q4_group_ok(group)) return fail(T81B200_EINVAL, "%s: groups of 32, 64 or 128 columns, not %d", name, group);
    if (dtype_size(b_dtype) == 0 || b_dtype < 0 || b_dtype > T81B200_F16 || c_dtype < 0 || c_dtype > T81B200_F16) return fail(T81B200_EINVAL, "%s: unknown dtype", name);
    if (M >= (1ll << 31) - 4096 || N >= (1ll << 31) - 4096 || K >= (1ll << 31) - 4096 || n_experts > kMostExperts || q4_row_tiles(M) * (n_experts > 0 ? n_experts : 1) >= (1ll << 31))
        return fail(T81B200_ELIMIT, "%s: dimension too large (at most %d experts)", name, kMostExperts);
    if (int rc = check_device()) return rc;
    if (M == 0 || N == 0) return T81B200_OK;
    if (!C || (K > 0 && (!B || !codes || !scales))) return fail(T81B200_EINVAL, "%s: null pointer", name);
    if (reinterpret_cast<uintptr_t>(codes) % 16 != 0 || reinterpret_cast<uintptr_t>(scales) % 16 != 0) return fail(T81B200_EALIGN, "%s: codes and scales must be 16-byte aligned", name);
    Q4Params p = {};
    p.codes = codes; p.scales = static_cast<const __nv_bfloat16 *>(scales); p.bias = bias;
    p.x = B; p.ldx = ldb; p.kx = (int)K;
    p.y = C; p.ldy = ldc; p.y_dtype = c_dtype;
    p.M = (int)M; p.rows = (int)N;
    p.offsets = offsets; p.n_experts = n_experts;
    p.bias_stride = M;
    p.col_tiles = (int)q4_col_tiles(K); p.groups = (int)q4_groups(K, group); p.units = (int)((K + 127) / 128); p.row_tiles = (int)q4_row_tiles(M);

    if (K > 0 && !in_place(B, b_dtype, ldb, K)) {
        const size_t need = (size_t)(b_dtype == T81B200_F32 ? 3 : 1) * N * staged_row(K) * 2;
        if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
            return fail(T81B200_EWORKSPACE, "%s: %zu bytes of 16-byte aligned workspace needed, %zu given", name, need, workspace_bytes);
        if (int rc = stage_planes(B, b_dtype, T81B200_LAYOUT_NK, ldb, N, K, 3, workspace, st)) return rc;
        p.x = workspace;
        p.ldx = staged_row(K);
        p.kx = (int)p.ldx;
        p.plane_elems = N * p.ldx;
    }
    const int planes = b_dtype == T81B200_F32 ? 3 : 1;
    if (K > 0 && (planes == 1 || 3 * N < (1ll << 31)) && tiles_are_faster(M, N, K, planes, offsets ? n_experts : 0))
        return gemm_q4_tc_launch(codes, scales, bias, C, M, p.x, b_dtype == T81B200_F16, planes, p.ldx, c_dtype, ldc, N, K, group, offsets, n_experts, st);
    if (b_dtype == T81B200_F32) return launch_shape<__nv_bfloat16, 3>(p, group, st);
    return b_dtype == T81B200_BF16 ? launch_shape<__nv_bfloat16, 1>(p, group, st) : launch_shape<__half, 1>(p, group, st);
}

}  // namespace

int gemv_q4_status(int reset) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_gemv_q4_status, sizeof v) != cudaSuccess) return T81B200_ECUDA;
    if (reset && v != 0) {
        const int zero = 0;
        if (cudaMemcpyToSymbol(g_gemv_q4_status, &zero, sizeof zero) != cudaSuccess) return T81B200_ECUDA;
    }
    return v;
}

}  // namespace t81b200

using namespace t81b200;

extern "C" size_t t81b200_linear_q4_workspace_bytes(const void *B, int b_dtype, int64_t ldb, int64_t N, int64_t K) {
    if (N <= 0 || K <= 0 || in_place(B, b_dtype, ldb, K)) return 0;
    return (size_t)(b_dtype == T81B200_F32 ? 3 : 1) * N * staged_row(K) * 2;
}

extern "C" int t81b200_linear_q4(const uint8_t *codes, const void *scales, const float *bias, void *C, int64_t M, const void *B, int b_dtype, int64_t ldb, int c_dtype, int64_t ldc,
                                 int64_t N, int64_t K, int group, void *workspace, size_t workspace_bytes, void *stream) {
    return product_q4("linear_q4", codes, scales, bias, C, M, B, b_dtype, ldb, c_dtype, ldc, N, K, group, nullptr, 0, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

extern "C" int t81b200_experts_q4(const uint8_t *codes, const void *scales, const float *bias, void *C, int64_t M, const void *B, int b_dtype, int64_t ldb, int c_dtype, int64_t ldc,
                                  int64_t N, int64_t K, int group, const int32_t *offsets, int n_experts, void *workspace, size_t workspace_bytes, void *stream) {
    if (!offsets || n_experts < 1) return fail(T81B200_EINVAL, "experts_q4: offsets of at least one expert are needed");
    return product_q4("experts_q4", codes, scales, bias, C, M, B, b_dtype, ldb, c_dtype, ldc, N, K, group, offsets, n_experts, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}
