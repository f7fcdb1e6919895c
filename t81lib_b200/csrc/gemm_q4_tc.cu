// Products of 4-bit weights (q4.cuh) on the 5th-generation tensor cores (tcgen05), for more activation rows than the streaming kernel
// serves well: 16-bit activations or float32 in three bf16 planes, one matrix or rows sorted by expert.
//
//   D[o][t] = sum_k W[o][k] * x[t][k]     o: output feature (256 per CTA pair, 128 per CTA), t: row of x (up to 256 per tile)
//
// The form is gemm_trit_tc.cu's: a pair of CTAs (cta_group::2) works on one tile, each expands its own 128 weight rows into its shared memory
// and loads half of the tile's activation rows by TMA; the even CTA issues the MMAs, and each CTA keeps its 128 accumulator rows in
// TMEM (2 x 256 columns, in turn).  What bounds it is shared memory: a 64-deep step writes and reads 16 KB of expanded weights per CTA and
// writes and reads its half of the activations.
//
// Weights: 128 columns (a chunk) of 128 rows are 8 KB of codes and up to 1 KB of scales, one TMA load each; a converter warp per 16 rows
// turns them into operands of 128-byte rows.  A pair of codes is a shift, an AND-OR and one packed FMA, v * s - 24 s on v = 16 + code + 8, which
// is exact: a code times its scale is a bf16 number.  Beside fp16 activations the scales of a row are first brought to 2^10 .. 2^11 at
// the largest by a power of two, which the result is divided by: fp16 holds all of a row's weights then whose scale is no less than 2^-30 of that.
// Where a converter meets a smaller scale, which counts as soon as the activations beside the large ones are small, the CTA
// goes over its tiles once more at its end and writes the results of such rows from sums in fp32 registers (mend_rows).
//
// float32 activations come as three bf16 planes (all 24 bits, stage_planes), each a product of its own with the same expanded weights.  The tensor
// core cuts an accumulator off at every 16 columns: 2.4e-7 of the result after 1024 columns, 5.6e-7 after 2048, 1.4e-6 after 4096, 7e-6
// after 14336 (bf16 values, whose products are exact).  So the first plane has an accumulator per 2048 columns, the other two share one, and
// the epilogue adds them.
//
// Rows sorted by expert: every CTA turns the experts' row counts into a list of tiles of its own (a sum over experts in shared memory) and the
// persistent clusters take tiles of it in turn.  An expert's rows are split evenly into tiles of whole 32 rows; rows of a tile past
// the expert's last are multiplied and not stored.
//
// Few tiles: the contraction is split over S = 2 to 4 pairs of a cluster, whose sums meet in shared memory and are added in rank order.
//
// 23 warps per CTA: 0 activations   1 MMA issuer (even CTA), TMEM allocation   2-5 epilogue   6-21 converters (two groups of eight that take
// alternate chunks)   22 codes and scales.
// Every mbarrier wait is bounded; on expiry the role records a status code and all roles fall through to the common teardown.
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

namespace {

constexpr int BM = 128, BK = 64, CHUNK = 128;
constexpr int A_ATOM_BYTES = BM * BK * 2, A_CHUNK_BYTES = 2 * A_ATOM_BYTES;  // 16 and 32 KB
constexpr int RAW_CODES = 8 * 1024;                                          // a chunk's codes; its scales lie behind them
constexpr int A_STAGES = 3, RAW_MAX = 8, B_MAX = 12, MAX_SPLITS = 4;
constexpr int NUM_THREADS = 23 * 32, EPILOGUE_WARP0 = 2, CONVERTER_WARP0 = 6, CONVERTERS = 8, RAW_WARP = 22;
constexpr int FINISHERS = (RAW_WARP - EPILOGUE_WARP0) / 4;  // groups of four warps that finish a tile alone in its launch
constexpr int BARRIER_BYTES = 512;
constexpr int SMEM_LIMIT = 227 * 1024;

enum { STATUS_PRODUCER = 1, STATUS_MMA = 2, STATUS_EPILOGUE = 3, STATUS_CONVERTER = 4 };

__device__ int g_q4_status = 0;

struct Q4TcParams {
    const __nv_bfloat16 *scales;
    const float *bias;
    void *C;
    const int32_t *offsets;
    int64_t ldc;
    int M, N;                   // output features (of an expert), rows of x
    int n_experts, row_tiles;   // 16-row tiles of an expert
    int groups;
    const uint8_t *codes;       // and x, for rows that fp16 does not hold
    const void *x;
    int64_t ldx;
    int K, group;
    int m_tiles, n_tiles;       // 256-row pair tiles; tiles of bn rows of x (one matrix)
    int bn;                     // most rows of x a tile, a multiple of 32
    int n_atoms, n_chunks;
    int splits, raw_stages, b_stages, one_tile, out_bytes, list_bytes;
    int vec;                    // 16-byte stores are possible
    int bufs, acc_cols;         // tiles whose sums TMEM holds at a time, and the columns of each
    int seg_chunks;             // three planes: chunks of the first plane that an accumulator takes
};

// Tensor maps of x.  One matrix: [0] with boxes of half a tile.  Experts, whose tiles differ: boxes of 128, 64, 32 and 16 rows, the binary digits of
// half a tile (in boxes of 16 alone 37 experts of 2048 x 4096 with 256 rows each took 119 us, 109 so).
struct XMaps {
    CUtensorMap m[4];
};

// What a tile is: its expert, first output feature, rows [tok, end) and their number rounded up to 32.
struct Tile {
    int expert, row0, tok, end, n;
};

template <bool EXPERTS> struct TileList;
template <> struct TileList<false> {
    __device__ __forceinline__ int build(const Q4TcParams &p, int32_t *) { return p.m_tiles * p.n_tiles; }
    __device__ __forceinline__ Tile tile(const Q4TcParams &p, int i, int half) const {
        const int tok = i / p.m_tiles * p.bn;
        return {0, (i % p.m_tiles * 2 + half) * BM, tok, min(tok + p.bn, p.N), p.bn};
    }
};
template <> struct TileList<true> {
    ExpertList list;
    __device__ __forceinline__ int build(const Q4TcParams &p, int32_t *memory) { return list.build(memory, p.offsets, p.n_experts, p.N, p.bn) * p.m_tiles; }
    __device__ __forceinline__ Tile tile(const Q4TcParams &p, int i, int half) const {
        const int at = i / p.m_tiles, e = list.expert_of(at, p.n_experts);
        const int2 here = list.at[e], then = list.at[e + 1];  // first row, tiles ahead
        const int tiles = then.y - here.y, width = ((then.x - here.x + tiles - 1) / tiles + 31) / 32 * 32;
        const int tok = here.x + (at - here.y) * width, end = min(tok + width, then.x);
        return {e, (i % p.m_tiles * 2 + half) * BM, tok, end, max((end - tok + 31) / 32 * 32, 32)};
    }
};

__device__ __forceinline__ bool epilogue_all(bool pred) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 q, %1, 0;\n\t"
        "barrier.cta.red.and.pred p, 2, 128, q;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)pred)
        : "memory");
    return r != 0;
}

// One warp's 32 features x 32 rows of x: rows of the result through a buffer of the warp's, 16 bytes a lane, or element by element.
template <typename CT>
__device__ __forceinline__ void emit(const Q4TcParams &p, const uint32_t (&v)[32], int feature0, int lane, float scale, float bias, int tok0, int end, CT *stage) {
    CT *const C = static_cast<CT *>(p.C);
    if (p.vec && feature0 + 32 <= p.M) {
        constexpr int PER = 16 / (int)sizeof(CT), PIECES = 32 / PER;  // of a row
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 32; ++i) stage[i * 32 + lane] = from_float<CT>(fmaf(__uint_as_float(v[i]), scale, bias));
        __syncwarp();
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int at = i * 32 + lane, tok = tok0 + at / PIECES;
            if (tok < end) *reinterpret_cast<uint4 *>(C + (int64_t)tok * p.ldc + feature0 + at % PIECES * PER) = reinterpret_cast<const uint4 *>(stage)[at];
        }
    } else if (feature0 + lane < p.M) {
        CT *dst = C + (int64_t)tok0 * p.ldc + feature0 + lane;
#pragma unroll
        for (int i = 0; i < 32; ++i, dst += p.ldc)
            if (tok0 + i < end) *dst = from_float<CT>(fmaf(__uint_as_float(v[i]), scale, bias));
    }
}

// 32 columns of a tile's sums: with three planes the accumulators of the first plane's segments, bn columns apart, and the others' behind them.
template <int PLANES>
__device__ __forceinline__ void load_sums(const Q4TcParams &p, uint32_t taddr, int segments, uint32_t (&v)[32]) {
    tmem_ld32(taddr, v);
    if constexpr (PLANES == 3)
#pragma unroll 1
        for (int s = 1; s <= segments; ++s) {
            taddr += (uint32_t)p.bn;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t more[8];
                tmem_ld8(taddr + (uint32_t)(8 * q), more);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[8 * q + i] = __float_as_uint(__uint_as_float(v[8 * q + i]) + __uint_as_float(more[i]));
            }
        }
}

// The power of two in a row's largest scale (1 for a row of zeros), as the exponent bits of a float; 2^-103 at least, the format's smallest.
__device__ __forceinline__ uint32_t row_exponent(const __nv_bfloat16 *scales, int64_t tile, int groups, int r) {
    const uint32_t bits = (uint32_t)__ldg(reinterpret_cast<const unsigned short *>(scales) + (tile * (groups + 1) + groups) * 16 + 2 * (r & 7) + (r >> 3)) & 0x7F80u;
    return bits ? max(bits << 16, 0x0C000000u) : 0x3F800000u;
}

// A row's scales beside fp16 activations are multiplied by 2^(kF16Up - e), 2^e being row_exponent: the largest weight is below 2^14 then, 24 scales below
// 2^16.  A scale of five bits is held to the last place of every code times it down to 2^-20, which is kF16Span below 2^e.
constexpr int kF16Up = 10, kF16Span = kF16Up + 20;

// Whether a scale (bf16 bits without the sign) is too small for that beside a row's largest.
__device__ __forceinline__ bool f16_loses(uint32_t scale, uint32_t exponent) { return scale != 0u && (int)scale < (int)(exponent >> 16) - (kF16Span << 7); }

// Results of a tile's rows with such scales, once more as the streaming kernel computes them: codes as whole numbers times fp16, the scale on the fp32
// sum.  16 rows and 16 rows of x at a time; a CTA's warps share the columns, and their sums meet in `part` in warp order.  For the
// few rows that want it, if any: 4096 x 14336, 64 rows of x 27 us, 76 with one such row, 406 where all are.
constexpr int MEND_WARPS = NUM_THREADS / 32, MEND_TOK = 16;
template <typename CT>
__device__ __noinline__ void mend_rows(const Q4TcParams &p, float (*part)[MEND_TOK][17], uint32_t *rows, int expert, int row0, int tok0, int end) {
    const int warp = (int)threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, col_tiles = (int)q4_col_tiles(p.K), halves_per_group = p.group / 32;
    const int64_t first_tile = (int64_t)expert * p.row_tiles + (row0 >> 4);
    if (threadIdx.x < BM / 32) rows[threadIdx.x] = 0u;
    __syncthreads();
    for (int tile16 = warp >> 1; tile16 < BM / 16 && row0 + 16 * tile16 < p.M; tile16 += MEND_WARPS / 2) {  // two warps each, a lane two rows of every eighth group
        const int64_t tile = first_tile + tile16;
        const int r = lane & 7;
        const uint32_t *scales = reinterpret_cast<const uint32_t *>(p.scales + tile * (p.groups + 1) * 16) + r;
        const uint32_t lower = row_exponent(p.scales, tile, p.groups, r), upper = row_exponent(p.scales, tile, p.groups, r + 8);
        uint32_t lost = 0u;
#pragma unroll 4
        for (int u = 4 * (warp & 1) + (lane >> 3); u < p.groups; u += 8) {
            const uint32_t pair = scales[(int64_t)u * 8];
            lost |= (f16_loses(pair & 0x7FFFu, lower) ? 1u : 0u) | (f16_loses(pair >> 16 & 0x7FFFu, upper) ? 256u : 0u);
        }
        if (lost) atomicOr(rows + (tile16 >> 1), lost << (r + 16 * (tile16 & 1)));
    }
    __syncthreads();
    const Q4Decode<__half> decode;
    for (int tile16 = 0; tile16 < BM / 16; ++tile16) {
        const uint32_t mine = rows[tile16 >> 1] >> (16 * (tile16 & 1)) & 0xFFFFu;
        if (mine == 0u) continue;
        const int64_t tile = first_tile + tile16;
        const uint8_t *codes = p.codes + tile * col_tiles * kQ4TileBytes + lane * 16;
        const __nv_bfloat16 *scales = p.scales + tile * (p.groups + 1) * 16 + 2 * g;
        for (int tok = tok0; tok < end; tok += MEND_TOK) {
            float sum[MEND_TOK / 8][4] = {};
            for (int c = warp; c < col_tiles; c += MEND_WARPS) {
                const uint4 q = *reinterpret_cast<const uint4 *>(codes + (int64_t)c * kQ4TileBytes);
                const uint32_t words[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int half = 0; half < 2; ++half) {  // (rows of x are whole pieces of eight, zeros from K on)
                    const int64_t col = 64 * (int64_t)c + 32 * half;
                    const uint32_t s = col < p.K ? *reinterpret_cast<const uint32_t *>(scales + (int64_t)((2 * c + half) / halves_per_group) * 16) : 0u;
                    uint4 x[MEND_TOK / 8];
#pragma unroll
                    for (int n = 0; n < MEND_TOK / 8; ++n) {
                        const __half *src = static_cast<const __half *>(p.x) + (int64_t)min(tok + 8 * n + g, end - 1) * p.ldx + col + 8 * t;
                        x[n] = col + 8 * t < p.K ? *reinterpret_cast<const uint4 *>(src) : make_uint4(0u, 0u, 0u, 0u);
                    }
                    uint32_t a[2][4];
                    q4_fragments(decode, words[2 * half], a[0]);
                    q4_fragments(decode, words[2 * half + 1], a[1]);
                    const float lo = __uint_as_float(s << 16), hi = __uint_as_float(s & 0xFFFF0000u);
#pragma unroll
                    for (int n = 0; n < MEND_TOK / 8; ++n) {
                        float d[4];
                        mma_16816<__half, false>(d, a[0], x[n].x, x[n].y);
                        mma_16816<__half, true>(d, a[1], x[n].z, x[n].w);
#pragma unroll
                        for (int k = 0; k < 4; ++k) sum[n][k] = fmaf(d[k], k < 2 ? lo : hi, sum[n][k]);
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < MEND_TOK / 8; ++n)
#pragma unroll
                for (int k = 0; k < 4; ++k) part[warp][8 * n + 2 * t + (k & 1)][g + 8 * (k >> 1)] = sum[n][k];
            __syncthreads();
            for (int i = threadIdx.x; i < 16 * MEND_TOK; i += NUM_THREADS) {
                const int r = i & 15, row = row0 + 16 * tile16 + r, at = tok + (i >> 4);
                if (!(mine >> r & 1u) || at >= end) continue;
                float v = p.bias ? p.bias[(int64_t)expert * p.M + row] : 0.0f;
                for (int w = 0; w < MEND_WARPS; ++w) v += part[w][i >> 4][r];
                static_cast<CT *>(p.C)[(int64_t)at * p.ldc + row] = from_float<CT>(v);
            }
            __syncthreads();
        }
    }
    __syncthreads();  // `rows` is the next tile's
}

// The same for every tile of a CTA that multiplies experts' rows.  `memory`: its shared memory, in which nothing is awaited any more; the list of experts lies
// behind the rings, what the epilogue stages and the barriers.
template <typename CT>
__device__ __noinline__ void mend_experts(const Q4TcParams &p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *const memory = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
    const uint32_t raw_bytes = RAW_CODES + 8 * (CHUNK / p.group) * 32;
    TileList<true> tiles;
    tiles.list.at = reinterpret_cast<int2 *>(memory + A_STAGES * A_CHUNK_BYTES + p.b_stages * (p.bn * BK) + p.raw_stages * raw_bytes + p.out_bytes + BARRIER_BYTES);
    const int total = tiles.list.before(p.n_experts) * p.m_tiles;
    for (int i = (int)blockIdx.x / 2; i < total; i += (int)gridDim.x / 2) {
        const Tile t = tiles.tile(p, i, (int)(blockIdx.x & 1u));
        mend_rows<CT>(p, reinterpret_cast<float (*)[MEND_TOK][17]>(memory + 16), reinterpret_cast<uint32_t *>(memory), t.expert, t.row0, t.tok, t.end);
    }
}

template <typename T, int PLANES, int GROUP, typename CT, bool EXPERTS>
__global__ void __launch_bounds__(NUM_THREADS, 1)
gemm_q4_tc_kernel(const __grid_constant__ CUtensorMap map_codes, const __grid_constant__ CUtensorMap map_scales, const __grid_constant__ XMaps map_x,
                  const __grid_constant__ Q4TcParams p) {
    constexpr bool F16 = std::is_same<T, __half>::value;
    constexpr int PER = CHUNK / GROUP;
    constexpr uint32_t RAW_BYTES = RAW_CODES + 8 * PER * 32;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *gen_base = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t b_stage_bytes = (uint32_t)(PLANES * p.bn) * (BK * 2 / 2);  // this CTA's half of the rows
    const uint32_t b_off = A_STAGES * A_CHUNK_BYTES, raw_off = b_off + (uint32_t)p.b_stages * b_stage_bytes, out_off = raw_off + (uint32_t)p.raw_stages * RAW_BYTES;
    const uint32_t bars = base + out_off + (uint32_t)p.out_bytes;
    auto a_full = [&](int s) { return bars + 8u * s; };
    auto a_empty = [&](int s) { return bars + 8u * (A_STAGES + s); };
    auto raw_full = [&](int s) { return bars + 8u * (2 * A_STAGES + s); };
    auto raw_empty = [&](int s) { return bars + 8u * (2 * A_STAGES + RAW_MAX + s); };
    auto acc_full = [&](int s) { return bars + 8u * (2 * A_STAGES + 2 * RAW_MAX + s); };
    auto acc_empty = [&](int s) { return bars + 8u * (2 * A_STAGES + 2 * RAW_MAX + 2 + s); };
    auto b_full = [&](int s) { return bars + 8u * (2 * A_STAGES + 2 * RAW_MAX + 4 + s); };
    auto b_empty = [&](int s) { return bars + 8u * (2 * A_STAGES + 2 * RAW_MAX + 4 + B_MAX + s); };
    const uint32_t tmem_slot = bars + 8u * (2 * A_STAGES + 2 * RAW_MAX + 4 + 2 * B_MAX);
    volatile int *const losses = reinterpret_cast<volatile int *>(gen_base + (tmem_slot + 4u - base));  // fp16: a scale of this CTA's rows was too small

    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int half = (int)(rank & 1u), slice = (int)(rank >> 1);
    if (threadIdx.x == 0) {
        for (int s = 0; s < A_STAGES; ++s) { mbar_init(a_full(s), 2 * CONVERTERS); mbar_init(a_empty(s), 1); }
        for (int s = 0; s < RAW_MAX; ++s) { mbar_init(raw_full(s), 1); mbar_init(raw_empty(s), CONVERTERS); }
        for (int s = 0; s < 2; ++s) { mbar_init(acc_full(s), 1); mbar_init(acc_empty(s), 8); }
        for (int s = 0; s < B_MAX; ++s) { mbar_init(b_full(s), 1); mbar_init(b_empty(s), 1); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        *losses = 0;
        prefetch_map(&map_codes);
        prefetch_map(&map_scales);
        prefetch_map(&map_x.m[0]);
    }
    __syncthreads();
    if (warp == 1) tmem_alloc_pair(tmem_slot);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_barrier();  // the other CTAs' barriers are initialised before anything arrives on them
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    // everything up to here overlaps the end of the kernel ahead; no thread touches global memory before this
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t *>(gen_base + (tmem_slot - base));

    TileList<EXPERTS> tiles;
    const int total_tiles = tiles.build(p, reinterpret_cast<int32_t *>(gen_base + (bars - base) + BARRIER_BYTES));
    const int n_clusters = (int)gridDim.x / (2 * p.splits), cluster_id = (int)blockIdx.x / (2 * p.splits);
    const int c0 = p.n_chunks * slice / p.splits, c1 = p.n_chunks * (slice + 1) / p.splits;
    const uint16_t pair_mask = (uint16_t)(3u << (rank & ~1u));
    const int segments = PLANES == 3 ? (c1 - c0 + p.seg_chunks - 1) / p.seg_chunks : 0;

    if constexpr (EXPERTS) {  // rows of no expert: a warp each
#pragma unroll 1
        for (int side = 0; side < 2; ++side) {  // ahead of the first one's and behind the last one's
            const int to = side ? p.N : tiles.list.first(0);
            for (int64_t row = (int64_t)(side ? tiles.list.first(p.n_experts) : 0) + blockIdx.x * (NUM_THREADS / 32) + warp; row < to; row += (int64_t)gridDim.x * (NUM_THREADS / 32)) {
                CT *dst = static_cast<CT *>(p.C) + row * p.ldc;
                if (p.vec && p.M % 8 == 0)
                    for (int i = lane; i < p.M / (16 / (int)sizeof(CT)); i += 32) reinterpret_cast<uint4 *>(dst)[i] = make_uint4(0u, 0u, 0u, 0u);
                else
                    for (int i = lane; i < p.M; i += 32) dst[i] = from_float<CT>(0.0f);
            }
        }
        __syncwarp();
    }
    // factor of the sums and bias of a feature
    auto factor_of = [&](const Tile &t, int r) {
        if (!F16 || t.row0 + r >= p.M) return 1.0f;
        return __uint_as_float(row_exponent(p.scales, (int64_t)t.expert * p.row_tiles + ((t.row0 + r) >> 4), p.groups, r & 15) - (kF16Up << 23));
    };
    auto bias_of = [&](const Tile &t, int r) { return p.bias && t.row0 + r < p.M ? __ldg(p.bias + (int64_t)t.expert * p.M + t.row0 + r) : 0.0f; };

    if (warp == 0) {
        // ---------------- this CTA's half of a tile's rows of x ----------------
        Ring b;
        bool ok = true;
        int chunks = 0;
        for (int i = cluster_id; i < total_tiles && ok; i += n_clusters) {
            const Tile t = tiles.tile(p, i, half);
            const int rows = t.n / 2, row = t.tok + half * rows;
            for (int c = c0; c < c1 && ok; ++c, ++chunks) {
                const int a1 = min(2 * c + 2, p.n_atoms);
                for (int a = 2 * c; a < a1; ++a) {
                    ok = mbar_wait(b_empty(b.stage), b.phase ^ 1);
                    if (!ok) break;
                    if (elect_one()) {
                        if (half == 0) mbar_arrive_expect_tx(b_full(b.stage), 2u * (uint32_t)(PLANES * rows) * (BK * 2));
                        uint32_t dst = base + b_off + (uint32_t)b.stage * b_stage_bytes;
#pragma unroll
                        for (int pl = 0; pl < PLANES; ++pl, dst += (uint32_t)rows * (BK * 2)) {
                            if constexpr (EXPERTS) {
                                int done = 0;
#pragma unroll
                                for (int k = 0; k < 4; ++k)
                                    if (rows & (128 >> k)) {
                                        tma_load_2d_pair(dst + (uint32_t)done * (BK * 2), &map_x.m[k], a * BK, pl * p.N + row + done, b_full(b.stage));
                                        done += 128 >> k;
                                    }
                            } else tma_load_2d_pair(dst, &map_x.m[0], a * BK, pl * p.N + row, b_full(b.stage));
                        }
                    }
                    __syncwarp();
                    b.advance(p.b_stages);
                }
            }
        }
        // The last commits' arrivals come from the pair's issuing CTA; this CTA may not end before they have landed.
        for (int i = 0; i < p.b_stages && ok; ++i) {
            ok = mbar_wait(b_empty(b.stage), b.phase ^ 1);
            b.advance(p.b_stages);
        }
        for (int i = chunks; i < chunks + A_STAGES && ok; ++i) ok = mbar_wait(a_empty(i % A_STAGES), ((uint32_t)(i / A_STAGES) & 1u) ^ 1u);
        if (!ok) give_up(&g_q4_status, STATUS_PRODUCER);
    } else if (warp == RAW_WARP) {
        // ---------------- codes and scales ----------------
        Ring raw;
        bool ok = true;
        for (int i = cluster_id; i < total_tiles && ok; i += n_clusters) {
            const Tile t = tiles.tile(p, i, half);
            const int y = t.expert * p.row_tiles + (t.row0 >> 4);
            for (int c = c0; c < c1; ++c) {
                ok = mbar_wait(raw_empty(raw.stage), raw.phase ^ 1);
                if (!ok) break;
                if (elect_one()) {
                    mbar_arrive_expect_tx(raw_full(raw.stage), RAW_BYTES);
                    const uint32_t dst = base + raw_off + (uint32_t)raw.stage * RAW_BYTES;
                    tma_load_2d(dst, &map_codes, c * 256, y, raw_full(raw.stage));
                    tma_load_2d(dst + RAW_CODES, &map_scales, c * PER * 16, y, raw_full(raw.stage));
                }
                __syncwarp();
                raw.advance(p.raw_stages);
            }
        }
        if (!ok) give_up(&g_q4_status, STATUS_PRODUCER);
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        if (half == 0) {
            Ring a, b;
            bool ok = true;
            int it = 0;
            for (int i = cluster_id; i < total_tiles && ok; i += n_clusters, ++it) {
                const Tile t = tiles.tile(p, i, half);
                const int buf = it & (p.bufs - 1);
                const uint32_t idesc = umma_instr_desc(t.n, F16);
                ok = mbar_wait(acc_empty(buf), ((uint32_t)(it >> (p.bufs - 1)) & 1u) ^ 1u);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                uint32_t d_tmem = tmem_base + (uint32_t)(buf * p.acc_cols);
                const uint32_t d_rest = d_tmem + (uint32_t)(segments * p.bn);
                int of_segment = 0;
                for (int c = c0; c < c1 && ok; ++c) {
                    ok = mbar_wait(a_full(a.stage), a.phase);
                    if (!ok) break;
                    const int atoms = min(p.n_atoms - 2 * c, 2);
                    for (int j = 0; j < atoms; ++j) {
                        ok = mbar_wait(b_full(b.stage), b.phase);
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        if (elect_one()) {
                            const uint64_t bd = umma_desc_k(base + b_off + (uint32_t)b.stage * b_stage_bytes);
                            const uint64_t ad = umma_desc_k(base + (uint32_t)a.stage * A_CHUNK_BYTES + (uint32_t)j * A_ATOM_BYTES);
#pragma unroll
                            for (int k = 0; k < BK / 16; ++k)
                                umma_pair(d_tmem, ad + (uint64_t)(2 * k), bd + (uint64_t)(2 * k), idesc, (PLANES == 3 ? of_segment > 0 : c > c0) || j > 0 || k > 0 ? 1u : 0u);
                            if constexpr (PLANES == 3)
#pragma unroll
                                for (int pl = 1; pl < 3; ++pl) {
                                    const uint64_t bp = bd + (uint64_t)((uint32_t)(pl * (t.n / 2)) * (BK * 2) >> 4);
#pragma unroll
                                    for (int k = 0; k < BK / 16; ++k)
                                        umma_pair(d_rest, ad + (uint64_t)(2 * k), bp + (uint64_t)(2 * k), idesc, c > c0 || j > 0 || pl > 1 || k > 0 ? 1u : 0u);
                                }
                            umma_commit_pair(b_empty(b.stage), pair_mask);
                        }
                        __syncwarp();
                        b.advance(p.b_stages);
                    }
                    if (!ok) break;
                    if (elect_one()) umma_commit_pair(a_empty(a.stage), pair_mask);
                    __syncwarp();
                    a.advance(A_STAGES);
                    if (PLANES == 3 && ++of_segment == p.seg_chunks) {
                        of_segment = 0;
                        d_tmem += (uint32_t)p.bn;
                    }
                }
                if (ok && elect_one()) umma_commit_pair(acc_full(buf), pair_mask);
                __syncwarp();
            }
            if (!ok) give_up(&g_q4_status, STATUS_MMA);
        }
    } else if (warp < CONVERTER_WARP0) {
        // ---------------- epilogue of all but one-tile launches, which are finished below ----------------
        const int quarter = warp & 3;
        CT *stage = reinterpret_cast<CT *>(gen_base + out_off) + quarter * 1024;
        bool ok = true;
        int it = 0;
        for (int i = cluster_id; i < total_tiles && ok; i += n_clusters, ++it) {
            const Tile t = tiles.tile(p, i, half);
            const int buf = it & (p.bufs - 1), r = quarter * 32 + lane;
            const float factor = p.one_tile ? 1.0f : factor_of(t, r), bias = p.one_tile ? 0.0f : bias_of(t, r);
            ok = epilogue_all(mbar_wait(acc_full(buf), (uint32_t)(it >> (p.bufs - 1)) & 1u));
            if (!ok || p.one_tile) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
            for (int b = 0; b < t.n / 32; ++b) {
                uint32_t v[32];
                load_sums<PLANES>(p, tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * p.acc_cols + b * 32), segments, v);
                emit<CT>(p, v, t.row0 + quarter * 32, lane, factor, bias, t.tok + b * 32, t.end, stage);
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive_leader(acc_empty(buf));
        }
        if (!ok) give_up(&g_q4_status, STATUS_EPILOGUE);
    } else {
        // ---------------- converters: 16 rows of a chunk each, the two groups take the chunks of the CTA's sequence in turn ----------------
        const int cw = (warp - CONVERTER_WARP0) & 7, group = (warp - CONVERTER_WARP0) >> 3, g = lane >> 2, t4 = lane & 3;
        const uint32_t swap = (uint32_t)(g & 1);  // lanes of odd rows store their second 32 columns first: eight lanes cover all banks
        uint32_t off[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) off[s] = (uint32_t)(cw * 16 + g) * 128u + (uint32_t)((4 * (s ^ (int)swap) + t4) ^ g) * 16u;
        const Q4Decode<T> decode;
        // Slots of the raw ring (an even number) stay with a group.  Those of the operand ring (three) change hands: a group waits for the MMAs of the slot's
        // last chunk, k - 3.  It has seen those of k - 5 end when it took its own last chunk, and MMAs end in order, so those of k - 6, the
        // slot's use before, have ended too, and the wait cannot be a whole use behind.
        Ring a, raw;
        if (group == 1) { a.advance(A_STAGES); raw.advance(p.raw_stages); }
        bool ok = true;
        float shrink[2] = {1.0f, 1.0f};
        // the smallest scales of the lane's two rows in a tile, bf16 bits plus 0x7FFF as signed 16-bit numbers: zeros are the largest
        constexpr uint32_t kNone = 0x7FFF7FFFu, kOne = 0x7F000000u + (kF16Up << 23);
        uint32_t least = kNone;
        auto look = [&]() {
#pragma unroll
            for (int r = 0; r < 2; ++r)
                if (f16_loses((((least >> (16 * r)) & 0xFFFFu) - 0x7FFFu) & 0xFFFFu, kOne - __float_as_uint(shrink[r]))) *losses = 1;
            least = kNone;
        };
        // the chunks of this CTA's tiles; `c`: of the tile's, where its rows' powers of two matter
        const int span = c1 - c0;
        int c = group, i = cluster_id;
        bool fresh = true;
        for (int left = (cluster_id < total_tiles ? (total_tiles - 1 - cluster_id) / n_clusters + 1 : 0) * span - group; left > 0; left -= 2) {
            if constexpr (F16) {
                for (; c >= span; c -= span, i += n_clusters) fresh = true;
                if (fresh) {
                    look();
                    const Tile t = tiles.tile(p, i, half);
                    const int64_t tile = (int64_t)t.expert * p.row_tiles + (t.row0 >> 4) + cw;
#pragma unroll
                    for (int r = 0; r < 2; ++r)
                        shrink[r] = t.row0 + cw * 16 < p.M ? __uint_as_float(kOne - row_exponent(p.scales, tile, p.groups, g + 8 * r)) : 0x1p100f;  // 2^(kF16Up - e); rows past M lose nothing
                    fresh = false;
                }
                c += 2;
            }
            ok = __all_sync(0xffffffffu, mbar_wait(raw_full(raw.stage), raw.phase));
            if (!ok) break;
            const uint8_t *src = gen_base + raw_off + raw.stage * RAW_BYTES;
            uint4 q[2];
            uint32_t s[PER];
#pragma unroll
            for (int k = 0; k < 2; ++k) q[k] = *reinterpret_cast<const uint4 *>(src + cw * 1024 + k * 512 + lane * 16);
#pragma unroll
            for (int u = 0; u < PER; ++u) s[u] = *reinterpret_cast<const uint32_t *>(src + RAW_CODES + (cw * PER + u) * 32 + g * 4);
            if constexpr (F16)
#pragma unroll
                for (int u = 0; u < PER; ++u) least = __vmins2(least, (s[u] & 0x7FFF7FFFu) + 0x7FFF7FFFu);
            // a row's scale twice in a word, and -24 times it
            uint32_t s2[2][PER], n2[2][PER];
#pragma unroll
            for (int u = 0; u < PER; ++u)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    if constexpr (F16) {
                        const __half h = __float2half_rn(__uint_as_float(r ? s[u] & 0xFFFF0000u : s[u] << 16) * shrink[r]);
                        const __half2 hh(h, h), nn = __hmul2(hh, __half2(__float2half_rn(-24.0f), __float2half_rn(-24.0f)));
                        s2[r][u] = *reinterpret_cast<const uint32_t *>(&hh);
                        n2[r][u] = *reinterpret_cast<const uint32_t *>(&nn);
                    } else {
                        s2[r][u] = __byte_perm(s[u], s[u], r ? 0x3232 : 0x1010);
                        n2[r][u] = fma_bf16x2(s2[r][u], 0xC1C0C1C0u, 0x80008000u);
                    }
                }
            ok = __all_sync(0xffffffffu, mbar_wait(a_empty(a.stage), a.phase ^ 1));
            if (!ok) break;
            uint8_t *dst = gen_base + a.stage * A_CHUNK_BYTES;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t w[4] = {swap ? q[k].z : q[k].x, swap ? q[k].w : q[k].y, swap ? q[k].x : q[k].z, swap ? q[k].y : q[k].w};
#pragma unroll
                for (int h = 0; h < 2; ++h)  // the lane's first and second half to be stored
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        uint32_t sc, nc;
                        if constexpr (GROUP == 32) {
                            sc = swap ? s2[r][2 * k + 1 - h] : s2[r][2 * k + h];
                            nc = swap ? n2[r][2 * k + 1 - h] : n2[r][2 * k + h];
                        } else {
                            sc = s2[r][GROUP == 64 ? k : 0];
                            nc = n2[r][GROUP == 64 ? k : 0];
                        }
                        uint32_t o[4];
#pragma unroll
                        for (int j = 0; j < 2; ++j)
#pragma unroll
                            for (int pr = 0; pr < 2; ++pr) {
                                const uint32_t x = w[2 * h + j];
                                const uint32_t v = r == 0 ? (pr == 0 ? decode.template biased<0>(x) : decode.template biased<2>(x))
                                                          : (pr == 0 ? decode.template biased<1>(x) : decode.template biased<3>(x));
                                o[2 * j + pr] = Q4Decode<T>::scaled(v, sc, nc);
                            }
                        *reinterpret_cast<uint4 *>(dst + k * A_ATOM_BYTES + off[h] + r * 1024) = make_uint4(o[0], o[1], o[2], o[3]);
                    }
            }
            // generic-proxy writes must be visible to the tensor core's async proxy
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            // The codes are handed back only now that they have been used: an arrival overtakes loads of shared memory that are still on their way
            // (16 warps' stores ahead of them), and the next copy overwrote what they were to read.
            if (lane == 0) {
                mbar_arrive_leader(a_full(a.stage));
                mbar_arrive(raw_empty(raw.stage));
            }
            raw.advance(p.raw_stages);
            raw.advance(p.raw_stages);
            a.advance(A_STAGES);
            a.advance(A_STAGES);
        }
        if constexpr (F16) look();
        if (!ok) give_up(&g_q4_status, STATUS_CONVERTER);
    }
    __syncwarp();

    if (p.one_tile) {
        // Groups of four warps take the tile's 32-row blocks in turn; what they stage goes into the activation ring, idle by now.  With
        // splits > 1 block b is finished by slice b % splits, the others write theirs into its shared memory first (the weight ring).
        const int group = (warp - EPILOGUE_WARP0) >> 2, quarter = warp & 3, S = p.splits, blocks = p.bn / 32;
        const bool worker = warp >= EPILOGUE_WARP0 && warp < RAW_WARP;
        const Tile t = tiles.tile(p, cluster_id, half);
        const uint32_t r = (uint32_t)(quarter * 32 + lane);
        const uint32_t t_lane = tmem_base + ((uint32_t)(quarter * 32) << 16);
        const float factor = factor_of(t, (int)r), bias = bias_of(t, (int)r);
        __syncthreads();
        if (S > 1) cluster_barrier();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (S > 1) {
            if (worker)
                for (int b = group; b < blocks; b += FINISHERS) {
                    const int to = b % S;
                    if (to == slice) continue;
                    uint32_t v[32];
                    load_sums<PLANES>(p, t_lane + (uint32_t)(b * 32), segments, v);
                    push_partial(v, base + partial_slot(b, S, slice, to) * 16384u + r * 4u, (uint32_t)(2 * to + half));
                }
            __syncthreads();
            cluster_barrier();
        }
        if (worker) {
            CT *stage = reinterpret_cast<CT *>(gen_base + b_off) + (group * 4 + quarter) * 1024;
            for (int b = slice + S * group; b < blocks; b += FINISHERS * S) {
                uint32_t v[32];
                load_sums<PLANES>(p, t_lane + (uint32_t)(b * 32), segments, v);
                if (S > 1) fold_partials(v, gen_base, b, S, slice, r);
                emit<CT>(p, v, t.row0 + quarter * 32, lane, factor, bias, t.tok + b * 32, t.end, stage);
            }
        }
    }
    // ---------------- teardown: no CTA leaves while its peer may still arrive on its barriers or read its operands ----------------
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_barrier();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        tmem_free_pair(tmem_base);
    }
    if constexpr (F16)
        if (*losses) {  // the cluster's results are written: those of rows that fp16 does not hold are written again
            // Two forms, because the registers that the call leaves to the rest of the kernel differ (us, without such rows, loop here and there: 32 experts of 2048 x
            // 4096, 2048 tokens 135 and 131; 4096 x 14336, 64 rows 27.6 and 28.1).
            if constexpr (EXPERTS) mend_experts<CT>(p);
            else
                for (int i = cluster_id; i < total_tiles; i += n_clusters) {
                    const Tile t = tiles.tile(p, i, half);
                    mend_rows<CT>(p, reinterpret_cast<float (*)[MEND_TOK][17]>(gen_base + 16), reinterpret_cast<uint32_t *>(gen_base), 0, t.row0, t.tok, t.end);
                }
        }
}

// Time of a 64-deep step at n columns, in ns: 18944 rows of 8192 columns (4096 for wide tiles of three planes), one tile a pair, 34 to 256 rows of
// x, without 5.5 us.
double step_cost(int n, int planes) {
    constexpr double one[9] = {235, 235, 236, 252, 259, 279, 297, 349, 375}, three[5] = {300, 300, 331, 417, 533};  // 0, 32, .. columns
    return planes == 3 ? three[n / 32] : one[n / 32];
}

// Three planes: chunks that an accumulator takes (2048 columns), and the widest tile whose accumulators TMEM holds: one per 2048 columns and one
// for the other planes.  (Beyond 30720 columns an accumulator takes more of them.)
constexpr int SEGMENT = 2048 / CHUNK;
int segments_of(int64_t K) {
    const int64_t n = (K + SEGMENT * CHUNK - 1) / (SEGMENT * CHUNK);
    return n < 1 ? 1 : (n > 15 ? 15 : (int)n);
}
int widest_of_planes(int64_t K) {
    const int s = segments_of(K);
    return s <= 3 ? 128 : (s <= 7 ? 64 : 32);
}

// Tile width and split of one matrix: the smallest estimate, in ns without the launch.
struct Shape {
    int bn = 0, n_tiles = 0, splits = 1;
    double ns = 1e30;
};
Shape pick_shape(int64_t M, int64_t N, int64_t K, int planes) {
    const int64_t m_tiles = (M + 255) / 256, chunks = (K + CHUNK - 1) / CHUNK, most = planes == 3 ? widest_of_planes(K) : 256, least = (N + most - 1) / most;
    Shape best;
    for (int64_t want = least; want <= least + 8 && want <= (N + 31) / 32; ++want) {
        const int bn = (int)(((N + want - 1) / want + 31) / 32 * 32);
        const int64_t n_tiles = (N + bn - 1) / bn, tiles = m_tiles * n_tiles;
        for (int s = 1; s <= MAX_SPLITS; ++s) {
            const int fit = resident_pair_clusters(s);
            if (s > chunks || (s > 1 && tiles > fit)) continue;
            const double ns = (double)((tiles + fit - 1) / fit) * (2.0 * (double)((chunks + s - 1) / s) * step_cost(bn, planes) + 700.0) + 5.0 * bn + (s > 1 ? 2200.0 + 5.0 * bn : 0.0);
            if (ns < best.ns) best = {bn, (int)n_tiles, s, ns};
        }
    }
    return best;
}

template <typename T, int PLANES, int GROUP, typename CT, bool EXPERTS>
int launch(const CUtensorMap &mc, const CUtensorMap &ms, const XMaps &mx, const Q4TcParams &p, int clusters, size_t smem, cudaStream_t st) {
    auto kern = gemm_q4_tc_kernel<T, PLANES, GROUP, CT, EXPERTS>;
    constexpr int most = SMEM_LIMIT;
    static std::atomic<bool> configured[64];
    int dev = 0;
    T81_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
        T81_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
        if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(clusters * 2 * p.splits));
    cfg.blockDim = dim3(NUM_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)(2 * p.splits);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    T81_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, mc, ms, mx, p));
    return T81B200_OK;
}

}  // namespace

int gemm_q4_tc_status(int reset) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_q4_status, sizeof v) != cudaSuccess) return T81B200_ECUDA;
    if (reset && v != 0) {
        const int zero = 0;
        if (cudaMemcpyToSymbol(g_q4_status, &zero, sizeof zero) != cudaSuccess) return T81B200_ECUDA;
    }
    return v;
}

// Time of a launch, for the choice between this and the streaming kernel.  Experts: of the number that N rows reach of a router without
// preferences, each with its share of the rows.
double gemm_q4_tc_estimate_us(int64_t M, int64_t N, int64_t K, int planes, int n_experts, double reached) {
    if (n_experts == 0) return 4.5 + 1e-3 * pick_shape(M, N, K, planes).ns;
    const double most = planes == 3 ? widest_of_planes(K) : 256;
    const double rows = (double)N / reached, tiles = reached * (double)((M + 255) / 256) * ceil(rows / most), fit = resident_pair_clusters(1);
    const int n = rows >= most ? (int)most : ((int)rows + 31) / 32 * 32;
    return 5.0 + 1e-3 * ceil(tiles / fit) * (2.0 * (double)((K + CHUNK - 1) / CHUNK) * step_cost(n, planes) + 700.0);
}

// x: 16-bit rows on 16-byte boundaries, K columns of them, N rows; with three planes three times N.  Arguments are checked by
// the caller.
int gemm_q4_tc_launch(const uint8_t *codes, const void *scales, const float *bias, void *C, int64_t M, const void *x, bool f16, int planes, int64_t ldx, int c_dtype, int64_t ldc, int64_t N,
                      int64_t K, int group, const int32_t *offsets, int n_experts, cudaStream_t st) {
    Q4TcParams p;
    memset(&p, 0, sizeof p);
    const int experts = offsets ? n_experts : 1;
    p.scales = static_cast<const __nv_bfloat16 *>(scales); p.bias = bias; p.C = C; p.offsets = offsets; p.ldc = ldc;
    p.M = (int)M; p.N = (int)N; p.n_experts = experts;
    p.row_tiles = (int)q4_row_tiles(M); p.groups = (int)q4_groups(K, group);
    p.codes = codes; p.x = x; p.ldx = ldx; p.K = (int)K; p.group = group;
    p.m_tiles = (int)((M + 255) / 256);
    p.n_atoms = (int)((K + BK - 1) / BK); p.n_chunks = (int)((K + CHUNK - 1) / CHUNK);
    p.splits = 1;
    p.vec = reinterpret_cast<uintptr_t>(C) % 16 == 0 && ldc * (int64_t)dtype_size(c_dtype) % 16 == 0;
    const int resident = resident_pair_clusters(1);
    int clusters;
    if (offsets) {
        // rows of an expert go evenly into tiles of at most 256
        p.bn = planes == 3 ? widest_of_planes(K) : 256;
        const int64_t most = (N / p.bn + (N < experts ? N : experts)) * p.m_tiles;
        clusters = (int)(most < resident ? (most < 1 ? 1 : most) : resident);
    } else {
        const Shape shape = pick_shape(M, N, K, planes);
        p.bn = shape.bn; p.n_tiles = shape.n_tiles; p.splits = shape.splits;
        const int tiles = p.m_tiles * p.n_tiles;
        p.one_tile = p.splits > 1 || tiles <= resident ? 1 : 0;
        clusters = p.one_tile ? tiles : resident;
    }
    p.out_bytes = p.one_tile ? 0 : 4 * 1024 * (int)dtype_size(c_dtype);
    p.list_bytes = offsets ? ExpertList::bytes(experts) : 0;
    // Two stages of codes for either group of converters, the rest for the activations (us with four, six and eight of codes: 14336 x 4096, 2048
    // tokens 153.9, 155.9, 162.9, 37 experts of 2048 x 4096 with 256 rows each 118.5, 118.8, 129.5); four where activations are narrow (18944 x
    // 8192, 64 tokens 38.1 and 35.7, 4096 x 14336 28.5 and 26.3).
    const int raw = RAW_CODES + CHUNK / group * 256, stage = planes * p.bn * BK;
    const int room = SMEM_LIMIT - A_STAGES * A_CHUNK_BYTES - p.out_bytes - BARRIER_BYTES - p.list_bytes - 1024;
    p.raw_stages = planes * p.bn <= 128 ? RAW_MAX : 4;
    p.b_stages = (room - p.raw_stages * raw) / stage;
    p.b_stages = p.b_stages > B_MAX ? B_MAX : p.b_stages;
    const size_t smem = (size_t)(SMEM_LIMIT - room) + (size_t)p.raw_stages * raw + (size_t)p.b_stages * stage;
    CUtensorMap mc, ms;
    XMaps mx;
    memset(&mx, 0, sizeof mx);
    const int64_t tiles16 = (int64_t)experts * p.row_tiles, ktiles = q4_col_tiles(K);
    if (int rc = make_map_2d(&mc, CU_TENSOR_MAP_DATA_TYPE_UINT32, codes, (uint64_t)ktiles * 128, (uint64_t)tiles16, (uint64_t)ktiles * kQ4TileBytes, 256, 8, CU_TENSOR_MAP_SWIZZLE_NONE)) return rc;
    if (int rc = make_map_2d(&ms, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, scales, (uint64_t)(p.groups + 1) * 16, (uint64_t)tiles16, (uint64_t)(p.groups + 1) * 32, (uint32_t)(CHUNK / group) * 16, 8,
                             CU_TENSOR_MAP_SWIZZLE_NONE))
        return rc;
    for (int k = 0; k < (offsets ? 4 : 1); ++k)
        if (int rc = make_map_2d(&mx.m[k], f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, x, (uint64_t)K, (uint64_t)(planes * N), (uint64_t)ldx * 2, BK,
                                 (uint32_t)(offsets ? 128 >> k : p.bn / 2), CU_TENSOR_MAP_SWIZZLE_128B))
            return rc;
    p.bufs = 2;
    p.acc_cols = 256;
    if (planes == 3) {
        const int share = (p.n_chunks + p.splits - 1) / p.splits, segments = segments_of((int64_t)share * CHUNK);
        p.seg_chunks = (share + segments - 1) / segments;
        p.acc_cols = (segments + 1) * p.bn;
        p.bufs = 2 * p.acc_cols <= (int)kTmemCols ? 2 : 1;
    }
    auto go = [&](auto t, auto pl, auto g, auto ct, auto e) {
        return launch<decltype(t), decltype(pl)::value, decltype(g)::value, decltype(ct), decltype(e)::value>(mc, ms, mx, p, clusters, smem, st);
    };
    using One = std::integral_constant<int, 1>;
    auto by_experts = [&](auto t, auto pl, auto g, auto ct) { return offsets ? go(t, pl, g, ct, std::true_type{}) : go(t, pl, g, ct, std::false_type{}); };
    auto by_out = [&](auto t, auto g) {
        auto by_planes = [&](auto ct) {
            if constexpr (std::is_same<decltype(t), __nv_bfloat16>::value)
                if (planes == 3) return by_experts(t, std::integral_constant<int, 3>{}, g, ct);
            return by_experts(t, One{}, g, ct);
        };
        switch (c_dtype) {
            case T81B200_F32: return by_planes(float{});
            case T81B200_BF16: return by_planes(__nv_bfloat16{});
            default: return by_planes(__half{});
        }
    };
    auto by_group = [&](auto t) {
        if (group == 32) return by_out(t, std::integral_constant<int, 32>{});
        if (group == 64) return by_out(t, std::integral_constant<int, 64>{});
        return by_out(t, std::integral_constant<int, 128>{});
    };
    return f16 ? by_group(__half{}) : by_group(__nv_bfloat16{});
}

}  // namespace t81b200
