// Products of 4-bit weights (q4.cuh) for few activation rows: y[t][o] = sum_k x[t][k] code[o][k] scale[o][k / group] (+ bias[o]).
//
// Bound by reading the weights (half a byte each and two bytes a group).  A warp streams 16-row tiles: a lane's 16 bytes of a tile are the
// A fragments of four mma.sync m16n8k16, the codes as exact numbers -8 .. 7, and its eight columns of an activation row are the B
// fragments of two of them, read where the row lies (L1 holds the few rows that a CTA's warps share; weights pass it by).  Sums of a
// group are scaled and added in fp32.  The warps of a CTA take units of 128 columns in turn and their sums meet in shared memory, in
// warp order: results do not depend on the schedule.
//
// float32 activations come as three bf16 planes (all 24 bits, stage_planes), each multiplied exactly; the first has sums of its own, since the
// tensor core cuts small terms beside large ones off.
//
// The same kernel multiplies rows sorted by expert (`offsets`): a block finds the expert of its number among those that have rows and
// takes that expert's rows; the blocks of the last number write zeros to rows behind the last expert's.
#include "common.cuh"
#include "launch_order.cuh"
#include "q4.cuh"
#include "tma.cuh"
#include "umma.cuh"

namespace t81b200 {

// gemm_q4_tc.cu
int gemm_q4_tc_launch(const uint8_t *codes, const void *scales, const float *bias, void *C, int64_t M, const void *x, bool f16, int64_t ldx, int c_dtype, int64_t ldc, int64_t N,
                      int64_t K, int group, const int32_t *offsets, int n_experts, cudaStream_t st);

namespace {

struct Q4Params {
    const uint8_t *codes;
    const __nv_bfloat16 *scales;
    const float *bias;
    const void *x;
    void *y;
    int64_t ldx, ldy, plane_elems;  // elements
    int64_t M, K, kx;               // kx: columns of x that may be read, a multiple of 8 (zeros past K)
    int64_t rows;                   // of x
    int64_t code_stride, scale_stride, bias_stride;  // from one expert to the next
    const int32_t *offsets;         // n_experts + 1, or null: one matrix for all rows
    int n_experts;
    int col_tiles, groups, units;
};

template <typename T> __device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma_16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Weights are read once: past L1.
__device__ __forceinline__ uint4 load_codes(const uint8_t *p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t load_scales(const void *p) {
    uint32_t v;
    asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}

template <typename T>
__device__ __forceinline__ void fragments(uint32_t w, uint32_t (&a)[4]) {
    a[0] = Q4Decode<T>::minus24(Q4Decode<T>::template biased<0>(w));
    a[1] = Q4Decode<T>::minus24(Q4Decode<T>::template biased<1>(w));
    a[2] = Q4Decode<T>::minus24(Q4Decode<T>::template biased<2>(w));
    a[3] = Q4Decode<T>::minus24(Q4Decode<T>::template biased<3>(w));
}

// T: type of the operands; PLANES: 1, or 3 of float32 activations; RT: row tiles a warp; NT: blocks of 8 rows of x at a time.
template <typename T, int PLANES, int RT, int NT, int GROUP, typename CT>
__global__ void __launch_bounds__(512) gemv_q4_kernel(const __grid_constant__ Q4Params p) {
    extern __shared__ float part[];  // [warps][RT * 16 rows][8 NT rows of x]
    constexpr int PER = 128 / GROUP, SUMS = PLANES == 1 ? 1 : 2, TOK = 8 * NT;
    wait_for_kernel_ahead();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5, g = lane >> 2, t = lane & 3;
    const int64_t tile0 = (int64_t)blockIdx.x * RT, row_tiles = (p.M + 15) >> 4;
    int64_t first = 0, end = p.rows;
    int expert = 0;
    if (p.offsets) {
        // this block's expert: number blockIdx.y of those with rows
        __shared__ int found[3];
        if (warp == 0) {
            int seen = 0, expert_here = -1;
            for (int e0 = 0; e0 < p.n_experts; e0 += 32) {
                const int e = e0 + lane;
                const bool some = e < p.n_experts && p.offsets[e + 1] > p.offsets[e];
                const uint32_t ballot = __ballot_sync(0xffffffffu, some);
                const int n = __popc(ballot);
                if (seen + n > (int)blockIdx.y) {
                    const int nth = (int)__fns(ballot, 0, (int)blockIdx.y - seen + 1);
                    expert_here = e0 + nth;
                    break;
                }
                seen += n;
            }
            if (lane == 0) {
                found[0] = expert_here;
                if (expert_here >= 0) {
                    found[1] = p.offsets[expert_here];
                    found[2] = p.offsets[expert_here + 1];
                }
            }
        }
        __syncthreads();
        expert = found[0];
        if (blockIdx.y == gridDim.y - 1) {  // rows of no expert
            const int64_t kept = p.offsets[p.n_experts] > 0 ? p.offsets[p.n_experts] : 0;
            for (int64_t i = threadIdx.x; i < (p.rows - kept) * (RT * 16); i += blockDim.x) {
                const int64_t row = tile0 * 16 + i % (RT * 16), tok = kept + i / (RT * 16);
                if (row < p.M) static_cast<CT *>(p.y)[tok * p.ldy + row] = from_float<CT>(0.0f);
            }
            return;
        }
        if (expert < 0) return;
        first = found[1] > 0 ? found[1] : 0;
        end = found[2] < p.rows ? found[2] : p.rows;  // whatever the offsets say, nothing lies outside the rows
    }
    const uint8_t *codes = p.codes + expert * p.code_stride;
    const __nv_bfloat16 *scales = p.scales + expert * p.scale_stride;
    const T *x = static_cast<const T *>(p.x);

    for (int64_t tok0 = first + (int64_t)blockIdx.z * TOK; tok0 < end; tok0 += (int64_t)gridDim.z * TOK) {
        float sum[RT][NT][SUMS][4] = {};
        auto read = [&](int unit, uint4 (&q)[RT][2], uint32_t (&s)[RT][PER]) {
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const bool there = tile0 + r < row_tiles && unit < p.units;
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    q[r][c] = there && 2 * unit + c < p.col_tiles ? load_codes(codes + ((tile0 + r) * p.col_tiles + 2 * unit + c) * kQ4TileBytes + lane * 16) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
                for (int i = 0; i < PER; ++i)
                    s[r][i] = there && unit * PER + i < p.groups ? load_scales(scales + ((tile0 + r) * (p.groups + 1) + unit * PER + i) * 16 + 2 * g) : 0u;
            }
        };
        uint4 q[RT][2], q_next[RT][2];
        uint32_t s[RT][PER], s_next[RT][PER];
        read(warp, q_next, s_next);
        for (int unit = warp; unit < p.units; unit += warps) {
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                q[r][0] = q_next[r][0];
                q[r][1] = q_next[r][1];
#pragma unroll
                for (int i = 0; i < PER; ++i) s[r][i] = s_next[r][i];
            }
            uint4 b[PLANES][NT][4];  // [.. 32 columns]
#pragma unroll
            for (int pl = 0; pl < PLANES; ++pl)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const int64_t tok = tok0 + 8 * n + g;
                    const T *src = x + pl * p.plane_elems + tok * p.ldx + (int64_t)unit * 128 + 8 * t;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        b[pl][n][i] = tok < end && (int64_t)unit * 128 + 32 * i + 8 * t < p.kx ? __ldg(reinterpret_cast<const uint4 *>(src + 32 * i)) : make_uint4(0u, 0u, 0u, 0u);
                }
            read(unit + warps, q_next, s_next);
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const uint32_t word[8] = {q[r][0].x, q[r][0].y, q[r][0].z, q[r][0].w, q[r][1].x, q[r][1].y, q[r][1].z, q[r][1].w};
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    float c[NT][SUMS][4] = {};
#pragma unroll
                    for (int j = i * (8 / PER); j < (i + 1) * (8 / PER); ++j) {
                        uint32_t a[4];
                        fragments<T>(word[j], a);
#pragma unroll
                        for (int pl = 0; pl < PLANES; ++pl)
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                const uint4 &v = b[pl][n][j >> 1];
                                mma_16816<T>(c[n][pl > 0 ? SUMS - 1 : 0], a, j & 1 ? v.z : v.x, j & 1 ? v.w : v.y);
                            }
                    }
                    const float lo = __uint_as_float(s[r][i] << 16), hi = __uint_as_float(s[r][i] & 0xFFFF0000u);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int u = 0; u < SUMS; ++u) {
                            sum[r][n][u][0] = fmaf(c[n][u][0], lo, sum[r][n][u][0]);
                            sum[r][n][u][1] = fmaf(c[n][u][1], lo, sum[r][n][u][1]);
                            sum[r][n][u][2] = fmaf(c[n][u][2], hi, sum[r][n][u][2]);
                            sum[r][n][u][3] = fmaf(c[n][u][3], hi, sum[r][n][u][3]);
                        }
                }
            }
        }
        // part[warp][row of x][row of the tiles]
        constexpr int WIDTH = RT * 16 + 1;
        if (tok0 != first + (int64_t)blockIdx.z * TOK) __syncthreads();
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
        for (int i = threadIdx.x; i < TOK * RT * 16; i += blockDim.x) {
            const int tok = i / (RT * 16), r = i % (RT * 16);
            const int64_t row = tile0 * 16 + r;
            if (tok0 + tok >= end || row >= p.M) continue;
            float v = 0.0f;
            for (int w = 0; w < warps; ++w) v += part[(w * TOK + tok) * WIDTH + r];
            if (p.bias) v += p.bias[expert * p.bias_stride + row];
            static_cast<CT *>(p.y)[(tok0 + tok) * p.ldy + row] = from_float<CT>(v);
        }
    }
}

template <typename T, int PLANES, int RT, int NT, int GROUP, typename CT>
int launch(const Q4Params &p, int warps, cudaStream_t st) {
    const int64_t blocks = (((p.M + 15) / 16) + RT - 1) / RT, passes = (p.rows + 8 * NT - 1) / (8 * NT);
    const dim3 grid((unsigned)blocks, p.offsets ? (unsigned)((p.rows < p.n_experts ? p.rows : p.n_experts) + 1) : 1u, p.offsets ? 1u : (unsigned)(passes < 65535 ? passes : 65535));
    const size_t smem = (size_t)warps * 8 * NT * (RT * 16 + 1) * sizeof(float);
    auto kernel = gemv_q4_kernel<T, PLANES, RT, NT, GROUP, CT>;
    if (smem > 48 * 1024) T81_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    T81_CUDA_TRY(launch_behind(kernel, grid, dim3(warps * 32), smem, st, p));
    return T81B200_OK;
}

template <typename T, int PLANES, int RT, int NT, int GROUP>
int launch_ct(const Q4Params &p, int c_dtype, int warps, cudaStream_t st) {
    switch (c_dtype) {
        case T81B200_F32: return launch<T, PLANES, RT, NT, GROUP, float>(p, warps, st);
        case T81B200_BF16: return launch<T, PLANES, RT, NT, GROUP, __nv_bfloat16>(p, warps, st);
        case T81B200_F16: return launch<T, PLANES, RT, NT, GROUP, __half>(p, warps, st);
    }
    return fail(T81B200_EINVAL, "linear_q4: unknown output dtype %d", c_dtype);
}

template <typename T, int PLANES, int RT, int NT>
int launch_group(const Q4Params &p, int group, int c_dtype, int warps, cudaStream_t st) {
    if (group == 32) return launch_ct<T, PLANES, RT, NT, 32>(p, c_dtype, warps, st);
    if (group == 64) return launch_ct<T, PLANES, RT, NT, 64>(p, c_dtype, warps, st);
    return launch_ct<T, PLANES, RT, NT, 128>(p, c_dtype, warps, st);
}

template <typename T, int PLANES>
int launch_shape(const Q4Params &p, int group, int c_dtype, cudaStream_t st) {
    const int warps = p.units >= 16 ? 16 : (p.units >= 8 ? 8 : 4);
    if constexpr (PLANES == 1)
        if (p.rows > 8) return launch_group<T, PLANES, 1, 2>(p, group, c_dtype, warps, st);
    return launch_group<T, PLANES, 1, 1>(p, group, c_dtype, warps, st);  // three planes of 16 rows do not fit the registers
}

// Rows that the kernels read where they are: 16-bit, on 16-byte boundaries, whole pieces of eight columns.
bool in_place(const void *B, int b_dtype, int64_t ldb, int64_t K) {
    return b_dtype != T81B200_F32 && reinterpret_cast<uintptr_t>(B) % 16 == 0 && ldb % 8 == 0 && K % 8 == 0;
}
int64_t staged_row(int64_t K) { return (K + 7) & ~(int64_t)7; }

int product_q4(const char *name, const uint8_t *codes, const void *scales, const float *bias, void *C, int64_t M, const void *B, int b_dtype, int64_t ldb, int c_dtype, int64_t ldc,
               int64_t N, int64_t K, int group, const int32_t *offsets, int n_experts, void *workspace, size_t workspace_bytes, cudaStream_t st) {
    if (M < 0 || N < 0 || K < 0 || ldb < K || ldc < M || n_experts < 0) return fail(T81B200_EINVAL, "%s: bad dimensions", name);
    if (!q4_group_ok(group)) return fail(T81B200_EINVAL, "%s: groups of 32, 64 or 128 columns, not %d", name, group);
    if (dtype_size(b_dtype) == 0 || b_dtype < 0 || b_dtype > T81B200_F16 || c_dtype < 0 || c_dtype > T81B200_F16) return fail(T81B200_EINVAL, "%s: unknown dtype", name);
    if (M >= (1ll << 31) || N >= (1ll << 31) || K >= (1ll << 31) || n_experts > 65534) return fail(T81B200_ELIMIT, "%s: dimension too large", name);
    if (int rc = check_device()) return rc;
    if (M == 0 || N == 0) return T81B200_OK;
    if (!C || (K > 0 && (!B || !codes || !scales))) return fail(T81B200_EINVAL, "%s: null pointer", name);
    if (reinterpret_cast<uintptr_t>(codes) % 16 != 0 || reinterpret_cast<uintptr_t>(scales) % 16 != 0) return fail(T81B200_EALIGN, "%s: codes and scales must be 16-byte aligned", name);
    Q4Params p = {};
    p.codes = codes; p.scales = static_cast<const __nv_bfloat16 *>(scales); p.bias = bias;
    p.x = B; p.ldx = ldb; p.kx = K;
    p.y = C; p.ldy = ldc;
    p.M = M; p.K = K; p.rows = N;
    p.offsets = offsets; p.n_experts = n_experts;
    p.code_stride = t81b200_q4_bytes(M, K); p.scale_stride = t81b200_q4_scales(M, K, group); p.bias_stride = M;
    p.col_tiles = (int)q4_col_tiles(K); p.groups = (int)q4_groups(K, group); p.units = (int)((K + 127) / 128);
    if (K > 0 && !in_place(B, b_dtype, ldb, K)) {
        const size_t need = (size_t)(b_dtype == T81B200_F32 ? 3 : 1) * N * staged_row(K) * 2;
        if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
            return fail(T81B200_EWORKSPACE, "%s: %zu bytes of 16-byte aligned workspace needed, %zu given", name, need, workspace_bytes);
        if (int rc = stage_planes(B, b_dtype, T81B200_LAYOUT_NK, ldb, N, K, 3, workspace, st)) return rc;
        p.x = workspace;
        p.ldx = p.kx = staged_row(K);
        p.plane_elems = N * p.ldx;
    }
    if (b_dtype != T81B200_F32 && K > 0 && n_experts <= 1024 && N >= (offsets ? 8 * (int64_t)n_experts : 33))
        return gemm_q4_tc_launch(codes, scales, bias, C, M, p.x, b_dtype == T81B200_F16, p.ldx, c_dtype, ldc, N, K, group, offsets, n_experts, st);
    if (b_dtype == T81B200_F32) return launch_shape<__nv_bfloat16, 3>(p, group, c_dtype, st);
    return b_dtype == T81B200_BF16 ? launch_shape<__nv_bfloat16, 1>(p, group, c_dtype, st) : launch_shape<__half, 1>(p, group, c_dtype, st);
}

}  // namespace
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
