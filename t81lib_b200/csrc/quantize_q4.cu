// Weights to 4-bit codes with group scales, and back (the format: q4.cuh).
//
// Quantise: m = the group's value of largest magnitude (the first of equals), scale s = m / -8 rounded to five significant bits, code =
// the whole number nearest to w / s, ties to even, held in -8 .. 7.  Eight steps reach from 0 to the largest value and seven the
// other way.  Five bits for the scale make code * s a bf16 number, and cost little: N(0, 1) weights in groups of 128 come back with
// a mean square error 0.3 % above that of an unrounded scale.
// The code is exact: w times 1 / s finds it or a neighbour, and the rest w - code * s, which has no rounding error (both are
// multiples of w's last place, and the difference is below s), decides.
//
// Bound by memory: a weight is read once, half a byte is written.  A warp holds 16 rows x 128 columns in registers, a lane eight columns
// of two rows at a time as the format has them: 64 (16-bit) or 128 bytes of a row side by side per load.
#include "common.cuh"
#include "launch_order.cuh"
#include "q4.cuh"

namespace t81b200 {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr float kMost = 8.507059173023462e37f;   // 2^126: larger magnitudes count as this, so that 8 s is finite
constexpr float kLeast = 7.888609052210118e-31f; // 2^-100: a group of smaller ones is zero (s would leave the normal numbers)

// Eight neighbouring elements of a row as fp32; columns at and past `left` are 0.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T *src, int64_t left, float (&v)[8]) {
    if (VEC && left >= 8) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = __ldcs(reinterpret_cast<const float4 *>(src)), b = __ldcs(reinterpret_cast<const float4 *>(src) + 1);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const uint4 a = __ldcs(reinterpret_cast<const uint4 *>(src));
            const T *e = reinterpret_cast<const T *>(&a);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = to_float<T>(e[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < left ? to_float<T>(src[i]) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] != v[i] ? 0.0f : fminf(fmaxf(v[i], -kMost), kMost);  // no number: 0
}

// The group's value of largest magnitude over the four lanes of a row, the first of equals: a lane's columns lie before the next one's.
__device__ __forceinline__ float largest_of_lanes(float m, int t) {
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
        const float o = __shfl_xor_sync(0xffffffffu, m, d);
        const bool other_first = (t & d) != 0;
        if (fabsf(o) > fabsf(m) || (other_first && fabsf(o) == fabsf(m))) m = o;
    }
    return m;
}
__device__ __forceinline__ float larger(float first, float then) { return fabsf(then) > fabsf(first) ? then : first; }

// m / -8 rounded to five significant bits, ties to even.
__device__ __forceinline__ float scale_of(float m) {
    if (fabsf(m) < kLeast) return 0.0f;
    uint32_t b = __float_as_uint(m * -0.125f);
    b += 0x3FFFFu + ((b >> 19) & 1u);
    return __uint_as_float(b & 0xFFF80000u);
}

// code + 8 of w.
__device__ __forceinline__ uint32_t code_of(float w, float s, float inverse) {
    float q = rintf(w * inverse);
    const float half = 0.5f * fabsf(s), rest = copysignf(1.0f, s) * fmaf(-q, s, w);
    const bool odd = (__float2int_rn(q) & 1) != 0;
    if (rest > half || (odd && rest == half)) q += 1.0f;
    else if (rest < -half || (odd && rest == -half)) q -= 1.0f;
    return (uint32_t)(__float2int_rn(fminf(fmaxf(q, -8.0f), 7.0f)) + 8);
}

// A block takes 16 rows, its warps units of 128 columns in turn.
template <typename T, int GROUP, bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_q4_kernel(const T *__restrict__ w, int64_t rows, int64_t cols, int64_t ld, int64_t matrix_stride,
                                                               uint4 *__restrict__ codes, __nv_bfloat16 *__restrict__ scales) {
    __shared__ float most[kWarps][16];
    const int64_t row_tiles = q4_row_tiles(rows), col_tiles = q4_col_tiles(cols), groups = q4_groups(cols, GROUP), units = (cols + 127) / 128;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int64_t matrix = blockIdx.y, T16 = blockIdx.x, out_tile = matrix * row_tiles + T16;
    float largest[2] = {0.0f, 0.0f};  // of the lane's rows
    for (int64_t unit = warp; unit < units; unit += kWarps) {
        float v[2][2][2][8];  // [tile][half of its columns][row of the lane]
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int64_t row = 16 * T16 + g + 8 * r, col = unit * 128 + 64 * c + 32 * half + 8 * t;
                    load8<T, VEC>(w + matrix * matrix_stride + row * ld + col, row < rows ? cols - col : 0, v[c][half][r]);
                }
        float m[2][2][2];
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float x = v[c][half][r][0];
#pragma unroll
                    for (int i = 1; i < 8; ++i) x = larger(x, v[c][half][r][i]);
                    m[c][half][r] = largest_of_lanes(x, t);
                }
        float s[2][2][2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            if (GROUP >= 64)
#pragma unroll
                for (int c = 0; c < 2; ++c) m[c][0][r] = m[c][1][r] = larger(m[c][0][r], m[c][1][r]);
            if (GROUP == 128) m[0][0][r] = m[0][1][r] = m[1][0][r] = m[1][1][r] = larger(m[0][0][r], m[1][0][r]);
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    s[c][half][r] = scale_of(m[c][half][r]);
                    largest[r] = fmaxf(largest[r], fabsf(s[c][half][r]));
                }
        }
        constexpr int PER = 128 / GROUP;  // groups of the 128 columns; lane t == 0 of a row writes them
        if (t == 0) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int64_t u = unit * PER + i;
                if (u >= groups) break;
                const int c = i * GROUP / 64, half = i * GROUP % 64 / 32;
                const __nv_bfloat162 pair(__float2bfloat16_rn(s[c][half][0]), __float2bfloat16_rn(s[c][half][1]));
                *reinterpret_cast<uint32_t *>(scales + (out_tile * (groups + 1) + u) * 16 + 2 * g) = bf162_bits(pair);
            }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            if (unit * 2 + c >= col_tiles) break;
            uint32_t word[4] = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float scale = s[c][half][r], inverse = scale != 0.0f ? 1.0f / scale : 0.0f;
#pragma unroll
                    for (int i = 0; i < 8; ++i)  // column 4 (j % 2) + 2 (register / 2) + h of the lane's eight
                        word[2 * half + (i >> 2)] |= (scale != 0.0f ? code_of(v[c][half][r][i], scale, inverse) : 8u) << (4 * (r + 2 * ((i >> 1) & 1)) + 16 * (i & 1));
                }
            codes[(out_tile * col_tiles + unit * 2 + c) * 32 + lane] = make_uint4(word[0], word[1], word[2], word[3]);
        }
    }
    if (t == 0) {
        most[warp][2 * g] = largest[0];
        most[warp][2 * g + 1] = largest[1];
    }
    __syncthreads();
    if (threadIdx.x < 16) {
        float x = most[0][threadIdx.x];
#pragma unroll
        for (int i = 1; i < kWarps; ++i) x = fmaxf(x, most[i][threadIdx.x]);
        scales[(out_tile * (groups + 1) + groups) * 16 + threadIdx.x] = __float2bfloat16_rn(x);
    }
}

// One warp per tile; every value is exact in fp32 and in bf16.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) dequantize_q4_kernel(const uint4 *__restrict__ codes, const __nv_bfloat16 *__restrict__ scales, int64_t matrices, int64_t rows,
                                                                 int64_t cols, int group, T *__restrict__ out) {
    wait_for_kernel_ahead();
    const int64_t row_tiles = q4_row_tiles(rows), col_tiles = q4_col_tiles(cols), groups = q4_groups(cols, group);
    const int64_t tile = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (tile >= matrices * row_tiles * col_tiles) return;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int64_t c = tile % col_tiles, all_T = tile / col_tiles, matrix = all_T / row_tiles, T16 = all_T % row_tiles;
    const uint4 q = codes[tile * 32 + lane];
    const uint32_t word[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int64_t col = 64 * c + 32 * half + 8 * t;
        if (col >= cols) continue;
        const uint32_t pair = *reinterpret_cast<const uint32_t *>(scales + (all_T * (groups + 1) + col / group) * 16 + 2 * g);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int64_t row = 16 * T16 + g + 8 * r;
            if (row >= rows) continue;
            const float s = __uint_as_float(r ? pair & 0xFFFF0000u : pair << 16);
            T v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                v[i] = from_float<T>((float)((int)((word[2 * half + (i >> 2)] >> (4 * (r + 2 * ((i >> 1) & 1)) + 16 * (i & 1))) & 15u) - 8) * s);
            T *dst = out + (matrix * rows + row) * cols + col;
            if (VEC && col + 8 <= cols) {
#pragma unroll
                for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4 *>(dst)[i] = reinterpret_cast<const uint4 *>(v)[i];
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) if (col + i < cols) dst[i] = v[i];
            }
        }
    }
}

template <typename T>
int launch_quantize(const void *w, int64_t matrices, int64_t rows, int64_t cols, int64_t ld, int64_t matrix_stride, int group, uint8_t *codes, void *scales, cudaStream_t st) {
    const int64_t blocks = q4_row_tiles(rows);
    if (blocks > 0x7FFFFFFF || matrices > 65535) return fail(T81B200_ELIMIT, "quantize_q4: matrix too large");
    const bool vec = reinterpret_cast<uintptr_t>(w) % 16 == 0 && ld * sizeof(T) % 16 == 0 && matrix_stride * sizeof(T) % 16 == 0;
    const dim3 grid((unsigned)blocks, (unsigned)matrices);
    auto go = [&](auto kernel) {
        kernel<<<grid, kThreads, 0, st>>>(static_cast<const T *>(w), rows, cols, ld, matrix_stride, reinterpret_cast<uint4 *>(codes), static_cast<__nv_bfloat16 *>(scales));
    };
    if (group == 32) vec ? go(quantize_q4_kernel<T, 32, true>) : go(quantize_q4_kernel<T, 32, false>);
    else if (group == 64) vec ? go(quantize_q4_kernel<T, 64, true>) : go(quantize_q4_kernel<T, 64, false>);
    else vec ? go(quantize_q4_kernel<T, 128, true>) : go(quantize_q4_kernel<T, 128, false>);
    T81_LAUNCH_CHECK("quantize_q4_kernel");
    return T81B200_OK;
}

template <typename T>
int launch_dequantize(const uint8_t *codes, const void *scales, int64_t matrices, int64_t rows, int64_t cols, int group, void *out, cudaStream_t st) {
    const int64_t blocks = (matrices * q4_row_tiles(rows) * q4_col_tiles(cols) + kWarps - 1) / kWarps;
    if (blocks > 0x7FFFFFFF) return fail(T81B200_ELIMIT, "dequantize_q4: matrix too large");
    const bool vec = reinterpret_cast<uintptr_t>(out) % 16 == 0 && cols * sizeof(T) % 16 == 0;
    T81_CUDA_TRY(launch_behind(vec ? dequantize_q4_kernel<T, true> : dequantize_q4_kernel<T, false>, dim3((unsigned)blocks), kThreads, 0, st,
                               reinterpret_cast<const uint4 *>(codes), static_cast<const __nv_bfloat16 *>(scales), matrices, rows, cols, group, static_cast<T *>(out)));
    return T81B200_OK;
}

}  // namespace
}  // namespace t81b200

using namespace t81b200;

extern "C" int64_t t81b200_q4_bytes(int64_t rows, int64_t cols) {
    if (rows < 0 || cols < 0) return -1;
    return q4_row_tiles(rows) * q4_col_tiles(cols) * kQ4TileBytes;
}

extern "C" int64_t t81b200_q4_scales(int64_t rows, int64_t cols, int group) {
    if (rows < 0 || cols < 0 || !q4_group_ok(group)) return -1;
    return q4_row_tiles(rows) * (q4_groups(cols, group) + 1) * 16;
}

extern "C" int t81b200_quantize_q4(const void *w, int w_dtype, int64_t matrices, int64_t rows, int64_t cols, int64_t ld, int64_t matrix_stride, int group, uint8_t *codes,
                                   void *scales, void *stream) {
    if (matrices < 0 || rows < 0 || cols < 0 || ld < cols || (matrices > 1 && matrix_stride < 0)) return fail(T81B200_EINVAL, "quantize_q4: bad dimensions");
    if (!q4_group_ok(group)) return fail(T81B200_EINVAL, "quantize_q4: groups of 32, 64 or 128 columns, not %d", group);
    if (int rc = check_device()) return rc;
    if (matrices == 0 || rows == 0 || cols == 0) return T81B200_OK;
    if (!w || !codes || !scales) return fail(T81B200_EINVAL, "quantize_q4: null pointer");
    if (reinterpret_cast<uintptr_t>(codes) % 16 != 0 || reinterpret_cast<uintptr_t>(scales) % 16 != 0) return fail(T81B200_EALIGN, "quantize_q4: the outputs must be 16-byte aligned");
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (w_dtype) {
        case T81B200_F32: return launch_quantize<float>(w, matrices, rows, cols, ld, matrix_stride, group, codes, scales, st);
        case T81B200_BF16: return launch_quantize<__nv_bfloat16>(w, matrices, rows, cols, ld, matrix_stride, group, codes, scales, st);
        case T81B200_F16: return launch_quantize<__half>(w, matrices, rows, cols, ld, matrix_stride, group, codes, scales, st);
    }
    return fail(T81B200_EINVAL, "quantize_q4: unknown dtype %d", w_dtype);
}

extern "C" int t81b200_dequantize_q4(const uint8_t *codes, const void *scales, int64_t matrices, int64_t rows, int64_t cols, int group, void *out, int out_dtype, void *stream) {
    if (matrices < 0 || rows < 0 || cols < 0) return fail(T81B200_EINVAL, "dequantize_q4: bad dimensions");
    if (!q4_group_ok(group)) return fail(T81B200_EINVAL, "dequantize_q4: groups of 32, 64 or 128 columns, not %d", group);
    if (int rc = check_device()) return rc;
    if (matrices == 0 || rows == 0 || cols == 0) return T81B200_OK;
    if (!codes || !scales || !out) return fail(T81B200_EINVAL, "dequantize_q4: null pointer");
    if (reinterpret_cast<uintptr_t>(codes) % 16 != 0 || reinterpret_cast<uintptr_t>(scales) % 16 != 0) return fail(T81B200_EALIGN, "dequantize_q4: codes and scales must be 16-byte aligned");
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (out_dtype) {
        case T81B200_F32: return launch_dequantize<float>(codes, scales, matrices, rows, cols, group, out, st);
        case T81B200_BF16: return launch_dequantize<__nv_bfloat16>(codes, scales, matrices, rows, cols, group, out, st);
        case T81B200_F16: return launch_dequantize<__half>(codes, scales, matrices, rows, cols, group, out, st);
    }
    return fail(T81B200_EINVAL, "dequantize_q4: unknown dtype %d", out_dtype);
}
