// Weights to 4-bit codes with group scales, and back (the format: q4.cuh).
//
// Quantise: m = the group's value of largest magnitude (the first of equals), scale s = m / -8 rounded to five significant bits, code =
// the whole number nearest to w / s, ties to even, held in -8 .. 7.  Eight steps reach from 0 to the largest value and seven the
// other way.  Five bits for the scale make code * s a bf16 number, and cost little: N(0, 1) weights in groups of 128 come back with
// a mean square error 0.15 % above that of an unrounded scale (0.6 % in groups of 32).
// A weight is read once, half a byte is written: 14336 x 4096 bf16 37 us, 0.62 of the copy rate, 68 % of the issue slots busy.  A warp holds 16 rows x
// 128 columns in registers (64 in groups of 32 and 64), a lane eight columns of two rows at a time as the format has them: 64
// (16-bit) or 128 bytes of a row side by side per load.
#include "common.cuh"
#include "launch_order.cuh"
#include "q4.cuh"

#include <type_traits>

namespace t81b200 {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr float kMost = 8.507059173023462e37f;   // 2^126: larger magnitudes count as this, so that 8 s is finite
constexpr float kLeast = 7.888609052210118e-31f; // 2^-100: a group of smaller ones is zero (s would leave the normal numbers)

// Eight neighbouring elements of a row as they lie in memory.
template <typename T> struct Eight { uint4 w[sizeof(T) / 2]; };

// Columns at and past `left` are 0.  VEC: the row lies on 16-byte boundaries.
template <typename T, bool VEC>
__device__ __forceinline__ Eight<T> load8(const T *src, int64_t left) {
    Eight<T> e;
    if (VEC && left >= 8) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) e.w[i] = __ldcs(reinterpret_cast<const uint4 *>(src) + i);
    } else {
        T v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < left ? src[i] : from_float<T>(0.0f);
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) e.w[i] = reinterpret_cast<const uint4 *>(v)[i];
    }
    return e;
}

// Largest and smallest of the elements, and whether one is no number or infinite (`probe` stays 0 otherwise): two elements at a time in
// 16-bit types.
template <typename T> struct Extremes {
    float high = 0.0f, low = 0.0f, probe = 0.0f;
    __device__ __forceinline__ void take(const Eight<T> &e) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = reinterpret_cast<const float *>(&e)[i];
            high = fmaxf(high, x);
            low = fminf(low, x);
            probe = fmaf(x, 0.0f, probe);
        }
    }
    __device__ __forceinline__ void done() {}
};
template <typename T, typename T2> struct Extremes16 {
    T2 high2 = T2(from_float<T>(0.0f), from_float<T>(0.0f)), low2 = high2, probe2 = high2;
    float high, low, probe;
    __device__ __forceinline__ void take(const Eight<T> &e) {
        const T2 zero(from_float<T>(0.0f), from_float<T>(0.0f));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const T2 x = reinterpret_cast<const T2 *>(&e)[i];
            high2 = __hmax2(high2, x);
            low2 = __hmin2(low2, x);
            probe2 = __hfma2(x, zero, probe2);
        }
    }
    __device__ __forceinline__ void done() {
        high = fmaxf(to_float<T>(high2.x), to_float<T>(high2.y));
        low = fminf(to_float<T>(low2.x), to_float<T>(low2.y));
        probe = to_float<T>(probe2.x) + to_float<T>(probe2.y);
    }
};
template <> struct Extremes<__nv_bfloat16> : Extremes16<__nv_bfloat16, __nv_bfloat162> {};
template <> struct Extremes<__half> : Extremes16<__half, __half2> {};

template <typename T> __device__ __forceinline__ float element(const Eight<T> &e, int i) {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(&e);
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16);
    else return __half2float(__ushort_as_half((unsigned short)(w[i >> 1] >> (16 * (i & 1)))));
}
// What the rule makes of it: no number counts as 0, magnitudes above kMost as that.
__device__ __forceinline__ float tamed(float v) { return v != v ? 0.0f : fminf(fmaxf(v, -kMost), kMost); }

// m / -8 rounded to five significant bits, ties to even.
__device__ __forceinline__ float scale_of(float m) {
    if (fabsf(m) < kLeast) return 0.0f;
    uint32_t b = __float_as_uint(m * -0.125f);
    b += 0x3FFFFu + ((b >> 19) & 1u);
    return __uint_as_float(b & 0xFFF80000u);
}

// 1.5 * 2^23 + 8 plus the code of w in its last bits.  The quotient is the correctly rounded one (Markstein's correction by the exact rest, from
// the correctly rounded reciprocal), which meets a border between two codes only where w / s does: w / s is at least 2^-23 / (s's
// mantissa) of its binade from one otherwise, more than half a last place.  Adding 1.5 * 2^23 rounds it, ties to even.
__device__ __forceinline__ uint32_t code_bits(float w, float s, float inverse) {
    float q = w * inverse;
    q = fmaf(fmaf(-q, s, w), inverse, q);
    return __float_as_uint(fminf(q, 7.0f) + 12582920.0f);  // (the largest of its sign comes to -8.26 at most, which is -8)
}
constexpr uint32_t kCodeBits = 0x4B400000u;  // what code_bits has beside the code

// A block takes 16 rows, its warps units of 128 columns in turn.
template <typename T, int GROUP, bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_q4_kernel(const T *__restrict__ w, int64_t rows, int64_t cols, int64_t ld, int64_t matrix_stride,
                                                               uint4 *__restrict__ codes, __nv_bfloat16 *__restrict__ scales) {
    // A step is a group of 128 columns, or 64 columns of smaller groups; a lane has eight columns of two rows of each half of 64.
    constexpr int TILES = GROUP == 128 ? 2 : 1, PER_TILE = GROUP == 32 ? 2 : 1;
    __shared__ float most[kWarps][16];
    const int64_t row_tiles = q4_row_tiles(rows), col_tiles = q4_col_tiles(cols), groups = q4_groups(cols, GROUP), steps = (col_tiles + TILES - 1) / TILES;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int64_t matrix = blockIdx.y, T16 = blockIdx.x, out_tile = matrix * row_tiles + T16;
    float largest[2] = {0.0f, 0.0f};  // of the lane's rows
    const T *const matrix_at = w + matrix * matrix_stride;
    auto load = [&](int64_t step, Eight<T>(&v)[TILES][2][2]) {
#pragma unroll
        for (int c = 0; c < TILES; ++c)
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int64_t row = 16 * T16 + g + 8 * r, col = step * (64 * TILES) + 64 * c + 32 * half + 8 * t;
                    v[c][half][r] = load8<T, VEC>(matrix_at + (row < rows ? row : 0) * ld + col, row < rows ? cols - col : 0);
                }
    };
    for (int64_t step = warp; step < steps; step += kWarps) {
        Eight<T> v[TILES][2][2];  // [tile][half of its columns][row of the lane]
        load(step, v);
        float s[PER_TILE][2];  // [group][row]
        bool wild = false;
#pragma unroll
        for (int u = 0; u < PER_TILE; ++u)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                Extremes<T> all;
#pragma unroll
                for (int c = 0; c < TILES; ++c)
#pragma unroll
                    for (int half = (GROUP == 32 ? u : 0); half < (GROUP == 32 ? u + 1 : 2); ++half) all.take(v[c][half][r]);
                all.done();
                float high = all.high, low = all.low;
#pragma unroll
                for (int d = 1; d < 4; d <<= 1) {
                    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, d));
                    low = fminf(low, __shfl_xor_sync(0xffffffffu, low, d));
                }
                float m = high > -low ? high : low;
                const bool here = all.probe != 0.0f || high > kMost || low < -kMost;
                wild = wild || here;
                if (__any_sync(0xffffffffu, here || (high == -low && high > 0.0f))) {
                    // equal magnitudes of both signs, the first of which gives the sign, or what the rule tames: element by element
                    m = 0.0f;
#pragma unroll
                    for (int c = 0; c < TILES; ++c)
#pragma unroll
                        for (int half = (GROUP == 32 ? u : 0); half < (GROUP == 32 ? u + 1 : 2); ++half) {
                            float mine = 0.0f;
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const float x = tamed(element(v[c][half][r], i));
                                if (fabsf(x) > fabsf(mine)) mine = x;
                            }
#pragma unroll
                            for (int d = 1; d < 4; d <<= 1) {  // a lane's columns lie before the next one's
                                const float o = __shfl_xor_sync(0xffffffffu, mine, d);
                                if (fabsf(o) > fabsf(mine) || ((t & d) != 0 && fabsf(o) == fabsf(mine))) mine = o;
                            }
                            if (fabsf(mine) > fabsf(m)) m = mine;
                        }
                }
                s[u][r] = scale_of(m);
            }
        const bool wild_warp = __any_sync(0xffffffffu, wild);
#pragma unroll
        for (int u = 0; u < PER_TILE; ++u) {
#pragma unroll
            for (int r = 0; r < 2; ++r) largest[r] = fmaxf(largest[r], fabsf(s[u][r]));
            const int64_t group = step * PER_TILE + u;
            if (t == 0 && group < groups) {
                const __nv_bfloat162 pair(__float2bfloat16_rn(s[u][0]), __float2bfloat16_rn(s[u][1]));
                *reinterpret_cast<uint32_t *>(scales + (out_tile * (groups + 1) + group) * 16 + 2 * g) = bf162_bits(pair);
            }
        }
#pragma unroll
        for (int c = 0; c < TILES; ++c) {
            if (TILES == 2 && step * 2 + c >= col_tiles) break;
            uint32_t word[4] = {0u, 0u, 0u, 0u};
            auto encode = [&](auto tame) {
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        // (a group of zeros: scale and reciprocal 0 make every code 0, that is 8)
                        const float scale = s[GROUP == 32 ? half : 0][r], inverse = scale != 0.0f ? 1.0f / scale : 0.0f;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {  // column 4 (j % 2) + 2 (register / 2) + h of the lane's eight
                            const float x = element(v[c][half][r], i);
                            const int shift = 4 * (r + 2 * ((i >> 1) & 1)) + 16 * (i & 1);
                            word[2 * half + (i >> 2)] += code_bits(decltype(tame)::value ? tamed(x) : x, scale, inverse) << shift;
                        }
                    }
            };
            if (wild_warp) encode(std::true_type{});
            else encode(std::false_type{});
            // what the codes' numbers have beside them, the same in every word
            constexpr uint32_t beside = kCodeBits * 0x11111111u;
#pragma unroll
            for (int j = 0; j < 4; ++j) word[j] -= beside;
            codes[(out_tile * col_tiles + step * TILES + c) * 32 + lane] = make_uint4(word[0], word[1], word[2], word[3]);
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

// Every value is exact in fp32 and in bf16.  A warp takes a tile; fp32 halves of eight columns change places between two lanes, so that a
// store fills whole sectors.  Rows off 16-byte boundaries go through shared memory, four tiles in turn, so that a warp's stores lie side by
// side.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) dequantize_q4_kernel(const uint4 *__restrict__ codes, const __nv_bfloat16 *__restrict__ scales, int64_t matrices, int64_t rows,
                                                                 int64_t cols, int group, T *__restrict__ out) {
    constexpr int TILES = VEC ? 1 : 4;
    __shared__ T through[VEC ? 1 : kWarps][VEC ? 1 : 16][VEC ? 1 : 65];
    wait_for_kernel_ahead();
    const int64_t row_tiles = q4_row_tiles(rows), col_tiles = q4_col_tiles(cols), groups = q4_groups(cols, group), across = (col_tiles + TILES - 1) / TILES;
    const int64_t at = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (at >= matrices * row_tiles * across) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int64_t c0 = at % across * TILES, all_T = at / across, matrix = all_T / row_tiles, T16 = all_T % row_tiles;
    T *const matrix_at = out + matrix * rows * cols;
    uint4 q[TILES];
    uint32_t pair[TILES][2];
#pragma unroll
    for (int c = 0; c < TILES; ++c) {
        const bool there = c0 + c < col_tiles;
        q[c] = there ? __ldcs(codes + (all_T * col_tiles + c0 + c) * 32 + lane) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int64_t col = 64 * (c0 + c) + 32 * half;
            pair[c][half] = col < cols ? *reinterpret_cast<const uint32_t *>(scales + (all_T * (groups + 1) + col / group) * 16 + 2 * g) : 0u;
        }
    }
#pragma unroll
    for (int c = 0; c < TILES; ++c) {
        if (c0 + c >= col_tiles) break;
        const uint32_t word[4] = {q[c].x, q[c].y, q[c].z, q[c].w};
        if (!VEC) __syncwarp();
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float s = __uint_as_float(r ? pair[c][half] & 0xFFFF0000u : pair[c][half] << 16);
                __align__(16) T v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    v[i] = from_float<T>((float)((int)((word[2 * half + (i >> 2)] >> (4 * (r + 2 * ((i >> 1) & 1)) + 16 * (i & 1))) & 15u) - 8) * s);
                if constexpr (VEC && sizeof(T) == 4) {  // (rows of whole 16 bytes end with one)
                    const bool odd = (t & 1) != 0;
                    float mine[4], other[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        other[i] = __shfl_xor_sync(0xffffffffu, odd ? v[i] : v[4 + i], 1);
                        mine[i] = odd ? v[4 + i] : v[i];
                    }
                    // the pair's sixteen columns: the even lane has columns 0 .. 3 and 8 .. 11, the odd one 4 .. 7 and 12 .. 15
                    const int64_t row = 16 * T16 + g + 8 * r, col = 64 * (c0 + c) + 32 * half + 16 * (t >> 1) + 4 * (t & 1);
                    float *at_row = reinterpret_cast<float *>(matrix_at) + row * cols + col;
                    if (row < rows && col < cols) *reinterpret_cast<float4 *>(at_row) = odd ? make_float4(other[0], other[1], other[2], other[3]) : make_float4(mine[0], mine[1], mine[2], mine[3]);
                    if (row < rows && col + 8 < cols) *reinterpret_cast<float4 *>(at_row + 8) = odd ? make_float4(mine[0], mine[1], mine[2], mine[3]) : make_float4(other[0], other[1], other[2], other[3]);
                } else if constexpr (VEC) {
                    const int64_t row = 16 * T16 + g + 8 * r, col = 64 * (c0 + c) + 32 * half + 8 * t;
                    if (row < rows && col < cols) *reinterpret_cast<uint4 *>(matrix_at + row * cols + col) = *reinterpret_cast<const uint4 *>(v);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) through[warp][g + 8 * r][32 * half + 8 * t + i] = v[i];
                }
            }
        if constexpr (!VEC) {
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int64_t row = 16 * T16 + i;
#pragma unroll
                for (int k = 0; k < 64; k += 32) {
                    const int64_t col = 64 * (c0 + c) + k + lane;
                    if (row < rows && col < cols) matrix_at[row * cols + col] = through[warp][i][k + lane];
                }
            }
        }
    }
}

// Scales in the matrix's order: a thread each, stores side by side.
__global__ void __launch_bounds__(kThreads) group_scales_kernel(const uint16_t *__restrict__ scales, int64_t rows, int64_t groups, int64_t total, uint16_t *__restrict__ out) {
    wait_for_kernel_ahead();
    const int64_t tiles = q4_row_tiles(rows);
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
        const int64_t u = i % groups, row_of_all = i / groups, matrix = row_of_all / rows, row = row_of_all % rows;
        out[i] = scales[((matrix * tiles + (row >> 4)) * (groups + 1) + u) * 16 + 2 * (row & 7) + ((row >> 3) & 1)];
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
    const bool vec = reinterpret_cast<uintptr_t>(out) % 16 == 0 && cols * sizeof(T) % 16 == 0;
    const int64_t blocks = (matrices * q4_row_tiles(rows) * (vec ? q4_col_tiles(cols) : (q4_col_tiles(cols) + 3) / 4) + kWarps - 1) / kWarps;
    if (blocks > 0x7FFFFFFF) return fail(T81B200_ELIMIT, "dequantize_q4: matrix too large");
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

extern "C" int t81b200_q4_group_scales(const void *scales, int64_t matrices, int64_t rows, int64_t cols, int group, void *out, void *stream) {
    if (matrices < 0 || rows < 0 || cols < 0) return fail(T81B200_EINVAL, "q4_group_scales: bad dimensions");
    if (!q4_group_ok(group)) return fail(T81B200_EINVAL, "q4_group_scales: groups of 32, 64 or 128 columns, not %d", group);
    if (int rc = check_device()) return rc;
    if (matrices == 0 || rows == 0 || cols == 0) return T81B200_OK;
    if (!scales || !out) return fail(T81B200_EINVAL, "q4_group_scales: null pointer");
    const int64_t groups = q4_groups(cols, group), total = matrices * rows * groups, blocks = (total + kThreads - 1) / kThreads, most = (int64_t)sm_count() * 16;
    T81_CUDA_TRY(launch_behind(group_scales_kernel, dim3((unsigned)(blocks < most ? blocks : most)), kThreads, 0, static_cast<cudaStream_t>(stream), static_cast<const uint16_t *>(scales), rows,
                               groups, total, static_cast<uint16_t *>(out)));
    return T81B200_OK;
}
