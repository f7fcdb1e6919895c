// The 4-bit weight format ("Q4") and what the kernels that read it share.
//
// Columns of a row go in groups of 32, 64 or 128.  A weight is code * scale, code in -8 .. 7, scale a bf16 number of five significant
// bits per row and group; so the weight itself is a bf16 number (3 + 5 bits), and kernels that multiply codes and scale the sums give
// the same products as ones that multiply the weights.
//
// Codes lie in tiles of 16 rows x 64 columns, 512 bytes, tile (T, c) at (T * ceil(cols / 64) + c) * 512, in the order of the mma.sync
// m16n8k16 A fragments: lane l = 4 g + t owns the four words at 16 l; word j holds in bits 4 r + 16 h (four of them) code + 8 of
//     row 16 T + g + 8 (r % 2),  column 64 c + 32 (j / 2) + 8 t + 4 (j % 2) + 2 (r / 2) + h.
// Words 0, 1 are columns 0 .. 31 and words 2, 3 columns 32 .. 63, so that no multiply mixes two groups, and a lane's eight columns of either
// half are 16 bytes of an activation row or of an operand tile.  Scales of tile row T and group u: 16 bf16 numbers at
// (T * (groups + 1) + u) * 16, row r of the tile at 2 (r % 8) + r / 8: a lane's two rows are one word.  Behind the groups' come the
// rows' largest magnitudes of a scale: kernels that hold weights in fp16 bring a row into its range by the power of two in it.
// Rows and columns past the matrix have code 0 (bits 8) and scale 0.
#pragma once

#include "common.cuh"

#include <type_traits>

namespace t81b200 {

constexpr int kQ4TileBytes = 512;

__host__ __device__ inline int64_t q4_row_tiles(int64_t rows) { return (rows + 15) / 16; }
__host__ __device__ inline int64_t q4_col_tiles(int64_t cols) { return (cols + 63) / 64; }
__host__ __device__ inline int64_t q4_groups(int64_t cols, int group) { return (cols + group - 1) / group; }

inline bool q4_group_ok(int group) { return group == 32 || group == 64 || group == 128; }

// Register r of a word as a pair of exact numbers -8 .. 7.  The four bits go to where the units 1 to 8 lie in the mantissa of 16 (bf16: bit
// 3, fp16: bit 6), which gives 16 + code + 8; one packed add takes the 24 away, or one packed FMA with a scale s and -24 s.
// What an instruction cannot hold of the constants is made opaque: known ones are made again for every use where registers are short, which
// doubled the instructions of the streaming kernel.
__device__ __forceinline__ uint32_t opaque(uint32_t v) {
    uint32_t r;
    asm volatile("mov.b32 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
template <uint32_t B> __device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t c) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "n"(B), "r"(c));
    return d;
}

// DOWN (bf16): the constants, and so the codes, times 2^-DOWN.
template <typename T, int DOWN = 0> struct Q4Decode;
template <int DOWN> struct Q4Decode<__nv_bfloat16, DOWN> {
    static constexpr uint32_t mask = 0x00780078u, down = (uint32_t)DOWN * 0x00800080u;
    uint32_t sixteen, minus24;
    __device__ __forceinline__ Q4Decode() : sixteen(opaque(0x41804180u - down)), minus24(opaque(0xC1C0C1C0u - down)) {}
    template <int R> __device__ __forceinline__ uint32_t biased(uint32_t w) const { return and_or<mask>(R == 0 ? w << 3 : w >> (4 * R - 3), sixteen); }
    __device__ __forceinline__ uint32_t code(uint32_t v) const {
        uint32_t d;
        asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(v), "r"(minus24));
        return d;
    }
    // (v - 24) s for n = -24 s (7 bits): one rounding, of an exact result
    static __device__ __forceinline__ uint32_t scaled(uint32_t v, uint32_t s, uint32_t n) { return fma_bf16x2(v, s, n); }
};
template <> struct Q4Decode<__half, 0> {
    static constexpr uint32_t mask = 0x03C003C0u;
    uint32_t sixteen, minus24;
    __device__ __forceinline__ Q4Decode() : sixteen(opaque(0x4C004C00u)), minus24(opaque(0xCE00CE00u)) {}
    template <int R> __device__ __forceinline__ uint32_t biased(uint32_t w) const { return and_or<mask>(R < 2 ? w << (6 - 4 * R) : w >> (4 * R - 6), sixteen); }
    __device__ __forceinline__ uint32_t code(uint32_t v) const {
        uint32_t d;
        asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(v), "r"(minus24));
        return d;
    }
    static __device__ __forceinline__ uint32_t scaled(uint32_t v, uint32_t s, uint32_t n) {
        uint32_t d;
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(v), "r"(s), "r"(n));
        return d;
    }
};

// c = a b, or (ADD) c += a b.
template <typename T, bool ADD> __device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
#define T81_MMA(TYPE)                                                                                                                                  \
    if constexpr (ADD)                                                                                                                                 \
        asm("mma.sync.aligned.m16n8k16.row.col.f32." TYPE "." TYPE ".f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"              \
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])                                                                                           \
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));                                                                           \
    else                                                                                                                                               \
        asm("mma.sync.aligned.m16n8k16.row.col.f32." TYPE "." TYPE ".f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"          \
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])                                                                                           \
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f))
    if constexpr (std::is_same<T, __half>::value) {
        T81_MMA("f16");
    } else {
        T81_MMA("bf16");
    }
#undef T81_MMA
}

template <typename Decode>
__device__ __forceinline__ void q4_fragments(const Decode &decode, uint32_t w, uint32_t (&a)[4]) {
    a[0] = decode.code(decode.template biased<0>(w));
    a[1] = decode.code(decode.template biased<1>(w));
    a[2] = decode.code(decode.template biased<2>(w));
    a[3] = decode.code(decode.template biased<3>(w));
}

// Rows sorted by expert as a list of pieces of at most `width` rows: in shared memory, made by every block from the experts' first rows.
struct ExpertList {
    int2 *at;  // [experts + 1]: an expert's first row, the pieces of experts ahead of it

    static __host__ __device__ constexpr int bytes(int n_experts) { return 2 * (n_experts + 1) * 4; }

    // Whole block; returns the number of pieces.  Whatever the offsets say, no row outside 0 .. rows - 1 is named.
    __device__ __forceinline__ int build(int32_t *memory, const int32_t *offsets, int n_experts, int rows, int width) {
        at = reinterpret_cast<int2 *>(memory);
        const int lane = (int)threadIdx.x;
        if (lane < 32) {
            int sum = 0;
            for (int e0 = 0; e0 <= n_experts; e0 += 32) {
                const int e = e0 + lane;
                const int row = e <= n_experts ? min(max(offsets[e], 0), rows) : 0, end = e < n_experts ? min(max(offsets[e + 1], 0), rows) : 0;
                const int pieces = e < n_experts && end > row ? (end - row + width - 1) / width : 0;
                int scan = pieces;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int o = __shfl_up_sync(0xffffffffu, scan, d);
                    if (lane >= d) scan += o;
                }
                if (e <= n_experts) at[e] = make_int2(row, sum + scan - pieces);
                sum += __shfl_sync(0xffffffffu, scan, 31);
            }
        }
        __syncthreads();
        return at[n_experts].y;
    }

    __device__ __forceinline__ int first(int e) const { return at[e].x; }
    __device__ __forceinline__ int before(int e) const { return at[e].y; }

    // The expert that a piece belongs to.
    __device__ __forceinline__ int expert_of(int piece, int n_experts) const {
        int lo = 0, hi = n_experts;  // the last one with no more pieces ahead of it has a piece
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (before(mid) <= piece) lo = mid;
            else hi = mid;
        }
        return lo;
    }
};

}  // namespace t81b200
