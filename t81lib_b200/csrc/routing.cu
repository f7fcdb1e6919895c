// Rows of a mixture of experts: (token, slot) pairs sorted by expert, rows gathered in that order and combined again, and the gradients.
//
//   sort     order[p] = flat index (token * top + slot) of sorted row p, position its inverse, offsets[e] the first row of expert e; a stable
//            counting sort, so pairs of one expert keep their order; ids outside 0 .. n_experts - 1 take no part (position -1) and order is -1
//            past the last row
//   gather   rows[p] = x[order[p] / top], 0 past the last row
//   combine  y[t] = sum_j w[t][j] rows[position[t][j]] in slot order, fp32, rounded once; slots without a row take no part.  Without
//            weights it is gather's gradient.
//   combine's gradient: grad_rows[p] = w[order[p]] grad_y[order[p] / top] (0 past the last row), grad_w[t][j] = <grad_y[t], rows[position[t][j]]>.
//
// Sort: one cluster of CTAs.  A warp counts its run of ids by expert in shared memory of its own (a step of 32 ids: lanes with equal ids find
// one another, the first adds their number), the counts become first positions by sums over warps, CTAs (distributed shared
// memory) and experts, and the warp goes through its run again.  No atomics: the order is always the same.
// The others are bound by memory: whole 16-byte pieces where rows allow, one read of each input row and one write of each result row
// (gather: a token's row is read once and written to its slots).
#include "common.cuh"
#include "launch_order.cuh"

#include <cooperative_groups.h>

#include <atomic>

namespace t81b200 {

namespace {

namespace cg = cooperative_groups;

constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32, kMostExperts = 1024, kSortCluster = 16, kSortKept = 4;

// The lanes with this lane's value, of `bits` bits: a vote per bit (match_any takes its turn on one unit of the SM: 131072 ids 42 us).
__device__ __forceinline__ uint32_t equal_lanes(int v, int bits) {
    uint32_t equal = 0xffffffffu;
    for (int b = 0; b < bits; ++b) {
        const bool one = ((v >> b) & 1) != 0;
        const uint32_t ones = __ballot_sync(0xffffffffu, one);
        equal &= one ? ones : ~ones;
    }
    return equal;
}

template <typename ID>
__global__ void __launch_bounds__(kSortThreads, 1) sort_by_expert_kernel(const ID *__restrict__ ids, int n, int n_experts, int run, int32_t *__restrict__ order,
                                                                         int32_t *__restrict__ position, int32_t *__restrict__ offsets) {
    extern __shared__ int32_t counts[];  // [warps][experts], then [experts] of this CTA
    __shared__ int32_t warp_sums[32];
    __shared__ int32_t kept;
    wait_for_kernel_ahead();
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int bits = 32 - __clz(n_experts);  // ids and n_experts itself
    const int pitch = n_experts | 1;  // odd: the warps' counts of an expert lie in different banks
    int32_t *mine = counts + warp * pitch, *cta_total = counts + kSortWarps * pitch;
    for (int i = threadIdx.x; i < kSortWarps * pitch; i += kSortThreads) counts[i] = 0;
    __syncthreads();
    const int64_t lo64 = (int64_t)(rank * kSortWarps + warp) * run;
    const int lo = lo64 < n ? (int)lo64 : n, hi = n - lo < run ? n : lo + run;
    auto expert_of = [&](int i) {
        if (i >= hi) return n_experts;
        const ID id = ids[i];
        return id >= 0 && id < (ID)n_experts ? (int)id : n_experts;
    };
    // the ids of a warp's first steps stay in registers for the second pass
    int kept_ids[kSortKept];
#pragma unroll
    for (int k = 0; k < kSortKept; ++k) kept_ids[k] = expert_of(lo + 32 * k + lane);
    auto steps = [&](auto &&body) {
#pragma unroll
        for (int k = 0; k < kSortKept; ++k)
            if (lo + 32 * k < hi) body(lo + 32 * k, kept_ids[k]);
        for (int i0 = lo + 32 * kSortKept; i0 < hi; i0 += 32) body(i0, expert_of(i0 + lane));
    };
    steps([&](int, int e) {
        const uint32_t equal = equal_lanes(e, bits);
        if (e < n_experts && lane == __ffs(equal) - 1) mine[e] += __popc(equal);
        __syncwarp();
    });
    __syncthreads();
    // counts to the number in warps ahead: a warp per expert, a lane per warp
    for (int x = warp; x < n_experts; x += kSortWarps) {
        const int32_t c = counts[lane * pitch + x];
        int32_t sum = c;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int32_t o = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += o;
        }
        counts[lane * pitch + x] = sum - c;
        if (lane == 31) cta_total[x] = sum;
    }
    cluster.sync();
    const int e = threadIdx.x;
    int32_t before = 0, all = 0;  // of this expert: in CTAs ahead, in all
    if (e < n_experts) {
        int32_t of[kSortCluster];
#pragma unroll
        for (int r = 0; r < kSortCluster; ++r) of[r] = r < ctas ? cluster.map_shared_rank(cta_total, r)[e] : 0;
#pragma unroll
        for (int r = 0; r < kSortCluster; ++r) {
            before += r < rank ? of[r] : 0;
            all += of[r];
        }
    }
    cluster.sync();  // nobody reads another CTA's counts from here on
    int32_t scan = all;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int32_t o = __shfl_up_sync(0xffffffffu, scan, d);
        if (lane >= d) scan += o;
    }
    if (lane == 31) warp_sums[warp] = scan;
    __syncthreads();
    int32_t ahead = 0;
    for (int w = 0; w < warp; ++w) ahead += warp_sums[w];
    const int32_t start = ahead + scan - all;
    if (e < n_experts) {
        cta_total[e] = start + before;
        if (rank == 0) offsets[e] = start;
    }
    if (e == n_experts - 1) {
        kept = start + all;
        if (rank == 0) offsets[n_experts] = kept;
    }
    __syncthreads();
    steps([&](int i0, int id) {
        const int i = i0 + lane;
        const uint32_t equal = equal_lanes(id, bits);
        if (id < n_experts) {
            const int32_t at = cta_total[id] + mine[id] + __popc(equal & ((1u << lane) - 1u));
            order[at] = i;
            position[i] = at;
        } else if (i < hi) position[i] = -1;
        __syncwarp();
        if (id < n_experts && lane == __ffs(equal) - 1) mine[id] += __popc(equal);
        __syncwarp();
    });
    for (int64_t p = (int64_t)kept + rank * kSortThreads + threadIdx.x; p < n; p += ctas * kSortThreads) order[p] = -1;
}

// ---- rows ----

constexpr int kThreads = 256, kWarps = kThreads / 32;

// Tokens first (row t of x to its slots), then the rows past the last expert's, which are zero.
template <typename P>
__global__ void __launch_bounds__(kThreads) gather_rows_kernel(const uint8_t *__restrict__ x, int64_t ld, int64_t tokens, int top, int64_t pieces, const int32_t *__restrict__ position,
                                                               const int32_t *__restrict__ kept, uint8_t *__restrict__ rows) {
    wait_for_kernel_ahead();
    const int64_t n = tokens * top, chunk = (int64_t)blockIdx.y * kThreads + threadIdx.x;
    if (chunk >= pieces) return;
    for (int64_t t = blockIdx.x; t < tokens; t += gridDim.x) {
        const P v = __ldg(reinterpret_cast<const P *>(x + t * ld) + chunk);
        for (int j = 0; j < top; ++j) {
            const int64_t p = position[t * top + j];
            if (p >= 0 && p < n) reinterpret_cast<P *>(rows)[p * pieces + chunk] = v;
        }
    }
    for (int64_t p = (int64_t)max(*kept, 0) + blockIdx.x; p < n; p += gridDim.x) reinterpret_cast<P *>(rows)[p * pieces + chunk] = P{};
}

template <typename T, int N> struct alignas(sizeof(T) * N) Piece { T v[N]; };

// y[t] of the block's piece of the row.  W: type of the weights.
template <typename T, int N, typename W>
__global__ void __launch_bounds__(kThreads) combine_rows_kernel(const T *__restrict__ rows, int64_t ld, int64_t tokens, int top, int64_t pieces, const int32_t *__restrict__ position,
                                                                const W *__restrict__ weights, T *__restrict__ y) {
    wait_for_kernel_ahead();
    const int64_t n = tokens * top, chunk = (int64_t)blockIdx.y * kThreads + threadIdx.x;
    if (chunk >= pieces) return;
    for (int64_t t = blockIdx.x; t < tokens; t += gridDim.x) {
        float sum[N] = {};
        for (int j0 = 0; j0 < top; j0 += 4) {  // four rows on their way at a time
            Piece<T, N> v[4];
            float w[4];
            bool there[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int64_t p = j0 + k < top ? position[t * top + j0 + k] : -1;
                there[k] = p >= 0 && p < n;
                v[k] = reinterpret_cast<const Piece<T, N> *>(rows + (there[k] ? p : 0) * ld)[chunk];  // (a slot without a row reads one all the same: no branch between loads)
                w[k] = weights && there[k] ? to_float<W>(weights[t * top + j0 + k]) : 1.0f;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (there[k])
#pragma unroll
                    for (int i = 0; i < N; ++i) sum[i] = fmaf(w[k], to_float<T>(v[k].v[i]), sum[i]);
        }
        Piece<T, N> out;
#pragma unroll
        for (int i = 0; i < N; ++i) out.v[i] = from_float<T>(sum[i]);
        reinterpret_cast<Piece<T, N> *>(y)[t * pieces + chunk] = out;
    }
}

// A warp per (token, slot): its piece of grad_rows and its weight's gradient; then the rows past the last expert's.
template <typename T, int N, typename W>
__global__ void __launch_bounds__(kThreads) combine_rows_grad_kernel(const T *__restrict__ grad_y, int64_t ld_y, const T *__restrict__ rows, int64_t ld, int64_t tokens, int top,
                                                                     int64_t pieces, const int32_t *__restrict__ position, const int32_t *__restrict__ kept,
                                                                     const W *__restrict__ weights, T *__restrict__ grad_rows, W *__restrict__ grad_weights) {
    wait_for_kernel_ahead();
    const int64_t n = tokens * top, stride = (int64_t)gridDim.x * kWarps, warp = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    for (int64_t i = warp; i < n; i += stride) {
        const int64_t p = position[i], t = i / top;
        float dot = 0.0f;
        if (p >= 0 && p < n) {
            const float w = weights ? to_float<W>(weights[i]) : 1.0f;
            const Piece<T, N> *gy = reinterpret_cast<const Piece<T, N> *>(grad_y + t * ld_y), *row = reinterpret_cast<const Piece<T, N> *>(rows + p * ld);
            Piece<T, N> *out = reinterpret_cast<Piece<T, N> *>(grad_rows) + p * pieces;
            for (int64_t c = lane; c < pieces; c += 32) {
                const Piece<T, N> g = gy[c];
                if (grad_weights) {
                    const Piece<T, N> r = row[c];
#pragma unroll
                    for (int k = 0; k < N; ++k) dot = fmaf(to_float<T>(g.v[k]), to_float<T>(r.v[k]), dot);
                }
                if (grad_rows) {
                    Piece<T, N> o;
#pragma unroll
                    for (int k = 0; k < N; ++k) o.v[k] = from_float<T>(w * to_float<T>(g.v[k]));
                    out[c] = o;
                }
            }
        }
        if (grad_weights) {
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
            if (lane == 0) grad_weights[i] = from_float<W>(dot);
        }
    }
    if (!grad_rows) return;
    for (int64_t p = (int64_t)max(*kept, 0) + warp; p < n; p += stride)
        for (int64_t c = lane; c < pieces; c += 32) {
            Piece<T, N> o;
#pragma unroll
            for (int k = 0; k < N; ++k) o.v[k] = from_float<T>(0.0f);
            reinterpret_cast<Piece<T, N> *>(grad_rows)[p * pieces + c] = o;
        }
}

template <typename ID>
int launch_sort(const void *ids, int64_t n, int n_experts, int32_t *order, int32_t *position, int32_t *offsets, cudaStream_t st) {
    const size_t smem = ((size_t)kSortWarps * (n_experts | 1) + n_experts) * sizeof(int32_t);
    auto kernel = sort_by_expert_kernel<ID>;
    T81_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)((kSortWarps + 1) * (kMostExperts + 1) * sizeof(int32_t))));
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kSortThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    auto shape = [&](int ctas) {
        cfg.gridDim = dim3((unsigned)ctas);
        attr[0].val.clusterDim.x = (unsigned)ctas;
    };
    // Sixteen CTAs where the device runs that many as a cluster (131072 ids 19 us, 30 with eight), eight for up to 8192 ids, one for up to 1024.
    int ctas = n > 8192 ? kSortCluster : (n > kSortThreads ? 8 : 1);
    if (ctas == kSortCluster) {
        static std::atomic<int> fits[64];  // 1: a cluster of sixteen fits, 2: it does not
        int dev = 0, known = 0;
        T81_CUDA_TRY(cudaGetDevice(&dev));
        if (dev >= 0 && dev < 64) known = fits[dev].load(std::memory_order_relaxed);
        if (known == 0) {
            int clusters = 0;
            shape(ctas);
            cfg.numAttrs = 1;
            cfg.dynamicSmemBytes = (kSortWarps + 1) * (kMostExperts + 1) * sizeof(int32_t);
            known = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
                            cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) == cudaSuccess && clusters > 0 ? 1 : 2;
            (void)cudaGetLastError();
            cfg.dynamicSmemBytes = smem;
            if (dev >= 0 && dev < 64) fits[dev].store(known, std::memory_order_relaxed);
        }
        if (known == 2) ctas = 8;
    }
    shape(ctas);
    cfg.numAttrs = 2;
    const int64_t run = ((n + (int64_t)ctas * kSortWarps - 1) / ((int64_t)ctas * kSortWarps) + 31) / 32 * 32;
    T81_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, static_cast<const ID *>(ids), (int)n, n_experts, (int)run, order, position, offsets));
    return T81B200_OK;
}

bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Blocks along the tokens and along a row's pieces.
dim3 row_grid(int64_t tokens, int64_t pieces) {
    const int64_t across = (pieces + kThreads - 1) / kThreads, most = 1 << 20;
    return dim3((unsigned)(tokens < 1 ? 1 : (tokens < most ? tokens : most)), (unsigned)across);
}

template <typename T, typename W>
int launch_combine(const void *rows, int64_t ld, int64_t tokens, int top, int64_t width, const int32_t *position, const void *weights, void *y, cudaStream_t st) {
    constexpr int N = 16 / (int)sizeof(T);
    const bool vec = width % N == 0 && ld % N == 0 && aligned16(rows) && aligned16(y);
    const int64_t pieces = vec ? width / N : width;
    const dim3 grid = row_grid(tokens, pieces);
    if (grid.y > 65535u) return fail(T81B200_ELIMIT, "combine_rows: rows too wide");
    T81_CUDA_TRY(launch_behind(vec ? combine_rows_kernel<T, N, W> : combine_rows_kernel<T, 1, W>, grid, kThreads, 0, st, static_cast<const T *>(rows), ld, tokens, top, pieces, position,
                               static_cast<const W *>(weights), static_cast<T *>(y)));
    return T81B200_OK;
}

template <typename T, typename W>
int launch_combine_grad(const void *grad_y, int64_t ld_y, const void *rows, int64_t ld, int64_t tokens, int top, int64_t width, const int32_t *position, const int32_t *kept,
                        const void *weights, void *grad_rows, void *grad_weights, cudaStream_t st) {
    constexpr int N = 16 / (int)sizeof(T);
    const bool vec = width % N == 0 && ld % N == 0 && ld_y % N == 0 && aligned16(rows) && aligned16(grad_y) && aligned16(grad_rows);
    const int64_t n = tokens * top, blocks = (n + kWarps - 1) / kWarps, most = 1 << 20;
    T81_CUDA_TRY(launch_behind(vec ? combine_rows_grad_kernel<T, N, W> : combine_rows_grad_kernel<T, 1, W>, dim3((unsigned)(blocks < most ? blocks : most)), kThreads, 0, st,
                               static_cast<const T *>(grad_y), ld_y, static_cast<const T *>(rows), ld, tokens, top, vec ? width / N : width, position, kept, static_cast<const W *>(weights),
                               static_cast<T *>(grad_rows), static_cast<W *>(grad_weights)));
    return T81B200_OK;
}

// f(T{}, W{}) for the two types.
template <typename F> int by_types(const char *name, int dtype, int w_dtype, F &&f) {
    auto inner = [&](auto t) -> int {
        switch (w_dtype) {
            case T81B200_F32: return f(t, float{});
            case T81B200_BF16: return f(t, __nv_bfloat16{});
            case T81B200_F16: return f(t, __half{});
        }
        return fail(T81B200_EINVAL, "%s: unknown dtype of the weights %d", name, w_dtype);
    };
    switch (dtype) {
        case T81B200_F32: return inner(float{});
        case T81B200_BF16: return inner(__nv_bfloat16{});
        case T81B200_F16: return inner(__half{});
    }
    return fail(T81B200_EINVAL, "%s: unknown dtype %d", name, dtype);
}

int check_rows(const char *name, int64_t tokens, int64_t top, int64_t width, int64_t ld) {
    if (tokens < 0 || top < 1 || width < 0 || ld < width) return fail(T81B200_EINVAL, "%s: bad dimensions", name);
    if (top > (1 << 20) || tokens > 0x7FFFFFFF / top) return fail(T81B200_ELIMIT, "%s: more than 2^31 - 1 (token, slot) pairs", name);
    return T81B200_OK;
}

}  // namespace
}  // namespace t81b200

using namespace t81b200;

extern "C" int t81b200_sort_by_expert(const void *ids, int id_bytes, int64_t n, int n_experts, int32_t *order, int32_t *position, int32_t *offsets, void *stream) {
    if (n < 0 || n_experts < 1 || (id_bytes != 4 && id_bytes != 8)) return fail(T81B200_EINVAL, "sort_by_expert: bad dimensions");
    if (n_experts > kMostExperts) return fail(T81B200_ELIMIT, "sort_by_expert: at most %d experts", kMostExperts);
    if (n > 0x7FFFFFFF - kSortCluster * kSortThreads * 32) return fail(T81B200_ELIMIT, "sort_by_expert: too many (token, slot) pairs");
    if (int rc = check_device()) return rc;
    if (!offsets || (n > 0 && (!ids || !order || !position))) return fail(T81B200_EINVAL, "sort_by_expert: null pointer");
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return id_bytes == 8 ? launch_sort<int64_t>(ids, n, n_experts, order, position, offsets, st) : launch_sort<int32_t>(ids, n, n_experts, order, position, offsets, st);
}

extern "C" int t81b200_gather_rows(const void *x, int dtype, int64_t ld, int64_t tokens, int64_t top, int64_t width, const int32_t *position, const int32_t *kept, void *rows,
                                   void *stream) {
    if (int rc = check_rows("gather_rows", tokens, top, width, ld)) return rc;
    if (dtype < T81B200_F32 || dtype > T81B200_F16) return fail(T81B200_EINVAL, "gather_rows: unknown dtype %d", dtype);
    if (int rc = check_device()) return rc;
    if (tokens == 0 || width == 0) return T81B200_OK;
    if (!x || !position || !kept || !rows) return fail(T81B200_EINVAL, "gather_rows: null pointer");
    const int64_t size = (int64_t)dtype_size(dtype);
    const bool vec = width * size % 16 == 0 && ld * size % 16 == 0 && aligned16(x) && aligned16(rows);
    const int64_t pieces = vec ? width * size / 16 : width;
    const dim3 grid = row_grid(tokens, pieces);
    if (grid.y > 65535u) return fail(T81B200_ELIMIT, "gather_rows: rows too wide");
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const uint8_t *src = static_cast<const uint8_t *>(x);
    uint8_t *dst = static_cast<uint8_t *>(rows);
    if (vec) T81_CUDA_TRY(launch_behind(gather_rows_kernel<uint4>, grid, kThreads, 0, st, src, ld * size, tokens, (int)top, pieces, position, kept, dst));
    else if (size == 4) T81_CUDA_TRY(launch_behind(gather_rows_kernel<uint32_t>, grid, kThreads, 0, st, src, ld * size, tokens, (int)top, pieces, position, kept, dst));
    else T81_CUDA_TRY(launch_behind(gather_rows_kernel<uint16_t>, grid, kThreads, 0, st, src, ld * size, tokens, (int)top, pieces, position, kept, dst));
    return T81B200_OK;
}

extern "C" int t81b200_combine_rows(const void *rows, int dtype, int64_t ld, int64_t tokens, int64_t top, int64_t width, const int32_t *position, const void *weights, int w_dtype,
                                    void *y, void *stream) {
    if (int rc = check_rows("combine_rows", tokens, top, width, ld)) return rc;
    if (int rc = check_device()) return rc;
    if (tokens == 0 || width == 0) return T81B200_OK;
    if (!rows || !position || !y) return fail(T81B200_EINVAL, "combine_rows: null pointer");
    return by_types("combine_rows", dtype, w_dtype, [&](auto t, auto w) {
        return launch_combine<decltype(t), decltype(w)>(rows, ld, tokens, (int)top, width, position, weights, y, static_cast<cudaStream_t>(stream));
    });
}

extern "C" int t81b200_combine_rows_grad(const void *grad_y, int64_t ld_y, const void *rows, int dtype, int64_t ld, int64_t tokens, int64_t top, int64_t width, const int32_t *position,
                                         const int32_t *kept, const void *weights, int w_dtype, void *grad_rows, void *grad_weights, void *stream) {
    if (int rc = check_rows("combine_rows_grad", tokens, top, width, ld)) return rc;
    if (ld_y < width) return fail(T81B200_EINVAL, "combine_rows_grad: bad dimensions");
    if (int rc = check_device()) return rc;
    if (tokens == 0) return T81B200_OK;
    if (!position || !kept || (width > 0 && (!grad_y || !rows))) return fail(T81B200_EINVAL, "combine_rows_grad: null pointer");
    return by_types("combine_rows_grad", dtype, w_dtype, [&](auto t, auto w) {
        return launch_combine_grad<decltype(t), decltype(w)>(grad_y, ld_y, rows, ld, tokens, (int)top, width, position, kept, weights, grad_rows, grad_weights,
                                                             static_cast<cudaStream_t>(stream));
    });
}
