// ops_orth.cu -- orthogonalising matrix updates by Newton-Schulz products.
//
//   X = M / (|M|_F + eps)   (transposed where M has more rows than columns)
//   `steps` times:  A = X X^T,  P = aI + bA + cA^2,  X = P X
//   (a, b, c) = (3.4445, -4.7750, 2.0315); the result is X in bf16.
//
// The quintic moves every singular value of M towards 1 and leaves the
// singular vectors; small singular values grow by a = 3.4445 a step, and so
// does whatever rounding has put beside them.  One bf16 rounding of X a step
// (2^-9) would come out up to 3.4445^5 = 485 times larger in the weak
// directions, so matrices are kept as pairs of fp16, high + low part, 22 bits:
// hi hi' + hi lo' + lo hi' are three tensor-core products into one fp32
// accumulator.  Norms of X stay below 1.3 and of P below 3.5, so a fixed factor
// 2^12 keeps both parts well inside fp16's range; it leaves as an exact power
// of two.
//
// Each step is three launches over tiles of 128 rows, A and P only on and
// above the diagonal (both are symmetric; a tile is written to both sides).
// tcgen05 reads both operands K-major: X for X X^T, and its transpose for P X,
// so the last product's epilogue writes both.
#include "ops_common.h"
#include "tc05.cuh"

namespace nesle {
namespace ops {
namespace {

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr float kScale = 4096.f;  // stored matrix = kScale * matrix

__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

__device__ __forceinline__ void split(float v, __half& hi, __half& lo) {
    hi = __float2half_rn(v);
    lo = __float2half_rn(v - __half2float(hi));
}

union Half8 {
    __half h[8];
    uint4 u;
};

// ----------------------------------------------------- norm, scaling, layout

constexpr int kNormThreads = 256;
constexpr int kNormRuns = 8;  // loads in flight a thread

// Partial sums of squares: block (i, b) takes every gridDim.x-th run of 2,048 loads of matrix b, row after row.  In 64
// bits: no update is too small or too large to be squared, and the partials are added in a fixed order.  4,096 x 2,048 bf16:
// 7.1 us.
template <class T>
__global__ void __launch_bounds__(kNormThreads) square_sums_kernel(const T* __restrict__ x, int64_t stride_b, int64_t stride_r,
                                                                  int64_t stride_c, uint32_t rows, uint32_t cols,
                                                                  double* __restrict__ partial) {
    grid_launch_next();
    const T* m = x + blockIdx.y * stride_b;
    double sum = 0;
    // Along the denser dimension, so that a warp's loads lie together; one long row where rows follow one another.
    const bool by_row = stride_c <= stride_r;
    const int64_t so = by_row ? stride_r : stride_c, si = by_row ? stride_c : stride_r;
    uint64_t outer = by_row ? rows : cols, inner = by_row ? cols : rows;
    if (so == static_cast<int64_t>(inner) * si) inner *= outer, outer = 1;
    // 16 bytes a load where every row is whole chunks on 16 bytes.
    constexpr uint32_t kPer = 16 / sizeof(T);
    const bool vector = si == 1 && inner % kPer == 0 && (outer == 1 || so % kPer == 0) && reinterpret_cast<uintptr_t>(m) % 16 == 0;
    const uint32_t run = kNormThreads * kNormRuns * (vector ? kPer : 1);
    const uint64_t runs = (inner + run - 1) / run;
    for (uint64_t i = blockIdx.x; i < outer * runs; i += gridDim.x) {
        const uint64_t o = outer == 1 ? 0 : i / runs, first = (outer == 1 ? i : i % runs) * run;
        const T* from = m + static_cast<int64_t>(o) * so;
        if (vector) {
            uint4 v[kNormRuns];
#pragma unroll
            for (int k = 0; k < kNormRuns; ++k) {
                const uint64_t e = first + (k * kNormThreads + threadIdx.x) * kPer;
                v[k] = e < inner ? __ldg(reinterpret_cast<const uint4*>(from + e)) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int k = 0; k < kNormRuns; ++k)
#pragma unroll
                for (uint32_t j = 0; j < kPer; ++j) {
                    const double e = to_f32(reinterpret_cast<const T*>(&v[k])[j]);
                    sum += e * e;
                }
        } else {
            float v[kNormRuns];
#pragma unroll
            for (int k = 0; k < kNormRuns; ++k) {
                const uint64_t e = first + k * kNormThreads + threadIdx.x;
                v[k] = e < inner ? to_f32(from[static_cast<int64_t>(e) * si]) : 0.f;
            }
#pragma unroll
            for (int k = 0; k < kNormRuns; ++k) sum += static_cast<double>(v[k]) * v[k];
        }
    }
    __shared__ double part[kNormThreads / 32];
#pragma unroll
    for (int d = 16; d; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < kNormThreads / 32; ++i) sum += part[i];
        partial[blockIdx.y * gridDim.x + blockIdx.x] = sum;
    }
}

// X = kScale M / (|M| + eps) as fp16 pairs, and its transpose, by tiles of 64 x 64 of X: high part, then low part, each
// rows x ld.  Four times the input is written: 32 us for 4,096 x 2,048 bf16, 2.6 TB/s.
constexpr int kMostPartials = 256;  // one a thread

template <class T>
__global__ void __launch_bounds__(256) scale_kernel(const T* __restrict__ x, int64_t stride_b, int64_t stride_r, int64_t stride_c,
                                                    uint32_t m, uint32_t n, const double* __restrict__ partial, uint32_t partials,
                                                    double eps, __half* __restrict__ out, uint32_t ld, __half* __restrict__ out_t,
                                                    uint32_t ld_t) {
    __shared__ float tile[64][65];
    __shared__ double part[8];
    grid_launch_next();
    const T* mat = x + blockIdx.z * stride_b;
    const uint32_t r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
    const bool by_row = stride_c <= stride_r;
    float v[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) {  // the caller's matrix: nothing before this launch writes it
        const int i = threadIdx.x + k * 256, r = by_row ? i / 64 : i % 64, c = by_row ? i % 64 : i / 64;
        v[k] = r0 + r < m && c0 + c < n ? to_f32(mat[static_cast<int64_t>(r0 + r) * stride_r + static_cast<int64_t>(c0 + c) * stride_c]) : 0.f;
    }
    grid_wait();
    double sum = threadIdx.x < partials ? partial[blockIdx.z * partials + threadIdx.x] : 0.0;
#pragma unroll
    for (int d = 16; d; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = sum;
    __syncthreads();
    sum = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += part[i];
    const double norm = sqrt(sum) + eps;
    const double factor = norm == 0 ? 0 : static_cast<double>(kScale) / norm;  // a matrix of zeros with eps = 0 stays zero
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        const int i = threadIdx.x + k * 256, r = by_row ? i / 64 : i % 64, c = by_row ? i % 64 : i / 64;
        tile[r][c] = static_cast<float>(v[k] * factor);
    }
    __syncthreads();
    __half* hi = out + static_cast<uint64_t>(blockIdx.z) * 2 * m * ld;
    __half* hi_t = out_t + static_cast<uint64_t>(blockIdx.z) * 2 * n * ld_t;
#pragma unroll
    for (int k = 0; k < 2; ++k) {  // 8 values a store; ld and ld_t are multiples of 8
        const uint32_t i = threadIdx.x + k * 256, a = i / 8, b = i % 8 * 8;
        Half8 h, l;
        if (r0 + a < m && c0 + b < n) {
#pragma unroll
            for (int q = 0; q < 8; ++q) split(tile[a][b + q], h.h[q], l.h[q]);
            const uint64_t at = static_cast<uint64_t>(r0 + a) * ld + c0 + b;
            *reinterpret_cast<uint4*>(hi + at) = h.u;
            *reinterpret_cast<uint4*>(hi + static_cast<uint64_t>(m) * ld + at) = l.u;
        }
        if (c0 + a < n && r0 + b < m) {
#pragma unroll
            for (int q = 0; q < 8; ++q) split(tile[b + q][a], h.h[q], l.h[q]);
            const uint64_t at = static_cast<uint64_t>(c0 + a) * ld_t + r0 + b;
            *reinterpret_cast<uint4*>(hi_t + at) = h.u;
            *reinterpret_cast<uint4*>(hi_t + static_cast<uint64_t>(n) * ld_t + at) = l.u;
        }
    }
}

// ------------------------------------------------------------------ products

enum Product { kGram, kPoly, kApply, kLast };

struct Job {
    uint32_t m, n, k;       // result m x n, sums over k
    uint32_t tiles_m, tiles_n;
    __half* out;            // result as fp16 pairs [2][m][ld]
    uint32_t ld;
    __half* out_t;          // and transposed [2][n][ld_t]; of a symmetric result the same matrix
    uint32_t ld_t;
    const __half* gram;     // kPoly: A as pairs [2][m][ld]
    __nv_bfloat16* last;    // kLast: the caller's result, [batch][m][n], or [batch][n][m] where `last_t`
    int last_t;
};

constexpr uint32_t kTile = 128, kSlice = 64;  // rows of a tile, k of a stage
constexpr int kThreads = 256;

template <int kBN>  // columns of a tile
struct Shape {
    static constexpr int kStages = 3;
    static constexpr int kA = kTile * kSlice * 2, kB = kBN * kSlice * 2;  // one fp16 part of an operand
    static constexpr int kStageBytes = 2 * (kA + kB);                     // A high, A low, B high, B low
    // A block's columns of a tile from every block of its cluster: rows of kBN / split floats, padded by 4.
    static constexpr int kShares = kBN == 64 ? 4 * kTile * (kBN / 4 + 4) * 4 : 0;
    static constexpr int kSmem = 1024 + kStages * kStageBytes + kShares + 256;
    static_assert(8 * 4 * 32 * 40 * 2 <= kStages * kStageBytes, "the warps' blocks of results take the place of the operands");
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_address(const void* p, uint32_t rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(tc::smem_u32(p)), "r"(rank));
    return at;
}

// A warp's 8 columns on their way to transposed storage: 32 rows of each, high and low parts.
struct alignas(16) WarpTile {
    __half h[2][8][40];  // 80 bytes a column: 16-byte reads of 8 columns fall on all banks
};

// Columns j..j+7 of row i0 + lane of a product, from its accumulators, by a whole warp; `mirror`: and transposed, which
// goes through shared memory so that a store is 8 rows of a column.
template <int kProduct>
__device__ __forceinline__ void emit_run(const Job& job, uint32_t batch, uint32_t i0, uint32_t j, bool mirror, const float (&acc)[8],
                                         WarpTile& wt, int lane) {
    const uint64_t plane = static_cast<uint64_t>(job.m) * job.ld, plane_t = static_cast<uint64_t>(job.n) * job.ld_t;
    if (i0 >= job.m || j >= job.n) return;  // the same for the warp
    const uint32_t i = i0 + lane;
    const bool inside = i < job.m;
    float f[8];
    const uint64_t at = static_cast<uint64_t>(i) * job.ld + j;
    if constexpr (kProduct == kPoly) {
        Half8 gh, gl;
        gh.u = gl.u = make_uint4(0, 0, 0, 0);
        if (inside) {
            const __half* g = job.gram + batch * 2 * plane + at;
            gh.u = *reinterpret_cast<const uint4*>(g);
            gl.u = *reinterpret_cast<const uint4*>(g + plane);
        }
#pragma unroll
        for (int q = 0; q < 8; ++q)
            f[q] = fmaf(kB, __half2float(gh.h[q]) + __half2float(gl.h[q]), fmaf(kC / kScale, acc[q], i == j + q ? kA * kScale : 0.f));
    } else {
        constexpr float kBack = kProduct == kLast ? 1.f / (kScale * kScale) : 1.f / kScale;
#pragma unroll
        for (int q = 0; q < 8; ++q) f[q] = acc[q] * kBack;
    }
    // what a lane stores of the transpose: 8 rows of column lane / 4
    const uint32_t tj = j + lane / 4, ti = i0 + lane % 4 * 8;
    const bool t_inside = tj < job.n && ti < job.m;
    if constexpr (kProduct == kLast) {
        union Bf8 {
            __nv_bfloat16 h[8];
            uint4 u;
        } b;
#pragma unroll
        for (int q = 0; q < 8; ++q) b.h[q] = __float2bfloat16_rn(f[q]);
        if (!job.last_t) {
            if (!inside) return;
            __nv_bfloat16* o = job.last + (static_cast<uint64_t>(batch) * job.m + i) * job.n + j;
            if (job.n % 8 == 0) {
                *reinterpret_cast<uint4*>(o) = b.u;
            } else {
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (j + q < job.n) o[q] = b.h[q];
            }
            return;
        }
        __nv_bfloat16(*tile)[40] = reinterpret_cast<__nv_bfloat16(*)[40]>(wt.h[0]);
#pragma unroll
        for (int q = 0; q < 8; ++q) tile[q][lane] = b.h[q];
        __syncwarp();
        if (t_inside) {
            b.u = *reinterpret_cast<const uint4*>(&tile[lane / 4][lane % 4 * 8]);
            __nv_bfloat16* o = job.last + (static_cast<uint64_t>(batch) * job.n + tj) * job.m + ti;
            if (job.m % 8 == 0) {
                *reinterpret_cast<uint4*>(o) = b.u;
            } else {
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (ti + q < job.m) o[q] = b.h[q];
            }
        }
        __syncwarp();
    } else {
        Half8 h, l;
#pragma unroll
        for (int q = 0; q < 8; ++q) split(f[q], h.h[q], l.h[q]);
        if (inside) {
            __half* o = job.out + batch * 2 * plane + at;
            *reinterpret_cast<uint4*>(o) = h.u;
            *reinterpret_cast<uint4*>(o + plane) = l.u;
        }
        if (!mirror) return;
#pragma unroll
        for (int q = 0; q < 8; ++q) wt.h[0][q][lane] = h.h[q], wt.h[1][q][lane] = l.h[q];
        __syncwarp();
        if (t_inside) {
            __half* t = job.out_t + batch * 2 * plane_t + static_cast<uint64_t>(tj) * job.ld_t + ti;
            *reinterpret_cast<uint4*>(t) = *reinterpret_cast<const uint4*>(&wt.h[0][lane / 4][lane % 4 * 8]);
            *reinterpret_cast<uint4*>(t + plane_t) = *reinterpret_cast<const uint4*>(&wt.h[1][lane / 4][lane % 4 * 8]);
        }
        __syncwarp();
    }
}

// 32 columns at once: a warp's 32 x 32 values of both parts and of their transposes, so that every access to global
// memory is 16 bytes a lane and 64 of a row (a lane a row, as emit_run stores, takes the memory pipe four times as long).
constexpr int kPitch = 40;  // 80 bytes a row: any 8 rows' 16-byte chunks fall on all banks
struct alignas(16) WarpBlock {
    __half h[2][32][kPitch], t[2][32][kPitch];
};

// h to t, transposed, by 8 x 8 blocks.
__device__ __forceinline__ void transpose_block(const __half (&h)[32][kPitch], __half (&t)[32][kPitch], int lane) {
#pragma unroll
    for (int c = 0; c < 32; c += 8) {
        uint32_t r[4];
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(tc::smem_u32(&h[lane][c]))
                     : "memory");
        asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(tc::smem_u32(&t[c + lane % 8][lane / 8 * 8])), "r"(r[0]),
                     "r"(r[1]), "r"(r[2]), "r"(r[3])
                     : "memory");
    }
}

// Rows of a warp's block to a row-major matrix of rows x cols, `ld` apart.
template <class T>
__device__ __forceinline__ void store_block(T* out, uint64_t ld, uint32_t rows, uint32_t cols, uint32_t r0, uint32_t c0, const __half (&h)[32][kPitch],
                                            bool vector, int lane) {
    const uint32_t c = c0 + lane % 4 * 8;
#pragma unroll
    for (int k = 0; k < 32; k += 8) {
        const uint32_t r = r0 + k + lane / 4;
        if (r >= rows || c >= cols) continue;
        const uint4 x = *reinterpret_cast<const uint4*>(&h[k + lane / 4][lane % 4 * 8]);
        T* to = out + r * ld + c;
        if (vector) {
            *reinterpret_cast<uint4*>(to) = x;
        } else {
            const T* v = reinterpret_cast<const T*>(&x);
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (c + q < cols) to[q] = v[q];
        }
    }
}

template <int kProduct>
__device__ __forceinline__ void emit_block(const Job& job, uint32_t batch, uint32_t i0, uint32_t j0, bool mirror, const uint32_t (&acc)[32],
                                           WarpBlock& wb, int lane) {
    if (i0 >= job.m || j0 >= job.n) return;  // the same for the warp
    const uint64_t plane = static_cast<uint64_t>(job.m) * job.ld, plane_t = static_cast<uint64_t>(job.n) * job.ld_t;
    if constexpr (kProduct == kPoly) {
        const __half* g = job.gram + batch * 2 * plane;
        const uint32_t c = j0 + lane % 4 * 8;
        uint4 x[2][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t r = i0 + k * 8 + lane / 4;
            const bool in = r < job.m && c < job.n;
            x[0][k] = in ? *reinterpret_cast<const uint4*>(g + static_cast<uint64_t>(r) * job.ld + c) : make_uint4(0, 0, 0, 0);
            x[1][k] = in ? *reinterpret_cast<const uint4*>(g + plane + static_cast<uint64_t>(r) * job.ld + c) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            *reinterpret_cast<uint4*>(&wb.t[0][k * 8 + lane / 4][lane % 4 * 8]) = x[0][k];
            *reinterpret_cast<uint4*>(&wb.t[1][k * 8 + lane / 4][lane % 4 * 8]) = x[1][k];
        }
        __syncwarp();
    }
    const uint32_t i = i0 + lane;
#pragma unroll
    for (int q8 = 0; q8 < 32; q8 += 8) {
        Half8 h, l, gh, gl;
        if constexpr (kProduct == kPoly) {
            gh.u = *reinterpret_cast<const uint4*>(&wb.t[0][lane][q8]);
            gl.u = *reinterpret_cast<const uint4*>(&wb.t[1][lane][q8]);
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            float f = __uint_as_float(acc[q8 + q]);
            if constexpr (kProduct == kPoly)
                f = fmaf(kB, __half2float(gh.h[q]) + __half2float(gl.h[q]), fmaf(kC / kScale, f, i == j0 + q8 + q ? kA * kScale : 0.f));
            else
                f *= kProduct == kLast ? 1.f / (kScale * kScale) : 1.f / kScale;
            if constexpr (kProduct == kLast) {
                const __nv_bfloat16 b = __float2bfloat16_rn(f);
                h.h[q] = reinterpret_cast<const __half&>(b);  // 16 bits to be moved
            } else {
                split(f, h.h[q], l.h[q]);
            }
        }
        *reinterpret_cast<uint4*>(&wb.h[0][lane][q8]) = h.u;
        if constexpr (kProduct != kLast) *reinterpret_cast<uint4*>(&wb.h[1][lane][q8]) = l.u;
    }
    __syncwarp();
    if constexpr (kProduct == kLast) {
        __nv_bfloat16* out = job.last + static_cast<uint64_t>(batch) * job.m * job.n;
        if (job.last_t) {
            transpose_block(wb.h[0], wb.t[0], lane);
            __syncwarp();
            store_block(out, job.m, job.n, job.m, j0, i0, wb.t[0], job.m % 8 == 0, lane);
        } else {
            store_block(out, job.n, job.m, job.n, i0, j0, wb.h[0], job.n % 8 == 0, lane);
        }
    } else {
        __half* out = job.out + batch * 2 * plane;
        store_block(out, job.ld, job.m, job.n, i0, j0, wb.h[0], true, lane);
        store_block(out + plane, job.ld, job.m, job.n, i0, j0, wb.h[1], true, lane);
        if (mirror) {
            transpose_block(wb.h[0], wb.t[0], lane);
            transpose_block(wb.h[1], wb.t[1], lane);
            __syncwarp();
            __half* out_t = job.out_t + batch * 2 * plane_t;
            store_block(out_t, job.ld_t, job.n, job.m, j0, i0, wb.t[0], true, lane);
            store_block(out_t + plane_t, job.ld_t, job.n, job.m, j0, i0, wb.t[1], true, lane);
        }
    }
    __syncwarp();
}

// One tile by a cluster of kSplit blocks, each over its share of k; every block sends the others their columns of its
// fp32 sums and adds up its own from all, in the order of the ranks.  (Fetching them from the others' shared memory took
// 4,000 to 6,000 clocks, sending them takes 1,400.)  A product of a 256 x 256 matrix takes 7 to 8 us by itself
// (ncu) and 5.5 in its chain, where a launch starts under the one before: its slices are 3, the epilogue 1 to 2
// and the rest starting and draining.
template <int kProduct, int kBN, int kSplit>
__global__ void __launch_bounds__(kThreads, 1)
    product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, Job job, unsigned int* stalls) {
    using S = Shape<kBN>;
    constexpr int kStages = S::kStages;
    constexpr bool kSymmetric = kProduct == kGram || kProduct == kPoly;
    extern __shared__ uint8_t raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    float* shares = reinterpret_cast<float*>(base + kStages * S::kStageBytes);
    uint64_t* full = reinterpret_cast<uint64_t*>(base + kStages * S::kStageBytes + S::kShares);
    uint64_t* empty = full + kStages;
    uint64_t* done = empty + kStages;
    uint32_t* slot = reinterpret_cast<uint32_t*>(done + 1);

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t rank = kSplit > 1 ? cluster_rank() : 0, batch = blockIdx.y;
    uint32_t ti, tj;
    {
        uint32_t t = blockIdx.x / kSplit;
        if constexpr (kSymmetric) {  // row ti holds the tiles from its diagonal block on
            ti = 0;
            for (uint32_t left = job.tiles_n; t >= left; left -= kTile / kBN, ++ti) t -= left;
            tj = ti * (kTile / kBN) + t;
        } else {
            ti = t % job.tiles_m;  // neighbours share X's columns
            tj = t / job.tiles_m;
        }
    }
    const uint32_t slices = (job.k + kSlice - 1) / kSlice;
    const uint32_t first = slices * rank / kSplit, last = slices * (rank + 1) / kSplit;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) {
            tc::mbar_init(&full[i], 1);
            tc::mbar_init(&empty[i], 1);
        }
        tc::mbar_init(done, 1);
        tc::mbar_init_fence();
        tc::prefetch_map(&map_a);
        tc::prefetch_map(&map_b);
    }
    if (warp == 1) tc::tmem_alloc(slot, kBN);
    tc::fence_before();
    if constexpr (kSplit > 1)
        cluster_sync();  // the others' shared memory is there
    else
        __syncthreads();
    tc::fence_after();
    const uint32_t tmem = *slot;
    grid_launch_next();
    grid_wait();  // what the launches before this one wrote
    bool ok = true;

    if (warp == 0 && tc::elect_one()) {
        uint32_t it = 0;
        for (uint32_t s = first; s < last; ++s, ++it) {
            const uint32_t i = it % kStages;
            if (!(ok = tc::mbar_wait(&empty[i], (it / kStages & 1) ^ 1))) break;
            uint8_t* st = base + i * S::kStageBytes;
            tc::mbar_expect_tx(&full[i], S::kStageBytes);
            tc::tma_load_3d(st, &map_a, &full[i], s * kSlice, ti * kTile, batch * 2);
            tc::tma_load_3d(st + 2 * S::kA, &map_b, &full[i], s * kSlice, tj * kBN, batch * 2);
            tc::tma_load_3d(st + S::kA, &map_a, &full[i], s * kSlice, ti * kTile, batch * 2 + 1);
            tc::tma_load_3d(st + 2 * S::kA + S::kB, &map_b, &full[i], s * kSlice, tj * kBN, batch * 2 + 1);
        }
        for (uint32_t s = it < kStages ? 0 : it - kStages; s < it; ++s)  // a load in flight lands before the block goes on
            ok = tc::mbar_wait(&full[s % kStages], s / kStages & 1) && ok;
    } else if (warp == 1 && tc::elect_one()) {
        constexpr uint32_t idesc = tc::idesc_f16(kBN);
        uint32_t it = 0;
        for (uint32_t s = first; s < last; ++s, ++it) {
            const uint32_t i = it % kStages;
            if (!(ok = tc::mbar_wait(&full[i], it / kStages & 1))) break;
            tc::fence_after();
            const uint8_t* st = base + i * S::kStageBytes;
            const uint64_t ah = tc::tile_desc(st), al = tc::tile_desc(st + S::kA), bh = tc::tile_desc(st + 2 * S::kA),
                           bl = tc::tile_desc(st + 2 * S::kA + S::kB);
#pragma unroll
            for (int kk = 0; kk < kSlice / 16; ++kk) {
                tc::mma_f16(tmem, al + 2 * kk, bh + 2 * kk, idesc, it > 0 || kk > 0);
                tc::mma_f16(tmem, ah + 2 * kk, bl + 2 * kk, idesc, true);
                tc::mma_f16(tmem, ah + 2 * kk, bh + 2 * kk, idesc, true);
            }
            tc::mma_commit(&empty[i]);
        }
        tc::mma_commit(done);
    }
    __syncwarp();
    ok = tc::mbar_wait_warp(done, 0) && ok;
    tc::fence_after();

    // This thread's row, and its columns: of its half of the tile, the rank's share.
    const int r = (warp % 4) * 32 + lane, half = warp / 4;
    constexpr int kHalf = kBN / 2, kMine = kHalf / kSplit;
    const uint32_t at_tmem = tmem + (static_cast<uint32_t>((warp % 4) * 32) << 16) + half * kHalf;
    const bool mirror = kProduct == kLast ? job.last_t : kProduct == kApply || (tj * kBN) / kTile != ti;

    __shared__ WarpTile warp_tiles[kThreads / 32];
    auto emit = [&](int c, const float (&acc)[8]) {
        emit_run<kProduct>(job, batch, ti * kTile + (warp % 4) * 32, tj * kBN + c, mirror, acc, warp_tiles[warp], lane);
    };
    if constexpr (kSplit == 1) {
        __syncthreads();  // nobody reads the operands any more
        WarpBlock* blocks = reinterpret_cast<WarpBlock*>(base);
#pragma unroll
        for (int c = 0; c < kHalf; c += 32) {
            uint32_t v[32];
            tc::tmem_ld32(at_tmem + c, v);
            tc::tmem_wait_ld();
            emit_block<kProduct>(job, batch, ti * kTile + (warp % 4) * 32, tj * kBN + half * kHalf + c, mirror, v, blocks[warp], lane);
        }
        tc::fence_before();
        __syncthreads();
        tc::fence_after();
        if (warp == 1) tc::tmem_free(tmem, kBN);
    } else {
        static_assert(kHalf == 32, "one load of tensor memory");
        constexpr int kPitch = kBN / kSplit + 4;
        uint32_t v[32];
        tc::tmem_ld32(at_tmem, v);
        tc::tmem_wait_ld();
#pragma unroll
        for (int x = 0; x < 32; x += 4) {
            const uint32_t at = peer_address(shares + (rank * kTile + r) * kPitch + half * kMine + x % kMine, x / kMine);
            asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v[x]), "r"(v[x + 1]), "r"(v[x + 2]), "r"(v[x + 3])
                         : "memory");
        }
        tc::fence_before();
        cluster_sync();
        tc::fence_after();
        if (warp == 1) tc::tmem_free(tmem, kBN);
#pragma unroll
        for (int c = 0; c < kMine; c += 8) {
            float acc[8] = {};
#pragma unroll
            for (int p = 0; p < kSplit; ++p) {
                const float* from = shares + (p * kTile + r) * kPitch + half * kMine + c;
                const float4 x = *reinterpret_cast<const float4*>(from), y = *reinterpret_cast<const float4*>(from + 4);
                acc[0] += x.x, acc[1] += x.y, acc[2] += x.z, acc[3] += x.w;
                acc[4] += y.x, acc[5] += y.y, acc[6] += y.z, acc[7] += y.w;
            }
            emit(half * kHalf + rank * kMine + c, acc);
        }
    }
    if (!ok) atomicAdd(stalls, 1u);
}

// Large matrices: tiles of 256 x 256, one a block, two accumulators of 128 x 256 that fill tensor memory.  What bounds
// the 128 x 128 tiles is their operands' way from L2 (48 bytes a clock and SM when all SMs read): 64 KB for 768 clocks of
// products.  Here 64 KB, a slice of 32, feed 1,536 clocks.  2,048 x 2,048 by 2,048 x 4,096: 87 us for three products,
// 1.2 PFLOP/s, 70% of what a bf16 library product reaches here.
struct Wide {
    static constexpr uint32_t kSide = 256, kSlice = 32;
    static constexpr int kStages = 3;
    static constexpr int kPart = kSide * kSlice * 2, kStageBytes = 4 * kPart;  // A high, A low, B high, B low
    static constexpr int kSmem = 1024 + kStages * kStageBytes + 256;
    static_assert(8 * sizeof(WarpBlock) <= kStages * kStageBytes, "the warps' blocks of results take the place of the operands");
};

template <int kProduct>
__global__ void __launch_bounds__(kThreads, 1)
    wide_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, Job job, unsigned int* stalls) {
    constexpr int kStages = Wide::kStages;
    constexpr uint32_t kSide = Wide::kSide;
    extern __shared__ uint8_t raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(base + kStages * Wide::kStageBytes);
    uint64_t* empty = full + kStages;
    uint64_t* done = empty + kStages;
    uint32_t* slot = reinterpret_cast<uint32_t*>(done + 1);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t batch = blockIdx.y;
    uint32_t ti, tj;
    {
        uint32_t t = blockIdx.x;
        if constexpr (kProduct == kGram || kProduct == kPoly) {
            ti = 0;
            for (uint32_t left = job.tiles_n; t >= left; --left, ++ti) t -= left;
            tj = ti + t;
        } else {
            ti = t % job.tiles_m;
            tj = t / job.tiles_m;
        }
    }
    const uint32_t slices = (job.k + Wide::kSlice - 1) / Wide::kSlice;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) {
            tc::mbar_init(&full[i], 1);
            tc::mbar_init(&empty[i], 1);
        }
        tc::mbar_init(done, 1);
        tc::mbar_init_fence();
        tc::prefetch_map(&map_a);
        tc::prefetch_map(&map_b);
    }
    if (warp == 1) tc::tmem_alloc(slot, 512);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = *slot;
    grid_launch_next();
    grid_wait();
    bool ok = true;
    if (warp == 0 && tc::elect_one()) {
        uint32_t it = 0;
        for (uint32_t s = 0; s < slices; ++s, ++it) {
            const uint32_t i = it % kStages;
            if (!(ok = tc::mbar_wait(&empty[i], (it / kStages & 1) ^ 1))) break;
            uint8_t* st = base + i * Wide::kStageBytes;
            tc::mbar_expect_tx(&full[i], Wide::kStageBytes);
            for (int part = 0; part < 2; ++part) {
                tc::tma_load_3d(st + part * Wide::kPart, &map_a, &full[i], s * Wide::kSlice, ti * kSide, batch * 2 + part);
                tc::tma_load_3d(st + (2 + part) * Wide::kPart, &map_b, &full[i], s * Wide::kSlice, tj * kSide, batch * 2 + part);
            }
        }
        for (uint32_t s = it < kStages ? 0 : it - kStages; s < it; ++s)  // a load in flight lands before the block goes on
            ok = tc::mbar_wait(&full[s % kStages], s / kStages & 1) && ok;
    } else if (warp == 1 && tc::elect_one()) {
        constexpr uint32_t idesc = tc::idesc_f16(kSide);
        uint32_t it = 0;
        for (uint32_t s = 0; s < slices; ++s, ++it) {
            const uint32_t i = it % kStages;
            if (!(ok = tc::mbar_wait(&full[i], it / kStages & 1))) break;
            tc::fence_after();
            const uint8_t* st = base + i * Wide::kStageBytes;
            const uint64_t bh = tc::tile_desc64(st + 2 * Wide::kPart), bl = tc::tile_desc64(st + 3 * Wide::kPart);
#pragma unroll
            for (int h = 0; h < 2; ++h) {  // rows 128 h and on
                const uint64_t ah = tc::tile_desc64(st + h * (Wide::kPart / 2)), al = tc::tile_desc64(st + Wide::kPart + h * (Wide::kPart / 2));
#pragma unroll
                for (int kk = 0; kk < Wide::kSlice / 16; ++kk) {
                    tc::mma_f16(tmem + h * kSide, al + 2 * kk, bh + 2 * kk, idesc, it > 0 || kk > 0);
                    tc::mma_f16(tmem + h * kSide, ah + 2 * kk, bl + 2 * kk, idesc, true);
                    tc::mma_f16(tmem + h * kSide, ah + 2 * kk, bh + 2 * kk, idesc, true);
                }
            }
            tc::mma_commit(&empty[i]);
        }
        tc::mma_commit(done);
    }
    __syncwarp();
    ok = tc::mbar_wait_warp(done, 0) && ok;
    tc::fence_after();
    __syncthreads();  // nobody reads the operands any more
    const bool mirror = kProduct == kLast ? job.last_t : kProduct == kApply || tj != ti;
    WarpBlock& mine = reinterpret_cast<WarpBlock*>(base)[warp];
    const uint32_t at = tmem + (static_cast<uint32_t>((warp % 4) * 32) << 16) + warp / 4 * kSide;
#pragma unroll 1
    for (uint32_t c = 0; c < kSide; c += 32) {
        uint32_t v[32];
        tc::tmem_ld32(at + c, v);
        tc::tmem_wait_ld();
        emit_block<kProduct>(job, batch, ti * kSide + warp / 4 * kTile + (warp % 4) * 32, tj * kSide + c, mirror, v, mine, lane);
    }
    if (!ok) atomicAdd(stalls, 1u);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    if (warp == 1) tc::tmem_free(tmem, 512);
}

// ----------------------------------------------------------------------- host

uint32_t up8(uint32_t v) { return (v + 7) / 8 * 8; }
uint64_t up256(uint64_t v) { return (v + 255) / 256 * 256; }
constexpr uint32_t kNormBlocks = kMostPartials;

uint32_t norm_blocks(uint64_t elements) {  // one run each while that is fewer
    const uint64_t runs = (elements + kNormThreads * kNormRuns - 1) / (kNormThreads * kNormRuns);
    return static_cast<uint32_t>(runs < kNormBlocks ? runs : kNormBlocks);
}

struct Layout {  // byte offsets of the workspace's parts
    uint32_t m, n, ld_n, ld_m;
    uint64_t partial, x[2], xt[2], gram, poly, bytes;
    explicit Layout(const nesle_orth_args& a) {
        m = static_cast<uint32_t>(a.rows < a.cols ? a.rows : a.cols);
        n = static_cast<uint32_t>(a.rows < a.cols ? a.cols : a.rows);
        ld_n = up8(n);
        ld_m = up8(m);
        const uint64_t mn = up256(a.batch * 4ull * m * ld_n), nm = up256(a.batch * 4ull * n * ld_m), mm = up256(a.batch * 4ull * m * ld_m);
        bytes = 0;
        auto take = [&](uint64_t n_) {
            const uint64_t at = bytes;
            bytes += n_;
            return at;
        };
        partial = take(up256(a.batch * kNormBlocks * sizeof(double)));
        x[0] = take(mn), x[1] = take(mn), xt[0] = take(nm), xt[1] = take(nm), gram = take(mm), poly = take(mm);
    }
};

int map_pair(CUtensorMap* map, const void* p, uint32_t rows, uint32_t cols, uint32_t ld, uint64_t batch, uint32_t box_rows) {
    const bool wide = box_rows == Wide::kSide;
    const uint64_t dims[3] = {cols, rows, batch * 2}, strides[2] = {ld * 2ull, static_cast<uint64_t>(rows) * ld * 2};
    const uint32_t box[3] = {wide ? Wide::kSlice : kSlice, box_rows, 1};
    return encode_map(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, p, dims, strides, box, wide ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int kProduct, int kBN, int kSplit>
int launch_product(const CUtensorMap& ma, const CUtensorMap& mb, const Job& job, uint32_t tiles, uint32_t batch, int device,
                   unsigned int* stalls, cudaStream_t st) {
    constexpr auto* kernel = [] {
        if constexpr (kBN == Wide::kSide)
            return wide_kernel<kProduct>;
        else
            return product_kernel<kProduct, kBN, kSplit>;
    }();
    constexpr int kBytes = [] {
        if constexpr (kBN == Wide::kSide)
            return Wide::kSmem;
        else
            return Shape<kBN>::kSmem;
    }();
    if (int rc = allow_smem<kernel>(kBytes, device, "orthogonalize")) return rc;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(tiles * kSplit, batch);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kBytes;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = kSplit;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = kSplit > 1 ? 2 : 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, kernel, ma, mb, job, stalls), "orthogonalize");
}

struct Operand {  // a stored pair as either side of a product
    const void* p;
    uint32_t rows, cols, ld;
    uint64_t batch;
    int map(CUtensorMap* m, uint32_t box_rows) const { return map_pair(m, p, rows, cols, ld, batch, box_rows); }
};

uint32_t count_tiles(bool symmetric, Job& job, uint32_t bm, uint32_t bn) {
    job.tiles_m = (job.m + bm - 1) / bm;
    job.tiles_n = (job.n + bn - 1) / bn;
    if (!symmetric) return job.tiles_m * job.tiles_n;
    uint32_t tiles = 0;
    for (uint32_t i = 0; i < job.tiles_m; ++i) tiles += job.tiles_n - i * (bm / bn);
    return tiles;
}

// Narrow tiles, and k split over a cluster where it is long enough to pay for that, as long as all blocks run at once; else
// wide ones, which read their operands less often: 256 x 256 where they fill two thirds of the SMs (a product of 2,048 x
// 4,096: 128 tiles 87 us, 512 of 128 x 128 104 us; a Gram matrix of 2,048 has 36 and 136 tiles, 44 us with the latter).
template <int kProduct>
int launch_sized(const Operand& a, const Operand& b, Job job, uint32_t batch, int device, unsigned int* stalls, cudaStream_t st) {
    const uint64_t sms = sm_count(device);
    const bool symmetric = kProduct == kGram || kProduct == kPoly;
    CUtensorMap ma, mb;
    auto maps = [&](uint32_t rows_a, uint32_t rows_b) {
        const int rc = a.map(&ma, rows_a);
        return rc ? rc : b.map(&mb, rows_b);
    };
    const uint64_t narrow = static_cast<uint64_t>(count_tiles(symmetric, job, kTile, 64)) * batch;
    if (narrow <= sms) {
        if (int rc = maps(kTile, 64)) return rc;
        const uint32_t tiles = static_cast<uint32_t>(narrow / batch), slices = (job.k + kSlice - 1) / kSlice;
        // A slice takes 1,000 clocks, joining a cluster's shares 3,500.
        if (narrow * 4 <= sms && slices >= 8) return launch_product<kProduct, 64, 4>(ma, mb, job, tiles, batch, device, stalls, st);
        if (narrow * 2 <= sms && slices >= 8) return launch_product<kProduct, 64, 2>(ma, mb, job, tiles, batch, device, stalls, st);
        return launch_product<kProduct, 64, 1>(ma, mb, job, tiles, batch, device, stalls, st);
    }
    const uint32_t wide = count_tiles(symmetric, job, Wide::kSide, Wide::kSide);
    if (static_cast<uint64_t>(wide) * batch * 3 >= sms * 2) {
        if (int rc = maps(Wide::kSide, Wide::kSide)) return rc;
        return launch_product<kProduct, Wide::kSide, 1>(ma, mb, job, wide, batch, device, stalls, st);
    }
    if (int rc = maps(kTile, kTile)) return rc;
    const uint32_t tiles = count_tiles(symmetric, job, kTile, kTile);
    return launch_product<kProduct, kTile, 1>(ma, mb, job, tiles, batch, device, stalls, st);
}

template <class T>
int launch_scaling(const nesle_orth_args& a, const Layout& lay, uint8_t* ws, int64_t sr, int64_t sc, cudaStream_t st) {
    const T* x = static_cast<const T*>(a.x);
    double* partial = reinterpret_cast<double*>(ws + lay.partial);
    const uint32_t partials = norm_blocks(static_cast<uint64_t>(lay.m) * lay.n);
    square_sums_kernel<T><<<dim3(partials, static_cast<unsigned>(a.batch)), kNormThreads, 0, st>>>(x, a.stride_b, sr, sc, lay.m, lay.n, partial);
    if (int rc = cuda_status(cudaGetLastError(), "orthogonalize")) return rc;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((lay.n + 63) / 64, (lay.m + 63) / 64, static_cast<unsigned>(a.batch));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, scale_kernel<T>, x, a.stride_b, sr, sc, lay.m, lay.n, static_cast<const double*>(partial),
                                          partials, a.eps, reinterpret_cast<__half*>(ws + lay.x[0]), lay.ld_n,
                                          reinterpret_cast<__half*>(ws + lay.xt[0]), lay.ld_m),
                       "orthogonalize");
}

int run(const nesle_orth_args& a, cudaStream_t st) {
    const Layout lay(a);
    uint8_t* ws = static_cast<uint8_t*>(a.workspace);
    const bool tall = a.rows > a.cols;
    const int64_t sr = tall ? a.stride_c : a.stride_r, sc = tall ? a.stride_r : a.stride_c;
    const uint32_t batch = static_cast<uint32_t>(a.batch), m = lay.m, n = lay.n;
    int rc;
    unsigned int* stalls = nullptr;
    if ((rc = stall_counter(a.device, &stalls))) return rc;
    switch (a.dtype) {
        case NESLE_F32: rc = launch_scaling<float>(a, lay, ws, sr, sc, st); break;
        case NESLE_BF16: rc = launch_scaling<__nv_bfloat16>(a, lay, ws, sr, sc, st); break;
        default: rc = launch_scaling<__half>(a, lay, ws, sr, sc, st); break;
    }
    if (rc) return rc;
    __half *gram = reinterpret_cast<__half*>(ws + lay.gram), *poly = reinterpret_cast<__half*>(ws + lay.poly);
    const Operand op_x[2] = {{ws + lay.x[0], m, n, lay.ld_n, batch}, {ws + lay.x[1], m, n, lay.ld_n, batch}};
    const Operand op_xt[2] = {{ws + lay.xt[0], n, m, lay.ld_m, batch}, {ws + lay.xt[1], n, m, lay.ld_m, batch}};
    const Operand op_g{gram, m, m, lay.ld_m, batch}, op_p{poly, m, m, lay.ld_m, batch};
    for (int step = 0; step < a.steps; ++step) {
        const int from = step & 1, to = from ^ 1;
        Job g{};
        g.m = g.n = m, g.k = n;
        g.out = g.out_t = gram;
        g.ld = g.ld_t = lay.ld_m;
        if ((rc = launch_sized<kGram>(op_x[from], op_x[from], g, batch, a.device, stalls, st))) return rc;
        Job p = g;
        p.k = m;
        p.gram = gram;
        p.out = p.out_t = poly;
        if ((rc = launch_sized<kPoly>(op_g, op_g, p, batch, a.device, stalls, st))) return rc;
        Job x{};
        x.m = m, x.n = n, x.k = m;
        x.out = reinterpret_cast<__half*>(ws + lay.x[to]);
        x.ld = lay.ld_n;
        x.out_t = reinterpret_cast<__half*>(ws + lay.xt[to]);
        x.ld_t = lay.ld_m;
        x.last = static_cast<__nv_bfloat16*>(a.out);
        x.last_t = tall;
        rc = step + 1 < a.steps ? launch_sized<kApply>(op_p, op_xt[from], x, batch, a.device, stalls, st)
                                : launch_sized<kLast>(op_p, op_xt[from], x, batch, a.device, stalls, st);
        if (rc) return rc;
    }
    return NESLE_OK;
}

const char* check(const nesle_orth_args& a) {
    if (a.steps < 1) return "orthogonalize: steps must be at least 1";
    if (!(a.eps >= 0)) return "orthogonalize: eps must not be negative";
    if (a.dtype != NESLE_F32 && a.dtype != NESLE_BF16 && a.dtype != NESLE_F16) return "orthogonalize: unknown element type";
    if (a.rows > 65536 || a.cols > 65536) return "orthogonalize: at most 65536 rows or columns";
    if (a.batch > 65535) return "orthogonalize: at most 65535 matrices";
    return nullptr;
}

}  // namespace
}  // namespace ops
}  // namespace nesle

using namespace nesle;

extern "C" {

uint64_t nesle_orth_workspace(const nesle_orth_args* a) {
    if (!a || ops::check(*a) || !a->batch || !a->rows || !a->cols) return 0;
    return ops::Layout(*a).bytes;
}

int nesle_orthogonalize(const nesle_orth_args* args, void* stream) {
    return ops::guarded([&]() -> int {
        if (!args) return ops::invalid("orthogonalize: null argument");
        const nesle_orth_args& a = *args;
        if (const char* why = ops::check(a)) return ops::invalid(why);
        if (!a.batch || !a.rows || !a.cols) return NESLE_OK;
        if (!a.x || !a.out) return ops::invalid("orthogonalize: null argument");
        if (reinterpret_cast<uintptr_t>(a.out) % 16) return ops::invalid("orthogonalize: out must be 16-byte aligned");
        if (!ops::all_on(ops::element_size(a.dtype), a.x)) return ops::invalid("orthogonalize: x must be aligned to its elements");
        if (!a.workspace || a.workspace_bytes < nesle_orth_workspace(args) || reinterpret_cast<uintptr_t>(a.workspace) % 256)
            return ops::invalid("orthogonalize: the workspace is missing, too small or not 256-byte aligned");
        ops::OnDevice on(a.device);
        if (!on.ok) return ops::invalid("orthogonalize: device ordinal out of range");
        return ops::run(a, static_cast<cudaStream_t>(stream));
    });
}

}  // extern "C"
