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
// Each step is three launches over tiles of 128 x 128, A and P only on and
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

// ----------------------------------------------------- norm, scaling, layout

constexpr int kNormThreads = 256;

// Partial sums of squares: block (i, b) takes every gridDim.x-th run of elements of matrix b.  In 64 bits: no update is
// too small or too large to be squared, and the partials are added in a fixed order.
template <class T>
__global__ void __launch_bounds__(kNormThreads) square_sums_kernel(const T* __restrict__ x, int64_t stride_b, int64_t stride_r,
                                                                  int64_t stride_c, uint32_t rows, uint32_t cols,
                                                                  double* __restrict__ partial) {
    const T* m = x + blockIdx.y * stride_b;
    double sum = 0;
    // Along the denser dimension, so that a warp's loads lie together.
    const bool by_row = stride_c <= stride_r;
    const uint32_t outer = by_row ? rows : cols, inner = by_row ? cols : rows;
    const int64_t so = by_row ? stride_r : stride_c, si = by_row ? stride_c : stride_r;
    const uint32_t runs = (inner + kNormThreads - 1) / kNormThreads;
    for (uint64_t i = blockIdx.x; i < static_cast<uint64_t>(outer) * runs; i += gridDim.x) {
        const uint32_t o = static_cast<uint32_t>(i / runs), at = static_cast<uint32_t>(i % runs) * kNormThreads + threadIdx.x;
        if (at < inner) {
            const double v = to_f32(m[o * so + at * si]);
            sum += v * v;
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
    grid_launch_next();
}

// X = kScale M / (|M| + eps) as fp16 pairs, and its transpose, by tiles of 64 x 64 of X.  `planes` of a pair: high part,
// then low part, each rows x ld.
template <class T>
__global__ void __launch_bounds__(256) scale_kernel(const T* __restrict__ x, int64_t stride_b, int64_t stride_r, int64_t stride_c,
                                                    uint32_t m, uint32_t n, const double* __restrict__ partial, uint32_t partials,
                                                    double eps, __half* __restrict__ out, uint32_t ld, __half* __restrict__ out_t,
                                                    uint32_t ld_t) {
    __shared__ float tile[64][65];
    grid_wait();
    grid_launch_next();
    double sum = 0;
    for (uint32_t i = 0; i < partials; ++i) sum += partial[blockIdx.z * partials + i];
    const double factor = static_cast<double>(kScale) / (sqrt(sum) + eps);
    const T* mat = x + blockIdx.z * stride_b;
    const uint32_t r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
    const bool by_row = stride_c <= stride_r;
    for (int i = threadIdx.x; i < 64 * 64; i += 256) {
        const int r = by_row ? i / 64 : i % 64, c = by_row ? i % 64 : i / 64;
        tile[r][c] = r0 + r < m && c0 + c < n
                         ? static_cast<float>(to_f32(mat[(r0 + r) * stride_r + (c0 + c) * stride_c]) * factor)
                         : 0.f;
    }
    __syncthreads();
    __half* hi = out + static_cast<uint64_t>(blockIdx.z) * 2 * m * ld;
    __half* hi_t = out_t + static_cast<uint64_t>(blockIdx.z) * 2 * n * ld_t;
    for (int i = threadIdx.x; i < 64 * 64; i += 256) {
        const uint32_t a = i / 64, b = i % 64;
        __half h, l;
        if (r0 + a < m && c0 + b < ld) {
            split(tile[a][b], h, l);
            const uint64_t at = static_cast<uint64_t>(r0 + a) * ld + c0 + b;
            hi[at] = h;
            hi[static_cast<uint64_t>(m) * ld + at] = l;
        }
        if (c0 + a < n && r0 + b < ld_t) {
            split(tile[b][a], h, l);
            const uint64_t at = static_cast<uint64_t>(c0 + a) * ld_t + r0 + b;
            hi_t[at] = h;
            hi_t[static_cast<uint64_t>(n) * ld_t + at] = l;
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

constexpr int kTile = 128, kSlice = 64, kStages = 3;
constexpr int kOperand = kTile * kSlice * 2;   // one fp16 part of one operand: 16 KB
constexpr int kStageBytes = 4 * kOperand;      // A high, A low, B high, B low
constexpr int kRow = kTile + 4;                // floats of a row of partial sums in shared memory
constexpr int kThreads = 256;
constexpr int kSmem = 1024 + kStages * kStageBytes + 256;
static_assert(kTile * kRow * 4 <= kStages * kStageBytes, "partial sums take the place of the operands");

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 peer_load(const float* p, uint32_t rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(tc::smem_u32(p)), "r"(rank));
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}

union Half4 {
    __half h[4];
    uint2 u;
};
union Half8 {
    __half h[8];
    uint4 u;
};

// One 128 x 128 tile by a cluster of kSplit blocks, each over its share of k; their fp32 partial sums meet in shared
// memory, block r adding rows r * 128 / kSplit and on, over the ranks in order.
template <int kProduct, int kSplit>
__global__ void __launch_bounds__(kThreads, 1)
    product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, Job job, unsigned int* stalls) {
    extern __shared__ uint8_t raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(base + kStages * kStageBytes);
    uint64_t* empty = full + kStages;
    uint64_t* done = empty + kStages;
    uint32_t* slot = reinterpret_cast<uint32_t*>(done + 1);
    float* sums = reinterpret_cast<float*>(base);

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t rank = kSplit > 1 ? cluster_rank() : 0, batch = blockIdx.y;
    uint32_t ti, tj;
    {
        uint32_t t = blockIdx.x / kSplit;
        if constexpr (kProduct == kGram || kProduct == kPoly) {  // row ti holds the tiles ti..tiles_n-1
            ti = 0;
            for (uint32_t row = job.tiles_n; t >= row; --row, ++ti) t -= row;
            tj = ti + t;
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
    if (warp == 1) tc::tmem_alloc(slot, kTile);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = *slot;
    grid_wait();  // what the launches before this one wrote
    grid_launch_next();
    bool ok = true;

    if (warp == 0 && tc::elect_one()) {
        uint32_t it = 0;
        for (uint32_t s = first; s < last; ++s, ++it) {
            const uint32_t i = it % kStages;
            if (!(ok = tc::mbar_wait(&empty[i], (it / kStages & 1) ^ 1))) break;
            uint8_t* st = base + i * kStageBytes;
            tc::mbar_expect_tx(&full[i], kStageBytes);
            tc::tma_load_3d(st, &map_a, &full[i], s * kSlice, ti * kTile, batch * 2);
            tc::tma_load_3d(st + kOperand, &map_a, &full[i], s * kSlice, ti * kTile, batch * 2 + 1);
            tc::tma_load_3d(st + 2 * kOperand, &map_b, &full[i], s * kSlice, tj * kTile, batch * 2);
            tc::tma_load_3d(st + 3 * kOperand, &map_b, &full[i], s * kSlice, tj * kTile, batch * 2 + 1);
        }
        for (uint32_t s = it < kStages ? 0 : it - kStages; s < it; ++s)  // a load in flight lands before the block goes on
            ok = tc::mbar_wait(&full[s % kStages], s / kStages & 1) && ok;
    } else if (warp == 1 && tc::elect_one()) {
        constexpr uint32_t idesc = tc::idesc_f16(kTile);
        uint32_t it = 0;
        for (uint32_t s = first; s < last; ++s, ++it) {
            const uint32_t i = it % kStages;
            if (!(ok = tc::mbar_wait(&full[i], it / kStages & 1))) break;
            tc::fence_after();
            const uint8_t* st = base + i * kStageBytes;
            const uint64_t ah = tc::tile_desc(st), al = tc::tile_desc(st + kOperand), bh = tc::tile_desc(st + 2 * kOperand),
                           bl = tc::tile_desc(st + 3 * kOperand);
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
    __syncthreads();  // nobody reads the operands any more
    {
        // warp w reads lanes (w % 4) * 32 and on, columns (w / 4) * 64 and on
        const int r = (warp % 4) * 32 + lane;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int c = (warp / 4) * 64 + h * 32;
            uint32_t v[32];
            tc::tmem_ld32(tmem + (static_cast<uint32_t>((warp % 4) * 32) << 16) + c, v);
            tc::tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 8; ++j)
                *reinterpret_cast<uint4*>(sums + r * kRow + c + 4 * j) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        }
    }
    tc::fence_before();
    if constexpr (kSplit > 1)
        cluster_sync();
    else
        __syncthreads();
    tc::fence_after();
    if (warp == 1) tc::tmem_free(tmem, kTile);

    constexpr int kRows = kTile / kSplit;
    const int row0 = rank * kRows;
    const uint64_t plane = static_cast<uint64_t>(job.m) * job.ld;
    __half* out = job.out + batch * 2 * plane;
#pragma unroll 4
    for (int e = threadIdx.x; e < kRows * (kTile / 4); e += kThreads) {
        const int r = row0 + e / (kTile / 4), c = e % (kTile / 4) * 4;
        float* mine = sums + r * kRow + c;
        float4 v;
        if constexpr (kSplit > 1) {
            v = peer_load(mine, 0);
#pragma unroll
            for (int p = 1; p < kSplit; ++p) {
                const float4 w = peer_load(mine, p);
                v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
            }
        } else {
            v = *reinterpret_cast<const float4*>(mine);
        }
        const uint32_t i = ti * kTile + r, j = tj * kTile + c;
        float f[4] = {v.x, v.y, v.z, v.w};
        const bool inside = i < job.m && j < job.n;
        const uint64_t at = static_cast<uint64_t>(i) * job.ld + j;
        if constexpr (kProduct == kPoly) {
            Half4 gh, gl;
            gh.u = gl.u = make_uint2(0, 0);
            if (inside) {
                const __half* g = job.gram + batch * 2 * plane;
                gh.u = *reinterpret_cast<const uint2*>(g + at);
                gl.u = *reinterpret_cast<const uint2*>(g + plane + at);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q)
                f[q] = fmaf(kB, __half2float(gh.h[q]) + __half2float(gl.h[q]),
                            fmaf(kC / kScale, f[q], i == j + q ? kA * kScale : 0.f));
        } else if constexpr (kProduct == kLast) {
#pragma unroll
            for (int q = 0; q < 4; ++q) f[q] *= 1.f / (kScale * kScale);
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) f[q] *= 1.f / kScale;
        }
        if constexpr (kProduct == kLast) {
            if (!job.last_t && inside) {
                __nv_bfloat16* o = job.last + (static_cast<uint64_t>(batch) * job.m + i) * job.n + j;
                if (job.n % 4 == 0) {
                    union { __nv_bfloat16 h[4]; uint2 u; } b;
#pragma unroll
                    for (int q = 0; q < 4; ++q) b.h[q] = __float2bfloat16_rn(f[q]);
                    *reinterpret_cast<uint2*>(o) = b.u;
                } else {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (j + q < job.n) o[q] = __float2bfloat16_rn(f[q]);
                }
            }
        } else if (inside) {
            Half4 h, l;
#pragma unroll
            for (int q = 0; q < 4; ++q) split(f[q], h.h[q], l.h[q]);
            *reinterpret_cast<uint2*>(out + at) = h.u;
            *reinterpret_cast<uint2*>(out + plane + at) = l.u;
        }
        *reinterpret_cast<float4*>(mine) = make_float4(f[0], f[1], f[2], f[3]);  // only this block reads its rows
    }
    __syncthreads();
    // The transpose: a thread takes one column's run of 8 rows, neighbours take neighbouring columns.
    if (kProduct == kLast ? job.last_t : (kProduct == kApply || ti != tj)) {
        for (int e = threadIdx.x; e < kTile * (kRows / 8); e += kThreads) {
            const int c = e % kTile, r = row0 + e / kTile * 8;
            const uint32_t j = tj * kTile + c, i = ti * kTile + r;
            if (j >= job.n || i >= job.m) continue;
            if constexpr (kProduct == kLast) {
                __nv_bfloat16* o = job.last + (static_cast<uint64_t>(batch) * job.n + j) * job.m + i;
                union { __nv_bfloat16 h[8]; uint4 u; } b;
#pragma unroll
                for (int q = 0; q < 8; ++q) b.h[q] = __float2bfloat16_rn(sums[(r + q) * kRow + c]);
                if (job.m % 8 == 0) {
                    *reinterpret_cast<uint4*>(o) = b.u;
                } else {
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        if (i + q < job.m) o[q] = b.h[q];
                }
            } else {
                const uint64_t plane_t = static_cast<uint64_t>(job.n) * job.ld_t, at = static_cast<uint64_t>(j) * job.ld_t + i;
                __half* o = job.out_t + batch * 2 * plane_t;
                Half8 h, l;
#pragma unroll
                for (int q = 0; q < 8; ++q) split(sums[(r + q) * kRow + c], h.h[q], l.h[q]);
                *reinterpret_cast<uint4*>(o + at) = h.u;
                *reinterpret_cast<uint4*>(o + plane_t + at) = l.u;
            }
        }
    }
    if (!ok) atomicAdd(stalls, 1u);
    if constexpr (kSplit > 1) cluster_sync();  // a peer may still read this block's sums
}

// ----------------------------------------------------------------------- host

uint32_t up8(uint32_t v) { return (v + 7) / 8 * 8; }
uint64_t up256(uint64_t v) { return (v + 255) / 256 * 256; }
constexpr uint32_t kNormBlocks = 64;

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

int map_pair(CUtensorMap* map, const void* p, uint32_t rows, uint32_t cols, uint32_t ld, uint64_t batch) {
    const uint64_t dims[3] = {cols, rows, batch * 2}, strides[2] = {ld * 2ull, static_cast<uint64_t>(rows) * ld * 2};
    const uint32_t box[3] = {kSlice, kTile, 1};
    return encode_map(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, p, dims, strides, box);
}

template <int kProduct, int kSplit>
int launch_product(const CUtensorMap& ma, const CUtensorMap& mb, const Job& job, uint32_t tiles, uint32_t batch, unsigned int* stalls,
                   cudaStream_t st) {
    auto* kernel = product_kernel<kProduct, kSplit>;
    if (int rc = cuda_status(allow_smem(kernel, kSmem), "orthogonalize")) return rc;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(tiles * kSplit, batch);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmem;
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

// k is split over a cluster while that leaves every block two slices and all blocks run at once.
template <int kProduct>
int launch_split(const CUtensorMap& ma, const CUtensorMap& mb, Job job, uint32_t batch, int sms, unsigned int* stalls, cudaStream_t st) {
    job.tiles_m = (job.m + kTile - 1) / kTile;
    job.tiles_n = (job.n + kTile - 1) / kTile;
    const bool symmetric = kProduct == kGram || kProduct == kPoly;
    const uint32_t tiles = symmetric ? job.tiles_n * (job.tiles_n + 1) / 2 : job.tiles_m * job.tiles_n;
    const uint32_t slices = (job.k + kSlice - 1) / kSlice;
    uint32_t s = 8;
    while (s > 1 && (static_cast<uint64_t>(tiles) * batch * s > static_cast<uint32_t>(sms) || slices < 2 * s)) s /= 2;
    switch (s) {
        case 8: return launch_product<kProduct, 8>(ma, mb, job, tiles, batch, stalls, st);
        case 4: return launch_product<kProduct, 4>(ma, mb, job, tiles, batch, stalls, st);
        case 2: return launch_product<kProduct, 2>(ma, mb, job, tiles, batch, stalls, st);
        default: return launch_product<kProduct, 1>(ma, mb, job, tiles, batch, stalls, st);
    }
}

template <class T>
int launch_scaling(const nesle_orth_args& a, const Layout& lay, uint8_t* ws, int64_t sr, int64_t sc, cudaStream_t st) {
    const T* x = static_cast<const T*>(a.x);
    double* partial = reinterpret_cast<double*>(ws + lay.partial);
    square_sums_kernel<T><<<dim3(kNormBlocks, static_cast<unsigned>(a.batch)), kNormThreads, 0, st>>>(x, a.stride_b, sr, sc, lay.m, lay.n, partial);
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
                                          kNormBlocks, a.eps, reinterpret_cast<__half*>(ws + lay.x[0]), lay.ld_n,
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
    switch (a.dtype) {
        case NESLE_F32: rc = launch_scaling<float>(a, lay, ws, sr, sc, st); break;
        case NESLE_BF16: rc = launch_scaling<__nv_bfloat16>(a, lay, ws, sr, sc, st); break;
        default: rc = launch_scaling<__half>(a, lay, ws, sr, sc, st); break;
    }
    if (rc) return rc;
    unsigned int* stalls = nullptr;
    if ((rc = stall_counter(a.device, &stalls))) return rc;
    const int sms = sm_count(a.device);
    __half *gram = reinterpret_cast<__half*>(ws + lay.gram), *poly = reinterpret_cast<__half*>(ws + lay.poly);
    CUtensorMap map_x[2], map_xt[2], map_g, map_p;
    for (int i = 0; i < 2; ++i) {
        if ((rc = map_pair(&map_x[i], ws + lay.x[i], m, n, lay.ld_n, batch))) return rc;
        if ((rc = map_pair(&map_xt[i], ws + lay.xt[i], n, m, lay.ld_m, batch))) return rc;
    }
    if ((rc = map_pair(&map_g, gram, m, m, lay.ld_m, batch))) return rc;
    if ((rc = map_pair(&map_p, poly, m, m, lay.ld_m, batch))) return rc;
    for (int step = 0; step < a.steps; ++step) {
        const int from = step & 1, to = from ^ 1;
        Job g{};
        g.m = g.n = m, g.k = n;
        g.out = g.out_t = gram;
        g.ld = g.ld_t = lay.ld_m;
        if ((rc = launch_split<kGram>(map_x[from], map_x[from], g, batch, sms, stalls, st))) return rc;
        Job p = g;
        p.k = m;
        p.gram = gram;
        p.out = p.out_t = poly;
        if ((rc = launch_split<kPoly>(map_g, map_g, p, batch, sms, stalls, st))) return rc;
        Job x{};
        x.m = m, x.n = n, x.k = m;
        x.out = reinterpret_cast<__half*>(ws + lay.x[to]);
        x.ld = lay.ld_n;
        x.out_t = reinterpret_cast<__half*>(ws + lay.xt[to]);
        x.ld_t = lay.ld_m;
        x.last = static_cast<__nv_bfloat16*>(a.out);
        x.last_t = tall;
        rc = step + 1 < a.steps ? launch_split<kApply>(map_p, map_xt[from], x, batch, sms, stalls, st)
                                : launch_split<kLast>(map_p, map_xt[from], x, batch, sms, stalls, st);
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
        if (!a.workspace || a.workspace_bytes < nesle_orth_workspace(args) || reinterpret_cast<uintptr_t>(a.workspace) % 256)
            return ops::invalid("orthogonalize: the workspace is missing, too small or not 256-byte aligned");
        ops::OnDevice on(a.device);
        if (!on.ok) return ops::invalid("orthogonalize: device ordinal out of range");
        return ops::run(a, static_cast<cudaStream_t>(stream));
    });
}

}  // extern "C"
