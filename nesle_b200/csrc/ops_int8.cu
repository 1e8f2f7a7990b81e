// ops_int8.cu -- quantisation of rows to 8 bits, and the product of 8-bit
// integers with a scale for each token and each channel.
#include <type_traits>

#include "ops_common.h"
#include "tc05.cuh"

namespace nesle {
namespace ops {
namespace {

// ------------------------------------------------------------- quantize_rows
//
// One pass: a row's 16-byte chunks stay in registers between the maximum and
// the rounding (4 chunks a thread; longer rows are read again, from L2).
// 65,536 x 1,024 bf16: 62 us, 3.2 TB/s, half of what a copy reaches: the
// conversions, products, roundings and tests of an element take 65% of the issue
// slots.  Small calls are a launch (2,048 x 512 bf16: 6.4 us).  Rows that are not
// aligned come element by element (65,536 x 1,021: 109 us; 32 elements a thread
// and a warp a row, to do without the block's barrier, was a tenth slower).  The maximum is taken on the bit
// patterns of |x|, where a NaN is above infinity and infinity above every
// number, so that a row with either says so in its scale.

constexpr int kQuantThreads = 256;
constexpr int kHeld = 4;

template <class T, bool kVec>
struct Chunk {
    static constexpr int kN = kVec ? 16 / sizeof(T) : 1;
    alignas(kVec ? 16 : sizeof(T)) T v[kN];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (kVec)
            *reinterpret_cast<uint4*>(v) = __ldg(reinterpret_cast<const uint4*>(p));
        else
            v[0] = *p;
    }
};

// rint(x / s), the quotient rounded to fp32 first, of a row whose largest magnitude is 127 s.  x times the reciprocal of s is
// within 3 roundings of the quotient, 127 * 3 * 2^-24 < 2^-14, so that only a chunk with a product this near to half an integer
// is divided (and all where s is below the normal numbers, whose reciprocal may be infinite); and a sum with 1.5 * 2^23
// has the nearest integer in its low bits.  65,536 x 1,024 bf16: 76 us by divisions and conversions, 62 so.  Only a scale
// below the normal numbers is rounded so coarsely that a quotient passes 127 (190 units over 127 round to one unit); such
// rows are divided, and clamped there.
struct Divisor {
    float value, reciprocal;
    __device__ __forceinline__ explicit Divisor(float s) : value(s), reciprocal(s >= 0x1p-120f ? 1.f / s : __builtin_nanf("")) {}
};

template <int N>
__device__ __forceinline__ void quantize(const float (&x)[N], const Divisor& d, int8_t (&out)[N]) {
    constexpr float kRound = 12582912.f;
    uint32_t bits[N];
    bool sure = true;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float q = x[i] * d.reciprocal, r = q + kRound;
        bits[i] = __float_as_uint(r);
        sure = sure && fabsf(q - (r - kRound)) < 0.5f - 0x1p-14f;  // not with a NaN
    }
    if (!sure) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float q = __fdiv_rn(x[i], d.value);
            bits[i] = __float_as_uint((q == q ? fminf(fmaxf(q, -127.f), 127.f) : 0.f) + kRound);
        }
    }
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4)
            reinterpret_cast<uint32_t*>(out)[i / 4] = __byte_perm(__byte_perm(bits[i], bits[i + 1], 0x0040), __byte_perm(bits[i + 2], bits[i + 3], 0x0040), 0x5410);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = static_cast<int8_t>(bits[i]);
    }
}

template <class T, bool kVec, int kPerRow>
__global__ void __launch_bounds__(kQuantThreads) quantize_rows_kernel(const T* __restrict__ x, uint64_t rows, uint64_t cols,
                                                                     int64_t ld_x, int8_t* __restrict__ q, int64_t ld_q,
                                                                     float* __restrict__ scale) {
    using C = Chunk<T, kVec>;
    constexpr int kN = C::kN, kRows = kQuantThreads / kPerRow;
    const int lane = threadIdx.x % kPerRow;
    const uint64_t row = static_cast<uint64_t>(blockIdx.x) * kRows + threadIdx.x / kPerRow;
    if (kPerRow == 32 && row >= rows) return;  // whole warps; a larger group is the block and has its row
    const T* xr = x + static_cast<int64_t>(row) * ld_x;
    const uint64_t chunks = cols / kN;  // kVec only where this is exact
    C held[kHeld];
    uint32_t most = 0;
    auto take = [&](const C& c) {
#pragma unroll
        for (int i = 0; i < kN; ++i) most = max(most, __float_as_uint(to_f32(c.v[i])) & 0x7FFFFFFFu);
    };
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
        const uint64_t c = lane + static_cast<uint64_t>(h) * kPerRow;
        if (c < chunks) {
            held[h].load(xr + c * kN);
            take(held[h]);
        }
    }
    for (uint64_t c = lane + static_cast<uint64_t>(kHeld) * kPerRow; c < chunks; c += kPerRow) {
        C t;
        t.load(xr + c * kN);
        take(t);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if constexpr (kPerRow > 32) {
        __shared__ uint32_t part[kQuantThreads / 32];
        if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = most;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kQuantThreads / 32; ++i) most = max(most, part[i]);
    }
    const float s = __fdiv_rn(__uint_as_float(most), 127.f);
    if (lane == 0) scale[row] = s;
    const Divisor divisor(s > 0.f || s != s ? s : 1.f);
    int8_t* qr = q + static_cast<int64_t>(row) * ld_q;
    auto put = [&](const C& c, uint64_t at) {
        float x[kN];
        alignas(8) int8_t b[kN];
#pragma unroll
        for (int i = 0; i < kN; ++i) x[i] = to_f32(c.v[i]);
        quantize(x, divisor, b);
        if constexpr (kN == 8)
            *reinterpret_cast<uint2*>(qr + at * kN) = *reinterpret_cast<const uint2*>(b);
        else if constexpr (kN == 4)
            *reinterpret_cast<uint32_t*>(qr + at * kN) = *reinterpret_cast<const uint32_t*>(b);
        else
            qr[at] = b[0];
    };
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
        const uint64_t c = lane + static_cast<uint64_t>(h) * kPerRow;
        if (c < chunks) put(held[h], c);
    }
    for (uint64_t c = lane + static_cast<uint64_t>(kHeld) * kPerRow; c < chunks; c += kPerRow) {
        C t;
        t.load(xr + c * kN);
        put(t, c);
    }
    if (cols + lane < static_cast<uint64_t>(ld_q) && lane < 16) qr[cols + lane] = 0;
}

template <class T>
cudaError_t launch_quantize(const void* x, uint64_t rows, uint64_t cols, int64_t ld_x, int8_t* q, int64_t ld_q, float* scale,
                            cudaStream_t st) {
    constexpr uint64_t kN = 16 / sizeof(T);
    const T* p = static_cast<const T*>(x);
    // 16-byte loads where every row starts on 16 bytes and is whole chunks, and the stores of a chunk are aligned.
    const bool vec = cols % kN == 0 && ld_x % kN == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && ld_q % 8 == 0 &&
                     reinterpret_cast<uintptr_t>(q) % 8 == 0;
    // A warp a row while its registers hold the row, else a block.
    const bool warp = cols <= 32 * kHeld * (vec ? kN : 1);
    const uint64_t blocks = warp ? (rows + kQuantThreads / 32 - 1) / (kQuantThreads / 32) : rows;
    const dim3 grid(static_cast<unsigned>(blocks));
    if (vec && warp)
        quantize_rows_kernel<T, true, 32><<<grid, kQuantThreads, 0, st>>>(p, rows, cols, ld_x, q, ld_q, scale);
    else if (vec)
        quantize_rows_kernel<T, true, kQuantThreads><<<grid, kQuantThreads, 0, st>>>(p, rows, cols, ld_x, q, ld_q, scale);
    else if (warp)
        quantize_rows_kernel<T, false, 32><<<grid, kQuantThreads, 0, st>>>(p, rows, cols, ld_x, q, ld_q, scale);
    else
        quantize_rows_kernel<T, false, kQuantThreads><<<grid, kQuantThreads, 0, st>>>(p, rows, cols, ld_x, q, ld_q, scale);
    return cudaGetLastError();
}

// ----------------------------------------------------------------- the product

struct Epilogue {
    const float* x_scale;
    float x_scale_value;
    const float* w_scale;
    const float* bias;
    void* y;
    int64_t ld_y;
    uint32_t m, k, n;
    int relu;
};

__device__ __forceinline__ float finish(int acc, float xs, float ws, float bias, int relu) {
    const float y = fmaf(static_cast<float>(acc) * xs, ws, bias);
    return relu && y < 0.f ? 0.f : y;  // a NaN passes
}

// Up to 16 bytes from anywhere, zeros after them.  They come as aligned words, each of which lies in one page with the byte
// of its that is asked for (rows of 65,536 x 2,047 laid out again: 46 us, byte by byte 82).
__device__ __forceinline__ uint4 load_any(const uint8_t* p, uint32_t bytes) {
    const uint32_t shift = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) & 3);
    const uint32_t* words = reinterpret_cast<const uint32_t*>(p - shift);
    uint32_t w[5], b[4];
#pragma unroll
    for (uint32_t j = 0; j < 5; ++j) w[j] = j * 4 < shift + bytes ? __ldg(words + j) : 0u;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
        const uint32_t left = bytes > j * 4 ? bytes - j * 4 : 0;  // of this word
        b[j] = __funnelshift_r(w[j], w[j + 1], shift * 8) & (left >= 4 ? ~0u : (1u << left * 8) - 1);
    }
    return make_uint4(b[0], b[1], b[2], b[3]);
}

// Rows of x copied to 16-byte aligned rows (many tokens of unaligned x only): zeros from k to ld.
__global__ void pad_rows_kernel(const uint8_t* __restrict__ x, int64_t ld_x, uint64_t rows, uint32_t k, uint8_t* __restrict__ out,
                                uint32_t ld) {
    const uint32_t per = ld / 16;
    const uint64_t total = rows * per;
    for (uint64_t i = blockIdx.x * static_cast<uint64_t>(blockDim.x) + threadIdx.x; i < total;
         i += static_cast<uint64_t>(gridDim.x) * blockDim.x) {
        const uint64_t r = i / per;
        const uint32_t c = static_cast<uint32_t>(i % per) * 16;
        *reinterpret_cast<uint4*>(out + r * ld + c) = load_any(x + static_cast<int64_t>(r) * ld_x + c, min(k - c, 16u));
    }
}

// Few tokens (m <= kFewTokens): latency and the weights' bytes bound it.  A
// block takes 16 tokens and 8 channels, its 8 warps split k, and the warps'
// exact integer sums meet in shared memory.  A lane's 16-byte chunk feeds two
// m16n8k32 products: any order of k is right as long as both operands have
// it, so a chunk's words 0, 1 and 2, 3 are the low and high halves of one
// product each.  The instruction takes uint8 by int8 as it is.  Tokens that are
// not aligned are read as they are.  16 x 2,048 to 512 channels: 6.0 us, most
// of it the launch and one trip to HBM.
constexpr uint32_t kFewTokens = 64;

__device__ __forceinline__ uint4 load16(const uint8_t* p, uint32_t at, uint32_t k) {
    if (at + 16 <= k) return __ldg(reinterpret_cast<const uint4*>(p + at));
    alignas(16) uint8_t b[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) b[j] = at + j < k ? p[at + j] : uint8_t(0);
    return *reinterpret_cast<const uint4*>(b);
}

template <bool kUnsigned>
__device__ __forceinline__ void mma_16832(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
    if constexpr (kUnsigned)
        asm volatile(
            "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <bool kUnsigned, class Out, bool kAligned>
__global__ void __launch_bounds__(256) int8_few_kernel(const uint8_t* __restrict__ x, int64_t ld_x, const uint8_t* __restrict__ w,
                                                      int64_t ld_w, Epilogue ep) {
    __shared__ int part[8][16][8];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, r = lane / 4, quad = lane % 4;
    const uint32_t m0 = blockIdx.y * 16, n0 = blockIdx.x * 8;
    const bool has0 = m0 + r < ep.m, has1 = m0 + r + 8 < ep.m, hasn = n0 + r < ep.n;
    const uint8_t* x0 = x + static_cast<int64_t>(has0 ? m0 + r : 0) * ld_x;
    const uint8_t* x1 = x + static_cast<int64_t>(has1 ? m0 + r + 8 : 0) * ld_x;
    const uint8_t* wn = w + static_cast<int64_t>(hasn ? n0 + r : 0) * ld_w;
    int c[4] = {};
    const uint4 zero = make_uint4(0, 0, 0, 0);
    auto token = [&](const uint8_t* row, uint32_t at) {
        if constexpr (kAligned)
            return load16(row, at, ep.k);
        else
            return load_any(row + at, min(ep.k - at, 16u));
    };
#pragma unroll 4
    for (uint32_t k0 = warp * 64; k0 < ep.k; k0 += 8 * 64) {
        const uint32_t at = k0 + quad * 16;
        const uint4 a = has0 && at < ep.k ? token(x0, at) : zero;
        const uint4 b = has1 && at < ep.k ? token(x1, at) : zero;
        const uint4 v = hasn && at < ep.k ? load16(wn, at, ep.k) : zero;
        mma_16832<kUnsigned>(c, a.x, b.x, a.y, b.y, v.x, v.y);
        mma_16832<kUnsigned>(c, a.z, b.z, a.w, b.w, v.z, v.w);
    }
    part[warp][r][quad * 2] = c[0];
    part[warp][r][quad * 2 + 1] = c[1];
    part[warp][r + 8][quad * 2] = c[2];
    part[warp][r + 8][quad * 2 + 1] = c[3];
    __syncthreads();
    if (threadIdx.x >= 128) return;
    const uint32_t i = threadIdx.x / 8, j = threadIdx.x % 8;
    if (m0 + i >= ep.m || n0 + j >= ep.n) return;
    int sum = 0;
#pragma unroll
    for (int s = 0; s < 8; ++s) sum += part[s][i][j];
    const float xs = ep.x_scale ? ep.x_scale[m0 + i] : ep.x_scale_value;
    static_cast<Out*>(ep.y)[static_cast<int64_t>(m0 + i) * ep.ld_y + n0 + j] =
        from_f32<Out>(finish(sum, xs, ep.w_scale[n0 + j], ep.bias ? ep.bias[n0 + j] : 0.f, ep.relu));
}

// Many tokens: persistent blocks, one an SM, over tiles of 128 tokens by kBN
// channels; TMA brings 128-byte slices of k of both operands, one thread issues
// tcgen05.mma (kind::i8), accumulators alternate between two halves of tensor
// memory so that a tile's epilogue runs under the next tile's products.
// 65,536 x 2,048 to 512: 62 us, 2.2 PFLOP/s, 3.2 TB/s of what HBM has to give
// and take.  The operands' way from L2 bounds it: 48 KB a slice at 48 bytes a
// clock and SM, 1,000 clocks for 512 clocks of products.
//
// Results leave by TMA where their rows start and end on 16 bytes, else from
// the same tile in shared memory a row at a time, neighbouring lanes at
// neighbouring columns, two a store where rows start on 4 bytes and are even
// (65,536 x 2,047 to 500: 79 us, one a store 92; a thread storing its own row
// 385).
//
// Unsigned tokens multiply the weights + 128, which are unsigned too, and
// sum_k x w = sum_k x (w + 128) - 128 sum_k x: four warps take the row sums of
// x from the tiles in shared memory as they pass (a dot product with ones,
// four bytes at a time).
constexpr int kBM = 128, kBK = 128;

template <int kBN>
struct Tile {
    static constexpr int kStages = kBN == 256 ? 4 : 6;
    static constexpr int kA = kBM * kBK, kB = kBN * kBK;
    static constexpr int kStage = kA + kB;
    static constexpr int kStaging = 4 * 32 * 128;  // 4 warps x 32 rows x 128 bytes on their way out
    static constexpr int kBars = 2 * kStages + 4;
    static constexpr int kChannels = 4 * 2 * 64 * 4;  // 4 warps' scales and biases of the columns at hand
    static constexpr int kSmem = 1024 + kStages * kStage + kStaging + kBars * 8 + 16 + 2 * kBM * 4 + kChannels;
    static constexpr uint32_t kCols = 2 * kBN < 32 ? 32 : 2 * kBN;
};

template <bool kUnsigned, class Out, int kBN, bool kTmaOut>
__global__ void __launch_bounds__(kUnsigned ? 320 : 192, 1)
    int8_tile_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                     const __grid_constant__ CUtensorMap map_y, Epilogue ep, unsigned int* stalls) {
    using T = Tile<kBN>;
    constexpr int S = T::kStages;
    extern __shared__ uint8_t raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    uint8_t* stage = base;
    uint8_t* staging = base + S * T::kStage;
    uint64_t* full = reinterpret_cast<uint64_t*>(staging + T::kStaging);
    uint64_t* empty = full + S;
    uint64_t* done = empty + S;  // a tile's accumulators (and row sums) are complete
    uint64_t* idle = done + 2;   // they have been read
    uint32_t* slot = reinterpret_cast<uint32_t*>(idle + 2);
    int* sums = reinterpret_cast<int*>(slot + 4);

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t tiles_n = (ep.n + kBN - 1) / kBN, tiles = tiles_n * ((ep.m + kBM - 1) / kBM);
    const uint32_t slices = (ep.k + kBK - 1) / kBK;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) {
            tc::mbar_init(&full[i], 1);
            tc::mbar_init(&empty[i], kUnsigned ? 5 : 1);
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&done[i], kUnsigned ? 5 : 1);
            tc::mbar_init(&idle[i], 4);
        }
        tc::mbar_init_fence();
        tc::prefetch_map(&map_x);
        tc::prefetch_map(&map_w);
    }
    if (warp == 1) tc::tmem_alloc(slot, T::kCols);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = *slot;
    bool ok = true;

    if (warp == 0) {
        if (tc::elect_one()) {
            uint32_t it = 0;
            for (uint32_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
                const int row = (tile / tiles_n) * kBM, col = (tile % tiles_n) * kBN;
                for (uint32_t s = 0; s < slices; ++s, ++it) {
                    const uint32_t i = it % S;
                    if (!(ok = tc::mbar_wait(&empty[i], (it / S & 1) ^ 1))) break;
                    tc::mbar_expect_tx(&full[i], T::kStage);
                    tc::tma_load_2d(stage + i * T::kStage, &map_x, &full[i], s * kBK, row);
                    tc::tma_load_2d(stage + i * T::kStage + T::kA, &map_w, &full[i], s * kBK, col);
                }
            }
            // a load in flight lands before the block leaves
            for (uint32_t s = it < S ? 0 : it - S; s < it; ++s) ok = tc::mbar_wait(&full[s % S], s / S & 1) && ok;
        }
    } else if (warp == 1) {
        if (tc::elect_one()) {
            constexpr uint32_t idesc = tc::idesc_i8(kBN, kUnsigned ? tc::kTypeU8 : tc::kTypeS8);
            uint32_t it = 0, n = 0;
            for (uint32_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x, ++n) {
                const uint32_t half = n & 1;
                if (!(ok = tc::mbar_wait(&idle[half], (n >> 1 & 1) ^ 1))) break;
                tc::fence_after();
                for (uint32_t s = 0; s < slices; ++s, ++it) {
                    const uint32_t i = it % S;
                    if (!(ok = tc::mbar_wait(&full[i], it / S & 1))) break;
                    tc::fence_after();
                    const uint64_t a = tc::tile_desc(stage + i * T::kStage), b = tc::tile_desc(stage + i * T::kStage + T::kA);
#pragma unroll
                    for (int kk = 0; kk < kBK / 32; ++kk)
                        tc::mma_i8(tmem + half * kBN, a + 2 * kk, b + 2 * kk, idesc, s > 0 || kk > 0);
                    tc::mma_commit(&empty[i]);
                }
                tc::mma_commit(&done[half]);
            }
        }
    } else if (warp < 6) {
        const int quarter = warp % 4;  // the lanes of tensor memory that this warp may read
        uint8_t* out = staging + (warp - 2) * 32 * 128;
        constexpr int kWide = 128 / sizeof(Out);  // columns of a 128-byte row on its way out
        float* scales = reinterpret_cast<float*>(sums + 2 * kBM) + (warp - 2) * 128;
        float* biases = scales + 64;
        uint32_t n = 0;
        for (uint32_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x, ++n) {
            const uint32_t half = n & 1;
            if (!(ok = tc::mbar_wait_warp(&done[half], n >> 1 & 1))) break;
            tc::fence_after();
            const uint32_t row = (tile / tiles_n) * kBM + quarter * 32 + lane, col = (tile % tiles_n) * kBN;
            const float xs = ep.x_scale ? (row < ep.m ? ep.x_scale[row] : 0.f) : ep.x_scale_value;
            const int less = kUnsigned ? sums[half * kBM + quarter * 32 + lane] * 128 : 0;
            const uint32_t at = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + half * kBN;
#pragma unroll 1
            for (int c = 0; c < kBN; c += kWide) {
                if (col + c >= ep.n) break;  // the same for the whole warp
                if constexpr (kTmaOut)
                    if (lane == 0) tc::bulk_wait_read();
#pragma unroll
                for (int j = lane; j < kWide; j += 32) {
                    const uint32_t cn = col + c + j;
                    scales[j] = cn < ep.n ? __ldg(ep.w_scale + cn) : 0.f;
                    biases[j] = ep.bias && cn < ep.n ? __ldg(ep.bias + cn) : 0.f;
                }
                __syncwarp();
#pragma unroll
                for (int p = 0; p < kWide; p += 32) {
                    uint32_t acc[32];
                    tc::tmem_ld32(at + c + p, acc);
                    tc::tmem_wait_ld();
                    alignas(16) Out v[32];
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const float4 ws = *reinterpret_cast<const float4*>(scales + p + j), be = *reinterpret_cast<const float4*>(biases + p + j);
                        v[j] = from_f32<Out>(finish(static_cast<int>(acc[j]) - less, xs, ws.x, be.x, ep.relu));
                        v[j + 1] = from_f32<Out>(finish(static_cast<int>(acc[j + 1]) - less, xs, ws.y, be.y, ep.relu));
                        v[j + 2] = from_f32<Out>(finish(static_cast<int>(acc[j + 2]) - less, xs, ws.z, be.z, ep.relu));
                        v[j + 3] = from_f32<Out>(finish(static_cast<int>(acc[j + 3]) - less, xs, ws.w, be.w, ep.relu));
                    }
                    constexpr int kChunks = 32 * sizeof(Out) / 16;
#pragma unroll
                    for (int j = 0; j < kChunks; ++j) {
                        const int chunk = (p * (int)sizeof(Out) / 16 + j) ^ (lane & 7);
                        *reinterpret_cast<uint4*>(out + lane * 128 + chunk * 16) = reinterpret_cast<const uint4*>(v)[j];
                    }
                }
                if constexpr (!kTmaOut) {  // a row at a time, neighbouring lanes neighbouring columns
                    constexpr int kPer = 16 / sizeof(Out);
                    __syncwarp();
                    const uint32_t row0 = row - lane, rows = ep.m > row0 ? ep.m - row0 : 0;
                    Out* y = static_cast<Out*>(ep.y) + static_cast<int64_t>(row0) * ep.ld_y + col + c;
                    auto staged = [&](uint32_t r, int j) { return out + r * 128 + (j / kPer ^ (r & 7)) * 16 + j % kPer * sizeof(Out); };
                    if (sizeof(Out) == 2 && ep.ld_y % 2 == 0 && ep.n % 2 == 0 && reinterpret_cast<uintptr_t>(ep.y) % 4 == 0) {  // two columns a store
                        const int j = lane * 2;
                        if (col + c + j < ep.n) {
#pragma unroll 16
                            for (uint32_t r = 0; r < 32; ++r)
                                if (r < rows) *reinterpret_cast<uint32_t*>(y + r * ep.ld_y + j) = *reinterpret_cast<const uint32_t*>(staged(r, j));
                        }
                    } else {
#pragma unroll 8
                        for (uint32_t r = 0; r < 32; ++r)
#pragma unroll
                            for (int j = lane; j < kWide; j += 32)
                                if (r < rows && col + c + j < ep.n) y[r * ep.ld_y + j] = *reinterpret_cast<const Out*>(staged(r, j));
                    }
                    __syncwarp();
                }
                if constexpr (kTmaOut) {
                    tc::fence_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tc::tma_store_2d(&map_y, out, col + c, (tile / tiles_n) * kBM + quarter * 32);
                        tc::bulk_commit();
                    }
                }
            }
            tc::fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&idle[half]);
        }
        if (kTmaOut && lane == 0) tc::bulk_wait();
    } else if constexpr (kUnsigned) {
        // The row of this thread in each slice; chunks are taken in an order that differs from lane to lane, so that
        // eight lanes' 16-byte reads fall on different banks (the order within a row does not matter to a sum).
        const int r = (warp - 6) * 32 + lane;
        uint32_t it = 0, n = 0;
        for (uint32_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x, ++n) {
            uint32_t sum = 0;
            for (uint32_t s = 0; s < slices; ++s, ++it) {
                const uint32_t i = it % S;
                if (!(ok = tc::mbar_wait_warp(&full[i], it / S & 1))) break;
                const uint8_t* rows = stage + i * T::kStage + r * 128;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint4 v = *reinterpret_cast<const uint4*>(rows + ((j + lane) & 7) * 16);
                    sum = __dp4a(v.x, 0x01010101u, sum);
                    sum = __dp4a(v.y, 0x01010101u, sum);
                    sum = __dp4a(v.z, 0x01010101u, sum);
                    sum = __dp4a(v.w, 0x01010101u, sum);
                }
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&empty[i]);
            }
            const uint32_t half = n & 1;
            if (!ok || !(ok = tc::mbar_wait_warp(&idle[half], (n >> 1 & 1) ^ 1))) break;
            sums[half * kBM + r] = static_cast<int>(sum);
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&done[half]);
        }
    }
    if (!ok) atomicAdd(stalls, 1u);
    __syncwarp();
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    if (warp == 1) tc::tmem_free(tmem, T::kCols);
}

bool aligned_x(const nesle_int8_args& a) { return reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.ld_x % 16 == 0; }
uint64_t padded(uint64_t k) { return (k + 15) / 16 * 16; }

const char* check(const nesle_int8_args& a) {
    if (a.m > 0x7FFFFFFFull || a.n > 0x7FFFFFFFull) return "int8_linear: m and n must be below 2^31";
    if (a.m && a.n && (!a.y || !a.w_scale)) return "int8_linear: null argument";
    if (a.m && a.n && a.k && (!a.x || !a.w || (a.x_unsigned && !a.w_biased))) return "int8_linear: null argument";
    if (a.k > (a.x_unsigned ? 33025ull : 131071ull))  // 255 * 255 k and 128 * 128 k are below 2^31
        return "int8_linear: k is above what 32-bit sums hold (33025 for uint8 tokens, 131071 for int8)";
    if (a.ld_x < (int64_t)a.k || a.ld_w < (int64_t)a.k || a.ld_y < (int64_t)a.n) return "int8_linear: a leading dimension is shorter than its row";
    if (a.ld_w % 16 || reinterpret_cast<uintptr_t>(a.w) % 16 || reinterpret_cast<uintptr_t>(a.w_biased) % 16)
        return "int8_linear: weights must be 16-byte aligned with rows a multiple of 16 bytes apart";
    if (a.y_dtype != NESLE_F32 && a.y_dtype != NESLE_BF16 && a.y_dtype != NESLE_F16) return "int8_linear: unknown output type";
    if (!all_on(4, a.x_scale, a.w_scale, a.bias) || !all_on(element_size(a.y_dtype), a.y)) return "int8_linear: scales, bias and y must be aligned to their elements";
    return nullptr;
}

template <bool kUnsigned, class Out, int kBN>
int launch_tiles(const nesle_int8_args& a, const uint8_t* x, int64_t ld_x, const Epilogue& ep, cudaStream_t st) {
    using T = Tile<kBN>;
    CUtensorMap mx, mw, my;
    const uint64_t dx[2] = {a.k, a.m}, sx[1] = {(uint64_t)ld_x}, dw[2] = {a.k, a.n}, sw[1] = {(uint64_t)a.ld_w};
    const uint32_t bx[2] = {kBK, kBM}, bw[2] = {kBK, kBN};
    const void* w = kUnsigned ? static_cast<const void*>(a.w_biased) : static_cast<const void*>(a.w);
    if (int rc = encode_map(&mx, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, x, dx, sx, bx)) return rc;
    if (int rc = encode_map(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, w, dw, sw, bw)) return rc;
    // A tiled store ends on 16 bytes, past n where n does not: such rows may have neighbours.
    const bool tma_out = reinterpret_cast<uintptr_t>(a.y) % 16 == 0 && a.ld_y * sizeof(Out) % 16 == 0 && a.n * sizeof(Out) % 16 == 0;
    if (tma_out) {
        const uint64_t dy[2] = {a.n, a.m}, sy[1] = {a.ld_y * sizeof(Out)};
        const uint32_t by[2] = {128 / sizeof(Out), 32};
        const CUtensorMapDataType ty = sizeof(Out) == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
        if (int rc = encode_map(&my, ty, 2, a.y, dy, sy, by)) return rc;
    } else {
        my = mx;
    }
    unsigned int* stalls = nullptr;
    if (int rc = stall_counter(a.device, &stalls)) return rc;
    const uint64_t tiles = ((a.m + kBM - 1) / kBM) * ((a.n + kBN - 1) / kBN);
    if (tiles > 0x7FFFFFFFull) return invalid("int8_linear: too many tiles");
    const unsigned grid = static_cast<unsigned>(tiles < (uint64_t)sm_count(a.device) ? tiles : sm_count(a.device));
    const int threads = kUnsigned ? 320 : 192;
    auto go = [&](auto tma) -> int {
        constexpr auto* kernel = int8_tile_kernel<kUnsigned, Out, kBN, decltype(tma)::value>;
        if (int rc = allow_smem<kernel>(T::kSmem, a.device, "int8_linear")) return rc;
        kernel<<<grid, threads, T::kSmem, st>>>(mx, mw, my, ep, stalls);
        return cuda_status(cudaGetLastError(), "int8_linear");
    };
    return tma_out ? go(std::true_type{}) : go(std::false_type{});
}

template <bool kUnsigned, class Out>
int run(const nesle_int8_args& a, cudaStream_t st) {
    Epilogue ep{a.x_scale, a.x_scale_value, a.w_scale, a.bias, a.y, a.ld_y, (uint32_t)a.m, (uint32_t)a.k, (uint32_t)a.n, a.relu};
    const uint8_t* x = static_cast<const uint8_t*>(a.x);
    int64_t ld_x = a.ld_x;
    if (a.m <= kFewTokens || !a.k) {  // k = 0 is the bias alone, of any number of tokens
        const uint8_t* w = reinterpret_cast<const uint8_t*>(a.w);
        constexpr uint64_t kMost = 65535 * 16;  // tokens of a grid
        for (uint64_t first = 0; first < a.m; first += kMost) {
            Epilogue part = ep;
            part.m = static_cast<uint32_t>(a.m - first < kMost ? a.m - first : kMost);
            part.x_scale = ep.x_scale ? ep.x_scale + first : nullptr;
            part.y = static_cast<Out*>(ep.y) + static_cast<int64_t>(first) * ep.ld_y;
            const dim3 grid(static_cast<unsigned>((a.n + 7) / 8), (part.m + 15) / 16);
            if (aligned_x(a))
                int8_few_kernel<kUnsigned, Out, true><<<grid, 256, 0, st>>>(x, a.ld_x, w, a.ld_w, part);
            else
                int8_few_kernel<kUnsigned, Out, false><<<grid, 256, 0, st>>>(x, a.ld_x, w, a.ld_w, part);
            if (int rc = cuda_status(cudaGetLastError(), "int8_linear")) return rc;
        }
        return NESLE_OK;
    }
    if (!aligned_x(a)) {
        ld_x = static_cast<int64_t>(padded(a.k));
        const uint64_t chunks = a.m * (ld_x / 16);
        const uint64_t most = 16ull * sm_count(a.device), want = (chunks + 255) / 256;
        pad_rows_kernel<<<static_cast<unsigned>(want < most ? want : most), 256, 0, st>>>(
            x, a.ld_x, a.m, static_cast<uint32_t>(a.k), static_cast<uint8_t*>(a.workspace), static_cast<uint32_t>(ld_x));
        if (int rc = cuda_status(cudaGetLastError(), "int8_linear")) return rc;
        x = static_cast<const uint8_t*>(a.workspace);
    }
    // The widest tile that n fills, whose operands are read least often from L2, where its tiles occupy half of the SMs; else
    // narrower ones (2,048 tokens of 512 to 256 channels: 16 blocks of 256 channels 11.5 us, 64 of 64 6.4 us).
    auto busy = [&](uint64_t bn) {
        return ((a.m + kBM - 1) / kBM) * ((a.n + bn - 1) / bn) * 2 >= static_cast<uint64_t>(sm_count(a.device));
    };
    if (a.n > 128 && busy(256)) return launch_tiles<kUnsigned, Out, 256>(a, x, ld_x, ep, st);
    if (a.n > 64 && busy(128)) return launch_tiles<kUnsigned, Out, 128>(a, x, ld_x, ep, st);
    return launch_tiles<kUnsigned, Out, 64>(a, x, ld_x, ep, st);
}

}  // namespace
}  // namespace ops
}  // namespace nesle

using namespace nesle;

extern "C" {

int nesle_quantize_rows(const void* x, int dtype, uint64_t rows, uint64_t cols, int64_t ld_x, int8_t* q, int64_t ld_q,
                        float* scale, int device, void* stream) {
    return ops::guarded([&]() -> int {
        if (!rows) return NESLE_OK;
        if (!scale || (cols && (!x || !q))) return ops::invalid("quantize_rows: null argument");
        if (ld_x < (int64_t)cols || ld_q < (int64_t)cols || ld_q - (int64_t)cols >= 16)
            return ops::invalid("quantize_rows: a leading dimension is shorter than its row, or ld_q 16 or more longer");
        if (rows > 0x7FFFFFFFull) return ops::invalid("quantize_rows: too many rows");
        if (!ops::all_on(4, scale) || !ops::all_on(ops::element_size(dtype), x)) return ops::invalid("quantize_rows: x and scale must be aligned to their elements");
        ops::OnDevice on(device);
        if (!on.ok) return ops::invalid("quantize_rows: device ordinal out of range");
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        cudaError_t e;
        switch (dtype) {
            case NESLE_F32: e = ops::launch_quantize<float>(x, rows, cols, ld_x, q, ld_q, scale, st); break;
            case NESLE_BF16: e = ops::launch_quantize<__nv_bfloat16>(x, rows, cols, ld_x, q, ld_q, scale, st); break;
            case NESLE_F16: e = ops::launch_quantize<__half>(x, rows, cols, ld_x, q, ld_q, scale, st); break;
            default: return ops::invalid("quantize_rows: unknown element type");
        }
        return ops::cuda_status(e, "quantize_rows");
    });
}

uint64_t nesle_int8_workspace(const nesle_int8_args* a) {
    return a && a->k && a->m > ops::kFewTokens && !ops::aligned_x(*a) ? a->m * ops::padded(a->k) : 0;
}

int nesle_int8_linear(const nesle_int8_args* args, void* stream) {
    return ops::guarded([&]() -> int {
        if (!args) return ops::invalid("int8_linear: null argument");
        const nesle_int8_args& a = *args;
        if (const char* why = ops::check(a)) return ops::invalid(why);
        if (!a.m || !a.n) return NESLE_OK;
        const int64_t size = ops::element_size(a.y_dtype);
        const ops::Memory y(a.y, a.m, a.ld_y * size, a.n * size);
        for (const ops::Memory& x : {ops::Memory(a.x, a.m, a.ld_x, a.k), ops::Memory(a.x_scale, 1, 0, a.m * 4), ops::Memory(a.bias, 1, 0, a.n * 4),
                                     ops::Memory(a.w, a.n, a.ld_w, a.k), ops::Memory(a.w_biased, a.n, a.ld_w, a.k), ops::Memory(a.w_scale, 1, 0, a.n * 4)})
            if (ops::may_overlap(y, x)) return set_error(NESLE_ERR_OVERLAP, "int8_linear: y shares memory with another argument");
        const uint64_t need = nesle_int8_workspace(args);
        if (need && (!a.workspace || a.workspace_bytes < need || reinterpret_cast<uintptr_t>(a.workspace) % 16))
            return ops::invalid("int8_linear: the workspace is missing, too small or not 16-byte aligned");
        ops::OnDevice on(a.device);
        if (!on.ok) return ops::invalid("int8_linear: device ordinal out of range");
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (a.x_unsigned) {
            if (a.y_dtype == NESLE_F32) return ops::run<true, float>(a, st);
            if (a.y_dtype == NESLE_BF16) return ops::run<true, __nv_bfloat16>(a, st);
            return ops::run<true, __half>(a, st);
        }
        if (a.y_dtype == NESLE_F32) return ops::run<false, float>(a, st);
        if (a.y_dtype == NESLE_BF16) return ops::run<false, __nv_bfloat16>(a, st);
        return ops::run<false, __half>(a, st);
    });
}

}  // extern "C"
