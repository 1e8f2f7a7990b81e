// ops_delta.cuh -- the gated delta rule over a sequence, and its gradients.
//
// For every env n and head h a state S (dk x dv, fp32) is a memory that maps
// keys to values.  A token decays it, reads what it holds for its key, and
// writes the difference to its value:
//
//   e_t = v_t - a_t S_{t-1}^T k_t     a_t = exp(g_t); S_{t-1} = 0 where reset_t
//   u_t = beta_t e_t
//   S_t = a_t S_{t-1} + k_t u_t^T
//   o_t = scale S_t^T q_t
//
// Token by token that is three products of a vector with a 64 x 64 matrix for
// a few hundred bytes of input.  Taken 16 tokens at a time (a chunk, within one
// episode) it is products of matrices: with D_ij = a_{j+1} ... a_i,
// gamma_i = a_1 ... a_i, eta_j = D_Cj and Gamma = gamma_C over the chunk,
//
//   u_i = beta_i (v_i - gamma_i S^T k_i - sum_{j<i} D_ij (k_i.k_j) u_j)
//   O   = scale (gamma Q S + (D o Q K^T) U)
//   S'  = Gamma S + (eta K)^T U
//
// 16 is the M of mma.sync, the triangular system is small enough to be solved
// by substitution (which no choice of keys can make inaccurate), and D comes
// from running products, never from differences of logarithms.
//
// Precision: states, errors and all sums are fp32.  Products run on the tensor
// cores with every fp32 operand as a sum of up to three bf16 (8 bits each, 24
// together; bf16 has fp32's range, so nothing needs scaling); terms below 2^-24
// of the largest are left out.  A bf16 input is one term, an fp16 input two, an
// fp32 input three.
#pragma once
#include <stddef.h>

#include "ops_common.h"
#include "tc05.cuh"

namespace nesle {
namespace ops {
namespace delta {

constexpr int kC = 16;  // tokens of a chunk

struct Strides {
    int64_t t, n, h;
};

struct Scan {
    const void *q, *k, *v;
    Strides sq, sk, sv;
    const float *g, *beta;
    Strides sg, sb;
    const uint8_t* reset;
    int64_t reset_t, reset_n;
    const float* state;
    int64_t t, n, h;
    int dk, dv;
    float scale;
    bool aligned;  // every row of q, k, v (and d_o) is whole 16-byte chunks and starts on 16 bytes
    void* o;
    float* final_state;
    float* errors;       // [t][n][h][dv], NULL where no gradient is wanted
    float* checkpoints;  // [n][h][ceil(t / 16)][dk][dv], the state before each chunk
    const void* d_o;     // contiguous
    const float* d_final;
    void *dq, *dk_out, *dv_out;
    float *dg, *dbeta, *dstate;
    unsigned int* stalls;
};

template <class T>
struct Terms;  // bf16 terms that hold a T exactly
template <>
struct Terms<__nv_bfloat16> { static constexpr int n = 1; };
template <>
struct Terms<__half> { static constexpr int n = 2; };
template <>
struct Terms<float> { static constexpr int n = 3; };

__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// x, y as sums of N bf16 each, packed pairwise.
template <int N>
__device__ __forceinline__ void split(float x, float y, uint32_t (&out)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        out[i] = pack(x, y);
        if (i + 1 < N) {
            x -= __uint_as_float(out[i] << 16);
            y -= __uint_as_float(out[i] & 0xFFFF0000u);
        }
    }
}

struct Acc {  // 16 x 8 of a result: rows lane/4 and lane/4 + 8, columns 2 (lane%4) and the next
    float v[4];
    __device__ __forceinline__ void zero() { v[0] = v[1] = v[2] = v[3] = 0.f; }
};

__device__ __forceinline__ void mma(Acc& c, const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c.v[0]), "+f"(c.v[1]), "+f"(c.v[2]), "+f"(c.v[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// c += A B with A in NA terms and B in NB; pairs of terms i + j < kMost, the smallest first.
template <int kMost, int NA, int NB>
__device__ __forceinline__ void mma_terms(Acc& c, const uint32_t (&a)[NA][4], const uint32_t (&b)[NB][2]) {
#pragma unroll
    for (int s = kMost - 1; s >= 0; --s)
#pragma unroll
        for (int i = 0; i < NA; ++i)
            if (s - i >= 0 && s - i < NB) mma(c, a[i], b[s - i][0], b[s - i][1]);
}

__device__ __forceinline__ uint32_t smem_at(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_at(p)));
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_at(p)));
}

// Tiles of 16 tokens x columns in shared memory come in two layouts.  As fetched (TMA): panels of 16 rows of 128 bytes, a
// row's eight 16-byte chunks permuted by the row (chunk c of row r at c ^ (r % 8)), so that eight rows of one chunk fall on
// all banks.  As bf16 terms: rows `ld` elements apart, ld * 2 an odd multiple of 16 bytes.
template <class T>
__device__ __forceinline__ int panel_at(int r, int c) {  // element (r, c) of a fetched tile
    constexpr int kPer = 16 / sizeof(T), kWide = 8 * kPer;
    return c / kWide * (kC * kWide) + r * kWide + ((c / kPer % 8) ^ (r & 7)) * kPer + c % kPer;
}
struct Panels {  // a fetched bf16 tile as an operand
    const __nv_bfloat16* tile;
    __device__ __forceinline__ const __nv_bfloat16* at(int r, int c) const { return tile + panel_at<__nv_bfloat16>(r, c); }
};
struct Rows {  // a tile of terms
    const __nv_bfloat16* tile;
    int ld;
    __device__ __forceinline__ const __nv_bfloat16* at(int r, int c) const { return tile + r * ld + c; }
};
// A operand, rows = tokens, k = columns c0..c0+15.  As a B operand with columns = tokens (K K^T) the same registers
// are {r0, r2} for tokens 0..7 and {r1, r3} for tokens 8..15.
template <class Tile>
__device__ __forceinline__ void load_rows(uint32_t (&r)[4], const Tile& t, int c0, int lane) {
    ldmatrix4(r, t.at(lane % 16, c0 + lane / 16 * 8));
}
// B operand, k = tokens, columns c0..c0+15: {r0, r1} for the first 8 columns, {r2, r3} for the next.
template <class Tile>
__device__ __forceinline__ void load_tokens(uint32_t (&r)[4], const Tile& t, int c0, int lane) {
    ldmatrix4_t(r, t.at(lane % 16, c0 + lane / 16 * 8));
}
// A operand, rows = columns c0..c0+15 of the tile, k = tokens.
template <class Tile>
__device__ __forceinline__ void load_columns(uint32_t (&r)[4], const Tile& t, int c0, int lane) {
    ldmatrix4_t(r, t.at(lane % 8 + lane / 16 * 8, c0 + lane / 8 % 2 * 8));
}

// 16 bytes, or zeros where not `in`.  (A byte count in a register instead of the predicate took 180 clocks a copy.)
__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool in) {
    asm volatile("{\n\t.reg .pred P;\n\tsetp.eq.u32 P, %2, 0;\n\tcp.async.cg.shared.global [%0], [%1], 16, P;\n\t}" ::"r"(smem_at(dst)),
                 "l"(src), "r"((uint32_t)in)
                 : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Rows t0.. of a (tokens, d) tensor into a tile of 16 x D with rows `ld` apart; zeros past the sequence and past d.
template <class T, int D>
__device__ __forceinline__ void stage(T* tile, int ld, const T* src, int64_t stride_t, int64_t t0, int64_t t_end, int d, bool aligned) {
    constexpr int kPer = 16 / sizeof(T), kRow = D / kPer;
    for (int i = threadIdx.x; i < kC * kRow; i += blockDim.x) {
        const int r = i / kRow, c = i % kRow * kPer;
        const bool in = t0 + r < t_end && c < d;
        T* to = tile + r * ld + c;
        const T* from = src + (in ? (t0 + r) * stride_t + c : 0);
        if (aligned) {
            cp_async16(to, from, in);
        } else {
#pragma unroll
            for (int j = 0; j < kPer; ++j) to[j] = in && c + j < d ? from[j] : from_f32<T>(0.f);
        }
    }
}

// A raw tile as its bf16 terms (bf16 itself is used in place).
template <class T, int D>
__device__ __forceinline__ void to_terms(__nv_bfloat16* terms, int ld, const T* raw, int ld_raw) {
    constexpr int N = Terms<T>::n;
    for (int i = threadIdx.x; i < kC * D / 2; i += blockDim.x) {
        const int r = i / (D / 2), c = i % (D / 2) * 2;
        uint32_t s[N];
        split(to_f32(raw[r * ld_raw + c]), to_f32(raw[r * ld_raw + c + 1]), s);
#pragma unroll
        for (int j = 0; j < N; ++j) *reinterpret_cast<uint32_t*>(terms + (j * kC + r) * ld + c) = s[j];
    }
}

// What a warp keeps of a chunk's scalars.
struct alignas(16) Decays {
    float d[kC][kC];   // D_ij, zero above the diagonal and outside the chunk's tokens
    float gamma[kC];   // zero outside, and all zero in a chunk that starts an episode
    float eta[kC];
    float beta[kC];    // zero outside
    float keep;        // Gamma
};

// Tokens r0..r1-1; lane i < 16 holds a_i (1 outside) and beta_i.
__device__ __forceinline__ void fill_decays(Decays& w, float a, float beta, int r0, int r1, bool fresh, int lane) {
    float run = 0.f, last = 0.f;
#pragma unroll
    for (int i = 0; i < kC; ++i) {
        const float ai = __shfl_sync(0xffffffffu, a, i);
        const bool in = i >= r0 && i < r1;
        if (lane == 16)
            run = i == r0 ? (fresh ? 0.f : ai) : run * ai;
        else
            run = i == lane ? (in ? 1.f : 0.f) : run * ai;
        if (lane < 16)
            w.d[i][lane] = in ? run : 0.f;
        else if (lane == 16)
            w.gamma[i] = in ? run : 0.f;
        if (i == r1 - 1) last = run;
    }
    if (lane < 16) {
        w.eta[lane] = lane < r1 ? last : 0.f;
        w.beta[lane] = lane >= r0 && lane < r1 ? beta : 0.f;
    } else if (lane == 16) {
        w.keep = last;
    }
    __syncwarp();
}

// Gate scalars of the 16 tokens of a block, lane i < 16 holding token i: loads only, so that they can be on their way
// while the block before is worked on.
struct Gates {
    float g, beta;
    uint32_t reset;
    __device__ __forceinline__ float decay() const { return expf(g); }
    __device__ __forceinline__ uint32_t starts() const { return __ballot_sync(0xffffffffu, reset != 0); }  // bit i: token i starts an episode
};
struct GatePointers {
    const float *g, *beta;
    const uint8_t* reset;
    int64_t g_t, b_t, r_t;
    __device__ __forceinline__ GatePointers(const Scan& p, int64_t n, int64_t h, int lane)
        : g(p.g + lane * p.sg.t + n * p.sg.n + h * p.sg.h), beta(p.beta + lane * p.sb.t + n * p.sb.n + h * p.sb.h),
          reset(p.reset ? p.reset + lane * p.reset_t + n * p.reset_n : nullptr), g_t(p.sg.t), b_t(p.sb.t), r_t(p.reset_t) {}
    __device__ __forceinline__ Gates load(int64_t t0, int64_t t_end, int lane) const {
        Gates s{0.f, 0.f, 0u};
        if (lane < kC && t0 + lane < t_end) {
            s.g = g[t0 * g_t];
            s.beta = beta[t0 * b_t];
            if (reset) s.reset = reset[t0 * r_t];
        }
        return s;
    }
};

__device__ __forceinline__ bool within(int i, int r0, int r1) { return i >= r0 && i < r1; }
// Halves of a register that holds tokens i and i + 1 of an operand: zero those outside the chunk, whatever they hold.
__device__ __forceinline__ uint32_t pair_mask(int i, int r0, int r1) {
    return (within(i, r0, r1) ? 0xFFFFu : 0u) | (within(i + 1, r0, r1) ? 0xFFFF0000u : 0u);
}

// ---------------------------------------------------------------- forward
//
// A block takes 64 columns of one (env, head)'s state: four warps with 16 each,
// and one helper.  Columns need nothing of one another, so a state warp keeps its
// columns, transposed (dv x dk), in registers for the whole sequence, and works
// in transposed form throughout,
//
//   R^T = V^T - (S^T K^T) gamma    E^T = R^T M^T    U = beta E
//   O^T = (S^T Q^T) gamma + U^T (D o Q K^T)^T       S^T <- Gamma S^T + (eta U)^T K
//
// because the accumulators of one product are then the A operand of the next:
// no state, error or update passes through shared memory.
//
// What the warps would all compute alike is the helper's, one chunk ahead: the
// loads (TMA, two blocks of 16 tokens ahead), the decays, Q K^T and K K^T,
// and M = (I + (D o K K^T) beta)^-1 by substitution, so that the triangular
// solve is a product too.  One barrier a chunk.

constexpr int kLdM = kC + 8;  // bf16 of a row of a 16 x 16 operand tile

struct alignas(16) Chunk {  // a chunk as the helper leaves it
    __nv_bfloat16 m[3][kC][kLdM];    // M, by terms
    __nv_bfloat16 att[3][kC][kLdM];  // D_ij q_i.k_j (i >= j), by terms
    float gamma[kC], eta[kC], beta[kC];
    float keep;
    int block, r0, r1;               // tokens 16 block + r0 .. r1 - 1; block < 0: the sequence is over
    int fresh;                       // starts an episode
};

constexpr int kLdD = 34;

struct alignas(16) HelperScratch {
    float d[kC][kLdD];    // D_ij; column 16: gamma_i; the rest is not read
    float b[kC][kC + 4];  // strictly lower part of the system
    float x[8][8];
};

// Decays of tokens r0..r1-1 (lane i holds a_i; 1 outside): D to scratch, gamma, eta, beta and keep to the chunk.
__device__ __forceinline__ void chunk_decays(float (&d)[kC][kLdD], float (&gamma)[kC], float (&eta)[kC], float (&beta_out)[kC],
                                             float& keep, float a, float beta, int r0, int r1, bool fresh, int lane) {
    // lane j < 16 runs down column j of D from its diagonal, lane 16 down the column before the chunk, which is gamma
    const int start = lane == 16 ? r0 : lane;
    float run = 0.f, last = 0.f;
#pragma unroll
    for (int i = 0; i < kC; ++i) {
        const float ai = __shfl_sync(0xffffffffu, a, i);
        const float begin = lane == 16 ? (fresh ? 0.f : ai) : 1.f;
        run = i == start ? begin : run * ai;
        d[i][lane] = run;
        last = i == r1 - 1 ? run : last;
    }
    __syncwarp();
    const bool in = within(lane, r0, r1);
    if (lane < 16) {
        gamma[lane] = in ? d[lane][16] : 0.f;
        eta[lane] = in ? last : 0.f;
        beta_out[lane] = in ? beta : 0.f;
    } else if (lane == 16) {
        keep = last;
    }
}

// The inverse of I + b, b strictly lower triangular 16 x 16, into b: two 8 x 8 inverses by substitution (lanes 0..7 and
// 8..15, a column each), then the block below them, -M22 b21 M11.
__device__ __forceinline__ void invert_lower(HelperScratch& hs, int lane) {
    if (lane < 16) {
        const int o = lane & 8, c = lane & 7;
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = i == c ? 1.f : 0.f;
#pragma unroll
        for (int j = 0; j < 7; ++j)
#pragma unroll
            for (int i = j + 1; i < 8; ++i) x[i] = fmaf(-hs.b[o + i][o + j], x[j], x[i]);
        __syncwarp(0xffffu);
#pragma unroll
        for (int i = 0; i < 8; ++i) hs.b[o + i][o + c] = x[i];
    }
    __syncwarp();
    const int i = lane / 4, j = lane % 4 * 2;  // 64 entries, two a lane
    float y0 = 0.f, y1 = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float l = hs.b[8 + i][k];
        y0 = fmaf(l, hs.b[k][j], y0);
        y1 = fmaf(l, hs.b[k][j + 1], y1);
    }
    hs.x[i][j] = y0;
    hs.x[i][j + 1] = y1;
    __syncwarp();
    y0 = y1 = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float l = hs.b[8 + i][8 + k];
        y0 = fmaf(-l, hs.x[k][j], y0);
        y1 = fmaf(-l, hs.x[k][j + 1], y1);
    }
    hs.b[8 + i][j] = y0;
    hs.b[8 + i][j + 1] = y1;
    hs.b[i][8 + j] = 0.f;
    hs.b[i][8 + j + 1] = 0.f;
    __syncwarp();
}

// A 16 x 16 fp32 matrix in scratch as N bf16 terms.
template <int N>
__device__ __forceinline__ void store_terms(__nv_bfloat16 (&out)[3][kC][kLdM], const float (&in)[kC][kC + 4], int lane) {
#pragma unroll
    for (int z = 0; z < 4; ++z) {
        const int i = z * 4 + lane / 8, j = lane % 8 * 2;
        const float2 v = *reinterpret_cast<const float2*>(&in[i][j]);
        uint32_t s[N];
        split(v.x, v.y, s);
#pragma unroll
        for (int x = 0; x < N; ++x) *reinterpret_cast<uint32_t*>(&out[x][i][j]) = s[x];
    }
}

// 16 x 16 operand tile as a B operand whose columns are the tile's rows.
template <int N>
__device__ __forceinline__ void load_operand(uint32_t (&r)[N][4], const __nv_bfloat16 (&tile)[3][kC][kLdM], int lane) {
#pragma unroll
    for (int x = 0; x < N; ++x) load_rows(r[x], Rows{&tile[x][0][0], kLdM}, 0, lane);
}

// One env and head's rows of a (t, n, h, d) tensor, 16 tokens at a time, into fetched tiles by one warp.  Where rows are
// whole 16-byte chunks at 16-byte strides (`aligned`) one lane asks TMA for each panel, which also fills with zeros past the
// sequence and past d; else the warp copies elements, and columns past d keep the zeros that the block put there.
// (Alternatives on the way here, a block of 16 tokens x 3 x 64: 12 cp.async a lane 1,150 clocks of the helper's time,
// 48 bulk copies of a row 3,550.)
template <class T, int D>
struct Fetch {
    static constexpr int kWide = 128 / sizeof(T), kPanels = (D + kWide - 1) / kWide;
    static constexpr int kElements = kPanels * kC * kWide;
    static __device__ __forceinline__ void run(T* tile, const CUtensorMap* map, const T* rows, int64_t stride_t, int64_t n, int64_t h,
                                               int col, int64_t t0, int count, int d, bool aligned, uint64_t* bar, int lane) {
        if (aligned) {
            if (lane == 0) {
#pragma unroll
                for (int i = 0; i < kPanels; ++i)
                    tc::tma_load_4d(tile + i * kC * kWide, map, bar, col + i * kWide, (int)h, (int)n, (int)t0);
            }
        } else {
            for (int r = 0; r < count; ++r)
                for (int c = lane; c < d; c += 32) tile[panel_at<T>(r, c)] = rows[(t0 + r) * stride_t + col + c];
        }
    }
};

template <class T, int D>
__device__ __forceinline__ void to_terms_warp(__nv_bfloat16* terms, int ld, const T* raw, int lane) {
    constexpr int N = Terms<T>::n;
    for (int i = lane; i < kC * D / 2; i += 32) {
        const int r = i / (D / 2), c = i % (D / 2) * 2;
        uint32_t s[N];
        const T* at = raw + panel_at<T>(r, c);
        split(to_f32(at[0]), to_f32(at[1]), s);
#pragma unroll
        for (int j = 0; j < N; ++j) *reinterpret_cast<uint32_t*>(terms + (j * kC + r) * ld + c) = s[j];
    }
}

constexpr int kLdOut = 24;  // 16-bit elements of a row of a warp's 16 x 16 tile on its way out

constexpr int kForwardWarps = 4;  // state warps of a block: 64 columns

template <class T, int DK>
struct ForwardSmem {
    static constexpr int kWidth = kForwardWarps * 16;
    static constexpr int kLdTerm = DK + 8;  // rows of terms
    static constexpr bool kInPlace = Terms<T>::n == 1;
    static constexpr int kBuffers = 4;  // state warps on one block, the helper on the next, two on their way
    static constexpr int kTileK = Fetch<T, DK>::kElements, kTileV = Fetch<T, kWidth>::kElements;
    static constexpr size_t kRaw = (size_t)(2 * kTileK + kTileV) * sizeof(T);                        // a buffer
    static constexpr size_t kTerms = kInPlace ? 0 : (size_t)2 * 2 * Terms<T>::n * kC * kLdTerm * 2;  // of two blocks
    static constexpr int kLdS = 20;  // floats of a row of a warp's columns of the state on their way out
    static constexpr size_t kOut = (size_t)DK * kLdS * 4;  // of a warp: that, or its 16 x 16 outputs
    static constexpr size_t kBytes = 1024 + kBuffers * kRaw + kTerms + 2 * sizeof(Chunk) + sizeof(HelperScratch) + kForwardWarps * kOut + 8 * kBuffers;
    static_assert(kRaw % 1024 == 0 && kTerms % 16 == 0 && kOut % 16 == 0 && kOut >= kC * kLdOut * 2, "layout");
};

template <class T, int DK>
__global__ void __launch_bounds__((kForwardWarps + 1) * 32, DK == 128 ? 2 : 3)
    scan_forward_kernel(const Scan p, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_q,
                        const __grid_constant__ CUtensorMap map_v) {
    using L = ForwardSmem<T, DK>;
    constexpr int NT = Terms<T>::n, kTiles = DK / 8, kSteps = DK / 16;
    constexpr int NO = NT == 3 ? 3 : 2;  // terms that o needs: 16 bits and more against its own 8 or 11
    extern __shared__ __align__(16) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + (1024 - (smem_at(smem_raw) & 1023) & 1023);
    constexpr int warps = kForwardWarps;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, row = lane / 4, quad = lane % 4;
    __nv_bfloat16* terms = reinterpret_cast<__nv_bfloat16*>(smem + L::kBuffers * L::kRaw);
    Chunk* chunks = reinterpret_cast<Chunk*>(smem + L::kBuffers * L::kRaw + L::kTerms);
    HelperScratch& hs = *reinterpret_cast<HelperScratch*>(chunks + 2);
    float* out_tiles = reinterpret_cast<float*>(&hs + 1);
    uint64_t* arrived = reinterpret_cast<uint64_t*>(out_tiles + warps * L::kOut / 4);  // a buffer's rows are there
    const int64_t seq = blockIdx.x, n = seq / p.h, h = seq % p.h;
    const int first_col = blockIdx.y * L::kWidth, cols = min(L::kWidth, p.dv - first_col);
    const int64_t blocks = (p.t + kC - 1) / kC;
    auto raw_tile = [&](int64_t b) { return reinterpret_cast<T*>(smem + b % L::kBuffers * L::kRaw); };
    // term x of K (which = 0) or Q (1) of a block as an operand
    auto operand = [&](int64_t b, int which, int x) {
        if constexpr (L::kInPlace)
            return Panels{reinterpret_cast<const __nv_bfloat16*>(raw_tile(b)) + which * L::kTileK};
        else
            return Rows{terms + ((b & 1) * 2 * NT + which * NT + x) * kC * L::kLdTerm, L::kLdTerm};
    };
    if (!p.aligned)
        for (int i = threadIdx.x; i < (int)(L::kBuffers * L::kRaw / 16); i += blockDim.x)
            reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kBuffers; ++i) tc::mbar_init(&arrived[i], 1);
        tc::mbar_init_fence();
        tc::prefetch_map(&map_k);
        tc::prefetch_map(&map_q);
        tc::prefetch_map(&map_v);
    }
    __syncthreads();

    if (warp == warps) {
        const T* q = static_cast<const T*>(p.q) + n * p.sq.n + h * p.sq.h;
        const T* k = static_cast<const T*>(p.k) + n * p.sk.n + h * p.sk.h;
        const T* v = static_cast<const T*>(p.v) + n * p.sv.n + h * p.sv.h;
        auto fetch = [&](int64_t b) {
            if (b >= blocks) return;
            T* to = raw_tile(b);
            uint64_t* bar = &arrived[b % L::kBuffers];
            const int count = (int)(p.t - b * kC < kC ? p.t - b * kC : kC);
            if (p.aligned && lane == 0) tc::mbar_expect_tx(bar, (uint32_t)L::kRaw);
            Fetch<T, DK>::run(to, &map_k, k, p.sk.t, n, h, 0, b * kC, count, p.dk, p.aligned, bar, lane);
            Fetch<T, DK>::run(to + L::kTileK, &map_q, q, p.sq.t, n, h, 0, b * kC, count, p.dk, p.aligned, bar, lane);
            Fetch<T, L::kWidth>::run(to + 2 * L::kTileK, &map_v, v, p.sv.t, n, h, first_col, b * kC, count, cols, p.aligned, bar, lane);
        };
        fetch(0);
        fetch(1);
        const GatePointers get_gates(p, n, h, lane);
        Gates gates{}, next = get_gates.load(0, p.t, lane);
        float decay = 1.f;
        uint32_t starts = 0;
        int64_t b = -1;
        int r0 = 0, count = 0;
        for (int turn = 0;; ++turn) {
            Chunk& ch = chunks[turn & 1];
            if (r0 >= count) {  // the next block of 16 tokens
                ++b;
                r0 = 0;
                if (b >= blocks) {
                    if (lane == 0) ch.block = -1;
                    __syncthreads();
                    break;
                }
                count = (int)(p.t - b * kC < kC ? p.t - b * kC : kC);
                gates = next;
                next = get_gates.load((b + 1) * kC, p.t, lane);
                decay = gates.decay();
                starts = gates.starts();
                if (p.aligned && !tc::mbar_wait_warp(&arrived[b % L::kBuffers], b / L::kBuffers & 1)) {
                    if (lane == 0) {
                        atomicAdd(p.stalls, 1u);
                        ch.block = -1;
                    }
                    __syncthreads();
                    break;
                }
                __syncwarp();
                fetch(b + 2);
                if constexpr (!L::kInPlace) {
                    __nv_bfloat16* to = terms + (b & 1) * 2 * NT * kC * L::kLdTerm;
                    to_terms_warp<T, DK>(to, L::kLdTerm, raw_tile(b), lane);
                    to_terms_warp<T, DK>(to + NT * kC * L::kLdTerm, L::kLdTerm, raw_tile(b) + L::kTileK, lane);
                    __syncwarp();
                }
            }
            const bool fresh = starts >> r0 & 1;
            const uint32_t later = starts & ~((2u << r0) - 1);
            const int r1 = later ? min(count, __ffs(later) - 1) : count;
            chunk_decays(hs.d, ch.gamma, ch.eta, ch.beta, ch.keep, within(lane, r0, r1) ? decay : 1.f, gates.beta, r0, r1, fresh, lane);
            if (lane == 0) ch.block = (int)b, ch.r0 = r0, ch.r1 = r1, ch.fresh = fresh;
            Acc kk[2], qk[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) kk[i].zero(), qk[i].zero();
#pragma unroll
            for (int st = 0; st < kSteps; ++st) {
                uint32_t ka[NT][4], qa[NT][4];
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    load_rows(ka[x], operand(b, 0, x), st * 16, lane);
                    load_rows(qa[x], operand(b, 1, x), st * 16, lane);
                }
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t kb[NT][2];
#pragma unroll
                    for (int x = 0; x < NT; ++x) kb[x][0] = ka[x][c], kb[x][1] = ka[x][c + 2];
                    mma_terms<3>(kk[c], ka, kb);
                    mma_terms<NO>(qk[c], qa, kb);
                }
            }
            __syncwarp();
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int i = row + half * 8, j = c * 8 + quad * 2;
                    const float2 d = *reinterpret_cast<const float2*>(&hs.d[i][j]);
                    const float2 be = *reinterpret_cast<const float2*>(&ch.beta[j]);
                    const bool in0 = within(i, r0, r1) && j >= r0, in1 = within(i, r0, r1) && j + 1 >= r0;  // and j <= i
                    *reinterpret_cast<float2*>(&hs.b[i][j]) = make_float2(in0 && i > j ? d.x * be.x * kk[c].v[half * 2] : 0.f,
                                                                          in1 && i > j + 1 ? d.y * be.y * kk[c].v[half * 2 + 1] : 0.f);
                    uint32_t s[NO];
                    split(in0 && i >= j ? d.x * qk[c].v[half * 2] : 0.f, in1 && i >= j + 1 ? d.y * qk[c].v[half * 2 + 1] : 0.f, s);
#pragma unroll
                    for (int x = 0; x < NO; ++x) *reinterpret_cast<uint32_t*>(&ch.att[x][i][j]) = s[x];
                }
            __syncwarp();
            invert_lower(hs, lane);
            store_terms<3>(ch.m, hs.b, lane);
            __syncwarp();  // scratch is free
            r0 = r1;
            __syncthreads();
        }
        return;
    }

    const int v0 = warp * 16, c0 = first_col + v0;  // this warp's columns of the state
    const bool whole = p.dk == DK && c0 + 16 <= p.dv;
    float* state_tile = out_tiles + warp * L::kOut / 4;
    __nv_bfloat16* out_tile = reinterpret_cast<__nv_bfloat16*>(state_tile);
    const bool s_aligned = p.dv % 4 == 0 && reinterpret_cast<uintptr_t>(p.checkpoints) % 16 == 0 &&
                           reinterpret_cast<uintptr_t>(p.final_state) % 16 == 0;
    const bool o_aligned = sizeof(T) == 2 && p.dv % 8 == 0 && reinterpret_cast<uintptr_t>(p.o) % 16 == 0;
    Acc s[kTiles];  // S^T: rows = columns c0.. of the state, columns = dk
    // where this thread's values of a (dk, dv) matrix lie: value e of tile i at i * 8 * dv + at(e)
    auto each_state = [&](auto&& f) {
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int kk = i * 8 + quad * 2 + e % 2, c = c0 + row + e / 2 * 8;
                f(s[i].v[e], kk * p.dv + c, whole || (kk < p.dk && c < p.dv));
            }
    };
    {
        const float* s0 = p.state ? p.state + seq * p.dk * p.dv : nullptr;
        each_state([&](float& x, int at, bool in) { x = s0 && in ? s0[at] : 0.f; });
    }
    // The state to a (dk, dv) matrix: through shared memory, 16 columns of a row at a time, so that stores are 16 bytes.
    auto put_state = [&](float* to) {
        if (whole && s_aligned) {
#pragma unroll
            for (int i = 0; i < kTiles; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) state_tile[(i * 8 + quad * 2 + e % 2) * L::kLdS + row + e / 2 * 8] = s[i].v[e];
            __syncwarp();
            float4* out = reinterpret_cast<float4*>(to + (lane / 4) * p.dv + c0 + lane % 4 * 4);
#pragma unroll
            for (int i = 0; i < DK / 8; ++i)
                __stcs(out + i * 2 * p.dv, *reinterpret_cast<const float4*>(state_tile + (i * 8 + lane / 4) * L::kLdS + lane % 4 * 4));
            __syncwarp();
        } else {
            each_state([&](float& x, int at, bool in) {
                if (in) to[at] = x;
            });
        }
    };
    const int64_t step_t = p.n * p.h * p.dv, first = (n * p.h + h) * p.dv + c0;
    for (int turn = 0;; ++turn) {
        __syncthreads();
        const Chunk& ch = chunks[turn & 1];
        const int64_t b = ch.block;
        if (b < 0) break;
        if (p.aligned) tc::mbar_wait_warp(&arrived[b % L::kBuffers], b / L::kBuffers & 1);  // long since; it makes the copies visible here
        const int r0 = ch.r0, r1 = ch.r1;
        if (p.checkpoints && r0 == 0) put_state(p.checkpoints + (seq * blocks + b) * p.dk * p.dv);
        if (ch.fresh) {
#pragma unroll
            for (int i = 0; i < kTiles; ++i) s[i].zero();
        }
        Acc ks[2], qs[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) ks[i].zero(), qs[i].zero();
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
            uint32_t sa[3][4];
#pragma unroll
            for (int z = 0; z < 4; ++z) {
                uint32_t tmp[3];
                const Acc& t = s[2 * st + z / 2];
                split(t.v[z % 2 * 2], t.v[z % 2 * 2 + 1], tmp);
#pragma unroll
                for (int x = 0; x < 3; ++x) sa[x][z] = tmp[x];
            }
            uint32_t ka[NT][4], qa[NT][4];
#pragma unroll
            for (int x = 0; x < NT; ++x) {
                load_rows(ka[x], operand(b, 0, x), st * 16, lane);
                load_rows(qa[x], operand(b, 1, x), st * 16, lane);
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t kb[NT][2], qb[NT][2];
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    kb[x][0] = ka[x][c], kb[x][1] = ka[x][c + 2];
                    qb[x][0] = qa[x][c], qb[x][1] = qa[x][c + 2];
                }
                mma_terms<3>(ks[c], sa, kb);
                mma_terms<NO>(qs[c], sa, qb);
            }
        }
        // R^T; tokens outside the chunk are zero whatever their inputs hold
        uint32_t ra[3][4];
        {
            const T* tv = raw_tile(b) + 2 * L::kTileK;
            uint32_t vv[4];
            if constexpr (L::kInPlace) load_columns(vv, Panels{reinterpret_cast<const __nv_bfloat16*>(tv)}, v0, lane);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int j = c * 8 + quad * 2;
                const float2 ga = *reinterpret_cast<const float2*>(&ch.gamma[j]);
                const bool in0 = within(j, r0, r1), in1 = within(j + 1, r0, r1);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float x0, x1;
                    if constexpr (L::kInPlace) {
                        x0 = __uint_as_float(vv[c * 2 + half] << 16);
                        x1 = __uint_as_float(vv[c * 2 + half] & 0xFFFF0000u);
                    } else {
                        x0 = to_f32(tv[panel_at<T>(j, v0 + row + half * 8)]);
                        x1 = to_f32(tv[panel_at<T>(j + 1, v0 + row + half * 8)]);
                    }
                    uint32_t tmp[3];
                    split(in0 ? fmaf(-ga.x, ks[c].v[half * 2], x0) : 0.f, in1 ? fmaf(-ga.y, ks[c].v[half * 2 + 1], x1) : 0.f, tmp);
#pragma unroll
                    for (int x = 0; x < 3; ++x) ra[x][c * 2 + half] = tmp[x];
                }
                qs[c].v[0] *= ga.x, qs[c].v[1] *= ga.y, qs[c].v[2] *= ga.x, qs[c].v[3] *= ga.y;
            }
        }
        uint32_t uo[NO][4], ue[3][4];  // U^T and (eta U)^T
        {
            uint32_t mb[3][4];
            load_operand(mb, ch.m, lane);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t bb[3][2];
#pragma unroll
                for (int x = 0; x < 3; ++x) bb[x][0] = mb[x][c], bb[x][1] = mb[x][c + 2];
                Acc e;
                e.zero();
                mma_terms<3>(e, ra, bb);
                const int j = c * 8 + quad * 2;
                if (p.errors) {
                    float* er = p.errors + (b * kC + j) * step_t + first + row;
#pragma unroll
                    for (int z = 0; z < 4; ++z)
                        if (within(j + z % 2, r0, r1) && (whole || c0 + row + z / 2 * 8 < p.dv)) __stcs(er + z % 2 * step_t + z / 2 * 8, e.v[z]);
                }
                const float2 be = *reinterpret_cast<const float2*>(&ch.beta[j]), et = *reinterpret_cast<const float2*>(&ch.eta[j]);
                const float h0 = be.x * et.x, h1 = be.y * et.y;  // rounded once more than beta e, then eta: 2^-24
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t t2[NO], t3[3];
                    split(be.x * e.v[half * 2], be.y * e.v[half * 2 + 1], t2);
                    split(h0 * e.v[half * 2], h1 * e.v[half * 2 + 1], t3);
#pragma unroll
                    for (int x = 0; x < NO; ++x) uo[x][c * 2 + half] = t2[x];
#pragma unroll
                    for (int x = 0; x < 3; ++x) ue[x][c * 2 + half] = t3[x];
                }
            }
        }
        {
            uint32_t ab[NO][4];
            load_operand(ab, ch.att, lane);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t bb[NO][2];
#pragma unroll
                for (int x = 0; x < NO; ++x) bb[x][0] = ab[x][c], bb[x][1] = ab[x][c + 2];
                mma_terms<NO>(qs[c], uo, bb);
            }
        }
        if (o_aligned && whole) {  // by a transposed tile in shared memory, 16 bytes a lane
            if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int z = 0; z < 4; ++z)
                        reinterpret_cast<T*>(out_tile)[(c * 8 + quad * 2 + z % 2) * kLdOut + row + z / 2 * 8] = from_f32<T>(p.scale * qs[c].v[z]);
                __syncwarp();
                const int i = lane / 2;
                if (within(i, r0, r1))
                    *reinterpret_cast<uint4*>(static_cast<T*>(p.o) + (b * kC + i) * step_t + first + lane % 2 * 8) =
                        *reinterpret_cast<const uint4*>(out_tile + i * kLdOut + lane % 2 * 8);
                __syncwarp();
            }
        } else {
            T* o = static_cast<T*>(p.o) + b * kC * step_t + first + row;
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    const int i = c * 8 + quad * 2 + z % 2;
                    if (within(i, r0, r1) && (whole || c0 + row + z / 2 * 8 < p.dv)) o[i * step_t + z / 2 * 8] = from_f32<T>(p.scale * qs[c].v[z]);
                }
        }
        const float keep = ch.keep;
        const uint32_t m0 = pair_mask(quad * 2, r0, r1), m1 = pair_mask(quad * 2 + 8, r0, r1);
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
            uint32_t kb[NT][4];
#pragma unroll
            for (int x = 0; x < NT; ++x) load_tokens(kb[x], operand(b, 0, x), st * 16, lane);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                Acc& acc = s[2 * st + c];
#pragma unroll
                for (int e = 0; e < 4; ++e) acc.v[e] *= keep;
                uint32_t bb[NT][2];
#pragma unroll
                for (int x = 0; x < NT; ++x) bb[x][0] = kb[x][2 * c] & m0, bb[x][1] = kb[x][2 * c + 1] & m1;
                mma_terms<3>(acc, ue, bb);
            }
        }
    }
    if (p.final_state) put_state(p.final_state + seq * p.dk * p.dv);
}

// --------------------------------------------------------------- backward
//
// Over the chunks from last to first, with dS the gradient of the state after
// the chunk, E and the state S before it kept by the forward pass:
//
//   dU = scale (D o Q K^T)^T dO + eta K dS        (I + L)^T dR = dU,  L = beta D o K K^T (i > j)
//   dV = beta dR    dbeta_i = dR_i . e_i    dL = -dR U^T    W = dO U^T
//   dA = scale D o W (i >= j)    dP = beta D o dL (i > j)
//   dQ = scale gamma dO S^T + dA K
//   dK = -beta gamma dR S^T + eta U dS^T + dA^T Q + (dP + dP^T) K
//   dS <- Gamma dS + (scale gamma Q)^T dO - (beta gamma K)^T dR
//   dg_l = sum_{i>=l>j} E_ij + sum_{i>=l} (q_i . dq_i^S + k_i . dk_i^S) + sum_{j<l} k_j . dk_j^{dS} + Gamma <dS, S>
//   E_ij = dA_ij q_i.k_j + dP_ij k_i.k_j
//
// (^S and ^{dS}: the parts of dq and dk that come through S and dS.)  A block
// takes one (env, head).  A warp has two parts: 16 columns of dS, transposed,
// for what sums over dk (dU), and 16 rows of dS for what sums over dv (dQ, dK);
// both copies stay in registers.  X = -beta gamma dR, Y = scale gamma dO and U
// go through shared memory as bf16 terms.

constexpr int kRowPad = 20;  // floats of a row of a warp's 16 x 16 scratch

template <class T, int DK, int DV>
struct BackwardSmem {
    static constexpr int kWarps = (DK > DV ? DK : DV) / 16, kWarpsV = DV / 16, kWarpsK = DK / 16;
    static constexpr int kPad = 16 / sizeof(T);
    static constexpr int kLdK = DK + kPad, kLdV = DV + kPad;   // raw rows
    static constexpr int kTk = DK + 8, kTv = DV + 8;           // rows of terms; the same for bf16
    static constexpr int NT = Terms<T>::n;
    static constexpr bool kInPlace = NT == 1;
    static constexpr int kLdE = DV + 4;
    static constexpr size_t kRaw = (size_t)kC * (2 * kLdK + kLdV) * sizeof(T) + (size_t)kC * kLdE * 4;  // of one buffer
    static constexpr size_t kTerms = kInPlace ? 0 : (size_t)NT * kC * (2 * kTk + kTv) * 2;
    static constexpr size_t kTile3 = (size_t)3 * kC * kTv * 2;
    struct alignas(16) Shared {
        float part[kWarpsV][2][kC][kC];      // W and dL by slices of dv
        float qk[kC][kC], kk[kC][kC];        // q_i.k_j, k_i.k_j
        float da[kC][kC + 1], dp[kC][kC + 1], ee[kC][kC + 1];
        float dot_i[kWarpsK][kC], dot_j[kWarpsK][kC], dot_s[kWarpsK], dbeta[kWarpsV][kC];
    };
    struct alignas(16) Warp {
        Decays w;
        float l[kC][kC];        // L_ij at [i][j]
        float r[kC][kRowPad];   // dU, then dR
    };
    static_assert(offsetof(Warp, r) % 16 == 0 && kRaw % 16 == 0 && kTerms % 16 == 0 && kTile3 % 16 == 0, "alignment of vector accesses");
    static constexpr size_t kBytes = 2 * kRaw + kTerms + 3 * kTile3 + sizeof(Shared) + kWarps * sizeof(Warp);
};

template <class T, int DK, int DV>
__global__ void __launch_bounds__((DK > DV ? DK : DV) * 2) scan_backward_kernel(const Scan p) {
    using L = BackwardSmem<T, DK, DV>;
    constexpr int NT = Terms<T>::n;
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, row = lane / 4, quad = lane % 4;
    __nv_bfloat16* terms = reinterpret_cast<__nv_bfloat16*>(smem + 2 * L::kRaw);
    __nv_bfloat16* ut = reinterpret_cast<__nv_bfloat16*>(smem + 2 * L::kRaw + L::kTerms);
    __nv_bfloat16* xt = ut + 3 * kC * L::kTv;
    __nv_bfloat16* yt = xt + 3 * kC * L::kTv;
    typename L::Shared& sh = *reinterpret_cast<typename L::Shared*>(smem + 2 * L::kRaw + L::kTerms + 3 * L::kTile3);
    typename L::Warp& ws = reinterpret_cast<typename L::Warp*>(&sh + 1)[warp];
    const int64_t seq = blockIdx.x, n = seq / p.h, h = seq % p.h;
    const T* q = static_cast<const T*>(p.q) + n * p.sq.n + h * p.sq.h;
    const T* k = static_cast<const T*>(p.k) + n * p.sk.n + h * p.sk.h;
    const int64_t out_t = p.n * p.h, out_0 = n * p.h + h;  // rows of contiguous (t, n, h, d) tensors
    const T* d_o = static_cast<const T*>(p.d_o) + out_0 * p.dv;
    const float* errors = p.errors + out_0 * p.dv;
    const int64_t blocks = (p.t + kC - 1) / kC;
    const bool has_v = warp < L::kWarpsV, has_k = warp < L::kWarpsK;
    const int c0 = warp * 16;
    const bool e_aligned = p.dv % 4 == 0;

    auto fetch = [&](int64_t b, int buf) {
        T* to = reinterpret_cast<T*>(smem + buf * L::kRaw);
        stage<T, DK>(to, L::kLdK, k, p.sk.t, b * kC, p.t, p.dk, p.aligned);
        stage<T, DK>(to + kC * L::kLdK, L::kLdK, q, p.sq.t, b * kC, p.t, p.dk, p.aligned);
        stage<T, DV>(to + 2 * kC * L::kLdK, L::kLdV, d_o, out_t * p.dv, b * kC, p.t, p.dv, p.aligned);
        stage<float, DV>(reinterpret_cast<float*>(to + kC * (2 * L::kLdK + L::kLdV)), L::kLdE, errors, out_t * p.dv, b * kC, p.t,
                         p.dv, e_aligned);
        cp_async_commit();
    };

    // dS twice: rows c0.. (dk) x dv, and columns c0.. (dv) x dk transposed.
    Acc ds[DV / 8], dst[DK / 8];
    const float* df = p.d_final ? p.d_final + seq * p.dk * p.dv : nullptr;
#pragma unroll
    for (int i = 0; i < DV / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int kk = c0 + row + e / 2 * 8, c = i * 8 + quad * 2 + e % 2;
            ds[i].v[e] = df && kk < p.dk && c < p.dv ? df[(int64_t)kk * p.dv + c] : 0.f;
        }
#pragma unroll
    for (int i = 0; i < DK / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int kk = i * 8 + quad * 2 + e % 2, c = c0 + row + e / 2 * 8;
            dst[i].v[e] = df && kk < p.dk && c < p.dv ? df[(int64_t)kk * p.dv + c] : 0.f;
        }

    if (blocks) fetch(blocks - 1, (blocks - 1) & 1);
    const GatePointers get_gates(p, n, h, lane);
    Gates next = get_gates.load((blocks - 1) * kC, p.t, lane);
    for (int64_t b = blocks - 1; b >= 0; --b) {
        const int buf = b & 1;
        cp_async_wait<0>();
        __syncthreads();
        if (b > 0) fetch(b - 1, buf ^ 1);
        const Gates gates = next;
        if (b > 0) next = get_gates.load((b - 1) * kC, p.t, lane);
        const uint32_t starts = gates.starts();
        const T* rk = reinterpret_cast<const T*>(smem + buf * L::kRaw);
        const T* rq = rk + kC * L::kLdK;
        const T* ro = rq + kC * L::kLdK;
        const float* er = reinterpret_cast<const float*>(ro + kC * L::kLdV);
        const __nv_bfloat16 *kt, *qt, *ot;
        if constexpr (L::kInPlace) {
            kt = reinterpret_cast<const __nv_bfloat16*>(rk);
            qt = reinterpret_cast<const __nv_bfloat16*>(rq);
            ot = reinterpret_cast<const __nv_bfloat16*>(ro);
        } else {
            kt = terms;
            qt = terms + NT * kC * L::kTk;
            ot = terms + 2 * NT * kC * L::kTk;
            to_terms<T, DK>(terms, L::kTk, rk, L::kLdK);
            to_terms<T, DK>(terms + NT * kC * L::kTk, L::kTk, rq, L::kLdK);
            to_terms<T, DV>(terms + 2 * NT * kC * L::kTk, L::kTv, ro, L::kLdV);
            __syncthreads();
        }
        const int count = (int)(p.t - b * kC < kC ? p.t - b * kC : kC);
        for (int r1 = count; r1 > 0;) {
            const uint32_t earlier = starts & ((1u << r1) - 1);
            const int r0 = earlier ? 31 - __clz(earlier) : 0;
            const bool fresh = starts >> r0 & 1;
            fill_decays(ws.w, within(lane, r0, r1) ? gates.decay() : 1.f, gates.beta, r0, r1, fresh, lane);
            const uint32_t m0 = pair_mask(quad * 2, r0, r1), m1 = pair_mask(quad * 2 + 8, r0, r1);

            // k_i.k_j, and k_j.q_i with tokens j as rows; dU through dS
            Acc kk[2], kq[2], du[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) kk[c].zero(), kq[c].zero(), du[c].zero();
#pragma unroll
            for (int st = 0; st < DK / 16; ++st) {
                uint32_t ka[NT][4], qa[NT][4];
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    load_rows(ka[x], Rows{kt + x * kC * L::kTk, L::kTk}, st * 16, lane);
                    load_rows(qa[x], Rows{qt + x * kC * L::kTk, L::kTk}, st * 16, lane);
                }
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t kb[NT][2], qb[NT][2], sb[3][2], lo[3], hi[3];
#pragma unroll
                    for (int x = 0; x < NT; ++x) {
                        kb[x][0] = ka[x][c], kb[x][1] = ka[x][c + 2];
                        qb[x][0] = qa[x][c], qb[x][1] = qa[x][c + 2];
                    }
                    mma_terms<3>(kk[c], ka, kb);
                    mma_terms<3>(kq[c], ka, qb);
                    split(dst[2 * st].v[2 * c], dst[2 * st].v[2 * c + 1], lo);
                    split(dst[2 * st + 1].v[2 * c], dst[2 * st + 1].v[2 * c + 1], hi);
#pragma unroll
                    for (int x = 0; x < 3; ++x) sb[x][0] = lo[x], sb[x][1] = hi[x];
                    mma_terms<3>(du[c], ka, sb);
                }
            }
            uint32_t att[3][4];  // scale (D o Q K^T)^T: rows j, k = i
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int x = row + half * 8, y = c * 8 + quad * 2;
                    float at[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const bool in = within(x, r0, r1) && within(y + e, r0, r1);
                        const float raw_kk = kk[c].v[half * 2 + e], raw_kq = kq[c].v[half * 2 + e];
                        ws.l[x][y + e] = in && x > y + e ? ws.w.beta[x] * ws.w.d[x][y + e] * raw_kk : 0.f;
                        at[e] = in && y + e >= x ? p.scale * ws.w.d[y + e][x] * raw_kq : 0.f;
                        if (warp == 0) {
                            sh.kk[x][y + e] = in ? raw_kk : 0.f;
                            sh.qk[y + e][x] = in ? raw_kq : 0.f;
                        }
                    }
                    uint32_t tmp[3];
                    split(at[0], at[1], tmp);
#pragma unroll
                    for (int z = 0; z < 3; ++z) att[z][c * 2 + half] = tmp[z];
                }
            if (has_v) {
                uint32_t ob[NT][4];
#pragma unroll
                for (int x = 0; x < NT; ++x) load_tokens(ob[x], Rows{ot + x * kC * L::kTv, L::kTv}, c0, lane);
                const float e0 = ws.w.eta[row], e1 = ws.w.eta[row + 8];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    du[c].v[0] *= e0, du[c].v[1] *= e0, du[c].v[2] *= e1, du[c].v[3] *= e1;
                    uint32_t bb[NT][2];
#pragma unroll
                    for (int x = 0; x < NT; ++x) bb[x][0] = ob[x][2 * c] & m0, bb[x][1] = ob[x][2 * c + 1] & m1;
                    mma_terms<3>(du[c], att, bb);
#pragma unroll
                    for (int half = 0; half < 2; ++half)
                        *reinterpret_cast<float2*>(&ws.r[row + half * 8][c * 8 + quad * 2]) =
                            make_float2(du[c].v[half * 2], du[c].v[half * 2 + 1]);
                }
                __syncwarp();
                float part[kC];
#pragma unroll
                for (int i = 0; i < kC; ++i) part[i] = 0.f;
                if (lane < 16) {  // one column each: back substitution
                    float x[kC];
#pragma unroll
                    for (int i = 0; i < kC; ++i) x[i] = ws.r[i][lane];
                    T* dv = static_cast<T*>(p.dv_out) + (b * kC * out_t + out_0) * p.dv + c0 + lane;
#pragma unroll
                    for (int i = kC - 1; i >= 0; --i) {
                        const bool in = within(i, r0, r1);
                        const float r = in ? x[i] : 0.f;
                        ws.r[i][lane] = r;
                        if (in && c0 + lane < p.dv) dv[i * out_t * p.dv] = from_f32<T>(ws.w.beta[i] * r);
                        part[i] = in ? r * er[i * L::kLdE + c0 + lane] : 0.f;
#pragma unroll
                        for (int j = 0; j < i; ++j) x[j] = fmaf(-ws.l[i][j], r, x[j]);
                    }
                }
                // dbeta: 16 sums over 16 lanes, halving the sums that a lane carries at each exchange
#pragma unroll
                for (int bit = 3; bit >= 0; --bit) {
                    const int w = 1 << bit;
                    const bool up = lane & w;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (i >= w) break;
                        const float give = up ? part[i] : part[i + w], have = up ? part[i + w] : part[i];
                        part[i] = have + __shfl_xor_sync(0xffffffffu, give, w);
                    }
                }
                if (lane < 16) sh.dbeta[warp][lane] = part[0];
                __syncwarp();
                // U, X, Y of this warp's columns as terms
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    const int i = z * 4 + lane / 8, c = lane % 8 * 2;
                    const bool in = within(i, r0, r1);
                    const float be = ws.w.beta[i], ga = ws.w.gamma[i];
                    const float2 e = *reinterpret_cast<const float2*>(er + i * L::kLdE + c0 + c);
                    const float2 r = *reinterpret_cast<const float2*>(&ws.r[i][c]);
                    const float y0 = to_f32(ro[i * L::kLdV + c0 + c]), y1 = to_f32(ro[i * L::kLdV + c0 + c + 1]);
                    uint32_t su[3], sx[3], sy[3];
                    split(in ? be * e.x : 0.f, in ? be * e.y : 0.f, su);
                    split(-be * ga * r.x, -be * ga * r.y, sx);
                    split(in ? p.scale * ga * y0 : 0.f, in ? p.scale * ga * y1 : 0.f, sy);
#pragma unroll
                    for (int x = 0; x < 3; ++x) {
                        const int at = (x * kC + i) * L::kTv + c0 + c;
                        *reinterpret_cast<uint32_t*>(ut + at) = su[x];
                        *reinterpret_cast<uint32_t*>(xt + at) = sx[x];
                        *reinterpret_cast<uint32_t*>(yt + at) = sy[x];
                    }
                }
                __syncwarp();
                // this slice's share of W = dO U^T and dL = -dR U^T
                uint32_t uu[3][4], oa[NT][4], ra[3][4];
#pragma unroll
                for (int x = 0; x < 3; ++x) load_rows(uu[x], Rows{ut + x * kC * L::kTv, L::kTv}, c0, lane);
#pragma unroll
                for (int x = 0; x < NT; ++x) load_rows(oa[x], Rows{ot + x * kC * L::kTv, L::kTv}, c0, lane);
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    const float2 r = *reinterpret_cast<const float2*>(&ws.r[row + z % 2 * 8][quad * 2 + z / 2 * 8]);
                    uint32_t tmp[3];
                    split(-r.x, -r.y, tmp);
#pragma unroll
                    for (int x = 0; x < 3; ++x) ra[x][z] = tmp[x];
                }
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t ub[3][2];
#pragma unroll
                    for (int x = 0; x < 3; ++x) ub[x][0] = uu[x][c], ub[x][1] = uu[x][c + 2];
                    Acc w, dl;
                    w.zero(), dl.zero();
                    mma_terms<3>(w, oa, ub);
                    mma_terms<3>(dl, ra, ub);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        *reinterpret_cast<float2*>(&sh.part[warp][0][row + half * 8][c * 8 + quad * 2]) = make_float2(w.v[half * 2], w.v[half * 2 + 1]);
                        *reinterpret_cast<float2*>(&sh.part[warp][1][row + half * 8][c * 8 + quad * 2]) = make_float2(dl.v[half * 2], dl.v[half * 2 + 1]);
                    }
                }
            }
            __syncthreads();
            for (int e = threadIdx.x; e < kC * kC; e += blockDim.x) {
                const int i = e / kC, j = e % kC;
                float w = 0.f, dl = 0.f;
#pragma unroll
                for (int x = 0; x < L::kWarpsV; ++x) w += sh.part[x][0][i][j], dl += sh.part[x][1][i][j];
                const bool in = within(i, r0, r1) && within(j, r0, r1);
                const float d = ws.w.d[i][j];
                const float da = in && i >= j ? p.scale * d * w : 0.f, dp = in && i > j ? ws.w.beta[i] * d * dl : 0.f;
                sh.da[i][j] = da;
                sh.dp[i][j] = dp;
                sh.ee[i][j] = i > j ? da * sh.qk[i][j] + dp * sh.kk[i][j] : 0.f;
            }
            Acc dq[2], dk[2], dku[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) dq[c].zero(), dk[c].zero(), dku[c].zero();
            if (has_k) {
                const float* s0 = p.checkpoints + (seq * blocks + b) * p.dk * p.dv;
                float dot = 0.f;
                const int k0 = c0 + row, k1 = k0 + 8;
                const bool in0 = !fresh && k0 < p.dk, in1 = !fresh && k1 < p.dk;
#pragma unroll
                for (int st = 0; st < DV / 16; ++st) {
                    uint32_t oa[NT][4], ua[3][4], xa[3][4];
#pragma unroll
                    for (int x = 0; x < NT; ++x) load_rows(oa[x], Rows{ot + x * kC * L::kTv, L::kTv}, st * 16, lane);
#pragma unroll
                    for (int x = 0; x < 3; ++x) {
                        load_rows(ua[x], Rows{ut + x * kC * L::kTv, L::kTv}, st * 16, lane);
                        load_rows(xa[x], Rows{xt + x * kC * L::kTv, L::kTv}, st * 16, lane);
                    }
                    Acc s[2];
#pragma unroll
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int c = st * 16 + x * 8 + quad * 2 + e;
                            s[x].v[e] = in0 && c < p.dv ? s0[(int64_t)k0 * p.dv + c] : 0.f;
                            s[x].v[2 + e] = in1 && c < p.dv ? s0[(int64_t)k1 * p.dv + c] : 0.f;
                        }
#pragma unroll
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int e = 0; e < 4; ++e) dot = fmaf(s[x].v[e], ds[2 * st + x].v[e], dot);
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t sb[3][2], db[3][2], lo[3], hi[3];
                        split(s[0].v[2 * c], s[0].v[2 * c + 1], lo);
                        split(s[1].v[2 * c], s[1].v[2 * c + 1], hi);
#pragma unroll
                        for (int x = 0; x < 3; ++x) sb[x][0] = lo[x], sb[x][1] = hi[x];
                        split(ds[2 * st].v[2 * c], ds[2 * st].v[2 * c + 1], lo);
                        split(ds[2 * st + 1].v[2 * c], ds[2 * st + 1].v[2 * c + 1], hi);
#pragma unroll
                        for (int x = 0; x < 3; ++x) db[x][0] = lo[x], db[x][1] = hi[x];
                        mma_terms<3>(dq[c], oa, sb);
                        mma_terms<3>(dk[c], xa, sb);
                        mma_terms<3>(dku[c], ua, db);
                    }
                }
                // the decays' gradients need q.dq and k.dk of these parts alone
                const float g0 = p.scale * ws.w.gamma[row], g1 = p.scale * ws.w.gamma[row + 8], e0 = ws.w.eta[row], e1 = ws.w.eta[row + 8];
                float di[2] = {0.f, 0.f}, dj[2] = {0.f, 0.f};
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int half = e / 2, at = (row + half * 8) * L::kLdK + c0 + c * 8 + quad * 2 + e % 2;
                        dq[c].v[e] *= half ? g1 : g0;
                        dku[c].v[e] *= half ? e1 : e0;
                        const float kv = to_f32(rk[at]);
                        di[half] += to_f32(rq[at]) * dq[c].v[e] + kv * dk[c].v[e];
                        dj[half] += kv * dku[c].v[e];
                    }
#pragma unroll
                for (int w = 1; w < 4; w *= 2) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        di[half] += __shfl_xor_sync(0xffffffffu, di[half], w);
                        dj[half] += __shfl_xor_sync(0xffffffffu, dj[half], w);
                    }
                }
#pragma unroll
                for (int w = 1; w < 32; w *= 2) dot += __shfl_xor_sync(0xffffffffu, dot, w);
                if (quad == 0) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        sh.dot_i[warp][row + half * 8] = di[half];
                        sh.dot_j[warp][row + half * 8] = dj[half];
                    }
                }
                if (lane == 0) sh.dot_s[warp] = ws.w.keep * dot;
            }
            __syncthreads();
            if (has_k) {
                uint32_t da[3][4], dat[3][4], dp[3][4], kb[NT][4], qb[NT][4];
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    const int x = row + z % 2 * 8, y = quad * 2 + z / 2 * 8;
                    uint32_t tmp[3];
                    split(sh.da[x][y], sh.da[x][y + 1], tmp);
#pragma unroll
                    for (int i = 0; i < 3; ++i) da[i][z] = tmp[i];
                    split(sh.da[y][x], sh.da[y + 1][x], tmp);
#pragma unroll
                    for (int i = 0; i < 3; ++i) dat[i][z] = tmp[i];
                    split(sh.dp[x][y] + sh.dp[y][x], sh.dp[x][y + 1] + sh.dp[y + 1][x], tmp);
#pragma unroll
                    for (int i = 0; i < 3; ++i) dp[i][z] = tmp[i];
                }
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    load_tokens(kb[x], Rows{kt + x * kC * L::kTk, L::kTk}, c0, lane);
                    load_tokens(qb[x], Rows{qt + x * kC * L::kTk, L::kTk}, c0, lane);
                }
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t k2[NT][2], q2[NT][2];
#pragma unroll
                    for (int x = 0; x < NT; ++x) {
                        k2[x][0] = kb[x][2 * c] & m0, k2[x][1] = kb[x][2 * c + 1] & m1;
                        q2[x][0] = qb[x][2 * c] & m0, q2[x][1] = qb[x][2 * c + 1] & m1;
                    }
                    mma_terms<3>(dq[c], da, k2);
#pragma unroll
                    for (int e = 0; e < 4; ++e) dk[c].v[e] += dku[c].v[e];
                    mma_terms<3>(dk[c], dat, q2);
                    mma_terms<3>(dk[c], dp, k2);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int i = row + half * 8, col = c0 + c * 8 + quad * 2;
                        if (within(i, r0, r1)) {
                            const int64_t at = ((b * kC + i) * out_t + out_0) * p.dk + col;
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                if (col + e < p.dk) {
                                    static_cast<T*>(p.dq)[at + e] = from_f32<T>(dq[c].v[half * 2 + e]);
                                    static_cast<T*>(p.dk_out)[at + e] = from_f32<T>(dk[c].v[half * 2 + e]);
                                }
                        }
                    }
                }
            }
            if (warp == 0) {
                // column j's sums of E from the last row up, then row l's first l columns
                float tail = 0.f;
                if (lane < 16)
                    for (int i = kC - 1; i >= 0; --i) {
                        tail += sh.ee[i][lane];
                        sh.ee[i][lane] = tail;
                    }
                __syncwarp();
                if (within(lane, r0, r1)) {
                    float dg = 0.f;
                    for (int j = 0; j < lane; ++j) dg += sh.ee[lane][j];
                    for (int x = 0; x < L::kWarpsK; ++x) {
                        for (int i = lane; i < r1; ++i) dg += sh.dot_i[x][i];
                        for (int j = r0; j < lane; ++j) dg += sh.dot_j[x][j];
                        dg += sh.dot_s[x];
                    }
                    float dbeta = 0.f;
                    for (int x = 0; x < L::kWarpsV; ++x) dbeta += sh.dbeta[x][lane];
                    const int64_t at = (b * kC + lane) * out_t + out_0;
                    p.dg[at] = dg;
                    p.dbeta[at] = dbeta;
                }
            }
            if (fresh) {  // the state before was dropped
#pragma unroll
                for (int i = 0; i < DV / 8; ++i) ds[i].zero();
#pragma unroll
                for (int i = 0; i < DK / 8; ++i) dst[i].zero();
            } else {
                const float keep = ws.w.keep;
                if (has_k) {
                    uint32_t qa[NT][4], ka[NT][4];  // rows = dk, k = tokens
#pragma unroll
                    for (int x = 0; x < NT; ++x) {
                        load_columns(qa[x], Rows{qt + x * kC * L::kTk, L::kTk}, c0, lane);
                        load_columns(ka[x], Rows{kt + x * kC * L::kTk, L::kTk}, c0, lane);
#pragma unroll
                        for (int z = 0; z < 4; ++z) {
                            qa[x][z] &= z < 2 ? m0 : m1;
                            ka[x][z] &= z < 2 ? m0 : m1;
                        }
                    }
#pragma unroll
                    for (int st = 0; st < DV / 16; ++st) {
                        uint32_t xb[3][4], yb[3][4];
#pragma unroll
                        for (int x = 0; x < 3; ++x) {
                            load_tokens(xb[x], Rows{xt + x * kC * L::kTv, L::kTv}, st * 16, lane);
                            load_tokens(yb[x], Rows{yt + x * kC * L::kTv, L::kTv}, st * 16, lane);
                        }
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            Acc& acc = ds[2 * st + c];
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc.v[e] *= keep;
                            uint32_t x2[3][2], y2[3][2];
#pragma unroll
                            for (int x = 0; x < 3; ++x) {
                                x2[x][0] = xb[x][2 * c], x2[x][1] = xb[x][2 * c + 1];
                                y2[x][0] = yb[x][2 * c], y2[x][1] = yb[x][2 * c + 1];
                            }
                            mma_terms<3>(acc, qa, y2);
                            mma_terms<3>(acc, ka, x2);
                        }
                    }
                }
                if (has_v) {
                    uint32_t xa[3][4], ya[3][4];  // rows = dv, k = tokens
#pragma unroll
                    for (int x = 0; x < 3; ++x) {
                        load_columns(xa[x], Rows{xt + x * kC * L::kTv, L::kTv}, c0, lane);
                        load_columns(ya[x], Rows{yt + x * kC * L::kTv, L::kTv}, c0, lane);
                    }
#pragma unroll
                    for (int st = 0; st < DK / 16; ++st) {
                        uint32_t kb[NT][4], qb[NT][4];
#pragma unroll
                        for (int x = 0; x < NT; ++x) {
                            load_tokens(kb[x], Rows{kt + x * kC * L::kTk, L::kTk}, st * 16, lane);
                            load_tokens(qb[x], Rows{qt + x * kC * L::kTk, L::kTk}, st * 16, lane);
                        }
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            Acc& acc = dst[2 * st + c];
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc.v[e] *= keep;
                            uint32_t k2[NT][2], q2[NT][2];
#pragma unroll
                            for (int x = 0; x < NT; ++x) {
                                k2[x][0] = kb[x][2 * c] & m0, k2[x][1] = kb[x][2 * c + 1] & m1;
                                q2[x][0] = qb[x][2 * c] & m0, q2[x][1] = qb[x][2 * c + 1] & m1;
                            }
                            mma_terms<3>(acc, ya, q2);
                            mma_terms<3>(acc, xa, k2);
                        }
                    }
                }
            }
            __syncthreads();  // U, X, Y and the sums are free for the next chunk
            r1 = r0;
        }
    }
    if (p.dstate && has_k) {
        float* to = p.dstate + seq * p.dk * p.dv;
#pragma unroll
        for (int i = 0; i < DV / 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int kk = c0 + row + e / 2 * 8, c = i * 8 + quad * 2 + e % 2;
                if (kk < p.dk && c < p.dv) to[(int64_t)kk * p.dv + c] = ds[i].v[e];
            }
    }
}

// ------------------------------------------------------------------- host

// A (t, n, h, d) tensor for Fetch.  Dimensions of one element have no stride to speak of.
template <class T>
int map_rows(CUtensorMap* map, const void* base, const Strides& s, const Scan& p, int d) {
    const uint64_t dims[4] = {(uint64_t)d, (uint64_t)p.h, (uint64_t)p.n, (uint64_t)p.t};
    auto bytes = [](int64_t count, int64_t stride) { return count > 1 ? (uint64_t)stride * sizeof(T) : 16u; };
    const uint64_t strides[3] = {bytes(p.h, s.h), bytes(p.n, s.n), bytes(p.t, s.t)};
    const uint32_t box[4] = {128 / sizeof(T), 1, 1, kC};
    const CUtensorMapDataType type = sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : Terms<T>::n == 1 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    return encode_map(map, type, 4, base, dims, strides, box);
}

template <class T, int DK>
int launch_forward_dk(const Scan& p, cudaStream_t st) {
    using L = ForwardSmem<T, DK>;
    auto* kernel = scan_forward_kernel<T, DK>;
    if (int rc = cuda_status(allow_smem(kernel, (int)L::kBytes), "delta_scan")) return rc;
    const dim3 grid(static_cast<unsigned>(p.n * p.h), (p.dv + L::kWidth - 1) / L::kWidth);
    CUtensorMap map_k{}, map_q{}, map_v{};
    if (p.aligned && p.t) {
        if (int rc = map_rows<T>(&map_k, p.k, p.sk, p, p.dk)) return rc;
        if (int rc = map_rows<T>(&map_q, p.q, p.sq, p, p.dk)) return rc;
        if (int rc = map_rows<T>(&map_v, p.v, p.sv, p, p.dv)) return rc;
    }
    kernel<<<grid, (kForwardWarps + 1) * 32, L::kBytes, st>>>(p, map_k, map_q, map_v);
    return cuda_status(cudaGetLastError(), "delta_scan");
}

template <class T, int DK, int DV>
int launch_backward_dk_dv(const Scan& p, cudaStream_t st) {
    using L = BackwardSmem<T, DK, DV>;
    auto* kernel = scan_backward_kernel<T, DK, DV>;
    if (int rc = cuda_status(allow_smem(kernel, (int)L::kBytes), "delta_scan_backward")) return rc;
    kernel<<<static_cast<unsigned>(p.n * p.h), L::kWarps * 32, L::kBytes, st>>>(p);
    return cuda_status(cudaGetLastError(), "delta_scan_backward");
}

template <class T, int DK>
int launch_backward_dk(const Scan& p, cudaStream_t st) {
    if (p.dv <= 32) return launch_backward_dk_dv<T, DK, 32>(p, st);
    if (p.dv <= 64) return launch_backward_dk_dv<T, DK, 64>(p, st);
    return launch_backward_dk_dv<T, DK, 128>(p, st);
}

// Head sizes are padded with zeros to the next of 32, 64 and 128.
template <class T>
int launch_forward(const Scan& p, cudaStream_t st) {
    if (p.dk <= 32) return launch_forward_dk<T, 32>(p, st);
    if (p.dk <= 64) return launch_forward_dk<T, 64>(p, st);
    return launch_forward_dk<T, 128>(p, st);
}
template <class T>
int launch_backward(const Scan& p, cudaStream_t st) {
    if (p.dk <= 32) return launch_backward_dk<T, 32>(p, st);
    if (p.dk <= 64) return launch_backward_dk<T, 64>(p, st);
    return launch_backward_dk<T, 128>(p, st);
}

extern template int launch_forward<__nv_bfloat16>(const Scan&, cudaStream_t);
extern template int launch_forward<__half>(const Scan&, cudaStream_t);
extern template int launch_forward<float>(const Scan&, cudaStream_t);
extern template int launch_backward<__nv_bfloat16>(const Scan&, cudaStream_t);
extern template int launch_backward<__half>(const Scan&, cudaStream_t);
extern template int launch_backward<float>(const Scan&, cudaStream_t);

}  // namespace delta
}  // namespace ops
}  // namespace nesle
