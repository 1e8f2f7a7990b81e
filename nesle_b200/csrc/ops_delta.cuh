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

#include <algorithm>
#include <type_traits>

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
    float* errors;       // as error_at() says, NULL where no gradient is wanted
    float* checkpoints;  // [n][h][ceil(t / 16)][dk][dv], the state before each chunk
    const void* d_o;     // contiguous
    const float* d_final;
    void *dq, *dk_out, *dv_out;
    float *dg, *dbeta, *dstate;
    int segments;        // 1, or what a sequence is cut into (launch_split)
    int64_t per;         // blocks of 16 tokens of a segment
    float* ends;         // [n][h][segments - 1]: the end of a segment (dk x dv), and what it makes of a state (dk x dk)
    int* restarts;       // [n][h][segments - 1]: an episode starts in the segment
    unsigned int* stalls;
    int device;
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
// Two fp32 in one instruction (fma.rn.f32x2): a * b + c.
__device__ __forceinline__ void fma2(float& x, float& y, float a0, float a1, float b0, float b1) {
    asm("{\n\t.reg .b64 A, B, C;\n\tmov.b64 A, {%2, %3};\n\tmov.b64 B, {%4, %5};\n\tmov.b64 C, {%0, %1};\n\t"
        "fma.rn.f32x2 C, A, B, C;\n\tmov.b64 {%0, %1}, C;\n\t}"
        : "+f"(x), "+f"(y)
        : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
__device__ __forceinline__ void mul2(float& x, float& y, float b) {
    asm("{\n\t.reg .b64 B, C;\n\tmov.b64 B, {%2, %2};\n\tmov.b64 C, {%0, %1};\n\tmul.rn.f32x2 C, C, B;\n\tmov.b64 {%0, %1}, C;\n\t}"
        : "+f"(x), "+f"(y)
        : "f"(b));
}

// x, y as sums of N bf16 each, packed pairwise.  kPaired takes both remainders in one instruction, which saves two of
// eleven and wants its registers in pairs: 2 to 4% of the forward pass's time, and 11% slower in the backward pass,
// whose registers are full.
template <bool kPaired = false, int N>
__device__ __forceinline__ void split(float x, float y, uint32_t (&out)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        out[i] = pack(x, y);
        if (i + 1 == N) break;
        const float hx = __uint_as_float(out[i] << 16), hy = __uint_as_float(out[i] & 0xFFFF0000u);
        if constexpr (kPaired)
            fma2(x, y, hx, hy, -1.f, -1.f);
        else
            x -= hx, y -= hy;
    }
}

struct Acc {  // 16 x 8 of a result: rows lane/4 and lane/4 + 8, columns 2 (lane%4) and the next
    float v[4];
    __device__ __forceinline__ void zero() { v[0] = v[1] = v[2] = v[3] = 0.f; }
};

__device__ __forceinline__ void mma(Acc& c, const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c.v[0]), "+f"(c.v[1]), "+f"(c.v[2]), "+f"(c.v[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

// The pairs of terms (i, j), i < NA, j < NB, i + j < kMost, the smallest products first.
template <int kMost, int NA, int NB>
struct Pairs {
    __host__ __device__ static constexpr int count() {
        int n = 0;
        for (int i = 0; i < NA; ++i)
            for (int j = 0; j < NB; ++j) n += i + j < kMost;
        return n;
    }
    __host__ __device__ static constexpr int at(int k) {  // 8 i + j of the k-th
        for (int s = kMost - 1; s >= 0; --s)
            for (int i = 0; i < NA; ++i)
                if (s - i >= 0 && s - i < NB && k-- == 0) return 8 * i + s - i;
        return 0;
    }
    static constexpr int n = count();
};

// One product after another into one accumulator waits for it 30-odd clocks each time, and a product takes 8 to issue: so
// products go round four accumulators or so.  Each call of a step adds pair k of one product to the accumulators of two
// neighbouring column tiles.
template <class P, int k, int NA, int NB>
__device__ __forceinline__ void step2(Acc& c0, Acc& c1, const uint32_t (&a)[NA][4], const uint32_t (&b0)[NB][2], const uint32_t (&b1)[NB][2]) {
    if constexpr (k < P::n) {
        constexpr int i = P::at(k) / 8, j = P::at(k) % 8;
        mma(c0, a[i], b0[j]);
        mma(c1, a[i], b1[j]);
    }
}
template <int k, int n, class F>
__device__ __forceinline__ void each_step(F&& f) {
    if constexpr (k < n) {
        f(std::integral_constant<int, k>{});
        each_step<k + 1, n>(f);
    }
}
// c += A b for two column tiles.
template <int kMost, int NA, int NB>
__device__ __forceinline__ void mma2(Acc (&c)[2], const uint32_t (&a)[NA][4], const uint32_t (&b)[2][NB][2]) {
    using P = Pairs<kMost, NA, NB>;
    each_step<0, P::n>([&](auto k) { step2<P, k.value>(c[0], c[1], a, b[0], b[1]); });
}
// Two products into accumulators of their own, in turn.
template <int kMostX, int kMostY, int NXA, int NXB, int NYA, int NYB>
__device__ __forceinline__ void mma2_zip(Acc (&x)[2], const uint32_t (&xa)[NXA][4], const uint32_t (&xb)[2][NXB][2], Acc (&y)[2],
                                         const uint32_t (&ya)[NYA][4], const uint32_t (&yb)[2][NYB][2]) {
    using X = Pairs<kMostX, NXA, NXB>;
    using Y = Pairs<kMostY, NYA, NYB>;
    each_step<0, (X::n > Y::n ? X::n : Y::n)>([&](auto k) {
        step2<X, k.value>(x[0], x[1], xa, xb[0], xb[1]);
        step2<Y, k.value>(y[0], y[1], ya, yb[0], yb[1]);
    });
}
// The same product over two pairs of accumulators, which are then added: for a product that stands alone.
template <int kMost, int NA, int NB>
__device__ __forceinline__ void mma2_split(Acc (&c)[2], const uint32_t (&a)[NA][4], const uint32_t (&b)[2][NB][2]) {
    using P = Pairs<kMost, NA, NB>;
    Acc d[2];
    d[0].zero(), d[1].zero();
    each_step<0, (P::n + 1) / 2>([&](auto k) {
        step2<P, 2 * k.value>(d[0], d[1], a, b[0], b[1]);
        step2<P, 2 * k.value + 1>(c[0], c[1], a, b[0], b[1]);
    });
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) c[i].v[e] += d[i].v[e];
}

// Registers of load_rows as a B operand whose columns are the tile's rows, of load_tokens as one whose columns are the
// tile's columns; tokens outside the chunk masked.
template <int N>
__device__ __forceinline__ void as_rows(uint32_t (&b)[2][N][2], const uint32_t (&r)[N][4]) {
#pragma unroll
    for (int x = 0; x < N; ++x)
#pragma unroll
        for (int c = 0; c < 2; ++c) b[c][x][0] = r[x][c], b[c][x][1] = r[x][c + 2];
}
template <int N>
__device__ __forceinline__ void as_columns(uint32_t (&b)[2][N][2], const uint32_t (&r)[N][4], uint32_t m0 = ~0u, uint32_t m1 = ~0u) {
#pragma unroll
    for (int x = 0; x < N; ++x)
#pragma unroll
        for (int c = 0; c < 2; ++c) b[c][x][0] = r[x][2 * c] & m0, b[c][x][1] = r[x][2 * c + 1] & m1;
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
//
// 1,024 envs x 4 heads x 128 tokens of 64 x 64, keeping states and errors for
// the gradients: 298 us, 3.6 TB/s, 314 with an episode's end in 200 tokens (an end
// makes two chunks of one).  No unit is full (44% of the issue slots at 13 warps an
// SM): a chunk is a chain of dependent products, and that many warps hide no more
// of it.  4 envs x 4 heads x 4,096 tokens of 128 x 128: 249 us in 6 segments
// (count_segments), 523 in one: 2.05 us a chunk where a block has an SM to itself, a
// chain of products as long as the helper's work.  The look for tokens that are not
// finite costs nothing there, 1 to 2% with 16 and 32 bits by terms, 4% with ragged values.

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

// Whether fetched tiles hold a NaN or an infinity: 0 * x adds up to zero over all else.
template <class T>
struct NotFinite {
    using Two = std::conditional_t<sizeof(T) == 4, float, std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>>;
    Two sum[4] = {zero(), zero(), zero(), zero()};
    static __device__ __forceinline__ Two zero() {
        const uint32_t bits = 0;
        return reinterpret_cast<const Two&>(bits);
    }
    template <int D>
    __device__ __forceinline__ void add(const T* tile, int lane) {
        const uint4* chunks = reinterpret_cast<const uint4*>(tile);
#pragma unroll
        for (int i = 0; i < Fetch<T, D>::kPanels * 4; ++i) {
            const uint4 x = chunks[i * 32 + lane];
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (sizeof(T) == 4)
                    sum[i % 4] = fmaf(__uint_as_float(w[j]), 0.f, sum[i % 4]);
                else
                    sum[i % 4] = __hfma2(reinterpret_cast<const Two&>(w[j]), zero(), sum[i % 4]);
            }
        }
    }
    static __device__ __forceinline__ float joined(Two x) {
        if constexpr (sizeof(T) == 4)
            return x;
        else
            return to_f32(x.x) + to_f32(x.y);
    }
    // Of the warp's lanes; `more` is a lane's own sum of this kind.
    __device__ __forceinline__ bool any(float more) const {
        more += joined((sum[0] + sum[1]) + (sum[2] + sum[3]));
        return __any_sync(0xffffffffu, more != more);
    }
    // Which tokens of a tile, bit i for token i: a token's chunks are 8 lanes', those of four tokens a warp's.  Rare, and
    // out of line for the registers of all else.
    template <int D>
    static __device__ __noinline__ uint32_t tokens(const T* tile, int lane) {
        uint32_t out = 0;
#pragma unroll 1
        for (int i = 0; i < Fetch<T, D>::kPanels * 4; ++i) {
            const uint4 x = reinterpret_cast<const uint4*>(tile)[i * 32 + lane];
            const T* v = reinterpret_cast<const T*>(&x);
            float f = 0.f;
#pragma unroll
            for (int j = 0; j < 16 / (int)sizeof(T); ++j) f = fmaf(to_f32(v[j]), 0.f, f);
            const uint32_t lanes = __ballot_sync(0xffffffffu, f != f);
#pragma unroll
            for (int g = 0; g < 4; ++g) out |= (lanes >> 8 * g & 0xFF ? 1u : 0u) << (i % 4 * 4 + g);
        }
        return out;
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

// Errors are kept as the accumulators hold them: for every 16 tokens and 16 columns two tiles, of 8 tokens each, a float4 a
// lane.  The index of a lane's float4.
__device__ __forceinline__ int64_t error_at(int64_t block, int slices, int slice, int tile, int lane) {
    return ((block * slices + slice) * 2 + tile) * 32 + lane;
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

template <class T, int DK, bool kRegular, bool kEnds>
__global__ void __launch_bounds__((kForwardWarps + 1) * 32, DK == 128 ? 2 : 3)
    scan_forward_kernel(const Scan p, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_q,
                        const __grid_constant__ CUtensorMap map_v) {
    using L = ForwardSmem<T, DK>;
    const bool aligned = kRegular || p.aligned;
    const int dk = kRegular ? DK : p.dk, dv = p.dv;
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
    const int value_blocks = (dv + L::kWidth - 1) / L::kWidth;
    const bool unit = kEnds && (int)blockIdx.y >= value_blocks;  // from a unit matrix, with no values: what the segment makes of a state
    const int wide = unit ? dk : dv, first_col = ((int)blockIdx.y - (unit ? value_blocks : 0)) * L::kWidth;
    const int cols = kRegular ? L::kWidth : min(L::kWidth, wide - first_col);
    const int segment = (int)blockIdx.z;
    if (unit && segment == 0) return;  // the state before the first token is known
    const int64_t all = (p.t + kC - 1) / kC, b0 = segment * p.per;  // blocks are counted from the segment's first
    const int64_t blocks = all - b0 < p.per ? all - b0 : p.per, t0 = b0 * kC;
    const int64_t slot = seq * (p.segments - 1) + segment;
    auto end_of = [&](int64_t at) { return p.ends + at * dk * (dk + dv); };
    auto raw_tile = [&](int64_t b) { return reinterpret_cast<T*>(smem + b % L::kBuffers * L::kRaw); };
    // term x of K (which = 0) or Q (1) of a block as an operand
    auto operand = [&](int64_t b, int which, int x) {
        if constexpr (L::kInPlace)
            return Panels{reinterpret_cast<const __nv_bfloat16*>(raw_tile(b)) + which * L::kTileK};
        else
            return Rows{terms + ((b & 1) * 2 * NT + which * NT + x) * kC * L::kLdTerm, L::kLdTerm};
    };
    if (!aligned)
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
            const int64_t t = t0 + b * kC;
            const int count = (int)(p.t - t < kC ? p.t - t : kC);
            if (aligned && lane == 0) tc::mbar_expect_tx(bar, (uint32_t)((kEnds ? L::kTileK : 2 * L::kTileK) + (unit ? 0 : L::kTileV)) * sizeof(T));
            Fetch<T, DK>::run(to, &map_k, k, p.sk.t, n, h, 0, t, count, dk, aligned, bar, lane);
            if constexpr (!kEnds) Fetch<T, DK>::run(to + L::kTileK, &map_q, q, p.sq.t, n, h, 0, t, count, dk, aligned, bar, lane);
            if (!unit) Fetch<T, L::kWidth>::run(to + 2 * L::kTileK, &map_v, v, p.sv.t, n, h, first_col, t, count, cols, aligned, bar, lane);
        };
        fetch(0);
        fetch(1);
        const GatePointers get_gates(p, n, h, lane);
        Gates gates{}, next = get_gates.load(t0, p.t, lane);
        float decay = 1.f;
        uint32_t starts = 0;  // bit i: token i starts an episode; bit 16 + i: it begins a chunk for another reason
        int64_t b = -1;
        int r0 = 0, count = 0, restarts = 0;
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
                count = (int)(p.t - t0 - b * kC < kC ? p.t - t0 - b * kC : kC);
                gates = next;
                next = get_gates.load(t0 + (b + 1) * kC, p.t, lane);
                decay = gates.decay();
                starts = gates.starts();
                if (aligned && !tc::mbar_wait_warp(&arrived[b % L::kBuffers], b / L::kBuffers & 1)) {
                    for (int64_t x = b; x < blocks && x < b + 2; ++x) tc::mbar_drain(&arrived[x % L::kBuffers], x / L::kBuffers & 1);
                    if (lane == 0) {
                        atomicAdd(p.stalls, 1u);
                        ch.block = -1;
                    }
                    __syncthreads();
                    break;
                }
                __syncwarp();
                fetch(b + 2);
                if constexpr (!kEnds) {
                    // A token whose key, value or gates are not finite begins a chunk: the products of a chunk multiply it by
                    // the zeros that stand for "later" too, and would spoil the tokens before it.
                    const T *tk = raw_tile(b), *tv = tk + 2 * L::kTileK;
                    const float gate = (decay + gates.beta) * 0.f;
                    NotFinite<T> look;
                    look.template add<DK>(tk, lane);
                    look.template add<L::kWidth>(tv, lane);
                    if (look.any(gate)) {
                        const uint32_t bad = look.template tokens<DK>(tk, lane) | look.template tokens<L::kWidth>(tv, lane) |
                                             __ballot_sync(0xffffffffu, gate != gate);
                        starts |= (bad & ((1u << count) - 1)) << 16;
                    }
                }
                if constexpr (!L::kInPlace) {
                    __nv_bfloat16* to = terms + (b & 1) * 2 * NT * kC * L::kLdTerm;
                    to_terms_warp<T, DK>(to, L::kLdTerm, raw_tile(b), lane);
                    if constexpr (!kEnds) to_terms_warp<T, DK>(to + NT * kC * L::kLdTerm, L::kLdTerm, raw_tile(b) + L::kTileK, lane);
                    __syncwarp();
                }
            }
            const bool fresh = starts >> r0 & 1;
            restarts |= fresh;
            const uint32_t later = (starts | starts >> 16) & ~((2u << r0) - 1);
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
                    if constexpr (!kEnds) load_rows(qa[x], operand(b, 1, x), st * 16, lane);
                }
                uint32_t kb[2][NT][2];
                as_rows(kb, ka);
                if constexpr (kEnds)
                    mma2<3>(kk, ka, kb);
                else
                    mma2_zip<3, NO>(kk, ka, kb, qk, qa, kb);
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
                    if constexpr (kEnds) continue;
                    uint32_t s[NO];
                    split<true>(in0 && i >= j ? d.x * qk[c].v[half * 2] : 0.f, in1 && i >= j + 1 ? d.y * qk[c].v[half * 2 + 1] : 0.f, s);
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
        if (kEnds && lane == 0 && blockIdx.y == 0) p.restarts[slot] = restarts;
        return;
    }

    const int v0 = warp * 16, c0 = first_col + v0;  // this warp's columns of the state
    const bool whole = kEnds ? dk == DK && c0 + 16 <= wide : kRegular || (dk == DK && c0 + 16 <= dv);
    float* state_tile = out_tiles + warp * L::kOut / 4;
    __nv_bfloat16* out_tile = reinterpret_cast<__nv_bfloat16*>(state_tile);
    const bool s_aligned = kRegular || (dv % 4 == 0 && (kEnds ? dk % 4 == 0 && reinterpret_cast<uintptr_t>(p.ends) % 16 == 0
                                                              : reinterpret_cast<uintptr_t>(p.checkpoints) % 16 == 0 &&
                                                                    reinterpret_cast<uintptr_t>(p.final_state) % 16 == 0));
    const bool o_aligned = sizeof(T) == 2 && (kRegular || (dv % 8 == 0 && reinterpret_cast<uintptr_t>(p.o) % 16 == 0));
    Acc s[kTiles];  // S^T: rows = columns c0.. of the state, columns = dk
    // where this thread's values of a (dk, dv) matrix lie: value e of tile i at i * 8 * dv + at(e)
    auto each_state = [&](auto&& f) {
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int kk = i * 8 + quad * 2 + e % 2, c = c0 + row + e / 2 * 8;
                f(s[i].v[e], kk * wide + c, whole || (kk < dk && c < wide));
            }
    };
    {
        const float* s0 = segment ? (kEnds ? nullptr : end_of(slot - 1)) : p.state ? p.state + seq * dk * dv : nullptr;
        if (unit)
            each_state([&](float& x, int at, bool in) { x = in && at % (dk + 1) == 0 ? 1.f : 0.f; });
        else
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
            float4* out = reinterpret_cast<float4*>(to + (lane / 4) * wide + c0 + lane % 4 * 4);
#pragma unroll
            for (int i = 0; i < DK / 8; ++i)
                __stcs(out + i * 2 * wide, *reinterpret_cast<const float4*>(state_tile + (i * 8 + lane / 4) * L::kLdS + lane % 4 * 4));
            __syncwarp();
        } else {
            each_state([&](float& x, int at, bool in) {
                if (in) to[at] = x;
            });
        }
    };
    const int slices = (dv + 15) / 16;
    const int64_t step_t = p.n * p.h * dv, first = (n * p.h + h) * dv + c0;
    for (int turn = 0;; ++turn) {
        __syncthreads();
        const Chunk& ch = chunks[turn & 1];
        const int64_t b = ch.block;
        if (b < 0) break;
        if (aligned) tc::mbar_see(&arrived[b % L::kBuffers], b / L::kBuffers & 1);  // the helper waited for them
        const int r0 = ch.r0, r1 = ch.r1;
        if (!kEnds && p.checkpoints && r0 == 0) put_state(p.checkpoints + (seq * all + b0 + b) * dk * dv);
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
                split<true>(t.v[z % 2 * 2], t.v[z % 2 * 2 + 1], tmp);
#pragma unroll
                for (int x = 0; x < 3; ++x) sa[x][z] = tmp[x];
            }
            uint32_t ka[NT][4], qa[NT][4];
#pragma unroll
            for (int x = 0; x < NT; ++x) {
                load_rows(ka[x], operand(b, 0, x), st * 16, lane);
                if constexpr (!kEnds) load_rows(qa[x], operand(b, 1, x), st * 16, lane);
            }
            uint32_t kb[2][NT][2], qb[2][NT][2];
            as_rows(kb, ka);
            if constexpr (kEnds) {
                mma2<3>(ks, sa, kb);
            } else {
                as_rows(qb, qa);
                mma2_zip<3, NO>(ks, sa, kb, qs, sa, qb);
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
                    if (unit) x0 = x1 = 0.f;
                    uint32_t tmp[3];
                    split<true>(in0 ? fmaf(-ga.x, ks[c].v[half * 2], x0) : 0.f, in1 ? fmaf(-ga.y, ks[c].v[half * 2 + 1], x1) : 0.f, tmp);
#pragma unroll
                    for (int x = 0; x < 3; ++x) ra[x][c * 2 + half] = tmp[x];
                }
                qs[c].v[0] *= ga.x, qs[c].v[1] *= ga.y, qs[c].v[2] *= ga.x, qs[c].v[3] *= ga.y;
            }
        }
        uint32_t uo[NO][4], ue[3][4];  // U^T and (eta U)^T
        {
            uint32_t mb[3][4], bb[2][3][2];
            load_operand(mb, ch.m, lane);
            as_rows(bb, mb);
            Acc ee[2];
            ee[0].zero(), ee[1].zero();
            mma2_split<3>(ee, ra, bb);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const Acc& e = ee[c];
                const int j = c * 8 + quad * 2;
                if (!kEnds && p.errors && first_col / 16 + warp < slices) {
                    float4* to = reinterpret_cast<float4*>(p.errors) + error_at(seq * all + b0 + b, slices, first_col / 16 + warp, c, lane);
                    if (r0 == 0 && r1 == kC) {
                        __stcs(to, make_float4(e.v[0], e.v[1], e.v[2], e.v[3]));
                    } else {
#pragma unroll
                        for (int z = 0; z < 4; ++z)
                            if (within(j + z % 2, r0, r1)) reinterpret_cast<float*>(to)[z] = e.v[z];
                    }
                }
                const float2 be = *reinterpret_cast<const float2*>(&ch.beta[j]), et = *reinterpret_cast<const float2*>(&ch.eta[j]);
                const float h0 = be.x * et.x, h1 = be.y * et.y;  // rounded once more than beta e, then eta: 2^-24
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t t2[NO], t3[3];
                    if constexpr (!kEnds) split<true>(be.x * e.v[half * 2], be.y * e.v[half * 2 + 1], t2);
                    split<true>(h0 * e.v[half * 2], h1 * e.v[half * 2 + 1], t3);
#pragma unroll
                    for (int x = 0; x < NO && !kEnds; ++x) uo[x][c * 2 + half] = t2[x];
#pragma unroll
                    for (int x = 0; x < 3; ++x) ue[x][c * 2 + half] = t3[x];
                }
            }
        }
        if constexpr (!kEnds) {
            uint32_t ab[NO][4], bb[2][NO][2];
            load_operand(ab, ch.att, lane);
            as_rows(bb, ab);
            mma2_split<NO>(qs, uo, bb);
        }
        if constexpr (kEnds) {
        } else if (o_aligned && whole) {  // by a transposed tile in shared memory, 16 bytes a lane
            if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int z = 0; z < 4; ++z)
                        reinterpret_cast<T*>(out_tile)[(c * 8 + quad * 2 + z % 2) * kLdOut + row + z / 2 * 8] = from_f32<T>(p.scale * qs[c].v[z]);
                __syncwarp();
                const int i = lane / 2;
                if (within(i, r0, r1))
                    *reinterpret_cast<uint4*>(static_cast<T*>(p.o) + (t0 + b * kC + i) * step_t + first + lane % 2 * 8) =
                        *reinterpret_cast<const uint4*>(out_tile + i * kLdOut + lane % 2 * 8);
                __syncwarp();
            }
        } else {
            T* o = static_cast<T*>(p.o) + (t0 + b * kC) * step_t + first + row;
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    const int i = c * 8 + quad * 2 + z % 2;
                    if (within(i, r0, r1) && (whole || c0 + row + z / 2 * 8 < dv)) o[i * step_t + z / 2 * 8] = from_f32<T>(p.scale * qs[c].v[z]);
                }
        }
        const float keep = ch.keep;
        const uint32_t m0 = pair_mask(quad * 2, r0, r1), m1 = pair_mask(quad * 2 + 8, r0, r1);
#pragma unroll
        for (int i = 0; i < kTiles; ++i) mul2(s[i].v[0], s[i].v[1], keep), mul2(s[i].v[2], s[i].v[3], keep);
#pragma unroll
        for (int st = 0; st < kSteps; st += 2) {
            uint32_t kb[2][NT][4], bb[2][2][NT][2];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
#pragma unroll
                for (int x = 0; x < NT; ++x) load_tokens(kb[half][x], operand(b, 0, x), (st + half) * 16, lane);
                as_columns(bb[half], kb[half], m0, m1);
            }
            using P = Pairs<3, 3, NT>;
            each_step<0, P::n>([&](auto k) {
                step2<P, k.value>(s[2 * st], s[2 * st + 1], ue, bb[0][0], bb[0][1]);
                step2<P, k.value>(s[2 * st + 2], s[2 * st + 3], ue, bb[1][0], bb[1][1]);
            });
        }
    }
    if constexpr (kEnds) {
        put_state(end_of(slot) + (unit ? dk * dv : 0));
    } else if (p.final_state && segment == p.segments - 1) {
        put_state(p.final_state + seq * dk * dv);
    }
}

// From segments' ends from zero (B) and what they make of a state (A) to their ends, in place and in order:
// S <- A S + B, or B where an episode starts in the segment.  A block has kJoinCols columns of one sequence's state, a
// warp 16 rows of them; products are of bf16 terms, as in the scan (by fused multiply-adds a segment of 128 x 128 took
// 2.8 to 4.4 us, bound by reads of shared memory; this 2.5).  The A and B of two segments come while the product of
// one is taken.
constexpr int kJoinCols = 16, kJoinThreads = 256, kMostSegments = 512;

template <int DK>
struct JoinSmem {
    static constexpr int kLd = DK + 8, kLdTerm = DK + 8;  // floats of a row of A; bf16 of a column of S
    static constexpr size_t kA = (size_t)DK * kLd * 4, kTerms = (size_t)3 * kJoinCols * kLdTerm * 2;
    static constexpr size_t kBytes = 3 * kA + kTerms + kMostSegments * 4;
};

template <int kBytes>
__device__ __forceinline__ void copy_async(float* to, const float* from) {
    if constexpr (kBytes == 16)  // not through L1, which this much shared memory leaves too small
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_at(to)), "l"(from) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_at(to)), "l"(from) : "memory");
}

template <int DK>
__global__ void __launch_bounds__(kJoinThreads) scan_join_kernel(const Scan p) {
    using L = JoinSmem<DK>;
    extern __shared__ __align__(16) uint8_t join_shared[];
    float* a = reinterpret_cast<float*>(join_shared);                                     // three of [DK][kLd]
    __nv_bfloat16* terms = reinterpret_cast<__nv_bfloat16*>(join_shared + 3 * L::kA);     // S, by terms: [3][kJoinCols][kLdTerm]
    int* joined = reinterpret_cast<int*>(join_shared + 3 * L::kA + L::kTerms);            // no episode starts in the segment
    const int dk = p.dk, dv = p.dv, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int r0 = warp * 16 + lane / 4, c0 = blockIdx.y * kJoinCols + lane % 4 * 2;
    const int64_t first = (int64_t)blockIdx.x * (p.segments - 1), size = (int64_t)dk * (dk + dv);
    const bool vec = dk % 4 == 0 && dv % 4 == 0 && reinterpret_cast<uintptr_t>(p.ends) % 16 == 0;
    for (int i = threadIdx.x; i < (int)((3 * L::kA + L::kTerms) / 16); i += kJoinThreads)  // rows and columns past dk stay zero
        reinterpret_cast<uint4*>(join_shared)[i] = make_uint4(0, 0, 0, 0);
    for (int i = threadIdx.x; i < p.segments; i += kJoinThreads) joined[i] = i > 0 && i + 1 < p.segments && !p.restarts[first + i];
    __syncthreads();
    auto fetch = [&](int i) {  // A of segment i, where it is needed
        if (i < p.segments && joined[i]) {
            const float* from = p.ends + (first + i) * size + dk * dv;
            float* to = a + i % 3 * DK * L::kLd;
            constexpr int kPer = DK / 4, kStep = kJoinThreads / kPer;
            const int row = threadIdx.x / kPer, c = threadIdx.x % kPer * 4;
            if (vec && dk == DK) {
#pragma unroll
                for (int j = 0; j < DK; j += kStep) copy_async<16>(to + (row + j) * L::kLd + c, from + (row + j) * DK + c);
            } else if (vec) {
                for (int j = row; j < dk; j += kStep)
                    if (c < dk) copy_async<16>(to + j * L::kLd + c, from + j * dk + c);
            } else {
                for (int j = warp; j < dk; j += kJoinThreads / 32)
                    for (int e = lane; e < dk; e += 32) copy_async<4>(to + j * L::kLd + e, from + j * dk + e);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto each_pair = [&](int i, auto&& f) {  // this thread's values of segment i's end, two neighbours at a time
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int r = r0 + half * 8, c = c0 + t * 8;
                if (i + 1 < p.segments && r < dk) f(t, half, p.ends + (first + i) * size + r * dv + c, c < dv, c + 1 < dv);
            }
    };
    auto load = [&](Acc (&x)[2], int i) {
        x[0].zero(), x[1].zero();
        each_pair(i, [&](int t, int half, const float* from, bool in0, bool in1) {
            if (vec && in1) {
                const float2 y = *reinterpret_cast<const float2*>(from);
                x[t].v[half * 2] = y.x, x[t].v[half * 2 + 1] = y.y;
            } else {
                if (in0) x[t].v[half * 2] = from[0];
                if (in1) x[t].v[half * 2 + 1] = from[1];
            }
        });
    };
    Acc end[2], next[2], after[2];
    load(end, 0);
    load(next, 1);
    fetch(1);
    for (int i = 0;; ++i) {
        fetch(i + 2);
        load(after, i + 2);
        if (joined[i] && warp * 16 < dk) {
            const float* row = a + i % 3 * DK * L::kLd + r0 * L::kLd + lane % 4 * 2;
#pragma unroll
            for (int k = 0; k < DK; k += 16) {
                uint32_t ta[3][4], tb[3][4], bb[2][3][2];
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    const float2 x = *reinterpret_cast<const float2*>(row + z % 2 * 8 * L::kLd + k + z / 2 * 8);
                    uint32_t t[3];
                    split(x.x, x.y, t);
#pragma unroll
                    for (int y = 0; y < 3; ++y) ta[y][z] = t[y];
                }
#pragma unroll
                for (int y = 0; y < 3; ++y) load_rows(tb[y], Rows{terms + y * kJoinCols * L::kLdTerm, L::kLdTerm}, k, lane);
                as_rows(bb, tb);
                mma2<3>(end, ta, bb);
            }
            each_pair(i, [&](int t, int half, float* to, bool in0, bool in1) {
                if (vec && in1) {
                    *reinterpret_cast<float2*>(to) = make_float2(end[t].v[half * 2], end[t].v[half * 2 + 1]);
                } else {
                    if (in0) to[0] = end[t].v[half * 2];
                    if (in1) to[1] = end[t].v[half * 2 + 1];
                }
            });
        }
        if (i + 2 >= p.segments) break;
        __syncthreads();  // S has been read
        if (warp * 16 < DK) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    uint32_t s[3];
                    split(end[t].v[e], end[t].v[2 + e], s);
#pragma unroll
                    for (int x = 0; x < 3; ++x) {
                        __nv_bfloat16* to = terms + (x * kJoinCols + t * 8 + lane % 4 * 2 + e) * L::kLdTerm + r0;
                        to[0] = __ushort_as_bfloat16((unsigned short)s[x]);
                        to[8] = __ushort_as_bfloat16((unsigned short)(s[x] >> 16));
                    }
                }
        }
        asm volatile("cp.async.wait_group 1;" ::: "memory");  // A of segment i + 1
        __syncthreads();
#pragma unroll
        for (int t = 0; t < 2; ++t) end[t] = next[t], next[t] = after[t];
    }
}

// --------------------------------------------------------------- backward
//
// Over the chunks from last to first, with dS the gradient of the state after
// the chunk, E and the state S before it kept by the forward pass:
//
//   dU = scale (D o Q K^T)^T dO + eta K dS        ubar = N^T dU,  N = (I + beta D o K K^T (i > j))^-1
//   dV = beta ubar    dbeta_i = ubar_i . e_i    dL = -ubar U^T    W = dO U^T
//   dA = scale D o W (i >= j)    dP = beta D o dL (i > j)
//   dQ = scale gamma dO S^T + dA K
//   dK = -beta gamma ubar S^T + eta U dS^T + dA^T Q + (dP + dP^T) K
//   dS <- Gamma dS + (scale gamma Q)^T dO - (beta gamma K)^T ubar
//   dg_l = sum_{i>=l>j} E_ij + sum_{i>=l} (q_i . dq_i^S + k_i . dk_i^S) + sum_{j<l} u_j . (eta_j dS^T k_j) + Gamma <dS, S>
//   E_ij = dA_ij q_i.k_j + dP_ij k_i.k_j
//
// (^S: the parts of dq and dk that come through S.)  A block takes one (env,
// head).  A warp has two parts.  For what sums over dk it owns 16 columns of dS,
// transposed in registers as in the forward pass, and takes dU, ubar and the
// update of dS without leaving them.  For what sums over dv (dQ, dK) it owns 16
// rows: dS goes through shared memory in fp32, U and ubar as bf16 terms, S comes
// from the checkpoint.  A helper prepares the next chunk (decays, Q K^T, K K^T,
// N) and finishes dg and dbeta of the last.  Two barriers a chunk.
//
// 1,024 envs x 4 heads x 128 tokens of 64 x 64: 762 us, 831 with an episode's end in
// 200 tokens.  No unit is full (36% of the issue slots, tensor cores 20% busy): 10
// warps an SM (168 registers a thread, 100 KB of shared memory a block) wait for
// their own chains of products.

struct alignas(16) BackChunk {
    __nv_bfloat16 n[3][kC][kLdM];    // N, by terms
    __nv_bfloat16 att[3][kC][kLdM];  // scale D_ij q_i.k_j (i >= j), by terms
    float fa[kC][kC], fp[kC][kC];    // scale D_ij (i >= j), beta_i D_ij (i > j); zero outside the chunk
    float qk[kC][kC], kk[kC][kC];    // q_i.k_j, k_i.k_j
    float gamma[kC], eta[kC], beta[kC];
    float keep;
    int block, r0, r1, fresh;
    int state;                       // S counts: the chunk begins its block and no episode
};

// What warps add up for a chunk's scalars.
template <int kWarpsK, int kWarpsV>
struct alignas(16) BackSums {
    float dot_i[kWarpsK][kC], dot_s[kWarpsK], dot_j[kWarpsV][kC], dbeta[kWarpsV][kC];
};

template <class T, int DK, int DV>
struct BackwardSmem {
    static constexpr int kWarpsK = DK / 16, kWarpsV = DV / 16, kWarps = DK > DV ? kWarpsK : kWarpsV;
    static constexpr int NT = Terms<T>::n;
    static constexpr bool kInPlace = NT == 1;
    // bf16 is used as fetched: warps on one block, the helper on the next, one on its way, for which heads of 128 have no
    // room.  Others are turned into terms on arrival, for two blocks, and one buffer is enough.
    static constexpr int kBuffers = kInPlace ? (DK + DV > 192 ? 2 : 3) : 1;
    static constexpr int kTileK = Fetch<T, DK>::kElements, kTileV = Fetch<T, DV>::kElements;
    static constexpr size_t kRaw = (size_t)(2 * kTileK + kTileV) * sizeof(T);
    static constexpr int kTk = DK + 8, kTv = DV + 8;  // rows of terms
    static constexpr size_t kTermBlock = kInPlace ? 0 : (size_t)NT * kC * (2 * kTk + kTv) * 2;
    static constexpr size_t kTile3 = (size_t)3 * kC * kTv * 2;    // U, ubar
    static constexpr int kLdS = DV + 8;
    static constexpr size_t kState = (size_t)DK * kLdS * 4;       // dS
    static constexpr size_t kFetched = (size_t)Fetch<float, DV>::kPanels * DK * 128;  // S, panels of 32 columns
    using Sums = BackSums<kWarpsK, kWarpsV>;
    struct alignas(16) Shared {
        BackChunk chunk[2];
        Sums sums[2];
        HelperScratch hs;
        __nv_bfloat16 da[3][kC][kLdM], dp[3][kC][kLdM];
        float ee[2][kC][kC + 1];  // E through dA, and through dP
        uint64_t arrived[kBuffers], state_arrived;
    };
    static constexpr size_t kOut = sizeof(T) == 2 ? (size_t)kC * kLdOut * 2 : 0;  // of a warp
    static constexpr size_t kBase = 1024 + kBuffers * kRaw + 2 * kTermBlock + 2 * kTile3 + kState + sizeof(Shared) + kWarps * kOut;
    // S is fetched a chunk ahead where it has room, else read from global memory when needed (1,024 envs of 64 x 64: 1,250 us
    // against 815 when both were built, although that leaves room for a third block on an SM).
    static constexpr bool kFetchState = kBase + kFetched <= 227 * 1024;
    static constexpr size_t kBytes = kBase + (kFetchState ? kFetched : 0);
    static_assert(kRaw % 1024 == 0 && kFetched % 1024 == 0 && kTermBlock % 16 == 0 && kTile3 % 16 == 0 && kState % 16 == 0, "layout");
    static_assert(kBytes <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ void store_columns(__nv_bfloat16* tile, int ld, int c0, const uint32_t (&r)[4], int lane) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(
                     smem_at(tile + (lane % 8 + lane / 16 * 8) * ld + c0 + lane / 8 % 2 * 8)),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
                 : "memory");
}

// Sums over a warp's rows of values that belong to columns (tokens 2 quad, 2 quad + 1 and those + 8).
__device__ __forceinline__ void add_over_rows(float (&x)[4]) {
#pragma unroll
    for (int w = 4; w < 32; w *= 2)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] += __shfl_xor_sync(0xffffffffu, x[i], w);
}

template <class T, int DK, int DV, bool kRegular>
__global__ void __launch_bounds__((DK > DV ? DK : DV) * 2 + 32, DK <= 64 && DV <= 64 ? 2 : 1)
    scan_backward_kernel(const Scan p, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_q,
                         const __grid_constant__ CUtensorMap map_o, const __grid_constant__ CUtensorMap map_s) {
    static_assert(!kRegular || DK == DV, "a warp of a regular head owns 16 of its keys and 16 of its values");
    using L = BackwardSmem<T, DK, DV>;
    const bool aligned = kRegular || p.aligned;
    const int dk_ = kRegular ? DK : p.dk, dv_ = kRegular ? DV : p.dv;
    constexpr int NT = Terms<T>::n, ND = NT == 3 ? 3 : 2;  // ND: terms of dS and U for dk alone, which leaves as T
    extern __shared__ __align__(16) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + (1024 - (smem_at(smem_raw) & 1023) & 1023);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, row = lane / 4, quad = lane % 4;
    float* fetched = reinterpret_cast<float*>(smem + L::kBuffers * L::kRaw);
    uint8_t* at = smem + L::kBuffers * L::kRaw + (L::kFetchState ? L::kFetched : 0);
    __nv_bfloat16* terms = reinterpret_cast<__nv_bfloat16*>(at);
    __nv_bfloat16* ut = reinterpret_cast<__nv_bfloat16*>(at + 2 * L::kTermBlock);  // U
    __nv_bfloat16* bt = ut + L::kTile3 / 2;                                        // ubar
    float* st = reinterpret_cast<float*>(bt + L::kTile3 / 2);                      // dS, rows = dk
    typename L::Shared& sh = *reinterpret_cast<typename L::Shared*>(st + L::kState / 4);
    const int64_t seq = blockIdx.x, n = seq / p.h, h = seq % p.h;
    const int64_t out_t = p.n * p.h, out_0 = n * p.h + h;  // rows of contiguous (t, n, h, d) tensors
    const int64_t blocks = (p.t + kC - 1) / kC;
    const int slices = (dv_ + 15) / 16;
    const bool fetch_state = L::kFetchState && (kRegular || dv_ % 4 == 0);
    auto raw_tile = [&](int64_t b) { return reinterpret_cast<T*>(smem + b % L::kBuffers * L::kRaw); };
    // term x of K (which = 0), Q (1) or dO (2) of a block as an operand
    auto operand = [&](int64_t b, int which, int x) {
        if constexpr (L::kInPlace)
            return Panels{reinterpret_cast<const __nv_bfloat16*>(raw_tile(b)) + which * L::kTileK};
        else
            return Rows{terms + (b & 1) * (L::kTermBlock / 2) + which * NT * kC * L::kTk + x * kC * (which == 2 ? L::kTv : L::kTk),
                        which == 2 ? L::kTv : L::kTk};
    };
    if (!aligned)
        for (int i = threadIdx.x; i < (int)(L::kBuffers * L::kRaw / 16); i += blockDim.x)
            reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kBuffers; ++i) tc::mbar_init(&sh.arrived[i], 1);
        tc::mbar_init(&sh.state_arrived, 1);
        tc::mbar_init_fence();
        tc::prefetch_map(&map_k);
        tc::prefetch_map(&map_q);
        tc::prefetch_map(&map_o);
    }
    __syncthreads();

    if (warp == L::kWarps) {
        const T* q = static_cast<const T*>(p.q) + n * p.sq.n + h * p.sq.h;
        const T* k = static_cast<const T*>(p.k) + n * p.sk.n + h * p.sk.h;
        const T* d_o = static_cast<const T*>(p.d_o) + out_0 * dv_;
        auto fetch = [&](int64_t b) {
            if (b < 0) return;
            T* to = raw_tile(b);
            uint64_t* bar = &sh.arrived[b % L::kBuffers];
            const int count = (int)(p.t - b * kC < kC ? p.t - b * kC : kC);
            if (aligned && lane == 0) tc::mbar_expect_tx(bar, (uint32_t)L::kRaw);
            Fetch<T, DK>::run(to, &map_k, k, p.sk.t, n, h, 0, b * kC, count, dk_, aligned, bar, lane);
            Fetch<T, DK>::run(to + L::kTileK, &map_q, q, p.sq.t, n, h, 0, b * kC, count, dk_, aligned, bar, lane);
            Fetch<T, DV>::run(to + 2 * L::kTileK, &map_o, d_o, out_t * dv_, n, h, 0, b * kC, count, dv_, aligned, bar, lane);
        };
        const GatePointers get_gates(p, n, h, lane);
        Gates gates{}, next = get_gates.load((blocks - 1) * kC, p.t, lane);
        float decay = 1.f;
        uint32_t starts = 0;
        int64_t b = blocks, turn_of_block = -1;
        int r1 = 0;
        if (L::kBuffers == 3) fetch(blocks - 1);
        uint32_t states = 0;  // fetched so far
        // The chunk before the last one prepared; false where a wait has given up.
        auto prepare = [&](BackChunk& ch) -> bool {
            if (r1 == 0) {
                --b;
                if (b < 0) {
                    if (lane == 0) ch.block = -1;
                    return true;
                }
                ++turn_of_block;
                r1 = (int)(p.t - b * kC < kC ? p.t - b * kC : kC);
                fetch(L::kBuffers == 3 ? b - 1 : b);  // the warps are on b + 1
                gates = next;
                if (b > 0) next = get_gates.load((b - 1) * kC, p.t, lane);
                decay = gates.decay();
                starts = gates.starts();
                // phases of a buffer's barrier count the blocks that it has held
                if (aligned && !tc::mbar_wait_warp(&sh.arrived[b % L::kBuffers], turn_of_block / L::kBuffers & 1)) {
                    if (lane == 0) atomicAdd(p.stalls, 1u);
                    return false;
                }
                __syncwarp();
                if constexpr (!L::kInPlace) {
                    __nv_bfloat16* to = terms + (b & 1) * (L::kTermBlock / 2);
                    to_terms_warp<T, DK>(to, L::kTk, raw_tile(b), lane);
                    to_terms_warp<T, DK>(to + NT * kC * L::kTk, L::kTk, raw_tile(b) + L::kTileK, lane);
                    to_terms_warp<T, DV>(to + 2 * NT * kC * L::kTk, L::kTv, raw_tile(b) + 2 * L::kTileK, lane);
                    tc::fence_async_smem();
                    __syncwarp();
                }
            }
            const uint32_t earlier = starts & ((1u << r1) - 1);
            const int r0 = earlier ? 31 - __clz(earlier) : 0;
            const bool fresh = starts >> r0 & 1;
            HelperScratch& hs = sh.hs;
            chunk_decays(hs.d, ch.gamma, ch.eta, ch.beta, ch.keep, within(lane, r0, r1) ? decay : 1.f, gates.beta, r0, r1, fresh, lane);
            if (lane == 0) ch.block = (int)b, ch.r0 = r0, ch.r1 = r1, ch.fresh = fresh, ch.state = !fresh;
            Acc kk[2], qk[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) kk[i].zero(), qk[i].zero();
#pragma unroll
            for (int s = 0; s < DK / 16; ++s) {
                uint32_t ka[NT][4], qa[NT][4];
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    load_rows(ka[x], operand(b, 0, x), s * 16, lane);
                    load_rows(qa[x], operand(b, 1, x), s * 16, lane);
                }
                uint32_t kb[2][NT][2];
                as_rows(kb, ka);
                mma2_zip<3, 3>(kk, ka, kb, qk, qa, kb);
            }
            __syncwarp();
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int i = row + half * 8, j = c * 8 + quad * 2;
                    const float2 d = *reinterpret_cast<const float2*>(&hs.d[i][j]);
                    const float be = ch.beta[i];
                    const bool in0 = within(i, r0, r1) && j >= r0, in1 = within(i, r0, r1) && j + 1 >= r0;
                    const float2 fa = make_float2(in0 && i >= j ? p.scale * d.x : 0.f, in1 && i >= j + 1 ? p.scale * d.y : 0.f);
                    const float2 fb = make_float2(in0 && i > j ? be * d.x : 0.f, in1 && i > j + 1 ? be * d.y : 0.f);
                    const float2 vq = make_float2(fa.x != 0.f ? qk[c].v[half * 2] : 0.f, fa.y != 0.f ? qk[c].v[half * 2 + 1] : 0.f);
                    // k_i.k_j counts where dP may, also at beta = 0, where dP is zero
                    const float2 vk = make_float2(in0 && i > j ? kk[c].v[half * 2] : 0.f, in1 && i > j + 1 ? kk[c].v[half * 2 + 1] : 0.f);
                    *reinterpret_cast<float2*>(&ch.fa[i][j]) = fa;
                    *reinterpret_cast<float2*>(&ch.fp[i][j]) = fb;
                    *reinterpret_cast<float2*>(&ch.qk[i][j]) = vq;
                    *reinterpret_cast<float2*>(&ch.kk[i][j]) = vk;
                    *reinterpret_cast<float2*>(&hs.b[i][j]) = make_float2(fb.x * vk.x, fb.y * vk.y);
                    uint32_t s[3];
                    split(fa.x * vq.x, fa.y * vq.y, s);
#pragma unroll
                    for (int x = 0; x < 3; ++x) *reinterpret_cast<uint32_t*>(&ch.att[x][i][j]) = s[x];
                }
            __syncwarp();
            invert_lower(hs, lane);
            store_terms<3>(ch.n, hs.b, lane);
            __syncwarp();
            r1 = r0;
            return true;
        };
        // After a wait that gave up no chunk follows the one at hand, and blocks on their way land before the block leaves.
        auto give_up = [&](BackChunk& ch) {
            for (int x = 0; aligned && x <= (L::kBuffers == 3) && b >= x; ++x)  // block b, and the one fetched ahead of it
                tc::mbar_drain(&sh.arrived[(b - x) % L::kBuffers], (turn_of_block + x) / L::kBuffers & 1);
            if (lane == 0) ch.block = -1;
        };
        // dg and dbeta of a chunk, from its sums
        auto finish = [&](const BackChunk& ch, const typename L::Sums& sums) {
            // column j's sums of E from the last row up, then row l's first l columns
            float tail = 0.f;
            if (lane < 16) {
#pragma unroll
                for (int i = kC - 1; i >= 0; --i) {
                    tail += sh.ee[0][i][lane] + sh.ee[1][i][lane];
                    sh.ee[0][i][lane] = tail;
                }
            }
            __syncwarp();
            // lane l: the sums over i >= l and over j < l, from the warps' parts
            const bool in = within(lane, ch.r0, ch.r1);
            float di = 0.f, dj = 0.f, dot = 0.f, dbeta = 0.f;
#pragma unroll
            for (int x = 0; x < L::kWarpsK; ++x) {
                di += in ? sums.dot_i[x][lane & 15] : 0.f;
                dot += sums.dot_s[x];
            }
#pragma unroll
            for (int x = 0; x < L::kWarpsV; ++x) {
                dj += in ? sums.dot_j[x][lane & 15] : 0.f;
                dbeta += sums.dbeta[x][lane & 15];
            }
#pragma unroll
            for (int w = 1; w < 16; w *= 2) {
                const float up = __shfl_down_sync(0xffffffffu, di, w, 16), down = __shfl_up_sync(0xffffffffu, dj, w, 16);
                if ((lane & 15) + w < 16) di += up;
                if ((lane & 15) >= w) dj += down;
            }
            const float before = __shfl_up_sync(0xffffffffu, dj, 1, 16);
            if (in) {
                float dg = di + ((lane & 15) ? before : 0.f) + dot;
#pragma unroll
                for (int j = 0; j < kC - 1; ++j)
                    if (j < lane) dg += sh.ee[0][lane][j];
                const int64_t to = (ch.block * (int64_t)kC + lane) * out_t + out_0;
                p.dg[to] = dg;
                p.dbeta[to] = dbeta;
            }
        };
        bool ok = prepare(sh.chunk[0]);
        if (!ok) give_up(sh.chunk[0]);
        __syncthreads();
        for (int turn = 0;; ++turn) {
            const BackChunk& ch = sh.chunk[turn & 1];
            if (states && !tc::mbar_wait_warp(&sh.state_arrived, (states - 1) & 1)) {  // the warps have read it
                tc::mbar_drain(&sh.state_arrived, (states - 1) & 1);
                if (lane == 0) atomicAdd(p.stalls, 1u);
                ok = false;
            }
            if (ok && ch.block >= 0 && ch.state && fetch_state) {
                ++states;
                if (lane == 0) {
                    tc::mbar_expect_tx(&sh.state_arrived, (uint32_t)L::kFetched);
#pragma unroll
                    for (int i = 0; i < Fetch<float, DV>::kPanels; ++i)
                        tc::tma_load_3d(fetched + i * DK * 32, &map_s, &sh.state_arrived, i * 32, 0, (int)(seq * blocks + ch.block));
                }
            }
            if (turn) finish(sh.chunk[(turn & 1) ^ 1], sh.sums[(turn & 1) ^ 1]);
            if (ch.block < 0) break;
            __syncwarp();
            __syncthreads();  // after U, ubar and dS are in shared memory
            BackChunk& next = sh.chunk[(turn & 1) ^ 1];
            if (!ok || !(ok = prepare(next))) give_up(next);
            __syncthreads();  // after dA and dP are
        }
        return;
    }

    const bool has_v = warp < L::kWarpsV, has_k = warp < L::kWarpsK;
    const int c0 = warp * 16;
    const bool whole_v = kRegular || c0 + 16 <= dv_, whole_k = kRegular || c0 + 16 <= dk_;
    const bool v_aligned = sizeof(T) == 2 && (kRegular || (dv_ % 8 == 0 && reinterpret_cast<uintptr_t>(p.dv_out) % 16 == 0));
    const bool k_pairs = sizeof(T) == 2 && (kRegular || (dk_ % 2 == 0 && (reinterpret_cast<uintptr_t>(p.dq) | reinterpret_cast<uintptr_t>(p.dk_out)) % 4 == 0));
    T* out_tile = reinterpret_cast<T*>(reinterpret_cast<uint8_t*>(&sh + 1) + warp * L::kOut);
    Acc ds[DK / 8];  // dS^T: rows = columns c0.. of the state, columns = dk
    auto each_state = [&](auto&& f) {
#pragma unroll
        for (int i = 0; i < DK / 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int kk = i * 8 + quad * 2 + e % 2, c = c0 + row + e / 2 * 8;
                f(ds[i].v[e], kk, c, kk < dk_ && c < dv_);
            }
    };
    {
        const float* df = p.d_final ? p.d_final + seq * dk_ * dv_ : nullptr;
        each_state([&](float& x, int kk, int c, bool in) { x = df && in ? df[kk * dv_ + c] : 0.f; });
    }
    uint32_t states = 0;  // fetched so far
    __syncthreads();
    for (int turn = 0;; ++turn) {
        const BackChunk& ch = sh.chunk[turn & 1];
        typename L::Sums& sums = sh.sums[turn & 1];
        const int64_t b = ch.block;
        if (b < 0) break;
        const int r0 = ch.r0, r1 = ch.r1;
        const bool state = ch.state;
        const uint32_t m0 = pair_mask(quad * 2, r0, r1), m1 = pair_mask(quad * 2 + 8, r0, r1);
        // the copies of this block were waited for by the helper; a wait that is over makes them visible here
        if constexpr (L::kInPlace)
            if (aligned) tc::mbar_see(&sh.arrived[b % L::kBuffers], (blocks - 1 - b) / L::kBuffers & 1);

        uint32_t xa[3][4];  // (-beta gamma ubar)^T for the update of dS
        if (has_v) {
            Acc e[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                e[c].zero();
                if (kRegular || warp < slices) {
                    const float4 x = __ldcs(reinterpret_cast<const float4*>(p.errors) + error_at(seq * blocks + b, slices, warp, c, lane));
                    e[c].v[0] = x.x, e[c].v[1] = x.y, e[c].v[2] = x.z, e[c].v[3] = x.w;
                }
            }
            // dS to shared memory, and (K dS)^T
            Acc du[2], du2[2];
            du[0].zero(), du[1].zero(), du2[0].zero(), du2[1].zero();
#pragma unroll
            for (int s = 0; s < DK / 16; ++s) {
                uint32_t sa[3][4], ka[NT][4];
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    uint32_t tmp[3];
                    const Acc& t = ds[2 * s + z / 2];
                    split(t.v[z % 2 * 2], t.v[z % 2 * 2 + 1], tmp);
#pragma unroll
                    for (int x = 0; x < 3; ++x) sa[x][z] = tmp[x];
                    float* to = st + (s * 16 + z / 2 * 8 + quad * 2) * L::kLdS + c0 + row + z % 2 * 8;
                    to[0] = t.v[z % 2 * 2];
                    to[L::kLdS] = t.v[z % 2 * 2 + 1];
                }
#pragma unroll
                for (int x = 0; x < NT; ++x) load_rows(ka[x], operand(b, 0, x), s * 16, lane);
                uint32_t kb[2][NT][2];
                as_rows(kb, ka);
                mma2<3>(s % 2 ? du2 : du, sa, kb);
            }
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int z = 0; z < 4; ++z) du[c].v[z] += du2[c].v[z];
            // U, and what eta gets: u_j . (dS^T k_j)
            uint32_t ua[3][4];
            float zj[4], be[4];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int j = c * 8 + quad * 2;
                const float2 b2 = *reinterpret_cast<const float2*>(&ch.beta[j]), et = *reinterpret_cast<const float2*>(&ch.eta[j]);
                const bool in0 = within(j, r0, r1), in1 = within(j + 1, r0, r1);
                float u[4];
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    const bool in = z % 2 ? in1 : in0;
                    e[c].v[z] = in ? e[c].v[z] : 0.f;
                    du[c].v[z] = in ? du[c].v[z] * (z % 2 ? et.y : et.x) : 0.f;
                    u[z] = e[c].v[z] * (z % 2 ? b2.y : b2.x);
                }
                zj[c * 2] = u[0] * du[c].v[0] + u[2] * du[c].v[2];
                zj[c * 2 + 1] = u[1] * du[c].v[1] + u[3] * du[c].v[3];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t tmp[3];
                    split(u[half * 2], u[half * 2 + 1], tmp);
#pragma unroll
                    for (int x = 0; x < 3; ++x) ua[x][c * 2 + half] = tmp[x];
                }
            }
#pragma unroll
            for (int x = 0; x < 3; ++x) store_columns(ut + x * kC * L::kTv, L::kTv, c0, ua[x], lane);
            // dU += dO^T (scale D o Q K^T), ubar^T = dU^T N
            uint32_t oa[NT][4], ab[3][4];
#pragma unroll
            for (int x = 0; x < NT; ++x) {
                load_columns(oa[x], operand(b, 2, x), c0, lane);
#pragma unroll
                for (int z = 0; z < 4; ++z) oa[x][z] &= z < 2 ? m0 : m1;
            }
#pragma unroll
            for (int x = 0; x < 3; ++x) load_tokens(ab[x], Rows{&ch.att[x][0][0], kLdM}, 0, lane);
            uint32_t da[3][4], bb[2][3][2];
            as_columns(bb, ab);
            mma2_split<3>(du, oa, bb);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t tmp[3];
                    split(du[c].v[half * 2], du[c].v[half * 2 + 1], tmp);
#pragma unroll
                    for (int x = 0; x < 3; ++x) da[x][c * 2 + half] = tmp[x];
                }
            }
#pragma unroll
            for (int x = 0; x < 3; ++x) load_tokens(ab[x], Rows{&ch.n[x][0][0], kLdM}, 0, lane);
            uint32_t ba[3][4];
            as_columns(bb, ab);
            Acc ubar[2];
            ubar[0].zero(), ubar[1].zero();
            mma2_split<3>(ubar, da, bb);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                Acc& ub = ubar[c];
                const int j = c * 8 + quad * 2;
                const float2 b2 = *reinterpret_cast<const float2*>(&ch.beta[j]), ga = *reinterpret_cast<const float2*>(&ch.gamma[j]);
                const bool in0 = within(j, r0, r1), in1 = within(j + 1, r0, r1);
#pragma unroll
                for (int z = 0; z < 4; ++z)
                    if (!(z % 2 ? in1 : in0)) ub.v[z] = 0.f;
                be[c * 2] = ub.v[0] * e[c].v[0] + ub.v[2] * e[c].v[2];
                be[c * 2 + 1] = ub.v[1] * e[c].v[1] + ub.v[3] * e[c].v[3];
                const float x0 = -b2.x * ga.x, x1 = -b2.y * ga.y;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t tmp[3], tmp2[3];
                    split(ub.v[half * 2], ub.v[half * 2 + 1], tmp);
                    split(x0 * ub.v[half * 2], x1 * ub.v[half * 2 + 1], tmp2);
#pragma unroll
                    for (int x = 0; x < 3; ++x) ba[x][c * 2 + half] = tmp[x], xa[x][c * 2 + half] = tmp2[x];
                }
                // dv = beta ubar
                if (v_aligned && whole_v) {
#pragma unroll
                    for (int z = 0; z < 4; ++z)
                        out_tile[(j + z % 2) * kLdOut + row + z / 2 * 8] = from_f32<T>((z % 2 ? b2.y : b2.x) * ub.v[z]);
                } else {
                    T* dv = static_cast<T*>(p.dv_out) + ((b * kC + j) * out_t + out_0) * dv_ + c0 + row;
#pragma unroll
                    for (int z = 0; z < 4; ++z)
                        if ((z % 2 ? in1 : in0) && c0 + row + z / 2 * 8 < dv_)
                            dv[z % 2 * out_t * dv_ + z / 2 * 8] = from_f32<T>((z % 2 ? b2.y : b2.x) * ub.v[z]);
                }
            }
#pragma unroll
            for (int x = 0; x < 3; ++x) store_columns(bt + x * kC * L::kTv, L::kTv, c0, ba[x], lane);
            if constexpr (sizeof(T) == 2) {
                if (v_aligned && whole_v) {
                    __syncwarp();
                    const int i = lane / 2;
                    if (within(i, r0, r1))
                        *reinterpret_cast<uint4*>(static_cast<T*>(p.dv_out) + ((b * kC + i) * out_t + out_0) * dv_ + c0 + lane % 2 * 8) =
                            *reinterpret_cast<const uint4*>(out_tile + i * kLdOut + lane % 2 * 8);
                }
            }
            add_over_rows(zj);
            add_over_rows(be);
            if (row == 0) {
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int j = x / 2 * 8 + quad * 2 + x % 2;
                    sums.dot_j[warp][j] = zj[x];
                    sums.dbeta[warp][j] = be[x];
                }
            }
        }
        __syncthreads();

        // W = dO U^T and dL = -ubar U^T, a half of one for each of the first four warps, into dA and dP
        for (int task = warp; task < 4; task += L::kWarps) {
            const int c = task & 1;
            const bool is_w = task < 2;
            Acc parts[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) parts[i].zero();
#pragma unroll
            for (int s = 0; s < DV / 16; ++s) {
                uint32_t uu[3][4], ub[3][2];
#pragma unroll
                for (int x = 0; x < 3; ++x) {
                    load_rows(uu[x], Rows{ut + x * kC * L::kTv, L::kTv}, s * 16, lane);
                    ub[x][0] = c ? uu[x][1] : uu[x][0], ub[x][1] = c ? uu[x][3] : uu[x][2];
                }
                if (is_w) {
                    uint32_t oa[NT][4];
#pragma unroll
                    for (int x = 0; x < NT; ++x) load_rows(oa[x], operand(b, 2, x), s * 16, lane);
                    using P = Pairs<3, NT, 3>;
                    each_step<0, P::n>([&](auto k) { mma(parts[(k.value + s) % 4], oa[P::at(k.value) / 8], ub[P::at(k.value) % 8]); });
                } else {
                    uint32_t ra[3][4];
#pragma unroll
                    for (int x = 0; x < 3; ++x) load_rows(ra[x], Rows{bt + x * kC * L::kTv, L::kTv}, s * 16, lane);
                    using P = Pairs<3, 3, 3>;
                    each_step<0, P::n>([&](auto k) { mma(parts[(k.value + s) % 4], ra[P::at(k.value) / 8], ub[P::at(k.value) % 8]); });
                }
            }
            Acc acc;
#pragma unroll
            for (int e = 0; e < 4; ++e) acc.v[e] = (parts[0].v[e] + parts[1].v[e]) + (parts[2].v[e] + parts[3].v[e]);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int i = row + half * 8, j = c * 8 + quad * 2;
                const float2 f = *reinterpret_cast<const float2*>(is_w ? &ch.fa[i][j] : &ch.fp[i][j]);
                const float2 g = *reinterpret_cast<const float2*>(is_w ? &ch.qk[i][j] : &ch.kk[i][j]);
                const float s = is_w ? 1.f : -1.f;
                const float x = f.x != 0.f ? s * f.x * acc.v[half * 2] : 0.f, y = f.y != 0.f ? s * f.y * acc.v[half * 2 + 1] : 0.f;
                uint32_t tmp[3];
                split(x, y, tmp);
#pragma unroll
                for (int z = 0; z < 3; ++z) *reinterpret_cast<uint32_t*>(is_w ? &sh.da[z][i][j] : &sh.dp[z][i][j]) = tmp[z];
                sh.ee[is_w ? 0 : 1][i][j] = i > j ? x * g.x : 0.f;
                sh.ee[is_w ? 0 : 1][i][j + 1] = i > j + 1 ? y * g.y : 0.f;
            }
        }

        Acc dq[2], dk[2], dku[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) dq[c].zero(), dk[c].zero(), dku[c].zero();
        if (has_k) {
            const float* s0 = p.checkpoints + (seq * blocks + b) * dk_ * dv_;
            if (fetch_state && state) tc::mbar_see(&sh.state_arrived, states & 1);
            float dot = 0.f;
#pragma unroll
            for (int s = 0; s < DV / 16; ++s) {
                uint32_t oa[NT][4], ra[3][4], ua[ND][4];
#pragma unroll
                for (int x = 0; x < NT; ++x) load_rows(oa[x], operand(b, 2, x), s * 16, lane);
#pragma unroll
                for (int x = 0; x < 3; ++x) load_rows(ra[x], Rows{bt + x * kC * L::kTv, L::kTv}, s * 16, lane);
#pragma unroll
                for (int x = 0; x < ND; ++x) load_rows(ua[x], Rows{ut + x * kC * L::kTv, L::kTv}, s * 16, lane);
                uint32_t sb[2][3][2], db[2][ND][2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {  // rows of the state c0 + 8 c + row
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int kk = c0 + c * 8 + row, col = s * 16 + half * 8 + quad * 2;
                        float2 x = make_float2(0.f, 0.f);
                        if (state) {
                            if (fetch_state) {
                                x = *reinterpret_cast<const float2*>(fetched + col / 32 * (DK * 32) + kk * 32 + ((col / 4 % 8) ^ (kk & 7)) * 4 + col % 4);
                            } else if (!L::kFetchState && dv_ % 2 == 0) {
                                if (kk < dk_ && col < dv_) x = __ldcs(reinterpret_cast<const float2*>(s0 + kk * dv_ + col));
                            } else if (kk < dk_) {
                                if (col < dv_) x.x = s0[kk * dv_ + col];
                                if (col + 1 < dv_) x.y = s0[kk * dv_ + col + 1];
                            }
                        }
                        const float2 y = *reinterpret_cast<const float2*>(st + kk * L::kLdS + col);
                        if (state) dot = fmaf(x.x, y.x, fmaf(x.y, y.y, dot));
                        uint32_t tmp[3], tmp2[ND];
                        split(x.x, x.y, tmp);
                        split(y.x, y.y, tmp2);
#pragma unroll
                        for (int z = 0; z < 3; ++z) sb[c][z][half] = tmp[z];
#pragma unroll
                        for (int z = 0; z < ND; ++z) db[c][z][half] = tmp2[z];
                    }
                }
                using X = Pairs<3, 3, 3>;    // dk: 6
                using Y = Pairs<3, NT, 3>;   // dq: 3 (5, 6), then
                using Z = Pairs<ND, ND, ND>; // U dS^T: 3 (3, 6)
                each_step<0, Y::n + Z::n>([&](auto k) {
                    step2<X, k.value>(dk[0], dk[1], ra, sb[0], sb[1]);
                    if constexpr (k.value < Y::n)
                        step2<Y, k.value>(dq[0], dq[1], oa, sb[0], sb[1]);
                    else
                        step2<Z, k.value - Y::n>(dku[0], dku[1], ua, db[0], db[1]);
                });
            }
            // the decays' gradients need q.dq and k.dk of the parts through S alone
            const float g0 = p.scale * ch.gamma[row], g1 = p.scale * ch.gamma[row + 8], e0 = ch.eta[row], e1 = ch.eta[row + 8];
            const float x0 = -ch.beta[row] * ch.gamma[row], x1 = -ch.beta[row + 8] * ch.gamma[row + 8];
            float di[2] = {0.f, 0.f};
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int half = e / 2;
                    const T* qv = raw_tile(b) + L::kTileK;
                    dq[c].v[e] *= half ? g1 : g0;
                    dk[c].v[e] *= half ? x1 : x0;
                    dku[c].v[e] *= half ? e1 : e0;
                    float kx, qx;
                    if constexpr (L::kInPlace) {
                        const int px = panel_at<T>(row + half * 8, c0 + c * 8 + quad * 2 + e % 2);
                        kx = to_f32(qv[px - L::kTileK]), qx = to_f32(qv[px]);
                    } else {
                        kx = qx = 0.f;
#pragma unroll
                        for (int x = NT - 1; x >= 0; --x) {
                            kx += __bfloat162float(*operand(b, 0, x).at(row + half * 8, c0 + c * 8 + quad * 2 + e % 2));
                            qx += __bfloat162float(*operand(b, 1, x).at(row + half * 8, c0 + c * 8 + quad * 2 + e % 2));
                        }
                    }
                    di[half] += qx * dq[c].v[e] + kx * dk[c].v[e];
                }
#pragma unroll
            for (int w = 1; w < 4; w *= 2)
#pragma unroll
                for (int half = 0; half < 2; ++half) di[half] += __shfl_xor_sync(0xffffffffu, di[half], w);
#pragma unroll
            for (int w = 1; w < 32; w *= 2) dot += __shfl_xor_sync(0xffffffffu, dot, w);
            if (quad == 0) sums.dot_i[warp][row] = di[0], sums.dot_i[warp][row + 8] = di[1];
            if (lane == 0) sums.dot_s[warp] = ch.keep * dot;
        }
        if (state) ++states;
        __syncthreads();

        if (has_k) {
            uint32_t da[3][4], dat[3][4], dp[3][4], dpt[3][4], kb[NT][4], qb[NT][4];
#pragma unroll
            for (int x = 0; x < 3; ++x) {
                load_rows(da[x], Rows{&sh.da[x][0][0], kLdM}, 0, lane);
                load_columns(dat[x], Rows{&sh.da[x][0][0], kLdM}, 0, lane);
                load_rows(dp[x], Rows{&sh.dp[x][0][0], kLdM}, 0, lane);
                load_columns(dpt[x], Rows{&sh.dp[x][0][0], kLdM}, 0, lane);
            }
#pragma unroll
            for (int x = 0; x < NT; ++x) {
                load_tokens(kb[x], operand(b, 0, x), c0, lane);
                load_tokens(qb[x], operand(b, 1, x), c0, lane);
            }
            uint32_t k2[2][NT][2], q2[2][NT][2];
            as_columns(k2, kb, m0, m1);
            as_columns(q2, qb, m0, m1);
            mma2_zip<ND, ND>(dq, da, k2, dk, dat, q2);
            mma2_zip<ND, ND>(dku, dp, k2, dk, dpt, k2);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int e = 0; e < 4; ++e) dk[c].v[e] += dku[c].v[e];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int i = row + half * 8, col = c0 + c * 8 + quad * 2;
                    if (!within(i, r0, r1)) continue;
                    const int64_t to = ((b * kC + i) * out_t + out_0) * dk_ + col;
                    if (k_pairs && whole_k) {
                        if constexpr (sizeof(T) == 2) {
                            union { T h[2]; uint32_t u; } x, y;
                            x.h[0] = from_f32<T>(dq[c].v[half * 2]), x.h[1] = from_f32<T>(dq[c].v[half * 2 + 1]);
                            y.h[0] = from_f32<T>(dk[c].v[half * 2]), y.h[1] = from_f32<T>(dk[c].v[half * 2 + 1]);
                            *reinterpret_cast<uint32_t*>(static_cast<T*>(p.dq) + to) = x.u;
                            *reinterpret_cast<uint32_t*>(static_cast<T*>(p.dk_out) + to) = y.u;
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            if (col + e < dk_) {
                                static_cast<T*>(p.dq)[to + e] = from_f32<T>(dq[c].v[half * 2 + e]);
                                static_cast<T*>(p.dk_out)[to + e] = from_f32<T>(dk[c].v[half * 2 + e]);
                            }
                    }
                }
            }
        }
        if (has_v) {
            if (ch.fresh) {  // the state before was dropped
#pragma unroll
                for (int i = 0; i < DK / 8; ++i) ds[i].zero();
            } else {
                const float keep = ch.keep;
                uint32_t ya[3][4];  // (scale gamma dO)^T
                {
                    uint32_t oa[NT][4];
#pragma unroll
                    for (int x = 0; x < NT; ++x) load_columns(oa[x], operand(b, 2, x), c0, lane);
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        const int j = z / 2 * 8 + quad * 2;
                        const float2 ga = *reinterpret_cast<const float2*>(&ch.gamma[j]);
                        float o0 = 0.f, o1 = 0.f;
#pragma unroll
                        for (int x = NT - 1; x >= 0; --x) {
                            o0 += __uint_as_float(oa[x][z] << 16);
                            o1 += __uint_as_float(oa[x][z] & 0xFFFF0000u);
                        }
                        uint32_t tmp[3];
                        split(within(j, r0, r1) ? p.scale * ga.x * o0 : 0.f, within(j + 1, r0, r1) ? p.scale * ga.y * o1 : 0.f, tmp);
#pragma unroll
                        for (int x = 0; x < 3; ++x) ya[x][z] = tmp[x];
                    }
                }
                // Of large heads dS comes back from shared memory: its registers are the others' in between (128 x 128 spills
                // 160 bytes a thread, 44 in the regular kernel, and spilled about twice as much without when that was measured;
                // 64 x 64 has few and is 8% faster without).
                constexpr bool kBack = DK > 64 || DV > 64;
#pragma unroll
                for (int i = 0; i < DK / 8; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        ds[i].v[e] = keep * (kBack ? st[(i * 8 + quad * 2 + e % 2) * L::kLdS + c0 + row + e / 2 * 8] : ds[i].v[e]);
#pragma unroll
                for (int s = 0; s < DK / 16; s += 2) {
                    using P = Pairs<3, 3, NT>;
#pragma unroll
                    for (int which = 0; which < 2; ++which) {
                        uint32_t kb[2][NT][4], bb[2][2][NT][2];
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
#pragma unroll
                            for (int x = 0; x < NT; ++x) load_tokens(kb[half][x], operand(b, which, x), (s + half) * 16, lane);
                            as_columns(bb[half], kb[half], m0, m1);
                        }
                        each_step<0, P::n>([&](auto k) {
                            step2<P, k.value>(ds[2 * s], ds[2 * s + 1], which ? ya : xa, bb[0][0], bb[0][1]);
                            step2<P, k.value>(ds[2 * s + 2], ds[2 * s + 3], which ? ya : xa, bb[1][0], bb[1][1]);
                        });
                    }
                }
            }
        }
    }
    if (p.dstate && has_v) {
        float* to = p.dstate + seq * dk_ * dv_;
        each_state([&](float& x, int kk, int c, bool in) {
            if (in) to[kk * dv_ + c] = x;
        });
    }
}

// ------------------------------------------------------------------- host

// Heads that fill their tiles, of tensors a tiled copy may fetch and 16-byte stores may write, take the
// kRegular kernels: the same code with every test of a ragged edge decided when it is compiled. 1,024 sequences
// x 4 heads x 128 steps of 64 in bfloat16 took 298 and 769 us forwards and back when that was split off, with the
// tests 307 and 814; 256 x 2 heads of 128 backwards 322 and 411.
inline bool on_16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// How many segments a few long sequences are cut into; 1 where that gains nothing.
//
// A sequence's chunks follow one another, so a few long ones leave most SMs idle.  The state after a segment is linear
// in the state before it, S' = A S + B: so first every segment's A and B at once, as scans from a unit matrix without
// values and from zero (outputs left out), then the ends in order, one small product each, then every segment's outputs
// at once from the state before it.  That is two passes of 1 / G of the chunks and G joins in place of one pass.  A pass
// takes as long as the SM with most blocks; how many an SM holds at once goes by the type and by dk, and they slow one
// another (kSharing).  Swept over 24 shapes and three types: the count chosen so is within 3% of the best on average, and
// nowhere slower than the sequence whole by more than measurements differ.  Cut and whole, us:
//
//   envs x heads x tokens, dk = dv   bfloat16                  float16                    float32
//   4 x 4 x 4,096 of 128             249 (6 segments) 523      696 (8) 1,318              834 (8) 1,626
//   4 x 4 x 4,096 of 64              106 (15) 420              171 (18) 773               197 (18) 992
//   4 x 4 x 512 of 128               58 (6) 70                 114 (3) 170                135 (3) 209
//   4 x 4 x 512 of 64                37 (8) 58                 47 (8) 101                 51 (8) 129
//   8 x 4 x 1,024 of 64              58 (8) 109                91 (6) 198                 105 (6) 252
//   8 x 4 x 1,024 of 128             whole: 136, 3 would too   whole: 336, 3 take 394     whole: 414, 3 take 472
//
// Costs are in tenths of a chunk's time, which is 1.6 to 2 us in bfloat16 and two to three times that in the others; the
// joins and the two more launches take the same time in all.
struct SplitCosts {
    int blocks;        // of the passes that an SM holds at once
    int join, launch;  // of a segment, and of the two more launches
};
template <class T>
inline SplitCosts split_costs(int dk) {
    auto fit = [](size_t bytes, int most) { return std::min(most, (int)(228 * 1024 / (bytes + 1024))); };  // 1 KB a block is the system's
    const int blocks = dk > 64 ? fit(ForwardSmem<T, 128>::kBytes, 2) : dk > 32 ? fit(ForwardSmem<T, 64>::kBytes, 3) : fit(ForwardSmem<T, 32>::kBytes, 3);
    return Terms<T>::n == 1 ? SplitCosts{blocks, 10, 100} : SplitCosts{blocks, 5, 50};
}

inline int count_segments(int64_t t, int64_t heads, int dk, int dv, int sms, const SplitCosts& c) {
    constexpr int kSharing[2][4] = {{0, 10, 10, 12}, {0, 10, 13, 13}};  // a chunk's time where so many blocks share an SM; dk > 64
    const int64_t all = (t + kC - 1) / kC, value_blocks = (dv + 63) / 64, key_blocks = (dk + 63) / 64;
    auto pass = [&](int64_t blocks) {
        const int64_t most = (blocks + sms - 1) / sms;
        return most / c.blocks * kSharing[dk > 64][c.blocks] + kSharing[dk > 64][most % c.blocks];
    };
    int64_t best = 1, best_cost = all * pass(heads * value_blocks);
    for (int64_t g = 3; g <= all && g <= kMostSegments && g * c.join + c.launch < best_cost; ++g) {
        const int64_t cost = (all + g - 1) / g * (pass(heads * ((g - 1) * value_blocks + (g - 2) * key_blocks)) + pass(heads * g * value_blocks)) +
                             g * c.join + c.launch;
        if (cost < best_cost) best = g, best_cost = cost;
    }
    const int64_t per = (all + best - 1) / best;
    return all ? (int)((all + per - 1) / per) : 1;
}

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
    const unsigned heads = static_cast<unsigned>(p.n * p.h), segments = p.segments;
    const unsigned value_blocks = (p.dv + L::kWidth - 1) / L::kWidth, key_blocks = (p.dk + L::kWidth - 1) / L::kWidth;
    CUtensorMap map_k{}, map_q{}, map_v{};
    if (p.aligned && p.t) {
        if (int rc = map_rows<T>(&map_k, p.k, p.sk, p, p.dk)) return rc;
        if (int rc = map_rows<T>(&map_q, p.q, p.sq, p, p.dk)) return rc;
        if (int rc = map_rows<T>(&map_v, p.v, p.sv, p, p.dv)) return rc;
    }
    auto go = [&](auto regular, auto ends, dim3 grid) -> int {
        constexpr auto* kernel = scan_forward_kernel<T, DK, decltype(regular)::value, decltype(ends)::value>;
        if (int rc = allow_smem<kernel>((int)L::kBytes, p.device, "delta_scan")) return rc;
        kernel<<<grid, (kForwardWarps + 1) * 32, L::kBytes, st>>>(p, map_k, map_q, map_v);
        return cuda_status(cudaGetLastError(), "delta_scan");
    };
    auto run = [&](auto regular) -> int {
        if (segments > 1) {
            if (int rc = go(regular, std::true_type{}, dim3(heads, value_blocks + key_blocks, segments - 1))) return rc;
            using J = JoinSmem<DK>;
            if (int rc = allow_smem<scan_join_kernel<DK>>((int)J::kBytes, p.device, "delta_scan")) return rc;
            scan_join_kernel<DK><<<dim3(heads, (p.dv + kJoinCols - 1) / kJoinCols), kJoinThreads, J::kBytes, st>>>(p);
            if (int rc = cuda_status(cudaGetLastError(), "delta_scan")) return rc;
        }
        return go(regular, std::false_type{}, dim3(heads, value_blocks, segments));
    };
    const bool regular = p.aligned && p.dk == DK && p.dv % L::kWidth == 0 && on_16(p.o) && on_16(p.final_state) &&
                         on_16(p.checkpoints) && on_16(p.ends);
    return regular ? run(std::true_type{}) : run(std::false_type{});
}

template <class T, int DK, int DV>
int launch_backward_dk_dv(const Scan& p, cudaStream_t st) {
    using L = BackwardSmem<T, DK, DV>;
    CUtensorMap map_k{}, map_q{}, map_o{}, map_s{};
    if (p.aligned) {
        const Strides so{p.n * p.h * p.dv, p.h * p.dv, p.dv};
        if (int rc = map_rows<T>(&map_k, p.k, p.sk, p, p.dk)) return rc;
        if (int rc = map_rows<T>(&map_q, p.q, p.sq, p, p.dk)) return rc;
        if (int rc = map_rows<T>(&map_o, p.d_o, so, p, p.dv)) return rc;
    }
    if (L::kFetchState && p.dv % 4 == 0) {
        const uint64_t dims[3] = {(uint64_t)p.dv, (uint64_t)p.dk, (uint64_t)(p.n * p.h * ((p.t + kC - 1) / kC))};
        const uint64_t strides[2] = {p.dv * 4ull, (uint64_t)p.dk * p.dv * 4};
        const uint32_t box[3] = {32, DK, 1};
        if (dims[2] > 0x7FFFFFFFull) return invalid("delta_scan_backward: more than 2^31 states");
        if (int rc = encode_map(&map_s, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, p.checkpoints, dims, strides, box)) return rc;
    }
    auto go = [&](auto regular) -> int {
        constexpr auto* kernel = scan_backward_kernel<T, DK, DV, decltype(regular)::value>;
        if (int rc = allow_smem<kernel>((int)L::kBytes, p.device, "delta_scan_backward")) return rc;
        kernel<<<static_cast<unsigned>(p.n * p.h), (L::kWarps + 1) * 32, L::kBytes, st>>>(p, map_k, map_q, map_o, map_s);
        return cuda_status(cudaGetLastError(), "delta_scan_backward");
    };
    if constexpr (DK == DV)
        if (p.aligned && p.dk == DK && p.dv == DV && on_16(p.dq) && on_16(p.dk_out) && on_16(p.dv_out)) return go(std::true_type{});
    return go(std::false_type{});
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
