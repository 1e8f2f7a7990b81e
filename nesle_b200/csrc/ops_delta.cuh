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
    bool aligned;  // every row of q, k, v (and d_o) starts on 16 bytes
    void* o;
    float* final_state;
    float* errors;       // [t][n][h][dv], NULL where no gradient is wanted
    float* checkpoints;  // [n][h][ceil(t / 16)][dk][dv], the state before each chunk
    const void* d_o;     // contiguous
    const float* d_final;
    void *dq, *dk_out, *dv_out;
    float *dg, *dbeta, *dstate;
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

// Tiles are 16 tokens x columns of bf16 in shared memory, rows `ld` elements apart.
// A operand, rows = tokens, k = columns c0..c0+15.  As a B operand with columns = tokens (K K^T) the same registers
// are {r0, r2} for tokens 0..7 and {r1, r3} for tokens 8..15.
__device__ __forceinline__ void load_rows(uint32_t (&r)[4], const __nv_bfloat16* tile, int ld, int c0, int lane) {
    ldmatrix4(r, tile + (lane % 16) * ld + c0 + lane / 16 * 8);
}
// B operand, k = tokens, columns c0..c0+15: {r0, r1} for the first 8 columns, {r2, r3} for the next.
__device__ __forceinline__ void load_tokens(uint32_t (&r)[4], const __nv_bfloat16* tile, int ld, int c0, int lane) {
    ldmatrix4_t(r, tile + (lane % 16) * ld + c0 + lane / 16 * 8);
}
// A operand, rows = columns c0..c0+15 of the tile, k = tokens.
__device__ __forceinline__ void load_columns(uint32_t (&r)[4], const __nv_bfloat16* tile, int ld, int c0, int lane) {
    ldmatrix4_t(r, tile + (lane % 8 + lane / 16 * 8) * ld + c0 + lane / 8 % 2 * 8);
}

__device__ __forceinline__ void cp_async16(void* dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_at(dst)), "l"(src), "r"(bytes) : "memory");
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
            cp_async16(to, from, in ? min(kPer, d - c) * (int)sizeof(T) : 0);
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

// Gate scalars of the 16 tokens of a block, lane i < 16 holding token i.
struct Gates {
    float a, beta;
    uint32_t resets;  // bit i: token i starts an episode
};
__device__ __forceinline__ Gates load_gates(const Scan& p, int64_t n, int64_t h, int64_t t0, int lane) {
    Gates s{1.f, 0.f, 0u};
    const int64_t t = t0 + lane;
    const bool in = lane < kC && t < p.t;
    bool reset = false;
    if (in) {
        s.a = expf(p.g[t * p.sg.t + n * p.sg.n + h * p.sg.h]);
        s.beta = p.beta[t * p.sb.t + n * p.sb.n + h * p.sb.h];
        reset = p.reset && p.reset[t * p.reset_t + n * p.reset_n] != 0;
    }
    s.resets = __ballot_sync(0xffffffffu, reset);
    return s;
}

__device__ __forceinline__ bool within(int i, int r0, int r1) { return i >= r0 && i < r1; }
// Halves of a register that holds tokens i and i + 1 of an operand: zero those outside the chunk, whatever they hold.
__device__ __forceinline__ uint32_t pair_mask(int i, int r0, int r1) {
    return (within(i, r0, r1) ? 0xFFFFu : 0u) | (within(i + 1, r0, r1) ? 0xFFFF0000u : 0u);
}

// ---------------------------------------------------------------- forward
//
// A block takes one (env, head); each warp 16 columns of the state, which need
// nothing of one another.  A warp holds its columns transposed (dv x dk) as
// accumulators of S^T += U^T K, which is also the register layout of the B
// operand of K S and Q S: the state never leaves the registers.  Inputs are
// fetched one block of 16 tokens ahead (cp.async), one barrier a block.

constexpr int kRowPad = 20;  // floats of a row of a warp's 16 x 16 scratch

struct alignas(16) WarpScratch {
    Decays w;
    float lt[kC][kC];         // D_ij k_i.k_j (i > j) at [j][i]
    float r[kC][kRowPad];     // K S, then U
};
static_assert(offsetof(WarpScratch, r) % 16 == 0, "rows are accessed two floats at a time");

template <class T, int DK>
struct ForwardSmem {
    static constexpr int kLd = DK + 16 / sizeof(T);      // raw rows
    static constexpr int kLdTerm = DK + 8;               // rows of terms; the same for bf16
    static constexpr bool kInPlace = Terms<T>::n == 1;
    __host__ __device__ static constexpr size_t raw(int dv16) { return 2 * kC * (2 * kLd + (size_t)dv16) * sizeof(T); }
    __host__ __device__ static constexpr size_t terms() { return kInPlace ? 0 : 2 * Terms<T>::n * kC * kLdTerm * 2; }
    static size_t bytes(int warps) { return raw(warps * 16 + 16) + terms() + warps * sizeof(WarpScratch); }
};

template <class T, int DK>
__global__ void __launch_bounds__(256) scan_forward_kernel(const Scan p) {
    using L = ForwardSmem<T, DK>;
    constexpr int NT = Terms<T>::n, kTiles = DK / 8, kSteps = DK / 16;
    constexpr int NO = NT == 3 ? 3 : 2;  // terms that o needs: 16 bits and more against its own 8 or 11
    extern __shared__ __align__(16) uint8_t smem[];
    const int warps = blockDim.x / 32, warp = threadIdx.x / 32, lane = threadIdx.x % 32, row = lane / 4, quad = lane % 4;
    const int ldv = warps * 16 + 16;
    T* raw = reinterpret_cast<T*>(smem);
    constexpr int kRaw = kC * L::kLd;
    const int raw_v = kC * ldv, raw_all = 2 * kRaw + raw_v;
    __nv_bfloat16* terms = reinterpret_cast<__nv_bfloat16*>(smem + L::raw(ldv));
    WarpScratch& ws = reinterpret_cast<WarpScratch*>(smem + L::raw(ldv) + L::terms())[warp];
    const int64_t seq = blockIdx.x, n = seq / p.h, h = seq % p.h;
    const T* q = static_cast<const T*>(p.q) + n * p.sq.n + h * p.sq.h;
    const T* k = static_cast<const T*>(p.k) + n * p.sk.n + h * p.sk.h;
    const T* v = static_cast<const T*>(p.v) + n * p.sv.n + h * p.sv.h;
    const int64_t blocks = (p.t + kC - 1) / kC;
    const int c0 = warp * 16;  // this warp's columns of the state

    auto fetch = [&](int64_t b, int buf) {
        T* to = raw + buf * raw_all;
        stage<T, DK>(to, L::kLd, k, p.sk.t, b * kC, p.t, p.dk, p.aligned);
        stage<T, DK>(to + kRaw, L::kLd, q, p.sq.t, b * kC, p.t, p.dk, p.aligned);
        constexpr int kPer = 16 / sizeof(T);
        const int per_row = warps * 16 / kPer;
        for (int i = threadIdx.x; i < kC * per_row; i += blockDim.x) {
            const int r = i / per_row, c = i % per_row * kPer;
            const bool in = b * kC + r < p.t && c < p.dv;
            T* dst = to + 2 * kRaw + r * ldv + c;
            const T* from = v + (in ? (b * kC + r) * p.sv.t + c : 0);
            if (p.aligned) {
                cp_async16(dst, from, in ? min(kPer, p.dv - c) * (int)sizeof(T) : 0);
            } else {
#pragma unroll
                for (int j = 0; j < kPer; ++j) dst[j] = in && c + j < p.dv ? from[j] : from_f32<T>(0.f);
            }
        }
        cp_async_commit();
    };

    Acc s[kTiles];  // S^T: rows = columns c0.. of the state, columns = dk
    const float* s0 = p.state ? p.state + seq * p.dk * p.dv : nullptr;
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int kk = i * 8 + quad * 2 + e % 2, c = c0 + row + e / 2 * 8;
            s[i].v[e] = s0 && kk < p.dk && c < p.dv ? s0[(int64_t)kk * p.dv + c] : 0.f;
        }

    fetch(0, 0);
    Gates next = load_gates(p, n, h, 0, lane);
    for (int64_t b = 0; b < blocks; ++b) {
        const int buf = b & 1;
        cp_async_wait<0>();
        __syncthreads();
        if (b + 1 < blocks) fetch(b + 1, buf ^ 1);
        const Gates gates = next;
        if (b + 1 < blocks) next = load_gates(p, n, h, (b + 1) * kC, lane);
        const T* tk = raw + buf * raw_all;
        const T* tv = tk + 2 * kRaw;
        const __nv_bfloat16 *kt, *qt;
        if constexpr (L::kInPlace) {
            kt = reinterpret_cast<const __nv_bfloat16*>(tk);
            qt = kt + kRaw;
        } else {
            to_terms<T, DK>(terms, L::kLdTerm, tk, L::kLd);
            to_terms<T, DK>(terms + NT * kC * L::kLdTerm, L::kLdTerm, tk + kRaw, L::kLd);
            kt = terms;
            qt = terms + NT * kC * L::kLdTerm;
            __syncthreads();
        }
        if (p.checkpoints) {
            float* to = p.checkpoints + (seq * blocks + b) * p.dk * p.dv;
#pragma unroll
            for (int i = 0; i < kTiles; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int kk = i * 8 + quad * 2 + e % 2, c = c0 + row + e / 2 * 8;
                    if (kk < p.dk && c < p.dv) to[(int64_t)kk * p.dv + c] = s[i].v[e];
                }
        }
        const int count = (int)(p.t - b * kC < kC ? p.t - b * kC : kC);
        for (int r0 = 0; r0 < count;) {
            const bool fresh = gates.resets >> r0 & 1;
            const uint32_t later = gates.resets & ~((2u << r0) - 1);
            const int r1 = later ? min(count, __ffs(later) - 1) : count;
            if (fresh) {
#pragma unroll
                for (int i = 0; i < kTiles; ++i) s[i].zero();
            }
            __syncwarp();
            fill_decays(ws.w, within(lane, r0, r1) ? gates.a : 1.f, gates.beta, r0, r1, fresh, lane);

            Acc kk[2], qk[2], ks[2], qs[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) kk[i].zero(), qk[i].zero(), ks[i].zero(), qs[i].zero();
#pragma unroll
            for (int st = 0; st < kSteps; ++st) {
                uint32_t ka[NT][4], qa[NT][4];
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    load_rows(ka[x], kt + x * kC * L::kLdTerm, L::kLdTerm, st * 16, lane);
                    load_rows(qa[x], qt + x * kC * L::kLdTerm, L::kLdTerm, st * 16, lane);
                }
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t kb[NT][2], sb[3][2], lo[3], hi[3];
#pragma unroll
                    for (int x = 0; x < NT; ++x) kb[x][0] = ka[x][c], kb[x][1] = ka[x][c + 2];
                    mma_terms<3>(kk[c], ka, kb);
                    mma_terms<NO>(qk[c], qa, kb);
                    split(s[2 * st].v[2 * c], s[2 * st].v[2 * c + 1], lo);
                    split(s[2 * st + 1].v[2 * c], s[2 * st + 1].v[2 * c + 1], hi);
#pragma unroll
                    for (int x = 0; x < 3; ++x) sb[x][0] = lo[x], sb[x][1] = hi[x];
                    mma_terms<3>(ks[c], ka, sb);
                    mma_terms<NO>(qs[c], qa, sb);
                }
            }
            // the triangular part to shared memory, D o Q K^T as the A operand of (D o Q K^T) U
            uint32_t att[NO][4];
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int i = row + half * 8, j = c * 8 + quad * 2;
                    float at[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float d = ws.w.d[i][j + e];
                        const bool in = within(i, r0, r1) && within(j + e, r0, r1);
                        ws.lt[j + e][i] = in && i > j + e ? d * kk[c].v[half * 2 + e] : 0.f;
                        at[e] = in && i >= j + e ? d * qk[c].v[half * 2 + e] : 0.f;
                    }
                    uint32_t tmp[NO];
                    split(at[0], at[1], tmp);
#pragma unroll
                    for (int x = 0; x < NO; ++x) att[x][c * 2 + half] = tmp[x];
                    *reinterpret_cast<float2*>(&ws.r[i][j]) = make_float2(ks[c].v[half * 2], ks[c].v[half * 2 + 1]);
                }
            __syncwarp();
            if (lane < 16) {  // one column of the state each: forward substitution
                float x[kC];
#pragma unroll
                for (int i = 0; i < kC; ++i) x[i] = to_f32(tv[i * ldv + c0 + lane]) - ws.w.gamma[i] * ws.r[i][lane];
                float* er = p.errors && c0 + lane < p.dv ? p.errors + ((b * kC * p.n + n) * p.h + h) * p.dv + c0 + lane : nullptr;
                const int64_t er_t = p.n * p.h * p.dv;
#pragma unroll
                for (int i = 0; i < kC; ++i) {
                    const bool in = within(i, r0, r1);
                    const float u = in ? ws.w.beta[i] * x[i] : 0.f;
                    if (er && in) er[i * er_t] = x[i];
                    ws.r[i][lane] = u;
#pragma unroll
                    for (int j = i + 1; j < kC; ++j) x[j] = fmaf(-ws.lt[i][j], u, x[j]);
                }
            }
            __syncwarp();
            // U as the B operand (tokens x columns) of (D o Q K^T) U, and eta U transposed as the A operand of the update
            uint32_t ua[3][4];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t ub[NO][2];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int i = quad * 2 + half * 8;
                    const float x = ws.r[i][c * 8 + row], y = ws.r[i + 1][c * 8 + row];
                    uint32_t tmp[NO], tmp3[3];
                    split(x, y, tmp);
                    split(x * ws.w.eta[i], y * ws.w.eta[i + 1], tmp3);
#pragma unroll
                    for (int z = 0; z < NO; ++z) ub[z][half] = tmp[z];
#pragma unroll
                    for (int z = 0; z < 3; ++z) ua[z][half * 2 + c] = tmp3[z];
                }
                const float g0 = ws.w.gamma[row], g1 = ws.w.gamma[row + 8];
                qs[c].v[0] *= g0, qs[c].v[1] *= g0, qs[c].v[2] *= g1, qs[c].v[3] *= g1;
                mma_terms<NO>(qs[c], att, ub);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int i = row + half * 8, col = c0 + c * 8 + quad * 2;
                    if (within(i, r0, r1)) {
                        T* o = static_cast<T*>(p.o) + (((b * kC + i) * p.n + n) * p.h + h) * p.dv + col;
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            if (col + e < p.dv) o[e] = from_f32<T>(p.scale * qs[c].v[half * 2 + e]);
                    }
                }
            }
            const float keep = ws.w.keep;
            const uint32_t m0 = pair_mask(quad * 2, r0, r1), m1 = pair_mask(quad * 2 + 8, r0, r1);
#pragma unroll
            for (int st = 0; st < kSteps; ++st) {
                uint32_t kb[NT][4];
#pragma unroll
                for (int x = 0; x < NT; ++x) load_tokens(kb[x], kt + x * kC * L::kLdTerm, L::kLdTerm, st * 16, lane);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    Acc& acc = s[2 * st + c];
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc.v[e] *= keep;
                    uint32_t bb[NT][2];
#pragma unroll
                    for (int x = 0; x < NT; ++x) bb[x][0] = kb[x][2 * c] & m0, bb[x][1] = kb[x][2 * c + 1] & m1;
                    mma_terms<3>(acc, ua, bb);
                }
            }
            r0 = r1;
        }
    }
    if (p.final_state) {
        float* to = p.final_state + seq * p.dk * p.dv;
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int kk = i * 8 + quad * 2 + e % 2, c = c0 + row + e / 2 * 8;
                if (kk < p.dk && c < p.dv) to[(int64_t)kk * p.dv + c] = s[i].v[e];
            }
    }
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
    Gates next = load_gates(p, n, h, (blocks - 1) * kC, lane);
    for (int64_t b = blocks - 1; b >= 0; --b) {
        const int buf = b & 1;
        cp_async_wait<0>();
        __syncthreads();
        if (b > 0) fetch(b - 1, buf ^ 1);
        const Gates gates = next;
        if (b > 0) next = load_gates(p, n, h, (b - 1) * kC, lane);
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
            const uint32_t earlier = gates.resets & ((1u << r1) - 1);
            const int r0 = earlier ? 31 - __clz(earlier) : 0;
            const bool fresh = gates.resets >> r0 & 1;
            fill_decays(ws.w, within(lane, r0, r1) ? gates.a : 1.f, gates.beta, r0, r1, fresh, lane);
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
                    load_rows(ka[x], kt + x * kC * L::kTk, L::kTk, st * 16, lane);
                    load_rows(qa[x], qt + x * kC * L::kTk, L::kTk, st * 16, lane);
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
                for (int x = 0; x < NT; ++x) load_tokens(ob[x], ot + x * kC * L::kTv, L::kTv, c0, lane);
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
                for (int x = 0; x < 3; ++x) load_rows(uu[x], ut + x * kC * L::kTv, L::kTv, c0, lane);
#pragma unroll
                for (int x = 0; x < NT; ++x) load_rows(oa[x], ot + x * kC * L::kTv, L::kTv, c0, lane);
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
                    for (int x = 0; x < NT; ++x) load_rows(oa[x], ot + x * kC * L::kTv, L::kTv, st * 16, lane);
#pragma unroll
                    for (int x = 0; x < 3; ++x) {
                        load_rows(ua[x], ut + x * kC * L::kTv, L::kTv, st * 16, lane);
                        load_rows(xa[x], xt + x * kC * L::kTv, L::kTv, st * 16, lane);
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
                    load_tokens(kb[x], kt + x * kC * L::kTk, L::kTk, c0, lane);
                    load_tokens(qb[x], qt + x * kC * L::kTk, L::kTk, c0, lane);
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
                        load_columns(qa[x], qt + x * kC * L::kTk, L::kTk, c0, lane);
                        load_columns(ka[x], kt + x * kC * L::kTk, L::kTk, c0, lane);
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
                            load_tokens(xb[x], xt + x * kC * L::kTv, L::kTv, st * 16, lane);
                            load_tokens(yb[x], yt + x * kC * L::kTv, L::kTv, st * 16, lane);
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
                        load_columns(xa[x], xt + x * kC * L::kTv, L::kTv, c0, lane);
                        load_columns(ya[x], yt + x * kC * L::kTv, L::kTv, c0, lane);
                    }
#pragma unroll
                    for (int st = 0; st < DK / 16; ++st) {
                        uint32_t kb[NT][4], qb[NT][4];
#pragma unroll
                        for (int x = 0; x < NT; ++x) {
                            load_tokens(kb[x], kt + x * kC * L::kTk, L::kTk, st * 16, lane);
                            load_tokens(qb[x], qt + x * kC * L::kTk, L::kTk, st * 16, lane);
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

template <class T, int DK>
int launch_forward_dk(const Scan& p, cudaStream_t st) {
    const int warps = (p.dv + 15) / 16;
    const size_t bytes = ForwardSmem<T, DK>::bytes(warps);
    auto* kernel = scan_forward_kernel<T, DK>;
    if (int rc = cuda_status(allow_smem(kernel, (int)bytes), "delta_scan")) return rc;
    kernel<<<static_cast<unsigned>(p.n * p.h), warps * 32, bytes, st>>>(p);
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
