// ops_delta.cu -- the gated delta rule: one token in place (delta_step), and
// the entry points of the sequence kernels (ops_delta.cuh).
#include "ops_delta.cuh"

namespace nesle {
namespace ops {
namespace delta {
namespace {

// One token of every (env, head):
//
//   e = v - a S^T k;  S <- a S + k (beta e)^T;  o = scale (a S^T q + (q.k) beta e)
//
// with S the state before (zero where reset, which is then not even read).
// 10 flop for 8 bytes of state: bound by reading and writing the states once.
// A warp takes 32 columns of one state: a lane holds 4 neighbouring columns of
// every fourth row, all loads in flight at once; S^T k and S^T q are summed in
// one pass and joined over the 4 row groups by shuffles.  No shared memory but
// the two vectors, no barrier.  2,048 envs x 4 heads of 64 x 64: 49.4 us,
// 5.5 TB/s, 84% of a copy.
struct Step {
    const void *q, *k, *v;
    int64_t q_n, q_h, k_n, k_h, v_n, v_h;
    const float *g, *beta;
    int64_t g_n, g_h, b_n, b_h;
    const uint8_t* reset;
    int64_t reset_n;
    float* state;
    int64_t s_n, s_h;
    void* o;
    int64_t n, h;
    int dk, dv;
    float scale;
};

constexpr int kStepWarps = 4;

template <class T, int DK, bool kVec>
__global__ void __launch_bounds__(kStepWarps * 32) step_kernel(const Step p) {
    constexpr int kRows = DK / 4;  // rows of a lane
    __shared__ float ks[kStepWarps][DK], qs[kStepWarps][DK];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, group = lane / 8;
    const int slices = (p.dv + 31) / 32;
    const int64_t item = (int64_t)blockIdx.x * kStepWarps + warp, seq = item / slices;
    if (seq >= p.n * p.h) return;
    const int64_t n = seq / p.h, h = seq % p.h;
    const int c = (int)(item % slices) * 32 + lane % 8 * 4;
    const bool reset = p.reset && p.reset[n * p.reset_n] != 0;
    float* st = p.state + n * p.s_n + h * p.s_h + c;
    float4 s[kRows];
    const int cols = min(4, p.dv - c);  // kVec: 4 or at most 0
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int r = i * 4 + group;
        s[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (reset || r >= p.dk) continue;
        const float* at = st + (int64_t)r * p.dv;
        if constexpr (kVec) {
            if (cols > 0) s[i] = __ldcs(reinterpret_cast<const float4*>(at));
        } else {
            if (cols > 0) s[i].x = at[0];
            if (cols > 1) s[i].y = at[1];
            if (cols > 2) s[i].z = at[2];
            if (cols > 3) s[i].w = at[3];
        }
    }
    const T* q = static_cast<const T*>(p.q) + n * p.q_n + h * p.q_h;
    const T* k = static_cast<const T*>(p.k) + n * p.k_n + h * p.k_h;
    const T* v = static_cast<const T*>(p.v) + n * p.v_n + h * p.v_h;
    const float a = expf(p.g[n * p.g_n + h * p.g_h]), beta = p.beta[n * p.b_n + h * p.b_h];
    float vv[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) vv[j] = j < cols ? to_f32(v[c + j]) : 0.f;
    float qk = 0.f;
    for (int i = lane; i < DK; i += 32) {
        const float kv = i < p.dk ? to_f32(k[i]) : 0.f, qv = i < p.dk ? to_f32(q[i]) : 0.f;
        ks[warp][i] = kv;
        qs[warp][i] = qv;
        qk = fmaf(kv, qv, qk);
    }
#pragma unroll
    for (int w = 16; w; w /= 2) qk += __shfl_xor_sync(0xffffffffu, qk, w);
    __syncwarp();
    float sk[4] = {0.f, 0.f, 0.f, 0.f}, sq[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const float kv = ks[warp][i * 4 + group], qv = qs[warp][i * 4 + group];
        sk[0] = fmaf(s[i].x, kv, sk[0]), sk[1] = fmaf(s[i].y, kv, sk[1]), sk[2] = fmaf(s[i].z, kv, sk[2]), sk[3] = fmaf(s[i].w, kv, sk[3]);
        sq[0] = fmaf(s[i].x, qv, sq[0]), sq[1] = fmaf(s[i].y, qv, sq[1]), sq[2] = fmaf(s[i].z, qv, sq[2]), sq[3] = fmaf(s[i].w, qv, sq[3]);
    }
    const float keep = reset ? 0.f : a;
    float u[4], o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        sk[j] += __shfl_xor_sync(0xffffffffu, sk[j], 8);
        sq[j] += __shfl_xor_sync(0xffffffffu, sq[j], 8);
        sk[j] += __shfl_xor_sync(0xffffffffu, sk[j], 16);
        sq[j] += __shfl_xor_sync(0xffffffffu, sq[j], 16);
        u[j] = beta * (vv[j] - keep * sk[j]);
        o[j] = p.scale * fmaf(qk, u[j], keep * sq[j]);
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int r = i * 4 + group;
        if (r >= p.dk) continue;
        const float kv = ks[warp][r];
        const float4 t = make_float4(fmaf(kv, u[0], keep * s[i].x), fmaf(kv, u[1], keep * s[i].y), fmaf(kv, u[2], keep * s[i].z),
                                     fmaf(kv, u[3], keep * s[i].w));
        float* at = st + (int64_t)r * p.dv;
        if constexpr (kVec) {
            if (cols > 0) __stcs(reinterpret_cast<float4*>(at), t);
        } else {
            if (cols > 0) at[0] = t.x;
            if (cols > 1) at[1] = t.y;
            if (cols > 2) at[2] = t.z;
            if (cols > 3) at[3] = t.w;
        }
    }
    if (group == 0) {
        T* out = static_cast<T*>(p.o) + seq * p.dv + c;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < cols) out[j] = from_f32<T>(o[j]);
    }
}

template <class T, int DK>
cudaError_t launch_step_dk(const Step& p, cudaStream_t st) {
    const int64_t items = p.n * p.h * ((p.dv + 31) / 32);
    const unsigned grid = static_cast<unsigned>((items + kStepWarps - 1) / kStepWarps);
    // 16 bytes at a time where every row of every state starts on 16 bytes.
    const bool vec = p.dv % 4 == 0 && p.s_n % 4 == 0 && p.s_h % 4 == 0 && reinterpret_cast<uintptr_t>(p.state) % 16 == 0;
    if (vec)
        step_kernel<T, DK, true><<<grid, kStepWarps * 32, 0, st>>>(p);
    else
        step_kernel<T, DK, false><<<grid, kStepWarps * 32, 0, st>>>(p);
    return cudaGetLastError();
}
template <class T>
cudaError_t launch_step(const Step& p, cudaStream_t st) {
    if (p.dk <= 32) return launch_step_dk<T, 32>(p, st);
    if (p.dk <= 64) return launch_step_dk<T, 64>(p, st);
    return launch_step_dk<T, 128>(p, st);
}

const char* check_common(int dtype, uint64_t n, uint64_t h, uint64_t dk, uint64_t dv) {
    if (dtype != NESLE_F32 && dtype != NESLE_BF16 && dtype != NESLE_F16) return "delta: unknown element type";
    if (dk < 1 || dk > 128 || dv < 1 || dv > 128) return "delta: head sizes must be 1 to 128";
    if (n > 0x0FFFFFFFull || h > 0x0FFFFFFFull || n * h > 0x0FFFFFFFull) return "delta: too many heads";
    return nullptr;
}

// What a tensor map takes: base and strides on 16 bytes, strides positive and below 2^40 bytes (dimensions of one element
// have none).
bool rows_aligned(const nesle_delta_args& x, const void* p, int64_t st, int64_t sn, int64_t sh, int size) {
    auto ok = [&](uint64_t count, int64_t stride) {
        return count <= 1 || (stride > 0 && stride * size % 16 == 0 && stride < (int64_t(1) << 40) / size);
    };
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ok(x.t, st) && ok(x.n, sn) && ok(x.h, sh) && x.t <= 0x7FFFFFFFull;
}

int segments_of(const nesle_delta_args& a) {
    const int dk = (int)a.dk;
    const SplitCosts c = a.dtype == NESLE_F32 ? split_costs<float>(dk) : a.dtype == NESLE_BF16 ? split_costs<__nv_bfloat16>(dk) : split_costs<__half>(dk);
    return count_segments((int64_t)a.t, (int64_t)(a.n * a.h), dk, (int)a.dv, sm_count(a.device), c);
}

Scan to_scan(const nesle_delta_args& a, bool backward) {
    Scan p{};
    p.q = a.q, p.k = a.k, p.v = a.v;
    p.sq = {a.q_t, a.q_n, a.q_h}, p.sk = {a.k_t, a.k_n, a.k_h}, p.sv = {a.v_t, a.v_n, a.v_h};
    p.g = a.g, p.beta = a.beta;
    p.sg = {a.g_t, a.g_n, a.g_h}, p.sb = {a.beta_t, a.beta_n, a.beta_h};
    p.reset = a.reset, p.reset_t = a.reset_t, p.reset_n = a.reset_n;
    p.state = a.state;
    p.t = (int64_t)a.t, p.n = (int64_t)a.n, p.h = (int64_t)a.h, p.dk = (int)a.dk, p.dv = (int)a.dv;
    p.scale = a.scale;
    const int size = a.dtype == NESLE_F32 ? 4 : 2;
    const int64_t dv = (int64_t)a.dv;
    p.aligned = a.dk * size % 16 == 0 && a.dv * size % 16 == 0 && rows_aligned(a, a.q, a.q_t, a.q_n, a.q_h, size) &&
                rows_aligned(a, a.k, a.k_t, a.k_n, a.k_h, size) &&
                (backward ? rows_aligned(a, a.d_o, p.n * p.h * dv, p.h * dv, dv, size) : rows_aligned(a, a.v, a.v_t, a.v_n, a.v_h, size));
    p.o = a.o, p.final_state = a.final_state, p.errors = a.errors, p.checkpoints = a.checkpoints;
    p.d_o = a.d_o, p.d_final = a.d_final, p.dq = a.dq, p.dk_out = a.d_k, p.dv_out = a.d_v, p.dg = a.dg, p.dbeta = a.dbeta;
    p.dstate = a.dstate;
    p.device = a.device;
    p.segments = 1, p.per = (p.t + kC - 1) / kC;
    return p;
}

}  // namespace
}  // namespace delta
}  // namespace ops
}  // namespace nesle

using namespace nesle;
using namespace nesle::ops;

extern "C" {

int nesle_delta_step(const nesle_delta_step_args* args, void* stream) {
    return guarded([&]() -> int {
        if (!args) return invalid("delta_step: null argument");
        const nesle_delta_step_args& a = *args;
        if (const char* why = delta::check_common(a.dtype, a.n, a.h, a.dk, a.dv)) return invalid(why);
        if (!a.n || !a.h) return NESLE_OK;
        if (!a.q || !a.k || !a.v || !a.g || !a.beta || !a.state || !a.o) return invalid("delta_step: null argument");
        if (!all_on(element_size(a.dtype), a.q, a.k, a.v, a.o) || !all_on(4, a.g, a.beta, a.state))
            return invalid("delta_step: arguments must be aligned to their elements");
        const int64_t size = element_size(a.dtype);
        auto heads = [&](const void* p, int64_t sn, int64_t sh, uint64_t bytes, int64_t element) {  // from the first to the last byte
            return Memory(p, 1, 0, ((a.n - 1) * sn + (a.h - 1) * sh) * element + bytes);
        };
        const Memory o(a.o, 1, 0, a.n * a.h * a.dv * size);
        for (const Memory& x : {heads(a.q, a.q_n, a.q_h, a.dk * size, size), heads(a.k, a.k_n, a.k_h, a.dk * size, size),
                                heads(a.v, a.v_n, a.v_h, a.dv * size, size), heads(a.g, a.g_n, a.g_h, 4, 4), heads(a.beta, a.beta_n, a.beta_h, 4, 4),
                                heads(a.state, a.state_n, a.state_h, a.dk * a.dv * 4, 4), Memory(a.reset, 1, 0, (a.n - 1) * a.reset_n + 1)})
            if (may_overlap(o, x)) return set_error(NESLE_ERR_OVERLAP, "delta_step: o shares memory with another argument");
        OnDevice on(a.device);
        if (!on.ok) return invalid("delta_step: device ordinal out of range");
        const delta::Step p{a.q, a.k, a.v, a.q_n, a.q_h, a.k_n, a.k_h, a.v_n, a.v_h, a.g, a.beta, a.g_n, a.g_h, a.beta_n, a.beta_h,
                            a.reset, a.reset_n, a.state, a.state_n, a.state_h, a.o, (int64_t)a.n, (int64_t)a.h, (int)a.dk,
                            (int)a.dv, a.scale};
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        cudaError_t e;
        if (a.dtype == NESLE_F32)
            e = delta::launch_step<float>(p, st);
        else if (a.dtype == NESLE_BF16)
            e = delta::launch_step<__nv_bfloat16>(p, st);
        else
            e = delta::launch_step<__half>(p, st);
        return cuda_status(e, "delta_step");
    });
}

uint64_t nesle_delta_checkpoint_floats(const nesle_delta_args* a) {
    return a ? a->n * a->h * ((a->t + delta::kC - 1) / delta::kC) * a->dk * a->dv : 0;
}

uint64_t nesle_delta_error_floats(const nesle_delta_args* a) {
    return a ? a->n * a->h * ((a->t + delta::kC - 1) / delta::kC) * ((a->dv + 15) / 16) * 16 * delta::kC : 0;
}

uint64_t nesle_delta_split_floats(const nesle_delta_args* a) {
    if (!a || delta::check_common(a->dtype, a->n, a->h, a->dk, a->dv) || !a->t || a->t > 0x7FFFFFFFull || !a->n || !a->h) return 0;
    const int segments = delta::segments_of(*a);
    return a->n * a->h * (uint64_t)(segments - 1) * (a->dk * (a->dk + a->dv) + 1);
}

int nesle_delta_scan(const nesle_delta_args* args, void* stream) { return nesle_delta_scan_split(args, nullptr, stream); }

int nesle_delta_scan_split(const nesle_delta_args* args, float* workspace, void* stream) {
    return guarded([&]() -> int {
        if (!args) return invalid("delta_scan: null argument");
        const nesle_delta_args& a = *args;
        if (const char* why = delta::check_common(a.dtype, a.n, a.h, a.dk, a.dv)) return invalid(why);
        if (!a.n || !a.h) return NESLE_OK;
        if (a.t && (!a.q || !a.k || !a.v || !a.g || !a.beta || !a.o)) return invalid("delta_scan: null argument");
        if (!all_on(element_size(a.dtype), a.q, a.k, a.v, a.o) || !all_on(4, a.g, a.beta, a.state, a.final_state, a.checkpoints))
            return invalid("delta_scan: arguments must be aligned to their elements");
        if (!a.errors != !a.checkpoints) return invalid("delta_scan: errors and checkpoints go together");
        if (!all_on(16, a.errors)) return invalid("delta_scan: errors must be 16-byte aligned");
        if (!all_on(4, workspace)) return invalid("delta_scan: workspace must be aligned");
        OnDevice on(a.device);
        if (!on.ok) return invalid("delta_scan: device ordinal out of range");
        delta::Scan p = delta::to_scan(a, false);
        if (workspace && a.t && a.t <= 0x7FFFFFFFull) {
            p.segments = delta::segments_of(a);
            const int64_t all = (p.t + delta::kC - 1) / delta::kC;
            p.per = (all + p.segments - 1) / p.segments;
            p.ends = workspace;
            p.restarts = reinterpret_cast<int*>(workspace + p.n * p.h * (p.segments - 1) * p.dk * (p.dk + p.dv));
        }
        if (int rc = stall_counter(a.device, &p.stalls)) return rc;
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (a.dtype == NESLE_F32) return delta::launch_forward<float>(p, st);
        if (a.dtype == NESLE_BF16) return delta::launch_forward<__nv_bfloat16>(p, st);
        return delta::launch_forward<__half>(p, st);
    });
}

int nesle_delta_scan_backward(const nesle_delta_args* args, void* stream) {
    return guarded([&]() -> int {
        if (!args) return invalid("delta_scan_backward: null argument");
        const nesle_delta_args& a = *args;
        if (const char* why = delta::check_common(a.dtype, a.n, a.h, a.dk, a.dv)) return invalid(why);
        if (!a.n || !a.h) return NESLE_OK;
        if (!a.t) return invalid("delta_scan_backward: no tokens");
        if (!a.q || !a.k || !a.v || !a.g || !a.beta || !a.d_o || !a.errors || !a.checkpoints || !a.dq || !a.d_k || !a.d_v || !a.dg ||
            !a.dbeta)
            return invalid("delta_scan_backward: null argument");
        if (!all_on(element_size(a.dtype), a.q, a.k, a.v, a.d_o, a.dq, a.d_k, a.d_v) ||
            !all_on(4, a.g, a.beta, a.d_final, a.dg, a.dbeta, a.dstate))
            return invalid("delta_scan_backward: arguments must be aligned to their elements");
        if (!all_on(16, a.errors, a.checkpoints)) return invalid("delta_scan_backward: errors and checkpoints must be 16-byte aligned");
        OnDevice on(a.device);
        if (!on.ok) return invalid("delta_scan_backward: device ordinal out of range");
        delta::Scan p = delta::to_scan(a, true);
        if (int rc = stall_counter(a.device, &p.stalls)) return rc;
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (a.dtype == NESLE_F32) return delta::launch_backward<float>(p, st);
        if (a.dtype == NESLE_BF16) return delta::launch_backward<__nv_bfloat16>(p, st);
        return delta::launch_backward<__half>(p, st);
    });
}

}  // extern "C"
