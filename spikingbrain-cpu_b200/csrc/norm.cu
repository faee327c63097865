// The step between two blocks of a residual network, in one pass:
//
//   h  = y                  or  y * rsqrt(mean(y^2) + eps) * w_post        (norm after a block)
//   r' = a * r + b * act(gate) * h                                         (gate, residual scale)
//   x  = r' * rsqrt(mean(r'^2) + eps) * w_pre                              (norm before the next block)
//
// (RMSNorm, spikingbrain_cpu/model.py:30-39, and Block.forward's residual additions, model.py:388-392.)
// A row is held in registers as fp32 between its loads and its stores, so y, r and the gate are read once
// and r' and x written once; both statistics are fp32 sums over fp32 values, and x is taken from r' before
// r' is rounded to the residual's type.
#include "w4_host.cuh"

namespace sbq {

struct NormParams {
    const void* y;
    const void* r;
    const void* gate;
    const float* w_post;
    const float* w_pre;
    void* r_out;
    void* x;
    int64_t ldy, ldr, ldg, ldro, ldx;
    int gcol;  // 1: one gate per column, 0: one gate per row
    int y_dtype, r_dtype, g_dtype, x_dtype, act;
    float a, b, eps;
    int64_t m;
    int d;
};

__device__ __forceinline__ float ld1(const void* p, int dtype, int64_t i) {
    if (dtype == SBQ_F32) return static_cast<const float*>(p)[i];
    if (dtype == SBQ_F16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

__device__ __forceinline__ void ld8(const void* p, int dtype, int64_t i, float (&v)[8]) {
    if (dtype == SBQ_F32) {
        const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
        const float4 a = q[0], b = q[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        return;
    }
    const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
    const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (dtype == SBQ_F16) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[j]));
            v[2 * j] = f.x, v[2 * j + 1] = f.y;
        } else {
            v[2 * j] = __uint_as_float(u[j] << 16);
            v[2 * j + 1] = __uint_as_float(u[j] & 0xFFFF0000u);
        }
    }
}

__device__ __forceinline__ void st8(void* p, int dtype, int64_t i, const float (&v)[8]) {
    if (dtype == SBQ_F32) {
        float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
        q[0] = make_float4(v[0], v[1], v[2], v[3]);
        q[1] = make_float4(v[4], v[5], v[6], v[7]);
        return;
    }
    uint32_t u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (dtype == SBQ_F16) {
            const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
            u[j] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
            u[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = make_uint4(u[0], u[1], u[2], u[3]);
}

__device__ __forceinline__ float gate_act(float g, int act) {
    if (act == SBQ_GATE_SIGMOID) return 1.0f / (1.0f + expf(-g));
    if (act == SBQ_GATE_SILU) return g / (1.0f + expf(-g));
    if (act == SBQ_GATE_TANH) return tanhf(g);
    return g;
}

// Sum over the TPR threads of a row (TPR = 32: a warp; otherwise the whole CTA).  `part` holds one float
// per warp; two calls in a row use different buffers, so one barrier per call is enough.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (TPR == 32) return v;
    const int lane = threadIdx.x & 31;
    if (lane == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < TPR / 32 ? part[lane] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

constexpr int norm_threads(int tpr) { return tpr == 32 ? 256 : tpr; }

// Element i (0..7) of a thread's chunk v: eight neighbours (VEC), or a stride of TPR so that the narrow
// accesses of a warp stay next to each other.
template <int TPR, bool VEC>
__device__ __forceinline__ int norm_col(int v, int i, int tid) {
    return VEC ? (v * TPR + tid) * 8 + i : (v * 8 + i) * TPR + tid;
}

template <int TPR, bool VEC>
__device__ __forceinline__ void norm_load(const void* p, int dtype, int64_t row0, int v, int tid, int d, float (&o)[8]) {
    if (VEC) {
        const int c = norm_col<TPR, true>(v, 0, tid);
        if (c < d) {
            ld8(p, dtype, row0 + c, o);
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = 0.0f;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = norm_col<TPR, false>(v, i, tid);
            o[i] = c < d ? ld1(p, dtype, row0 + c) : 0.0f;
        }
    }
}

template <int TPR, bool VEC>
__device__ __forceinline__ void norm_store(void* p, int dtype, int64_t row0, int v, int tid, int d, const float (&o)[8]) {
    if (VEC) {
        const int c = norm_col<TPR, true>(v, 0, tid);
        if (c < d) st8(p, dtype, row0 + c, o);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = norm_col<TPR, false>(v, i, tid);
            if (c < d) w4_store(p, dtype, row0 + c, o[i]);
        }
    }
}

// The gated branch of one chunk added to the scaled residual: o = a * r + b * act(gate) * (y * inv * w_post).
template <int TPR, bool VEC>
__device__ __forceinline__ void norm_combine(const NormParams& p, int64_t row, int v, int tid, float inv,
                                             const float (&y)[8], const float (&r)[8], float (&o)[8]) {
    float w[8], g[8];
    if (p.w_post) norm_load<TPR, VEC>(p.w_post, SBQ_F32, 0, v, tid, p.d, w);
    if (p.gate && p.gcol) norm_load<TPR, VEC>(p.gate, p.g_dtype, row * p.ldg, v, tid, p.d, g);
    const float g0 = p.gate && !p.gcol ? ld1(p.gate, p.g_dtype, row * p.ldg) : 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float h = 0.0f;
        if (p.y) {
            h = y[i];
            if (p.w_post) h = h * inv * w[i];
            if (p.gate) h *= gate_act(p.gcol ? g[i] : g0, p.act);
            h *= p.b;
        }
        o[i] = p.y ? fmaf(p.a, r[i], h) : p.a * r[i];
    }
}

// One row per TPR threads, V chunks of 8 elements per thread.
template <int TPR, int V, bool VEC>
__global__ void __launch_bounds__(norm_threads(TPR)) norm_kernel(const NormParams p) {
    __shared__ float part[2][32];
    const int tid = TPR == 32 ? (int)(threadIdx.x & 31) : (int)threadIdx.x;
    const int64_t row = TPR == 32 ? (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5) : (int64_t)blockIdx.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (row >= p.m) return;  // whole warps; with TPR > 32 there is one row per CTA
    float y[V][8], r[V][8];
    float ss = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        if (p.y) norm_load<TPR, VEC>(p.y, p.y_dtype, row * p.ldy, v, tid, p.d, y[v]);
        norm_load<TPR, VEC>(p.r, p.r_dtype, row * p.ldr, v, tid, p.d, r[v]);
    }
    float inv = 1.0f;
    if (p.y && p.w_post) {
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(y[v][i], y[v][i], ss);
        inv = rsqrtf(row_sum<TPR>(ss, part[0]) / (float)p.d + p.eps);
    }
    ss = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        float o[8];
        norm_combine<TPR, VEC>(p, row, v, tid, inv, y[v], r[v], o);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            r[v][i] = norm_col<TPR, VEC>(v, i, tid) < p.d ? o[i] : 0.0f;
            ss = fmaf(r[v][i], r[v][i], ss);
        }
        if (p.r_out) norm_store<TPR, VEC>(p.r_out, p.r_dtype, row * p.ldro, v, tid, p.d, r[v]);
    }
    if (!p.x) return;
    inv = rsqrtf(row_sum<TPR>(ss, part[1]) / (float)p.d + p.eps);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        float w[8], o[8];
        norm_load<TPR, VEC>(p.w_pre, SBQ_F32, 0, v, tid, p.d, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = r[v][i] * inv * w[i];
        norm_store<TPR, VEC>(p.x, p.x_dtype, row * p.ldx, v, tid, p.d, o);
    }
}

// Rows longer than the registers of one CTA: the row is read again for each statistic (from L2), and
// nothing is written before the last pass, so r_out may be r and x may be y.
constexpr int kLongTpr = 512;
template <bool VEC>
__global__ void __launch_bounds__(kLongTpr) norm_long_kernel(const NormParams p) {
    __shared__ float part[2][32];
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    const int chunks = (p.d + kLongTpr * 8 - 1) / (kLongTpr * 8);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    float y[8], r[8], o[8], inv = 1.0f, ss = 0.0f;
    if (p.y && p.w_post) {
        for (int v = 0; v < chunks; ++v) {
            norm_load<kLongTpr, VEC>(p.y, p.y_dtype, row * p.ldy, v, tid, p.d, y);
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(y[i], y[i], ss);
        }
        inv = rsqrtf(row_sum<kLongTpr>(ss, part[0]) / (float)p.d + p.eps);
    }
    float inv2 = 1.0f;
    for (int pass = p.x ? 0 : 1; pass < 2; ++pass) {
        ss = 0.0f;
        for (int v = 0; v < chunks; ++v) {
            if (p.y) norm_load<kLongTpr, VEC>(p.y, p.y_dtype, row * p.ldy, v, tid, p.d, y);
            norm_load<kLongTpr, VEC>(p.r, p.r_dtype, row * p.ldr, v, tid, p.d, r);
            norm_combine<kLongTpr, VEC>(p, row, v, tid, inv, y, r, o);
            if (pass == 0) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (norm_col<kLongTpr, VEC>(v, i, tid) < p.d) ss = fmaf(o[i], o[i], ss);
            } else {
                if (p.r_out) norm_store<kLongTpr, VEC>(p.r_out, p.r_dtype, row * p.ldro, v, tid, p.d, o);
                if (p.x) {
                    norm_load<kLongTpr, VEC>(p.w_pre, SBQ_F32, 0, v, tid, p.d, r);
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[i] = o[i] * inv2 * r[i];
                    norm_store<kLongTpr, VEC>(p.x, p.x_dtype, row * p.ldx, v, tid, p.d, o);
                }
            }
        }
        if (pass == 0) inv2 = rsqrtf(row_sum<kLongTpr>(ss, part[1]) / (float)p.d + p.eps);
    }
}

template <int TPR, int V>
static cudaError_t launch_norm(const NormParams& p, bool vec, cudaStream_t s) {
    const unsigned grid = (unsigned)(TPR == 32 ? ceil_div(p.m, 8) : p.m);
    return vec ? w4_launch(norm_kernel<TPR, V, true>, grid, norm_threads(TPR), 0, s, p)
               : w4_launch(norm_kernel<TPR, V, false>, grid, norm_threads(TPR), 0, s, p);
}

template <int V>
static cudaError_t launch_norm_v(const NormParams& p, bool vec, cudaStream_t s) {
    if (p.d <= 256 * V) return launch_norm<32, V>(p, vec, s);
    if (p.d <= 512 * V) return launch_norm<64, V>(p, vec, s);
    if (p.d <= 1024 * V) return launch_norm<128, V>(p, vec, s);
    if (p.d <= 2048 * V) return launch_norm<256, V>(p, vec, s);
    if (p.d <= 4096 * V) return launch_norm<512, V>(p, vec, s);
    return vec ? w4_launch(norm_long_kernel<true>, (unsigned)p.m, kLongTpr, 0, s, p)
               : w4_launch(norm_long_kernel<false>, (unsigned)p.m, kLongTpr, 0, s, p);
}

static bool norm_dtype(int t) { return t == SBQ_F32 || t == SBQ_F16 || t == SBQ_BF16; }

// One operand: its type, stride and element alignment; *vec stays true while 8-element accesses are aligned.
static int check_operand(const void* p, int dtype, int64_t ld, int64_t width, int64_t m, const char* what, bool* vec) {
    if (!norm_dtype(dtype)) return set_error(SBQ_ERR_UNSUPPORTED, "%s dtype %d (f32, f16, bf16)", what, dtype);
    const int es = w4_elem(dtype);
    if (reinterpret_cast<uintptr_t>(p) % es) return set_error(SBQ_ERR_ALIGNMENT, "%s must be aligned to its element size", what);
    if (m > 1 && ld < width) return set_error(SBQ_ERR_INVALID_ARGUMENT, "%s row stride smaller than the row", what);
    if (reinterpret_cast<uintptr_t>(p) % 16 || (m > 1 && (ld * es) % 16)) *vec = false;
    return SBQ_OK;
}

}  // namespace sbq

using namespace sbq;

extern "C" int sbq_residual_norm(const sbq_residual_norm_args* a, void* stream) {
    if (!a) return set_error(SBQ_ERR_INVALID_ARGUMENT, "null arguments");
    const int64_t m = a->m, d = a->d;
    if (m <= 0 || d <= 0) return set_error(SBQ_ERR_INVALID_ARGUMENT, "m and d must be positive (m=%lld d=%lld)", (long long)m, (long long)d);
    if (m > (int64_t(1) << 31) - 16 || d >= (int64_t(1) << 30)) return set_error(SBQ_ERR_UNSUPPORTED, "shape too large");
    if (!a->residual) return set_error(SBQ_ERR_INVALID_ARGUMENT, "null residual");
    if (!a->residual_out && !a->out) return set_error(SBQ_ERR_INVALID_ARGUMENT, "no output given");
    if ((a->out != nullptr) != (a->pre_weight != nullptr))
        return set_error(SBQ_ERR_INVALID_ARGUMENT, "the normed output and pre_weight go together");
    if (!a->branch && (a->post_weight || a->gate))
        return set_error(SBQ_ERR_INVALID_ARGUMENT, "post_weight and gate need a branch");
    if (a->gate_act < SBQ_GATE_NONE || a->gate_act > SBQ_GATE_TANH)
        return set_error(SBQ_ERR_UNSUPPORTED, "gate activation %d", a->gate_act);
    if (a->gate_mode != SBQ_GATE_PER_COLUMN && a->gate_mode != SBQ_GATE_PER_ROW && a->gate_mode != SBQ_GATE_FULL)
        return set_error(SBQ_ERR_UNSUPPORTED, "gate mode %d", a->gate_mode);
    if (!(a->eps >= 0.0f)) return set_error(SBQ_ERR_INVALID_ARGUMENT, "eps must not be negative");
    bool vec = d % 8 == 0;
    NormParams p{};
    int st = check_operand(a->residual, a->residual_dtype, a->ld_residual, d, m, "residual", &vec);
    if (!st && a->branch) st = check_operand(a->branch, a->branch_dtype, a->ld_branch, d, m, "branch", &vec);
    if (!st && a->residual_out)
        st = check_operand(a->residual_out, a->residual_dtype, a->ld_residual_out, d, m, "residual output", &vec);
    if (!st && a->out) st = check_operand(a->out, a->out_dtype, a->ld_out, d, m, "output", &vec);
    if (!st && a->gate && a->gate_mode == SBQ_GATE_FULL)
        st = check_operand(a->gate, a->gate_dtype, a->ld_gate, d, m, "gate", &vec);
    else if (!st && a->gate) {
        bool row_vec = true;
        st = check_operand(a->gate, a->gate_dtype, a->ld_gate, 0, 1, "gate", &row_vec);
        if (a->gate_mode == SBQ_GATE_PER_COLUMN) vec = vec && row_vec;
    }
    if (!st && a->pre_weight) st = check_operand(a->pre_weight, SBQ_F32, d, d, 1, "pre_weight", &vec);
    if (!st && a->post_weight) st = check_operand(a->post_weight, SBQ_F32, d, d, 1, "post_weight", &vec);
    if (st) return st;
    p.y = a->branch, p.r = a->residual, p.gate = a->gate, p.w_post = a->post_weight, p.w_pre = a->pre_weight;
    p.r_out = a->residual_out, p.x = a->out;
    p.ldy = a->ld_branch, p.ldr = a->ld_residual, p.ldro = a->ld_residual_out, p.ldx = a->ld_out;
    p.ldg = a->gate_mode == SBQ_GATE_PER_COLUMN ? 0 : a->ld_gate;
    p.gcol = a->gate_mode != SBQ_GATE_PER_ROW;
    p.y_dtype = a->branch_dtype, p.r_dtype = a->residual_dtype, p.g_dtype = a->gate_dtype, p.x_dtype = a->out_dtype;
    p.act = a->gate_act, p.a = a->residual_scale, p.b = a->branch_scale, p.eps = a->eps;
    p.m = m, p.d = (int)d;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    // one chunk per thread while there are fewer rows than SMs (more threads on each row), else two
    const cudaError_t e = m <= w4_sm_count() ? launch_norm_v<1>(p, vec, s) : launch_norm_v<2>(p, vec, s);
    if (e != cudaSuccess) return set_error(SBQ_ERR_CUDA, "residual_norm launch: %s", cudaGetErrorString(e));
    return check_launch("residual_norm");
}
