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
//
// The bytes bound it.  Measured on B200: 8192 x 4096, fp32 in and fp16 out, without a post norm 69.5 us (6.8 TB/s, 1.03 of
// the measured copy rate), with it 75 us; 1 x 4096 2.9 us (a launch); 16-bit rows with a gate per element, which have
// half the bytes per element and twice the arithmetic, 3001 x 2560 19.7 us (3.9 TB/s) and 3001 x 2559 29 us (up to 22 and
// 34 on some machines): there instruction issue bounds it (75 to 78 % of the slots, 64 and 102 instructions per 32 elements).
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

__device__ __forceinline__ void unpack8(const uint4& a, int dtype, float (&v)[8]) {
    const uint32_t u[4] = {a.x, a.y, a.z, a.w};
    if (dtype == SBQ_F16) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[j]));
            v[2 * j] = f.x, v[2 * j + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[2 * j] = __uint_as_float(u[j] << 16), v[2 * j + 1] = __uint_as_float(u[j] & 0xFFFF0000u);
    }
}

__device__ __forceinline__ void ld8(const void* p, int dtype, int64_t i, float (&v)[8]) {
    if (dtype == SBQ_F32) {
        const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
        const float4 a = q[0], b = q[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        return;
    }
    unpack8(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i), dtype, v);
}

__device__ __forceinline__ void st8(void* p, int dtype, int64_t i, const float (&v)[8]) {
    if (dtype == SBQ_F32) {
        float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
        q[0] = make_float4(v[0], v[1], v[2], v[3]);
        q[1] = make_float4(v[4], v[5], v[6], v[7]);
        return;
    }
    uint32_t u[4];
    if (dtype == SBQ_F16) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
            u[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
            u[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = make_uint4(u[0], u[1], u[2], u[3]);
}

// Eight fp32 weights from column c on, any c in [0, d - 8]: three aligned quads and a shift that is the same for a
// row (eight single loads cost three times the L1 cycles).
__device__ __forceinline__ void ld8_weight(const float* w, int c, int d, float (&o)[8]) {
    const int s = c & 3;
    const float4* q = reinterpret_cast<const float4*>(w + (c - s));
    const float4 a = __ldg(q), b = __ldg(q + 1);
    // the third quad holds columns of this chunk only if s > 0, and all of it may lie past the end
    float4 e = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (s > 0) {
        if (c - s + 12 <= d) {
            e = __ldg(q + 2);
        } else {
            const float* t = w + (c - s + 8);
            e.x = __ldg(t);
            if (s > 1) e.y = __ldg(t + 1);
            if (s > 2) e.z = __ldg(t + 2);
        }
    }
    const float v[12] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w, e.x, e.y, e.z, e.w};
    if (s == 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = v[i];
    } else if (s == 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = v[i + 1];
    } else if (s == 2) {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = v[i + 2];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = v[i + 3];
    }
}

// Elements lo .. hi - 1 of eight.
__device__ __forceinline__ void st8_some(void* p, int dtype, int64_t i, int lo, int hi, const float (&v)[8]) {
    if (dtype == SBQ_F32) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j >= lo && j < hi) static_cast<float*>(p)[i + j] = v[j];
    } else if (dtype == SBQ_F16) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j >= lo && j < hi) static_cast<__half*>(p)[i + j] = __float2half_rn(v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j >= lo && j < hi) static_cast<__nv_bfloat16*>(p)[i + j] = __float2bfloat16_rn(v[j]);
    }
}

__device__ __forceinline__ float ex2_approx(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float rcp_approx(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// 1 / (1 + 2^(-g log2 e)) from the hardware's power of two and reciprocal, for every type of result.  Relative error at
// most (2 + 0.32 |g|) 2^-22 for g down to -87, 0 below: the rounding of the exponent (2^-24) and of log2 e (2^-26) count |g|
// times, the power of two is good to 2^-22, the rest adds about as much.  So a gate of -20 is off by 2e-6 of itself, which
// is 2e-9; 16-bit results round far above it.  (expf and an exact division made the gated step instruction-bound.)
__device__ __forceinline__ float sigmoid_approx(float g) { return rcp_approx(1.0f + ex2_approx(-1.44269504f * g)); }

__device__ __forceinline__ void gate_act8(float (&g)[8], int act) {
    if (act == SBQ_GATE_SIGMOID) {
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = sigmoid_approx(g[i]);
    } else if (act == SBQ_GATE_SILU) {
        // g * sigmoid(g): an infinite negative g gives -inf * 0 = NaN, where the limit is 0
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] *= sigmoid_approx(g[i]);
    } else if (act == SBQ_GATE_TANH) {
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = tanhf(g[i]);
    }
}

// Threads per row: TPR (8, 16, 32: several rows per CTA, a row's threads are neighbouring lanes) or, for TPR = 0, the
// whole CTA, of any number of warps.
template <int TPR>
__device__ __forceinline__ int row_threads() { return TPR ? TPR : (int)blockDim.x; }

// Sum over a row's threads.  `part` holds one float per warp; two calls in a row use different buffers, so one
// barrier per call is enough.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* part) {
#pragma unroll
    for (int o = (TPR ? TPR : 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (TPR) return v;
    const int lane = threadIdx.x & 31;
    if (lane == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < (int)(blockDim.x >> 5) ? part[lane] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// How a row is cut into chunks of 8 elements per thread.
//   kAligned  every access of a chunk is aligned (the weights' too);
//   kShifted  the rows of all operands start at the same distance `phase` past an 8-element boundary (any width,
//             contiguous operands): the chunks start `phase` elements before the row, so that their accesses are
//             aligned.  A row's first and last chunk are read whole where that stays inside the operand (the
//             neighbours' elements are dropped) and stored element by element; weights by shifted quads;
//   kStrided  anything else: a thread's elements lie a row's threads apart, so that the narrow accesses of a warp are neighbours.
enum NormMode { kAligned, kShifted, kStrided };

template <int TPR, int MODE>
__device__ __forceinline__ int norm_col(int v, int i, int tid, int phase) {
    const int n = row_threads<TPR>();
    if (MODE == kStrided) return (v * 8 + i) * n + tid;
    return (v * n + tid) * 8 + i - (MODE == kShifted ? phase : 0);
}

// One chunk of row `row` (row stride ld) of an operand of m rows; outside the row: zeros.
template <int TPR, int MODE>
__device__ __forceinline__ void norm_load(const void* p, int dtype, int64_t row, int64_t ld, int v, int tid,
                                          const NormParams& q, int phase, float (&o)[8]) {
    const int c0 = norm_col<TPR, MODE>(v, 0, tid, phase), d = q.d;
    const int64_t at = row * ld + c0;
    if (MODE != kStrided && (MODE == kAligned ? c0 < d : c0 >= 0 && c0 + 8 <= d)) {
        ld8(p, dtype, at, o);
        return;
    }
    if (MODE == kShifted && c0 < d && at >= 0 && at + 8 <= (q.m - 1) * ld + d) {
        ld8(p, dtype, at, o);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if ((unsigned)(c0 + i) >= (unsigned)d) o[i] = 0.0f;
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int c = norm_col<TPR, MODE>(v, i, tid, phase);
        o[i] = MODE != kAligned && (unsigned)c < (unsigned)d ? ld1(p, dtype, row * ld + c) : 0.0f;
    }
}

// The same of a vector [d].
template <int TPR, int MODE>
__device__ __forceinline__ void norm_load_vec(const void* p, int dtype, int v, int tid, int d, int phase, float (&o)[8]) {
    const int c0 = norm_col<TPR, MODE>(v, 0, tid, phase);
    if (MODE == kAligned && c0 < d) {
        ld8(p, dtype, c0, o);
        return;
    }
    if (MODE == kShifted && c0 >= 0 && c0 + 8 <= d && dtype == SBQ_F32 && !(reinterpret_cast<uintptr_t>(p) & 15)) {
        ld8_weight(static_cast<const float*>(p), c0, d, o);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int c = norm_col<TPR, MODE>(v, i, tid, phase);
        o[i] = MODE != kAligned && (unsigned)c < (unsigned)d ? ld1(p, dtype, c) : 0.0f;
    }
}

template <int TPR, int MODE>
__device__ __forceinline__ void norm_store(void* p, int dtype, int64_t row0, int v, int tid, int d, int phase,
                                           const float (&o)[8]) {
    const int c0 = norm_col<TPR, MODE>(v, 0, tid, phase);
    if (MODE == kStrided) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = norm_col<TPR, MODE>(v, i, tid, phase);
            if (c < d) w4_store(p, dtype, row0 + c, o[i]);
        }
    } else if (MODE == kAligned ? c0 < d : c0 >= 0 && c0 + 8 <= d) {
        st8(p, dtype, row0 + c0, o);
    } else if (MODE == kShifted && c0 < d) {
        st8_some(p, dtype, row0 + c0, c0 < 0 ? -c0 : 0, d - c0 < 8 ? d - c0 : 8, o);
    }
}

template <int MODE>
__device__ __forceinline__ int norm_phase(const NormParams& p, int64_t row) {
    return MODE == kShifted ? (int)((row * p.ldr) & 7) : 0;
}

// The gate of one chunk, before its activation.
template <int TPR, int MODE>
__device__ __forceinline__ void norm_gate(const NormParams& p, int64_t row, int v, int tid, int phase, float (&g)[8]) {
    if (!p.gcol) {
        const float g0 = ld1(p.gate, p.g_dtype, row * p.ldg);
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = g0;
    } else if (p.ldg) {
        norm_load<TPR, MODE>(p.gate, p.g_dtype, row, p.ldg, v, tid, p, phase, g);
    } else {
        norm_load_vec<TPR, MODE>(p.gate, p.g_dtype, v, tid, p.d, phase, g);
    }
}

// One chunk: r = a * r + b * act(g) * (y * inv * w_post).
template <int TPR, int MODE, bool GATE>
__device__ __forceinline__ void norm_combine(const NormParams& p, int v, int tid, int phase, float inv, float (&y)[8],
                                             float (&g)[8], float (&r)[8]) {
    if (!p.y) {
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] *= p.a;
        return;
    }
    if (p.w_post) {
        float w[8];
        norm_load_vec<TPR, MODE>(p.w_post, SBQ_F32, v, tid, p.d, phase, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = y[i] * inv * w[i];
    }
    if (GATE) {
        gate_act8(g, p.act);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] *= g[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = fmaf(p.a, r[i], p.b * y[i]);
}

// Columns of a chunk outside the row were loaded as zeros and stay zeros.
__device__ __forceinline__ float square8(const float (&r)[8], float ss) {
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(r[i], r[i], ss);
    return ss;
}

// CTAs per SM that the register kernel is compiled for (above 512 threads: two of them as long as that spills little).
__host__ __device__ constexpr int norm_ctas(int threads, int chunks, int mode) {
    return threads == 512                 ? (mode == kAligned ? 4 : 3)
           : chunks == 1 && threads == 768  ? (mode == kShifted ? 1 : 2)
           : chunks == 1 && threads == 1024 ? (mode == kAligned ? 2 : 1)
                                            : 1;
}

// V chunks of 8 elements per thread, everything a row needs from memory (but the weights) requested at the start.
template <int TPR, int V, int MAXT, int MODE, bool GATE>
__global__ void __launch_bounds__(MAXT, norm_ctas(MAXT, V, MODE)) norm_kernel(const NormParams p) {
    __shared__ float part[2][32];
    const int n = row_threads<TPR>(), tid = (int)threadIdx.x % n;
    const int64_t first = TPR ? (int64_t)blockIdx.x * (MAXT / (TPR ? TPR : 1)) + threadIdx.x / n : (int64_t)blockIdx.x;
    // rows that share a warp go on together: one past the end repeats the last row and stores nothing
    const bool live = first < p.m;
    const int64_t row = live ? first : p.m - 1;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int phase = norm_phase<MODE>(p, row);
    float y[V][8], r[V][8], g[GATE ? V : 1][8];
    float ss = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        if (p.y) norm_load<TPR, MODE>(p.y, p.y_dtype, row, p.ldy, v, tid, p, phase, y[v]);
        norm_load<TPR, MODE>(p.r, p.r_dtype, row, p.ldr, v, tid, p, phase, r[v]);
        if (GATE) norm_gate<TPR, MODE>(p, row, v, tid, phase, g[GATE ? v : 0]);
    }
    float inv = 1.0f;
    if (p.y && p.w_post) {
#pragma unroll
        for (int v = 0; v < V; ++v) ss = square8(y[v], ss);
        inv = rsqrtf(row_sum<TPR>(ss, part[0]) / (float)p.d + p.eps);
    }
    ss = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        norm_combine<TPR, MODE, GATE>(p, v, tid, phase, inv, y[v], g[GATE ? v : 0], r[v]);
        ss = square8(r[v], ss);
        if (p.r_out && live) norm_store<TPR, MODE>(p.r_out, p.r_dtype, row * p.ldro, v, tid, p.d, phase, r[v]);
    }
    if (!p.x) return;
    inv = rsqrtf(row_sum<TPR>(ss, part[1]) / (float)p.d + p.eps);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        float w[8];
        norm_load_vec<TPR, MODE>(p.w_pre, SBQ_F32, v, tid, p.d, phase, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) r[v][i] = r[v][i] * inv * w[i];
        if (live) norm_store<TPR, MODE>(p.x, p.x_dtype, row * p.ldx, v, tid, p.d, phase, r[v]);
    }
}

// The same with the row in shared memory: each thread copies the chunks that it will read itself (so that nobody waits for
// another's copies) into 16-byte planes [warp][chunk][plane][lane], and goes over them in rolled loops.  Registers no longer
// grow with the chunks of a thread, so a thread can take several, which share what a row costs besides its elements (sums
// over the CTA, square roots, addresses).
template <bool L1>
__device__ __forceinline__ void stage16(uint4* dst, const void* src) {
    const uint32_t to = (uint32_t)__cvta_generic_to_shared(dst);
    if (L1)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(to), "l"(src) : "memory");
    else
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(src) : "memory");
}

// Requests one chunk of an operand; what lies outside the row is dropped by stage_read.  A chunk of fp32 is a whole
// sector that is copied in two halves: through L1, or it would be fetched twice (8192 x 4096: 119 and 103 us).
template <int MODE>
__device__ __forceinline__ void stage_row(const void* p, int dtype, int64_t row, int64_t ld, int c0, const NormParams& q, uint4* dst) {
    const int64_t at = row * ld + c0;
    if (c0 >= q.d) return;
    bool whole = true;
    if (MODE != kAligned) whole = (c0 >= 0 && c0 + 8 <= q.d) || (at >= 0 && at + 8 <= (q.m - 1) * ld + q.d);
    if (whole) {
        if (dtype == SBQ_F32) {
            stage16<true>(dst, static_cast<const float*>(p) + at);
            stage16<true>(dst + 32, static_cast<const float*>(p) + at + 4);
        } else {
            stage16<false>(dst, static_cast<const uint16_t*>(p) + at);
        }
    } else {
        for (int i = 0; i < 8; ++i) {
            if ((unsigned)(c0 + i) >= (unsigned)q.d) continue;
            if (dtype == SBQ_F32)
                reinterpret_cast<float*>(dst + (i >> 2) * 32)[i & 3] = static_cast<const float*>(p)[at + i];
            else
                reinterpret_cast<uint16_t*>(dst)[i] = static_cast<const uint16_t*>(p)[at + i];
        }
    }
}

template <int MODE>
__device__ __forceinline__ void stage_read(const uint4* src, int dtype, int c0, int d, float (&v)[8]) {
    const uint4 a = src[0];
    if (dtype == SBQ_F32) {
        const uint4 b = src[32];
        const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(u[i]);
    } else {
        unpack8(a, dtype, v);
    }
    if (MODE == kShifted && (c0 < 0 || c0 + 8 > d)) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if ((unsigned)(c0 + i) >= (unsigned)d) v[i] = 0.0f;
    }
}

constexpr int kStagedThreads = 512;
constexpr int kStagedBytes = 220 * 1024, kStagedHalf = 110 * 1024;  // one and two CTAs per SM
template <int MODE, bool GATE>
__global__ void __launch_bounds__(kStagedThreads, 3) norm_staged_kernel(const NormParams p, int chunks, int y_planes, int planes) {
    extern __shared__ uint4 stage[];
    __shared__ float part[2][32];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int tid = threadIdx.x, d = p.d, hop = (int)blockDim.x * 8, step = planes * 32;
    const int64_t row = blockIdx.x;
    const int phase = norm_phase<MODE>(p, row), first = tid * 8 - phase;
    uint4* const mine = stage + (tid >> 5) * chunks * step + (tid & 31);
    const int at_r = y_planes * 32, at_g = at_r + (p.r_dtype == SBQ_F32 ? 64 : 32);
    const bool staged_gate = GATE && p.gcol && p.ldg;
    uint4* s = mine;
    if (p.y)
        for (int v = 0, c = first; v < chunks; ++v, c += hop, s += step) stage_row<MODE>(p.y, p.y_dtype, row, p.ldy, c, p, s);
    asm volatile("cp.async.commit_group;" ::: "memory");
    s = mine;
    for (int v = 0, c = first; v < chunks; ++v, c += hop, s += step) {
        stage_row<MODE>(p.r, p.r_dtype, row, p.ldr, c, p, s + at_r);
        if (staged_gate) stage_row<MODE>(p.gate, p.g_dtype, row, p.ldg, c, p, s + at_g);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    float inv = 1.0f, ss = 0.0f;
    if (p.y && p.w_post) {
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        s = mine;
        for (int v = 0, c = first; v < chunks; ++v, c += hop, s += step) {
            if (c >= d) continue;
            float y[8];
            stage_read<MODE>(s, p.y_dtype, c, d, y);
            ss += square8(y, 0.0f);
        }
        inv = rsqrtf(row_sum<0>(ss, part[0]) / (float)d + p.eps);
        ss = 0.0f;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    s = mine;
    for (int v = 0, c = first; v < chunks; ++v, c += hop, s += step) {
        if (c >= d) continue;
        float y[8], r[8], g[8];
        if (p.y) stage_read<MODE>(s, p.y_dtype, c, d, y);
        stage_read<MODE>(s + at_r, p.r_dtype, c, d, r);
        if (GATE) {
            if (staged_gate)
                stage_read<MODE>(s + at_g, p.g_dtype, c, d, g);
            else
                norm_gate<0, MODE>(p, row, v, tid, phase, g);
        }
        norm_combine<0, MODE, GATE>(p, v, tid, phase, inv, y, g, r);
        ss += square8(r, 0.0f);
        if (p.r_out) norm_store<0, MODE>(p.r_out, p.r_dtype, row * p.ldro, v, tid, d, phase, r);
        if (p.x) {  // r' in fp32 takes the place of the chunk's operands
            s[0] = make_uint4(__float_as_uint(r[0]), __float_as_uint(r[1]), __float_as_uint(r[2]), __float_as_uint(r[3]));
            s[32] = make_uint4(__float_as_uint(r[4]), __float_as_uint(r[5]), __float_as_uint(r[6]), __float_as_uint(r[7]));
        }
    }
    if (!p.x) return;
    inv = rsqrtf(row_sum<0>(ss, part[1]) / (float)d + p.eps);
    s = mine;
    for (int v = 0, c = first; v < chunks; ++v, c += hop, s += step) {
        if (c >= d) continue;
        float r[8], w[8];
        stage_read<kAligned>(s, SBQ_F32, c, d, r);
        norm_load_vec<0, MODE>(p.w_pre, SBQ_F32, v, tid, d, phase, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = r[i] * inv * w[i];
        norm_store<0, MODE>(p.x, p.x_dtype, row * p.ldx, v, tid, d, phase, r);
    }
}

// Rows longer than the registers of one CTA: the row is read again for each statistic (from L2), and
// nothing is written before the last pass, so r_out may be r and x may be y.
constexpr int kLongThreads = 512;
template <int MODE, bool GATE>
__global__ void __launch_bounds__(kLongThreads) norm_long_kernel(const NormParams p) {
    __shared__ float part[2][32];
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    const int phase = norm_phase<MODE>(p, row), chunks = (p.d + phase + kLongThreads * 8 - 1) / (kLongThreads * 8);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    float y[8], r[8], g[8], inv = 1.0f, ss = 0.0f;
    if (p.y && p.w_post) {
        for (int v = 0; v < chunks; ++v) {
            norm_load<0, MODE>(p.y, p.y_dtype, row, p.ldy, v, tid, p, phase, y);
            ss = square8(y, ss);
        }
        inv = rsqrtf(row_sum<0>(ss, part[0]) / (float)p.d + p.eps);
    }
    float inv2 = 1.0f;
    for (int pass = p.x ? 0 : 1; pass < 2; ++pass) {
        ss = 0.0f;
        for (int v = 0; v < chunks; ++v) {
            if (p.y) norm_load<0, MODE>(p.y, p.y_dtype, row, p.ldy, v, tid, p, phase, y);
            norm_load<0, MODE>(p.r, p.r_dtype, row, p.ldr, v, tid, p, phase, r);
            if (GATE) norm_gate<0, MODE>(p, row, v, tid, phase, g);
            norm_combine<0, MODE, GATE>(p, v, tid, phase, inv, y, g, r);
            if (pass == 0) {
                ss = square8(r, ss);
            } else {
                if (p.r_out) norm_store<0, MODE>(p.r_out, p.r_dtype, row * p.ldro, v, tid, p.d, phase, r);
                if (p.x) {
                    norm_load_vec<0, MODE>(p.w_pre, SBQ_F32, v, tid, p.d, phase, y);
#pragma unroll
                    for (int i = 0; i < 8; ++i) r[i] = r[i] * inv2 * y[i];
                    norm_store<0, MODE>(p.x, p.x_dtype, row * p.ldx, v, tid, p.d, phase, r);
                }
            }
        }
        if (pass == 0) inv2 = rsqrtf(row_sum<0>(ss, part[1]) / (float)p.d + p.eps);
    }
}

// TPR = 0: `threads` for each row; otherwise 256 threads for 256 / TPR rows.
template <int TPR, int V, int MAXT, int MODE>
static cudaError_t launch_norm_m(const NormParams& p, int threads, cudaStream_t s) {
    const unsigned grid = (unsigned)(TPR ? ceil_div(p.m, MAXT / (TPR ? TPR : 1)) : p.m);
    return p.gate ? w4_launch(norm_kernel<TPR, V, MAXT, MODE, true>, grid, (unsigned)threads, 0, s, p)
                  : w4_launch(norm_kernel<TPR, V, MAXT, MODE, false>, grid, (unsigned)threads, 0, s, p);
}

template <int TPR, int V, int MAXT>
static cudaError_t launch_norm(const NormParams& p, int mode, int threads, cudaStream_t s) {
    if (mode == kAligned) return launch_norm_m<TPR, V, MAXT, kAligned>(p, threads, s);
    if (mode == kShifted) return launch_norm_m<TPR, V, MAXT, kShifted>(p, threads, s);
    return launch_norm_m<TPR, V, MAXT, kStrided>(p, threads, s);
}

template <int MODE, bool GATE>
static cudaError_t launch_norm_staged_g(const NormParams& p, int threads, int chunks, int planes, cudaStream_t s) {
    static std::atomic<uint64_t> allowed{0};
    const cudaError_t e = w4_allow_smem(norm_staged_kernel<MODE, GATE>, kStagedBytes, allowed);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)p.m);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)threads * chunks * planes * 16;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, norm_staged_kernel<MODE, GATE>, p, chunks, p.y ? (p.y_dtype == SBQ_F32 ? 2 : 1) : 0, planes);
}

template <int MODE>
static cudaError_t launch_norm_staged(const NormParams& p, int threads, int chunks, int planes, cudaStream_t s) {
    return p.gate ? launch_norm_staged_g<MODE, true>(p, threads, chunks, planes, s)
                  : launch_norm_staged_g<MODE, false>(p, threads, chunks, planes, s);
}

template <int MODE>
static cudaError_t launch_norm_long(const NormParams& p, cudaStream_t s) {
    return p.gate ? w4_launch(norm_long_kernel<MODE, true>, (unsigned)p.m, kLongThreads, 0, s, p)
                  : w4_launch(norm_long_kernel<MODE, false>, (unsigned)p.m, kLongThreads, 0, s, p);
}

// In registers, one chunk per thread up to 8192 columns (1024 threads), on as many warps as the row fills: two chunks
// hold twice the registers (8192 x 4096 fp32 with both norms 75 and 78 us).  What hides a row's chain of loads and sums is
// other rows on the SM, so registers are held down to what norm_ctas needs (8192 x 8192 fp32: one CTA per SM 219, two 160 us;
// the gated kernels then spill 24 to 104 bytes a thread, staged ones 32 to 84, which is 2 to 3 % of their instructions).
// Measured on B200, in registers and staged, two norms and a full gate in bf16: 3001 x 2560 22.2 and 19.7 us, 3001 x 2559
// 35.6 and 29.1, 3001 x 6144 58.8 and 44.5, 3001 x 8191 174 and 77, 3001 x 20480 241 and 184; one wave of rows or less is
// faster in registers (592 x 4096 7.7 and 9.8 us: a thread's chunks come one after the other), and so are fp32 rows (3001 x
// 4096 31.9 and 40.4 us).  Weights requested early, persistent CTAs that request their next row early, and one warp
// per row were slower.
static cudaError_t launch_norm_any(const NormParams& p, int mode, cudaStream_t s) {
    const int span = p.d + (mode == kShifted ? 7 : 0);
    // More elements than one wave of full SMs takes at 8 per thread, in rows that are worth several chunks per thread: the
    // staged kernel for 16-bit rows, and for others where the registers leave one CTA per SM.  Two CTAs of it must fit on
    // an SM if the registers do better than one (aligned rows up to 16384 columns).
    if (mode != kStrided && span > 1024 && p.m * p.d > (int64_t)16384 * w4_sm_count()) {
        const bool full_gate = p.gate && p.gcol && p.ldg, y32 = p.y && p.y_dtype == SBQ_F32, r32 = p.r_dtype == SBQ_F32,
                   g32 = full_gate && p.g_dtype == SBQ_F32;
        int planes = 1 + r32 + (p.y != nullptr) + y32 + full_gate + g32;
        planes = planes < 2 ? 2 : planes;  // r' in fp32
        const int pieces = (span + 7) / 8, most = (int)ceil_div(pieces, kStagedThreads), chunks = most < 2 ? 2 : most;
        const int threads = (int)ceil_div(ceil_div(pieces, chunks), 32) * 32;
        const bool wide = y32 || r32 || g32, crowded = span > (mode == kShifted ? 4096 : 8192);
        const int room = mode == kShifted || span > 16384 ? kStagedBytes : kStagedHalf;
        if ((!wide || crowded) && (int64_t)threads * chunks * planes * 16 <= room)
            return mode == kAligned ? launch_norm_staged<kAligned>(p, threads, chunks, planes, s)
                                    : launch_norm_staged<kShifted>(p, threads, chunks, planes, s);
    }
    if (span <= 64) return launch_norm<8, 1, 256>(p, mode, 256, s);
    if (span <= 128) return launch_norm<16, 1, 256>(p, mode, 256, s);
    if (span <= 256) return launch_norm<32, 1, 256>(p, mode, 256, s);
    const int one = (span + 255) / 256 * 32, two = (span + 511) / 512 * 32;  // threads for one or two chunks each
    if (one <= 512) return launch_norm<0, 1, 512>(p, mode, one, s);
    if (one <= 768) return launch_norm<0, 1, 768>(p, mode, one, s);
    if (one <= 1024) return launch_norm<0, 1, 1024>(p, mode, one, s);
    if (two <= 1024) return launch_norm<0, 2, 1024>(p, mode, two, s);
    if (mode == kAligned) return launch_norm_long<kAligned>(p, s);
    if (mode == kShifted) return launch_norm_long<kShifted>(p, s);
    return launch_norm_long<kStrided>(p, s);
}

static bool norm_dtype(int t) { return t == SBQ_F32 || t == SBQ_F16 || t == SBQ_BF16; }

// What the operands' addresses allow: `aligned` 8-element accesses in every row, or rows that all start at the same
// distance past an 8-element boundary (`shifted`; `step`: their stride modulo 8, -1 before the first operand).
struct NormLayout {
    bool aligned = true, shifted = true;
    int step = -1;
};

// One operand: its type, stride and element alignment.  rows: whether it has m rows of d elements (else a vector).
static int check_operand(const void* p, int dtype, int64_t ld, int64_t width, int64_t m, const char* what, NormLayout* l,
                         bool rows) {
    if (!norm_dtype(dtype)) return set_error(SBQ_ERR_UNSUPPORTED, "%s dtype %d (f32, f16, bf16)", what, dtype);
    const int es = w4_elem(dtype);
    if (reinterpret_cast<uintptr_t>(p) % es) return set_error(SBQ_ERR_ALIGNMENT, "%s must be aligned to its element size", what);
    if (m > 1 && ld < width) return set_error(SBQ_ERR_INVALID_ARGUMENT, "%s row stride smaller than the row", what);
    if (reinterpret_cast<uintptr_t>(p) % 16 || (m > 1 && (ld * es) % 16)) l->aligned = false;
    if (rows) {
        const int step = m > 1 ? (int)(ld & 7) : 0;
        if (reinterpret_cast<uintptr_t>(p) % 16 || (l->step >= 0 && l->step != step)) l->shifted = false;
        l->step = step;
    }
    return SBQ_OK;
}

// Each element of a row is read by the thread that writes it, before it does: an output may take the place of an
// operand with the same rows, and share no byte with another.  What every thread of a row reads (a gate per row) or every
// row (weights, a gate per column) lies under no output at all: nothing orders those reads before another thread's stores.
static bool norm_in_the_way(const W4Rows& out, const W4Rows& in, int64_t m) {
    if (!out.p || !in.p || !w4_overlap(out, in, m)) return false;
    return out.p != in.p || (m > 1 && out.ld != in.ld) || out.width != in.width;
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
    NormLayout l;
    l.aligned = d % 8 == 0;
    NormParams p{};
    int st = check_operand(a->residual, a->residual_dtype, a->ld_residual, d, m, "residual", &l, true);
    if (!st && a->branch) st = check_operand(a->branch, a->branch_dtype, a->ld_branch, d, m, "branch", &l, true);
    if (!st && a->residual_out)
        st = check_operand(a->residual_out, a->residual_dtype, a->ld_residual_out, d, m, "residual output", &l, true);
    if (!st && a->out) st = check_operand(a->out, a->out_dtype, a->ld_out, d, m, "output", &l, true);
    if (!st && a->gate) {
        NormLayout any;  // one gate per row sets no condition
        const bool full = a->gate_mode == SBQ_GATE_FULL;
        st = check_operand(a->gate, a->gate_dtype, a->ld_gate, full ? d : 0, full ? m : 1, "gate",
                           a->gate_mode == SBQ_GATE_PER_ROW ? &any : &l, full);
    }
    if (!st && a->pre_weight) st = check_operand(a->pre_weight, SBQ_F32, d, d, 1, "pre_weight", &l, false);
    if (!st && a->post_weight) st = check_operand(a->post_weight, SBQ_F32, d, d, 1, "post_weight", &l, false);
    if (st) return st;
    const auto rows = [&](const void* q, int dtype, int64_t ld) { return W4Rows{q, ld * w4_elem(dtype), d * w4_elem(dtype)}; };
    const W4Rows r = rows(a->residual, a->residual_dtype, a->ld_residual), y = rows(a->branch, a->branch_dtype, a->ld_branch),
                 // one row: a gate per column is a full one
                 g = rows(a->gate_mode == SBQ_GATE_FULL || (a->gate_mode == SBQ_GATE_PER_COLUMN && m == 1) ? a->gate : nullptr,
                          a->gate_dtype, a->ld_gate),
                 ro = rows(a->residual_out, a->residual_dtype, a->ld_residual_out), x = rows(a->out, a->out_dtype, a->ld_out);
    for (const W4Rows* in : {&r, &y, &g})
        if (norm_in_the_way(ro, *in, m) || norm_in_the_way(x, *in, m))
            return set_error(SBQ_ERR_INVALID_ARGUMENT, "an output overlaps an operand with other rows");
    // a gate per row as rows of one element, from the lowest address on; neighbours in memory as one range
    const int64_t gs = w4_elem(a->gate_dtype), gld = m > 1 ? a->ld_gate * gs : gs;
    const W4Rows gate{static_cast<const char*>(a->gate) + (gld < 0 ? (m - 1) * gld : 0), gld < 0 ? -gld : gld, gs};
    for (const W4Rows* out : {&ro, &x}) {
        if (!out->p) continue;
        bool meet = (a->pre_weight && w4_overlap(*out, a->pre_weight, 4 * d, m)) ||
                    (a->post_weight && w4_overlap(*out, a->post_weight, 4 * d, m));
        if (a->gate && a->gate_mode == SBQ_GATE_PER_ROW)
            meet = meet || (gate.ld > gs ? w4_overlap(*out, gate, m) : w4_overlap(*out, gate.p, gate.ld == gs ? m * gs : gs, m));
        if (a->gate && a->gate_mode == SBQ_GATE_PER_COLUMN && m > 1) meet = meet || w4_overlap(*out, a->gate, d * gs, m);
        if (meet) return set_error(SBQ_ERR_INVALID_ARGUMENT, "an output overlaps a weight or a gate");
    }
    if (a->residual_out && a->out && w4_overlap(ro, x, m))
        return set_error(SBQ_ERR_INVALID_ARGUMENT, "the outputs overlap");
    const int mode = l.aligned ? kAligned : l.shifted ? kShifted : kStrided;
    p.y = a->branch, p.r = a->residual, p.gate = a->gate, p.w_post = a->post_weight, p.w_pre = a->pre_weight;
    p.r_out = a->residual_out, p.x = a->out;
    p.ldy = a->ld_branch, p.ldr = a->ld_residual, p.ldro = a->ld_residual_out, p.ldx = a->ld_out;
    p.ldg = a->gate_mode == SBQ_GATE_PER_COLUMN ? 0 : a->ld_gate;
    p.gcol = a->gate_mode != SBQ_GATE_PER_ROW;
    p.y_dtype = a->branch_dtype, p.r_dtype = a->residual_dtype, p.g_dtype = a->gate_dtype, p.x_dtype = a->out_dtype;
    p.act = a->gate_act, p.a = a->residual_scale, p.b = a->branch_scale, p.eps = a->eps;
    p.m = m, p.d = (int)d;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = launch_norm_any(p, mode, s);
    if (e != cudaSuccess) return set_error(SBQ_ERR_CUDA, "residual_norm launch: %s", cudaGetErrorString(e));
    return check_launch("residual_norm");
}
