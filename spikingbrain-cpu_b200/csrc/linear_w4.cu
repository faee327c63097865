// Entry points of the 4-bit format: argument checks, the activation's 16-bit parts, and the choice of
// kernel (decode product up to 16 rows, the tensor-memory product above).
#include <atomic>

#include "w4_host.cuh"

namespace sbq {

// SMs of the current device, cached per device.
int w4_sm_count() {
    static std::atomic<int> count[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    int c = count[dev].load(std::memory_order_relaxed);
    if (c == 0) {
        cudaDeviceGetAttribute(&c, cudaDevAttrMultiProcessorCount, dev);
        c = c > 0 ? c : 148;
        count[dev].store(c, std::memory_order_relaxed);
    }
    return c;
}

// ---- the activation as the kernels read it ------------------------------------------------------------
// fp16 x, and bf16 x up to 16 rows, are read in place when k is a multiple of 16.  Otherwise one launch writes x into
// the workspace, its rows filled with zeros up to a multiple of 16 columns:
//   fp32 x               row r times 2^(14 - e), 2^e <= max |x[r]| < 2^(e + 1) over its finite values, as two fp16 parts
//                        hi + lo (22 bits, the difference x - hi is exact; below 2^-17 of the row's largest 2^-39 of it),
//                        inv[r] = 2^(e - 14);
//   bf16 x, over 16 rows the same in one fp16 part (exact unless an element is below 2^-31 of the row's largest);
//   16-bit x             as it is.
// Infinities and NaN stay what they are.
constexpr int kActThreads = 512;
enum ActSource { kActF32, kActBF16, kActCopy };

struct ActParams {
    const void* x;
    int64_t ldx;
    uint16_t* hi;
    uint16_t* lo;  // fp32 x
    float* inv;    // fp32 and bf16 x
    int k, k16;    // columns of x, and of the parts
    int aligned;   // every 8 columns of x are one (fp32: two) 16-byte accesses, and k = k16
};

// Columns c .. c + 7 of row `row`, zeros past k: fp32 and bf16 as values, other 16-bit types as their bits.
template <int SRC>
__device__ __forceinline__ void act_load8(const ActParams& p, int64_t row, int c, float (&v)[8]) {
    const int64_t at = row * p.ldx + c;
    if (SRC == kActF32) {
        const float* x = static_cast<const float*>(p.x) + at;
        if (p.aligned) {
            const float4 a = reinterpret_cast<const float4*>(x)[0], b = reinterpret_cast<const float4*>(x)[1];
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = c + i < p.k ? x[i] : 0.0f;
        }
    } else {
        const uint16_t* x = static_cast<const uint16_t*>(p.x) + at;
        uint32_t u[8];
        if (p.aligned) {
            const uint4 a = *reinterpret_cast<const uint4*>(x);
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xFFFFu;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = c + i < p.k ? x[i] : 0u;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(SRC == kActBF16 ? u[i] << 16 : u[i]);
    }
}

// One row per CTA.  V chunks of 8 columns per thread stay in registers between the maximum and the conversion; V = 0:
// any k, the row is read twice.
template <int SRC, int V>
__global__ void __launch_bounds__(kActThreads) w4_acts_kernel(const ActParams p) {
    __shared__ float part[kActThreads / 32];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int64_t row = blockIdx.x, o0 = row * p.k16;
    constexpr int kStep = kActThreads * 8;
    float keep[V ? V : 1][8], mul = 1.0f;
    if (V) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = threadIdx.x * 8 + i * kStep;
            if (c < p.k16) act_load8<SRC>(p, row, c, keep[i]);
        }
    }
    if (SRC != kActCopy) {
        float big = 0.0f;
        auto widen = [&](const float (&v)[8]) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (isfinite(v[i])) big = fmaxf(big, fabsf(v[i]));
        };
        if (V) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if ((int)threadIdx.x * 8 + i * kStep < p.k16) widen(keep[i]);
        } else {
            for (int c = threadIdx.x * 8; c < p.k16; c += kStep) {
                act_load8<SRC>(p, row, c, keep[0]);
                widen(keep[0]);
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = big;
        __syncthreads();
        big = part[threadIdx.x & (kActThreads / 32 - 1)];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
        // exponents clamped so that both the factor and its inverse are normal numbers
        int e = big > 0.0f ? 14 - ilogbf(big) : 0;
        e = e > 126 ? 126 : e < -126 ? -126 : e;
        mul = scalbnf(1.0f, e);
        if (threadIdx.x == 0) p.inv[row] = scalbnf(1.0f, -e);
    }
    auto put = [&](const float (&v)[8], int c) {
        uint32_t h[4], l[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (SRC == kActCopy) {
                h[j] = __float_as_uint(v[2 * j]) | __float_as_uint(v[2 * j + 1]) << 16;
                continue;
            }
            const float a = v[2 * j] * mul, b = v[2 * j + 1] * mul;
            const __half2 hh = __floats2half2_rn(a, b);
            h[j] = *reinterpret_cast<const uint32_t*>(&hh);
            if (SRC == kActF32) {
                const float2 hf = __half22float2(hh);
                // an infinity has no low part (inf - inf)
                const __half2 ll = __floats2half2_rn(isinf(a) ? 0.0f : a - hf.x, isinf(b) ? 0.0f : b - hf.y);
                l[j] = *reinterpret_cast<const uint32_t*>(&ll);
            }
        }
        *reinterpret_cast<uint4*>(p.hi + o0 + c) = make_uint4(h[0], h[1], h[2], h[3]);
        if (SRC == kActF32) *reinterpret_cast<uint4*>(p.lo + o0 + c) = make_uint4(l[0], l[1], l[2], l[3]);
    };
    if (V) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = threadIdx.x * 8 + i * kStep;
            if (c < p.k16) put(keep[i], c);
        }
    } else {
        for (int c = threadIdx.x * 8; c < p.k16; c += kStep) {
            act_load8<SRC>(p, row, c, keep[0]);
            put(keep[0], c);
        }
    }
}

template <int SRC>
static cudaError_t launch_acts(const ActParams& p, int64_t m, cudaStream_t s) {
    if (p.k16 <= kActThreads * 8) return w4_launch(w4_acts_kernel<SRC, 1>, (unsigned)m, kActThreads, 0, s, p);
    if (p.k16 <= kActThreads * 24) return w4_launch(w4_acts_kernel<SRC, 3>, (unsigned)m, kActThreads, 0, s, p);
    return w4_launch(w4_acts_kernel<SRC, 0>, (unsigned)m, kActThreads, 0, s, p);
}

constexpr int64_t kW4GemvRows = 16;  // up to this many rows: the decode product

static size_t align256(size_t v) { return (v + 255) & ~size_t(255); }

static int64_t round16(int64_t k) { return (k + 15) / 16 * 16; }

static bool w4_needs_parts(int64_t m, int64_t k, int x_dtype) {
    return x_dtype == SBQ_F32 || (x_dtype == SBQ_BF16 && m > kW4GemvRows) || k % 16 != 0;
}

// x in the workspace and its factors; the factors are read 16 or 32 at a time, up to the end of the last token tile
// (of at most 256).
static size_t act_bytes(int64_t m, int64_t k, int x_dtype) {
    if (!w4_needs_parts(m, k, x_dtype)) return 0;
    return (x_dtype == SBQ_F32 ? 2 : 1) * align256((size_t)m * round16(k) * 2) + (size_t)ceil_div(m + 256, 256) * 1024;
}

static int check_w4_call(const void* x, int x_dtype, int64_t ldx, const W4Call& c, int group, int nmat) {
    if (!x || !c.y) return set_error(SBQ_ERR_INVALID_ARGUMENT, "null pointer");
    for (int i = 0; i < nmat; ++i) {
        if (!c.w[i].packed || !c.w[i].scales || !c.w[i].rowmul) return set_error(SBQ_ERR_INVALID_ARGUMENT, "null pointer");
        if (reinterpret_cast<uintptr_t>(c.w[i].packed) % 256 || reinterpret_cast<uintptr_t>(c.w[i].scales) % 256)
            return set_error(SBQ_ERR_ALIGNMENT, "packed weight and scales must be 256-byte aligned");
    }
    if (c.m <= 0 || c.n <= 0 || c.k <= 0)
        return set_error(SBQ_ERR_INVALID_ARGUMENT, "m, n, k must be positive (m=%lld n=%lld k=%lld)", (long long)c.m,
                         (long long)c.n, (long long)c.k);
    if (!c.gpt) return set_error(SBQ_ERR_UNSUPPORTED, "group size %d (32, 64, 128)", group);
    if (x_dtype != SBQ_F32 && x_dtype != SBQ_F16 && x_dtype != SBQ_BF16)
        return set_error(SBQ_ERR_UNSUPPORTED, "activation dtype %d (f16, bf16, f32)", x_dtype);
    if (c.y_dtype != SBQ_F32 && c.y_dtype != SBQ_F16 && c.y_dtype != SBQ_BF16)
        return set_error(SBQ_ERR_UNSUPPORTED, "output dtype %d (f32, f16, bf16)", c.y_dtype);
    if (ldx < c.k || c.ldy < c.n) return set_error(SBQ_ERR_INVALID_ARGUMENT, "row stride smaller than the row");
    const int xs = w4_elem(x_dtype);
    if (c.k % 16 == 0 && (reinterpret_cast<uintptr_t>(x) % 16 || (c.m > 1 && (ldx * xs) % 16)))
        return set_error(SBQ_ERR_ALIGNMENT, "activation rows must be 16-byte aligned (k a multiple of 16)");
    if (reinterpret_cast<uintptr_t>(x) % xs) return set_error(SBQ_ERR_ALIGNMENT, "activation must be aligned to its element size");
    if (reinterpret_cast<uintptr_t>(c.y) % w4_elem(c.y_dtype))
        return set_error(SBQ_ERR_ALIGNMENT, "output must be aligned to its element size");
    for (int i = 0; i < nmat; ++i)
        if (reinterpret_cast<uintptr_t>(c.w[i].rowmul) % 4) return set_error(SBQ_ERR_ALIGNMENT, "rowmul must be 4-byte aligned");
    if (reinterpret_cast<uintptr_t>(c.bias) % 4) return set_error(SBQ_ERR_ALIGNMENT, "bias must be 4-byte aligned");
    if (c.n > (int64_t(1) << 31) - 256 || c.k >= (int64_t(1) << 30) || c.m > (int64_t(1) << 31) - 256)
        return set_error(SBQ_ERR_UNSUPPORTED, "shape too large");
    const int ys = w4_elem(c.y_dtype);  // one CTA may store its part of y while another still reads x
    if (w4_overlap({x, ldx * xs, c.k * xs}, {c.y, c.ldy * ys, c.n * ys}, c.m))
        return set_error(SBQ_ERR_INVALID_ARGUMENT, "output and activation must not overlap");
    return SBQ_OK;
}

static int w4_run(const void* x, int x_dtype, int64_t ldx, W4Call c, int group, int nmat, void* workspace,
                  size_t workspace_bytes) {
    int st = check_w4_call(x, x_dtype, ldx, c, group, nmat);
    if (st) return st;
    const size_t need = sbq_linear_w4_workspace_bytes(c.m, c.n, c.k, x_dtype, nmat), acts = act_bytes(c.m, c.k, x_dtype);
    if (need) {
        if (!workspace) return set_error(SBQ_ERR_INVALID_ARGUMENT, "this call needs a workspace of %zu bytes", need);
        if (reinterpret_cast<uintptr_t>(workspace) % 256)
            return set_error(SBQ_ERR_ALIGNMENT, "workspace must be 256-byte aligned");
        if (workspace_bytes < need) return set_error(SBQ_ERR_WORKSPACE, "workspace needs %zu bytes", need);
    }
    W4Acts a{};
    a.bf16 = x_dtype == SBQ_BF16;
    a.part[0] = x;
    a.ld = ldx;
    a.scratch = static_cast<uint8_t*>(workspace) + acts;
    const int64_t k16 = round16(c.k);
    if (acts) {
        const size_t one = align256((size_t)c.m * k16 * 2);
        uint8_t* ws = static_cast<uint8_t*>(workspace);
        const bool f32 = x_dtype == SBQ_F32, scaled = f32 || (x_dtype == SBQ_BF16 && c.m > kW4GemvRows);
        ActParams p{};
        p.x = x;
        p.ldx = ldx;
        p.hi = reinterpret_cast<uint16_t*>(ws);
        p.lo = f32 ? reinterpret_cast<uint16_t*>(ws + one) : nullptr;
        p.inv = scaled ? reinterpret_cast<float*>(ws + (f32 ? 2 : 1) * one) : nullptr;
        p.k = (int)c.k;
        p.k16 = (int)k16;
        p.aligned = c.k == k16;  // rows 16-byte aligned then (checked)
        const cudaError_t e = f32      ? launch_acts<kActF32>(p, c.m, c.stream)
                              : scaled ? launch_acts<kActBF16>(p, c.m, c.stream)
                                       : launch_acts<kActCopy>(p, c.m, c.stream);
        if (e != cudaSuccess) return set_error(SBQ_ERR_CUDA, "w4 activation launch: %s", cudaGetErrorString(e));
        a.part[0] = p.hi;
        a.part[1] = p.lo;
        a.ld = k16;
        a.inv = p.inv;
        if (scaled) a.bf16 = false;
    }
    c.k = k16;  // the weight's columns past k are zeros, in the same tiles
    return c.m <= kW4GemvRows ? gemv_w4_run(c, a) : gemm_w4_run(c, a);
}

}  // namespace sbq

using namespace sbq;

extern "C" size_t sbq_linear_w4_workspace_bytes(int64_t m, int64_t n, int64_t k, int x_dtype, int matrices) {
    if (m <= 0 || n <= 0 || k <= 0) return 0;
    return act_bytes(m, k, x_dtype) + (m > kW4GemvRows ? gemm_w4_workspace(m, n, round16(k), x_dtype == SBQ_F32, matrices == 2 ? 2 : 1) : 0);
}

extern "C" int sbq_linear_w4_plan(int64_t m, int64_t n, int64_t k, int x_dtype, int matrices, int* plan) {
    if (!plan) return set_error(SBQ_ERR_INVALID_ARGUMENT, "null pointer");
    if (m <= 0 || n <= 0 || k <= 0) return set_error(SBQ_ERR_INVALID_ARGUMENT, "m, n, k must be positive");
    plan[0] = plan[2] = plan[3] = 0;
    plan[1] = 8;
    if (m > kW4GemvRows)
        gemm_w4_plan(m, n, round16(k), x_dtype == SBQ_F32, matrices == 2 ? 2 : 1, plan);
    else if (m > 8)
        plan[1] = 16;
    return SBQ_OK;
}

extern "C" int sbq_linear_w4(const void* x, int x_dtype, int64_t ldx, const void* packed, const void* scales,
                             const float* rowmul, int group, const float* bias, int64_t m, int64_t n, int64_t k, void* y,
                             int y_dtype, int64_t ldy, void* workspace, size_t workspace_bytes, void* stream) {
    W4Call c{};
    c.w[0] = {static_cast<const uint8_t*>(packed), static_cast<const __nv_bfloat16*>(scales), rowmul};
    c.gpt = w4_groups_per_tile(group);
    c.bias = bias;
    c.m = m, c.n = n, c.k = k;
    c.y = y, c.y_dtype = y_dtype, c.ldy = ldy;
    c.stream = static_cast<cudaStream_t>(stream);
    return w4_run(x, x_dtype, ldx, c, group, 1, workspace, workspace_bytes);
}

extern "C" int sbq_mlp_gateup_w4(const void* x, int x_dtype, int64_t ldx, const void* packed_gate,
                                 const void* scales_gate, const float* rowmul_gate, const void* packed_up,
                                 const void* scales_up, const float* rowmul_up, int group, int64_t m, int64_t n, int64_t k,
                                 void* h, int h_dtype, int64_t ldh, void* workspace, size_t workspace_bytes, void* stream) {
    W4Call c{};
    c.w[0] = {static_cast<const uint8_t*>(packed_gate), static_cast<const __nv_bfloat16*>(scales_gate), rowmul_gate};
    c.w[1] = {static_cast<const uint8_t*>(packed_up), static_cast<const __nv_bfloat16*>(scales_up), rowmul_up};
    c.gpt = w4_groups_per_tile(group);
    c.m = m, c.n = n, c.k = k;
    c.y = h, c.y_dtype = h_dtype, c.ldy = ldh;
    c.stream = static_cast<cudaStream_t>(stream);
    return w4_run(x, x_dtype, ldx, c, group, 2, workspace, workspace_bytes);
}
