// Preparation of 4-bit weights: quantisation by group on the device, packing of given codes, and back.
//
// For each output channel and group of `group` input features:
//   s = bf16(max(max|w|, 1e-8) / 7)              (fp32 division, then one rounding to bf16)
//   q = clamp(rint(w / s), -7, 7)                (fp32 division, ties to even)
// The scale is rounded before q is taken, so q fits the scale that is stored: |w| / s is at most
// 7 (1 + 2^-8), which rounds to 7.  A bf16 scale is enough (its rounding is 2^-8 of a step that is
// itself 1/14 of the group's range) and makes q * s exact in fp16 up to a power of two (w4.cuh).
// A group that holds an infinity or a NaN has no scale: it gets NaN, and so do the results of its row.
#include "w4.cuh"

namespace sbq {

template <typename T>
__device__ __forceinline__ float w4_f32(T v);
template <>
__device__ __forceinline__ float w4_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float w4_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float w4_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

constexpr int kPackThreads = 128;

// The larger of two values, NaN if either is (fmaxf would drop it).
__device__ __forceinline__ float w4_max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// The power of two that brings m (the row's largest |scale|) into [2^10, 2^11).
__device__ __forceinline__ float w4_rowmul(float m) {
    if (!(m > 0.0f) || !isfinite(m)) return 1.0f;
    int e = 10 - ilogbf(m);
    e = e > 126 ? 126 : e;
    return scalbnf(1.0f, e);
}

__device__ __forceinline__ void w4_store_rowmul(float smax, float* rowmul) {
    __shared__ float part[kPackThreads / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) smax = fmaxf(smax, __shfl_xor_sync(0xffffffffu, smax, o));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = smax;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < kPackThreads / 32; ++i) smax = fmaxf(smax, part[i]);
        *rowmul = w4_rowmul(smax);
    }
}

// One CTA per packed row (rows past n are written as zeros), one thread per 8 columns; the threads of a
// group are neighbouring lanes.
template <typename T>
__global__ void __launch_bounds__(kPackThreads) w4_quantize_kernel(const T* __restrict__ w, int64_t n, int64_t k,
                                                                   int64_t ldw, int group, uint8_t* __restrict__ packed,
                                                                   __nv_bfloat16* __restrict__ scales,
                                                                   float* __restrict__ rowmul) {
    const int64_t r = blockIdx.x, kt_total = w4_tiles_k(k), words = kt_total * 16;
    const int lanes = group / 8, gpt = w4_groups_per_tile(group);
    float smax = 0.0f;
    // whole warps run together (words is a multiple of 16: the second half of a warp may be past the end)
    for (int64_t c0 = 0; c0 < words; c0 += kPackThreads) {
        const int64_t c8 = c0 + threadIdx.x;
        float v[8], amax = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t c = c8 * 8 + i;
            v[i] = (r < n && c < k) ? w4_f32(w[r * ldw + c]) : 0.0f;
            amax = w4_max_nan(amax, fabsf(v[i]));
        }
        for (int o = lanes >> 1; o > 0; o >>= 1) amax = w4_max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if (isinf(amax)) amax = __int_as_float(0x7FC00000);
        const bool real = r < n && c8 / lanes * group < k;  // the group has columns of the weight
        const __nv_bfloat16 sb = __float2bfloat16_rn(real ? __fdiv_rn(w4_max_nan(amax, 1e-8f), 7.0f) : 0.0f);
        const float s = __bfloat162float(sb);
        smax = fmaxf(smax, s);
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            int q = 0;
            if (real) q = (int)fminf(fmaxf(rintf(__fdiv_rn(v[i], s)), -7.0f), 7.0f);
            word |= (uint32_t)(q + 8) << (4 * (i >> 1) + 16 * (i & 1));
        }
        if (c8 < words) {
            *reinterpret_cast<uint32_t*>(packed + w4_word_offset(r, c8, kt_total)) = word;
            if (c8 % lanes == 0) scales[w4_scale_index(r, c8 / lanes, kt_total, gpt)] = sb;
        }
    }
    w4_store_rowmul(smax, rowmul + r);
}

// Given codes and scales (row strides ldq, lds) -> packed.  Codes outside [-8, 7] are clamped to it.
__global__ void __launch_bounds__(kPackThreads) w4_pack_kernel(const int8_t* __restrict__ q, int64_t ldq,
                                                               const __nv_bfloat16* __restrict__ s, int64_t lds,
                                                               int64_t n, int64_t k, int group,
                                                               uint8_t* __restrict__ packed,
                                                               __nv_bfloat16* __restrict__ scales,
                                                               float* __restrict__ rowmul) {
    const int64_t r = blockIdx.x, kt_total = w4_tiles_k(k), words = kt_total * 16;
    const int lanes = group / 8, gpt = w4_groups_per_tile(group);
    float smax = 0.0f;
    for (int64_t c8 = threadIdx.x; c8 < words; c8 += kPackThreads) {
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t c = c8 * 8 + i;
            int v = (r < n && c < k) ? (int)q[r * ldq + c] : 0;
            v = v < -8 ? -8 : v > 7 ? 7 : v;
            word |= (uint32_t)(v + 8) << (4 * (i >> 1) + 16 * (i & 1));
        }
        *reinterpret_cast<uint32_t*>(packed + w4_word_offset(r, c8, kt_total)) = word;
        if (c8 % lanes == 0) {
            const int64_t gi = c8 / lanes;
            const bool real = r < n && gi * group < k;
            const __nv_bfloat16 sb = real ? s[r * lds + gi] : __float2bfloat16_rn(0.0f);
            scales[w4_scale_index(r, gi, kt_total, gpt)] = sb;
            smax = fmaxf(smax, fabsf(__bfloat162float(sb)));
        }
    }
    w4_store_rowmul(smax, rowmul + r);
}

// Packed -> codes [n, k] and scales [n, ceil(k / group)] (either may be null).
__global__ void __launch_bounds__(kPackThreads) w4_unpack_kernel(const uint8_t* __restrict__ packed,
                                                                 const __nv_bfloat16* __restrict__ scales, int64_t n,
                                                                 int64_t k, int group, int8_t* __restrict__ q,
                                                                 int64_t ldq, __nv_bfloat16* __restrict__ s,
                                                                 int64_t lds) {
    const int64_t r = blockIdx.x, kt_total = w4_tiles_k(k);
    const int gpt = w4_groups_per_tile(group);
    if (q) {
        for (int64_t c8 = threadIdx.x; c8 * 8 < k; c8 += kPackThreads) {
            const uint32_t word = *reinterpret_cast<const uint32_t*>(packed + w4_word_offset(r, c8, kt_total));
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c8 * 8 + i < k)
                    q[r * ldq + c8 * 8 + i] = (int8_t)((int)((word >> (4 * (i >> 1) + 16 * (i & 1))) & 15u) - 8);
        }
    }
    if (s) {
        for (int64_t gi = threadIdx.x; gi * group < k; gi += kPackThreads)
            s[r * lds + gi] = scales[w4_scale_index(r, gi, kt_total, gpt)];
    }
}

static bool off_element(const void* p, size_t size) { return reinterpret_cast<uintptr_t>(p) % size != 0; }

static int check_w4_pack(const void* a, const void* packed, const void* scales, int64_t n, int64_t k, int64_t ld,
                         int group) {
    if (!a || !packed || !scales) return set_error(SBQ_ERR_INVALID_ARGUMENT, "null pointer");
    if (n <= 0 || k <= 0)
        return set_error(SBQ_ERR_INVALID_ARGUMENT, "n and k must be positive (n=%lld k=%lld)", (long long)n, (long long)k);
    if (!w4_groups_per_tile(group)) return set_error(SBQ_ERR_UNSUPPORTED, "group size %d (32, 64, 128)", group);
    if (ld < k) return set_error(SBQ_ERR_INVALID_ARGUMENT, "row stride %lld < k %lld", (long long)ld, (long long)k);
    if (reinterpret_cast<uintptr_t>(packed) % 256 || reinterpret_cast<uintptr_t>(scales) % 256)
        return set_error(SBQ_ERR_ALIGNMENT, "packed weight and scales must be 256-byte aligned");
    if (n > (int64_t(1) << 31) - 16 || k >= (int64_t(1) << 30)) return set_error(SBQ_ERR_UNSUPPORTED, "weight too large");
    return SBQ_OK;
}

}  // namespace sbq

using namespace sbq;

extern "C" size_t sbq_w4_packed_bytes(int64_t n, int64_t k) {
    if (n <= 0 || k <= 0) return 0;
    return (size_t)(ceil_div(n, kTileRows) * w4_tiles_k(k) * kW4TileBytes);
}

extern "C" size_t sbq_w4_scale_bytes(int64_t n, int64_t k, int group) {
    if (n <= 0 || k <= 0) return 0;
    return (size_t)(ceil_div(n, kTileRows) * w4_tiles_k(k)) * 32 * w4_groups_per_tile(group);
}

extern "C" int sbq_w4_quantize_pack(const void* w, int w_dtype, int64_t n, int64_t k, int64_t ldw, int group,
                                    void* packed, void* scales, float* rowmul, void* stream) {
    int st = check_w4_pack(w, packed, scales, n, k, ldw, group);
    if (st) return st;
    if (!rowmul) return set_error(SBQ_ERR_INVALID_ARGUMENT, "null rowmul pointer");
    if (off_element(w, w_dtype == SBQ_F32 ? 4 : 2) || off_element(rowmul, 4))
        return set_error(SBQ_ERR_ALIGNMENT, "weight and rowmul must be aligned to their element size");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const unsigned grid = (unsigned)(ceil_div(n, kTileRows) * kTileRows);
    uint8_t* out = static_cast<uint8_t*>(packed);
    __nv_bfloat16* sc = static_cast<__nv_bfloat16*>(scales);
    switch (w_dtype) {
        case SBQ_F32:
            w4_quantize_kernel<float><<<grid, kPackThreads, 0, s>>>(static_cast<const float*>(w), n, k, ldw, group, out, sc, rowmul);
            break;
        case SBQ_F16:
            w4_quantize_kernel<__half><<<grid, kPackThreads, 0, s>>>(static_cast<const __half*>(w), n, k, ldw, group, out, sc, rowmul);
            break;
        case SBQ_BF16:
            w4_quantize_kernel<__nv_bfloat16>
                <<<grid, kPackThreads, 0, s>>>(static_cast<const __nv_bfloat16*>(w), n, k, ldw, group, out, sc, rowmul);
            break;
        default:
            return set_error(SBQ_ERR_UNSUPPORTED, "weight dtype %d not supported (f32, f16, bf16)", w_dtype);
    }
    return packed_launch("w4_quantize_pack", s);
}

extern "C" int sbq_w4_pack(const int8_t* q, int64_t ldq, const void* scale, int64_t lds, int64_t n, int64_t k,
                           int group, void* packed, void* scales, float* rowmul, void* stream) {
    int st = check_w4_pack(q, packed, scales, n, k, ldq, group);
    if (st) return st;
    if (!scale || !rowmul) return set_error(SBQ_ERR_INVALID_ARGUMENT, "null pointer");
    if (off_element(scale, 2) || off_element(rowmul, 4))
        return set_error(SBQ_ERR_ALIGNMENT, "scale and rowmul must be aligned to their element size");
    if (lds < ceil_div(k, group)) return set_error(SBQ_ERR_INVALID_ARGUMENT, "scale row stride smaller than the row");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    w4_pack_kernel<<<(unsigned)(ceil_div(n, kTileRows) * kTileRows), kPackThreads, 0, s>>>(
        q, ldq, static_cast<const __nv_bfloat16*>(scale), lds, n, k, group, static_cast<uint8_t*>(packed),
        static_cast<__nv_bfloat16*>(scales), rowmul);
    return packed_launch("w4_pack", s);
}

extern "C" int sbq_w4_unpack(const void* packed, const void* scales, int64_t n, int64_t k, int group, int8_t* q,
                             int64_t ldq, void* scale, int64_t lds, void* stream) {
    int st = check_w4_pack(packed, packed, scales, n, k, q ? ldq : k, group);
    if (st) return st;
    if (scale && lds < ceil_div(k, group)) return set_error(SBQ_ERR_INVALID_ARGUMENT, "scale row stride smaller than the row");
    if (off_element(scale, 2)) return set_error(SBQ_ERR_ALIGNMENT, "scale must be aligned to its element size");
    if (!q && !scale) return SBQ_OK;
    w4_unpack_kernel<<<(unsigned)n, kPackThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const uint8_t*>(packed), static_cast<const __nv_bfloat16*>(scales), n, k, group, q, ldq,
        static_cast<__nv_bfloat16*>(scale), lds);
    return check_launch("w4_unpack");
}
