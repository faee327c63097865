// What the 4-bit entry points and kernels share on the host, and the device helpers of their epilogues.
#pragma once

#include <atomic>

#include "w4.cuh"

namespace sbq {

// One checked call of sbq_linear_w4 (w[1] null) or sbq_mlp_gateup_w4.
struct W4Call {
    W4Weight w[2];
    int gpt;  // groups per 128-column tile
    const float* bias;
    int64_t m, n, k;
    void* y;
    int y_dtype;
    int64_t ldy;
    cudaStream_t stream;
};

// The activation as the kernels read it: 16-bit parts [m, k] with row stride ld.  fp16 and bf16 inputs
// are read in place; the parts of an fp32 input (and of a bf16 input above 16 rows) are fp16 made by
// w4_acts_kernel, each row multiplied by a power of two whose inverse is inv[row].
struct W4Acts {
    const void* part[2];
    int64_t ld;
    const float* inv;
    bool bf16;
    void* scratch;  // gemm_w4_workspace bytes
};

int gemv_w4_run(const W4Call& c, const W4Acts& x);  // up to 16 rows
int gemm_w4_run(const W4Call& c, const W4Acts& x);  // fp16 parts only
size_t gemm_w4_workspace(int64_t m, int64_t n, int64_t k, bool split, int nmat);
void gemm_w4_plan(int64_t m, int64_t n, int64_t k, bool split, int nmat, int* plan);
int w4_sm_count();

inline int w4_elem(int dtype) { return dtype == SBQ_F32 ? 4 : 2; }

// m rows of `width` bytes, `ld` bytes apart.
struct W4Rows {
    const void* p;
    int64_t ld, width;
};

// Whether rows of a and b share a byte.  Columns of one buffer (same ld) do not, however their ranges interleave; with
// different strides, ranges that meet count as shared.
inline bool w4_overlap(const W4Rows& a, const W4Rows& b, int64_t m) {
    const intptr_t pa = reinterpret_cast<intptr_t>(a.p), pb = reinterpret_cast<intptr_t>(b.p);
    if (pa + (m - 1) * a.ld + a.width <= pb || pb + (m - 1) * b.ld + b.width <= pa) return false;
    if (m == 1 || a.ld != b.ld || a.ld <= 0) return true;
    const int64_t off = ((pb - pa) % a.ld + a.ld) % a.ld;
    return off < a.width || off + b.width > a.ld;
}

// Whether one of m rows shares a byte with the `bytes` bytes at q.
inline bool w4_overlap(const W4Rows& a, const void* q, int64_t bytes, int64_t m) {
    const int64_t off = reinterpret_cast<intptr_t>(q) - reinterpret_cast<intptr_t>(a.p);
    if (off + bytes <= 0 || off >= (m - 1) * a.ld + a.width) return false;
    if (off < 0 || m == 1 || a.ld <= 0) return true;
    const int64_t at = off % a.ld;  // behind the start of the row before it, and then before the start of the next one
    return at < a.width || at + bytes > a.ld;
}

// Lets a kernel use `bytes` of dynamic shared memory on the current device: once per kernel and device (`done`, the
// kernel's own), since the call costs as much host time as a tenth of a launch.
template <class K>
cudaError_t w4_allow_smem(K kernel, int bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
    if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    const cudaError_t s = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (s == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return s;
}

// A launch as a programmatic dependent of the previous kernel on the stream.  Each kernel launched
// this way reads nothing but packed weights before its griddepcontrol.wait and lets its own dependents
// begin only after that wait.
template <class K, class P>
cudaError_t w4_launch(K kernel, dim3 grid, unsigned block, size_t smem, cudaStream_t s, const P& p) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

__device__ __forceinline__ float w4_silu(float v) { return v / (1.0f + expf(-v)); }

__device__ __forceinline__ void w4_store(void* y, int dtype, int64_t i, float v) {
    if (dtype == SBQ_F32)
        static_cast<float*>(y)[i] = v;
    else if (dtype == SBQ_F16)
        static_cast<__half*>(y)[i] = __float2half_rn(v);
    else
        static_cast<__nv_bfloat16*>(y)[i] = __float2bfloat16_rn(v);
}

}  // namespace sbq
