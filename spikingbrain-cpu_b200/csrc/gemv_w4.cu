// Decode product of 4-bit weights with group scales, and its fused gate/up form:
//
//   y[m, n] = sum_g s[n, g] * (sum_{k in g} x[m, k] q[n, k]) (+ bias[n])         m <= 16
//   h[m, n] = silu(gate[m, n]) * up[m, n], gate and up as y with their own weights
//
// One warp takes a 16-channel tile row (or every W-th 128-column tile of it): per tile two 16-byte loads
// of codes per lane, q in fp16 or bf16 (exact integers), m16n8k16 tensor-core products with the rows
// of x as the n dimension, fp32 partial sums per group that are scaled and added in fp32.  So the
// weight takes part exactly and every sum is fp32.
#include <atomic>

#include "w4.cuh"
#include "w4_host.cuh"

namespace sbq {

constexpr int kG4Warps = 8;
constexpr int kG4Threads = kG4Warps * 32;

struct GemvW4Params {
    const void* x[2];        // 16-bit activation [m, k]; x[1]: low part of a split fp32 activation
    int64_t ldx;
    const float* xinv;       // per row factor of a split activation, or null
    const uint8_t* w[2];     // codes (gate and up of the fused form)
    const uint32_t* s[2];    // scales, row pairs (w4.cuh)
    const float* bias;
    void* y;
    int64_t ldy;
    int y_dtype;
    int m, n, k;
    int kt_total;            // 128-column tiles
    int tile_rows;
    int wsplit;              // warps per tile row (a power of two up to 8)
};

template <int MT>
struct XFrag4 {
    uint4 v[MT][4];  // [row block][word]: 8 consecutive columns of row 8 * block + g
};

// One word (8 columns x rows g, g + 8): two k16 products per row block.
template <bool BF16, int MT, int PARTS>
__device__ __forceinline__ void w4_word_mma(float (&part)[MT][4], uint32_t wa, uint32_t wb, int w,
                                            const XFrag4<MT> (&xf)[PARTS]) {
    uint32_t a[4], b[4];
    if (BF16) {
        w4_to_bf16(wa, a);
        w4_to_bf16(wb, b);
    } else {
        w4_to_half(wa, a);
        w4_to_half(wb, b);
    }
#pragma unroll
    for (int p = 0; p < PARTS; ++p)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const uint4 v = xf[p].v[mt][w];
            if (BF16) {
                mma_bf16(part[mt], a[0], b[0], a[1], b[1], v.x, v.y);
                mma_bf16(part[mt], a[2], b[2], a[3], b[3], v.z, v.w);
            } else {
                mma_f16(part[mt], a[0], b[0], a[1], b[1], v.x, v.y);
                mma_f16(part[mt], a[2], b[2], a[3], b[3], v.z, v.w);
            }
        }
}

template <bool BF16, int MT, int PARTS, int NMAT, int GPT>
__global__ void __launch_bounds__(kG4Threads) gemv_w4_kernel(const GemvW4Params p) {
    __shared__ float red[kG4Warps][NMAT][MT * 8][17];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int W = p.wsplit, rows_per_cta = kG4Warps / W;
    const int tr = blockIdx.x * rows_per_cta + warp / W, ks = warp % W;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    float acc[NMAT][MT][4];
#pragma unroll
    for (int a = 0; a < NMAT; ++a)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[a][mt][e] = 0.0f;
    if (tr < p.tile_rows) {
        for (int kt = ks; kt < p.kt_total; kt += W) {
            const int64_t tile = (int64_t)tr * p.kt_total + kt;
            XFrag4<MT> xf[PARTS];
#pragma unroll
            for (int q = 0; q < PARTS; ++q)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const int row = 8 * mt + g, c = kt * kW4TileCols + 32 * w + 8 * t;
                        xf[q].v[mt][w] = make_uint4(0, 0, 0, 0);
                        if (row < p.m && c < p.k)
                            xf[q].v[mt][w] = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.x[q]) +
                                                                             ((int64_t)row * p.ldx + c) * 2);
                    }
#pragma unroll
            for (int a = 0; a < NMAT; ++a) {
                const uint8_t* src = p.w[a] + tile * kW4TileBytes + lane * 16;
                const uint4 wa = ld_stream(src), wb = ld_stream(src + 512);
                const uint32_t wa_[4] = {wa.x, wa.y, wa.z, wa.w}, wb_[4] = {wb.x, wb.y, wb.z, wb.w};
#pragma unroll
                for (int gi = 0; gi < GPT; ++gi) {
                    float part[MT][4];
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) part[mt][e] = 0.0f;
#pragma unroll
                    for (int w = gi * (4 / GPT); w < (gi + 1) * (4 / GPT); ++w)
                        w4_word_mma<BF16, MT, PARTS>(part, wa_[w], wb_[w], w, xf);
                    const uint32_t sc = __ldg(p.s[a] + (tile * 8 + g) * GPT + gi);
                    const float s0 = __uint_as_float(sc << 16), s1 = __uint_as_float(sc & 0xFFFF0000u);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        acc[a][mt][0] = fmaf(s0, part[mt][0], acc[a][mt][0]);
                        acc[a][mt][1] = fmaf(s0, part[mt][1], acc[a][mt][1]);
                        acc[a][mt][2] = fmaf(s1, part[mt][2], acc[a][mt][2]);
                        acc[a][mt][3] = fmaf(s1, part[mt][3], acc[a][mt][3]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int a = 0; a < NMAT; ++a)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e) red[warp][a][8 * mt + 2 * t + (e & 1)][g + 8 * (e >> 1)] = acc[a][mt][e];
    __syncthreads();
    for (int e = threadIdx.x; e < rows_per_cta * MT * 8 * 16; e += kG4Threads) {
        const int r = e & 15, tl = (e >> 4) % rows_per_cta, tok = (e >> 4) / rows_per_cta;
        const int64_t n = (int64_t)(blockIdx.x * rows_per_cta + tl) * 16 + r;
        if (tok >= p.m || n >= p.n) continue;
        float v[NMAT];
#pragma unroll
        for (int a = 0; a < NMAT; ++a) {
            v[a] = 0.0f;
            for (int w = 0; w < W; ++w) v[a] += red[tl * W + w][a][tok][r];
            if (p.xinv) v[a] *= p.xinv[tok];
        }
        float out = v[0];
        if (NMAT == 2)
            out = w4_silu(v[0]) * v[NMAT - 1];
        else if (p.bias)
            out += p.bias[n];
        w4_store(p.y, p.y_dtype, (int64_t)tok * p.ldy + n, out);
    }
}

template <bool BF16, int MT, int PARTS, int NMAT>
static cudaError_t launch_gemv_w4(const GemvW4Params& p, int gpt, cudaStream_t s) {
    const unsigned grid = (unsigned)ceil_div(p.tile_rows, kG4Warps / p.wsplit);
    switch (gpt) {
        case 1: return w4_launch(gemv_w4_kernel<BF16, MT, PARTS, NMAT, 1>, grid, kG4Threads, 0, s, p);
        case 2: return w4_launch(gemv_w4_kernel<BF16, MT, PARTS, NMAT, 2>, grid, kG4Threads, 0, s, p);
        default: return w4_launch(gemv_w4_kernel<BF16, MT, PARTS, NMAT, 4>, grid, kG4Threads, 0, s, p);
    }
}

template <int MT, int NMAT>
static cudaError_t launch_gemv_w4_x(const GemvW4Params& p, bool bf16, bool split, int gpt, cudaStream_t s) {
    if (split) return launch_gemv_w4<false, MT, 2, NMAT>(p, gpt, s);
    if (bf16) return launch_gemv_w4<true, MT, 1, NMAT>(p, gpt, s);
    return launch_gemv_w4<false, MT, 1, NMAT>(p, gpt, s);
}

int gemv_w4_run(const W4Call& c, const W4Acts& x) {
    for (int64_t m0 = 0; m0 < c.m; m0 += 16) {
        GemvW4Params p{};
        p.m = (int)(c.m - m0 < 16 ? c.m - m0 : 16);
        p.ldx = x.ld;
        for (int i = 0; i < 2; ++i) p.x[i] = x.part[i] ? static_cast<const uint8_t*>(x.part[i]) + m0 * x.ld * 2 : nullptr;
        p.xinv = x.inv ? x.inv + m0 : nullptr;
        for (int i = 0; i < 2; ++i) {
            p.w[i] = c.w[i].packed;
            p.s[i] = reinterpret_cast<const uint32_t*>(c.w[i].scales);
        }
        p.bias = c.bias;
        p.y = static_cast<uint8_t*>(c.y) + m0 * c.ldy * w4_elem(c.y_dtype);
        p.ldy = c.ldy;
        p.y_dtype = c.y_dtype;
        p.n = (int)c.n;
        p.k = (int)c.k;
        p.kt_total = (int)w4_tiles_k(c.k);
        p.tile_rows = (int)ceil_div(c.n, kTileRows);
        p.wsplit = 1;
        while (p.wsplit < 8 && p.tile_rows * (int64_t)p.wsplit < (int64_t)w4_sm_count() * 16 && 2 * p.wsplit <= p.kt_total)
            p.wsplit *= 2;
        const bool two = c.w[1].packed != nullptr, bf16 = x.bf16, split = x.part[1] != nullptr;
        cudaError_t e;
        if (p.m > 8)
            e = two ? launch_gemv_w4_x<2, 2>(p, bf16, split, c.gpt, c.stream) : launch_gemv_w4_x<2, 1>(p, bf16, split, c.gpt, c.stream);
        else
            e = two ? launch_gemv_w4_x<1, 2>(p, bf16, split, c.gpt, c.stream) : launch_gemv_w4_x<1, 1>(p, bf16, split, c.gpt, c.stream);
        if (e != cudaSuccess) return set_error(SBQ_ERR_CUDA, "gemv_w4 launch: %s", cudaGetErrorString(e));
    }
    return check_launch("gemv_w4");
}

}  // namespace sbq
