// Product of 4-bit weights with group scales for more than 16 rows of x, and its fused gate/up form, on
// the fifth-generation tensor cores:
//
//   y[t, n] = xinv[t] / rowmul[n] * sum_k xh[t, k] * (q[n, k] s[n, k / group] rowmul[n])  (+ bias[n])
//
// xh is x in fp16 (x itself, or its power-of-two-scaled parts, linear_w4.cu), and q * s * rowmul is exact in
// fp16 (w4.cuh), so the products are those of the definition and the sums are fp32 in tensor memory.
//
// Channels are the MMA's M, tokens its N.  Per 128 columns of k (one packed tile):
//   * warp 0 (one thread) loads the tokens' x (TMA, 128-byte swizzle), the codes (64 bytes per channel, 64-byte
//     swizzle, so that 32 rows read 16 bytes each without bank conflicts) and the scales into a ring of stages;
//   * warps 4-11, two converter warpgroups taking alternate k-blocks, one channel per thread, turn the codes
//     into scaled fp16 weights and write them to tensor memory (the MMA's A operand, a ring of its own);
//   * warp 1 (one thread) issues tcgen05.mma, A from tensor memory, x from shared memory.
//
// Conversion: a code moved to bits 6..9 under the fp16 exponent of 16 reads as 16 + u, and
// (16 + u) * s - 24 * s = q * s is one fused multiply-add: 24 * s is exact (2 + 8 bits), the result too.  With a
// shift and a mask per pair of columns that is 3 instructions for 2 weights.
//
// Tensor-core accumulation truncates: measured on B200, the relative error of a sum grows by about 1.3e-8 per
// k16 step (1.2e-5 at k = 12288).  Where the result is kept in fp32 the sum is therefore cut into segments
// of 32 steps (kSegSteps) that alternate between two accumulators; the converter warps add each finished
// segment to fp32 registers (round to nearest) while the other one fills.  128-token tiles have room
// for that (64 sums per thread), 256-token tiles, which read half the weight per product, do not, and
// serve 16-bit results, whose own rounding (2^-12 and up) is far above it.
#include "tc.cuh"
#include "w4_host.cuh"

namespace sbq {

constexpr int kW4Threads = 384;   // producer, MMA, tensor-memory, idle warp, two converter warpgroups
constexpr int kW4Rows = 128;      // channels (tensor-memory lanes) per CTA
constexpr int kSegSteps = 32;     // MMA steps per accumulation segment

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
            tc::smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(tc::smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}

struct GemmW4Params {
    int m, n, kt, parts;
    const float* rowmul[2];
    const float* bias;
    const float* xinv;
    void* y;
    int64_t ldy;
    int y_dtype;
};

// Sizes of one kernel.  XROWS: tokens of x this CTA loads per stage; N: the MMA's tokens.
template <int XROWS, int N, int PARTS, bool SEG, int TMEM, int RING>
struct W4Shape {
    static constexpr int kXSub = XROWS * 128;               // 64 columns of k: a 128-byte row per token
    static constexpr int kXBytes = 2 * PARTS * kXSub;       // [64-column half][part]
    static constexpr int kCodes = kW4Rows * 64;
    static constexpr int kStage = kXBytes + kCodes + 1024;  // scales: at most 1 KiB
    static constexpr int kStages = RING / kStage < 8 ? RING / kStage : 8;
    static constexpr int kACol = SEG ? 2 * N : N;            // accumulator(s) first
    static constexpr int kABufs0 = (TMEM - kACol) / 64;
    static constexpr int kABufs = kABufs0 < kStages ? kABufs0 : kStages;  // 64 columns per 128 k
    static constexpr int kSegBlocks = kSegSteps / (8 * PARTS);
    static constexpr int kBarOff = kStages * kStage;
    static constexpr int kBytes = kBarOff + 512 + kW4Rows * 8 + 1024;
    static_assert(kStages >= 2 && kABufs >= 2, "pipeline depth");
    static_assert((4 * kStages + 4) * 8 + 4 <= 512, "barriers");
    static_assert(kBytes <= 227 * 1024, "shared memory");
};

// One channel's 128 codes (64 bytes of row `row`, 64-byte swizzle) -> words 16 w + 4 t + i = columns
// 32 w + 8 t + 2 i, + 1 of the scaled fp16 weight.  `half` 0 / 1: the words of columns 0..63 / 64..127.
template <int GPT>
__device__ __forceinline__ void w4_convert_half(const uint4 (&raw)[4], const uint32_t (&s2)[GPT], const uint32_t (&c2)[GPT],
                                                int half, uint32_t (&h)[32]) {
#pragma unroll
    for (int w2 = 0; w2 < 2; ++w2)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const uint32_t v = half ? (w2 ? raw[t].w : raw[t].z) : (w2 ? raw[t].y : raw[t].x);
            const int gi = (2 * half + w2) * GPT / 4;
            uint32_t* o = h + 16 * w2 + 4 * t;
            o[0] = hfma2(lop3_and_or(v << 6, 0x03C003C0u, 0x4C004C00u), s2[gi], c2[gi]);
            o[1] = hfma2(lop3_and_or(v << 2, 0x03C003C0u, 0x4C004C00u), s2[gi], c2[gi]);
            o[2] = hfma2(lop3_and_or(v >> 2, 0x03C003C0u, 0x4C004C00u), s2[gi], c2[gi]);
            o[3] = hfma2(lop3_and_or(v >> 6, 0x03C003C0u, 0x4C004C00u), s2[gi], c2[gi]);
        }
}

// A converter thread's stage: codes and scales of channel `row` -> 64 tensor-memory columns.
template <int GPT>
__device__ __forceinline__ void w4_convert_stage(const uint8_t* codes, const uint8_t* scales, int row, float rowmul,
                                                 uint32_t tmem_dst) {
    uint32_t s2[GPT], c2[GPT];
#pragma unroll
    for (int gi = 0; gi < GPT; ++gi) {
        const uint16_t u = *reinterpret_cast<const uint16_t*>(
            scales + (((row >> 4) * 8 + (row & 7)) * GPT + gi) * 4 + ((row >> 3) & 1) * 2);
        const __half2 s = __float2half2_rn(__uint_as_float((uint32_t)u << 16) * rowmul);
        s2[gi] = *reinterpret_cast<const uint32_t*>(&s);
        const __half2 c = __hmul2(s, __float2half2_rn(-24.0f));
        c2[gi] = *reinterpret_cast<const uint32_t*>(&c);
    }
    uint4 raw[4];
#pragma unroll
    for (int t = 0; t < 4; ++t)
        raw[t] = *reinterpret_cast<const uint4*>(codes + row * 64 + ((t ^ ((row >> 1) & 3)) << 4));
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        uint32_t h[32];
        w4_convert_half<GPT>(raw, s2, c2, half, h);
        tc::tmem_st_32x32b_x32(tmem_dst + half * 32, h);
    }
}

// Adds `COLS` accumulator columns at `taddr` to a thread's sums (FIRST: takes them).
template <int COLS>
__device__ __forceinline__ void w4_take_segment(uint32_t taddr, float (&sum)[COLS], bool first) {
#pragma unroll
    for (int c = 0; c < COLS / 32; ++c) {
        uint32_t r[32];
        tc::tmem_ld_32x32b_x32(taddr + c * 32, r);
        tc::tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            const float v = __uint_as_float(r[j]);
            sum[32 * c + j] = first ? v : sum[32 * c + j] + v;
        }
    }
}

// Channel of tensor-memory lane `row` (CTA's first channel n0): with two matrices lanes 0..63 are the
// gate's channels n0.., lanes 64..127 the up projection's.
template <int NMAT>
__device__ __forceinline__ int w4_channel(int n0, int row) { return n0 + (NMAT == 2 ? row & 63 : row); }

// Up to 128 named-barrier threads of one converter warpgroup.
__device__ __forceinline__ void group_sync(int grp) { asm volatile("bar.sync %0, 128;" ::"r"(1 + grp) : "memory"); }

// Epilogue of one 32-token slice: v holds lane `row`'s sums of tokens tb.., already scaled.  With two matrices
// the up lanes hand theirs over through `xch` ([token][64]) and the gate lanes finish.
template <int NMAT>
__device__ __forceinline__ void w4_finish(const GemmW4Params& p, const float (&v)[32], int tb, int n, int row, int grp,
                                          float bias, float* xch, bool ok) {
    if (NMAT == 2) {
        if (row >= 64) {
#pragma unroll
            for (int j = 0; j < 32; ++j) xch[j * 64 + (row & 63)] = v[j];
        }
        group_sync(grp);
        if (row < 64 && n < p.n && ok) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (tb + j < p.m) w4_store(p.y, p.y_dtype, (int64_t)(tb + j) * p.ldy + n, w4_silu(v[j]) * xch[j * 64 + row]);
        }
        group_sync(grp);
    } else if (n < p.n && ok) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (tb + j < p.m) w4_store(p.y, p.y_dtype, (int64_t)(tb + j) * p.ldy + n, v[j] + bias);
    }
}

// ---------------------------------------------------------------------------------------------
// More than 128 rows: CTA pairs (cta_group::2), 256 channels x TOK tokens per pair.  Each CTA converts its own
// 128 channels and loads half of the tokens.  SEG (TOK 128): segmented sums.
// ---------------------------------------------------------------------------------------------
template <int TOK, int PARTS>
using W4Pair = W4Shape<TOK / 2, TOK, PARTS, TOK == 128, 512, 224 * 1024>;

template <int TOK, int PARTS, int NMAT, int GPT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kW4Threads, 1)
    gemm_w4_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_lo,
                        const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_w2,
                        const __grid_constant__ CUtensorMap map_s, const __grid_constant__ CUtensorMap map_s2,
                        const __grid_constant__ GemmW4Params p) {
    using S = W4Pair<TOK, PARTS>;
    constexpr bool SEG = TOK == 128;
    constexpr int NS = S::kStages, NA = S::kABufs, COLS = TOK / 2;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* wfull = reinterpret_cast<uint64_t*>(smem + S::kBarOff);  // this CTA's codes and scales landed
    uint64_t* ready = wfull + NS;      // leader: both CTAs' x landed and both CTAs' converters wrote
    uint64_t* conv_done = ready + NS;  // this CTA's converters have read the codes
    uint64_t* mma_done = conv_done + NS;
    uint64_t* done = mma_done + NS;    // per accumulator: its segment's (without segments: all) MMAs completed
    uint64_t* taken = done + 2;        // leader, per accumulator: both CTAs' converters have added it up
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(taken + 2);
    float* s_mul = reinterpret_cast<float*>(smem + S::kBarOff + 512);
    float* s_bias = s_mul + kW4Rows;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = tc::cluster_ctarank();
    const bool leader = rank == 0;
    constexpr int kCh = kW4Rows / NMAT;
    const int n0 = (int)blockIdx.x * kCh, t0 = blockIdx.y * TOK;

    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; ++s) {
            tc::mbar_init(&wfull[s], 1);
            tc::mbar_init(&ready[s], 1 + 8);
            tc::mbar_init(&conv_done[s], 4);
            tc::mbar_init(&mma_done[s], 1);
        }
        tc::mbar_init(&done[0], 1);
        tc::mbar_init(&done[1], 1);
        tc::mbar_init(&taken[0], 16);
        tc::mbar_init(&taken[1], 16);
        tc::fence_mbar_init();
        tc::prefetch_tmap(&map_x);
        tc::prefetch_tmap(&map_w);
        tc::prefetch_tmap(&map_s);
    }
    if (warp == 2) {
        tc::tmem_alloc_pair(tmem_slot, 512);
        tc::tmem_relinquish_pair();
    }
    for (int i = threadIdx.x; i < kW4Rows; i += blockDim.x) {
        const int n = w4_channel<NMAT>(n0, i);
        s_mul[i] = n < p.n ? p.rowmul[NMAT == 2 ? i >> 6 : 0][n] : 1.0f;
        s_bias[i] = p.bias && n < p.n ? p.bias[n] : 0.0f;
    }
    tc::fence_before_sync();
    tc::cluster_sync();
    tc::fence_after_sync();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            const int tr = t0 + (int)rank * (TOK / 2);
            auto load_w = [&](int kb) {
                const int s = kb % NS;
                uint8_t* ws = smem + s * S::kStage + S::kXBytes;
                tc::mbar_arrive_expect_tx(&wfull[s], S::kCodes + 256 * GPT);
                tc::tma_load_4d(ws, &map_w, &wfull[s], 0, 0, kb, n0 / 16);
                tma_load_3d(ws + S::kCodes, &map_s, &wfull[s], 0, kb, n0 / 16);
                if (NMAT == 2) {
                    tc::tma_load_4d(ws + S::kCodes / 2, &map_w2, &wfull[s], 0, 0, kb, n0 / 16);
                    tma_load_3d(ws + S::kCodes + 128 * GPT, &map_s2, &wfull[s], 0, kb, n0 / 16);
                }
            };
            auto load_x = [&](int kb) {
                const int s = kb % NS;
                uint8_t* xs = smem + s * S::kStage;
                const uint32_t xb = tc::cluster_addr(&ready[s], 0);
                if (leader) tc::mbar_arrive_expect_tx(&ready[s], 2 * S::kXBytes);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    tc::tma_load_2d_pair(xs + h * PARTS * S::kXSub, &map_x, xb, kb * 128 + h * 64, tr);
                    if (PARTS == 2) tc::tma_load_2d_pair(xs + (h * PARTS + 1) * S::kXSub, &map_lo, xb, kb * 128 + h * 64, tr);
                }
            };
            const int pre = p.kt < NS ? p.kt : NS;
            for (int kb = 0; kb < pre; ++kb) load_w(kb);
            asm volatile("griddepcontrol.wait;" ::: "memory");
            asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
            for (int kb = 0; kb < pre; ++kb) load_x(kb);
            for (int kb = pre; kb < p.kt; ++kb) {
                const int s = kb % NS;
                const uint32_t ph = (kb / NS) & 1;
                if (!tc::mbar_wait(&conv_done[s], ph ^ 1)) break;
                if (!tc::mbar_wait(&mma_done[s], ph ^ 1)) break;
                load_w(kb);
                load_x(kb);
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && leader) {
            constexpr uint32_t idesc = tc::idesc_f16(2 * kW4Rows, TOK, false);
            for (int kb = 0; kb < p.kt; ++kb) {
                const int s = kb % NS, seg = SEG ? kb / S::kSegBlocks : 0;
                const bool fresh = SEG ? kb % S::kSegBlocks == 0 : kb == 0;
                if (SEG && fresh && seg >= 2 && !tc::mbar_wait_cluster(&taken[seg & 1], ((seg >> 1) - 1) & 1)) break;
                if (!tc::mbar_wait_cluster(&ready[s], (kb / NS) & 1)) break;
                tc::fence_after_sync();
                const uint8_t* xs = smem + s * S::kStage;
                const uint32_t d = tmem + (seg & 1) * TOK, a = tmem + S::kACol + (kb % NA) * 64;
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int q = 0; q < PARTS; ++q) {
                        const uint64_t bd = tc::smem_desc(xs + ((j >> 2) * PARTS + q) * S::kXSub + (j & 3) * 32, tc::kSwizzle128B, 1024);
                        tc::mma_f16_ts_pair(d, a + j * 8, bd, idesc, !(fresh && j == 0 && q == 0));
                    }
                tc::mma_commit_pair(tc::cluster_addr(&mma_done[s], 0));
                tc::mma_commit_pair(tc::cluster_addr(&mma_done[s], 1));
                if (kb + 1 == p.kt || (SEG && (kb + 1) % S::kSegBlocks == 0)) {
                    tc::mma_commit_pair(tc::cluster_addr(&done[seg & 1], 0));
                    tc::mma_commit_pair(tc::cluster_addr(&done[seg & 1], 1));
                }
            }
        }
    } else if (warp >= 4) {
        const int grp = (warp - 4) >> 2, wq = (warp - 4) & 3, row = wq * 32 + lane;
        const uint32_t lane_tmem = tmem + ((uint32_t)(wq * 32) << 16);
        const float mul = s_mul[row];
        float sum[SEG ? COLS : 32];
        int taken_segs = 0;
        // the next segment: waits for its MMAs.  A segment's accumulator is filled again only after it was
        // taken, so its barrier is never more than one phase ahead.
        auto take = [&]() -> bool {
            if constexpr (SEG) {
                if (!__all_sync(0xffffffffu, tc::mbar_wait(&done[taken_segs & 1], (taken_segs >> 1) & 1))) return false;
                tc::fence_after_sync();
                w4_take_segment<COLS>(lane_tmem + (taken_segs & 1) * TOK + grp * COLS, sum, taken_segs == 0);
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive_cluster(tc::cluster_addr(&taken[taken_segs & 1], 0));
                ++taken_segs;
            }
            return true;
        };
        bool ok = true;
        for (int kb = grp; kb < p.kt; kb += 2) {
            const int s = kb % NS;
            // the operand buffer was last read by k-block kb - NA; waiting for its MMAs also puts every
            // earlier phase of this stage's barriers behind us (NA <= NS), so a parity names one phase
            if (kb >= NA) {
                const int prev = kb - NA;
                if (!__all_sync(0xffffffffu, tc::mbar_wait(&mma_done[prev % NS], (prev / NS) & 1))) { ok = false; break; }
            }
            if (!__all_sync(0xffffffffu, tc::mbar_wait(&wfull[s], (kb / NS) & 1))) { ok = false; break; }
            tc::fence_after_sync();
            const uint8_t* codes = smem + s * S::kStage + S::kXBytes;
            w4_convert_stage<GPT>(codes, codes + S::kCodes, row, mul, lane_tmem + S::kACol + (kb % NA) * 64);
            tc::tmem_wait_st();
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                tc::mbar_arrive_cluster(tc::cluster_addr(&ready[s], 0));
                tc::mbar_arrive(&conv_done[s]);
            }
            // a segment is taken NA blocks after its last one: its MMAs are done by then (the wait above), and
            // the MMAs of the segment after the next, which need its accumulator, are not due yet
            if (SEG && kb - NA + 1 >= (taken_segs + 1) * S::kSegBlocks && !(ok = take())) break;
        }
        if constexpr (SEG) {
            while (ok && taken_segs * S::kSegBlocks < p.kt) ok = take();
        } else {
            ok = __all_sync(0xffffffffu, ok && tc::mbar_wait(&done[0], 0));
            tc::fence_after_sync();
        }
        asm volatile("griddepcontrol.wait;" ::: "memory");  // before y is written, and xinv read
        const int n = w4_channel<NMAT>(n0, row);
        const float inv = 1.0f / mul, bias = s_bias[row];
        float* xch = reinterpret_cast<float*>(smem) + grp * 32 * 64;
        // every MMA of the pair is done, so the ring is free for the exchange
#pragma unroll
        for (int c = 0; c < COLS / 32; ++c) {
            const int tb = t0 + grp * COLS + c * 32;
            float v[32];
            if constexpr (SEG) {
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = sum[32 * c + j] * inv;
            } else {
                uint32_t r[32];
                tc::tmem_ld_32x32b_x32(lane_tmem + grp * COLS + c * 32, r);
                tc::tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]) * inv;
            }
            if (p.xinv) {
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] *= tb + j < p.m ? p.xinv[tb + j] : 0.0f;
            }
            w4_finish<NMAT>(p, v, tb, n, row, grp, bias, xch, ok);
        }
    }
    tc::fence_before_sync();
    tc::cluster_sync();
    if (warp == 2) {
        tc::fence_after_sync();
        tc::tmem_dealloc_pair(tmem, 512);
    }
}

// ---------------------------------------------------------------------------------------------
// 17..128 rows: 128 channels x 64 tokens per CTA, two CTAs per SM, k split over the CTAs of a cluster when
// the tiles alone are too few: each pushes its fp32 sums into the shared memory of the CTA that owns the
// channel, which adds them in part order.
// ---------------------------------------------------------------------------------------------
constexpr int kSTok4 = 64;
template <int PARTS>
using W4Small = W4Shape<kSTok4, kSTok4, PARTS, true, 256, 108 * 1024>;

template <int PARTS, int NMAT, int GPT>
__global__ void __launch_bounds__(kW4Threads, 2)
    gemm_w4_small_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_lo,
                         const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_w2,
                         const __grid_constant__ CUtensorMap map_s, const __grid_constant__ CUtensorMap map_s2,
                         const __grid_constant__ GemmW4Params p) {
    using S = W4Small<PARTS>;
    constexpr int NS = S::kStages, NA = S::kABufs;
    static_assert(2 * (S::kBytes + 1024) <= 228 * 1024, "two CTAs per SM");
    static_assert(kSTok4 * kW4Rows * 4 <= S::kBarOff, "the receive buffer fits in the ring");
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* wfull = reinterpret_cast<uint64_t*>(smem + S::kBarOff);
    uint64_t* ready = wfull + NS;
    uint64_t* conv_done = ready + NS;
    uint64_t* mma_done = conv_done + NS;
    uint64_t* done = mma_done + NS;
    uint64_t* taken = done + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(taken + 2);
    float* s_mul = reinterpret_cast<float*>(smem + S::kBarOff + 512);
    float* s_bias = s_mul + kW4Rows;
    float* recv = reinterpret_cast<float*>(smem);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kCh = kW4Rows / NMAT;
    const int n0 = (int)blockIdx.x * kCh, t0 = blockIdx.y * kSTok4;
    const int part = p.parts > 1 ? (int)tc::cluster_ctarank() : 0;
    const int kb0 = part * p.kt / p.parts, nkb = (part + 1) * p.kt / p.parts - kb0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; ++s) {
            tc::mbar_init(&wfull[s], 1);
            tc::mbar_init(&ready[s], 1 + 4);
            tc::mbar_init(&conv_done[s], 4);
            tc::mbar_init(&mma_done[s], 1);
        }
        tc::mbar_init(&done[0], 1);
        tc::mbar_init(&done[1], 1);
        tc::mbar_init(&taken[0], 8);
        tc::mbar_init(&taken[1], 8);
        tc::fence_mbar_init();
        tc::prefetch_tmap(&map_x);
        tc::prefetch_tmap(&map_w);
        tc::prefetch_tmap(&map_s);
    }
    if (warp == 2) {
        tc::tmem_alloc(tmem_slot, 256);
        tc::tmem_relinquish();
    }
    for (int i = threadIdx.x; i < kW4Rows; i += blockDim.x) {
        const int n = w4_channel<NMAT>(n0, i);
        s_mul[i] = n < p.n ? p.rowmul[NMAT == 2 ? i >> 6 : 0][n] : 1.0f;
        s_bias[i] = p.bias && n < p.n ? p.bias[n] : 0.0f;
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    float sum[32];

    if (warp == 0) {
        if (lane == 0) {
            auto load_w = [&](int i) {
                const int s = i % NS, kb = kb0 + i;
                uint8_t* ws = smem + s * S::kStage + S::kXBytes;
                tc::mbar_arrive_expect_tx(&wfull[s], S::kCodes + 256 * GPT);
                tc::tma_load_4d(ws, &map_w, &wfull[s], 0, 0, kb, n0 / 16);
                tma_load_3d(ws + S::kCodes, &map_s, &wfull[s], 0, kb, n0 / 16);
                if (NMAT == 2) {
                    tc::tma_load_4d(ws + S::kCodes / 2, &map_w2, &wfull[s], 0, 0, kb, n0 / 16);
                    tma_load_3d(ws + S::kCodes + 128 * GPT, &map_s2, &wfull[s], 0, kb, n0 / 16);
                }
            };
            auto load_x = [&](int i) {
                const int s = i % NS, kb = kb0 + i;
                uint8_t* xs = smem + s * S::kStage;
                tc::mbar_arrive_expect_tx(&ready[s], S::kXBytes);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    tc::tma_load_2d(xs + h * PARTS * S::kXSub, &map_x, &ready[s], kb * 128 + h * 64, t0);
                    if (PARTS == 2) tc::tma_load_2d(xs + (h * PARTS + 1) * S::kXSub, &map_lo, &ready[s], kb * 128 + h * 64, t0);
                }
            };
            const int pre = nkb < NS ? nkb : NS;
            for (int i = 0; i < pre; ++i) load_w(i);
            asm volatile("griddepcontrol.wait;" ::: "memory");
            asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
            for (int i = 0; i < pre; ++i) load_x(i);
            for (int i = pre; i < nkb; ++i) {
                const int s = i % NS;
                const uint32_t ph = (i / NS) & 1;
                if (!tc::mbar_wait(&conv_done[s], ph ^ 1)) break;
                if (!tc::mbar_wait(&mma_done[s], ph ^ 1)) break;
                load_w(i);
                load_x(i);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = tc::idesc_f16(kW4Rows, kSTok4, false);
            for (int i = 0; i < nkb; ++i) {
                const int s = i % NS, seg = i / S::kSegBlocks;
                const bool fresh = i % S::kSegBlocks == 0;
                if (fresh && seg >= 2 && !tc::mbar_wait(&taken[seg & 1], ((seg >> 1) - 1) & 1)) break;
                if (!tc::mbar_wait(&ready[s], (i / NS) & 1)) break;
                tc::fence_after_sync();
                const uint8_t* xs = smem + s * S::kStage;
                const uint32_t d = tmem + (seg & 1) * kSTok4, a = tmem + S::kACol + (i % NA) * 64;
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int q = 0; q < PARTS; ++q) {
                        const uint64_t bd = tc::smem_desc(xs + ((j >> 2) * PARTS + q) * S::kXSub + (j & 3) * 32, tc::kSwizzle128B, 1024);
                        tc::mma_f16_ts(d, a + j * 8, bd, idesc, !(fresh && j == 0 && q == 0));
                    }
                tc::mma_commit(&mma_done[s]);
                if (i + 1 == nkb || (i + 1) % S::kSegBlocks == 0) tc::mma_commit(&done[seg & 1]);
            }
        }
    } else if (warp >= 4) {
        const int grp = (warp - 4) >> 2, wq = (warp - 4) & 3, row = wq * 32 + lane;
        const uint32_t lane_tmem = tmem + ((uint32_t)(wq * 32) << 16);
        const float mul = s_mul[row];
        int taken_segs = 0;
#pragma unroll
        for (int j = 0; j < 32; ++j) sum[j] = 0.0f;
        auto take = [&]() -> bool {
            if (!__all_sync(0xffffffffu, tc::mbar_wait(&done[taken_segs & 1], (taken_segs >> 1) & 1))) return false;
            tc::fence_after_sync();
            w4_take_segment<32>(lane_tmem + (taken_segs & 1) * kSTok4 + grp * 32, sum, false);
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&taken[taken_segs & 1]);
            ++taken_segs;
            return true;
        };
        bool ok = true;
        for (int i = grp; i < nkb; i += 2) {
            const int s = i % NS;
            if (i >= NA) {
                const int prev = i - NA;
                if (!__all_sync(0xffffffffu, tc::mbar_wait(&mma_done[prev % NS], (prev / NS) & 1))) { ok = false; break; }
            }
            if (!__all_sync(0xffffffffu, tc::mbar_wait(&wfull[s], (i / NS) & 1))) { ok = false; break; }
            tc::fence_after_sync();
            const uint8_t* codes = smem + s * S::kStage + S::kXBytes;
            w4_convert_stage<GPT>(codes, codes + S::kCodes, row, mul, lane_tmem + S::kACol + (i % NA) * 64);
            tc::tmem_wait_st();
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                tc::mbar_arrive(&ready[s]);
                tc::mbar_arrive(&conv_done[s]);
            }
            if (i - NA + 1 >= (taken_segs + 1) * S::kSegBlocks && !(ok = take())) break;
        }
        while (ok && taken_segs * S::kSegBlocks < nkb) ok = take();
        asm volatile("griddepcontrol.wait;" ::: "memory");  // before y is written, and xinv read
        const float inv = 1.0f / mul;
#pragma unroll
        for (int j = 0; j < 32; ++j) sum[j] *= inv;
        if (p.parts == 1) {
            const int tb = t0 + grp * 32;
            if (p.xinv) {
#pragma unroll
                for (int j = 0; j < 32; ++j) sum[j] *= tb + j < p.m ? p.xinv[tb + j] : 0.0f;
            }
            w4_finish<NMAT>(p, sum, tb, w4_channel<NMAT>(n0, row), row, grp, s_bias[row], recv + grp * 32 * 64, ok);
        }
    }
    if (p.parts > 1) {
        // (1) every CTA of the cluster has left its main loop, so every ring is free; (2) sums go to the owner of
        // the channel, [part][token][matrix][owner's channel], neighbouring lanes next to each other; (3) the
        // owner adds them in part order.
        tc::cluster_sync();
        const int share = kCh / p.parts;  // a power of two, at least 8
        if (warp >= 4) {
            const int grp = (warp - 4) >> 2, row = ((warp - 4) & 3) * 32 + lane;
            const int mat = NMAT == 2 ? row >> 6 : 0, c = NMAT == 2 ? row & 63 : row, owner = c / share;
            const uint32_t dst = tc::cluster_addr(recv + ((part * kSTok4 + grp * 32) * NMAT + mat) * share + c % share, (uint32_t)owner);
#pragma unroll
            for (int j = 0; j < 32; ++j)
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + (uint32_t)(j * NMAT * share * 4)), "f"(sum[j]) : "memory");
        }
        tc::cluster_sync();
        asm volatile("griddepcontrol.wait;" ::: "memory");
        for (int e = threadIdx.x; e < share * kSTok4; e += blockDim.x) {
            const int c = e % share, t = e / share, ch = part * share + c, n = n0 + ch;
            if (t0 + t >= p.m || n >= p.n) continue;
            float v[NMAT];
#pragma unroll
            for (int a = 0; a < NMAT; ++a) {
                v[a] = 0.0f;
                for (int q = 0; q < p.parts; ++q) v[a] += recv[((q * kSTok4 + t) * NMAT + a) * share + c];
                if (p.xinv) v[a] *= p.xinv[t0 + t];
            }
            const float out = NMAT == 2 ? w4_silu(v[0]) * v[NMAT - 1] : v[0] + s_bias[ch];
            w4_store(p.y, p.y_dtype, (int64_t)(t0 + t) * p.ldy + n, out);
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    if (warp == 2) {
        tc::fence_after_sync();
        tc::tmem_dealloc(tmem, 256);
    }
}

SBQ_DEFINE_ERROR_POLL(poll_error_w4)

struct W4Maps {
    CUtensorMap x, lo, w[2], s[2];
};

static int make_maps(W4Maps& m, const W4Call& c, const W4Acts& x, int x_rows) {
    const uint64_t xd[2] = {(uint64_t)c.k, (uint64_t)c.m}, xs[1] = {(uint64_t)x.ld * 2};
    const uint32_t xb[2] = {64, (uint32_t)x_rows};
    int st = encode_tmap(&m.x, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, x.part[0], xd, xs, xb, CU_TENSOR_MAP_SWIZZLE_128B);
    m.lo = m.x;
    if (!st && x.part[1]) st = encode_tmap(&m.lo, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, x.part[1], xd, xs, xb, CU_TENSOR_MAP_SWIZZLE_128B);
    const int nmat = c.w[1].packed ? 2 : 1;
    const uint64_t kt = (uint64_t)w4_tiles_k(c.k), nt = (uint64_t)ceil_div(c.n, kTileRows), sb = 32 * (uint64_t)c.gpt;
    const uint32_t rows = kW4Rows / 16 / nmat;
    for (int i = 0; i < nmat && !st; ++i) {
        const uint64_t wd[4] = {64, 16, kt, nt}, ws[3] = {64, 1024, kt * 1024};
        const uint32_t wb[4] = {64, 16, 1, rows};
        st = encode_tmap(&m.w[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, c.w[i].packed, wd, ws, wb, CU_TENSOR_MAP_SWIZZLE_64B);
        const uint64_t sd[3] = {sb, kt, nt}, ss[2] = {sb, kt * sb};
        const uint32_t bb[3] = {(uint32_t)sb, 1, rows};
        if (!st) st = encode_tmap(&m.s[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, c.w[i].scales, sd, ss, bb, CU_TENSOR_MAP_SWIZZLE_NONE);
    }
    if (nmat == 1) m.w[1] = m.w[0], m.s[1] = m.s[0];
    return st;
}

template <class K>
static cudaError_t launch_maps(K kernel, dim3 grid, int smem, int parts, cudaStream_t s, const W4Maps& m, const GemmW4Params& p) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kW4Threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;  // the pair kernel has its own compiled in
    attr[1].val.clusterDim.x = 1;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = (unsigned)parts;
    cfg.attrs = attr;
    cfg.numAttrs = parts > 0 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, m.x, m.lo, m.w[0], m.w[1], m.s[0], m.s[1], p);
}

template <int PARTS, int NMAT, int GPT>
static cudaError_t launch_gemm_w4(int tok, const W4Maps& m, const GemmW4Params& p, cudaStream_t s) {
    constexpr int kCh = kW4Rows / NMAT;
    if (tok == kSTok4)
        return launch_maps(gemm_w4_small_kernel<PARTS, NMAT, GPT>,
                           dim3((unsigned)ceil_div(p.n, kCh), (unsigned)ceil_div(p.m, kSTok4), (unsigned)p.parts),
                           W4Small<PARTS>::kBytes, p.parts, s, m, p);
    const unsigned gx = 2 * (unsigned)ceil_div(p.n, 2 * kCh);
    if (tok == 128)
        return launch_maps(gemm_w4_pair_kernel<128, PARTS, NMAT, GPT>, dim3(gx, (unsigned)ceil_div(p.m, 128)),
                           W4Pair<128, PARTS>::kBytes, 0, s, m, p);
    return launch_maps(gemm_w4_pair_kernel<256, PARTS, NMAT, GPT>, dim3(gx, (unsigned)ceil_div(p.m, 256)),
                       W4Pair<256, PARTS>::kBytes, 0, s, m, p);
}

template <int PARTS, int NMAT>
static cudaError_t launch_gemm_w4_g(int gpt, int tok, const W4Maps& m, const GemmW4Params& p, cudaStream_t s) {
    if (gpt == 1) return launch_gemm_w4<PARTS, NMAT, 1>(tok, m, p, s);
    if (gpt == 2) return launch_gemm_w4<PARTS, NMAT, 2>(tok, m, p, s);
    return launch_gemm_w4<PARTS, NMAT, 4>(tok, m, p, s);
}

constexpr int64_t kW4SmallRows = 128;

int gemm_w4_run(const W4Call& c, const W4Acts& x) {
    const int nmat = c.w[1].packed ? 2 : 1, ch = kW4Rows / nmat, sms = w4_sm_count();
    GemmW4Params p{};
    p.m = (int)c.m;
    p.n = (int)c.n;
    p.kt = (int)w4_tiles_k(c.k);
    p.parts = 1;
    p.rowmul[0] = c.w[0].rowmul;
    p.rowmul[1] = c.w[1].rowmul;
    p.bias = c.bias;
    p.xinv = x.inv;
    p.y = c.y;
    p.ldy = c.ldy;
    p.y_dtype = c.y_dtype;
    int tok;
    if (c.m <= kW4SmallRows) {
        tok = kSTok4;
        // k parts: the largest power of two up to 8 that keeps the grid within 7/8 of the CTA slots (two per
        // SM; a cluster needs all of its CTAs at once) and gives every part at least two tiles
        const int64_t tiles = ceil_div(c.n, ch) * ceil_div(c.m, kSTok4);
        while (p.parts < 8 && tiles * (2 * p.parts) * 8 <= (int64_t)2 * sms * 7 && p.kt / (2 * p.parts) >= 2) p.parts *= 2;
    } else {
        // 256-token tiles for 16-bit results (see the top), unless they leave SMs without work
        const int64_t cols = ceil_div(c.n, 2 * ch), pairs = cols * ceil_div(c.m, 256);
        tok = c.y_dtype == SBQ_F32 || pairs * 10 < (int64_t)(sms / 2) * 9 ? 128 : 256;
    }
    W4Maps maps;
    const int st = make_maps(maps, c, x, tok == kSTok4 ? kSTok4 : tok / 2);
    if (st) return st;
    const cudaError_t e = x.part[1] ? (nmat == 2 ? launch_gemm_w4_g<2, 2>(c.gpt, tok, maps, p, c.stream)
                                                 : launch_gemm_w4_g<2, 1>(c.gpt, tok, maps, p, c.stream))
                                    : (nmat == 2 ? launch_gemm_w4_g<1, 2>(c.gpt, tok, maps, p, c.stream)
                                                 : launch_gemm_w4_g<1, 1>(c.gpt, tok, maps, p, c.stream));
    if (e != cudaSuccess) return set_error(SBQ_ERR_CUDA, "gemm_w4 launch: %s", cudaGetErrorString(e));
    return check_launch("gemm_w4");
}

}  // namespace sbq
