// Product of 4-bit weights with group scales for more than 16 rows of x, and its fused gate/up form, on
// the fifth-generation tensor cores:
//
//   y[t, n] = xinv[t] / rowmul[n] * sum_k xh[t, k] * (q[n, k] s[n, k / group] rowmul[n])  (+ bias[n])
//
// xh is x in fp16 (x itself, or its power-of-two-scaled parts, linear_w4.cu), and q * s * rowmul is exact in
// fp16 (w4.cuh, down to scales of 2^-27 of the row's largest), so the products are those of the definition and the
// sums are fp32 in tensor memory.
//
// Channels are the MMA's M, tokens its N.  Per 128 columns of k (one packed tile):
//   * warp 0 (one thread) loads the tokens' x (TMA, 128-byte swizzle), the codes (64 bytes per channel, 64-byte
//     swizzle, so that 32 rows read 16 bytes each without bank conflicts) and the scales into a ring of stages;
//   * two converter warpgroups, one channel per thread, turn the codes into scaled fp16 weights and write them to
//     tensor memory (the MMA's A operand, a ring of its own);
//   * warp 1 (one thread) issues tcgen05.mma, A from tensor memory, x from shared memory.
//
// Conversion: a code moved to bits 6..9 under the fp16 exponent of 16 reads as 16 + u, and
// (16 + u) * s - 24 * s = q * s is one fused multiply-add: 24 * s is exact (2 + 8 bits), the result too.  With a
// shift and a mask per pair of columns that is 3 instructions for 2 weights.
//
// Tensor-core accumulation truncates: measured on B200, the relative error of a sum grows by about 1.3e-8 per
// k16 step (1.2e-5 at k = 12288).  Where the result is kept in fp32 the sum is therefore cut into segments
// of kSegSteps = 32 steps, and each finished segment is added to fp32 registers (round to nearest): 3e-7 (bf16 x) to
// 6e-7 (fp32 x) at any k from 512 to 12288, with 64 steps 1.2e-6.  16-bit results are summed in one piece: that error is
// relative to the largest partial sum, so it lies far below the result's own rounding (2^-12 or 2^-9 of its value) unless
// the sum cancels to a few hundredths of its parts or k passes about 100,000.
//
// Measured on B200, groups of 128, in bursts of a few ms (the power cap not yet reached): 4096 x 4096 x 12288 fp16 271 us (1.52
// PFLOP/s, 0.92 of cuBLAS's measured bf16 burst rate), 2048 x 4096 x 12288 fp16 144 us, with fp32 results 170 us (a segment
// ends in the wait for the accumulator to be read); gate/up 2048 x 4096 x 12288 293 us with bf16 x.  Call after call, under the
// power cap, 310 to 316 us and 340 to 345 us.  Long products are bound by the tensor cores (active 72 to 75 % of the cycles at
// the lowered clock); one tile per pair (512 x 4096 x 4096, 24.5 us) by about 8 us of set-up, first loads and stores and
// 0.5 us per block of 128 k; 64 x 4096 x 12288 (20 us) by x, read again for every 128 channels (100 MB of L2 traffic for 27 of
// weight).  The gate/up instances of the pair kernel spill up to 180 bytes a thread in the takers' exchange, once per tile
// and beside the MMAs (0.7 % of all instructions).
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
    int seg_blocks;  // blocks of 128 k per accumulation segment
    // pair kernel: rounds of whole tiles, then tail_tiles tiles cut into tail_parts parts along k
    int rounds, tail_tiles, tail_parts;
    int tok;  // tokens of a tile: a multiple of 32 up to 256
    float* partial;  // [tail tile][part][token][lane of both CTAs]: sums of a cut tile's parts, or null
    const float* rowmul[2];
    const float* bias;
    const float* xinv;
    void* y;
    int64_t ldy;
    int y_dtype;
};

// Sizes of one kernel.  XROWS: tokens of x this CTA loads per block of 128 k; N: the MMA's tokens; ND:
// accumulators; XCH: bytes for the gate / up exchange.
template <int XROWS, int N, int PARTS, int ND, int TMEM, int RING, int XCH>
struct W4Shape {
    static constexpr int kXSub = XROWS * 128;               // 64 columns of k: a 128-byte row per token
    static constexpr int kXBytes = 2 * PARTS * kXSub;       // [64-column half][part]
    static constexpr int kCodes = kW4Rows * 64;
    static constexpr int kStage = kXBytes + kCodes + 1024;  // scales: at most 1 KiB
    static constexpr int kStages = (RING - XCH) / kStage < 8 ? (RING - XCH) / kStage : 8;
    static constexpr int kACol = ND * N;                    // accumulators first
    static constexpr int kABufs0 = (TMEM - kACol) / 64;
    static constexpr int kABufs1 = kABufs0 < 4 ? kABufs0 : 4;
    static constexpr int kABufs = kABufs1 < kStages ? kABufs1 : kStages;  // 64 columns per 128 k
    static constexpr int kXchOff = kStages * kStage;
    static constexpr int kBarOff = kXchOff + XCH;
    static constexpr int kBytes = kBarOff + 512 + 1024;  // barriers, alignment
    static_assert(kStages >= 2 && kABufs >= 2, "pipeline depth");
    static_assert((4 * kStages + 4) * 8 + 4 <= 512, "barriers");
    static_assert(kBytes <= 227 * 1024, "shared memory");
};

// fp16 scale pairs (s, s) and (-24 s, -24 s) of one channel's groups in a tile.
template <int GPT>
__device__ __forceinline__ void w4_scales(const uint8_t* scales, int row, float rowmul, int g0, uint32_t* s2, uint32_t* c2,
                                          int count) {
#pragma unroll
    for (int i = 0; i < count; ++i) {
        const uint16_t u = *reinterpret_cast<const uint16_t*>(
            scales + (((row >> 4) * 8 + (row & 7)) * GPT + g0 + i) * 4 + ((row >> 3) & 1) * 2);
        const __half2 s = __float2half2_rn(__uint_as_float((uint32_t)u << 16) * rowmul);
        s2[i] = *reinterpret_cast<const uint32_t*>(&s);
        const __half2 c = __hmul2(s, __float2half2_rn(-24.0f));
        c2[i] = *reinterpret_cast<const uint32_t*>(&c);
    }
}

// Eight codes -> four words of scaled fp16 weights.
__device__ __forceinline__ void w4_convert_word(uint32_t v, uint32_t s, uint32_t c, uint32_t* o) {
    o[0] = hfma2(lop3_and_or(v << 6, 0x03C003C0u, 0x4C004C00u), s, c);
    o[1] = hfma2(lop3_and_or(v << 2, 0x03C003C0u, 0x4C004C00u), s, c);
    o[2] = hfma2(lop3_and_or(v >> 2, 0x03C003C0u, 0x4C004C00u), s, c);
    o[3] = hfma2(lop3_and_or(v >> 6, 0x03C003C0u, 0x4C004C00u), s, c);
}

__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// 32 lanes x 16 tensor-memory columns: thread t of the warp gets lane (base lane + t).
__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

// Columns 64 half .. 64 half + 63 of channel `row` of one tile (64 bytes of codes, 64-byte swizzle) -> 32
// tensor-memory columns.
template <int GPT>
__device__ __forceinline__ void w4_convert_half(const uint8_t* codes, const uint8_t* scales, int row, float rowmul, int half,
                                                uint32_t tmem_dst) {
    constexpr int NG = GPT == 4 ? 2 : 1;  // groups in 64 columns
    uint32_t s2[NG], c2[NG], h[16];
    w4_scales<GPT>(scales, row, rowmul, half * GPT / 2, s2, c2, NG);
    uint2 v[4];
#pragma unroll
    for (int t = 0; t < 4; ++t)
        v[t] = *reinterpret_cast<const uint2*>(codes + row * 64 + ((t ^ ((row >> 1) & 3)) << 4) + half * 8);
#pragma unroll
    for (int t = 0; t < 4; ++t) w4_convert_word(v[t].x, s2[0], c2[0], h + 4 * t);
    tmem_st_x16(tmem_dst, h);
#pragma unroll
    for (int t = 0; t < 4; ++t) w4_convert_word(v[t].y, s2[NG - 1], c2[NG - 1], h + 4 * t);
    tmem_st_x16(tmem_dst + 16, h);
}

// Channel of tensor-memory lane `row` (CTA's first channel n0): with two matrices lanes 0..63 are the
// gate's channels n0.., lanes 64..127 the up projection's.
template <int NMAT>
__device__ __forceinline__ int w4_channel(int n0, int row) { return n0 + (NMAT == 2 ? row & 63 : row); }

// Up to 128 named-barrier threads of one converter warpgroup.
__device__ __forceinline__ void group_sync(int grp) { asm volatile("bar.sync %0, 128;" ::"r"(1 + grp) : "memory"); }

// ---------------------------------------------------------------------------------------------
// Many rows: CTA pairs (cta_group::2), persistent.  A pair computes tiles of 256 channels x TOK tokens one
// after the other; blocks of 128 k run through the rings without a break between tiles.  Each CTA converts its
// own 128 channels and loads half of the tokens.  With two matrices a CTA's lanes 0..63 are gate channels and
// lanes 64..127 the same channels of the up projection (128 channels per pair).
//
// Roles: warp 0 producer, warp 1 MMA (leader), warp 2 tensor memory; warps 4-11 converters, each on one half of the
// columns of every block; warps 12-19 takers: they read a finished segment (tile) out of the accumulator, let the
// MMAs go on, and scale and store a finished tile under the next one's MMAs.  Registers are dealt to the roles
// by setmaxnreg: a taker holds up to 128 fp32 sums.
//
// Tiles are up to 256 tokens wide (that accumulator and four operand buffers fill tensor memory).  An MMA of N tokens
// whose A operand comes from tensor memory takes about 50 + 0.39 N cycles (N = 128: 100), so wide tiles are
// the efficient ones and narrow ones serve products that would leave pairs without a tile.  The last token tile's
// MMAs are as wide as its tokens.
//
// The tiles of the last, incomplete round are cut along k so that every pair has a part; a cut tile's parts go to
// `partial` as fp32 sums and w4_reduce_kernel adds them in order.
// ---------------------------------------------------------------------------------------------
constexpr int kPairThreads = 640;
constexpr int kRegsIssue = 40, kRegsConvert = 56, kRegsTake = 160;
static_assert(kRegsIssue + 2 * kRegsConvert + 2 * kRegsTake <= 5 * 96, "the launch's registers: 96 x 640 threads");

template <int N>
__device__ __forceinline__ void regs_more() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_less() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

constexpr int kTok = 256;  // tokens of a tile, at most
template <int PARTS, int NMAT>
using W4Pair = W4Shape<kTok / 2, kTok, PARTS, 1, 512, 224 * 1024, NMAT == 2 ? 32 * 1024 : 0>;

// One piece of a pair's work: blocks kb0 .. kb1 - 1 of a tile; slot: its place in `partial`, -1 for a whole tile.
struct W4Item {
    int tile, kb0, kb1, slot;
};

__device__ __forceinline__ int w4_items(const GemmW4Params& p, int pair) {
    return p.rounds + (pair < p.tail_tiles * p.tail_parts ? 1 : 0);
}

__device__ __forceinline__ W4Item w4_item(const GemmW4Params& p, int pair, int npairs, int i) {
    W4Item w;
    if (i < p.rounds) {
        w.tile = i * npairs + pair, w.kb0 = 0, w.kb1 = p.kt, w.slot = -1;
    } else {
        const int P = p.tail_parts, part = pair % P;
        w.tile = p.rounds * npairs + pair / P;
        w.kb0 = part * p.kt / P, w.kb1 = (part + 1) * p.kt / P;
        w.slot = P > 1 ? pair : -1;
    }
    return w;
}

// Tokens of the MMAs of a tile: its rows of x rounded up to 32.
__device__ __forceinline__ int w4_tile_tokens(const GemmW4Params& p, int t0) {
    const int left = (p.m - t0 + 31) & ~31;
    return left < p.tok ? left : p.tok;
}

template <class T>
__device__ __forceinline__ T w4_round(float v);
template <>
__device__ __forceinline__ float w4_round<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half w4_round<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 w4_round<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// One channel's results of CNT tokens from t0 on: consecutive lanes hold consecutive channels.
template <class T, int CNT, class F>
__device__ __forceinline__ void w4_put_as(const GemmW4Params& p, int t0, int n, F value) {
    T* y = static_cast<T*>(p.y) + (int64_t)t0 * p.ldy + n;
    if (t0 + CNT <= p.m) {
#pragma unroll
        for (int j = 0; j < CNT; ++j, y += p.ldy) *y = w4_round<T>(value(j));
    } else {
#pragma unroll
        for (int j = 0; j < CNT; ++j, y += p.ldy)
            if (t0 + j < p.m) *y = w4_round<T>(value(j));
    }
}

template <int CNT, class F>
__device__ __forceinline__ void w4_put(const GemmW4Params& p, int t0, int n, F value) {
    if (n >= p.n) return;
    if (p.y_dtype == SBQ_F32)
        w4_put_as<float, CNT>(p, t0, n, value);
    else if (p.y_dtype == SBQ_F16)
        w4_put_as<__half, CNT>(p, t0, n, value);
    else
        w4_put_as<__nv_bfloat16, CNT>(p, t0, n, value);
}

// CNT tokens' factors (the array is padded to a multiple of 256 values).
template <int CNT>
__device__ __forceinline__ void w4_times_xinv(const float* xinv, int t0, float* v) {
#pragma unroll
    for (int j = 0; j < CNT / 4; ++j) {
        const float4 f = __ldg(reinterpret_cast<const float4*>(xinv + t0) + j);
        v[4 * j] *= f.x, v[4 * j + 1] *= f.y, v[4 * j + 2] *= f.z, v[4 * j + 3] *= f.w;
    }
}

template <int PARTS, int NMAT, int GPT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    gemm_w4_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_lo,
                        const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_w2,
                        const __grid_constant__ CUtensorMap map_s, const __grid_constant__ CUtensorMap map_s2,
                        const __grid_constant__ GemmW4Params p) {
    using S = W4Pair<PARTS, NMAT>;
    constexpr int NS = S::kStages, NA = S::kABufs, COLS = kTok / 2;  // COLS: tokens per taker warpgroup
    constexpr int kCh = kW4Rows / NMAT;                             // channels of this CTA's tile
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* wfull = reinterpret_cast<uint64_t*>(smem + S::kBarOff);  // this CTA's codes and scales landed
    uint64_t* ready = wfull + NS;      // leader: both CTAs' x landed and both CTAs' converters wrote
    uint64_t* conv_done = ready + NS;  // this CTA's converters have read the codes
    uint64_t* mma_done = conv_done + NS;
    uint64_t* done = mma_done + NS;    // a segment's MMAs completed
    uint64_t* taken = done + 1;        // leader: both CTAs' takers have read the accumulator
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(taken + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = tc::cluster_ctarank();
    const bool leader = rank == 0;
    const int pair = (int)(blockIdx.x >> 1), npairs = (int)(gridDim.x >> 1);
    const int cols = (p.n + 2 * kCh - 1) / (2 * kCh);  // tiles are numbered channels first
    const int items = w4_items(p, pair);

    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; ++s) {
            tc::mbar_init(&wfull[s], 1);
            tc::mbar_init(&ready[s], 1 + 16);
            tc::mbar_init(&conv_done[s], 8);
            tc::mbar_init(&mma_done[s], 1);
        }
        tc::mbar_init(done, 1);
        tc::mbar_init(taken, 16);
        tc::fence_mbar_init();
        tc::prefetch_tmap(&map_x);
        tc::prefetch_tmap(&map_w);
        tc::prefetch_tmap(&map_s);
    }
    if (warp == 2) {
        tc::tmem_alloc_pair(tmem_slot, 512);
        tc::tmem_relinquish_pair();
    }
    tc::fence_before_sync();
    tc::cluster_sync();
    tc::fence_after_sync();
    const uint32_t tmem = *tmem_slot;

    if (warp < 4) {
        regs_less<kRegsIssue>();
        if (warp == 0 && lane == 0) {
            auto load_w = [&](int s, int tile, int kb) {
                uint8_t* ws = smem + s * S::kStage + S::kXBytes;
                const int nt = (tile % cols) * (2 * kCh / 16) + (int)rank * (kCh / 16);
                tc::mbar_arrive_expect_tx(&wfull[s], S::kCodes + 256 * GPT);
                tc::tma_load_4d(ws, &map_w, &wfull[s], 0, 0, kb, nt);
                tma_load_3d(ws + S::kCodes, &map_s, &wfull[s], 0, kb, nt);
                if (NMAT == 2) {
                    tc::tma_load_4d(ws + S::kCodes / 2, &map_w2, &wfull[s], 0, 0, kb, nt);
                    tma_load_3d(ws + S::kCodes + 128 * GPT, &map_s2, &wfull[s], 0, kb, nt);
                }
            };
            auto load_x = [&](int s, int tile, int kb) {
                uint8_t* xs = smem + s * S::kStage;
                const int t0 = (tile / cols) * p.tok, tr = t0 + (int)rank * (w4_tile_tokens(p, t0) / 2);
                const uint32_t xb = tc::cluster_addr(&ready[s], 0);
                if (leader) tc::mbar_arrive_expect_tx(&ready[s], (uint32_t)p.tok * (PARTS * 256));  // both CTAs' boxes
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    tc::tma_load_2d_pair(xs + h * PARTS * S::kXSub, &map_x, xb, kb * 128 + h * 64, tr);
                    if (PARTS == 2) tc::tma_load_2d_pair(xs + (h * PARTS + 1) * S::kXSub, &map_lo, xb, kb * 128 + h * 64, tr);
                }
            };
            // codes of the first stages before the wait for the previous kernel, x after it
            int pre = 0;
            for (int i = 0; i < items && pre < NS; ++i) {
                const W4Item w = w4_item(p, pair, npairs, i);
                for (int kb = w.kb0; kb < w.kb1 && pre < NS; ++kb) load_w(pre++, w.tile, kb);
            }
            asm volatile("griddepcontrol.wait;" ::: "memory");
            asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
            int s = 0, g = 0;
            uint32_t ph = 1;  // of the blocks that used the stages before
            bool ok = true;
            for (int i = 0; i < items && ok; ++i) {
                const W4Item w = w4_item(p, pair, npairs, i);
                for (int kb = w.kb0; kb < w.kb1; ++kb, ++g) {
                    if (g >= pre) {
                        if (!tc::mbar_wait(&conv_done[s], ph) || !tc::mbar_wait(&mma_done[s], ph)) {
                            ok = false;
                            break;
                        }
                        load_w(s, w.tile, kb);
                    }
                    load_x(s, w.tile, kb);
                    if (++s == NS) s = 0, ph ^= 1;
                }
            }
        } else if (warp == 1 && lane == 0 && leader) {
            // One thread issues everything, so its instructions per block are kept few: a descriptor is the first
            // stage's plus a multiple of 16 bytes, ring positions are counted along.
            const uint64_t desc0 = tc::smem_desc(smem, tc::kSwizzle128B, 1024);
            const uint32_t bar_done0 = tc::cluster_addr(mma_done, 0), bar_done1 = tc::cluster_addr(mma_done, 1);
            const uint32_t bar_seg0 = tc::cluster_addr(done, 0), bar_seg1 = tc::cluster_addr(done, 1);
            int s = 0, ab = 0, seg = 0;  // stage, operand buffer, segment
            uint32_t ph = 0;
            bool ok = true;
            for (int i = 0; i < items && ok; ++i) {
                const W4Item w = w4_item(p, pair, npairs, i);
                const uint32_t idesc = tc::idesc_f16(2 * kW4Rows, w4_tile_tokens(p, (w.tile / cols) * p.tok), false);
                int left = 0;  // blocks left in the segment
                for (int kb = w.kb0; kb < w.kb1; ++kb) {
                    const bool fresh = left == 0;
                    if (fresh) {
                        left = p.seg_blocks < w.kb1 - kb ? p.seg_blocks : w.kb1 - kb;
                        if (seg > 0 && !tc::mbar_wait_cluster(taken, (seg - 1) & 1)) {
                            ok = false;
                            break;
                        }
                    }
                    if (!tc::mbar_wait_cluster(&ready[s], ph)) {
                        ok = false;
                        break;
                    }
                    tc::fence_after_sync();
                    const uint64_t xd = desc0 + (uint64_t)(s * (S::kStage / 16));
                    const uint32_t op = tmem + S::kACol + ab * 64;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int q = 0; q < PARTS; ++q)
                            tc::mma_f16_ts_pair(tmem, op + j * 8, xd + (((j >> 2) * PARTS + q) * S::kXSub + (j & 3) * 32) / 16,
                                                idesc, j == 0 && q == 0 ? !fresh : 1u);
                    tc::mma_commit_pair(bar_done0 + s * 8);
                    tc::mma_commit_pair(bar_done1 + s * 8);
                    if (--left == 0) {
                        tc::mma_commit_pair(bar_seg0);
                        tc::mma_commit_pair(bar_seg1);
                        ++seg;
                    }
                    if (++s == NS) s = 0, ph ^= 1;
                    if (++ab == NA) ab = 0;
                }
            }
        }
    } else if (warp < 12) {
        regs_less<kRegsConvert>();
        const int half = (warp - 4) >> 2, wq = warp & 3, row = wq * 32 + lane;
        const uint32_t dst0 = tmem + ((uint32_t)(wq * 32) << 16) + S::kACol + half * 32;
        const uint32_t ready0 = tc::cluster_addr(ready, 0);
        const float* rowmul = p.rowmul[NMAT == 2 ? row >> 6 : 0];
        const int cn = (int)rank * kCh + (NMAT == 2 ? row & 63 : row);
        auto mul_of = [&](int i) {
            const int n = i < items ? (w4_item(p, pair, npairs, i).tile % cols) * (2 * kCh) + cn : p.n;
            return n < p.n ? __ldg(rowmul + n) : 1.0f;
        };
        // ring positions are counted along: stage s in its phase ph, operand buffer ab, and the stage sa of the
        // block that used that buffer before, in its phase pa
        int g = 0, s = 0, ab = 0, sa = 0;
        uint32_t ph = 0, pa = 0;
        bool ok = true;
        float mul = mul_of(0);
        for (int i = 0; i < items && ok; ++i) {
            const W4Item w = w4_item(p, pair, npairs, i);
            const float next_mul = mul_of(i + 1);
            for (int kb = w.kb0; kb < w.kb1; ++kb, ++g) {
                if (g >= NA) {
                    // the operand buffer was last read by block g - NA.  Every warp takes every block, and
                    // NA <= NS, so each barrier is at most one phase from the one awaited
                    if (!__all_sync(0xffffffffu, tc::mbar_wait(&mma_done[sa], pa))) { ok = false; break; }
                    if (++sa == NS) sa = 0, pa ^= 1;
                }
                if (!__all_sync(0xffffffffu, tc::mbar_wait(&wfull[s], ph))) { ok = false; break; }
                tc::fence_after_sync();
                const uint8_t* codes = smem + s * S::kStage + S::kXBytes;
                w4_convert_half<GPT>(codes, codes + S::kCodes, row, mul, half, dst0 + ab * 64);
                tc::tmem_wait_st();
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    tc::mbar_arrive_cluster(ready0 + s * 8);
                    tc::mbar_arrive(&conv_done[s]);
                }
                if (++s == NS) s = 0, ph ^= 1;
                if (++ab == NA) ab = 0;
            }
            mul = next_mul;
        }
    } else {
        regs_more<kRegsTake>();
        const int grp = (warp - 12) >> 2, wq = warp & 3, row = wq * 32 + lane;
        const int half = p.tok / 2;  // tokens of this warpgroup
        const uint32_t src = tmem + ((uint32_t)(wq * 32) << 16) + grp * half;
        const uint32_t taken0 = tc::cluster_addr(taken, 0);
        const int mat = NMAT == 2 ? row >> 6 : 0, cn = (int)rank * kCh + (NMAT == 2 ? row & 63 : row);
        float* xch = reinterpret_cast<float*>(smem + S::kXchOff) + grp * 32 * kW4Rows;
        asm volatile("griddepcontrol.wait;" ::: "memory");  // before y is written, and xinv read
        uint32_t ph = 0;
        bool ok = true;  // a warp whose wait ran out stores nothing more, but stays for the group's barriers
        for (int i = 0; i < items; ++i) {
            const W4Item w = w4_item(p, pair, npairs, i);
            const int n = (w.tile % cols) * (2 * kCh) + cn, t0 = (w.tile / cols) * p.tok + grp * half;
            const float inv = 1.0f / (n < p.n ? __ldg(p.rowmul[mat] + n) : 1.0f);
            const float bias = NMAT == 1 && p.bias && n < p.n ? __ldg(p.bias + n) : 0.0f;
            float sum[COLS];
            for (int kb = w.kb0; kb < w.kb1; kb += p.seg_blocks) {
                ok = ok && __all_sync(0xffffffffu, tc::mbar_wait(done, ph));
                if (!ok) break;
                ph ^= 1;
                tc::fence_after_sync();
                if (kb == w.kb0) {
#pragma unroll
                    for (int c = 0; c < COLS / 16; ++c)
                        if (c * 16 < half) tmem_ld_x16(src + c * 16, reinterpret_cast<uint32_t*>(sum) + c * 16);
                    tc::tmem_wait_ld();
                } else {
#pragma unroll
                    for (int c = 0; c < COLS / 16; ++c) {
                        if (c * 16 >= half) continue;
                        uint32_t r[16];
                        tmem_ld_x16(src + c * 16, r);
                        tc::tmem_wait_ld();
#pragma unroll
                        for (int j = 0; j < 16; ++j) sum[c * 16 + j] += __uint_as_float(r[j]);
                    }
                }
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive_cluster(taken0);
            }
            // ---- the tile's sums are here, the MMAs go on
            if (w.slot >= 0) {
                float* out = p.partial + ((int64_t)w.slot * kTok + grp * half) * (2 * kW4Rows) + (int)rank * kW4Rows + row;
                if (ok) {
#pragma unroll
                    for (int j = 0; j < COLS; ++j)
                        if (j < half && t0 + j < p.m) __stcg(out + j * (2 * kW4Rows), sum[j]);
                }
                continue;
            }
#pragma unroll
            for (int c = 0; c < COLS / 16; ++c) {
                if (c * 16 >= half) continue;
#pragma unroll
                for (int j = 0; j < 16; ++j) sum[c * 16 + j] *= inv;
                if (p.xinv) w4_times_xinv<16>(p.xinv, t0 + c * 16, sum + c * 16);
                if (NMAT == 1 && ok) w4_put<16>(p, t0 + c * 16, n, [&](int j) { return sum[c * 16 + j] + bias; });
            }
            if (NMAT == 2) {
                // of every 32 tokens the gate lanes finish the first 16, the up lanes the others: each hands the other its
                // values.  Two buffers, so one barrier per 32 tokens
                const bool up = mat == 1;
#pragma unroll
                for (int c = 0; c < COLS / 32; ++c) {
                    if (c * 32 >= half) continue;
                    float* buf = xch + (c & 1) * 16 * kW4Rows;
#pragma unroll
                    for (int j = 0; j < 16; ++j) buf[j * kW4Rows + row] = up ? sum[c * 32 + j] : sum[c * 32 + 16 + j];
                    group_sync(grp);
                    float res[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) res[j] = buf[j * kW4Rows + (row ^ 64)];
                    // a 16-bit result: the approximate exponential (documented to 2 + 1.2 |g| units of 2^-23) and
                    // division are off by 2^-16 of silu at most, at gates near -87, and by 2^-19 above -10, under its rounding
                    // of 2^-12 or 2^-9.  The reduction of cut tiles and the few-row kernel, with fewer results to a
                    // thread, take expf and an exact division
                    if (p.y_dtype == SBQ_F32) {
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            res[j] = up ? w4_silu(res[j]) * sum[c * 32 + 16 + j] : w4_silu(sum[c * 32 + j]) * res[j];
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const float gv = up ? res[j] : sum[c * 32 + j], uv = up ? sum[c * 32 + 16 + j] : res[j];
                            res[j] = __fdividef(gv, 1.0f + __expf(-gv)) * uv;
                        }
                    }
                    if (ok) w4_put<16>(p, t0 + c * 32 + (up ? 16 : 0), n, [&](int j) { return res[j]; });
                }
            }
        }
    }
    tc::fence_before_sync();
    tc::cluster_sync();
    if (warp == 2) {
        tc::fence_after_sync();
        tc::tmem_dealloc_pair(tmem, 512);
    }
}

// Cut tiles: one CTA per tile and 4 tokens (two matrices: 8), one thread per lane of the pair (two matrices: 4 of the
// 8 tokens of a channel's two lanes).  Every thread's loads of a part are independent of each other.
template <int NMAT>
__global__ void __launch_bounds__(2 * kW4Rows) w4_reduce_kernel(const GemmW4Params p, int npairs) {
    constexpr int kCh = kW4Rows / NMAT, kLanes = 2 * kW4Rows, T = 4;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int cols = (p.n + 2 * kCh - 1) / (2 * kCh);
    const int cut = (int)blockIdx.y, tile = p.rounds * npairs + cut;
    const int tid = (int)threadIdx.x, ch = NMAT == 2 ? tid & 127 : tid;
    const int j0 = ((int)blockIdx.x * NMAT + (NMAT == 2 ? tid >> 7 : 0)) * T, t0 = (tile / cols) * p.tok + j0;
    const int lane0 = NMAT == 2 ? (ch >> 6) * kW4Rows + (ch & 63) : ch;
    const int n = (tile % cols) * (2 * kCh) + ch;
    if (n >= p.n || t0 >= p.m || j0 >= p.tok) return;
    const int count = p.m - t0 < T ? p.m - t0 : T;
    const float* base = p.partial + ((int64_t)cut * p.tail_parts * kTok + j0) * kLanes + lane0;
    float v[NMAT][T];
#pragma unroll
    for (int a = 0; a < NMAT; ++a)
#pragma unroll
        for (int j = 0; j < T; ++j) v[a][j] = 0.0f;
#pragma unroll 2
    for (int q = 0; q < p.tail_parts; ++q, base += (int64_t)kTok * kLanes) {
#pragma unroll
        for (int a = 0; a < NMAT; ++a)
#pragma unroll
            for (int j = 0; j < T; ++j) v[a][j] += j < count ? __ldcg(base + j * kLanes + a * 64) : 0.0f;
    }
    const float bias = NMAT == 1 && p.bias ? __ldg(p.bias + n) : 0.0f;
#pragma unroll
    for (int a = 0; a < NMAT; ++a) {
        const float inv = 1.0f / __ldg(p.rowmul[a] + n);
#pragma unroll
        for (int j = 0; j < T; ++j) {
            v[a][j] *= inv;
            if (p.xinv && j < count) v[a][j] *= __ldg(p.xinv + t0 + j);
        }
    }
    w4_put<T>(p, t0, n, [&](int j) { return NMAT == 2 ? w4_silu(v[0][j]) * v[NMAT - 1][j] : v[0][j] + bias; });
}

// ---------------------------------------------------------------------------------------------
// Few rows: 128 channels x 64 tokens per CTA, two CTAs per SM, k split over the CTAs of a cluster when
// the tiles alone are too few: each pushes its fp32 sums into the shared memory of the CTA that owns the
// channel, which adds them in part order.  The two converter warpgroups take alternate blocks (each warp on half of
// every block, as in the pair kernel, was 15 % slower: with two CTAs on an SM the waits of a block count) and both
// take the sums, 32 tokens each.
// ---------------------------------------------------------------------------------------------
constexpr int kSTok4 = 64;
template <int PARTS>
using W4Small = W4Shape<kSTok4, kSTok4, PARTS, 1, 256, 108 * 1024, 0>;

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
    uint64_t* taken = done + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(taken + 1);
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
        tc::mbar_init(done, 1);
        tc::mbar_init(taken, 8);
        tc::fence_mbar_init();
        tc::prefetch_tmap(&map_x);
        tc::prefetch_tmap(&map_w);
        tc::prefetch_tmap(&map_s);
    }
    if (warp == 2) {
        tc::tmem_alloc(tmem_slot, 256);
        tc::tmem_relinquish();
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    float sum[32];

    if (warp == 0) {
        if (lane == 0) {
            auto load_w = [&](int s, int kb) {
                uint8_t* ws = smem + s * S::kStage + S::kXBytes;
                tc::mbar_arrive_expect_tx(&wfull[s], S::kCodes + 256 * GPT);
                tc::tma_load_4d(ws, &map_w, &wfull[s], 0, 0, kb, n0 / 16);
                tma_load_3d(ws + S::kCodes, &map_s, &wfull[s], 0, kb, n0 / 16);
                if (NMAT == 2) {
                    tc::tma_load_4d(ws + S::kCodes / 2, &map_w2, &wfull[s], 0, 0, kb, n0 / 16);
                    tma_load_3d(ws + S::kCodes + 128 * GPT, &map_s2, &wfull[s], 0, kb, n0 / 16);
                }
            };
            auto load_x = [&](int s, int kb) {
                uint8_t* xs = smem + s * S::kStage;
                tc::mbar_arrive_expect_tx(&ready[s], S::kXBytes);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    tc::tma_load_2d(xs + h * PARTS * S::kXSub, &map_x, &ready[s], kb * 128 + h * 64, t0);
                    if (PARTS == 2) tc::tma_load_2d(xs + (h * PARTS + 1) * S::kXSub, &map_lo, &ready[s], kb * 128 + h * 64, t0);
                }
            };
            const int pre = nkb < NS ? nkb : NS;
            for (int i = 0; i < pre; ++i) load_w(i, kb0 + i);
            asm volatile("griddepcontrol.wait;" ::: "memory");
            asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
            for (int i = 0; i < pre; ++i) load_x(i, kb0 + i);
            int s = 0;
            uint32_t ph = 0;
            for (int i = pre; i < nkb; ++i) {
                if (!tc::mbar_wait(&conv_done[s], ph)) break;
                if (!tc::mbar_wait(&mma_done[s], ph)) break;
                load_w(s, kb0 + i);
                load_x(s, kb0 + i);
                if (++s == NS) s = 0, ph ^= 1;
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const int tokens = p.m - t0 < kSTok4 ? (p.m - t0 + 15) & ~15 : kSTok4;
            const uint32_t idesc = tc::idesc_f16(kW4Rows, tokens, false);
            const uint64_t desc0 = tc::smem_desc(smem, tc::kSwizzle128B, 1024);
            int s = 0, ab = 0, seg = 0, left = 0;
            uint32_t ph = 0;
            for (int i = 0; i < nkb; ++i) {
                const bool fresh = left == 0;
                if (fresh) {
                    left = p.seg_blocks < nkb - i ? p.seg_blocks : nkb - i;
                    if (seg > 0 && !tc::mbar_wait(taken, (seg - 1) & 1)) break;
                }
                if (!tc::mbar_wait(&ready[s], ph)) break;
                tc::fence_after_sync();
                const uint64_t xd = desc0 + (uint64_t)(s * (S::kStage / 16));
                const uint32_t op = tmem + S::kACol + ab * 64;
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int q = 0; q < PARTS; ++q)
                        tc::mma_f16_ts(tmem, op + j * 8, xd + (((j >> 2) * PARTS + q) * S::kXSub + (j & 3) * 32) / 16, idesc,
                                       j == 0 && q == 0 ? !fresh : 1u);
                tc::mma_commit(&mma_done[s]);
                if (--left == 0) {
                    tc::mma_commit(done);
                    ++seg;
                }
                if (++s == NS) s = 0, ph ^= 1;
                if (++ab == NA) ab = 0;
            }
        }
    } else if (warp >= 4) {
        const int half = (warp - 4) >> 2, wq = warp & 3, row = wq * 32 + lane;
        const uint32_t lane_tmem = tmem + ((uint32_t)(wq * 32) << 16);
        const int n = w4_channel<NMAT>(n0, row);
        const float mul = n < p.n ? __ldg(p.rowmul[NMAT == 2 ? row >> 6 : 0] + n) : 1.0f;
        // the next segment to take: its parity and its last block
        uint32_t tk_ph = 0;
        int tk_last = p.seg_blocks < nkb ? p.seg_blocks - 1 : nkb - 1;
#pragma unroll
        for (int j = 0; j < 32; ++j) sum[j] = 0.0f;
        auto take = [&]() -> bool {
            if (!__all_sync(0xffffffffu, tc::mbar_wait(done, tk_ph))) return false;
            tk_ph ^= 1;
            tc::fence_after_sync();
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t r[16];
                tmem_ld_x16(lane_tmem + half * 32 + c * 16, r);
                tc::tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; ++j) sum[c * 16 + j] += __uint_as_float(r[j]);
            }
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(taken);
            // the last segment has no next: past the end
            tk_last = tk_last == nkb - 1 ? nkb : tk_last + p.seg_blocks < nkb - 1 ? tk_last + p.seg_blocks : nkb - 1;
            return true;
        };
        bool ok = true;
        for (int i = half; i < nkb; i += 2) {
            const int s = i % NS;
            if (i >= NA) {
                // the operand buffer's last reader, block i - NA; a segment is taken when its last block's MMAs
                // are done, or this warp's next block would wait for MMAs that wait for the taking
                const int prev = i - NA;
                if (!__all_sync(0xffffffffu, tc::mbar_wait(&mma_done[prev % NS], (prev / NS) & 1))) { ok = false; break; }
                while (ok && tk_last < prev + 2) ok = take();
                if (!ok) break;
            }
            if (!__all_sync(0xffffffffu, tc::mbar_wait(&wfull[s], (i / NS) & 1))) { ok = false; break; }
            tc::fence_after_sync();
            const uint8_t* codes = smem + s * S::kStage + S::kXBytes;
            const uint32_t dst = lane_tmem + S::kACol + (i % NA) * 64;
            w4_convert_half<GPT>(codes, codes + S::kCodes, row, mul, 0, dst);
            w4_convert_half<GPT>(codes, codes + S::kCodes, row, mul, 1, dst + 32);
            tc::tmem_wait_st();
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                tc::mbar_arrive(&ready[s]);
                tc::mbar_arrive(&conv_done[s]);
            }
        }
        while (ok && tk_last < nkb) ok = take();
        asm volatile("griddepcontrol.wait;" ::: "memory");  // before y is written, and xinv read
        const float inv = 1.0f / mul;
#pragma unroll
        for (int j = 0; j < 32; ++j) sum[j] *= inv;
        if (p.parts == 1) {
            const int tb = t0 + half * 32;
            if (p.xinv) w4_times_xinv<32>(p.xinv, tb, sum);
            const float bias = p.bias && n < p.n ? __ldg(p.bias + n) : 0.0f;
            if (NMAT == 1) {
                if (ok) w4_put<32>(p, tb, n, [&](int j) { return sum[j] + bias; });
            } else {
                // the up lanes hand their values to the gate lanes, which finish; no load is on its way into the ring
                float* xch = recv + half * 32 * 64;
                if (row >= 64) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) xch[j * 64 + (row & 63)] = sum[j];
                }
                group_sync(half);
                if (row < 64 && ok) w4_put<32>(p, tb, n, [&](int j) { return w4_silu(sum[j]) * xch[j * 64 + row]; });
            }
        }
    }
    if (p.parts > 1) {
        // (1) every CTA of the cluster has left its main loop, so every ring is free; (2) sums go to the owner of
        // the channel, [part][token][matrix][owner's channel], neighbouring lanes next to each other; (3) the
        // owner adds them in part order.
        tc::cluster_sync();
        const int share = kCh / p.parts;  // a power of two, at least 8
        if (warp >= 4) {
            const int half = (warp - 4) >> 2, row = (warp & 3) * 32 + lane;
            const int mat = NMAT == 2 ? row >> 6 : 0, c = NMAT == 2 ? row & 63 : row, owner = c / share;
            const uint32_t dst = tc::cluster_addr(recv + ((part * kSTok4 + half * 32) * NMAT + mat) * share + c % share, (uint32_t)owner);
#pragma unroll
            for (int j = 0; j < 32; ++j)
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + (uint32_t)(j * NMAT * share * 4)), "f"(sum[j]) : "memory");
        }
        tc::cluster_sync();
        asm volatile("griddepcontrol.wait;" ::: "memory");
        for (int e = threadIdx.x; e < share * kSTok4; e += blockDim.x) {
            const int c = e % share, t = e / share, n = n0 + part * share + c;
            if (t0 + t >= p.m || n >= p.n) continue;
            float v[NMAT];
#pragma unroll
            for (int a = 0; a < NMAT; ++a) {
                v[a] = 0.0f;
                for (int q = 0; q < p.parts; ++q) v[a] += recv[((q * kSTok4 + t) * NMAT + a) * share + c];
                if (p.xinv) v[a] *= p.xinv[t0 + t];
            }
            const float out = NMAT == 2 ? w4_silu(v[0]) * v[NMAT - 1] : p.bias ? v[0] + __ldg(p.bias + n) : v[0];
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

// x in boxes of `x_rows` tokens, codes and scales in boxes of `w_rows` channels (per matrix).
static int make_maps(W4Maps& m, const W4Call& c, const W4Acts& x, int x_rows, int w_rows) {
    const uint64_t xd[2] = {(uint64_t)c.k, (uint64_t)c.m}, xs[1] = {(uint64_t)x.ld * 2};
    const uint32_t xb[2] = {64, (uint32_t)x_rows};
    int st = encode_tmap(&m.x, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, x.part[0], xd, xs, xb, CU_TENSOR_MAP_SWIZZLE_128B);
    m.lo = m.x;
    if (!st && x.part[1]) st = encode_tmap(&m.lo, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, x.part[1], xd, xs, xb, CU_TENSOR_MAP_SWIZZLE_128B);
    const int nmat = c.w[1].packed ? 2 : 1;
    const uint64_t kt = (uint64_t)w4_tiles_k(c.k), nt = (uint64_t)ceil_div(c.n, kTileRows), sb = 32 * (uint64_t)c.gpt;
    for (int i = 0; i < nmat && !st; ++i) {
        const uint64_t wd[4] = {64, 16, kt, nt}, ws[3] = {64, 1024, kt * 1024};
        const uint32_t wb[4] = {64, 16, 1, (uint32_t)w_rows / 16};
        st = encode_tmap(&m.w[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, c.w[i].packed, wd, ws, wb, CU_TENSOR_MAP_SWIZZLE_64B);
        const uint64_t sd[3] = {sb, kt, nt}, ss[2] = {sb, kt * sb};
        const uint32_t bb[3] = {(uint32_t)sb, 1, (uint32_t)w_rows / 16};
        if (!st) st = encode_tmap(&m.s[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, c.w[i].scales, sd, ss, bb, CU_TENSOR_MAP_SWIZZLE_NONE);
    }
    if (nmat == 1) m.w[1] = m.w[0], m.s[1] = m.s[0];
    return st;
}

template <auto kernel>
static cudaError_t launch_maps(dim3 grid, int threads, int smem, int parts, cudaStream_t s, const W4Maps& m, const GemmW4Params& p) {
    static std::atomic<uint64_t> allowed{0};
    const cudaError_t e = w4_allow_smem(kernel, smem, allowed);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
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
static cudaError_t launch_gemm_w4(bool small, int npairs, const W4Maps& m, GemmW4Params p, cudaStream_t s) {
    p.seg_blocks = p.y_dtype == SBQ_F32 ? kSegSteps / (8 * PARTS) : p.kt;
    if (small)
        return launch_maps<gemm_w4_small_kernel<PARTS, NMAT, GPT>>(
                           dim3((unsigned)ceil_div(p.n, kW4Rows / NMAT), (unsigned)ceil_div(p.m, kSTok4), (unsigned)p.parts),
                           kW4Threads, W4Small<PARTS>::kBytes, p.parts, s, m, p);
    return launch_maps<gemm_w4_pair_kernel<PARTS, NMAT, GPT>>(dim3(2 * (unsigned)npairs), kPairThreads,
                       W4Pair<PARTS, NMAT>::kBytes, 0, s, m, p);
}

template <int PARTS, int NMAT>
static cudaError_t launch_gemm_w4_g(int gpt, bool small, int npairs, const W4Maps& m, const GemmW4Params& p, cudaStream_t s) {
    if (gpt == 1) return launch_gemm_w4<PARTS, NMAT, 1>(small, npairs, m, p, s);
    if (gpt == 2) return launch_gemm_w4<PARTS, NMAT, 2>(small, npairs, m, p, s);
    return launch_gemm_w4<PARTS, NMAT, 4>(small, npairs, m, p, s);
}

// Which kernel, and its schedule, by a model of the time (us) fitted to measurements on B200 (k 2560 to 12288, n 1024 to
// 12288, 130 to 1024 rows; mostly within 10 %).  It counts blocks of 128 k on the longest path.
//   Pair kernel: eight MMAs per block (two parts of x: sixteen, and two more for the pauses in which the accumulator is
//   read) of 50 + 0.39 N cycles, or what it takes to bring and convert the operands, whichever is longer; tiles in rounds over the pairs, the
//   last round's cut along k or not.  Cutting costs 3 us (a second launch) and 80 ns for every part's 256 KiB of sums,
//   and the cut tiles end no earlier than the stores of the round before.
//   Small kernel: 64 tokens per tile, two CTAs per SM; with k split a CTA shares its SM all the time.
// Fp16 rows: 200 x 4096 x 4096 18.6 us (16 tiles in four parts; 64 narrow tiles uncut 23.0), 300 x 9728 x 2560 27.1 (20 in three;
// uncut 46.8), 512 x 4096 x 4096 23.9 (64 uncut), 300 x 4096 x 1024 11.7 with the small kernel (cut tiles 14.8, uncut 21.0).
struct W4Plan {
    int small_parts;  // small kernel: CTAs of a cluster along k; 0: pair kernel
    int tok, npairs, rounds, tail_tiles, tail_parts;
};

static W4Plan w4_plan(int64_t m, int64_t n, int64_t k, bool split, int nmat) {
    const int64_t sms = w4_sm_count(), pairs = sms / 2, kt = w4_tiles_k(k);
    W4Plan best{};
    // k parts per tile (the cluster size): the largest power of two up to 8 that keeps the grid within 7/8 of the
    // CTA slots (two per SM) and gives every part at least two blocks.  A cluster needs all of its CTAs in one
    // GPC at once: 64 x 4096 x 12288 (96 tiles) takes 20.1 us with 2 parts, 28.2 us with 3 (288 of 296 slots)
    const int64_t small_tiles = ceil_div(n, kW4Rows / nmat) * ceil_div(m, kSTok4);
    int64_t parts = 1;
    while (parts < 8 && small_tiles * (2 * parts) * 8 <= 2 * sms * 7 && kt / (2 * parts) >= 2) parts *= 2;
    best.small_parts = (int)parts;
    if (m <= kSTok4) return best;  // a pair's tile would be no fuller
    const int64_t waves = ceil_div(small_tiles * parts, 2 * sms);
    const double small_block = parts > 1 ? (split ? 1.4 : 0.84) : waves > 1 ? (split ? 1.25 : 0.68) : (split ? 1.15 : 0.57);
    // its token tiles are the grid's y dimension: above 65535 of them the pair kernel takes the call
    double best_t = ceil_div(m, kSTok4) > 65535 ? 1e30 : (split ? 7.5 : 6.5) + (double)(waves * ceil_div(kt, parts)) * small_block;
    // with two matrices a taker warpgroup finishes whole sets of 32 tokens
    const int set = 32 * nmat, widest = m < kTok ? (int)ceil_div(m, set) * set : kTok;
    for (int tok = widest; tok >= set; tok -= set) {
        const int64_t tiles = ceil_div(n, 2 * kW4Rows / nmat) * ceil_div(m, tok), rounds = tiles / pairs, tail = tiles % pairs;
        const double mma = (split ? 18 : 8) * (50 + 0.39 * tok) / 1850, least = split ? 0.92 : 0.53,
                     block = mma > least ? mma : least, fixed = (split ? 10 : 8) + (double)(rounds * kt) * block;
        for (int64_t cut = 1; cut == 1 || (cut <= 16 && cut * tail <= pairs && 2 * cut <= kt); ++cut) {
            double end = tail > 0 ? (double)ceil_div(kt, cut) * block : 0.0;
            if (cut > 1) {
                if (rounds > 0 && end < 8.0) end = 8.0;
                end += 3.0 + 0.08 * (double)(cut * tail) * tok / kTok;
            }
            // a schedule with more tiles or parts must gain 3 %: it reads more than the model knows
            if (fixed + end < 0.97 * best_t) {
                best_t = fixed + end;
                best = W4Plan{0, tok, (int)(rounds > 0 ? pairs : tail * cut), (int)rounds, (int)tail, (int)cut};
            }
            if (tail == 0) break;
        }
    }
    return best;
}

size_t gemm_w4_workspace(int64_t m, int64_t n, int64_t k, bool split, int nmat) {
    const W4Plan pl = w4_plan(m, n, k, split, nmat);
    return !pl.small_parts && pl.tail_parts > 1 ? (size_t)pl.tail_tiles * pl.tail_parts * kTok * 2 * kW4Rows * 4 : 0;
}

void gemm_w4_plan(int64_t m, int64_t n, int64_t k, bool split, int nmat, int* plan) {
    const W4Plan pl = w4_plan(m, n, k, split, nmat);
    plan[0] = pl.small_parts ? 1 : 2;
    plan[1] = pl.small_parts ? kSTok4 : pl.tok;
    plan[2] = pl.small_parts ? pl.small_parts : pl.tail_parts;
    plan[3] = pl.small_parts ? 0 : pl.rounds;
}

int gemm_w4_run(const W4Call& c, const W4Acts& x) {
    const int nmat = c.w[1].packed ? 2 : 1, ch = kW4Rows / nmat;
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
    const W4Plan pl = w4_plan(c.m, c.n, c.k, x.part[1] != nullptr, nmat);
    const bool small = pl.small_parts > 0;
    if (small) {
        p.parts = pl.small_parts;
    } else {
        p.rounds = pl.rounds;
        p.tail_tiles = pl.tail_tiles;
        p.tail_parts = pl.tail_parts;
        p.tok = pl.tok;
        p.partial = static_cast<float*>(x.scratch);
    }
    W4Maps maps;
    const int st = make_maps(maps, c, x, small ? kSTok4 : p.tok / 2, ch);
    if (st) return st;
    cudaError_t e = x.part[1] ? (nmat == 2 ? launch_gemm_w4_g<2, 2>(c.gpt, small, pl.npairs, maps, p, c.stream)
                                           : launch_gemm_w4_g<2, 1>(c.gpt, small, pl.npairs, maps, p, c.stream))
                              : (nmat == 2 ? launch_gemm_w4_g<1, 2>(c.gpt, small, pl.npairs, maps, p, c.stream)
                                           : launch_gemm_w4_g<1, 1>(c.gpt, small, pl.npairs, maps, p, c.stream));
    if (e == cudaSuccess && p.tail_parts > 1) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)(kTok / (4 * nmat)), (unsigned)pl.tail_tiles);
        cfg.blockDim = dim3(2 * kW4Rows);
        cfg.stream = c.stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        e = nmat == 2 ? cudaLaunchKernelEx(&cfg, w4_reduce_kernel<2>, p, pl.npairs)
                      : cudaLaunchKernelEx(&cfg, w4_reduce_kernel<1>, p, pl.npairs);
    }
    if (e != cudaSuccess) return set_error(SBQ_ERR_CUDA, "gemm_w4 launch: %s", cudaGetErrorString(e));
    return check_launch("gemm_w4");
}

}  // namespace sbq
