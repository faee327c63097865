// Decode product of 4-bit weights with group scales, and its fused gate/up form:
//
//   y[m, n] = sum_g s[n, g] * (sum_{k in g} x[m, k] q[n, k]) (+ bias[n])         m <= 16
//   h[m, n] = silu(gate[m, n]) * up[m, n], gate and up as y with their own weights
//
// The weight's bytes bound it: half a byte and a share of a scale per weight, read once.  A CTA's warps split the k
// tiles of a 16-channel tile row (W warps per tile row); a warp walks through its tiles of all of its CTA's tile
// rows as one stream and keeps DEPTH - 1 of them on the way into shared memory (each lane copies what it will read
// itself, so no barrier is needed; held in registers the same depth spilled), also across tile rows and, at the
// start, across the wait for the previous kernel.  Per tile: two 16-byte reads of codes per lane, q in fp16 or bf16 (exact
// integers), m16n8k16 tensor-core products with the rows of x as the n dimension (columns past m repeat row 0 and
// are dropped), fp32 partial sums per group that are scaled and added in fp32.  So the weight takes part exactly
// and every sum is fp32; the order of the additions is fixed.
//
// With two streams (gate and up, or two tile rows of one weight) a fragment of x serves two tiles (four: slower, the
// registers leave one CTA per SM).
//
// Measured on B200, groups of 128: 1 x 2560 x 151936 42 us with fp16 x (4.8 TB/s of weight and scales, 0.73 of the copy
// rate) and 47 us with bf16; gate/up 1 x 4096 x 12288 14.6 us (3.6 TB/s; up to 19 on some machines); 1 x 4096 x 4096
// 4.5 us, of which an empty launch is 2.6.  Long launches are bound by instruction issue: 141 instructions per 1 KiB tile
// (bf16 157), 72 (88) of them the conversion, at 2.4 per cycle and SM (counted with ncu on the first two).
#include "w4.cuh"
#include "w4_host.cuh"

namespace sbq {

constexpr int kG4Warps = 8;
constexpr int kG4Threads = kG4Warps * 32;

struct GemvW4Params {
    const uint8_t* x[2];     // 16-bit activation [m, k]; x[1]: low part of a split fp32 activation
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
    int units;               // CTA-sized pieces: 8 / wsplit tile rows per stream each
};

// Copies of `BYTES` (4, 8, 16) from global to shared memory, counted in groups per thread.
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
    if (BYTES == 16)
        asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint32_t word_of(const uint4& v, int w) { return w == 0 ? v.x : w == 1 ? v.y : w == 2 ? v.z : v.w; }

// m16n8k16 product, d = a b (first) or d += a b.
template <bool BF16>
__device__ __forceinline__ void mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1, bool first) {
    if (!first) {
        BF16 ? mma_bf16(d, a0, a1, a2, a3, b0, b1) : mma_f16(d, a0, a1, a2, a3, b0, b1);
        return;
    }
    if (BF16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// Shared memory of one instance: [warp][slot][stream]: codes (1 KiB), then every lane's scales.
template <int NSTR, int GPT>
struct GemvW4Smem {
    static constexpr int kDepth = NSTR == 2 ? 4 : 6;
    static constexpr int kTile = kW4TileBytes + 128 * GPT;
    static constexpr int kWarp = kDepth * NSTR * kTile;
    static constexpr int kBytes = kG4Warps * kWarp;
};

template <bool BF16, int MT, int PARTS, int NSTR, bool GATED, int GPT>
__global__ void __launch_bounds__(kG4Threads, MT * PARTS * NSTR == 1 ? 3 : 2) gemv_w4_kernel(const GemvW4Params p) {
    using SM = GemvW4Smem<NSTR, GPT>;
    constexpr int DEPTH = SM::kDepth;
    __shared__ float red[2][kG4Warps][NSTR][MT * 8][17];
    extern __shared__ __align__(128) uint8_t ring[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int W = p.wsplit, rows_per_unit = kG4Warps / W, KT = p.kt_total, ks = warp % W;
    const int cnt = (KT - ks + W - 1) / W;  // this warp's tiles of a tile row (W <= KT)
    const int my_units = (p.units - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x, total = my_units * cnt;

    // ---- the stream of tiles: (unit, k tile) of the next copy, and its slot
    int pu = blockIdx.x, pk = ks;
    const uint8_t* wp[NSTR];
    const uint32_t* sp[NSTR];
    // this lane's codes in a slot are at 16 * lane (+ 512), its scales at kW4TileBytes + 4 GPT * lane
    uint8_t* const ring0 = ring + warp * SM::kWarp + lane * 16;
    const int scale_off = kW4TileBytes + lane * (4 * GPT - 16);
    constexpr int kSlot = NSTR * SM::kTile;
    const uint32_t put0 = (uint32_t)__cvta_generic_to_shared(ring0);
    uint32_t put = put0;
    auto seek = [&]() {
#pragma unroll
        for (int a = 0; a < NSTR; ++a) {
            int tr = (pu * rows_per_unit + warp / W) * (GATED ? 1 : NSTR) + (GATED ? 0 : a);
            tr = tr < p.tile_rows ? tr : p.tile_rows - 1;  // past the last tile row: its results are dropped
            const int64_t tile = (int64_t)tr * KT + ks;
            wp[a] = p.w[GATED ? a : 0] + tile * kW4TileBytes + lane * 16;
            sp[a] = p.s[GATED ? a : 0] + (tile * 8 + g) * GPT;
        }
    };
    auto issue = [&]() {
        if (pu < p.units) {
#pragma unroll
            for (int a = 0; a < NSTR; ++a) {
                const uint32_t dst = put + a * SM::kTile;
                copy_async<16>(dst, wp[a]);
                copy_async<16>(dst + 512, wp[a] + 512);
                copy_async<4 * GPT>(dst + scale_off, sp[a]);
                wp[a] += (int64_t)W * kW4TileBytes;
                sp[a] += W * 8 * GPT;
            }
            pk += W;
            if (pk >= KT) {
                pk = ks;
                pu += gridDim.x;
                if (pu < p.units) seek();
            }
        }
        put = put == put0 + (DEPTH - 1) * kSlot ? put0 : put + kSlot;
        copy_commit();
    };
    seek();
#pragma unroll
    for (int d = 0; d < DEPTH - 1; ++d) issue();
    asm volatile("griddepcontrol.wait;" ::: "memory");  // x, and y
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // this lane's x of the tile that is consumed next: rows g (and 8 + g), columns 8 t .. of each word
    const uint8_t* xp[PARTS][MT];
#pragma unroll
    for (int q = 0; q < PARTS; ++q)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const int row = 8 * mt + g < p.m ? 8 * mt + g : 0;
            xp[q][mt] = p.x[q] + ((int64_t)row * p.ldx + 8 * t + ks * kW4TileCols) * 2;
        }
    float acc[NSTR][MT][4];
    auto clear = [&]() {
#pragma unroll
        for (int a = 0; a < NSTR; ++a)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[a][mt][e] = 0.0f;
    };
    clear();

    auto consume = [&](const uint4 (&ca)[NSTR], const uint4 (&cb)[NSTR], const uint32_t (&sc)[NSTR][GPT], int kt) {
        constexpr bool AHEAD = PARTS * MT < 4;  // the tile's x at once, or (64 registers of it) word by word
        uint4 xv[4][PARTS][MT];
        const int left = p.k - kt * kW4TileCols - 8 * t;  // columns of x from this lane's first on
        auto load_x = [&](int w0, int w1) {
#pragma unroll
            for (int w = w0; w < w1; ++w)
#pragma unroll
                for (int q = 0; q < PARTS; ++q)
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        if (left >= kW4TileCols - 24) {
                            xv[w][q][mt] = *reinterpret_cast<const uint4*>(xp[q][mt] + 64 * w);
                        } else {
                            // x past k must read as zero (0 * inf is not), and not be touched
                            xv[w][q][mt] = make_uint4(0, 0, 0, 0);
                            if (32 * w < left) xv[w][q][mt] = *reinterpret_cast<const uint4*>(xp[q][mt] + 64 * w);
                        }
                    }
        };
        if (AHEAD) load_x(0, 4);
#pragma unroll
        for (int gi = 0; gi < GPT; ++gi) {
            float part[NSTR][MT][4];
#pragma unroll
            for (int w = gi * (4 / GPT); w < (gi + 1) * (4 / GPT); ++w) {
                if (!AHEAD) load_x(w, w + 1);
#pragma unroll
                for (int a = 0; a < NSTR; ++a) {
                    uint32_t h0[4], h1[4];
                    if (BF16) {
                        w4_to_bf16(word_of(ca[a], w), h0);
                        w4_to_bf16(word_of(cb[a], w), h1);
                    } else {
                        w4_to_half(word_of(ca[a], w), h0);
                        w4_to_half(word_of(cb[a], w), h1);
                    }
#pragma unroll
                    for (int q = 0; q < PARTS; ++q)
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            const uint4 v = xv[w][q][mt];
                            mma_first<BF16>(part[a][mt], h0[0], h1[0], h0[1], h1[1], v.x, v.y, w == gi * (4 / GPT) && q == 0);
                            mma_first<BF16>(part[a][mt], h0[2], h1[2], h0[3], h1[3], v.z, v.w, false);
                        }
                }
            }
#pragma unroll
            for (int a = 0; a < NSTR; ++a) {
                const float s0 = __uint_as_float(sc[a][gi] << 16), s1 = __uint_as_float(sc[a][gi] & 0xFFFF0000u);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    acc[a][mt][0] = fmaf(s0, part[a][mt][0], acc[a][mt][0]);
                    acc[a][mt][1] = fmaf(s0, part[a][mt][1], acc[a][mt][1]);
                    acc[a][mt][2] = fmaf(s1, part[a][mt][2], acc[a][mt][2]);
                    acc[a][mt][3] = fmaf(s1, part[a][mt][3], acc[a][mt][3]);
                }
            }
        }
    };

    // ---- end of a unit: the warps' sums meet in shared memory (two buffers: one barrier per unit)
    int done = 0;
    auto finish = [&]() {
        const int unit = (int)blockIdx.x + done * (int)gridDim.x;
        float(*rb)[NSTR][MT * 8][17] = red[done & 1];
#pragma unroll
        for (int a = 0; a < NSTR; ++a)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int e = 0; e < 4; ++e) rb[warp][a][8 * mt + 2 * t + (e & 1)][g + 8 * (e >> 1)] = acc[a][mt][e];
        // the W warps of a tile row, by a barrier of their own
        const int tl = warp / W;
        if (W == 1)
            __syncwarp();
        else
            asm volatile("bar.sync %0, %1;" ::"r"(1 + tl), "r"(32 * W) : "memory");
        constexpr int outs = GATED ? 1 : NSTR;
        for (int e = ks * 32 + lane; e < outs * 16 * p.m; e += 32 * W) {
            const int r = e & 15, a0 = (e >> 4) % outs, tok = (e >> 4) / outs;
            const int64_t n = ((int64_t)(unit * rows_per_unit + tl) * outs + a0) * 16 + r;
            if (n >= p.n) continue;
            float v[2] = {0.0f, 0.0f};
            for (int w = 0; w < W; ++w) {
                v[0] += rb[tl * W + w][a0][tok][r];
                if (GATED) v[1] += rb[tl * W + w][NSTR - 1][tok][r];
            }
            if (p.xinv) {
                const float f = __ldg(p.xinv + tok);
                v[0] *= f, v[1] *= f;
            }
            const float out = GATED ? w4_silu(v[0]) * v[1] : p.bias ? v[0] + __ldg(p.bias + n) : v[0];
            w4_store(p.y, p.y_dtype, (int64_t)tok * p.ldy + n, out);
        }
        ++done;
        clear();
    };

    int kt = ks;
    const uint8_t* get = ring0;
    for (int i = 0; i < total; ++i) {
        copy_wait<DEPTH - 2>();  // tile i is here
        uint4 ca[NSTR], cb[NSTR];
        uint32_t sc[NSTR][GPT];
#pragma unroll
        for (int a = 0; a < NSTR; ++a) {
            const uint8_t* src = get + a * SM::kTile;
            ca[a] = *reinterpret_cast<const uint4*>(src);
            cb[a] = *reinterpret_cast<const uint4*>(src + 512);
#pragma unroll
            for (int gi = 0; gi < GPT; ++gi) sc[a][gi] = *reinterpret_cast<const uint32_t*>(src + scale_off + 4 * gi);
        }
        issue();  // into the slot of tile i - 1, whose values have been used
        get = get == ring0 + (DEPTH - 1) * kSlot ? ring0 : get + kSlot;
        consume(ca, cb, sc, kt);
        kt += W;
        const bool end = kt >= KT;
        const int64_t step = (int64_t)(end ? ks - kt + W : W) * (2 * kW4TileCols);
#pragma unroll
        for (int q = 0; q < PARTS; ++q)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) xp[q][mt] += step;
        if (end) {
            kt = ks;
            finish();
        }
    }
    copy_wait<0>();
}

template <bool BF16, int MT, int PARTS, int NSTR, bool GATED, int GPT>
static cudaError_t launch_gemv_w4(GemvW4Params p, cudaStream_t s) {
    auto kernel = gemv_w4_kernel<BF16, MT, PARTS, NSTR, GATED, GPT>;
    constexpr int smem = GemvW4Smem<NSTR, GPT>::kBytes;
    static std::atomic<uint64_t> allowed{0};
    const cudaError_t e = w4_allow_smem(kernel, smem, allowed);
    if (e != cudaSuccess) return e;
    // CTAs that fit on an SM at once (the same on every device the library runs on)
    static const int per_sm = [&] {
        int c = 0;
        return cudaOccupancyMaxActiveBlocksPerMultiprocessor(&c, kernel, kG4Threads, smem) == cudaSuccess && c > 0 ? c : 1;
    }();
    const int slots = per_sm * w4_sm_count(), rows = GATED ? 1 : NSTR;
    // Warps per tile row: the fewest steps on the longest path - rounds of units over the CTA slots, each a warp's
    // tiles and about two more for the joining of the sums.
    int64_t best = INT64_MAX;
    for (int w = 1; w <= 8 && w <= p.kt_total; w *= 2) {
        const int64_t units = ceil_div(p.tile_rows, (int64_t)(kG4Warps / w) * rows);
        const int64_t steps = ceil_div(units, slots) * (ceil_div(p.kt_total, w) * NSTR + 2);
        if (steps <= best) best = steps, p.wsplit = w, p.units = (int)units;
    }
    return w4_launch(kernel, (unsigned)(p.units < slots ? p.units : slots), kG4Threads, smem, s, p);
}

template <bool BF16, int MT, int PARTS, int NSTR, bool GATED>
static cudaError_t launch_gemv_w4_g(const GemvW4Params& p, int gpt, cudaStream_t s) {
    if (gpt == 1) return launch_gemv_w4<BF16, MT, PARTS, NSTR, GATED, 1>(p, s);
    if (gpt == 2) return launch_gemv_w4<BF16, MT, PARTS, NSTR, GATED, 2>(p, s);
    return launch_gemv_w4<BF16, MT, PARTS, NSTR, GATED, 4>(p, s);
}

template <int MT, int NSTR, bool GATED>
static cudaError_t launch_gemv_w4_x(const GemvW4Params& p, bool bf16, int gpt, cudaStream_t s) {
    if (p.x[1]) return launch_gemv_w4_g<false, MT, 2, NSTR, GATED>(p, gpt, s);
    if (bf16) return launch_gemv_w4_g<true, MT, 1, NSTR, GATED>(p, gpt, s);
    return launch_gemv_w4_g<false, MT, 1, NSTR, GATED>(p, gpt, s);
}

int gemv_w4_run(const W4Call& c, const W4Acts& x) {
    GemvW4Params p{};
    p.m = (int)c.m;
    p.ldx = x.ld;
    p.xinv = x.inv;
    for (int i = 0; i < 2; ++i) {
        p.x[i] = static_cast<const uint8_t*>(x.part[i]);
        p.w[i] = c.w[i].packed;
        p.s[i] = reinterpret_cast<const uint32_t*>(c.w[i].scales);
    }
    p.bias = c.bias;
    p.y = c.y;
    p.ldy = c.ldy;
    p.y_dtype = c.y_dtype;
    p.n = (int)c.n;
    p.k = (int)c.k;
    p.kt_total = (int)w4_tiles_k(c.k);
    p.tile_rows = (int)ceil_div(c.n, kTileRows);
    // two tile rows per warp where there are plenty of them
    const bool two = p.tile_rows >= 8 * w4_sm_count();
    cudaError_t e;
    if (p.m > 8)
        e = c.w[1].packed ? launch_gemv_w4_x<2, 2, true>(p, x.bf16, c.gpt, c.stream)
            : two         ? launch_gemv_w4_x<2, 2, false>(p, x.bf16, c.gpt, c.stream)
                          : launch_gemv_w4_x<2, 1, false>(p, x.bf16, c.gpt, c.stream);
    else
        e = c.w[1].packed ? launch_gemv_w4_x<1, 2, true>(p, x.bf16, c.gpt, c.stream)
            : two         ? launch_gemv_w4_x<1, 2, false>(p, x.bf16, c.gpt, c.stream)
                          : launch_gemv_w4_x<1, 1, false>(p, x.bf16, c.gpt, c.stream);
    if (e != cudaSuccess) return set_error(SBQ_ERR_CUDA, "gemv_w4 launch: %s", cudaGetErrorString(e));
    return check_launch("gemv_w4");
}

}  // namespace sbq
