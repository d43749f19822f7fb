// Products with 4-bit weights for sm_100a: y = x W^T, its gradient with respect
// to x and to the group scales, for one matrix or one per run of rows.
//
// e q has at most 4 + 4 significant bits, so it is a bfloat16 (and a float16)
// without rounding: the tensor cores multiply it by the activations exactly
// and add in float32; the matrix's s multiplies the finished sum.
#include "uq_q4.cuh"
#include "uq_tc5.cuh"

#include <algorithm>

namespace {

using namespace uq::q4;
namespace tc5 = uq::tc5;
namespace tma = uq::tma;

__device__ int g_mm_bad_offset, g_mm_timeout;

// ----------------------------------------------------------------------------
// Tiles: 128 weight columns of the result by up to `bt` rows of one matrix's
// run, by one of `splits` parts of the contraction.
// ----------------------------------------------------------------------------
struct Runs {
    const int32_t *offsets;   // null: one matrix, all rows
    int64_t T, mats;
    int bt;                   // rows of a tile
    int wtiles, splits;
};

struct Tile {
    int64_t mat, row0;
    int rows, wt, split;
};

// Finds a warp's tiles in rising order: the 32 lanes hold 32 matrices' runs at a
// time.  An offset counts as at least its predecessors and at most T.
struct Finder {
    int64_t first, base, lo, hi, incl, top, begin;   // matrices and row tiles before this block of 32; this lane's run
    bool loaded;

    __device__ __forceinline__ void start(const Runs &r) {
        first = base = 0;
        loaded = false;
        if (r.offsets) {
            const int64_t o = r.offsets[0];
            top = min(max(o, int64_t(0)), r.T);
            if (o != top) g_mm_bad_offset = 1;
        } else {
            top = 0;
        }
        begin = top;
    }
    __device__ __forceinline__ void load(const Runs &r) {
        const int lane = threadIdx.x & 31;
        const int64_t i = first + lane;
        int64_t o = i < r.mats ? int64_t(r.offsets[i + 1]) : 0;
        int64_t m = i < r.mats ? min(max(o, int64_t(0)), r.T) : 0;
        m = max(m, top);
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, m, d);
            if (lane >= d) m = max(m, v);
        }
        if (i < r.mats && o != m) g_mm_bad_offset = 1;
        hi = m;
        lo = __shfl_up_sync(0xffffffffu, m, 1);
        if (lane == 0) lo = top;
        incl = (hi - lo + r.bt - 1) / r.bt;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, incl, d);
            if (lane >= d) incl += v;
        }
        top = __shfl_sync(0xffffffffu, hi, 31);
        loaded = true;
    }
    // Tile number `t`; false beyond the last.
    __device__ __forceinline__ bool find(const Runs &r, int64_t t, Tile &tile) {
        tile.split = int(t % r.splits);
        const int64_t u = t / r.splits;
        tile.wt = int(u % r.wtiles);
        const int64_t rt = u / r.wtiles;
        if (!r.offsets) {
            tile.mat = 0;
            tile.row0 = rt * r.bt;
            if (tile.row0 >= r.T) return false;
            tile.rows = int(min(r.T - tile.row0, int64_t(r.bt)));
            return true;
        }
        for (;;) {
            if (!loaded) {
                if (first >= r.mats) return false;
                load(r);
            }
            const int64_t all = __shfl_sync(0xffffffffu, incl, 31);
            if (rt < base + all) break;
            base += all;
            first += 32;
            loaded = false;
        }
        const int at = __popc(__ballot_sync(0xffffffffu, base + incl <= rt));   // runs that end before the tile
        const int64_t before = __shfl_sync(0xffffffffu, incl, at > 0 ? at - 1 : 0);
        const int64_t l = __shfl_sync(0xffffffffu, lo, at), h = __shfl_sync(0xffffffffu, hi, at);
        tile.mat = first + at;
        tile.row0 = l + (rt - base - (at > 0 ? before : 0)) * r.bt;
        tile.rows = int(min(h - tile.row0, int64_t(r.bt)));
        return true;
    }
    // The end of the last run, once find() has gone beyond the last tile.
    __device__ __forceinline__ int64_t end(const Runs &r) const { return r.offsets ? top : r.T; }
};

// ----------------------------------------------------------------------------
// Weights in 16-bit halves
// ----------------------------------------------------------------------------
// The pair (2 i, 2 i + 1) of a word as 16 + u in two halves: u moved to the top
// bits of the significand of 16.0.  Then e (16 + u) - 24 e = e q in one fused
// multiply-add: 24 e and e q have at most 8 bits, so nothing rounds.
template <bool BF16> struct Halves;
template <> struct Halves<true> {
    using T = __nv_bfloat16;
    static __device__ __forceinline__ uint32_t raw(uint32_t w, int i) {
        const uint32_t v = i == 0 ? w << 3 : w >> (4 * i - 3);
        return (v & 0x00780078u) | 0x41804180u;
    }
    static __device__ __forceinline__ uint32_t pair(float e) {
        const __nv_bfloat162 p = __float2bfloat162_rn(e);
        return *reinterpret_cast<const uint32_t *>(&p);
    }
    static __device__ __forceinline__ uint32_t fma(uint32_t a, uint32_t b, uint32_t c) {
        uint32_t d;
        asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
        return d;
    }
};
template <> struct Halves<false> {
    using T = __half;
    static __device__ __forceinline__ uint32_t raw(uint32_t w, int i) {
        const uint32_t v = i == 0 ? w << 6 : i == 1 ? w << 2 : w >> (4 * i - 6);
        return (v & 0x03c003c0u) | 0x4c004c00u;
    }
    static __device__ __forceinline__ uint32_t pair(float e) {
        const __half2 p = __float2half2_rn(e);
        return *reinterpret_cast<const uint32_t *>(&p);
    }
    static __device__ __forceinline__ uint32_t fma(uint32_t a, uint32_t b, uint32_t c) {
        uint32_t d;
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
        return d;
    }
};

// 32 codes of one group -> 16 registers of two halves each, in order.
template <bool BF16> __device__ __forceinline__ void widen32(const uint4 &c, float e, uint32_t *out) {
    const uint32_t s = Halves<BF16>::pair(e), z = Halves<BF16>::pair(-24.0f * e);
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) out[4 * j + i] = Halves<BF16>::fma(Halves<BF16>::raw(w[j], i), s, z);
}

__device__ __forceinline__ uint4 lds128(unsigned addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void sts128(unsigned addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" :: "r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

struct Weights {
    const uint8_t *scales;
    const float *scale;
    int64_t N, K;
    int gshift;       // group = 2^gshift
};

// The scale bytes that one lane needs for a chunk of four stages, in one word;
// 0 (e = 0, so that whatever the codes are the weights are 0) beyond the matrix.
// Forward: byte j is group j of the chunk's 256 values of weight row `row`.
// DX: bytes 0, 1 and 2, 3 are the two pieces of 32 values in this lane's row of
// stages `half` and `half` + 2.
template <bool DX>
__device__ __forceinline__ uint64_t chunk_scales(const Weights &w, const uint8_t *e0, int64_t groups, int64_t row, int wt, int stage, int half, int quad) {
    uint64_t v = 0;
    if (DX) {
        const int64_t k0 = int64_t(wt) * 128 + (quad >> 1) * 64;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t n = int64_t(stage + half + 2 * i) * 64 + (quad & 1) * 32 + (threadIdx.x & 31);
            if (n >= w.N) continue;
            const uint8_t *p = e0 + n * groups;
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (k0 + 32 * j < w.K) v |= uint64_t(__ldg(p + ((k0 + 32 * j) >> w.gshift))) << (16 * i + 8 * j);
        }
    } else if (row < w.N) {
        const int64_t g0 = (int64_t(stage) * 64) >> w.gshift;
        const int count = 256 >> w.gshift;   // 8, 4, 2 or 1, aligned where rows are whole chunks
        const uint8_t *p = e0 + g0;
        if ((w.K & 255) == 0) {
            if (count == 8) v = __ldg(reinterpret_cast<const unsigned long long *>(p));
            else if (count == 4) v = __ldg(reinterpret_cast<const unsigned *>(p));
            else if (count == 2) v = __ldg(reinterpret_cast<const unsigned short *>(p));
            else v = __ldg(p);
        } else {
            for (int j = 0; j < count; ++j)
                if (g0 + j < groups) v |= uint64_t(__ldg(p + j)) << (8 * j);
        }
    }
    return v;
}

struct Out {
    void *out;        // (rows, J) of 16 bits, or with splits the workspace: (splits, T, J) floats
    int64_t ld, J, T;
    bool zero_rest;
};

// Register j of lane i: row j, column i of a 32 x 32 piece of the result.
// Rows [0, rows) and columns below J are written; one row's 32 columns are one
// line of 64 (or 128) bytes.
template <bool BF16>
__device__ __forceinline__ void store_piece(const uint32_t (&r)[32], float s, const Out &o, int split, int splits, int64_t row0, int rows, int64_t col) {
    using T = typename Halves<BF16>::T;
    if (col >= o.J) return;
    if (splits > 1) {
        float *p = static_cast<float *>(o.out) + (int64_t(split) * o.T + row0) * o.J + col;
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (j < rows) p[int64_t(j) * o.J] = __uint_as_float(r[j]);
    } else {
        T *p = static_cast<T *>(o.out) + row0 * o.ld + col;
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (j < rows) p[int64_t(j) * o.ld] = from_float<T>(s * __uint_as_float(r[j]));
    }
}

// Rows outside every run, a share of them for each block's eight warps.
template <typename T> __device__ void zero_rows(const Out &o, int64_t begin, int64_t end) {
    const int64_t rest = o.T - (end - begin);
    for (int64_t i = blockIdx.x; i < rest; i += gridDim.x) {
        T *p = static_cast<T *>(o.out) + (i < begin ? i : end + i - begin) * o.ld;
        for (int64_t j = threadIdx.x; j < o.J; j += 256) p[j] = from_float<T>(0.0f);
    }
}

// ----------------------------------------------------------------------------
// The product kernel.  The result is formed transposed, weight columns in the
// 128 lanes of tensor memory and up to BT rows in its columns, so that few rows
// make a narrow instruction.  Stages of 64 contraction steps: `full_b` the rows'
// tile (TMA, 128-byte swizzle), `full_a` the widened weights, `empty` both free
// again.
//   forward: lane n; the weights go from registers into tensor memory (32
//            columns a stage), codes by TMA in chunks of 256 steps
//   DX:      lane k; a stage is 64 rows n of 128 codes, widened into shared
//            memory with k contiguous
// Warps 0 .. 7 widen (four a stage, in turn) and write results; warp 8 copies
// the rows, warp 9 the codes, warp 10 issues the products.
// ----------------------------------------------------------------------------
constexpr int kThreads = 352;

template <int BT, bool DX> struct Cfg {
    // stages: an even number, so that each slot is always widened by the same four warps
    static constexpr int NS = DX ? (BT == 256 ? 4 : 6) : BT == 256 ? 4 : BT == 128 ? 6 : 8;
    static constexpr int kChunks = DX ? (BT == 64 ? 4 : 2) : BT == 256 ? 4 : BT == 128 ? 6 : 8;
    static constexpr int kB = BT * 128, kA = DX ? 16384 : 0, kC = 16384;
    static constexpr int kBar = 3 * NS + 2 * kChunks + 2;
    static constexpr int kSmem = 1024 + NS * (kB + kA) + kChunks * kC + kBar * 8 + 16;
    static constexpr int kTmem = 512;
    static_assert(kSmem <= 232448, "shared memory of one block");
    static_assert(DX ? BT <= 512 : BT + 32 * NS <= 512, "tensor memory");
};

template <int BT, bool BF16, bool DX>
__global__ void __launch_bounds__(kThreads, 1)
q4_product_kernel(const __grid_constant__ CUtensorMap map_rows, const __grid_constant__ CUtensorMap map_codes, Runs runs, Weights w, Out o) {
    using C = Cfg<BT, DX>;
    constexpr int NS = C::NS, NC = C::kChunks, kBox = BT / 4;
    extern __shared__ uint8_t smem_raw[];
    const unsigned base = (tc5::smem_addr(smem_raw) + 1023u) & ~1023u;
    const unsigned sb = base, sa = sb + NS * C::kB, sc = sa + NS * C::kA, bars = sc + NC * C::kC;
    const unsigned full_b = bars, full_a = bars + 8 * NS, empty = bars + 16 * NS, full_c = bars + 24 * NS, empty_c = full_c + 8 * NC,
                   done = empty_c + 8 * NC, drained = done + 8, misc = drained + 8;
    volatile int *gave_up = reinterpret_cast<volatile int *>(smem_raw + (misc + 4 - tc5::smem_addr(smem_raw)));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == 10) tc5::tmem_alloc<C::kTmem>(misc);
    if (threadIdx.x == 0) {
        *gave_up = 0;
        for (int i = 0; i < NS; ++i) {
            tma::mbar_init(full_b + 8 * i, 1);
            tma::mbar_init(full_a + 8 * i, 4);
            tma::mbar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < NC; ++i) {
            tma::mbar_init(full_c + 8 * i, 1);
            tma::mbar_init(empty_c + 8 * i, 8);
        }
        tma::mbar_init(done, 1);
        tma::mbar_init(drained, 8);
        tma::mbar_init(misc + 8, 1);   // products in flight, where a wait gave up
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    tc5::fence_before();
    __syncthreads();
    tc5::fence_after();
    unsigned tmem;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(misc));
    const unsigned tmem_a = tmem + BT;

    tc5::Waiter wt{gave_up, &g_mm_timeout};
    Finder find;
    find.start(runs);
    Tile t;
    const int64_t depth = DX ? w.N : w.K;
    const int all = int((depth + 63) / 64);                                       // stages of the whole contraction
    const int per = runs.splits > 1 ? ((all + 4 * runs.splits - 1) / (4 * runs.splits)) * 4 : all;   // of one part, whole chunks
    unsigned it = 0, ct = 0, tiles = 0;                                           // stages, chunks, tiles so far

    if (warp == 8) {
        // rows
        for (int64_t tile = blockIdx.x; !wt.fail && find.find(runs, tile, t); tile += gridDim.x) {
            const int s0 = t.split * per, n = max(0, min(per, all - s0));
            const int boxes = (((t.rows + 15) & ~15) + kBox - 1) / kBox;
            for (int s = 0; s < n; ++s, ++it) {
                const int slot = it % NS;
                if (!wt.wait(empty + 8 * slot, ((it / NS) & 1) ^ 1)) break;
                if (lane == 0) {
                    tma::mbar_arrive_expect_tx(full_b + 8 * slot, boxes * kBox * 128);
                    for (int b = 0; b < boxes; ++b)
                        tma::load2d(sb + slot * C::kB + b * kBox * 128, &map_rows, (s0 + s) * 64, int(t.row0) + b * kBox, full_b + 8 * slot);
                }
            }
        }
        if (wt.fail)   // copies in flight land before the block ends
            for (unsigned i = it > NS ? it - NS : 0; i < it; ++i) tc5::Waiter::drain(full_b + 8 * (i % NS), (i / NS) & 1);
    } else if (warp == 9) {
        // codes: 128 rows of 256 codes, or 256 rows of 128
        for (int64_t tile = blockIdx.x; !wt.fail && find.find(runs, tile, t); tile += gridDim.x) {
            const int s0 = t.split * per, n = max(0, min(per, all - s0));
            for (int s = 0; s < n; s += 4, ++ct) {
                const int slot = ct % NC;
                if (!wt.wait(empty_c + 8 * slot, ((ct / NC) & 1) ^ 1)) break;
                if (lane == 0) {
                    tma::mbar_arrive_expect_tx(full_c + 8 * slot, C::kC);
                    const int64_t row = t.mat * w.N;
                    if (DX) tma::load2d(sc + slot * C::kC, &map_codes, t.wt * 64, int(row + (s0 + s) * 64), full_c + 8 * slot);
                    else tma::load2d(sc + slot * C::kC, &map_codes, (s0 + s) * 32, int(row + t.wt * 128), full_c + 8 * slot);
                }
            }
        }
        if (wt.fail)
            for (unsigned i = ct > NC ? ct - NC : 0; i < ct; ++i) tc5::Waiter::drain(full_c + 8 * (i % NC), (i / NC) & 1);
    } else if (warp == 10) {
        // products
        for (int64_t tile = blockIdx.x; !wt.fail && find.find(runs, tile, t); tile += gridDim.x, ++tiles) {
            const int s0 = t.split * per, n = max(0, min(per, all - s0));
            const uint32_t idesc = tc5::idesc_f16(BF16, (t.rows + 15) & ~15, DX, false);
            if (!wt.wait(drained, (tiles & 1) ^ 1)) break;
            for (int s = 0; s < n; ++s, ++it) {
                const int slot = it % NS;
                const unsigned par = (it / NS) & 1;
                if (!wt.wait(full_b + 8 * slot, par) || !wt.wait(full_a + 8 * slot, par)) break;
                tc5::fence_after();
                if (lane == 0) {
                    const uint64_t b = tc5::desc128(sb + slot * C::kB, 16, 1024);
                    const uint64_t a = tc5::desc128(sa + slot * C::kA, 8192, 1024);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if (DX) tc5::mma_ss(tmem, a + k * 128, b + k * 2, idesc, s > 0 || k > 0);
                        else tc5::mma_ts(tmem, tmem_a + slot * 32 + k * 8, b + k * 2, idesc, s > 0 || k > 0);
                    }
                    tc5::commit(empty + 8 * slot);
                }
                __syncwarp();
            }
            if (!wt.fail && lane == 0) tc5::commit(done);
            __syncwarp();
        }
        if (wt.fail) {   // products in flight end before the block does
            if (lane == 0) tc5::commit(misc + 8);
            __syncwarp();
            tc5::Waiter::drain(misc + 8, 0);
        }
    } else {
        // widen, then write the result
        const int half = warp >> 2, quad = warp & 3;
        const int64_t groups = w.K >> w.gshift;
        bool more;
        for (int64_t tile = blockIdx.x; (more = find.find(runs, tile, t)) && !wt.fail; tile += gridDim.x, ++tiles) {
            const int s0 = t.split * per, n = max(0, min(per, all - s0));
            const float scale = __ldg(w.scale + t.mat);
            const int64_t row = int64_t(t.wt) * 128 + quad * 32 + lane;   // forward: this lane's weight row
            const uint8_t *const e0 = w.scales + (t.mat * w.N + (DX ? 0 : min(row, w.N - 1))) * groups;
            uint64_t eraw = chunk_scales<DX>(w, e0, groups, row, t.wt, s0, half, quad);
            for (int c = 0; c < n; c += 4, ++ct) {
                const int cslot = ct % NC, cn = min(4, n - c);
                const unsigned cpar = (ct / NC) & 1;
                const uint64_t ecur = eraw;
                if (c + 4 < n) eraw = chunk_scales<DX>(w, e0, groups, row, t.wt, s0 + c + 4, half, quad);   // a chunk ahead
                bool seen = false;
                for (int s = half; s < cn; s += 2) {
                    const int slot = (it + s) % NS;
                    if (!seen && !wt.wait(full_c + 8 * cslot, cpar)) break;
                    seen = true;
                    if (!wt.wait(empty + 8 * slot, (((it + s) / NS) & 1) ^ 1)) break;
                    float e[2];
#pragma unroll
                    for (int p = 0; p < 2; ++p) e[p] = e4m3_value(uint8_t(ecur >> (8 * (DX ? (s & 2) + p : (2 * s + p) >> (w.gshift - 5)))));
                    if (DX) {
                        // row rr of 128 codes (64 bytes, 64-byte swizzle): this warp's 64 values are pieces 2 h, 2 h + 1
                        const int rr = s * 64 + (quad & 1) * 32 + lane, h = quad >> 1;
                        const unsigned line = sa + slot * C::kA + h * 8192 + ((quad & 1) * 32 + lane) * 128;
#pragma unroll
                        for (int p = 0; p < 2; ++p) {
                            uint32_t v[16];
                            widen32<BF16>(lds128(sc + cslot * C::kC + rr * 64 + (((2 * h + p) ^ ((rr >> 1) & 3)) << 4)), e[p], v);
#pragma unroll
                            for (int q = 0; q < 4; ++q)
                                sts128(line + (((4 * p + q) ^ (lane & 7)) << 4), v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
                        }
                        tma::fence_proxy_async();
                    } else {
                        const int rr = quad * 32 + lane;
                        uint32_t v[32];
#pragma unroll
                        for (int p = 0; p < 2; ++p)
                            widen32<BF16>(lds128(sc + cslot * C::kC + rr * 128 + (((2 * s + p) ^ (rr & 7)) << 4)), e[p], v + 16 * p);
                        tc5::fence_after();
                        tc5::st32(tmem_a + slot * 32 + (unsigned(quad * 32) << 16), v);
                        tc5::wait_st();
                        tc5::fence_before();
                    }
                    __syncwarp();
                    if (lane == 0) tc5::mbar_arrive(full_a + 8 * slot);
                }
                if (wt.fail) break;
                it += cn;
                __syncwarp();
                if (lane == 0) tc5::mbar_arrive(empty_c + 8 * cslot);
            }
            if (!wt.wait(done, tiles & 1)) break;
            tc5::fence_after();
            const int64_t col = int64_t(t.wt) * 128 + quad * 32 + lane;
            for (int c = half; c * 32 < t.rows; c += 2) {
                uint32_t r[32];
                tc5::ld32(tmem + c * 32 + (unsigned(quad * 32) << 16), r);
                tc5::wait_ld();
                if (n == 0) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) r[j] = 0;
                }
                store_piece<BF16>(r, scale, o, t.split, runs.splits, t.row0 + c * 32, t.rows - c * 32, col);
            }
            tc5::fence_before();
            __syncwarp();
            if (lane == 0) tc5::mbar_arrive(drained);
        }
        if (o.zero_rest && runs.offsets && !wt.fail) zero_rows<typename Halves<BF16>::T>(o, find.begin, find.end(runs));
    }
    __syncthreads();
    if (warp == 10) {
        tc5::fence_after();
        tc5::tmem_free<C::kTmem>(tmem);
    }
}

// ----------------------------------------------------------------------------
// Few rows: bound by reading the codes once.  A block takes 32 weight rows; its
// eight warps take every eighth step of 256 values of k each and add up in
// shared memory at the end, so that even a 4096 x 4096 matrix gives every SM
// 7 warps whose loads are all in flight at once.  The widened codes are operand
// A of m16n8k16 products straight from registers: the contraction order is free
// as long as both operands agree, so lane quarter q takes 64 consecutive values
// of a row (two 16-byte loads) where the instruction says "columns 2 q, 2 q + 1,
// 2 q + 8, 2 q + 9".  Widening costs the same for 1 row as for 8.
// ----------------------------------------------------------------------------
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool bf16) {
    if (bf16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

constexpr int kFewWarps = 8, kFewRows = 32;

// One lane's codes and scales of a step: 4 rows (g, g + 8, g + 16, g + 24) of 64 values.
struct Step {
    uint4 c[4][2];
    uint32_t e;        // two rows' bytes; see load_step
    uint32_t e2;
};

__device__ __forceinline__ void load_step(Step &st, const uint8_t *codes, const Weights &w, int64_t mrow, int64_t n0, int64_t k, int64_t groups) {
    const int g = (threadIdx.x & 31) >> 2;
    st.e = st.e2 = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t n = n0 + g + 8 * i;
        const uint8_t *c = codes + ((mrow + n) * w.K + k) / 2;
        const uint8_t *e = w.scales + (mrow + n) * groups;
        uint32_t eb = 0;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const bool in = n < w.N && k + 32 * p < w.K;
            st.c[i][p] = in ? __ldg(reinterpret_cast<const uint4 *>(c) + p) : make_uint4(0, 0, 0, 0);
            eb |= in ? uint32_t(__ldg(e + ((k + 32 * p) >> w.gshift))) << (8 * p) : 0u;
        }
        if (i < 2) st.e |= eb << (16 * i);
        else st.e2 |= eb << (16 * (i - 2));
    }
}

template <bool BF16, int NT>
__global__ void __launch_bounds__(256, 2)
q4_few_kernel(const void *x, int64_t ldx, const uint8_t *codes, Runs runs, Weights w, Out o, int section) {
    using T = typename Halves<BF16>::T;
    extern __shared__ __align__(16) uint8_t few_smem[];   // the rows of a section of k, then the warps' sums
    const unsigned sx = tc5::smem_addr(few_smem);
    float *const sums = reinterpret_cast<float *>(few_smem);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, q = lane & 3, tok = lane >> 2;
    const int64_t groups = w.K >> w.gshift;
    Finder find;
    find.start(runs);
    Tile t;
    for (int64_t tile = blockIdx.x; find.find(runs, tile, t); tile += gridDim.x) {
        const int64_t n0 = int64_t(t.wt) * kFewRows, mrow = t.mat * w.N;
        float acc[2][NT][4] = {};
        for (int64_t sec = 0; sec < w.K; sec += section) {
            const int len = int(min(w.K - sec, int64_t(section))), steps = (len + 255) >> 8;
            Step cur;
            int s = warp;
            if (s < steps) load_step(cur, codes, w, mrow, n0, sec + s * 256 + q * 64, groups);
            // rows into shared memory: 64 values a line, its eight pieces swizzled by the line's place in a step and the row
            __syncthreads();
            const int pieces = steps * 32;
            for (int r = 0; r < t.rows; ++r) {
                const T *src = static_cast<const T *>(x) + (t.row0 + r) * ldx + sec;
                for (int p = tid; p < pieces; p += 256) {
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (p * 8 < len) v = __ldg(reinterpret_cast<const uint4 *>(src + p * 8));
                    const int line = p >> 3, sw = (line & 3) | ((r & 1) << 2);
                    sts128(sx + ((r * steps * 4 + line) * 8 + ((p & 7) ^ sw)) * 16, v.x, v.y, v.z, v.w);
                }
            }
            __syncthreads();
            for (; s < steps; s += kFewWarps) {
                Step next;
                if (s + kFewWarps < steps) load_step(next, codes, w, mrow, n0, sec + (s + kFewWarps) * 256 + q * 64, groups);
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    uint32_t es[4], ez[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float e = e4m3_value(uint8_t((i < 2 ? cur.e : cur.e2) >> (16 * (i & 1) + 8 * p)));
                        es[i] = Halves<BF16>::pair(e);
                        ez[i] = Halves<BF16>::pair(-24.0f * e);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint4 b[NT];
#pragma unroll
                        for (int u = 0; u < NT; ++u) {
                            const int r = tok + 8 * u, sw = q | ((r & 1) << 2);
                            b[u] = make_uint4(0, 0, 0, 0);
                            if (r < t.rows) b[u] = lds128(sx + ((r * steps * 4 + s * 4 + q) * 8 + ((4 * p + j) ^ sw)) * 16);
                        }
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            uint32_t lo[4], hi[4];
                            const uint4 &c0 = cur.c[2 * m][p], &c1 = cur.c[2 * m + 1][p];
                            const uint32_t w0 = j == 0 ? c0.x : j == 1 ? c0.y : j == 2 ? c0.z : c0.w;
                            const uint32_t w1 = j == 0 ? c1.x : j == 1 ? c1.y : j == 2 ? c1.z : c1.w;
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                lo[i] = Halves<BF16>::fma(Halves<BF16>::raw(w0, i), es[2 * m], ez[2 * m]);
                                hi[i] = Halves<BF16>::fma(Halves<BF16>::raw(w1, i), es[2 * m + 1], ez[2 * m + 1]);
                            }
                            const uint32_t a0[4] = {lo[0], hi[0], lo[1], hi[1]}, a1[4] = {lo[2], hi[2], lo[3], hi[3]};
#pragma unroll
                            for (int u = 0; u < NT; ++u) {
                                mma16816(acc[m][u], a0, b[u].x, b[u].y, BF16);
                                mma16816(acc[m][u], a1, b[u].z, b[u].w, BF16);
                            }
                        }
                    }
                }
                cur = next;
            }
        }
        __syncthreads();
        // sums[warp][row of x][weight row]
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int u = 0; u < NT; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    sums[(warp * 8 * NT + 8 * u + 2 * q + (i & 1)) * kFewRows + 16 * m + tok + 8 * (i >> 1)] = acc[m][u][i];
        __syncthreads();
        const float scale = __ldg(w.scale + t.mat);
        for (int i = tid; i < 8 * NT * kFewRows; i += 256) {
            const int r = i / kFewRows, c = i % kFewRows;
            float v = 0.0f;
#pragma unroll
            for (int k = 0; k < kFewWarps; ++k) v += sums[(k * 8 * NT + r) * kFewRows + c];
            if (r < t.rows && n0 + c < w.N) static_cast<T *>(o.out)[(t.row0 + r) * o.ld + n0 + c] = from_float<T>(scale * v);
        }
        __syncthreads();
    }
    if (o.zero_rest && runs.offsets) zero_rows<T>(o, find.begin, find.end(runs));
}

// The parts of a split contraction, added in their order.
template <bool BF16>
__global__ void __launch_bounds__(256) q4_join_parts_kernel(const float *part, int splits, int64_t T, int64_t J, const float *scale, void *out, int64_t ld) {
    using Ty = typename Halves<BF16>::T;
    const float s = __ldg(scale);
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < T * J; i += int64_t(gridDim.x) * 256) {
        float v = part[i];
        for (int p = 1; p < splits; ++p) v += part[int64_t(p) * T * J + i];
        static_cast<Ty *>(out)[(i / J) * ld + i % J] = from_float<Ty>(s * v);
    }
}

// ----------------------------------------------------------------------------
// Gradient of the group scales: dW = dy^T x over the rows of a matrix, reduced
// with the codes before it leaves the chip (a 32nd to a 256th of dW is written).
// One tile: 128 rows n by 256 columns k; both operands come as lines of 64
// columns, one line per row t, in stages of 64 rows.  The sums of kPromote
// stages are taken from tensor memory (two accumulators in turn), multiplied by
// q and added in float32 registers, so that no long sum runs in the tensor core.
// Warps 0 .. 7 reduce, warp 8 copies, warp 9 issues, warp 10 clears the rows
// behind the last one of a run (they are another matrix's, and may be NaN).
// ----------------------------------------------------------------------------
constexpr int kPromote = 8, kBand = 12;

struct DsCfg {
    static constexpr int NS = 4, kA = 16384, kB = 32768, kBar = 3 * NS + 4;
    static constexpr int kSmem = 1024 + NS * (kA + kB) + kBar * 8 + 32 + 512;
};

struct DsTile {
    int64_t mat, lo, rows;
    int nt, kt;
};

// Tile number -> matrix, run and place.  Consecutive tiles of a matrix form
// bands of kBand row tiles, so that the blocks running at one time share both
// operands' lines in L2.
struct DsFinder {
    int64_t at = -1, top = 0, lo = 0;   // runs up to matrix `at` are read
    __device__ __forceinline__ bool find(const Runs &r, int64_t t, int ntiles, int ktiles, DsTile &d) {
        const int64_t per = int64_t(ntiles) * ktiles;
        d.mat = t / per;
        if (d.mat >= r.mats) return false;
        if (!r.offsets) {
            d.lo = 0;
            d.rows = r.T;
        } else {
            const int lane = threadIdx.x & 31;
            if (at < 0) {
                const int64_t o = r.offsets[0];
                top = min(max(o, int64_t(0)), r.T);
                if (o != top) g_mm_bad_offset = 1;
            }
            while (at < d.mat) {   // 32 offsets at a time: their running maximum
                const int64_t n = min(d.mat - at, int64_t(32)), i = at + 1 + min(int64_t(lane), n - 1);
                const int64_t o = r.offsets[i + 1];
                int64_t m = max(min(max(o, int64_t(0)), r.T), top);
#pragma unroll
                for (int s = 1; s < 32; s <<= 1) {
                    const int64_t v = __shfl_up_sync(0xffffffffu, m, s);
                    if (lane >= s) m = max(m, v);
                }
                if (o != m && lane < n) g_mm_bad_offset = 1;
                lo = n > 1 ? __shfl_sync(0xffffffffu, m, int(n) - 2) : top;
                top = __shfl_sync(0xffffffffu, m, int(n) - 1);
                at += n;
            }
            d.lo = lo;
            d.rows = top - lo;
        }
        const int64_t u = t - d.mat * per, band = u / (int64_t(kBand) * ktiles), v = u - band * kBand * ktiles;
        const int high = min(kBand, ntiles - int(band) * kBand);
        d.nt = int(band) * kBand + int(v % high);
        d.kt = int(v / high);
        return true;
    }
};

template <bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
q4_dscale_kernel(const __grid_constant__ CUtensorMap map_dy, const __grid_constant__ CUtensorMap map_x, Runs runs, const uint8_t *codes, int64_t N,
                 int64_t K, int gshift, int ntiles, int ktiles, float *dc) {
    using C = DsCfg;
    constexpr int NS = C::NS;
    extern __shared__ uint8_t smem_raw[];
    const unsigned base = (tc5::smem_addr(smem_raw) + 1023u) & ~1023u;
    const unsigned sa = base, sb = sa + NS * C::kA, bars = sb + NS * C::kB;
    const unsigned full = bars, fixed = full + 8 * NS, empty = fixed + 8 * NS, done = empty + 8 * NS, drained = done + 16, misc = drained + 16;
    uint8_t *const misc_ptr = smem_raw + (misc - tc5::smem_addr(smem_raw));
    volatile int *gave_up = reinterpret_cast<volatile int *>(misc_ptr + 4);
    const unsigned sums_full = misc + 16, sums_empty = misc + 24;
    float *const other = reinterpret_cast<float *>(misc_ptr + 32);   // 128 sums of the second half
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == 9) tc5::tmem_alloc<512>(misc);
    if (threadIdx.x == 0) {
        *gave_up = 0;
        for (int i = 0; i < NS; ++i) {
            tma::mbar_init(full + 8 * i, 1);
            tma::mbar_init(fixed + 8 * i, 1);
            tma::mbar_init(empty + 8 * i, 2);
        }
        for (int i = 0; i < 2; ++i) {
            tma::mbar_init(done + 8 * i, 1);
            tma::mbar_init(drained + 8 * i, 8);
        }
        tma::mbar_init(misc + 8, 1);
        tma::mbar_init(sums_full, 4);
        tma::mbar_init(sums_empty, 4);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    tc5::fence_before();
    __syncthreads();
    tc5::fence_after();
    unsigned tmem;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(misc));

    tc5::Waiter wt{gave_up, &g_mm_timeout};
    DsFinder find;
    DsTile t;
    unsigned it = 0, part = 0;   // stages, promoted parts so far

    if (warp == 8) {
        for (int64_t tile = blockIdx.x; !wt.fail && find.find(runs, tile, ntiles, ktiles, t); tile += gridDim.x) {
            const int n = int((t.rows + 63) / 64);
            for (int s = 0; s < n; ++s, ++it) {
                const int slot = it % NS;
                if (!wt.wait(empty + 8 * slot, ((it / NS) & 1) ^ 1)) break;
                if (lane == 0) {
                    tma::mbar_arrive_expect_tx(full + 8 * slot, C::kA + C::kB);
                    const int row = int(t.lo) + s * 64;
#pragma unroll
                    for (int c = 0; c < 2; ++c) tma::load2d(sa + slot * C::kA + c * 8192, &map_dy, t.nt * 128 + c * 64, row, full + 8 * slot);
#pragma unroll
                    for (int c = 0; c < 4; ++c) tma::load2d(sb + slot * C::kB + c * 8192, &map_x, t.kt * 256 + c * 64, row, full + 8 * slot);
                }
            }
        }
        if (wt.fail)
            for (unsigned i = it > NS ? it - NS : 0; i < it; ++i) tc5::Waiter::drain(full + 8 * (i % NS), (i / NS) & 1);
    } else if (warp == 10) {
        for (int64_t tile = blockIdx.x; !wt.fail && find.find(runs, tile, ntiles, ktiles, t); tile += gridDim.x) {
            const int n = int((t.rows + 63) / 64);
            for (int s = 0; s < n; ++s, ++it) {   // every stage, so that no phase of `full` goes by unseen
                const int slot = it % NS, left = int(min(t.rows - int64_t(s) * 64, int64_t(64)));
                if (!wt.wait(full + 8 * slot, (it / NS) & 1)) break;
                if (left & 15) {
                    const int rows = 16 - (left & 15);
                    for (int i = lane; i < rows * 48; i += 32) {   // 6 blocks of lines, 8 pieces a line
                        const int l = left + i / 48, b = i % 48;
                        const unsigned at = b < 16 ? sa + slot * C::kA + (b >> 3) * 8192 : sb + slot * C::kB + ((b - 16) >> 3) * 8192;
                        sts128(at + l * 128 + (b & 7) * 16, 0, 0, 0, 0);
                    }
                    tma::fence_proxy_async();
                }
                __syncwarp();
                if (lane == 0) {
                    if (left & 15) tc5::mbar_arrive(fixed + 8 * slot);
                    tc5::mbar_arrive(empty + 8 * slot);
                }
            }
        }
    } else if (warp == 9) {
        unsigned parity = 0;   // bit per slot: of its next clearing
        constexpr uint32_t idesc = tc5::idesc_f16(BF16, 256, true, true);
        for (int64_t tile = blockIdx.x; !wt.fail && find.find(runs, tile, ntiles, ktiles, t); tile += gridDim.x) {
            const int n = int((t.rows + 63) / 64);
            for (int s = 0; s < n; ++s, ++it) {
                const int slot = it % NS;
                const bool begin = s % kPromote == 0, end = s % kPromote == kPromote - 1 || s + 1 == n;
                if (begin && !wt.wait(drained + 8 * (part & 1), ((part >> 1) & 1) ^ 1)) break;
                if (!wt.wait(full + 8 * slot, (it / NS) & 1)) break;
                const int left = int(min(t.rows - int64_t(s) * 64, int64_t(64)));
                if (left & 15) {
                    if (!wt.wait(fixed + 8 * slot, (parity >> slot) & 1)) break;
                    parity ^= 1u << slot;
                }
                tc5::fence_after();
                if (lane == 0) {
                    const uint64_t a = tc5::desc128(sa + slot * C::kA, 8192, 1024), b = tc5::desc128(sb + slot * C::kB, 8192, 1024);
                    const int steps = (left + 15) >> 4;
                    for (int k = 0; k < steps; ++k) tc5::mma_ss(tmem + (part & 1) * 256, a + k * 128, b + k * 128, idesc, !begin || k > 0);
                    tc5::commit(empty + 8 * slot);
                    if (end) tc5::commit(done + 8 * (part & 1));
                }
                __syncwarp();
                part += end;
            }
        }
        if (wt.fail) {
            if (lane == 0) tc5::commit(misc + 8);
            __syncwarp();
            tc5::Waiter::drain(misc + 8, 0);
        }
    } else {
        const int half = warp >> 2, quad = warp & 3;
        const int64_t groups = K >> gshift;
        unsigned tiles = 0;
        for (int64_t tile = blockIdx.x; !wt.fail && find.find(runs, tile, ntiles, ktiles, t); tile += gridDim.x, ++tiles) {
            const int parts = int((t.rows + 64 * kPromote - 1) / (64 * kPromote));
            const int64_t n = int64_t(t.nt) * 128 + quad * 32 + lane, k0 = int64_t(t.kt) * 256 + half * 128;
            uint4 code[4];
            float sum[4] = {};
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                code[p] = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
                if (n < N && k0 + 32 * p < K) code[p] = __ldg(reinterpret_cast<const uint4 *>(codes + ((t.mat * N + n) * K + k0 + 32 * p) / 2));
            }
            for (int c = 0; c < parts; ++c, ++part) {
                if (!wt.wait(done + 8 * (part & 1), (part >> 1) & 1)) break;
                tc5::fence_after();
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    uint32_t r[32];
                    tc5::ld32(tmem + (part & 1) * 256 + half * 128 + p * 32 + (unsigned(quad * 32) << 16), r);
                    tc5::wait_ld();
                    uint32_t w[4] = {code[p].x, code[p].y, code[p].z, code[p].w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) asm volatile("" : "+r"(w[i]));   // widened anew each part: 128 kept floats would spill
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        // u under the significand of 2^23: q = (2^23 + u) - (2^23 + 8)
                        const uint32_t u = (w[i >> 3] >> (4 * (((i & 7) >> 1) + 4 * (i & 1)))) & 15u;
                        sum[p] = fmaf(__uint_as_float(r[i]), __uint_as_float(0x4b000000u | u) - 8388616.0f, sum[p]);
                    }
                }
                tc5::fence_before();
                __syncwarp();
                if (lane == 0) tc5::mbar_arrive(drained + 8 * (part & 1));
            }
            if (wt.fail) break;
            float *const row = dc + (t.mat * N + n) * groups;
            if (gshift < 8) {
                const int span = 1 << (gshift - 5);   // pieces of a group
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    if ((p & (span - 1)) || n >= N || k0 + 32 * p >= K) continue;
                    float v = sum[p];
                    if (span >= 2) v += sum[p | 1];
                    if (span == 4) v += sum[2] + sum[3];
                    row[(k0 + 32 * p) >> gshift] = v;
                }
            } else {
                const float v = (sum[0] + sum[1]) + (sum[2] + sum[3]);
                if (half) {
                    if (!wt.wait(sums_empty, (tiles & 1) ^ 1)) break;
                    other[quad * 32 + lane] = v;
                    __syncwarp();
                    if (lane == 0) tc5::mbar_arrive(sums_full);
                } else {
                    if (!wt.wait(sums_full, tiles & 1)) break;
                    if (n < N && k0 < K) row[k0 >> gshift] = v + other[quad * 32 + lane];
                    __syncwarp();
                    if (lane == 0) tc5::mbar_arrive(sums_empty);
                }
            }
        }
    }
    __syncthreads();
    if (warp == 9) {
        tc5::fence_after();
        tc5::tmem_free<512>(tmem);
    }
}

constexpr int64_t kMost = (int64_t(1) << 31) - 256;

// Arguments that the three products share; `a` and `b`: the row operands (b may
// be an output without alignment rules) with `na`, `nb` values a row.
int check_args(const char *what, int dtype, int64_t T, int64_t mats, int64_t N, int64_t K, int group, const int32_t *offsets,
               const uint8_t *codes, const void *a, int64_t lda, int64_t na, const void *b, int64_t ldb, int64_t nb, bool b_read) {
    if (dtype != UQ_BF16 && dtype != UQ_F16) return uq::fail(UQ_ERR_INVALID, "%s: dtype code %d is not built (bfloat16, float16)", what, dtype);
    if (T < 0 || mats < 0 || N < 0 || K <= 0 || !group_ok(group) || K % group || (!offsets && mats != 1) || mats > 65535 ||
        T > kMost || N > kMost || K > kMost || mats * N > kMost)
        return uq::fail(UQ_ERR_INVALID, "%s: bad shape (T=%lld mats=%lld N=%lld K=%lld group=%d)", what, (long long)T, (long long)mats,
                        (long long)N, (long long)K, group);
    if (T == 0 || N == 0 || mats == 0) return UQ_OK;
    if (!codes || !a || !b) return uq::fail(UQ_ERR_INVALID, "%s: null pointer", what);
    if ((T > 1 && (lda < na || ldb < nb)) || lda % 8 || (b_read && ldb % 8))
        return uq::fail(UQ_ERR_INVALID, "%s: row strides %lld and %lld of rows of %lld and %lld (those that are read: multiples of 8)", what,
                        (long long)lda, (long long)ldb, (long long)na, (long long)nb);
    if (!al16(codes) || !al16(a) || (b_read && !al16(b)))
        return uq::fail(UQ_ERR_INVALID, "%s: codes and the rows that are read have to be 16-byte aligned", what);
    return UQ_OK;
}

struct Plan {
    int width;        // BT of the kernel
    int bt;           // rows of a tile
    int splits;
    int64_t tiles;    // at most
};

// J result columns, `depth` contraction steps.
Plan plan_for(int64_t T, int64_t mats, bool runs, int64_t J, int64_t depth) {
    Plan p;
    const int64_t each = std::max<int64_t>(1, T / std::max<int64_t>(mats, 1));   // rows a matrix, if even
    p.width = each <= 64 ? 64 : each <= 128 ? 128 : 256;
    p.bt = p.width;
    p.splits = 1;
    const int64_t wt = (J + 127) / 128;
    const int64_t rt = runs ? std::min(T, T / p.bt + mats) : (T + p.bt - 1) / p.bt;
    p.tiles = rt * wt;
    const int sms = uq::num_sms();
    if (!runs && p.tiles * 2 <= sms) {
        const int64_t chunks = (depth + 255) / 256;
        p.splits = int(std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(sms / p.tiles, chunks / 2), 16)));
        p.tiles *= p.splits;
    }
    return p;
}

template <int BT, bool BF16, bool DX>
int launch(const void *rows, int64_t lda, const uint8_t *codes, int64_t mats, const Runs &r, const Weights &w, const Out &o, int64_t tiles, cudaStream_t st) {
    using C = Cfg<BT, DX>;
    CUtensorMap mr, mc;
    auto kernel = q4_product_kernel<BT, BF16, DX>;
    // before the maps: in a thread without a context (autograd's, at its first call) this binds the device's, which the
    // map encoder needs
    if (uq::set_smem_attr(reinterpret_cast<const void *>(kernel), C::kSmem) != cudaSuccess) return uq::check_cuda("q4_product_kernel attribute");
    const int64_t depth = DX ? w.N : w.K;
    if (!tc5::encode2d(&mr, BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rows, uint64_t(depth), uint64_t(r.T),
                       uint64_t(lda) * 2, 64, BT / 4, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !tc5::encode2d(&mc, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, uint64_t(w.K / 2), uint64_t(mats * w.N), uint64_t(w.K / 2), DX ? 64 : 128,
                       DX ? 256 : 128, DX ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B))
        return uq::fail(UQ_ERR_CUDA, "tensor map of a 4-bit product");
    const int grid = int(std::min<int64_t>(tiles, uq::num_sms()));
    uq::ProfScope _p(DX ? "q4_dx" : "q4_linear", st);
    kernel<<<grid, kThreads, C::kSmem, st>>>(mr, mc, r, w, o);
    return uq::check_cuda("q4_product_kernel launch");
}

// Rows (for several matrices, rows each if even) up to which the kernel for few
// rows is taken.
constexpr int64_t kFewMost = 16;

template <bool BF16, int NT>
int few(const void *x, int64_t ldx, int64_t T, const uint8_t *codes, const Weights &w, int64_t mats, const int32_t *offsets, void *y, int64_t ldy, bool zero,
        cudaStream_t st) {
    auto kernel = q4_few_kernel<BF16, NT>;
    const int64_t rows = std::min<int64_t>(T, 8 * NT), wide = (w.K + 255) / 256 * 256;
    const int section = int(std::min<int64_t>(wide, 98304 / (2 * rows) / 256 * 256));
    const int smem = int(std::max<int64_t>(rows * section * 2, kFewWarps * 8 * NT * kFewRows * 4));
    if (uq::set_smem_attr(reinterpret_cast<const void *>(kernel), 98304) != cudaSuccess) return uq::check_cuda("q4_few_kernel attribute");
    const Runs r{offsets, T, mats, 8 * NT, int((w.N + kFewRows - 1) / kFewRows), 1};
    const Out o{y, ldy, w.N, T, zero};
    const int64_t tiles = (offsets ? std::min(T, T / (8 * NT) + mats) : 1) * r.wtiles;
    uq::ProfScope _p("q4_few", st);
    kernel<<<unsigned(std::min<int64_t>(tiles, offsets ? int64_t(uq::num_sms()) * 2 : int64_t(1) << 30)), 256, smem, st>>>(x, ldx, codes, r, w, o, section);
    return uq::check_cuda("q4_few_kernel launch");
}

template <bool BF16, bool DX>
int product(const void *rows, int64_t lda, int64_t T, const uint8_t *codes, const Weights &w, int64_t mats, const int32_t *offsets, void *out,
            int64_t ldo, bool zero, void *ws, size_t ws_bytes, cudaStream_t st) {
    const int64_t J = DX ? w.K : w.N, depth = DX ? w.N : w.K;
    const Plan p = plan_for(T, mats, offsets != nullptr, J, depth);
    if (p.splits > 1 && (!ws || ws_bytes < size_t(p.splits) * T * J * 4))
        return uq::fail(UQ_ERR_WORKSPACE, "4-bit product: workspace of %zu bytes, %zu needed", ws_bytes, size_t(p.splits) * T * J * 4);
    const Runs r{offsets, T, mats, p.bt, int((J + 127) / 128), p.splits};
    const Out o{p.splits > 1 ? ws : out, ldo, J, T, zero};
    int rc = p.width == 64    ? launch<64, BF16, DX>(rows, lda, codes, mats, r, w, o, p.tiles, st)
             : p.width == 128 ? launch<128, BF16, DX>(rows, lda, codes, mats, r, w, o, p.tiles, st)
                              : launch<256, BF16, DX>(rows, lda, codes, mats, r, w, o, p.tiles, st);
    if (rc || p.splits == 1) return rc;
    uq::ProfScope _p("q4_join_parts", st);
    q4_join_parts_kernel<BF16><<<unsigned(std::min<int64_t>((T * J + 255) / 256, 1184)), 256, 0, st>>>(static_cast<const float *>(ws), p.splits, T, J, w.scale, out, ldo);
    return uq::check_cuda("q4_join_parts_kernel launch");
}

template <bool BF16>
int dscale(const void *dy, const void *x, int64_t T, int64_t lddy, int64_t ldx, const uint8_t *codes, int64_t mats, int64_t N, int64_t K, int group,
           const int32_t *offsets, float *dc, cudaStream_t st) {
    const CUtensorMapDataType ty = BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    CUtensorMap md, mx;
    auto kernel = q4_dscale_kernel<BF16>;
    // before the maps, see launch()
    if (uq::set_smem_attr(reinterpret_cast<const void *>(kernel), DsCfg::kSmem) != cudaSuccess) return uq::check_cuda("q4_dscale_kernel attribute");
    if (!tc5::encode2d(&md, ty, dy, uint64_t(N), uint64_t(T), uint64_t(lddy) * 2, 64, 64, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !tc5::encode2d(&mx, ty, x, uint64_t(K), uint64_t(T), uint64_t(ldx) * 2, 64, 64, CU_TENSOR_MAP_SWIZZLE_128B))
        return uq::fail(UQ_ERR_CUDA, "tensor map of the scales' gradient");
    const Runs r{offsets, T, mats, 0, 0, 1};
    const int ntiles = int((N + 127) / 128), ktiles = int((K + 255) / 256);
    const int grid = int(std::min<int64_t>(mats * ntiles * int64_t(ktiles), uq::num_sms()));
    uq::ProfScope _p("q4_dscale", st);
    kernel<<<grid, kThreads, DsCfg::kSmem, st>>>(md, mx, r, codes, N, K, uq::ilog2(group), ntiles, ktiles, dc);
    return uq::check_cuda("q4_dscale_kernel launch");
}

size_t product_workspace(int64_t T, int64_t mats, int64_t J, int64_t depth) {
    if (T <= 0 || mats != 1 || J <= 0 || depth <= 0 || T > kMost || J > kMost || depth > kMost) return 0;
    const Plan p = plan_for(T, mats, false, J, depth);
    return p.splits > 1 ? size_t(p.splits) * T * J * 4 : 0;
}

}  // namespace

namespace uq {
namespace q4 {
bool mm_take_flags(int *timeout, int *offset) {
    const int zero = 0;
    return cudaMemcpyFromSymbol(offset, g_mm_bad_offset, sizeof(int)) == cudaSuccess &&
           cudaMemcpyFromSymbol(timeout, g_mm_timeout, sizeof(int)) == cudaSuccess &&
           (!*offset || cudaMemcpyToSymbol(g_mm_bad_offset, &zero, sizeof(int)) == cudaSuccess) &&
           (!*timeout || cudaMemcpyToSymbol(g_mm_timeout, &zero, sizeof(int)) == cudaSuccess);
}
}  // namespace q4
}  // namespace uq

extern "C" {

size_t uq_q4_linear_workspace_bytes(int64_t T, int64_t mats, int64_t N, int64_t K) { return T <= kFewMost ? 0 : product_workspace(T, mats, N, K); }

int uq_q4_linear(const void *x, int dtype, int64_t T, int64_t ldx, const uint8_t *codes, const uint8_t *scales, const float *scale,
                 int64_t mats, int64_t N, int64_t K, int group, const int32_t *offsets, void *y, int64_t ldy, int zero_rest,
                 void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check_args("uq_q4_linear", dtype, T, mats, N, K, group, offsets, codes, x, ldx, K, y, ldy, N, false)) return rc;
    if (T == 0 || N == 0 || mats == 0) return UQ_OK;
    if (!scales || !scale) return uq::fail(UQ_ERR_INVALID, "uq_q4_linear: null pointer");
    const Weights w{scales, scale, N, K, uq::ilog2(group)};
    const cudaStream_t st = UQ_STREAM(stream);
    if (T <= kFewMost * mats) {
        if (T <= 8 * mats)
            return dtype == UQ_BF16 ? few<true, 1>(x, ldx, T, codes, w, mats, offsets, y, ldy, zero_rest, st)
                                    : few<false, 1>(x, ldx, T, codes, w, mats, offsets, y, ldy, zero_rest, st);
        return dtype == UQ_BF16 ? few<true, 2>(x, ldx, T, codes, w, mats, offsets, y, ldy, zero_rest, st)
                                : few<false, 2>(x, ldx, T, codes, w, mats, offsets, y, ldy, zero_rest, st);
    }
    return dtype == UQ_BF16 ? product<true, false>(x, ldx, T, codes, w, mats, offsets, y, ldy, zero_rest, workspace, workspace_bytes, st)
                            : product<false, false>(x, ldx, T, codes, w, mats, offsets, y, ldy, zero_rest, workspace, workspace_bytes, st);
}

size_t uq_q4_linear_dx_workspace_bytes(int64_t T, int64_t mats, int64_t N, int64_t K) { return product_workspace(T, mats, K, N); }

int uq_q4_linear_dx(const void *dy, int dtype, int64_t T, int64_t lddy, const uint8_t *codes, const uint8_t *scales, const float *scale,
                    int64_t mats, int64_t N, int64_t K, int group, const int32_t *offsets, void *dx, int64_t lddx, int zero_rest,
                    void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check_args("uq_q4_linear_dx", dtype, T, mats, N, K, group, offsets, codes, dy, lddy, N, dx, lddx, K, false)) return rc;
    if (T == 0 || N == 0 || mats == 0) return UQ_OK;
    if (!scales || !scale) return uq::fail(UQ_ERR_INVALID, "uq_q4_linear_dx: null pointer");
    const Weights w{scales, scale, N, K, uq::ilog2(group)};
    const cudaStream_t st = UQ_STREAM(stream);
    return dtype == UQ_BF16 ? product<true, true>(dy, lddy, T, codes, w, mats, offsets, dx, lddx, zero_rest, workspace, workspace_bytes, st)
                            : product<false, true>(dy, lddy, T, codes, w, mats, offsets, dx, lddx, zero_rest, workspace, workspace_bytes, st);
}

size_t uq_q4_linear_dscale_workspace_bytes(int64_t, int64_t, int64_t, int64_t, int) { return 0; }

int uq_q4_linear_dscale(const void *dy, const void *x, int dtype, int64_t T, int64_t lddy, int64_t ldx, const uint8_t *codes, int64_t mats,
                        int64_t N, int64_t K, int group, const int32_t *offsets, float *dc, void *, size_t, void *stream) {
    if (int rc = check_args("uq_q4_linear_dscale", dtype, T, mats, N, K, group, offsets, codes, dy, lddy, N, x, ldx, K, true)) return rc;
    if (N == 0 || mats == 0) return UQ_OK;
    if (!dc) return uq::fail(UQ_ERR_INVALID, "uq_q4_linear_dscale: null pointer");
    const cudaStream_t st = UQ_STREAM(stream);
    if (T == 0)
        return cudaMemsetAsync(dc, 0, size_t(mats) * N * (K / group) * 4, st) == cudaSuccess ? UQ_OK : uq::check_cuda("uq_q4_linear_dscale");
    return dtype == UQ_BF16 ? dscale<true>(dy, x, T, lddy, ldx, codes, mats, N, K, group, offsets, dc, st)
                            : dscale<false>(dy, x, T, lddy, ldx, codes, mats, N, K, group, offsets, dc, st);
}

}  // extern "C"
