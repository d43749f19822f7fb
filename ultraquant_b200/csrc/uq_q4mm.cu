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
// Tiles: `wtiles` ranges of weight columns of the result by up to `bt` rows of
// one matrix's run.  Those from number `whole` on are `splits` parts of the
// contraction each (one matrix for all rows only).
// ----------------------------------------------------------------------------
struct Runs {
    const int32_t *offsets;   // null: one matrix, all rows
    int64_t T, mats;
    int bt;                   // rows of a tile
    int wtiles, splits;
    int64_t whole;
};

struct Tile {
    int mat, row0, rows, wt, split;
};

// Finds a warp's tiles in rising order: the 32 lanes hold 32 matrices' runs at a
// time.  An offset counts as at least its predecessors and at most T.
// RUNS: whether there are offsets; without them none of the state is kept.
template <bool RUNS> struct Finder {
    int first, lo, incl, top, begin;   // matrices before this block of 32; this lane's run: first row, row tiles up to its end
    int64_t base;                      // row tiles before this block
    bool loaded;

    __device__ __forceinline__ void start(const Runs &r) {
        first = 0;
        base = 0;
        loaded = false;
        top = 0;
        if (RUNS) {
            const int o = r.offsets[0];
            top = min(max(o, 0), int(r.T));
            if (o != top) g_mm_bad_offset = 1;
        }
        begin = top;
    }
    __device__ __forceinline__ void load(const Runs &r) {
        const int lane = threadIdx.x & 31, i = first + lane, n = int(r.mats), T = int(r.T);
        const int o = i < n ? r.offsets[i + 1] : 0;
        int m = max(i < n ? min(max(o, 0), T) : 0, top);
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, m, d);
            if (lane >= d) m = max(m, v);
        }
        if (i < n && o != m) g_mm_bad_offset = 1;
        lo = __shfl_up_sync(0xffffffffu, m, 1);
        if (lane == 0) lo = top;
        incl = (m - lo + r.bt - 1) / r.bt;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, d);
            if (lane >= d) incl += v;
        }
        top = __shfl_sync(0xffffffffu, m, 31);
        loaded = true;
    }
    // Tile number `t`; false beyond the last.
    __device__ __forceinline__ bool find(const Runs &r, int64_t t, Tile &tile) {
        int64_t u = t;
        tile.split = -1;          // the whole contraction, else the part's number
        if (!RUNS && t >= r.whole) {
            tile.split = int(t - r.whole);     // below 2^27 parts
            u = r.whole + int(unsigned(tile.split) / unsigned(r.splits));
        }
        const int64_t rt = u < r.wtiles ? 0 : u / r.wtiles;   // few rows: no division on the way to the first copy
        tile.wt = int(u - rt * r.wtiles);
        if constexpr (!RUNS) {
            tile.mat = 0;
            if (rt * r.bt >= r.T) return false;
            tile.row0 = int(rt) * r.bt;
            tile.rows = min(int(r.T) - tile.row0, r.bt);
        } else {
            for (;;) {
                if (!loaded) {
                    if (first >= r.mats) return false;
                    load(r);
                }
                const int all = __shfl_sync(0xffffffffu, incl, 31);
                if (rt < base + all) break;
                base += all;
                first += 32;
                loaded = false;
            }
            const int at = __popc(__ballot_sync(0xffffffffu, base + incl <= rt));   // runs that end before the tile
            const int before = __shfl_sync(0xffffffffu, incl, at > 0 ? at - 1 : 0);
            const int l = __shfl_sync(0xffffffffu, lo, at), next = __shfl_sync(0xffffffffu, lo, at < 31 ? at + 1 : 31);
            tile.mat = first + at;
            tile.row0 = l + int(rt - base - (at > 0 ? before : 0)) * r.bt;
            tile.rows = min((at < 31 ? next : top) - tile.row0, r.bt);
        }
        return true;
    }
    // The end of the last run, once find() has gone beyond the last tile.
    __device__ __forceinline__ int64_t end(const Runs &r) const { return RUNS ? top : r.T; }
};

// ----------------------------------------------------------------------------
// Weights in 16-bit halves
// ----------------------------------------------------------------------------
// Eight codes become four words of two halves with one shift: nibbles 0, 4 and
// 1, 5 of the word and of the word shifted by 8 are masked in place and read as
// numbers that are linear in u; one fused multiply-add each makes e q of them,
// times kUnit, a power of two that is taken back from the finished sum.  Nothing
// rounds or overflows (|e| <= 448 with 4 significant bits, 9 x 15 and 17 x 15 have
// 8 bits, 129 x 15 has 11):
//   bfloat16, kUnit 2^-14: the masked bits are 2^-133 u and 2^-129 u, subnormal or
//     of the least exponent, which continues them; times e 2^119 and e 2^115, less
//     8 e 2^-14
//   float16, kUnit 1/8: under the significand of 1024, 1024 + u and 1024 + 16 u;
//     times e / 8 and e / 128, less 129 e and 9 e
template <bool BF16> struct Halves;
template <> struct Halves<true> {
    using T = __nv_bfloat16;
    static constexpr float kBack = 16384.0f;   // 1 / kUnit
    struct Scale { uint32_t e, e16, z; };
    // e: two E4M3 values as float16; which: 0 or 1
    static __device__ __forceinline__ Scale scale(uint32_t e, int which) {
        const float f = __half2float(__ushort_as_half((unsigned short)(which ? e >> 16 : e)));
        uint32_t d;
        Scale s;
        asm("cvt.rn.bf16x2.f32 %0, %1, %1;" : "=r"(d) : "f"(f));
        asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(s.e) : "r"(d), "r"(0x7b007b00u));     // 2^119
        asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(s.e16) : "r"(d), "r"(0x79007900u));   // 2^115
        asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(s.z) : "r"(d), "r"(0xba00ba00u));     // -2^-11
        return s;
    }
    static __device__ __forceinline__ void widen8(uint32_t w, const Scale &s, uint32_t *out) {
        const uint32_t h = w >> 8;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t v = (i < 2 ? w : h) & (i & 1 ? 0x00f000f0u : 0x000f000fu);
            asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(out[i]) : "r"(v), "r"(i & 1 ? s.e16 : s.e), "r"(s.z));
        }
    }
};
template <> struct Halves<false> {
    using T = __half;
    static constexpr float kBack = 8.0f;
    struct Scale { uint32_t e, e16, z, z16; };
    static __device__ __forceinline__ Scale scale(uint32_t e, int which) {
        const uint32_t d = __byte_perm(e, 0, which ? 0x3232 : 0x1010);
        Scale s;
        asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(s.e) : "r"(d), "r"(0x30003000u));     // 1 / 8
        asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(s.e16) : "r"(d), "r"(0x20002000u));   // 1 / 128
        asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(s.z) : "r"(d), "r"(0xd808d808u));     // -129
        asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(s.z16) : "r"(d), "r"(0xc880c880u));   // -9
        return s;
    }
    static __device__ __forceinline__ void widen8(uint32_t w, const Scale &s, uint32_t *out) {
        const uint32_t h = w >> 8;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t v = ((i < 2 ? w : h) & (i & 1 ? 0x00f000f0u : 0x000f000fu)) | 0x64006400u;
            asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(out[i]) : "r"(v), "r"(i & 1 ? s.e16 : s.e), "r"(i & 1 ? s.z16 : s.z));
        }
    }
};

// Two E4M3 bytes as two float16 (E4M3 is a subset; NaN stays NaN).
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t b) {
    uint32_t h;
    asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(h) : "r"(b));
    return h;
}

// 32 codes of one group -> 16 registers of two halves each, in order.
template <bool BF16> __device__ __forceinline__ void widen32(const uint4 &c, const typename Halves<BF16>::Scale &s, uint32_t *out) {
    Halves<BF16>::widen8(c.x, s, out);
    Halves<BF16>::widen8(c.y, s, out + 4);
    Halves<BF16>::widen8(c.z, s, out + 8);
    Halves<BF16>::widen8(c.w, s, out + 12);
}

// A plain load (not asm), so that the compiler may order it among the arithmetic
// but not across a barrier.
__device__ __forceinline__ uint4 lds128(const uint8_t *smem, unsigned smem_at, unsigned addr) {
    return *reinterpret_cast<const uint4 *>(smem + (addr - smem_at));
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

// A chunk's scales on their way to shared memory, four rows of eight pieces of 32
// values a lane, or (DX) eight rows of four.  Where a row's bytes of the chunk are
// one aligned word (`packed`), it is kept as it is; else the pieces' bytes are
// gathered.  Nothing here waits for a load: the words are taken apart when they
// are stored.
struct Scales { uint32_t w[8]; };

// Bytes of the four pieces from value k on, 0 beyond K.
__device__ __forceinline__ uint32_t gather4(const Weights &w, const uint8_t *row, int64_t k) {
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = k + 32 * i < w.K ? __ldg(row + ((k + 32 * i) >> w.gshift)) : 0u;
    return v[0] | v[1] << 8 | v[2] << 16 | v[3] << 24;
}
// Rows lane + 32 j (below `rows`) of `groups` bytes each, from `p` on: a word of
// WORD's size of each, 0 for a row that is not there.
template <typename WORD, int R> __device__ __forceinline__ void load_rows(uint32_t (&w)[8], const uint8_t *p, int64_t groups, int rows) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int j = 0; j < R; ++j) {
        WORD v = {};
        if (lane + 32 * j < rows) v = __ldg(reinterpret_cast<const WORD *>(p + (lane + 32 * j) * groups));
        if constexpr (sizeof(WORD) == 8) {
            w[2 * j] = v.x;
            w[2 * j + 1] = v.y;
        } else {
            w[8 / R * j] = v;
        }
    }
}
// The scales from value k on; `p`: the first row's bytes.
template <bool DX>
__device__ __forceinline__ void load_scales(Scales &v, const Weights &w, bool packed, const uint8_t *p, int64_t groups, int rows, int64_t k) {
    constexpr int R = DX ? 8 : 4, W = 8 / R;   // rows, words of each
    const int bytes = (DX ? 128 : 256) >> w.gshift;
    if (k >= w.K) rows = 0;                    // DX: columns beyond the matrix
    const uint8_t *const at = p + (k >> w.gshift);
    if (!packed) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int j = 0; j < R; ++j)
#pragma unroll
            for (int i = 0; i < W; ++i) v.w[W * j + i] = lane + 32 * j < rows ? gather4(w, p + (lane + 32 * j) * groups, k + 128 * i) : 0u;
    } else if (W == 2 && bytes == 8) {
        if constexpr (W == 2) load_rows<uint2, R>(v.w, at, groups, rows);
    } else if (bytes == 4) {
        load_rows<unsigned, R>(v.w, at, groups, rows);
    } else if (bytes == 2) {
        load_rows<unsigned short, R>(v.w, at, groups, rows);
    } else {
        load_rows<unsigned char, R>(v.w, at, groups, rows);
    }
}

struct Out {
    void *out;        // (rows, J) of 16 bits
    int64_t ld, J, T;
    bool zero_rest;
    float *parts;     // of split tiles: (tile, part, bt, 256)
};

// A finished sum times the matrix's s, then 1 / kUnit: sum / kUnit alone may be beyond
// float32 where the result is not (weights of 2^-10 and bfloat16 activations of 2^115).
// In this order nothing passes the range before the result does; a result below 2^-112
// is off by at most 2^-136 more (half of float32's least step, times 2^14), a quarter
// of bfloat16's least rounding.
template <bool BF16> __device__ __forceinline__ float finish(float v, float s) { return (s * v) * Halves<BF16>::kBack; }

// Register j of lane i: row j, column i of a 32 x 32 piece of the result.
// pack_piece: rows 2 j and 2 j + 1 in the halves of v[j], scaled and rounded.
template <bool BF16> __device__ __forceinline__ void pack_piece(const uint32_t (&r)[32], float s, uint32_t (&v)[16]) {
    using T = typename Halves<BF16>::T;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        T two[2] = {from_float<T>(finish<BF16>(__uint_as_float(r[2 * j]), s)), from_float<T>(finish<BF16>(__uint_as_float(r[2 * j + 1]), s))};
        v[j] = *reinterpret_cast<const uint32_t *>(two);
    }
}
// Writes rows [0, rows) and columns below J.  Where two columns share an aligned
// word (`wide`) neighbouring lanes trade halves, so that each writes both columns
// of one row: half the store instructions, a row's 32 columns still one line of
// 64 bytes.
__device__ __forceinline__ void store_piece(const uint32_t (&v)[16], void *out, int64_t ld, int64_t J, bool wide, int row0, int rows, int64_t col) {
    const int odd = threadIdx.x & 1;
    if (wide) {
        char *p = static_cast<char *>(out) + (int64_t(row0 + odd) * ld + (col - odd)) * 2;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const uint32_t got = __shfl_xor_sync(0xffffffffu, v[j], 1);
            const uint32_t word = odd ? __byte_perm(got, v[j], 0x7632) : __byte_perm(v[j], got, 0x5410);
            if (2 * j + odd < rows && col < J) *reinterpret_cast<uint32_t *>(p) = word;
            p += ld * 4;
        }
    } else if (col < J) {
        unsigned short *p = static_cast<unsigned short *>(out) + int64_t(row0) * ld + col;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            if (j < rows) *p = (unsigned short)(v[j >> 1] >> (16 * (j & 1)));
            p += ld;
        }
    }
}
// A tile's share of one warp, out of line so that the widening loop keeps its
// registers: 32 lanes' columns of `pieces` times 32 rows, every 128 rows.  Once
// the values are in registers the tensor memory is free (`drained`).
template <bool BF16, int PIECES>
__device__ __noinline__ void write_tile(unsigned at, unsigned drained, float scale, void *out, int64_t ld, int64_t J, bool wide, int row0, int rows, int64_t col) {
    uint32_t v[PIECES][16];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        uint32_t r[32];
        tc5::ld32(at + i * 128, r);   // beyond the tile's rows: whatever is there, not written
        tc5::wait_ld();
        pack_piece<BF16>(r, scale, v[i]);
    }
    tc5::fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) tc5::mbar_arrive_remote(drained);
#pragma unroll
    for (int i = 0; i < PIECES; ++i)
        if (i * 128 < rows) store_piece(v[i], out, ld, J, wide, row0 + i * 128, rows - i * 128, col);
}
// The same for a part of a split contraction: floats, unscaled, 256 a row.
__device__ __noinline__ void write_part(unsigned at, unsigned drained, float *out, int rows) {
    for (int i = 0; i < rows; i += 128) {
        uint32_t r[32];
        tc5::ld32(at + i, r);
        tc5::wait_ld();
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (i + j < rows) out[(i + j) * 256] = __uint_as_float(r[j]);
    }
    tc5::fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) tc5::mbar_arrive_remote(drained);
}

// Rows outside every run, a share of them for the first `threads` threads of each block.
template <typename T> __device__ void zero_rows(const Out &o, int64_t begin, int64_t end, int threads) {
    const int64_t rest = o.T - (end - begin);
    for (int64_t i = blockIdx.x; i < rest; i += gridDim.x) {
        T *p = static_cast<T *>(o.out) + (i < begin ? i : end + i - begin) * o.ld;
        for (int64_t j = threadIdx.x; j < o.J; j += threads) p[j] = from_float<T>(0.0f);
    }
}

// ----------------------------------------------------------------------------
// The product kernel.  The result is formed transposed, weight columns in the
// lanes of tensor memory and up to BT rows in its columns, so that few rows make
// a narrow instruction.  A pair of CTAs takes 256 weight columns, 128 each, and
// each CTA brings half of the tile's rows: alone, a CTA needed 64 bytes a clock
// of rows from L2, and L2 gave 12 TB/s, 43 a clock and SM.  Stages of 64
// contraction steps: `full` (in the first CTA) its half of the rows (TMA, 128-byte
// swizzle), the second CTA's word that its half is there, and the widened weights
// of both, one barrier for all, since the issuing warp's waits bound the rate;
// `empty` both free again.
//   forward: lane n; the weights go from registers into tensor memory (32
//            columns a stage), codes by TMA in chunks of 256 steps
//   DX:      lane k; a stage is 64 rows n of 128 codes, widened into shared
//            memory with k contiguous
// Warps 0 .. 15 widen (warps 4 s .. 4 s + 3 stage s of each chunk) and write
// results, those of a tile after the next tile's first chunk is widened, so that
// the tensor cores have work meanwhile; warp 16 copies the rows, warp 17 the
// codes; warp 18 issues the products (first CTA) or tells the first CTA that its
// rows are there (second); warp 19 brings each chunk's scales, an odd few bytes
// from every row, which loaded by the widening warps a chunk ahead still cost 7 %
// forward and 30 % of DX (4096 x 4096 x 14336: 460 us, 316 without any scales).
// Bound by the tensor cores from about 215 rows a tile on (forward 2047 x 14336 x 4096
// 156 us, 1.54 PFLOP/s; DX 4096 x 4096 x 14336 344 us, 1.40 PFLOP/s).  Below, a stage
// takes some 430 cycles however few its rows, about three times what its bytes need, by
// neither the widening's arithmetic nor the products but by the way of a chunk through
// copies, barriers and the store of A.  28672 x 8192 in us, as it is / without the
// arithmetic / without the products / without both: forward 32 rows 58 / 57 / 56 / 55,
// 128 rows 67 / 65 / 63 / 61, 256 rows 93 / 92 / 65 / 71; DX 32 rows 62 / 61 / 61 / 60,
// 256 rows 119 / 112 / 95 / 92.
// The sums of a tile's whole contraction stay in the tensor core's float32
// accumulator, unlike those of q4_dscale_kernel: the result is rounded to 16 bits, and
// what sums of 14336 terms are off (some 6e-6 of the results' size: 0.16 % of them round
// to the neighbour) is a 300th of that rounding.
// 640 threads leave 96 registers each.  Spilled (bytes stored and loaded): nothing
// forward without offsets, 112 and 220 by DX in bfloat16 and 256 rows, up to 264 and
// 156 by the forms with offsets; up to 30 and 46 by write_tile.
// ----------------------------------------------------------------------------
constexpr int kWiden = 16, kThreads = (kWiden + 4) * 32;

template <int BT, bool DX> struct Cfg {
    static constexpr int NS = DX ? (BT == 256 ? 5 : 6) : 8;                  // stages
    static constexpr int kChunks = DX ? (BT == 64 ? 4 : BT == 128 ? 3 : 3) : BT == 256 ? 5 : 8;
    static constexpr int kB = BT * 64, kA = DX ? 16384 : 0, kC = 16384, kE = 1024;   // kE: a chunk's scales, 512 pairs
    static constexpr int kBar = 2 * NS + 2 * kChunks + 2;
    static constexpr int kSmem = 1024 + NS * (kB + kA) + kChunks * (kC + kE) + kBar * 8 + 16;
    static_assert(kSmem <= 232448, "shared memory of one block");
    static_assert(DX || BT + 32 * NS <= 512, "tensor memory");
};

template <int BT, bool BF16, bool DX, bool RUNS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
q4_product_kernel(const __grid_constant__ CUtensorMap map_rows, const __grid_constant__ CUtensorMap map_codes, Runs runs, Weights w, Out o) {
    using C = Cfg<BT, DX>;
    constexpr int NS = C::NS, NC = C::kChunks, kBox = BT / 4;   // rows of one copy: half of a CTA's share
    extern __shared__ uint8_t smem_raw[];
    const unsigned smem_at = tc5::smem_addr(smem_raw), base = (smem_at + 1023u) & ~1023u;
    const unsigned sb = base, sa = sb + NS * C::kB, sc = sa + NS * C::kA, se = sc + NC * C::kC, bars = se + NC * C::kE;
    const unsigned full = bars, empty = bars + 8 * NS, full_c = bars + 16 * NS, empty_c = full_c + 8 * NC, done = empty_c + 8 * NC, drained = done + 8, misc = drained + 8;
    volatile int *gave_up = reinterpret_cast<volatile int *>(smem_raw + (misc + 4 - tc5::smem_addr(smem_raw)));
    const int warp = tc5::warp_id(), lane = threadIdx.x & 31;
    const unsigned rank = tc5::cluster_rank();
    if (warp == kWiden + 2) tc5::tmem_alloc<512>(misc);
    if (threadIdx.x == 0) {
        *gave_up = 0;
        for (int i = 0; i < NS; ++i) {
            tma::mbar_init(full + 8 * i, rank == 0 ? 10 : 1);
            tma::mbar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < NC; ++i) {
            tma::mbar_init(full_c + 8 * i, 2);   // codes, scales
            tma::mbar_init(empty_c + 8 * i, kWiden);
        }
        tma::mbar_init(done, 1);
        tma::mbar_init(drained, 2 * kWiden);
        tma::mbar_init(misc + 8, 1);   // products in flight, where a wait gave up
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    tc5::fence_before();
    __syncthreads();
    tc5::cluster_sync();
    tc5::fence_after();
    unsigned tmem;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(misc));
    tmem = __shfl_sync(0xffffffffu, tmem, 0);
    const unsigned tmem_a = tmem + BT;

    tc5::Waiter wt{gave_up, &g_mm_timeout};
    Finder<RUNS> find;
    find.start(runs);
    Tile t;
    const int64_t step = gridDim.x >> 1, first = blockIdx.x >> 1;                 // pairs
    const int64_t depth = DX ? w.N : w.K;
    // stages of the whole contraction and of one part of it, whole chunks of four: what lies beyond the end is zero, and every
    // warp takes part in every chunk, so that no barrier goes by two phases unseen by one that will wait for it
    const int all = int((depth + 255) / 256) * 4, per = (all / 4 + runs.splits - 1) / runs.splits * 4;
    const auto first_of = [&](const Tile &i) { return RUNS || i.split < 0 ? 0 : i.split % runs.splits * per; };   // a tile's stages
    const auto count_of = [&](const Tile &i) { return RUNS || i.split < 0 ? all : min(per, all - first_of(i)); };
    unsigned it = 0, ct = 0, tiles = 0;                                           // stages, chunks, tiles so far

    if (warp == kWiden) {
        // rows: this CTA's half of the product's N
        for (int64_t tile = first; !wt.fail && find.find(runs, tile, t); tile += step) {
            const int s0 = first_of(t), n = count_of(t);
            const int half = ((t.rows + 31) & ~31) >> 1, boxes = (half + kBox - 1) / kBox, row = int(t.row0) + int(rank) * half;
            for (int s = 0; s < n; ++s, ++it) {
                const int slot = it % NS;
                if (!wt.wait(empty + 8 * slot, ((it / NS) & 1) ^ 1)) break;
                if (lane == 0) {
                    tma::mbar_arrive_expect_tx(full + 8 * slot, boxes * kBox * 128);
                    for (int b = 0; b < boxes; ++b)
                        tma::load2d(sb + slot * C::kB + b * kBox * 128, &map_rows, (s0 + s) * 64, row + b * kBox, full + 8 * slot);
                }
                __syncwarp();
            }
        }
        if (wt.fail)   // copies in flight land before the block ends
            for (unsigned i = it > NS ? it - NS : 0; i < it; ++i) tc5::Waiter::drain(full + 8 * (i % NS), (i / NS) & 1);
    } else if (warp == kWiden + 1) {
        // codes: 128 rows of 256 codes, or 256 rows of 128
        for (int64_t tile = first; !wt.fail && find.find(runs, tile, t); tile += step) {
            const int s0 = first_of(t), n = count_of(t);
            const int64_t row = t.mat * w.N;
            const int wtile = t.wt * 2 + int(rank);
            for (int s = 0; s < n; s += 4, ++ct) {
                const int slot = ct % NC;
                if (!wt.wait(empty_c + 8 * slot, ((ct / NC) & 1) ^ 1)) break;
                if (lane == 0) {
                    tma::mbar_arrive_expect_tx(full_c + 8 * slot, C::kC);
                    if (DX) tma::load2d(sc + slot * C::kC, &map_codes, wtile * 64, int(row + (s0 + s) * 64), full_c + 8 * slot);
                    else tma::load2d(sc + slot * C::kC, &map_codes, (s0 + s) * 32, int(row + int64_t(wtile) * 128), full_c + 8 * slot);
                }
                __syncwarp();
            }
        }
        if (wt.fail)
            for (unsigned i = ct > NC ? ct - NC : 0; i < ct; ++i) tc5::Waiter::drain(full_c + 8 * (i % NC), (i / NC) & 1);
    } else if (warp == kWiden + 2 && rank == 1) {
        for (int64_t tile = first; !wt.fail && find.find(runs, tile, t); tile += step) {
            const int s0 = first_of(t), n = count_of(t);
            for (int s = 0; s < n; ++s, ++it) {
                const int slot = it % NS;
                if (!wt.wait(full + 8 * slot, (it / NS) & 1)) break;
                if (lane == 0) tc5::mbar_arrive_remote(tc5::leader_addr(full + 8 * slot));
                __syncwarp();
            }
        }
    } else if (warp == kWiden + 2) {
        // products
        unsigned slot = 0, par = 0;
        bool ready = false;
        for (int64_t tile = first; !wt.fail && find.find(runs, tile, t); tile += step, ++tiles) {
            const int s0 = first_of(t), n = count_of(t);
            const uint32_t idesc = tc5::idesc_f16(BF16, (t.rows + 31) & ~31, DX, false);
            if (!wt.wait(drained, (tiles & 1) ^ 1)) break;
            for (int s = 0; s < n; ++s) {
                if (!ready && !wt.wait(full + 8 * slot, par)) break;
                tc5::fence_after();
                const uint64_t b = tc5::desc128(sb + slot * C::kB, 16, 1024), a = tc5::desc128(sa + slot * C::kA, 8192, 1024);
                // whether the next stage is there: asked for before this one's products are issued, since the answer takes as
                // long as they do
                const unsigned next = slot + 1 == NS ? 0 : slot + 1, npar = par ^ (slot + 1 == NS);
                ready = __all_sync(0xffffffffu, tc5::mbar_test(full + 8 * next, npar));
                if (tc5::elect()) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if (DX) tc5::mma_ss(tmem, a + k * 128, b + k * 2, idesc, s > 0 || k > 0);
                        else tc5::mma_ts(tmem, tmem_a + slot * 32 + k * 8, b + k * 2, idesc, s > 0 || k > 0);
                    }
                    tc5::commit(empty + 8 * slot);
                }
                __syncwarp();
                slot = next;
                par = npar;
            }
            if (!wt.fail && tc5::elect()) tc5::commit(done);
            __syncwarp();
        }
        if (wt.fail) {   // products in flight end before the block does
            if (tc5::elect()) tc5::commit(misc + 8);
            __syncwarp();
            tc5::Waiter::drain(misc + 8, 0);
        }
    } else if (warp == kWiden + 3) {
        // scales, two chunks' loads ahead of the ring
        const int64_t groups = w.K >> w.gshift;
        const bool packed = (w.K & (DX ? 127 : 255)) == 0;
        // bytes of the kept words that are a pair's: those of pieces 2 i and 2 i + 1
        const int shift = packed ? w.gshift - 5 : 0;
        uint32_t pick[DX ? 2 : 4];
#pragma unroll
        for (int i = 0; i < (DX ? 2 : 4); ++i) pick[i] = uint32_t((2 * i) >> shift) | uint32_t((2 * i + 1) >> shift) << 4;
        int64_t tile = first;
        int c = 0, n = 0, s0 = 0;       // chunk's first stage in the tile, its stages, the first
        bool on = true;
        Scales a, b;
        auto fetch = [&](Scales &v) -> bool {   // the next chunk's; false beyond the last
            if (c >= n) {
                if (!on || !(on = find.find(runs, tile, t))) return false;
                tile += step;
                c = 0;
                s0 = first_of(t);
                n = count_of(t);
            }
            const int64_t k0 = int64_t(s0 + c) * 64, mrow = t.mat * w.N, col = (int64_t(t.wt) * 2 + rank) * 128;
            const int64_t row = DX ? k0 : col;
            load_scales<DX>(v, w, packed, w.scales + (mrow + row) * groups, groups, int(min(w.N - row, int64_t(DX ? 256 : 128))), DX ? col : k0);
            c += 4;
            return true;
        };
        unsigned slot = 0, par = 1;
        auto put = [&](const Scales &v) -> bool {
            if (!wt.wait(empty_c + 8 * slot, par)) return false;
            uint8_t *const to = smem_raw + (se + slot * C::kE - smem_at);
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int i = DX ? j & 1 : j & 3, r = DX ? j >> 1 : j >> 2, at = i * (DX ? 256 : 128) + r * 32;   // [half][row n] or [stage][row n]
                reinterpret_cast<unsigned short *>(to)[at + lane] =
                    (unsigned short)(DX ? __byte_perm(v.w[r], 0, pick[i]) : __byte_perm(v.w[2 * r], v.w[2 * r + 1], pick[i]));
            }
            __syncwarp();
            if (lane == 0) tc5::mbar_arrive(full_c + 8 * slot);
            if (++slot == NC) { slot = 0; par ^= 1; }
            return true;
        };
        bool more_a = fetch(a), more_b = more_a && fetch(b);
        while (more_a) {
            if (!put(a)) break;
            more_a = more_b && fetch(a);
            if (!more_b || !put(b)) break;
            more_b = more_a && fetch(b);
        }
    } else {
        // widen, then write the result
        const int stage = warp >> 2, quad = warp & 3;      // of each chunk; lanes of tensor memory
        unsigned cslot = 0, cpar = 0, slot0 = 0, par0 = 1;   // chunk slot and parity; the chunk's first stage and its parity of `empty`
        const unsigned full0 = tc5::leader_addr(full), drained0 = tc5::leader_addr(drained);
        const bool wide = !((o.ld | o.J) & 1) && !(reinterpret_cast<uintptr_t>(o.out) & 3);
        // this lane's scales in a chunk's table: forward those of its row and stage, DX of its row n and half
        const int eat = DX ? (quad >> 1) * 256 + stage * 64 + (quad & 1) * 32 + lane : stage * 128 + quad * 32 + lane;
        Tile prev = {}, next = {};
        bool have = false, more = find.find(runs, first, next);   // `prev` has still to be written
        for (int64_t tile = first; !wt.fail; tile += step) {
            const bool live = more;
            int n = 0;
            if (live) {
                t = next;
                more = find.find(runs, tile + step, next);
                n = count_of(t);
            }
            int c = 0;
            do {
                if (live) {
                    const unsigned wrap = slot0 + stage >= NS, slot = slot0 + stage - (wrap ? NS : 0);
                    if (!wt.wait(full_c + 8 * cslot, cpar)) break;
                    const uint32_t ep = e4m3_pair(reinterpret_cast<const unsigned short *>(smem_raw + (se + cslot * C::kE - smem_at))[eat]);
                    const typename Halves<BF16>::Scale e[2] = {Halves<BF16>::scale(ep, 0), Halves<BF16>::scale(ep, 1)};
                    if (DX) {
                        // row rr of 128 codes (64 bytes, 64-byte swizzle): this warp's 64 values are pieces 2 h, 2 h + 1
                        const int rr = stage * 64 + (quad & 1) * 32 + lane, h = quad >> 1;
                        const unsigned line = sa + slot * C::kA + h * 8192 + ((quad & 1) * 32 + lane) * 128;
                        uint4 code[2];
#pragma unroll
                        for (int p = 0; p < 2; ++p) code[p] = lds128(smem_raw, smem_at, sc + cslot * C::kC + rr * 64 + (((2 * h + p) ^ ((rr >> 1) & 3)) << 4));
                        if (!wt.wait(empty + 8 * slot, par0 ^ wrap)) break;
#pragma unroll
                        for (int p = 0; p < 2; ++p) {
                            uint32_t v[16];
                            widen32<BF16>(code[p], e[p], v);
#pragma unroll
                            for (int q = 0; q < 4; ++q)
                                sts128(line + (((4 * p + q) ^ (lane & 7)) << 4), v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
                        }
                        tma::fence_proxy_async();
                    } else {
                        const int rr = quad * 32 + lane;
                        uint32_t v[32];
#pragma unroll
                        for (int p = 0; p < 2; ++p) widen32<BF16>(lds128(smem_raw, smem_at, sc + cslot * C::kC + rr * 128 + (((2 * stage + p) ^ (rr & 7)) << 4)), e[p], v + 16 * p);
                        if (!wt.wait(empty + 8 * slot, par0 ^ wrap)) break;
                        tc5::fence_after();
                        tc5::st32(tmem_a + slot * 32 + (unsigned(quad * 32) << 16), v);
                        tc5::wait_st();
                        tc5::fence_before();
                    }
                    __syncwarp();
                    if (lane == 0) tc5::mbar_arrive_remote(full0 + 8 * slot);
                    __syncwarp();
                    if (lane == 0) tc5::mbar_arrive(empty_c + 8 * cslot);
                    slot0 += 4;
                    if (slot0 >= NS) { slot0 -= NS; par0 ^= 1; }
                    if (++cslot == NC) { cslot = 0; cpar ^= 1; }
                }
                if (have) {
                    // the tile before: its products are done; once its values are in registers the next tile's may begin
                    have = false;
                    if (!wt.wait(done, tiles & 1)) break;
                    ++tiles;
                    tc5::fence_after();
                    const int64_t col = (int64_t(prev.wt) * 2 + rank) * 128 + quad * 32 + lane;
                    const unsigned at = tmem + stage * 32 + (unsigned(quad * 32) << 16);
                    const int r0 = prev.row0 + stage * 32, rows = prev.rows - stage * 32;
                    if (!RUNS && prev.split >= 0) {
                        write_part(at, drained0, o.parts + (int64_t(prev.split) * runs.bt + stage * 32) * 256 + rank * 128 + quad * 32 + lane, rows);
                    } else
                        write_tile<BF16, BT == 256 ? 2 : 1>(at, drained0, __ldg(w.scale + prev.mat), o.out, o.ld, o.J, wide, r0, rows, col);
                }
                c += 4;
            } while (c < n);
            if (!live || wt.fail) break;
            prev = t;
            have = true;
        }
        if (RUNS && o.zero_rest && !wt.fail) zero_rows<typename Halves<BF16>::T>(o, find.begin, find.end(runs), kWiden * 32);
    }
    tc5::fence_before();
    __syncthreads();
    tc5::cluster_sync();   // the other CTA's products read this one's memory, its warps arrive here
    if (warp == kWiden + 2) {
        tc5::fence_after();
        tc5::tmem_free<512>(tmem);
    }
}

// ----------------------------------------------------------------------------
// Few rows: bound by reading the codes once, and next to that by the
// instructions that widen them.  (57344 x 8192, 1 row: 57 us, 4.3 TB/s.  The copies
// alone take 42 us; the arithmetic alone 52, of which the masks and shifts, on a pipe
// of half rate, with the products of pairs by their scale are 40.)  A block takes
// 128 weight rows, 32 for each of four warps (16 of eight for more than 8 rows); one
// more copies chunks of 256 values of k, codes and rows, into a ring (TMA).  Four
// blocks an SM with two stages: 57 us; three with three: 63.  Where there are few
// tiles a cluster of 2, 4 or 8 blocks shares one, each a part of k, and adds up
// through distributed shared memory.  The widened codes are operand A of m16n8k16
// products straight from registers: the contraction order is free as long as both operands agree, so lane quarter q
// takes 64 consecutive values of a row (two 16-byte pieces) where the instruction
// says "columns 2 q, 2 q + 1, 2 q + 8, 2 q + 9".  Widening costs the same for 1 row
// as for 8.  (Through q4_product_kernel the codes pass at a third of memory's rate
// however few rows there are.)
// ----------------------------------------------------------------------------
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool bf16) {
    if (bf16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

constexpr int kFewRows = 128, kFewParts = 8;   // weight rows of a tile; most parts of k

// NT: blocks of 8 rows; MT: blocks of 16 weight rows of a warp.  A quarter of a
// chunk's rows is one copy of up to 8 NT lines of 64 values; each quarter begins two
// lines further round the 128-byte swizzle, so that the four lanes of a row read
// different banks.
template <int NT> struct FewCfg {
    // two weight blocks a warp share the loads of the rows and the steps of the loop; with more rows the registers do not reach
    static constexpr int MT = NT == 1 ? 2 : 1, kWarps = 8 / MT, kThreads = (kWarps + 1) * 32;
    static constexpr int NS = NT == 2 ? 4 : 2, kBlocks = NT == 1 ? 4 : 2;     // stages, blocks an SM
    static constexpr int kC = 16384, kQuarter = 8 * NT * 128 + 256, kX = 4 * kQuarter, kStage = kC + kX;
    static constexpr int kSums = kFewRows * 8 * NT * 4;                       // of one block, for its cluster
    static constexpr int kSmem = 1024 + NS * kStage + kSums + NS * 16 + 16;
    static_assert(kStage % 1024 == 0 && kBlocks * (kSmem + 1024) <= 233472, "shared memory of an SM");
};

template <bool BF16, int NT, bool RUNS>
__global__ void __launch_bounds__(FewCfg<NT>::kThreads, FewCfg<NT>::kBlocks)
q4_few_kernel(const __grid_constant__ CUtensorMap map_rows, const __grid_constant__ CUtensorMap map_codes, Runs runs, Weights w, Out o, int box) {
    using T = typename Halves<BF16>::T;
    using C = FewCfg<NT>;
    constexpr int NS = C::NS, MT = C::MT, kFewWarps = C::kWarps;
    extern __shared__ uint8_t smem_raw[];
    const unsigned smem_at = tc5::smem_addr(smem_raw), base = (smem_at + 1023u) & ~1023u, sums_at = base + NS * C::kStage, full = sums_at + C::kSums, empty = full + 8 * NS, misc = empty + 8 * NS;
    volatile int *gave_up = reinterpret_cast<volatile int *>(smem_raw + (misc - smem_at));
    const int warp = tc5::warp_id(), lane = threadIdx.x & 31;
    const int parts = RUNS ? 1 : runs.splits, part = parts > 1 ? int(tc5::cluster_rank()) : 0;   // blocks of a cluster: parts of k
    if (threadIdx.x == 0) {
        *gave_up = 0;
        for (int i = 0; i < NS; ++i) {
            tma::mbar_init(full + 8 * i, 1);
            tma::mbar_init(empty + 8 * i, kFewWarps);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    tc5::Waiter wt{gave_up, &g_mm_timeout};
    Finder<RUNS> find;
    find.start(runs);
    Tile t;
    const int chunks = int((w.K + 255) >> 8), c0 = int(int64_t(chunks) * part / parts), c1 = int(int64_t(chunks) * (part + 1) / parts);
    unsigned slot = 0, phase = 0;

    if (warp == kFewWarps) {
        unsigned n = 0;
        for (int64_t tile = blockIdx.x; !wt.fail && find.find(runs, tile, t); tile += gridDim.x) {
            const int row = int(t.mat * w.N + int64_t(t.wt) * kFewRows);
            for (int c = c0; c < c1; ++c, ++n) {
                if (!wt.wait(empty + 8 * slot, phase ^ 1)) break;
                if (tc5::elect()) {
                    const unsigned at = base + slot * C::kStage, bar = full + 8 * slot;
                    tma::mbar_arrive_expect_tx(bar, C::kC + 4 * box * 128);
                    tma::load2d(at, &map_codes, c * 128, row, bar);
#pragma unroll
                    for (int q = 0; q < 4; ++q) tma::load2d(at + C::kC + q * C::kQuarter, &map_rows, c * 256 + q * 64, t.row0, bar);
                }
                __syncwarp();
                if (++slot == NS) { slot = 0; phase ^= 1; }
            }
        }
        if (wt.fail)   // copies in flight land before the block ends
            for (unsigned i = n > NS ? n - NS : 0; i < n; ++i) tc5::Waiter::drain(full + 8 * (i % NS), (i / NS) & 1);
    } else {
        const int q = lane & 3, g = lane >> 2;
        const int64_t groups = w.K >> w.gshift;
        Tile next;
        bool more = find.find(runs, blockIdx.x, next);
        const bool pairs = w.gshift == 5, both = pairs && (groups & 1) == 0;   // two scales a quarter; as one word
        constexpr int R = 2 * MT;        // this lane's rows: 8 apart
        const uint8_t *es = nullptr;     // the tile's scales from this part on
        uint32_t ro[R];                  // the rows' from there; beyond N the last row's, not written
        uint32_t elo[R], ehi[R];         // the bytes of this lane's 64 values, as they come from memory: put together when used
        auto scales_of = [&](const Tile &tt) {
            const int64_t n0 = int64_t(tt.wt) * kFewRows;
            es = w.scales + (tt.mat * w.N + n0) * groups;
#pragma unroll
            for (int i = 0; i < R; ++i) ro[i] = uint32_t(min(int64_t(warp * 16 * MT + g + 8 * i), w.N - 1 - n0)) * uint32_t(groups) + (q * 64 >> w.gshift);
        };
        // the rows' bytes for chunk c; of a quarter that begins beyond K the row's last, for values that are zero
        auto scales_at = [&](int c) {
            const int first = c * 256 >> w.gshift;
            const uint8_t *const p = es + first;
            uint32_t back = 0, step = 1;
            if (int64_t(c) * 256 + 256 > w.K) {
                const int at = q * 64 >> w.gshift, last = int(groups) - 1 - first;
                back = max(at - (both ? last - 1 : last), 0);
                step = at < last;
            }
#pragma unroll
            for (int i = 0; i < R; ++i) {
                if (both) elo[i] = __ldg(reinterpret_cast<const unsigned short *>(p + (ro[i] - back)));
                else elo[i] = __ldg(p + (ro[i] - back));
                if (pairs && !both) ehi[i] = __ldg(p + (ro[i] - back + step));
            }
        };
        if (more) {
            scales_of(next);
            scales_at(c0);
        }
        for (int64_t tile = blockIdx.x; more && !wt.fail; tile += gridDim.x) {
            t = next;
            more = find.find(runs, tile + gridDim.x, next);
            float acc[MT][2][NT][4] = {};   // two sums each, so that a product need not wait for the one before
            unsigned tok[NT];           // this lane's row of x (of one that is not there: the last one's)
#pragma unroll
            for (int u = 0; u < NT; ++u) tok[u] = min(g + 8 * u, t.rows - 1);
            for (int c = c0; c < c1; ++c) {
                uint32_t eh[R];
#pragma unroll
                for (int i = 0; i < R; ++i) eh[i] = e4m3_pair(both ? elo[i] : pairs ? elo[i] | ehi[i] << 8 : elo[i] * 0x101u);
                if (c + 1 < c1) {
                    scales_at(c + 1);
                } else if (more) {   // the next tile's
                    scales_of(next);
                    scales_at(c0);
                }
                if (!wt.wait(full + 8 * slot, phase)) break;
                const uint8_t *const stage = smem_raw + (base + slot * C::kStage - smem_at);
                // rows g, g + 8, ... of the warp's (the same swizzle): pieces 2 q, 2 q + 1
                const uint8_t *const code = stage + (warp * 16 * MT + g) * 128;
                const uint8_t *xs[NT];
#pragma unroll
                for (int u = 0; u < NT; ++u) xs[u] = stage + C::kC + q * C::kQuarter + tok[u] * 128;
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const int at = ((2 * q + p) ^ g) << 4;
                    uint4 cw[R];
                    typename Halves<BF16>::Scale sc[R];
#pragma unroll
                    for (int i = 0; i < R; ++i) {
                        cw[i] = *reinterpret_cast<const uint4 *>(code + i * 1024 + at);
                        sc[i] = Halves<BF16>::scale(eh[i], p);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint4 b[NT];
#pragma unroll
                        for (int u = 0; u < NT; ++u) b[u] = *reinterpret_cast<const uint4 *>(xs[u] + (((4 * p + j) ^ ((tok[u] + 2 * q) & 7)) << 4));
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            uint32_t lo[4], hi[4];
                            const uint4 &w0 = cw[2 * m], &w1 = cw[2 * m + 1];
                            Halves<BF16>::widen8(j == 0 ? w0.x : j == 1 ? w0.y : j == 2 ? w0.z : w0.w, sc[2 * m], lo);
                            Halves<BF16>::widen8(j == 0 ? w1.x : j == 1 ? w1.y : j == 2 ? w1.z : w1.w, sc[2 * m + 1], hi);
                            const uint32_t a0[4] = {lo[0], hi[0], lo[1], hi[1]}, a1[4] = {lo[2], hi[2], lo[3], hi[3]};
#pragma unroll
                            for (int u = 0; u < NT; ++u) {
                                mma16816(acc[m][0][u], a0, b[u].x, b[u].y, BF16);
                                mma16816(acc[m][1][u], a1, b[u].z, b[u].w, BF16);
                            }
                        }
                    }
                }
                // the copies into this stage come after the reads above, which may still be on their way: the arrival alone
                // does not wait for them (cold, with 7 chunks a block, one call in 8 read a part of a later chunk)
                tma::fence_proxy_async();
                __syncwarp();
                if (lane == 0) tc5::mbar_arrive(empty + 8 * slot);
                if (++slot == NS) { slot = 0; phase ^= 1; }
            }
            if (wt.fail) break;
            // element i of a lane: row of x 8 u + 2 q + (i & 1), weight row 16 m + g + 8 (i >> 1)
            const float scale = __ldg(w.scale + t.mat);
            float *const sums = reinterpret_cast<float *>(smem_raw + (sums_at - smem_at));   // [row of x][weight row]; one tile a block
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int u = 0; u < NT; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = 8 * u + 2 * q + (i & 1), c = (warp * MT + m) * 16 + g + 8 * (i >> 1);
                        const float v = acc[m][0][u][i] + acc[m][1][u][i];
                        const int64_t n = int64_t(t.wt) * kFewRows + c;
                        if (parts > 1) sums[r * kFewRows + c] = v;
                        else if (r < t.rows && n < w.N) static_cast<T *>(o.out)[int64_t(t.row0 + r) * o.ld + n] = from_float<T>(finish<BF16>(v, scale));
                    }
        }
        if (RUNS && o.zero_rest && !wt.fail) zero_rows<T>(o, find.begin, find.end(runs), kFewWarps * 32);
    }
    if (parts > 1) {
        tc5::cluster_sync();
        // this block's share of the tile's weight rows, the parts added in their order
        find.start(runs);
        if (find.find(runs, blockIdx.x, t)) {
            const float scale = __ldg(w.scale);
            const int first = kFewRows * part / parts, share = kFewRows * (part + 1) / parts - first;
            for (int i = threadIdx.x; i < share * t.rows; i += C::kThreads) {
                const int r = i / share, n = first + i % share;
                float v = 0.0f, f[kFewParts];   // on their way together
#pragma unroll
                for (int p = 0; p < kFewParts; ++p) {
                    f[p] = 0.0f;
                    if (p >= parts) continue;
                    unsigned from;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(from) : "r"(sums_at + (r * kFewRows + n) * 4), "r"(p));
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f[p]) : "r"(from) : "memory");
                }
#pragma unroll
                for (int p = 0; p < kFewParts; ++p) v += f[p];
                const int64_t col = int64_t(t.wt) * kFewRows + n;
                if (col < w.N) static_cast<T *>(o.out)[int64_t(t.row0 + r) * o.ld + col] = from_float<T>(finish<BF16>(v, scale));
            }
        }
        tc5::cluster_sync();   // no block leaves while another reads its sums
    }
}

// The parts of the split tiles, added in their order, four columns a thread.
template <bool BF16>
__global__ void __launch_bounds__(256) q4_join_parts_kernel(Runs r, const float *scale, Out o, int64_t rows) {
    using T = typename Halves<BF16>::T;
    const float s = __ldg(scale);
    const bool wide = !((o.ld | o.J) & 3) && !(reinterpret_cast<uintptr_t>(o.out) & 7);
    for (int64_t i = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6); i < rows; i += int64_t(gridDim.x) * 4) {   // row of a tile
        const int64_t at = i / r.bt, u = r.whole + at, t = u / r.wtiles * r.bt + i % r.bt;
        const int64_t col = u % r.wtiles * 256 + (threadIdx.x & 63) * 4;
        if (t >= r.T) continue;
        const float4 *p = reinterpret_cast<const float4 *>(o.parts) + ((at * r.splits) * r.bt + i % r.bt) * 64 + (threadIdx.x & 63);
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int k = 0; k < r.splits; ++k) {
            const float4 a = p[int64_t(k) * r.bt * 64];
            v.x += a.x;
            v.y += a.y;
            v.z += a.z;
            v.w += a.w;
        }
        union { T h[4]; uint2 both; } f;
        f.h[0] = from_float<T>(finish<BF16>(v.x, s));
        f.h[1] = from_float<T>(finish<BF16>(v.y, s));
        f.h[2] = from_float<T>(finish<BF16>(v.z, s));
        f.h[3] = from_float<T>(finish<BF16>(v.w, s));
        T *const to = static_cast<T *>(o.out) + t * o.ld + col;
        if (wide && col < o.J) {
            *reinterpret_cast<uint2 *>(to) = f.both;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (col + j < o.J) to[j] = f.h[j];
        }
    }
}

// ----------------------------------------------------------------------------
// Gradient of the group scales: dW = dy^T x over the rows of a matrix, reduced
// with the codes before it leaves the chip (a 32nd to a 256th of dW is written).
// One tile of a pair of CTAs: 256 rows n (128 each) by 256 columns k (each brings
// half); both operands come as lines of 64 columns, one line per row t, in stages
// of 64 rows.  The sums of kPromote
// stages are taken from tensor memory (two accumulators in turn), multiplied by
// q and added in float32 registers: the result is float32, where what a longer sum
// loses in the tensor core would show (5.4e-7 of the result at 4096 rows).
// Warps 0 .. 7 reduce, warp 8 copies, warp 9 issues (first CTA), warp 10 clears the
// rows behind the last one of a run (they are another matrix's, and may be NaN)
// and tells the first CTA that the stage is there.  Bound by the tensor cores: 4096 x
// 4096 x 14336 in 304 us, 1.58 PFLOP/s.
// ----------------------------------------------------------------------------
constexpr int kPromote = 8, kBand = 8, kDsThreads = 352;

struct DsCfg {
    static constexpr int NS = 6, kA = 16384, kB = 16384, kBar = 3 * NS + 4;
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
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kDsThreads, 1)
q4_dscale_kernel(const __grid_constant__ CUtensorMap map_dy, const __grid_constant__ CUtensorMap map_x, Runs runs, const uint8_t *codes, int64_t N,
                 int64_t K, int gshift, int ntiles, int ktiles, float *dc) {
    using C = DsCfg;
    constexpr int NS = C::NS;
    extern __shared__ uint8_t smem_raw[];
    const unsigned base = (tc5::smem_addr(smem_raw) + 1023u) & ~1023u;
    const unsigned sa = base, sb = sa + NS * C::kA, bars = sb + NS * C::kB;
    const unsigned full = bars, ready = full + 8 * NS, empty = ready + 8 * NS, done = empty + 8 * NS, drained = done + 16, misc = drained + 16;
    uint8_t *const misc_ptr = smem_raw + (misc - tc5::smem_addr(smem_raw));
    volatile int *gave_up = reinterpret_cast<volatile int *>(misc_ptr + 4);
    const unsigned sums_full = misc + 16, sums_empty = misc + 24;
    float *const other = reinterpret_cast<float *>(misc_ptr + 32);   // 128 sums of the second half
    const int warp = tc5::warp_id(), lane = threadIdx.x & 31;
    const unsigned rank = tc5::cluster_rank();
    const int64_t step = gridDim.x >> 1, first = blockIdx.x >> 1;   // pairs
    if (warp == 9) tc5::tmem_alloc<512>(misc);
    if (threadIdx.x == 0) {
        *gave_up = 0;
        for (int i = 0; i < NS; ++i) {
            tma::mbar_init(full + 8 * i, 1);
            tma::mbar_init(ready + 8 * i, 2);
            tma::mbar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            tma::mbar_init(done + 8 * i, 1);
            tma::mbar_init(drained + 8 * i, 16);
        }
        tma::mbar_init(misc + 8, 1);
        tma::mbar_init(sums_full, 4);
        tma::mbar_init(sums_empty, 4);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    tc5::fence_before();
    __syncthreads();
    tc5::cluster_sync();
    tc5::fence_after();
    unsigned tmem;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(misc));
    tmem = __shfl_sync(0xffffffffu, tmem, 0);

    tc5::Waiter wt{gave_up, &g_mm_timeout};
    DsFinder find;
    DsTile t;
    unsigned it = 0, part = 0;   // stages, promoted parts so far

    if (warp == 8) {
        for (int64_t tile = first; !wt.fail && find.find(runs, tile, ntiles, ktiles, t); tile += step) {
            const int n = int((t.rows + 63) / 64);
            for (int s = 0; s < n; ++s, ++it) {
                const int slot = it % NS;
                if (!wt.wait(empty + 8 * slot, ((it / NS) & 1) ^ 1)) break;
                if (lane == 0) {
                    tma::mbar_arrive_expect_tx(full + 8 * slot, C::kA + C::kB);
                    const int row = int(t.lo) + s * 64;
#pragma unroll
                    for (int c = 0; c < 2; ++c) tma::load2d(sa + slot * C::kA + c * 8192, &map_dy, t.nt * 256 + int(rank) * 128 + c * 64, row, full + 8 * slot);
#pragma unroll
                    for (int c = 0; c < 2; ++c) tma::load2d(sb + slot * C::kB + c * 8192, &map_x, t.kt * 256 + int(rank) * 128 + c * 64, row, full + 8 * slot);
                }
            }
        }
        if (wt.fail)
            for (unsigned i = it > NS ? it - NS : 0; i < it; ++i) tc5::Waiter::drain(full + 8 * (i % NS), (i / NS) & 1);
    } else if (warp == 10) {
        for (int64_t tile = first; !wt.fail && find.find(runs, tile, ntiles, ktiles, t); tile += step) {
            const int n = int((t.rows + 63) / 64);
            for (int s = 0; s < n; ++s, ++it) {
                const int slot = it % NS, left = int(min(t.rows - int64_t(s) * 64, int64_t(64)));
                if (!wt.wait(full + 8 * slot, (it / NS) & 1)) break;
                if (left & 15) {
                    const int rows = 16 - (left & 15);
                    for (int i = lane; i < rows * 32; i += 32) {   // 4 blocks of lines, 8 pieces a line
                        const int l = left + i / 32, b = i % 32;
                        const unsigned at = b < 16 ? sa + slot * C::kA + (b >> 3) * 8192 : sb + slot * C::kB + ((b - 16) >> 3) * 8192;
                        sts128(at + l * 128 + (b & 7) * 16, 0, 0, 0, 0);
                    }
                    tma::fence_proxy_async();
                }
                __syncwarp();
                if (lane == 0) tc5::mbar_arrive_remote(tc5::leader_addr(ready + 8 * slot));
                __syncwarp();
            }
        }
    } else if (warp == 9 && rank == 1) {
        // the first CTA issues for both
    } else if (warp == 9) {
        constexpr uint32_t idesc = tc5::idesc_f16(BF16, 256, true, true);
        for (int64_t tile = first; !wt.fail && find.find(runs, tile, ntiles, ktiles, t); tile += step) {
            const int n = int((t.rows + 63) / 64);
            for (int s = 0; s < n; ++s, ++it) {
                const int slot = it % NS;
                const bool begin = s % kPromote == 0, end = s % kPromote == kPromote - 1 || s + 1 == n;
                if (begin && !wt.wait(drained + 8 * (part & 1), ((part >> 1) & 1) ^ 1)) break;
                if (!wt.wait(ready + 8 * slot, (it / NS) & 1)) break;
                const int left = int(min(t.rows - int64_t(s) * 64, int64_t(64)));
                tc5::fence_after();
                const uint64_t a = tc5::desc128(sa + slot * C::kA, 8192, 1024), b = tc5::desc128(sb + slot * C::kB, 8192, 1024);
                const int steps = (left + 15) >> 4;
                const unsigned d = tmem + (part & 1) * 256;
                if (tc5::elect()) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (k < steps) tc5::mma_ss(d, a + k * 128, b + k * 128, idesc, !begin || k > 0);
                    tc5::commit(empty + 8 * slot);
                    if (end) tc5::commit(done + 8 * (part & 1));
                }
                __syncwarp();
                part += end;
            }
        }
        if (wt.fail) {
            if (tc5::elect()) tc5::commit(misc + 8);
            __syncwarp();
            tc5::Waiter::drain(misc + 8, 0);
        }
    } else {
        const int half = warp >> 2, quad = warp & 3;
        const int64_t groups = K >> gshift;
        unsigned tiles = 0;
        for (int64_t tile = first; !wt.fail && find.find(runs, tile, ntiles, ktiles, t); tile += step, ++tiles) {
            const int parts = int((t.rows + 64 * kPromote - 1) / (64 * kPromote));
            const int64_t n = int64_t(t.nt) * 256 + rank * 128 + quad * 32 + lane, k0 = int64_t(t.kt) * 256 + half * 128;
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
                if (lane == 0) tc5::mbar_arrive_remote(tc5::leader_addr(drained + 8 * (part & 1)));
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
    tc5::fence_before();
    __syncthreads();
    tc5::cluster_sync();   // the other CTA's products read this one's memory, its warps arrive here
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
    int splits;       // of each tile from number `whole` on
    int64_t whole, tiles;    // tiles: with the parts, at most
};

// J result columns, `depth` contraction steps.  The tiles that do not fill a round
// of all pairs are split along k, so that the last round is a short one.  The width
// and the parts have the least estimated cycles: a stage of 64 steps takes 2 cycles a
// row of the tile in the tensor cores and about 430 to pass the ring, a tile some 4500
// for its start and end, and joining parts a launch (5700) and their way to memory
// and back.  Measured: 2047 x 14336 x 4096 (448 tiles, 74 pairs) 156 us, 168 with the
// last 4 tiles whole; 4096 x 4096 x 14336 (256 tiles) 294 against 334; 4096 x 4096 at
// 64 rows 15.5 us in four parts, 20 in one, at 512 rows 24 us as 64 tiles of 128
// rows, 34 as two parts of 32 tiles of 256.
Plan plan_for(int64_t T, int64_t mats, bool runs, int64_t J, int64_t depth) {
    Plan p{};
    const int64_t wt = (J + 255) / 256, chunks = (depth + 255) / 256, pairs = uq::num_sms() / 2;
    if (runs) {   // the runs' lengths are not known here: as if they were even
        const int64_t each = std::max<int64_t>(1, T / std::max<int64_t>(mats, 1));
        p.width = p.bt = each <= 64 ? 64 : each <= 128 ? 128 : 256;
        p.splits = 1;
        p.whole = INT64_MAX;
        p.tiles = std::min(T, T / p.bt + mats) * wt;
        return p;
    }
    double best = 0;
    for (int width = 64; width <= 256; width *= 2) {
        const int64_t n = (T + width - 1) / width, tiles = n * wt, bt = ((T + n - 1) / n + 31) / 32 * 32;
        const int64_t whole = tiles / pairs * pairs, rest = tiles - whole;
        for (int64_t s = 1; s <= std::min<int64_t>(16, chunks); ++s) {
            const int64_t part = (chunks + s - 1) / s;
            if (s > 1 && ((chunks + part - 1) / part != s || rest == 0 || rest * s > pairs)) continue;   // an empty part; more than one round
            const auto tile = [&](int64_t c) { return double(c * 4) * std::max(2.0 * double(bt), 430.0) + 4500.0; };
            const double cost = double(whole / pairs) * tile(chunks) + (rest ? tile(part) : 0.0) +
                                (s > 1 ? 5700.0 + double(rest * s * bt) * 256 * 8 / 2100.0 : 0.0);
            if (p.width == 0 || cost < best) {
                best = cost;
                p.width = width;
                p.bt = int(bt);
                p.splits = int(s);
                p.whole = s > 1 ? whole : INT64_MAX;
                p.tiles = s > 1 ? whole + rest * s : tiles;
            }
        }
    }
    return p;
}

size_t parts_bytes(const Plan &p) { return p.splits > 1 ? size_t(p.tiles - p.whole) * p.bt * 256 * 4 : 0; }

template <int BT, bool BF16, bool DX, bool RUNS>
int launch(const void *rows, int64_t lda, const uint8_t *codes, int64_t mats, const Runs &r, const Weights &w, const Out &o, int64_t tiles, cudaStream_t st) {
    using C = Cfg<BT, DX>;
    CUtensorMap mr, mc;
    auto kernel = q4_product_kernel<BT, BF16, DX, RUNS>;
    // before the maps: in a thread without a context (autograd's, at its first call) this binds the device's, which the
    // map encoder needs
    if (uq::set_smem_attr(reinterpret_cast<const void *>(kernel), C::kSmem) != cudaSuccess) return uq::check_cuda("q4_product_kernel attribute");
    const int64_t depth = DX ? w.N : w.K;
    if (!tc5::encode2d(&mr, BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rows, uint64_t(depth), uint64_t(r.T),
                       uint64_t(lda) * 2, 64, BT / 4, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !tc5::encode2d(&mc, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, uint64_t(w.K / 2), uint64_t(mats * w.N), uint64_t(w.K / 2), DX ? 64 : 128,
                       DX ? 256 : 128, DX ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B))
        return uq::fail(UQ_ERR_CUDA, "tensor map of a 4-bit product");
    const int grid = 2 * int(std::min<int64_t>(tiles, uq::num_sms() / 2));
    uq::ProfScope _p(DX ? "q4_dx" : "q4_linear", st);
    kernel<<<grid, kThreads, C::kSmem, st>>>(mr, mc, r, w, o);
    return uq::check_cuda("q4_product_kernel launch");
}

// Whether the kernel for few rows is taken.  Up to 16 rows (for several matrices:
// 16 each if they were even): 4096 x 4096 at 16 rows 7.9 us, by pairs 14; 28672 x
// 8192 44 against 57.  Up to 32 where a single matrix has so few tiles that the
// pairs would have to split k: 4096 x 4096 at 32 rows 10.6 us against 14, but
// 28672 x 8192 68 against 59.
bool few_rows(int64_t T, int64_t mats, bool runs, int64_t N) {
    return T <= 16 * mats || (!runs && T <= 32 && (N + 255) / 256 * 2 <= uq::num_sms() / 2);
}

template <bool BF16, int NT>
int few(const void *x, int64_t ldx, int64_t T, const uint8_t *codes, const Weights &w, int64_t mats, const int32_t *offsets, void *y, int64_t ldy, bool zero,
        cudaStream_t st) {
    using C = FewCfg<NT>;
    const auto kernel = offsets ? q4_few_kernel<BF16, NT, true> : q4_few_kernel<BF16, NT, false>;
    if (uq::set_smem_attr(reinterpret_cast<const void *>(kernel), C::kSmem) != cudaSuccess) return uq::check_cuda("q4_few_kernel attribute");
    int box = 1;   // rows of a copy
    while (box < std::min<int64_t>(T, 8 * NT)) box *= 2;
    CUtensorMap mr, mc;
    if (!tc5::encode2d(&mr, BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, x, uint64_t(w.K), uint64_t(T), uint64_t(ldx) * 2, 64,
                       box, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !tc5::encode2d(&mc, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, uint64_t(w.K / 2), uint64_t(mats * w.N), uint64_t(w.K / 2), 128, kFewRows,
                       CU_TENSOR_MAP_SWIZZLE_128B))
        return uq::fail(UQ_ERR_CUDA, "tensor map of a 4-bit product");
    const int64_t wtiles = (w.N + kFewRows - 1) / kFewRows, tiles = (offsets ? std::min(T, T / (8 * NT) + mats) : 1) * wtiles;
    const int64_t slots = int64_t(uq::num_sms()) * C::kBlocks, chunks = (w.K + 255) / 256;
    // Parts of k: the least time of the busiest SM, in 0.35 us.  m blocks at a time take m + 1 a chunk between them, and 8 to
    // start and end; adding up the parts takes 4 a block of 8 rows.  (1 row, parts 1, 2, 4, 8: 4096 x 4096 13.2, 9.5, 7.3,
    // 7.0 us; 28672 x 8192 34.0, 33.3, 34.0, 37.8.  16 rows of 14336 x 4096 15.4, 17.4, 21.0, 27.4.)
    const auto cost = [&](int64_t p) {
        const int64_t blocks = (tiles * p + uq::num_sms() - 1) / uq::num_sms(), c = (chunks + p - 1) / p, rest = blocks % C::kBlocks;
        return blocks / C::kBlocks * ((C::kBlocks + 1) * c + 8) + (rest ? (rest + 1) * c + 8 : 0) + (p > 1 ? 4 * NT : 0);
    };
    int parts = 1;
    for (int p = 2; p <= kFewParts && !offsets && p <= chunks; p *= 2)
        if (cost(p) < cost(parts)) parts = p;
    const Runs r{offsets, T, mats, 8 * NT, int(wtiles), parts, 0};
    const Out o{y, ldy, w.N, T, zero, nullptr};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = unsigned(parts > 1 ? tiles * parts : std::min(tiles, slots));
    cfg.blockDim = C::kThreads;
    cfg.dynamicSmemBytes = C::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = unsigned(parts);
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    uq::ProfScope _p("q4_few", st);
    if (cudaLaunchKernelEx(&cfg, kernel, mr, mc, r, w, o, box) != cudaSuccess) return uq::check_cuda("q4_few_kernel launch");
    return uq::check_cuda("q4_few_kernel launch");
}

template <bool BF16, bool DX>
int product(const void *rows, int64_t lda, int64_t T, const uint8_t *codes, const Weights &w, int64_t mats, const int32_t *offsets, void *out,
            int64_t ldo, bool zero, void *ws, size_t ws_bytes, cudaStream_t st) {
    const int64_t J = DX ? w.K : w.N, depth = DX ? w.N : w.K;
    const Plan p = plan_for(T, mats, offsets != nullptr, J, depth);
    if (const size_t need = parts_bytes(p); need && (!ws || ws_bytes < need || !al16(ws)))
        return uq::fail(UQ_ERR_WORKSPACE, "4-bit product: workspace of %zu bytes, %zu needed (16-byte aligned)", ws_bytes, need);
    const Runs r{offsets, T, mats, p.bt, int((J + 255) / 256), p.splits, p.whole};
    const Out o{out, ldo, J, T, zero, static_cast<float *>(ws)};
    const auto go = offsets ? p.width == 64    ? launch<64, BF16, DX, true>
                              : p.width == 128 ? launch<128, BF16, DX, true>
                                               : launch<256, BF16, DX, true>
                    : p.width == 64  ? launch<64, BF16, DX, false>
                    : p.width == 128 ? launch<128, BF16, DX, false>
                                     : launch<256, BF16, DX, false>;
    const int rc = go(rows, lda, codes, mats, r, w, o, p.tiles, st);
    if (rc || p.splits == 1) return rc;
    uq::ProfScope _p("q4_join_parts", st);
    const int64_t split_rows = (p.tiles - p.whole) / p.splits * p.bt;
    q4_join_parts_kernel<BF16><<<unsigned(std::min<int64_t>((split_rows + 3) / 4, 1184)), 256, 0, st>>>(r, w.scale, o, split_rows);
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
    const Runs r{offsets, T, mats, 0, 0, 1, 0};
    const int ntiles = int((N + 255) / 256), ktiles = int((K + 255) / 256);
    const int grid = 2 * int(std::min<int64_t>(mats * ntiles * int64_t(ktiles), uq::num_sms() / 2));
    uq::ProfScope _p("q4_dscale", st);
    kernel<<<grid, kDsThreads, DsCfg::kSmem, st>>>(md, mx, r, codes, N, K, uq::ilog2(group), ntiles, ktiles, dc);
    return uq::check_cuda("q4_dscale_kernel launch");
}

// In one step, so that what a kernel on another stream meets meanwhile is either
// told now or kept.
__global__ void q4_take_flags_kernel(int *out) {
    out[0] = atomicExch(&g_mm_timeout, 0);
    out[1] = atomicExch(&g_mm_bad_offset, 0);
}

// The products' wait on a barrier at which nothing arrives, of two warps: the second
// wait of each ends at once.
__global__ void __launch_bounds__(64) q4_wait_selftest_kernel() {
    __shared__ uint64_t bar;
    __shared__ int gave_up;
    if (threadIdx.x == 0) {
        gave_up = 0;
        tma::mbar_init(tc5::smem_addr(&bar), 1);
    }
    __syncthreads();
    tc5::WaiterFor<50> wt{&gave_up, &g_mm_timeout};
    wt.wait(tc5::smem_addr(&bar), 0);
    wt.wait(tc5::smem_addr(&bar), 0);
}

// No matrix: every row is outside every run.
int no_matrix(void *out, int64_t ld, int64_t T, int64_t J, bool zero, cudaStream_t st) {
    if (!zero || T == 0 || J == 0) return UQ_OK;
    if (!out || (T > 1 && ld < J)) return uq::fail(UQ_ERR_INVALID, "4-bit product: output (null pointer or row stride)");
    return cudaMemset2DAsync(out, size_t(std::max(ld, J)) * 2, 0, size_t(J) * 2, size_t(T), st) == cudaSuccess ? UQ_OK : uq::check_cuda("4-bit product");
}

size_t product_workspace(int64_t T, int64_t mats, int64_t J, int64_t depth) {
    if (T <= 0 || mats != 1 || J <= 0 || depth <= 0 || T > kMost || J > kMost || depth > kMost) return 0;
    const Plan p = plan_for(T, mats, false, J, depth);
    return parts_bytes(p);
}

}  // namespace

namespace uq {
namespace q4 {
void mm_take_flags(int *out, cudaStream_t st) {
    uq::ProfScope _p("q4_take_flags", st);
    q4_take_flags_kernel<<<1, 1, 0, st>>>(out);
}
}  // namespace q4
}  // namespace uq

extern "C" {

int uq_q4_wait_selftest(void *stream) {
    q4_wait_selftest_kernel<<<1, 64, 0, UQ_STREAM(stream)>>>();
    return uq::check_cuda("q4_wait_selftest_kernel launch");
}

size_t uq_q4_linear_workspace_bytes(int64_t T, int64_t mats, int64_t N, int64_t K) {
    return T > 0 && mats == 1 && !few_rows(T, 1, false, N) ? product_workspace(T, mats, N, K) : 0;
}

int uq_q4_linear(const void *x, int dtype, int64_t T, int64_t ldx, const uint8_t *codes, const uint8_t *scales, const float *scale,
                 int64_t mats, int64_t N, int64_t K, int group, const int32_t *offsets, void *y, int64_t ldy, int zero_rest,
                 void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check_args("uq_q4_linear", dtype, T, mats, N, K, group, offsets, codes, x, ldx, K, y, ldy, N, false)) return rc;
    if (mats == 0) return no_matrix(y, ldy, T, N, zero_rest, UQ_STREAM(stream));
    if (T == 0 || N == 0) return UQ_OK;
    if (!scales || !scale) return uq::fail(UQ_ERR_INVALID, "uq_q4_linear: null pointer");
    if (!al16(scales)) return uq::fail(UQ_ERR_INVALID, "uq_q4_linear: scales have to be 16-byte aligned");
    const Weights w{scales, scale, N, K, uq::ilog2(group)};
    const cudaStream_t st = UQ_STREAM(stream);
    if (few_rows(T, mats, offsets != nullptr, N)) {
        const auto go = dtype == UQ_BF16 ? T <= 8 * mats ? few<true, 1> : T <= 16 * mats ? few<true, 2> : few<true, 4>
                        : T <= 8 * mats  ? few<false, 1>
                        : T <= 16 * mats ? few<false, 2>
                                         : few<false, 4>;
        return go(x, ldx, T, codes, w, mats, offsets, y, ldy, zero_rest, st);
    }
    return dtype == UQ_BF16 ? product<true, false>(x, ldx, T, codes, w, mats, offsets, y, ldy, zero_rest, workspace, workspace_bytes, st)
                            : product<false, false>(x, ldx, T, codes, w, mats, offsets, y, ldy, zero_rest, workspace, workspace_bytes, st);
}

size_t uq_q4_linear_dx_workspace_bytes(int64_t T, int64_t mats, int64_t N, int64_t K) { return product_workspace(T, mats, K, N); }

int uq_q4_linear_dx(const void *dy, int dtype, int64_t T, int64_t lddy, const uint8_t *codes, const uint8_t *scales, const float *scale,
                    int64_t mats, int64_t N, int64_t K, int group, const int32_t *offsets, void *dx, int64_t lddx, int zero_rest,
                    void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check_args("uq_q4_linear_dx", dtype, T, mats, N, K, group, offsets, codes, dy, lddy, N, dx, lddx, K, false)) return rc;
    if (mats == 0) return no_matrix(dx, lddx, T, K, zero_rest, UQ_STREAM(stream));
    if (T == 0 || N == 0) return UQ_OK;
    if (!scales || !scale) return uq::fail(UQ_ERR_INVALID, "uq_q4_linear_dx: null pointer");
    if (!al16(scales)) return uq::fail(UQ_ERR_INVALID, "uq_q4_linear_dx: scales have to be 16-byte aligned");
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
