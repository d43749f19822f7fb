// 4-bit weights with group scales for sm_100a: codec, rounding of trained
// scales, row lookup and the lookup's gradient with respect to the scales.
#include "uq_q4.cuh"

#include <algorithm>

namespace {

using namespace uq::q4;

__device__ int g_q4_bad_token;   // a lookup met a token outside its table

// ----------------------------------------------------------------------------
// Codec
// ----------------------------------------------------------------------------

// Least power of two s >= 2^-117 with top <= 1.75 2^p s, from the bits of top
// (finite, >= 0); 1 if top is 0.  1.75 2^11 = 8 x 448: the largest value is -8
// steps of the largest E4M3 scale.  At s >= 2^-117 the smallest step, 2^-9 s,
// is a normal number.
__device__ __forceinline__ float scale_for(uint32_t top, int p) {
    if (top == 0) return 1.0f;
    int k = int(top >> 23) - 127 - p + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    k = k < -117 ? -117 : k;
    return __uint_as_float(uint32_t(k + 127) << 23);
}

// E4M3 of v, never 0 for v != 0, NaN for a non-finite v.
__device__ __forceinline__ uint8_t e4m3_of(float v) {
    if (!(fabsf(v) <= 448.0f)) return 0x7f;
    const uint8_t b = uint8_t(__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3));
    return (b & 0x7f) == 0 && v != 0.0f ? uint8_t(b | 1) : b;
}

template <typename T> __device__ __forceinline__ void load_weights(const T *p, bool vec, float (&x)[8]) {
    if (vec) {
        load8(p, x);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_float(p[i]);
    }
}

// Largest |x| (as bits) of the group of 8 * lanes values that `lanes`
// neighbouring threads hold eight each.
__device__ __forceinline__ uint32_t group_top(const float (&x)[8], int lanes) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    for (int o = lanes >> 1; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}

// blockIdx.y: matrix.  `words` of eight values a matrix, `wrow` a row; `flat`:
// rows follow one another, so that a word's place needs no division.
struct EncArgs {
    int64_t words, wrow, ldw;
    int group, blocks;       // blocks: of a matrix in q4_top_kernel
    bool vec, flat;
};
constexpr int kWords = 4;    // a thread's loads in flight

template <typename T> __device__ __forceinline__ void load_word(const T *W, const EncArgs &a, int64_t i, float (&x)[8]) {
    load_weights(W + (a.flat ? i * 8 : (i / a.wrow) * a.ldw + (i % a.wrow) * 8), a.vec, x);
}

// top[matrix][block] = max |x| bits over the groups without a non-finite value.
// Bound by memory (4096 x 14336 float32: 49 us, 4.8 TB/s); a group is looked at as a
// whole only where a warp has met such a value.
template <typename T> __global__ void __launch_bounds__(256) q4_top_kernel(const T *W, EncArgs a, int64_t mat_stride, uint32_t *top) {
    __shared__ uint32_t warp_top[8];
    W += blockIdx.y * mat_stride;
    uint32_t best = 0;
    for (int64_t base = int64_t(blockIdx.x) * 256 * kWords; base < a.words; base += int64_t(gridDim.x) * 256 * kWords) {
        float x[kWords][8];
#pragma unroll
        for (int u = 0; u < kWords; ++u) {
            const int64_t i = base + u * 256 + threadIdx.x;
            if (i < a.words) {
                load_word(W, a, i, x[u]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[u][j] = 0.0f;
            }
        }
#pragma unroll
        for (int u = 0; u < kWords; ++u) {
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(x[u][j]) & 0x7fffffffu);
            if (__any_sync(0xffffffffu, m >= 0x7f800000u)) {
                m = group_top(x[u], a.group / 8);
                if (m >= 0x7f800000u) m = 0;
            }
            best = max(best, m);
        }
    }
    best = __reduce_max_sync(0xffffffffu, best);
    if ((threadIdx.x & 31) == 0) warp_top[threadIdx.x >> 5] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int i = 1; i < 8; ++i) best = max(best, warp_top[i]);
        top[int64_t(blockIdx.y) * gridDim.x + blockIdx.x] = best;
    }
}

// `lanes`: threads of a group, eight values each (a constant: the reductions unroll).
// The second reading goes backwards: what the first read last is still in L2
// (4096 x 14336 float32 in 60 us).
template <typename T, int lanes>
__global__ void __launch_bounds__(256) q4_encode_kernel(const T *W, EncArgs a, int64_t mat_stride, const uint32_t *top, float *scale, uint32_t *codes, uint8_t *scales) {
    __shared__ uint32_t warp_top[8];
    uint32_t best = 0;
    for (int i = threadIdx.x; i < a.blocks; i += 256) best = max(best, top[int64_t(blockIdx.y) * a.blocks + i]);
    best = __reduce_max_sync(0xffffffffu, best);
    if ((threadIdx.x & 31) == 0) warp_top[threadIdx.x >> 5] = best;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) best = max(best, warp_top[i]);
    const float s = scale_for(best, 11), inv = __fdiv_rn(0.125f, s);   // s >= 2^-117, and below 2^118: inv is a normal number
    if (blockIdx.x == 0 && threadIdx.x == 0) scale[blockIdx.y] = s;
    W += blockIdx.y * mat_stride;
    codes += blockIdx.y * a.words;
    scales += blockIdx.y * (a.words / lanes);
    const int64_t spans = (a.words + 256 * kWords - 1) / (256 * kWords);
    for (int64_t span = spans - 1 - blockIdx.x; span >= 0; span -= gridDim.x) {
        float xs[kWords][8];
#pragma unroll
        for (int u = 0; u < kWords; ++u) {
            const int64_t i = span * 256 * kWords + u * 256 + threadIdx.x;
            if (i < a.words) {
                load_word(W, a, i, xs[u]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) xs[u][j] = 0.0f;
            }
        }
#pragma unroll
        for (int u = 0; u < kWords; ++u) {
            const int64_t i = span * 256 * kWords + u * 256 + threadIdx.x;
            const float (&x)[8] = xs[u];
            const int sub = int(threadIdx.x) & (lanes - 1);
            // the group's largest and smallest value; `odd` is NaN where one is not finite
            float hi = x[0], lo = x[0], odd = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                hi = fmaxf(hi, x[j]);
                lo = fminf(lo, x[j]);
                odd = fmaf(x[j], 0.0f, odd);
            }
#pragma unroll
            for (int o = lanes >> 1; o > 0; o >>= 1) {
                hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
                lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
                odd += __shfl_xor_sync(0xffffffffu, odd, o);
            }
            const bool finite = odd == 0.0f;
            bool negative = -lo > hi;     // the first value of largest size
            if (__any_sync(0xffffffffu, -lo == hi && hi != 0.0f)) {   // both signs: the one that comes first
                uint32_t first = 0xffffffffu;
#pragma unroll
                for (int j = 7; j >= 0; --j)
                    if (fabsf(x[j]) == hi) first = uint32_t(sub * 8 + j) * 2 + (x[j] < 0.0f ? 1 : 0);
                for (int o = lanes >> 1; o > 0; o >>= 1) first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
                if (-lo == hi) negative = first & 1u;
            }
            if (i >= a.words) continue;   // whole groups: the shuffles above are over
            const float m = fmaxf(hi, -lo);
            // m / (8 s): s is a power of two, so the quotient is exact (or underflows, and e4m3_of keeps its sign)
            const float size = m * inv;
            uint8_t e = finite ? e4m3_of(size == 0.0f && m != 0.0f ? 0x1p-20f : size) : uint8_t(0x7f);
            if (finite && m != 0.0f && !negative) e |= 0x80;   // a positive largest value takes a negative scale
            uint32_t word = 0x88888888u;
            if (finite && m != 0.0f) {
                const float c = s * e4m3_value(e), rc = __frcp_rn(c), half = 0.5f * fabsf(c);
                constexpr float kMagic = 12582912.0f;   // 1.5 2^23: adding it rounds to a whole number, ties to even
                float q[8];
                bool border = false;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    // q = rint(x / c) exactly: t is within 2^-22 of x / c relatively, so rint(t) is off by at most one and
                    // only next to a border; the remainder x - q c is exact (q c has 8 bits) and shows it
                    q[j] = (x[j] * rc + kMagic) - kMagic;
                    border |= fabsf(fmaf(-q[j], c, x[j])) >= half;
                }
                if (border) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float r = fmaf(-q[j], c, x[j]);
                        if (fabsf(r) > half || (fabsf(r) == half && (int(q[j]) & 1))) q[j] += ((r < 0.0f) != (c < 0.0f)) ? -1.0f : 1.0f;
                    }
                }
                // q + 8 in four bits each, gathered in floats of 16 bits: elements 0 2 4 6 and 1 3 5 7
                float pack[2] = {0.0f, 0.0f};
#pragma unroll
                for (int j = 7; j >= 0; --j) pack[j & 1] = fmaf(pack[j & 1], 16.0f, fminf(fmaxf(q[j], -8.0f), 7.0f) + 8.0f);
                word = __byte_perm(__float_as_uint(pack[0] + 8388608.0f), __float_as_uint(pack[1] + 8388608.0f), 0x5410);
            }
            codes[i] = word;
            if (sub == 0) scales[uint64_t(i) / lanes] = e;
        }
    }
}

// A thread writes 16 bytes at a time, so that a warp's store is one run of lines:
// eight values of 16 bits, or (float32) the four of half a word.  Bound by the writes:
// 4096 x 14336 to float32 in 45 us, 5.9 TB/s.
template <typename T>
__global__ void __launch_bounds__(256) q4_decode_kernel(const uint32_t *codes, const uint8_t *scales, const float *scale, int64_t words, int lshift, T *out) {
    constexpr int P = 16 / int(sizeof(T)), H = 8 / P;   // values a store, stores a word
    const float s = __ldg(scale + blockIdx.y);
    codes += blockIdx.y * words;
    scales += blockIdx.y * (words >> lshift);
    out += blockIdx.y * words * 8;
    const int64_t n = words * H, step = int64_t(gridDim.x) * 256 * kWords;
    uint32_t w[kWords];
    uint8_t e[kWords];
    auto load = [&](int64_t at) {
#pragma unroll
        for (int u = 0; u < kWords; ++u) {
            const int64_t i = min(at + u * 256, n - 1) / H;
            w[u] = __ldg(codes + i);
            e[u] = __ldg(scales + (i >> lshift));
        }
    };
    int64_t base = int64_t(blockIdx.x) * 256 * kWords + threadIdx.x;
    if (base < n) load(base);
    for (; base < n; base += step) {
        uint4 r[kWords];
#pragma unroll
        for (int u = 0; u < kWords; ++u) {
            const float c = s * e4m3_value(e[u]);
            const uint32_t v = H == 2 && ((base + u * 256) & 1) ? w[u] >> 8 : w[u];   // elements 4 .. 7 are 8 bits up
            union { uint4 v4; T t[P]; } t;
#pragma unroll
            for (int j = 0; j < P; ++j) t.t[j] = from_float<T>(q_of(v, j) * c);
            r[u] = t.v4;
        }
        if (base + step < n) load(base + step);   // on their way during the stores
#pragma unroll
        for (int u = 0; u < kWords; ++u)
            if (base + u * 256 < n) __stcs(reinterpret_cast<uint4 *>(out) + base + u * 256, r[u]);
    }
}

__global__ void q4_scale_kernel(float *scale, int64_t mats, int p) {
    const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
    if (i < mats) scale[i] = scale_for(__float_as_uint(scale[i]), p);
}

__global__ void __launch_bounds__(256) q4_scales_top_kernel(const float *c, int64_t n, uint32_t *top) {
    uint32_t m = 0;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) {
        const uint32_t b = __float_as_uint(__ldg(c + int64_t(blockIdx.y) * n + i)) & 0x7fffffffu;
        if (b < 0x7f800000u) m = max(m, b);
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0 && m) atomicMax(top + blockIdx.y, m);
}

__global__ void __launch_bounds__(256) q4_round_scales_kernel(const float *c, int64_t n, const float *scale, uint8_t *scales) {
    const float s = scale[blockIdx.y];
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) {
        const float v = __ldg(c + int64_t(blockIdx.y) * n + i);
        const float t = __fdiv_rn(v, s);
        scales[int64_t(blockIdx.y) * n + i] = e4m3_of(t == 0.0f && v != 0.0f ? copysignf(0x1p-20f, v) : t);
    }
}

// ----------------------------------------------------------------------------
// Lookup
// ----------------------------------------------------------------------------

template <typename I> __device__ __forceinline__ int64_t token_at(const I *tokens, int64_t t, int64_t V) {
    const int64_t v = int64_t(__ldg(tokens + t));
    return v >= 0 && v < V ? v : -1;
}

// A block takes a token's row at a time, two words a thread on the way, the next
// token already read: 16384 rows of 4096 in 32 us, 5.2 TB/s, bound by the writes.
// (Four rows on the way a block took more registers, fewer blocks and 49 us.)
template <typename I, typename T>
__global__ void __launch_bounds__(256) q4_embed_kernel(const I *tokens, int64_t n, const uint32_t *codes, const uint8_t *scales,
                                                       const float *scale, int64_t V, int wrow, int lshift, float alpha, T *out) {
    const float f = alpha * __ldg(scale);
    const int per = wrow >> lshift;
    int64_t t = blockIdx.x, v = t < n ? token_at(tokens, t, V) : -1;
    for (; t < n; t += gridDim.x) {
        const int64_t now = v;
        if (t + gridDim.x < n) v = token_at(tokens, t + gridDim.x, V);
        if (now < 0 && threadIdx.x == 0) atomicExch(&g_q4_bad_token, 1);
        const uint32_t *const row = codes + now * wrow;
        const uint8_t *const erow = scales + now * per;
        for (int i = threadIdx.x; i < wrow; i += 512) {
            const bool two = i + 256 < wrow;
            uint32_t w[2] = {0, 0};
            float c[2] = {__int_as_float(0x7fc00000), __int_as_float(0x7fc00000)};
            if (now >= 0) {
                w[0] = __ldg(row + i);
                const uint8_t e0 = __ldg(erow + (i >> lshift));
                uint8_t e1 = 0;
                if (two) {
                    w[1] = __ldg(row + i + 256);
                    e1 = __ldg(erow + ((i + 256) >> lshift));
                }
                c[0] = f * e4m3_value(e0);
                c[1] = f * e4m3_value(e1);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                if (u && !two) break;
                float x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = q_of(w[u], j) * c[u];
                store8(out + (t * wrow + i + 256 * u) * 8, x);
            }
        }
    }
}

// ----------------------------------------------------------------------------
// Gradient of the lookup: positions sorted by token (stable), then each
// token's rows added in order
// ----------------------------------------------------------------------------

constexpr int kTile = 1024, kMaxBits = 9, kMaxBins = 1 << kMaxBits, kMaxChunks = 64;

struct SortPlan {
    int passes, bits;       // digits of `bits` bits
    int64_t chunk;          // consecutive entries of one block, a multiple of kTile
    int chunks;
};

SortPlan sort_plan(int64_t T, int64_t V) {
    SortPlan p;
    int need = 1;
    while ((int64_t(1) << need) <= V) ++need;   // keys 0 .. V (V: no token)
    p.passes = (need + kMaxBits - 1) / kMaxBits;
    p.bits = (need + p.passes - 1) / p.passes;
    const int64_t tiles = (T + kTile - 1) / kTile;
    p.chunk = (tiles + kMaxChunks - 1) / kMaxChunks * kTile;
    p.chunks = int((T + p.chunk - 1) / p.chunk);
    return p;
}

struct Keys {
    const void *tokens;   // first pass: the tokens themselves
    int tokens64;
    int64_t V;
    const uint32_t *keys;
};

__device__ __forceinline__ uint32_t key_at(const Keys &k, int64_t i) {
    if (k.keys) return k.keys[i];
    const int64_t v = k.tokens64 ? token_at(static_cast<const int64_t *>(k.tokens), i, k.V)
                                 : token_at(static_cast<const int32_t *>(k.tokens), i, k.V);
    return v < 0 ? uint32_t(k.V) : uint32_t(v);
}

// The sort's few blocks leave most SMs free: the blocks behind them clear a share
// of the gradient, float4 [lo, hi) of it.
struct Clear {
    float4 *p;
    int64_t lo, hi;
};
__device__ __forceinline__ bool clear_share(const Clear &z, int sorting) {
    if (int(blockIdx.x) < sorting) return false;
    for (int64_t i = z.lo + int64_t(blockIdx.x - sorting) * kTile + threadIdx.x; i < z.hi; i += int64_t(gridDim.x - sorting) * kTile)
        z.p[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    return true;
}

// hist[bin * chunks + chunk]
__global__ void __launch_bounds__(kTile) q4_hist_kernel(Keys k, int64_t T, int64_t chunk, int chunks, int shift, int bits, int *hist, Clear z) {
    __shared__ int h[kMaxBins];
    if (clear_share(z, chunks)) return;
    const int bins = 1 << bits;
    for (int b = threadIdx.x; b < bins; b += kTile) h[b] = 0;
    __syncthreads();
    const int64_t lo = int64_t(blockIdx.x) * chunk, hi = min(lo + chunk, T);
    for (int64_t i = lo + threadIdx.x; i < hi; i += kTile) atomicAdd(h + ((key_at(k, i) >> shift) & (bins - 1)), 1);
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kTile) hist[b * chunks + blockIdx.x] = h[b];
}

// Moves each entry to its place: entries of smaller digits, then those of the
// same digit in earlier chunks, earlier tiles, earlier warps, earlier lanes.
__global__ void __launch_bounds__(kTile) q4_scatter_kernel(Keys k, const uint32_t *pos_in, int64_t T, int64_t chunk, int chunks, int shift, int bits,
                                                           const int *hist, uint32_t *keys_out, uint32_t *pos_out, Clear z) {
    __shared__ int start[kMaxBins];
    __shared__ int wsum[kTile / 32];
    __shared__ unsigned short count[kTile / 32][kMaxBins];
    if (clear_share(z, chunks)) return;
    const int bins = 1 << bits, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int total = 0, before = 0;
    if (tid < bins) {
        for (int c = 0; c < chunks; ++c) {
            const int v = hist[tid * chunks + c];
            before += c < int(blockIdx.x) ? v : 0;
            total += v;
        }
    }
    int incl = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) wsum[warp] = incl;
    __syncthreads();
    int off = 0;
    for (int w = 0; w < warp; ++w) off += wsum[w];
    if (tid < bins) start[tid] = off + incl - total + before;
    const int64_t lo = int64_t(blockIdx.x) * chunk, hi = min(lo + chunk, T);
    for (int64_t base = lo; base < hi; base += kTile) {
        for (int b = lane; b < bins; b += 32) count[warp][b] = 0;
        __syncthreads();
        const int64_t i = base + tid;
        const bool ok = i < hi;
        const uint32_t key = ok ? key_at(k, i) : 0;
        const uint32_t pos = ok ? (pos_in ? pos_in[i] : uint32_t(i)) : 0;
        const int digit = ok ? int((key >> shift) & uint32_t(bins - 1)) : -1;
        const unsigned same = __match_any_sync(0xffffffffu, digit);
        const int rank = __popc(same & ((1u << lane) - 1u));
        if (ok && rank == 0) count[warp][digit] = (unsigned short)__popc(same);
        __syncthreads();
        int sum = 0;
        if (tid < bins) {
            for (int w = 0; w < kTile / 32; ++w) {
                const int v = count[w][tid];
                count[w][tid] = (unsigned short)sum;
                sum += v;
            }
        }
        __syncthreads();
        if (ok) {
            const int at = start[digit] + count[warp][digit] + rank;
            keys_out[at] = key;
            pos_out[at] = pos;
        }
        __syncthreads();
        if (tid < bins) start[tid] += sum;
    }
}

// A block adds the rows of kSeg consecutive sorted entries, 2048 columns.  A
// token whose entries all lie in the piece is written out; of one that goes
// on from the piece before (head) or into the next (tail) the piece's part
// goes to part[piece][head / tail].  Bound by the rows that it gathers: 16384 of
// 4096 values, of 131072 tokens, 49 us, 3.4 TB/s; the sort before it 18 us, the join
// 7.  (Pieces of 16 with four rows on the way 44 us here, but more to join; of 64, 50.)
constexpr int kSeg = 32;

// Eight values of a row as loaded, and as floats.
template <typename T> struct Raw8 {
    union { uint4 v[sizeof(T) / 2]; T t[8]; };
    __device__ __forceinline__ Raw8() {}
    __device__ __forceinline__ void load(const T *p, bool ok) {
#pragma unroll
        for (int i = 0; i < int(sizeof(T)) / 2; ++i) v[i] = ok ? __ldg(reinterpret_cast<const uint4 *>(p) + i) : make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ float at(int j) const { return to_float(t[j]); }
};

template <typename T>
__global__ void __launch_bounds__(256) q4_segment_kernel(const uint32_t *keys, const uint32_t *pos, int64_t n, const T *dout, int64_t ld,
                                                         const uint32_t *codes, int64_t V, int wrow, int lshift, float alpha, float *dc,
                                                         float *part) {
    __shared__ uint32_t skey[kSeg + 2], spos[kSeg];
    const int64_t lo = int64_t(blockIdx.x) * kSeg;
    const int m = int(min(int64_t(kSeg), n - lo));
    // skey[0]: the key before the piece, skey[m + 1]: the one behind it
    for (int i = threadIdx.x; i < m + 2; i += 256) {
        const int64_t j = lo + i - 1;
        skey[i] = j >= 0 && j < n ? keys[j] : 0xffffffffu;
    }
    if (threadIdx.x < m) spos[threadIdx.x] = pos[lo + threadIdx.x];
    __syncthreads();
    const int col = blockIdx.y * 256 + threadIdx.x;   // word of the row
    const bool in = col < wrow;
    const int lanes = 1 << lshift, per = wrow >> lshift;
    float acc[8] = {};
    bool head = skey[0] == skey[1];
    constexpr int U = sizeof(T) == 4 ? 4 : 8;      // rows on the way
    for (int b = 0; b < m; b += U) {
        Raw8<T> d[U];
        uint32_t w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool ok = in && b + u < m && skey[b + u + 1] < uint32_t(V);
            w[u] = ok ? __ldg(codes + int64_t(skey[b + u + 1]) * wrow + col) : 0;
            d[u].load(dout + (ok ? int64_t(spos[b + u]) * ld + col * 8 : 0), ok);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (b + u >= m) break;
            const uint32_t key = skey[b + u + 1];
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] += d[u].at(j);
            const bool last = b + u + 1 == m;
            if (key >= uint32_t(V) || (!last && skey[b + u + 2] == key)) continue;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                sum = fmaf(q_of(w[u], j), acc[j], sum);
                acc[j] = 0.f;
            }
            for (int o = lanes >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (in && (threadIdx.x & (lanes - 1)) == 0) {
                const int g = col >> lshift;
                const bool tail = last && skey[m + 1] == key;
                if (head || tail) part[(int64_t(blockIdx.x) * 2 + (head ? 0 : 1)) * per + g] = sum;
                else dc[int64_t(key) * per + g] = alpha * sum;
            }
            head = false;
        }
    }
}

// Adds the parts of each token that crosses pieces, in order.  Block: the
// piece in which such a token begins (its tail part), then the head parts of
// the pieces that follow while the token goes on.  A padding token has
// a million rows, and a float32 sum of their pieces one by one would be off by more
// the more there are: what each addition rounds away is kept (the two-sum, exact) and
// added up beside it.  (Gradient of 16384 rows of which half are one token: 107 us;
// 112 without that and with half as many loads on the way; in 64 bits 185.)
constexpr int kJoin = 16;
__global__ void __launch_bounds__(256) q4_join_kernel(const uint32_t *keys, int64_t n, int64_t V, int per, float alpha, const float *part, float *dc) {
    const int64_t pieces = (n + kSeg - 1) / kSeg;
    const int64_t p = blockIdx.x;
    if (p + 1 >= pieces) return;
    const int64_t end = (p + 1) * kSeg;              // first entry of the next piece
    const uint32_t key = keys[end - 1];
    if (key >= uint32_t(V) || keys[end] != key) return;                      // nothing goes on from here
    if (p > 0 && keys[p * kSeg] == key && keys[p * kSeg - 1] == key) return;   // it began earlier
    // last piece with this key: the first entry beyond p's that differs
    int64_t lo = p + 1, hi = pieces - 1;             // piece lo begins with the key
    while (lo < hi) {
        const int64_t mid = (lo + hi + 1) / 2;
        if (keys[mid * kSeg] == key) lo = mid; else hi = mid - 1;
    }
    for (int g = threadIdx.x; g < per; g += 256) {
        float sum = part[(p * 2 + 1) * per + g], rest = 0.0f;
        for (int64_t i = p + 1; i <= lo; i += kJoin) {
            float v[kJoin];   // on their way together
#pragma unroll
            for (int u = 0; u < kJoin; ++u) v[u] = i + u <= lo ? part[(i + u) * 2 * per + g] : 0.0f;
#pragma unroll
            for (int u = 0; u < kJoin; ++u) {
                const float next = sum + v[u], got = next - sum;
                rest += (sum - (next - got)) + (v[u] - got);
                sum = next;
            }
        }
        dc[int64_t(key) * per + g] = isfinite(sum) ? float(double(alpha) * (double(sum) + double(rest))) : alpha * sum;
    }
}

// In one step: see uq_q4mm.cu.
__global__ void q4_take_token_flag_kernel(int *out) { *out = atomicExch(&g_q4_bad_token, 0); }

int blocks_for(int64_t work, int per_sm) {
    return int(std::max<int64_t>(1, std::min<int64_t>(work, int64_t(uq::num_sms()) * per_sm)));
}

int top_blocks(int64_t words) { return blocks_for((words + 256 * kWords - 1) / (256 * kWords), 8); }

template <typename T>
int encode(const T *W, int64_t mats, int64_t rows, int64_t cols, int64_t ldw, int group, uint8_t *codes, uint8_t *scales, float *scale, uint32_t *top, cudaStream_t st) {
    EncArgs a;
    a.wrow = cols / 8;
    a.words = rows * a.wrow;
    a.ldw = ldw;
    a.group = group;
    a.blocks = top_blocks(a.words);
    a.vec = al16(W) && ldw * int64_t(sizeof(T)) % 16 == 0;
    a.flat = ldw == cols;
    const dim3 grid(unsigned(a.blocks), unsigned(mats));
    { uq::ProfScope _p("q4_top", st); q4_top_kernel<T><<<grid, 256, 0, st>>>(W, a, rows * ldw, top); }
    {
        uq::ProfScope _p("q4_encode", st);
        uint32_t *const cw = reinterpret_cast<uint32_t *>(codes);
        switch (group) {
            case 32: q4_encode_kernel<T, 4><<<grid, 256, 0, st>>>(W, a, rows * ldw, top, scale, cw, scales); break;
            case 64: q4_encode_kernel<T, 8><<<grid, 256, 0, st>>>(W, a, rows * ldw, top, scale, cw, scales); break;
            case 128: q4_encode_kernel<T, 16><<<grid, 256, 0, st>>>(W, a, rows * ldw, top, scale, cw, scales); break;
            default: q4_encode_kernel<T, 32><<<grid, 256, 0, st>>>(W, a, rows * ldw, top, scale, cw, scales); break;
        }
    }
    return uq::check_cuda("q4_encode_kernel launch");
}

bool form_ok(int64_t mats, int64_t rows, int64_t cols, int group) {
    return mats >= 0 && mats <= 65535 && rows >= 0 && group_ok(group) && cols > 0 && cols % group == 0 && cols < (int64_t(1) << 31) &&
           (rows == 0 || mats < (int64_t(1) << 48) / rows / cols);
}

struct Carve {
    uint32_t *key[2], *pos[2];
    int *hist;
    float *part;
    size_t bytes;
};

Carve carve(void *ws, size_t cap, int64_t T, const SortPlan &p, int64_t per) {
    uq::Carver c(ws, cap);
    Carve r;
    for (int i = 0; i < 2; ++i) {
        r.key[i] = c.take<uint32_t>(size_t(T));
        r.pos[i] = c.take<uint32_t>(size_t(T));
    }
    r.hist = c.take<int>(size_t(p.chunks) << p.bits);
    r.part = c.take<float>(size_t((T + kSeg - 1) / kSeg) * 2 * size_t(per));
    r.bytes = c.off;
    return r;
}

template <typename T>
void segments(const Carve &c, int last, int64_t n, const void *dout, int64_t ld, const uint8_t *codes, int64_t V, int64_t K, int lshift,
              float alpha, float *dc, cudaStream_t st) {
    const int wrow = int(K / 8);
    const dim3 grid(unsigned((n + kSeg - 1) / kSeg), unsigned((wrow + 255) / 256));
    { uq::ProfScope _p("q4_segment", st);
      q4_segment_kernel<T><<<grid, 256, 0, st>>>(c.key[last], c.pos[last], n, static_cast<const T *>(dout), ld,
                                                reinterpret_cast<const uint32_t *>(codes), V, wrow, lshift, alpha, dc, c.part); }
    if (grid.x > 1) { uq::ProfScope _p("q4_join", st); q4_join_kernel<<<grid.x - 1, 256, 0, st>>>(c.key[last], n, V, wrow >> lshift, alpha, c.part, dc); }
}

int lane_shift(int group) { return uq::ilog2(group) - 3; }

}  // namespace

extern "C" {

size_t uq_q4_encode_workspace_bytes(int64_t mats, int64_t rows, int64_t cols) {
    return mats > 0 && rows >= 0 && cols > 0 ? size_t(mats) * top_blocks(rows * (cols / 8)) * 4 : 0;
}

int uq_q4_encode(const void *W, int w_dtype, int64_t mats, int64_t rows, int64_t cols, int64_t ldw, int group, uint8_t *codes,
                 uint8_t *scales, float *scale, void *workspace, size_t workspace_bytes, void *stream) {
    if (!form_ok(mats, rows, cols, group) || ldw < cols)
        return uq::fail(UQ_ERR_INVALID, "uq_q4_encode: bad shape (mats=%lld rows=%lld cols=%lld ld=%lld group=%d; cols must be whole groups of 32, 64, 128 or 256)",
                        (long long)mats, (long long)rows, (long long)cols, (long long)ldw, group);
    if (mats == 0) return UQ_OK;
    if (!scale || (rows && (!W || !codes || !scales))) return uq::fail(UQ_ERR_INVALID, "uq_q4_encode: null pointer");
    if (!al16(codes)) return uq::fail(UQ_ERR_INVALID, "uq_q4_encode: codes not 16-byte aligned");
    if (w_dtype < UQ_F32 || w_dtype > UQ_F16) return uq::fail(UQ_ERR_INVALID, "uq_q4_encode: unknown dtype code %d", w_dtype);
    const size_t need = uq_q4_encode_workspace_bytes(mats, rows, cols);
    if (!workspace || workspace_bytes < need) return uq::fail(UQ_ERR_WORKSPACE, "uq_q4_encode: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    const cudaStream_t st = UQ_STREAM(stream);
    uint32_t *const top = static_cast<uint32_t *>(workspace);
    switch (w_dtype) {
        case UQ_F32: return encode(static_cast<const float *>(W), mats, rows, cols, ldw, group, codes, scales, scale, top, st);
        case UQ_F64: return encode(static_cast<const double *>(W), mats, rows, cols, ldw, group, codes, scales, scale, top, st);
        case UQ_BF16: return encode(static_cast<const __nv_bfloat16 *>(W), mats, rows, cols, ldw, group, codes, scales, scale, top, st);
        default: return encode(static_cast<const __half *>(W), mats, rows, cols, ldw, group, codes, scales, scale, top, st);
    }
}

int uq_q4_decode(const uint8_t *codes, const uint8_t *scales, const float *scale, int64_t mats, int64_t rows, int64_t cols, int group,
                 void *out, int out_dtype, void *stream) {
    if (!form_ok(mats, rows, cols, group))
        return uq::fail(UQ_ERR_INVALID, "uq_q4_decode: bad shape (mats=%lld rows=%lld cols=%lld group=%d)", (long long)mats, (long long)rows, (long long)cols, group);
    if (mats == 0 || rows == 0) return UQ_OK;
    if (!codes || !scales || !scale || !out) return uq::fail(UQ_ERR_INVALID, "uq_q4_decode: null pointer");
    if (!al16(codes) || !al16(out)) return uq::fail(UQ_ERR_INVALID, "uq_q4_decode: codes or out not 16-byte aligned");
    const int64_t words = rows * cols / 8;
    const cudaStream_t st = UQ_STREAM(stream);
    const dim3 grid(unsigned(top_blocks(words * (out_dtype == UQ_F32 ? 2 : 1))), unsigned(mats));
    const int ls = lane_shift(group);
    const uint32_t *cw = reinterpret_cast<const uint32_t *>(codes);
    uq::ProfScope _p("q4_decode", st);
    switch (out_dtype) {
        case UQ_F32: q4_decode_kernel<<<grid, 256, 0, st>>>(cw, scales, scale, words, ls, static_cast<float *>(out)); break;
        case UQ_BF16: q4_decode_kernel<<<grid, 256, 0, st>>>(cw, scales, scale, words, ls, static_cast<__nv_bfloat16 *>(out)); break;
        case UQ_F16: q4_decode_kernel<<<grid, 256, 0, st>>>(cw, scales, scale, words, ls, static_cast<__half *>(out)); break;
        default: return uq::fail(UQ_ERR_INVALID, "uq_q4_decode: dtype code %d is not built", out_dtype);
    }
    return uq::check_cuda("q4_decode_kernel launch");
}

int uq_q4_round_scales(const float *c, int64_t mats, int64_t n, uint8_t *scales, float *scale, void *stream) {
    if (mats < 0 || n < 0 || mats > 65535) return uq::fail(UQ_ERR_INVALID, "uq_q4_round_scales: bad shape (mats=%lld n=%lld)", (long long)mats, (long long)n);
    if (mats == 0) return UQ_OK;
    if (!scale || (n && (!c || !scales))) return uq::fail(UQ_ERR_INVALID, "uq_q4_round_scales: null pointer");
    const cudaStream_t st = UQ_STREAM(stream);
    if (cudaMemsetAsync(scale, 0, size_t(mats) * 4, st) != cudaSuccess) return uq::check_cuda("uq_q4_round_scales");
    const dim3 grid(unsigned(std::max<int64_t>(1, std::min<int64_t>((n + 1023) / 1024, 1184 / std::min<int64_t>(mats, 1184)))), unsigned(mats));
    { uq::ProfScope _p("q4_scales_top", st); q4_scales_top_kernel<<<grid, 256, 0, st>>>(c, n, reinterpret_cast<uint32_t *>(scale)); }
    { uq::ProfScope _p("q4_scale", st); q4_scale_kernel<<<unsigned((mats + 255) / 256), 256, 0, st>>>(scale, mats, 8); }
    if (n) { uq::ProfScope _p("q4_round_scales", st); q4_round_scales_kernel<<<grid, 256, 0, st>>>(c, n, scale, scales); }
    return uq::check_cuda("q4_round_scales_kernel launch");
}

int uq_q4_embed(const void *tokens, int tokens64, int64_t T, const uint8_t *codes, const uint8_t *scales, const float *scale, int64_t V,
                int64_t K, int group, float alpha, void *out, int out_dtype, void *stream) {
    if (T < 0 || !form_ok(1, V, K, group))
        return uq::fail(UQ_ERR_INVALID, "uq_q4_embed: bad shape (T=%lld V=%lld K=%lld group=%d)", (long long)T, (long long)V, (long long)K, group);
    if (T == 0) return UQ_OK;
    if (!tokens || !out || !scale || (V && (!codes || !scales))) return uq::fail(UQ_ERR_INVALID, "uq_q4_embed: null pointer");
    if (!al16(codes) || !al16(out)) return uq::fail(UQ_ERR_INVALID, "uq_q4_embed: codes or out not 16-byte aligned");
    const cudaStream_t st = UQ_STREAM(stream);
    const int grid = blocks_for(T, 16), ls = lane_shift(group), wrow = int(K / 8);
    const uint32_t *cw = reinterpret_cast<const uint32_t *>(codes);
    uq::ProfScope _p("q4_embed", st);
#define UQ_EMBED(TY)                                                                                                                     \
    if (tokens64)                                                                                                                        \
        q4_embed_kernel<<<grid, 256, 0, st>>>(static_cast<const int64_t *>(tokens), T, cw, scales, scale, V, wrow, ls, alpha, static_cast<TY *>(out)); \
    else                                                                                                                                 \
        q4_embed_kernel<<<grid, 256, 0, st>>>(static_cast<const int32_t *>(tokens), T, cw, scales, scale, V, wrow, ls, alpha, static_cast<TY *>(out))
    switch (out_dtype) {
        case UQ_F32: UQ_EMBED(float); break;
        case UQ_BF16: UQ_EMBED(__nv_bfloat16); break;
        case UQ_F16: UQ_EMBED(__half); break;
        default: return uq::fail(UQ_ERR_INVALID, "uq_q4_embed: dtype code %d is not built", out_dtype);
    }
#undef UQ_EMBED
    return uq::check_cuda("q4_embed_kernel launch");
}

size_t uq_q4_embed_dscale_workspace_bytes(int64_t T, int64_t V, int64_t K, int group) {
    if (T <= 0 || T >= (int64_t(1) << 30) || !form_ok(1, V, K, group) || V >= (int64_t(1) << 31) - 1) return 0;
    return carve(nullptr, 0, T, sort_plan(T, V), K / group).bytes;
}

int uq_q4_embed_dscale(const void *tokens, int tokens64, int64_t T, const void *dout, int dtype, int64_t ld, const uint8_t *codes, int64_t V,
                       int64_t K, int group, float alpha, float *dc, void *workspace, size_t workspace_bytes, void *stream) {
    if (T < 0 || T >= (int64_t(1) << 30) || !form_ok(1, V, K, group) || V >= (int64_t(1) << 31) - 1 || (T > 1 && ld < K) || K > (int64_t(1) << 26))
        return uq::fail(UQ_ERR_INVALID, "uq_q4_embed_dscale: bad shape (T=%lld V=%lld K=%lld group=%d ld=%lld)", (long long)T, (long long)V, (long long)K, group, (long long)ld);
    if (V == 0) return UQ_OK;
    if (!dc || !codes || (T && (!tokens || !dout))) return uq::fail(UQ_ERR_INVALID, "uq_q4_embed_dscale: null pointer");
    if (dtype != UQ_F32 && dtype != UQ_BF16 && dtype != UQ_F16) return uq::fail(UQ_ERR_INVALID, "uq_q4_embed_dscale: dtype code %d is not built", dtype);
    if (!al16(codes) || !al16(dc) || !al16(dout) || ld % 8) return uq::fail(UQ_ERR_INVALID, "uq_q4_embed_dscale: codes, dout and dc have to be 16-byte aligned, ld a multiple of 8");
    const cudaStream_t st = UQ_STREAM(stream);
    const int64_t per = K / group;
    if (T == 0) return cudaMemsetAsync(dc, 0, size_t(V * per) * 4, st) == cudaSuccess ? UQ_OK : uq::check_cuda("uq_q4_embed_dscale");
    {
        const SortPlan p = sort_plan(T, V);
        const Carve c = carve(workspace, workspace_bytes, T, p, per);
        if (!workspace || c.bytes > workspace_bytes)
            return uq::fail(UQ_ERR_WORKSPACE, "uq_q4_embed_dscale: workspace of %zu bytes, %zu needed", workspace_bytes, c.bytes);
        // the gradient is cleared beside the sort, a share in each launch; up to three odd floats at its end before
        const int64_t vecs = V * per / 4, launches = 2 * p.passes;
        if (V * per % 4 && cudaMemsetAsync(dc + vecs * 4, 0, size_t(V * per % 4) * 4, st) != cudaSuccess) return uq::check_cuda("uq_q4_embed_dscale");
        const auto share = [&](int i) { return Clear{reinterpret_cast<float4 *>(dc), vecs * i / launches, vecs * (i + 1) / launches}; };
        const unsigned grid = unsigned(p.chunks + std::min<int64_t>(uq::num_sms() * 2, (vecs / launches + kTile) / kTile));
        for (int i = 0; i < p.passes; ++i) {
            const Keys k{tokens, tokens64, V, i ? c.key[(i - 1) & 1] : nullptr};
            { uq::ProfScope _p("q4_hist", st); q4_hist_kernel<<<grid, kTile, 0, st>>>(k, T, p.chunk, p.chunks, i * p.bits, p.bits, c.hist, share(2 * i)); }
            { uq::ProfScope _p("q4_scatter", st);
              q4_scatter_kernel<<<grid, kTile, 0, st>>>(k, i ? c.pos[(i - 1) & 1] : nullptr, T, p.chunk, p.chunks, i * p.bits, p.bits, c.hist, c.key[i & 1], c.pos[i & 1],
                                                        share(2 * i + 1)); }
        }
        const int last = (p.passes - 1) & 1, ls = lane_shift(group);
        switch (dtype) {
            case UQ_F32: segments<float>(c, last, T, dout, ld, codes, V, K, ls, alpha, dc, st); break;
            case UQ_BF16: segments<__nv_bfloat16>(c, last, T, dout, ld, codes, V, K, ls, alpha, dc, st); break;
            default: segments<__half>(c, last, T, dout, ld, codes, V, K, ls, alpha, dc, st); break;
        }
    }
    return uq::check_cuda("q4_segment_kernel launch");
}

int uq_q4_errors(void *stream) {
    const cudaStream_t st = UQ_STREAM(stream);
    if (cudaStreamSynchronize(st) != cudaSuccess) return uq::check_cuda("uq_q4_errors");
    int met[3] = {0, 0, 0}, *taken = nullptr;   // a wait that gave up, an offset, a token
    if (cudaMallocAsync(&taken, sizeof(met), st) != cudaSuccess) return uq::check_cuda("uq_q4_errors");
    mm_take_flags(taken, st);
    { uq::ProfScope _p("q4_take_token_flag", st); q4_take_token_flag_kernel<<<1, 1, 0, st>>>(taken + 2); }
    const int rc = uq::check_cuda("q4_take_flags_kernel launch");
    const cudaError_t copied = cudaMemcpyAsync(met, taken, sizeof(met), cudaMemcpyDeviceToHost, st);
    cudaFreeAsync(taken, st);
    if (cudaStreamSynchronize(st) != cudaSuccess || copied != cudaSuccess) return uq::check_cuda("read 4-bit operator flags");
    if (rc) return rc;
    if (!met[0] && !met[1] && !met[2]) return UQ_OK;
    return uq::fail(met[0] ? UQ_ERR_TIMEOUT : UQ_ERR_INVALID, "%s%s%s%s%s",
                    met[0] ? "a bounded device wait of a 4-bit product timed out" : "", met[0] && (met[1] || met[2]) ? "; " : "",
                    met[2] ? "a token lies outside the table" : "", met[2] && met[1] ? "; " : "",
                    met[1] ? "offsets fall, or go beyond the rows" : "");
}

}  // extern "C"
