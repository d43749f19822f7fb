// Products with 4-bit weights for sm_100a: y = x W^T, its gradient with respect
// to x and to the group scales, for one matrix or one per run of rows.
#include "uq_q4.cuh"

#include <algorithm>

namespace {

using namespace uq::q4;

__device__ int g_mm_bad_offset;

struct Mat {
    const uint8_t *codes, *scales;
    const float *scale;
    int64_t N, K;
    int gshift;
};

// Rows [lo, hi) of matrix i: each offset at least its predecessors, at most T.
__device__ void run_of(const int32_t *offsets, int64_t i, int64_t T, int64_t &lo, int64_t &hi) {
    if (!offsets) { lo = 0; hi = T; return; }
    int64_t top = 0;
    for (int64_t j = 0; j <= i; ++j) {
        const int64_t o = offsets[j];
        if (o < top || o > T) g_mm_bad_offset = 1;
        top = min(max(top, o), T);
    }
    lo = top;
    const int64_t o = offsets[i + 1];
    if (o < top || o > T) g_mm_bad_offset = 1;
    hi = min(max(top, o), T);
}

__device__ __forceinline__ float weight(const Mat &m, int64_t mat, int64_t n, int64_t k) {
    const int64_t row = mat * m.N + n;
    const uint32_t w = reinterpret_cast<const uint32_t *>(m.codes)[(row * m.K + k) >> 3];
    return float(nibble(w, int(k & 7)) - 8) * e4m3_value(m.scales[(row * m.K + k) >> m.gshift]);
}

// out[t, j] = scale sum_i a[t, i] w(i, j): forward i = k, j = n; DX i = n, j = k.
template <typename T, bool DX>
__global__ void __launch_bounds__(256) q4_product_kernel(const T *a, int64_t lda, int64_t rows, Mat m, const int32_t *offsets, T *out, int64_t ldo) {
    __shared__ float sa[64][17], sw[64][17];
    const int64_t mat = blockIdx.z, I = DX ? m.N : m.K, J = DX ? m.K : m.N;
    int64_t lo, hi;
    run_of(offsets, mat, rows, lo, hi);
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int64_t j0 = int64_t(blockIdx.x) * 64;
    for (int64_t t0 = lo + int64_t(blockIdx.y) * 64; t0 < hi; t0 += int64_t(gridDim.y) * 64) {
        float acc[4][4] = {};
        for (int64_t i0 = 0; i0 < I; i0 += 16) {
            for (int e = threadIdx.x; e < 1024; e += 256) {
                const int r = e >> 4, c = e & 15;
                sa[r][c] = t0 + r < hi && i0 + c < I ? to_float(a[(t0 + r) * lda + i0 + c]) : 0.f;
                const int64_t j = j0 + r, i = i0 + c;
                sw[r][c] = j < J && i < I ? (DX ? weight(m, mat, i, j) : weight(m, mat, j, i)) : 0.f;
            }
            __syncthreads();
#pragma unroll
            for (int c = 0; c < 16; ++c)
#pragma unroll
                for (int p = 0; p < 4; ++p)
#pragma unroll
                    for (int q = 0; q < 4; ++q) acc[p][q] = fmaf(sa[ty + 16 * p][c], sw[tx + 16 * q][c], acc[p][q]);
            __syncthreads();
        }
        const float s = m.scale[mat];
        for (int p = 0; p < 4; ++p)
            for (int q = 0; q < 4; ++q) {
                const int64_t t = t0 + ty + 16 * p, j = j0 + tx + 16 * q;
                if (t < hi && j < J) out[t * ldo + j] = from_float<T>(s * acc[p][q]);
            }
    }
}

template <typename T> __global__ void q4_rest_kernel(const int32_t *offsets, int64_t mats, int64_t rows, int64_t J, T *out, int64_t ldo) {
    int64_t lo, hi, d;
    run_of(offsets, 0, rows, lo, d);
    run_of(offsets, mats - 1, rows, d, hi);
    for (int64_t t = blockIdx.x; t < rows; t += gridDim.x)
        if (t < lo || t >= hi)
            for (int64_t j = threadIdx.x; j < J; j += 256) out[t * ldo + j] = from_float<T>(0.f);
}

// One block: 8 weight rows x one group.
template <typename T>
__global__ void __launch_bounds__(256) q4_dscale_kernel(const T *dy, const T *x, int64_t lddy, int64_t ldx, int64_t rows, Mat m, const int32_t *offsets, float *dc) {
    const int64_t mat = blockIdx.z, n = int64_t(blockIdx.y) * 8 + (threadIdx.x >> 5), g = blockIdx.x;
    int64_t lo, hi;
    run_of(offsets, mat, rows, lo, hi);
    if (n >= m.N) return;
    const int lane = threadIdx.x & 31;
    const int64_t row = mat * m.N + n, per = m.K >> m.gshift;
    float sum = 0.f;
    for (int64_t k = (g << m.gshift) + lane; k < ((g + 1) << m.gshift); k += 32) {
        float d = 0.f;
        for (int64_t t = lo; t < hi; ++t) d = fmaf(to_float(dy[t * lddy + n]), to_float(x[t * ldx + k]), d);
        const uint32_t w = reinterpret_cast<const uint32_t *>(m.codes)[(row * m.K + k) >> 3];
        sum = fmaf(float(nibble(w, int(k & 7)) - 8), d, sum);
    }
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) dc[row * per + g] = sum;
}

// Arguments that the three products share; `a` and `b`: the row operands (b may
// be an output without alignment rules) with `na`, `nb` values a row.
int check_args(const char *what, int dtype, int64_t T, int64_t mats, int64_t N, int64_t K, int group, const int32_t *offsets,
               const uint8_t *codes, const void *a, int64_t lda, int64_t na, const void *b, int64_t ldb, int64_t nb, bool b_read) {
    if (dtype != UQ_BF16 && dtype != UQ_F16) return uq::fail(UQ_ERR_INVALID, "%s: dtype code %d is not built (bfloat16, float16)", what, dtype);
    constexpr int64_t most = (int64_t(1) << 31) - 256;
    if (T < 0 || mats < 0 || N < 0 || K <= 0 || !group_ok(group) || K % group || (!offsets && mats != 1) || mats > 65535 ||
        T > most || N > most || K > most)
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

template <bool DX, typename T>
void product(const void *a, int64_t lda, int64_t rows, Mat m, int64_t mats, const int32_t *offsets, void *out, int64_t ldo, bool zero, cudaStream_t st) {
    const int64_t J = DX ? m.K : m.N;
    const dim3 grid(unsigned((J + 63) / 64), unsigned(std::min<int64_t>((rows + 63) / 64, 64)), unsigned(mats));
    { uq::ProfScope _p(DX ? "q4_dx" : "q4_linear", st);
      q4_product_kernel<T, DX><<<grid, 256, 0, st>>>(static_cast<const T *>(a), lda, rows, m, offsets, static_cast<T *>(out), ldo); }
    if (zero && offsets) { uq::ProfScope _p("q4_rest", st); q4_rest_kernel<T><<<148, 256, 0, st>>>(offsets, mats, rows, J, static_cast<T *>(out), ldo); }
}

}  // namespace

namespace uq {
namespace q4 {
bool mm_take_flags(int *timeout, int *offset) {
    const int zero = 0;
    *timeout = 0;
    return cudaMemcpyFromSymbol(offset, g_mm_bad_offset, sizeof(int)) == cudaSuccess &&
           (!*offset || cudaMemcpyToSymbol(g_mm_bad_offset, &zero, sizeof(int)) == cudaSuccess);
}
}  // namespace q4
}  // namespace uq

extern "C" {

size_t uq_q4_linear_workspace_bytes(int64_t, int64_t, int64_t, int64_t) { return 0; }

int uq_q4_linear(const void *x, int dtype, int64_t T, int64_t ldx, const uint8_t *codes, const uint8_t *scales, const float *scale,
                 int64_t mats, int64_t N, int64_t K, int group, const int32_t *offsets, void *y, int64_t ldy, int zero_rest,
                 void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check_args("uq_q4_linear", dtype, T, mats, N, K, group, offsets, codes, x, ldx, K, y, ldy, N, false)) return rc;
    if (T == 0 || N == 0 || mats == 0) return UQ_OK;
    if (!scales || !scale) return uq::fail(UQ_ERR_INVALID, "uq_q4_linear: null pointer");
    const Mat m{codes, scales, scale, N, K, uq::ilog2(group)};
    if (dtype == UQ_BF16) product<false, __nv_bfloat16>(x, ldx, T, m, mats, offsets, y, ldy, zero_rest, UQ_STREAM(stream));
    else product<false, __half>(x, ldx, T, m, mats, offsets, y, ldy, zero_rest, UQ_STREAM(stream));
    return uq::check_cuda("q4_product_kernel launch");
}

size_t uq_q4_linear_dx_workspace_bytes(int64_t, int64_t, int64_t, int64_t) { return 0; }

int uq_q4_linear_dx(const void *dy, int dtype, int64_t T, int64_t lddy, const uint8_t *codes, const uint8_t *scales, const float *scale,
                    int64_t mats, int64_t N, int64_t K, int group, const int32_t *offsets, void *dx, int64_t lddx, int zero_rest,
                    void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check_args("uq_q4_linear_dx", dtype, T, mats, N, K, group, offsets, codes, dy, lddy, N, dx, lddx, K, false)) return rc;
    if (T == 0 || N == 0 || mats == 0) return UQ_OK;
    if (!scales || !scale) return uq::fail(UQ_ERR_INVALID, "uq_q4_linear_dx: null pointer");
    const Mat m{codes, scales, scale, N, K, uq::ilog2(group)};
    if (dtype == UQ_BF16) product<true, __nv_bfloat16>(dy, lddy, T, m, mats, offsets, dx, lddx, zero_rest, UQ_STREAM(stream));
    else product<true, __half>(dy, lddy, T, m, mats, offsets, dx, lddx, zero_rest, UQ_STREAM(stream));
    return uq::check_cuda("q4_product_kernel launch");
}

size_t uq_q4_linear_dscale_workspace_bytes(int64_t, int64_t, int64_t, int64_t, int) { return 0; }

int uq_q4_linear_dscale(const void *dy, const void *x, int dtype, int64_t T, int64_t lddy, int64_t ldx, const uint8_t *codes, int64_t mats,
                        int64_t N, int64_t K, int group, const int32_t *offsets, float *dc, void *workspace, size_t workspace_bytes,
                        void *stream) {
    if (int rc = check_args("uq_q4_linear_dscale", dtype, T, mats, N, K, group, offsets, codes, dy, lddy, N, x, ldx, K, true)) return rc;
    if (N == 0 || mats == 0) return UQ_OK;
    if (!dc) return uq::fail(UQ_ERR_INVALID, "uq_q4_linear_dscale: null pointer");
    const Mat m{codes, nullptr, nullptr, N, K, uq::ilog2(group)};
    const dim3 grid(unsigned(K / group), unsigned((N + 7) / 8), unsigned(mats));
    const cudaStream_t st = UQ_STREAM(stream);
    uq::ProfScope _p("q4_dscale", st);
    if (dtype == UQ_BF16)
        q4_dscale_kernel<<<grid, 256, 0, st>>>(static_cast<const __nv_bfloat16 *>(dy), static_cast<const __nv_bfloat16 *>(x), lddy, ldx, T, m, offsets, dc);
    else
        q4_dscale_kernel<<<grid, 256, 0, st>>>(static_cast<const __half *>(dy), static_cast<const __half *>(x), lddy, ldx, T, m, offsets, dc);
    return uq::check_cuda("q4_dscale_kernel launch");
}

}  // extern "C"
