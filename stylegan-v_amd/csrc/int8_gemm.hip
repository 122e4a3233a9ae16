// Matrix product in 8-bit integers with one scale per row of either operand (sgv_int8_gemm):
//
//   C[m,n] = act( (sum_k A[m,k] B[n,k]) * a_scale[m] * b_scale[n] + bias[n] ) * gain        A [M,K], B [N,K] signed bytes, sums in 32-bit integers
//
// Both operands are contiguous along k, which is how the matrix instructions want them: a lane of v_mfma_i32_16x16x64_i8 holds 16 consecutive bytes of one row.
// The integer sums are exact whatever their order, so K may be split freely and the result does not depend on the split.
#include "sgv_common.h"

#include <algorithm>

namespace sgv_i8 {

typedef int i32x4 __attribute__((ext_vector_type(4)));

struct args {
    const int8_t* a; const int8_t* b; const float* a_scale; const float* b_scale; const float* bias; void* c;
    int64_t lda, ldb, ldc;
    int m, n, k;
    int lrelu;
    float alpha, gain;
};

// 16 bytes of a row at k; bytes at or behind K are cleared (one operand is enough: 0 times anything is 0)
__device__ __forceinline__ i32x4 mask_tail(i32x4 v, int left) {
#pragma unroll
    for (int w = 0; w < 4; w++) {
        const int bytes = left - 4 * w;
        if (bytes <= 0) v[w] = 0;
        else if (bytes < 4) v[w] &= (int)((1u << (8 * bytes)) - 1u);
    }
    return v;
}

__device__ __forceinline__ float finish(const args& p, int acc, float sa, float sb, float bias) {
    float v = __builtin_fmaf((float)acc * sa, sb, bias);
    if (p.lrelu) v = v > 0.f ? v : v * p.alpha;
    return v * p.gain;
}

// Few rows: a workgroup owns 16 MT rows x 16 columns, its waves split K, the partial sums meet in LDS.  Operands go from memory to registers: each is used MT (B) or
// one (A) times per wave, there is nothing to share.
template <typename T, int MT>
__global__ __launch_bounds__(1024) void int8_rows_kernel(const args p) {
    extern __shared__ int red[];                 // [waves][MT * 256]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * (16 * MT);
    const int r = lane & 15, kq = (lane >> 4) * 16;
    const int8_t* b = p.b + (int64_t)min(n0 + r, p.n - 1) * p.ldb + kq;
    const int8_t* a[MT];
#pragma unroll
    for (int t = 0; t < MT; t++) a[t] = p.a + (int64_t)min(m0 + 16 * t + r, p.m - 1) * p.lda + kq;
    i32x4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; t++) acc[t] = i32x4{0, 0, 0, 0};
    constexpr int U = 4;
    const int steps = (p.k + 63) / 64;
    for (int s0 = wave; s0 < steps; s0 += waves * U) {
        i32x4 av[U][MT], bv[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int k0 = (s0 + u * waves) * 64;
            const bool ok = k0 + kq < p.k;
            bv[u] = ok ? *(const i32x4*)(b + k0) : i32x4{0, 0, 0, 0};
#pragma unroll
            for (int t = 0; t < MT; t++) av[u][t] = ok ? *(const i32x4*)(a[t] + k0) : i32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int left = p.k - ((s0 + u * waves) * 64 + kq);
            if (left < 16) bv[u] = mask_tail(bv[u], left);
#pragma unroll
            for (int t = 0; t < MT; t++) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(av[u][t], bv[u], acc[t], 0, 0, 0);
        }
    }
    // C layout of the instruction: column = lane & 15, row = 4 * (lane >> 4) + e
#pragma unroll
    for (int t = 0; t < MT; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) red[wave * (MT * 256) + t * 256 + ((lane >> 4) * 4 + e) * 16 + r] = acc[t][e];
    __syncthreads();
    for (int i = threadIdx.x; i < MT * 256; i += blockDim.x) {
        const int m = m0 + (i >> 4), n = n0 + (i & 15);
        if (m >= p.m || n >= p.n) continue;
        int s = red[i];
        for (int w = 1; w < waves; w++) s += red[w * (MT * 256) + i];
        sgv_traits<T>::store((T*)p.c + (int64_t)m * p.ldc + n, finish(p, s, p.a_scale[m], p.b_scale[n], p.bias ? p.bias[n] : 0.f));
    }
}

template <typename T>
static void launch(const args& p, hipStream_t stream) {
    const int tiles = p.m <= 16 ? 1 : p.m <= 32 ? 2 : 4;
    const int steps = (p.k + 63) / 64;
    const int waves = std::max(1, std::min(tiles == 4 ? 8 : 16, steps));
    const dim3 grid((unsigned)((p.n + 15) / 16), (unsigned)((p.m + 16 * tiles - 1) / (16 * tiles))), block(64 * waves);
    const size_t lds = (size_t)waves * tiles * 1024;
    if (tiles == 1) hipLaunchKernelGGL((int8_rows_kernel<T, 1>), grid, block, lds, stream, p);
    else if (tiles == 2) hipLaunchKernelGGL((int8_rows_kernel<T, 2>), grid, block, lds, stream, p);
    else hipLaunchKernelGGL((int8_rows_kernel<T, 4>), grid, block, lds, stream, p);
}

}  // namespace sgv_i8

extern "C" int sgv_int8_gemm(const sgv_int8_gemm_params* q, int dtype, void* stream_) {
    if (!q) return sgv_fail(SGV_ERR_INVALID_ARG, "int8_gemm: params is NULL");
    if (dtype != SGV_F32 && dtype != SGV_F16 && dtype != SGV_BF16) return sgv_fail(SGV_ERR_UNSUPPORTED, "int8_gemm: the output is fp32, fp16 or bf16");
    if (q->m < 0 || q->n < 0 || q->k < 1) return sgv_fail(SGV_ERR_INVALID_ARG, "int8_gemm: m and n must be >= 0 and k >= 1");
    if (q->k > 131071) return sgv_fail(SGV_ERR_TOO_LARGE, "int8_gemm: k is at most 131071 (a sum of 128 * 128 * k has to fit in 32 bits)");
    if (q->act != 1 && q->act != 3) return sgv_fail(SGV_ERR_INVALID_ARG, "int8_gemm: act must be 1 (linear) or 3 (lrelu)");
    if (q->m == 0 || q->n == 0) return SGV_OK;
    if (!q->a || !q->b || !q->a_scale || !q->b_scale || !q->c) return sgv_fail(SGV_ERR_INVALID_ARG, "int8_gemm: NULL pointer");
    if (((uintptr_t)q->a) % 16 || ((uintptr_t)q->b) % 16 || q->lda % 16 || q->ldb % 16 || q->lda < 0 || q->ldb < 0)
        return sgv_fail(SGV_ERR_INVALID_ARG, "int8_gemm: rows of a and b start on 16 bytes and can be read up to the next multiple of 16 columns");
    if (q->ldc < q->n) return sgv_fail(SGV_ERR_INVALID_ARG, "int8_gemm: rows of c overlap");
    if (((int64_t)q->m + 63) / 64 > 65535) return sgv_fail(SGV_ERR_TOO_LARGE, "int8_gemm: too many rows");
    sgv_i8::args p{};
    p.a = (const int8_t*)q->a; p.b = (const int8_t*)q->b; p.a_scale = q->a_scale; p.b_scale = q->b_scale; p.bias = q->bias; p.c = q->c;
    p.lda = q->lda; p.ldb = q->ldb; p.ldc = q->ldc; p.m = q->m; p.n = q->n; p.k = q->k;
    p.lrelu = q->act == 3; p.alpha = q->alpha; p.gain = q->gain;
    hipStream_t stream = (hipStream_t)stream_;
    const double m = q->m, n = q->n, k = q->k;
    sgv_launch_scope scope(SGV_K_INT8_GEMM, stream, m * k + n * k + m * n * (double)sgv_dtype_size(dtype), 2.0 * m * n * k);
    if (dtype == SGV_F32) sgv_i8::launch<float>(p, stream);
    else if (dtype == SGV_F16) sgv_i8::launch<sgv_half_t>(p, stream);
    else sgv_i8::launch<sgv_bf16_t>(p, stream);
    return sgv_check_launch("int8_gemm kernel");
}
