// sgv_rms_norm and sgv_dequantize_rows; the mathematics and the layout: rms_norm_kernel.h
#include "rms_norm_kernel.h"

namespace sgv_rn {

struct args {
    const void* x; const void* residual; const void* weight;
    void* y; void* h; float* inv_rms; int8_t* q; float* q_scale;
    int64_t rows, x_stride, residual_stride, q_stride;
    int cols, q_cols;            // q_cols: cols rounded up to 16 -- the 8-bit rows are written that far, with zeros
    int weight_f32, normalize, stream;       // stream: the call moves more than the caches hold
    float eps, inv_cols;
};

// does fp32 hold the sum of squares?  (a sum below the range matters only where eps does not cover it)
__device__ __forceinline__ bool sum_in_range(float ss, float eps) { return ss < 1e37f && (ss > 1e-30f || eps > 1e-20f); }

// The 8-bit values of VEC columns, four to a word.  x(j): 384 + the value in steps of the row -- between 257 and 511, where the float's last place is 2^-15 -- so that its
// bits, shifted by one, hold the whole number in byte 2 (off by 128) and the fraction in the two bytes below: one addition rounds, and values within NEAR / 2^16 of a border
// between two steps show in the low half.  (x is good to 3.5 / 2^16: rcp, two products and the sum of the largest at 2^-24 .. 2^-23 each, 127 times that, and half a last
// place.)  They are decided by the exact sign of 127 u - (N - 1/2) max|u|, halves to the even neighbour; u64(j): the exact u.
constexpr unsigned NEAR = 4;
template <int VEC, typename X, typename U>
__device__ __forceinline__ void quantise(X x, U u64, double amax, unsigned* word) {
    unsigned y[VEC];
    unsigned short near = 0xffff;
    unsigned half = 0x808000u + NEAR;
    asm("" : "+s"(half));                 // (in a register: the shift and the addition are one instruction then, which takes no literal)
#pragma unroll
    for (int j = 0; j < VEC; j++) {
        const float s = x(j);
        y[j] = (__float_as_uint(s) << 1) + half;
        near = min(near, (unsigned short)y[j]);
    }
    if (near < 2 * NEAR) {
#pragma unroll
        for (int j = 0; j < VEC; j++)
            if ((unsigned short)y[j] < 2 * NEAR) {
                const int n = (int)(y[j] << 8) >> 24;
                const double m = (double)n - 0.5, p = amax * m, e = __builtin_fma(u64(j), 127.0, -p) - __builtin_fma(amax, m, -p);
                if (e < 0.0 || (e == 0.0 && (n & 1))) y[j] -= 0x10000u;
            }
    }
#pragma unroll
    for (int w = 0; w < VEC / 4; w++)
        word[w] = __builtin_amdgcn_perm(y[4 * w + 1], y[4 * w], 0x0c0c0602u) | __builtin_amdgcn_perm(y[4 * w + 3], y[4 * w + 2], 0x06020c0cu);
}
template <int VEC>
__device__ __forceinline__ void store_bytes(int8_t* q, const unsigned* word) {
    if constexpr (VEC == 8) ((any_u32x2*)q)->v = u32x2{word[0], word[1]};
    else ((any_u32*)q)->v = word[0];
}

// OUT8: q and its scale, else y.  TEAM threads (up to 64: of a wave, 256 / TEAM rows to a workgroup; else the workgroup) hold a row as NV vectors each and walk over rows; the next
// row's loads are in flight while one is reduced and written.
template <typename T, bool STREAM, bool OUT8, int WK, int TEAM, int NV>
__global__ __launch_bounds__(TEAM <= 64 ? 256 : TEAM) void rms_norm_kernel(const args p) {
    constexpr int VEC = io<T>::VEC, RPB = TEAM <= 64 ? 256 / TEAM : 1;
    constexpr bool TAIL = TEAM == 1;
    // (1024 threads have 128 registers each: rows in flight beside fp32 rows with a weight spill, [4096, 16384] to 8 bits 82 -> 86 us; bf16 without one 60 -> 49)
    constexpr bool AHEAD = TEAM < 1024 || VEC == 8 || !OUT8 || WK == W_NONE;
    __shared__ red_slots red;
    int turn = 0;
    const int t = threadIdx.x % TEAM;
    const bool partial = p.cols % VEC != 0;
    int col[NV], shared[NV];
#pragma unroll
    for (int v = 0; v < NV; v++) col[v] = vec_column<TEAM, VEC>(v, t, p.cols, shared[v]);
    u32x4 xv[NV], rv[NV];
    auto load = [&](int64_t row) {
        const T* x = (const T*)p.x + row * p.x_stride;
        const T* r = p.residual ? (const T*)p.residual + row * p.residual_stride : x;
        load_row<T, STREAM, TAIL, NV>(x, col, p.cols, xv);
        if (p.residual) load_row<T, STREAM, TAIL, NV>(r, col, p.cols, rv);
    };
    const int64_t stride = (int64_t)gridDim.x * RPB;
    int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TEAM;
    if (AHEAD && row < p.rows) load(row);
    held_weight<T, WK, TAIL, NV> weight;
#pragma unroll
    for (int v = 0; v < NV; v++) weight.load(p.weight, v, col[v], p.cols);
    for (; row < p.rows; row += stride) {
        if (!AHEAD) load(row);
        weight.fresh();
        float h[NV][VEC];
#pragma unroll
        for (int v = 0; v < NV; v++) io<T>::unpack(xv[v], h[v]);
        if (p.residual) {
#pragma unroll
            for (int v = 0; v < NV; v++) {
                float rf[VEC];
                io<T>::unpack(rv[v], rf);
#pragma unroll
                for (int j = 0; j < VEC; j++) h[v][j] += rf[j];
                const u32x4 hv = io<T>::pack(h[v]);
                io<T>::unpack(hv, h[v]);
                put_vec<T, STREAM, TAIL>((T*)p.h + row * p.cols, col[v], p.cols, hv);
            }
        }
        if (AHEAD && row + stride < p.rows) load(row + stride);
        float ss = 0.f;
        unsigned top = 0;
#pragma unroll
        for (int v = 0; v < NV; v++) {
            float part = ss;
#pragma unroll
            for (int j = 0; j < VEC; j++) part = __builtin_fmaf(h[v][j], h[v][j], part);
            if (partial && shared[v] > 0) {
                part = ss;
#pragma unroll
                for (int j = 0; j < VEC; j++) part = j >= shared[v] ? __builtin_fmaf(h[v][j], h[v][j], part) : part;
            }
            ss = part;
            if constexpr (OUT8) {
                float w[VEC];
                weight.get(v, w);
                if constexpr (WK == W_NONE) {            // a NaN does not show in this maximum, but in the sum of squares
#pragma unroll
                    for (int j = 0; j < VEC; j += 2) top = max3_abs(top, h[v][j], h[v][j + 1]);
                } else {
#pragma unroll
                    for (int j = 0; j < VEC; j++) top = max(top, abs_bits(h[v][j] * w[j]));
                }
            }
        }
        const unsigned mine = top;
        team_reduce<TEAM, OUT8>(ss, top, red, turn);
        float inv = 1.f;
        if (p.normalize) {
            inv = __builtin_amdgcn_rsqf(__builtin_fmaf(ss, p.inv_cols, p.eps));
            if (!sum_in_range(ss, p.eps)) {
                double s2 = 0.0;
#pragma unroll
                for (int v = 0; v < NV; v++)
#pragma unroll
                    for (int j = 0; j < VEC; j++) s2 += j >= shared[v] ? (double)h[v][j] * h[v][j] : 0.0;
                s2 = team_wide<TEAM>(s2, red, turn, add_op());
                inv = (float)(1.0 / __builtin_sqrt(s2 / p.cols + p.eps));
            }
            if (p.inv_rms && t == 0) p.inv_rms[row] = inv;
        }
        if constexpr (!OUT8) {
#pragma unroll
            for (int v = 0; v < NV; v++) {
                float w[VEC], y[VEC];
                weight.get(v, w);
#pragma unroll
                for (int j = 0; j < VEC; j++) y[j] = WK == W_NONE ? h[v][j] * inv : h[v][j] * inv * w[j];
                put_vec<T, STREAM, TAIL>((T*)p.y + row * p.cols, col[v], p.cols, io<T>::pack(y));
            }
        } else {
            // EXACT: fp32 holds every product h * w (all there is without a weight, and products of two 16-bit values), the maximum too.  Elsewhere the largest product is
            // among those that round to the largest.
            constexpr bool EXACT = WK == W_NONE || (WK == W_ROWS && VEC == 8);
            const float peak = WK == W_NONE && ss != ss ? ss : __uint_as_float(top);
            // wide: the maximum, or that of y, leaves fp32's range or comes near its end (rows of zeros are among these)
            const bool wide = !(peak > 1e-30f && peak < 1e37f && peak * inv < 1e38f);
            double amax = (double)peak, k64 = 0.0;
            bool fine = true;
            float k, scale;
            auto exact_top = [&] {
                double top64 = 0.0;
#pragma unroll
                for (int v = 0; v < NV; v++) {
                    float w[VEC];
                    weight.get(v, w);
#pragma unroll
                    for (int j = 0; j < VEC; j++) top64 = __builtin_fmax(top64, __builtin_fabs((double)h[v][j] * w[j]));
                }
                return top64;
            };
            if (wide) {
                if (peak == peak) amax = team_wide<TEAM>(exact_top(), red, turn, max_op());
                fine = amax > 0.0 && amax < __builtin_inf();
                scale = fine || amax == 0.0 ? (float)(amax * inv / 127.0) : __builtin_nanf("");
                k64 = fine ? 127.0 / amax : 0.0;
                k = 0.f;
            } else {
                if constexpr (!EXACT) {
                    const bool any = mine == top;
                    amax = team_top<TEAM>(any ? exact_top() : 0.0, any, red, turn);
                }
                k = 127.f * __builtin_amdgcn_rcpf(peak);
                scale = peak * inv * (1.f / 127.f);
            }
            if (t == 0) p.q_scale[row] = scale;
            int8_t* q = p.q + row * p.q_stride;
#pragma unroll
            for (int v = 0; v < NV; v++) {
                unsigned word[VEC / 4];
                float w[VEC];
                weight.get(v, w);
                auto u64 = [&](int j) { return (double)h[v][j] * w[j]; };
                if (!fine) {
#pragma unroll
                    for (int e = 0; e < VEC / 4; e++) word[e] = 0u;
                } else if (wide) quantise<VEC>([&](int j) { return (float)(u64(j) * k64) + 384.f; }, u64, amax, word);
                else quantise<VEC>([&](int j) { return __builtin_fmaf(WK == W_NONE ? h[v][j] : h[v][j] * w[j], k, 384.f); }, u64, amax, word);
                if (col[v] < p.cols) store_bytes<VEC>(q + col[v], word);
            }
            for (int i = p.cols + t; i < p.q_cols; i += TEAM) q[i] = 0;
        }
    }
}

// Rows longer than a workgroup holds in registers: TEAM threads walk over the row once per step.  With a residual, the later walks read the h that the same thread wrote.
template <typename T, bool OUT8, int TEAM>
__global__ __launch_bounds__(TEAM) void rms_norm_long_kernel(const args p) {
    constexpr int VEC = io<T>::VEC;
    __shared__ red_slots red;
    int turn = 0;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = (const T*)p.x + row * p.x_stride;
        const T* r = p.residual ? (const T*)p.residual + row * p.residual_stride : nullptr;
        T* hout = r ? (T*)p.h + row * p.cols : nullptr;
        const T* again = r ? (const T*)hout : x;
        double ss = 0.0;                                // (fp64: a thread adds up cols / TEAM squares)
        for (int i = threadIdx.x * VEC; i < p.cols; i += TEAM * VEC) {
            float h[VEC];
            io<T>::unpack(load_vec<T, true>(x, i, p.cols), h);
            if (r) {
                float rf[VEC];
                io<T>::unpack(load_vec<T, true>(r, i, p.cols), rf);
#pragma unroll
                for (int j = 0; j < VEC; j++) h[j] += rf[j];
                const u32x4 hv = io<T>::pack(h);
                io<T>::unpack(hv, h);
                store_vec<T, true>(hout, i, p.cols, hv);
            }
#pragma unroll
            for (int j = 0; j < VEC; j++) ss += (double)h[j] * h[j];
        }
        float inv = 1.f;
        if (p.normalize) {
            ss = team_wide<TEAM>(ss, red, turn, add_op());
            inv = (float)(1.0 / __builtin_sqrt(ss / p.cols + p.eps));
            if (p.inv_rms && threadIdx.x == 0) p.inv_rms[row] = inv;
        }
        if constexpr (!OUT8) {
            for (int i = threadIdx.x * VEC; i < p.cols; i += TEAM * VEC) {
                float h[VEC], w[VEC];
                io<T>::unpack(load_vec<T, true>(again, i, p.cols), h);
                load_weight<T, true>(p.weight, p.weight_f32, i, p.cols, w);
#pragma unroll
                for (int j = 0; j < VEC; j++) h[j] = h[j] * inv * w[j];
                store_vec<T, true>((T*)p.y + row * p.cols, i, p.cols, io<T>::pack(h));
            }
        } else {
            double top = 0.0, bad = 0.0;                // (a maximum passes over NaN)
            for (int i = threadIdx.x * VEC; i < p.cols; i += TEAM * VEC) {
                float h[VEC], w[VEC];
                io<T>::unpack(load_vec<T, true>(again, i, p.cols), h);
                load_weight<T, true>(p.weight, p.weight_f32, i, p.cols, w);
#pragma unroll
                for (int j = 0; j < VEC; j++)
                    if (i + j < p.cols) {
                        const double u = (double)h[j] * w[j];
                        top = __builtin_fmax(top, __builtin_fabs(u));
                        if (u != u) bad = 1.0;
                    }
            }
            top = team_wide<TEAM>(top, red, turn, max_op());
            bad = team_wide<TEAM>(bad, red, turn, max_op());
            const double amax = bad > 0.0 ? __builtin_nan("") : top;
            const bool fine = amax > 0.0 && amax < __builtin_inf();
            if (threadIdx.x == 0) p.q_scale[row] = fine || amax == 0.0 ? (float)(amax * inv / 127.0) : __builtin_nanf("");
            const double k64 = fine ? 127.0 / amax : 0.0;
            for (int i = threadIdx.x * VEC; i < p.q_cols; i += TEAM * VEC) {
                float h[VEC], w[VEC];
                unsigned word[VEC / 4];
#pragma unroll
                for (int j = 0; j < VEC; j++) h[j] = w[j] = 0.f;
                if (i < p.cols) {
                    io<T>::unpack(load_vec<T, true>(again, i, p.cols), h);
                    load_weight<T, true>(p.weight, p.weight_f32, i, p.cols, w);
                }
                if (fine) quantise<VEC>([&](int j) { return i + j < p.cols ? (float)((double)h[j] * w[j] * k64) + 384.f : 384.f; }, [&](int j) { return i + j < p.cols ? (double)h[j] * w[j] : 0.0; }, amax, word);
                else {
#pragma unroll
                    for (int e = 0; e < VEC / 4; e++) word[e] = 0u;
                }
                store_bytes<VEC>(p.q + row * p.q_stride + i, word);
            }
        }
    }
}

// `team` threads to a row, up to four vectors to a thread in flight, the team's width apart: neighbouring lanes store neighbouring 16 bytes
template <typename T>
__global__ __launch_bounds__(256) void dequantize_rows_kernel(const int8_t* q, int64_t q_stride, const float* scale, T* out, int64_t rows, int cols, int team, int stream) {
    constexpr int VEC = io<T>::VEC;
    const int t = threadIdx.x & (team - 1), rpb = 256 / team;
    for (int64_t row = (int64_t)blockIdx.x * rpb + threadIdx.x / team; row < rows; row += (int64_t)gridDim.x * rpb) {
        const float s = scale[row];
        const int8_t* src = q + row * q_stride;
        T* dst = out + row * cols;
        for (int i0 = t * VEC; i0 < cols; i0 += 4 * team * VEC) {
            u32x2 b[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int i = i0 + u * team * VEC;
                b[u] = u32x2{0u, 0u};
                if (i + VEC <= cols) {
                    if constexpr (VEC == 8) b[u] = ((const any_u32x2*)(src + i))->v;
                    else b[u][0] = ((const any_u32*)(src + i))->v;
                }
            }
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int i = i0 + u * team * VEC;
                if (i + VEC <= cols) {
                    float f[VEC];
#pragma unroll
                    for (int e = 0; e < VEC; e++) f[e] = (float)(int8_t)(b[u][e >> 2] >> (8 * (e & 3))) * s;
                    if (stream) stream_vec(dst, i, io<T>::pack(f)); else store_vec<T, false>(dst, i, cols, io<T>::pack(f));
                } else if (i < cols) {
                    for (int e = i; e < cols; e++) sgv_traits<T>::store(dst + e, (float)src[e] * s);
                }
            }
        }
    }
}

template <typename T, bool STREAM, bool OUT8, int WK>
struct forward_go {
    const args& p; int64_t blocks; hipStream_t stream;
    template <int TEAM, int NV> void go() const { hipLaunchKernelGGL((rms_norm_kernel<T, STREAM, OUT8, WK, TEAM, NV>), dim3((unsigned)blocks), dim3(TEAM <= 64 ? 256 : TEAM), 0, stream, p); }
};
template <typename T, bool STREAM, bool OUT8>
static void launch_forward(const args& p, const shape& s, hipStream_t stream) {
    const int64_t blocks = groups(p.rows, s, false);
    if (!p.weight) for_shape<T>(s, forward_go<T, STREAM, OUT8, W_NONE>{p, blocks, stream});
    else if (io<T>::VEC == 8 && p.weight_f32) { if constexpr (io<T>::VEC == 8) for_shape<T>(s, forward_go<T, STREAM, OUT8, W_F32>{p, blocks, stream}); }
    else for_shape<T>(s, forward_go<T, STREAM, OUT8, W_ROWS>{p, blocks, stream});
}
template <typename T, bool OUT8>
static void launch_forward(const args& p, hipStream_t stream) {
    const shape s = row_shape(p.cols, io<T>::VEC);
    const dim3 grid((unsigned)groups(p.rows, s, false));
    if (s.elems == 0) hipLaunchKernelGGL((rms_norm_long_kernel<T, OUT8, 1024>), grid, dim3(1024), 0, stream, p);
    else if (p.stream) launch_forward<T, true, OUT8>(p, s, stream);
    else launch_forward<T, false, OUT8>(p, s, stream);
}
template <typename T>
static void launch_forward(const args& p, hipStream_t stream) {
    if (p.q) launch_forward<T, true>(p, stream); else launch_forward<T, false>(p, stream);
}

}  // namespace sgv_rn

extern "C" int sgv_rms_norm(const sgv_rms_norm_params* q, int dtype, void* stream_) {
    if (!q) return sgv_fail(SGV_ERR_INVALID_ARG, "rms_norm: params is NULL");
    if (!sgv_rn::row_dtype(dtype)) return sgv_fail(SGV_ERR_UNSUPPORTED, "rms_norm: rows are fp32, fp16 or bf16");
    if (q->rows < 0 || q->cols < 1) return sgv_fail(SGV_ERR_INVALID_ARG, "rms_norm: rows must be >= 0 and cols >= 1");
    if (q->cols > sgv_rn::MAX_COLS) return sgv_fail(SGV_ERR_TOO_LARGE, "rms_norm: rows are too long");
    if (!(q->eps >= 0.f)) return sgv_fail(SGV_ERR_INVALID_ARG, "rms_norm: eps must be >= 0");
    if (q->rows == 0) return SGV_OK;
    if (!q->x || (!q->y && !q->q)) return sgv_fail(SGV_ERR_INVALID_ARG, "rms_norm: NULL pointer");
    if (q->y && q->q) return sgv_fail(SGV_ERR_INVALID_ARG, "rms_norm: one output, in the rows' type or in 8 bits");
    if ((q->residual != nullptr) != (q->h != nullptr)) return sgv_fail(SGV_ERR_INVALID_ARG, "rms_norm: a residual comes with the stream it makes, and the other way round");
    if (!q->normalize && !q->q) return sgv_fail(SGV_ERR_INVALID_ARG, "rms_norm: rows that are not normalised have the 8-bit output only");
    const int q_cols = (q->cols + 15) / 16 * 16;
    if (q->q) {
        if (!q->q_scale) return sgv_fail(SGV_ERR_INVALID_ARG, "rms_norm: the 8-bit output needs its scales");
        if (q->q_stride < q_cols || q->q_stride % 16 || ((uintptr_t)q->q) % 16)
            return sgv_fail(SGV_ERR_INVALID_ARG, "rms_norm: 8-bit rows start on 16 bytes and are written up to the next multiple of 16 columns");
    }
    if (q->x_stride < 0 || q->residual_stride < 0) return sgv_fail(SGV_ERR_INVALID_ARG, "rms_norm: negative strides");
    sgv_rn::args p{};
    p.x = q->x; p.residual = q->residual; p.weight = q->weight; p.y = q->y; p.h = q->h; p.inv_rms = q->inv_rms; p.q = (int8_t*)q->q; p.q_scale = q->q_scale;
    p.rows = q->rows; p.x_stride = q->x_stride; p.residual_stride = q->residual_stride; p.q_stride = q->q_stride;
    p.cols = q->cols; p.q_cols = q_cols; p.weight_f32 = q->weight_f32; p.normalize = q->normalize; p.eps = q->eps;
    hipStream_t stream = (hipStream_t)stream_;
    const double es = (double)sgv_dtype_size(dtype), n = (double)q->rows * q->cols, bytes = n * (es * (q->residual ? 3 : 1) + (q->q ? 1.0 : es));
    p.inv_cols = (float)(1.0 / q->cols);
    // (8 bits out: a call mostly reads, and gains from 320 MB: [16384, 4096] fp32 62 -> 56 us; [16384, 4096] bf16, 201 MB, 38.2 -> 38.8 with it)
    p.stream = sgv_rn::streams(q->q ? 1.2 * bytes : bytes, dtype, q->cols, {{q->x, q->x_stride}, {q->residual, q->residual_stride}, {q->h, q->cols}, {q->y, q->cols}});
    sgv_launch_scope scope(SGV_K_RMS_NORM, stream, bytes);
    const bool held = sgv_rn::row_shape(q->cols, dtype == SGV_F32 ? 4 : 8).elems > 0;
    sgv_note_variant(!held ? SGV_V_rms_norm_walked : p.stream ? SGV_V_rms_norm_held_past_caches : SGV_V_rms_norm_held);
    if (dtype == SGV_F32) sgv_rn::launch_forward<float>(p, stream);
    else if (dtype == SGV_F16) sgv_rn::launch_forward<sgv_half_t>(p, stream);
    else sgv_rn::launch_forward<sgv_bf16_t>(p, stream);
    return sgv_check_launch("rms_norm_kernel");
}

extern "C" int sgv_dequantize_rows(const void* q, int64_t q_stride, const float* scale, void* out, int64_t rows, int32_t cols, int dtype, void* stream_) {
    if (!sgv_rn::row_dtype(dtype)) return sgv_fail(SGV_ERR_UNSUPPORTED, "dequantize_rows: the output is fp32, fp16 or bf16");
    if (rows < 0 || cols < 1 || q_stride < 0) return sgv_fail(SGV_ERR_INVALID_ARG, "dequantize_rows: rows must be >= 0 and cols >= 1");
    if (cols > sgv_rn::MAX_COLS) return sgv_fail(SGV_ERR_TOO_LARGE, "dequantize_rows: rows are too long");
    if (rows == 0) return SGV_OK;
    if (!q || !scale || !out) return sgv_fail(SGV_ERR_INVALID_ARG, "dequantize_rows: NULL pointer");
    hipStream_t stream = (hipStream_t)stream_;
    sgv_launch_scope scope(SGV_K_RMS_NORM, stream, (double)rows * cols * (1.0 + sgv_dtype_size(dtype)));
    // two vectors to a thread, up to a workgroup ([262144, 128] to bf16: 8 threads to a row 16 us, one 44, 64 52; [1000000, 5] to fp32: one thread 8.6 us, 64 138)
    const int vec = dtype == SGV_F32 ? 4 : 8;
    int team = 1;
    while (team < 256 && 2 * team * vec < cols) team *= 2;
    // (a call that mostly writes gains from 128 MB: [8192, 8192] to fp32 5.4 -> 6.8 TB/s)
    const int past = sgv_rn::streams(3.0 * rows * cols * sgv_dtype_size(dtype), dtype, cols, {{out, cols}});
    const dim3 grid((unsigned)std::min<int64_t>((rows * team + 255) / 256, 1 << 16));
    const int8_t* in = (const int8_t*)q;
    if (dtype == SGV_F32) hipLaunchKernelGGL((sgv_rn::dequantize_rows_kernel<float>), grid, dim3(256), 0, stream, in, q_stride, scale, (float*)out, rows, cols, team, past);
    else if (dtype == SGV_F16) hipLaunchKernelGGL((sgv_rn::dequantize_rows_kernel<sgv_half_t>), grid, dim3(256), 0, stream, in, q_stride, scale, (sgv_half_t*)out, rows, cols, team, past);
    else hipLaunchKernelGGL((sgv_rn::dequantize_rows_kernel<sgv_bf16_t>), grid, dim3(256), 0, stream, in, q_stride, scale, (sgv_bf16_t*)out, rows, cols, team, past);
    return sgv_check_launch("dequantize_rows_kernel");
}
