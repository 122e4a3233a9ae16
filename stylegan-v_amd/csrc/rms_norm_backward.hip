// sgv_rms_norm_backward; the mathematics and the layout: rms_norm_kernel.h
#include "rms_norm_kernel.h"

namespace sgv_rn {

struct bwd_args {
    const void* dy; const void* h; const void* dh; const void* weight; const float* inv_rms;
    void* dx; float* partials;       // partials [gridDim.x, cols]: sums of dy * xh over the rows of a workgroup (NULL: no weight gradient)
    int64_t rows, dy_stride, h_stride, dh_stride;
    int cols, weight_f32, stream;
    float inv_cols;
};

template <typename T, bool STREAM, bool DW, int WK, int TEAM, int NV>
__global__ __launch_bounds__(TEAM <= 64 ? 256 : TEAM) void rms_norm_backward_kernel(const bwd_args p) {
    constexpr int VEC = io<T>::VEC, RPB = TEAM <= 64 ? 256 / TEAM : 1;
    constexpr bool TAIL = TEAM == 1;
    // (1024 threads have 128 registers each: [8192, 9000] fp16 without the weight's gradient 87 -> 74 us with rows in flight, [4096, 10240] fp32 84 -> 111: spilled)
    constexpr bool AHEAD = TEAM < 1024 || (!DW && VEC == 8);
    const bool partial = p.cols % VEC != 0;
    __shared__ red_slots red;
    __shared__ float part[DW && TEAM <= 64 ? 3 * TEAM * NV * VEC : 1];
    int turn = 0;
    const int t = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    int col[NV], shared[NV];
#pragma unroll
    for (int v = 0; v < NV; v++) col[v] = vec_column<TEAM, VEC>(v, t, p.cols, shared[v]);
    u32x4 gv[NV], hv[NV], ev[NV];
    float inv;
    auto load = [&](int64_t row) {
        load_row<T, STREAM, TAIL, NV>((const T*)p.dy + row * p.dy_stride, col, p.cols, gv);
        load_row<T, STREAM, TAIL, NV>((const T*)p.h + row * p.h_stride, col, p.cols, hv);
        if (p.dh) load_row<T, STREAM, TAIL, NV>((const T*)p.dh + row * p.dh_stride, col, p.cols, ev);
        inv = p.inv_rms[row];
    };
    const int64_t stride = (int64_t)gridDim.x * RPB;
    int64_t row = (int64_t)blockIdx.x * RPB + team;
    if (AHEAD && row < p.rows) load(row);
    held_weight<T, WK, TAIL, NV> weight;
#pragma unroll
    for (int v = 0; v < NV; v++) weight.load(p.weight, v, col[v], p.cols);
    float dw[DW ? NV : 1][VEC];
    if constexpr (DW) {
#pragma unroll
        for (int v = 0; v < NV; v++)
#pragma unroll
            for (int j = 0; j < VEC; j++) dw[v][j] = 0.f;
    }
    for (; row < p.rows; row += stride) {
        if (!AHEAD) load(row);
        weight.fresh();
        float g[NV][VEC], xh[NV][VEC], c = 0.f;
        u32x4 e[NV];
        const float iv = inv;
#pragma unroll
        for (int v = 0; v < NV; v++) { io<T>::unpack(gv[v], g[v]); io<T>::unpack(hv[v], xh[v]); e[v] = ev[v]; }
        if (AHEAD && row + stride < p.rows) load(row + stride);
#pragma unroll
        for (int v = 0; v < NV; v++) {
            float w[VEC];
            weight.get(v, w);
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                xh[v][j] *= iv;
                if constexpr (DW) dw[v][j] = __builtin_fmaf(g[v][j], xh[v][j], dw[v][j]);
                if constexpr (WK != W_NONE) g[v][j] *= w[j];
            }
            float sum = c;
#pragma unroll
            for (int j = 0; j < VEC; j++) sum = __builtin_fmaf(g[v][j], xh[v][j], sum);
            if (partial && shared[v] > 0) {
                sum = c;
#pragma unroll
                for (int j = 0; j < VEC; j++) sum = j >= shared[v] ? __builtin_fmaf(g[v][j], xh[v][j], sum) : sum;
            }
            c = sum;
        }
        c = team_sum<TEAM>(c, red, turn) * p.inv_cols;
        if (p.dx) {
#pragma unroll
            for (int v = 0; v < NV; v++) {
                float d[VEC];
                if (p.dh) io<T>::unpack(e[v], d);
                else {
#pragma unroll
                    for (int j = 0; j < VEC; j++) d[j] = 0.f;
                }
#pragma unroll
                for (int j = 0; j < VEC; j++) d[j] = __builtin_fmaf(iv, __builtin_fmaf(-xh[v][j], c, g[v][j]), d[j]);
                put_vec<T, STREAM, TAIL>((T*)p.dx + row * p.cols, col[v], p.cols, io<T>::pack(d));
            }
        }
    }
    if constexpr (DW) {
        if constexpr (TEAM <= 64) {       // the sums of a wave's rows, then those of the four waves, in the order of the waves
            for (int off = TEAM; off < 64; off <<= 1)
#pragma unroll
                for (int v = 0; v < NV; v++)
#pragma unroll
                    for (int j = 0; j < VEC; j++) dw[v][j] += __shfl_xor(dw[v][j], off, 64);
            const int wave = threadIdx.x >> 6;
            if (wave > 0 && (threadIdx.x & 63) < TEAM) {
#pragma unroll
                for (int v = 0; v < NV; v++)
#pragma unroll
                    for (int j = 0; j < VEC; j++) part[((wave - 1) * NV + v) * TEAM * VEC + j * TEAM + t] = dw[v][j];
            }
            __syncthreads();
            if (threadIdx.x >= TEAM) return;
#pragma unroll
            for (int w = 0; w < 3; w++)
#pragma unroll
                for (int v = 0; v < NV; v++)
#pragma unroll
                    for (int j = 0; j < VEC; j++) dw[v][j] += part[(w * NV + v) * TEAM * VEC + j * TEAM + t];
        }
        float* out = p.partials + (int64_t)blockIdx.x * p.cols;
#pragma unroll
        for (int v = 0; v < NV; v++)
            if (TAIL) {
#pragma unroll
                for (int j = 0; j < VEC; j++) if (j < p.cols) out[j] = dw[v][j];
            } else if (col[v] < p.cols) {
#pragma unroll
                for (int q = 0; q < VEC / 4; q++) ((any_f32x4*)(out + col[v] + 4 * q))->v = f32x4{dw[v][4 * q], dw[v][4 * q + 1], dw[v][4 * q + 2], dw[v][4 * q + 3]};
            }
    }
}

// rows that are not held in registers: two walks; a workgroup's weight-gradient sums live in its own row of `partials`
template <typename T, int TEAM>
__global__ __launch_bounds__(TEAM) void rms_norm_backward_long_kernel(const bwd_args p) {
    constexpr int VEC = io<T>::VEC;
    __shared__ red_slots red;
    int turn = 0;
    float* out = p.partials ? p.partials + (int64_t)blockIdx.x * p.cols : nullptr;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* dy = (const T*)p.dy + row * p.dy_stride;
        const T* h = (const T*)p.h + row * p.h_stride;
        const T* dh = p.dh ? (const T*)p.dh + row * p.dh_stride : nullptr;
        const float inv = p.inv_rms[row];
        const bool first = row == (int64_t)blockIdx.x;
        double along = 0.0;
        for (int i = threadIdx.x * VEC; i < p.cols; i += TEAM * VEC) {
            float g[VEC], xh[VEC], w[VEC];
            io<T>::unpack(load_vec<T, true>(dy, i, p.cols), g);
            io<T>::unpack(load_vec<T, true>(h, i, p.cols), xh);
            load_weight<T, true>(p.weight, p.weight_f32, i, p.cols, w);
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                xh[j] *= inv;
                if (out && i + j < p.cols) out[i + j] = first ? g[j] * xh[j] : __builtin_fmaf(g[j], xh[j], out[i + j]);
                along += (double)(g[j] * w[j]) * xh[j];
            }
        }
        const float c = (float)(team_wide<TEAM>(along, red, turn, add_op()) / p.cols);
        if (p.dx)
            for (int i = threadIdx.x * VEC; i < p.cols; i += TEAM * VEC) {
                float g[VEC], xh[VEC], w[VEC], e[VEC];
                io<T>::unpack(load_vec<T, true>(dy, i, p.cols), g);
                io<T>::unpack(load_vec<T, true>(h, i, p.cols), xh);
                load_weight<T, true>(p.weight, p.weight_f32, i, p.cols, w);
#pragma unroll
                for (int j = 0; j < VEC; j++) e[j] = 0.f;
                if (dh) io<T>::unpack(load_vec<T, true>(dh, i, p.cols), e);
#pragma unroll
                for (int j = 0; j < VEC; j++) e[j] = __builtin_fmaf(inv, __builtin_fmaf(-(xh[j] * inv), c, g[j] * w[j]), e[j]);
                store_vec<T, true>((T*)p.dx + row * p.cols, i, p.cols, io<T>::pack(e));
            }
    }
}

// dw[k] = sum of the workgroups' partial rows: 16 columns per workgroup at a time, 64 threads to a column (a wave adds up a column in the end); the order is fixed, so the
// result is too.  A workgroup walks over columns only where a launch of one to every 16 would have 2^32 threads.
constexpr int DW_GROUPS = 1 << 21;
template <typename W>
__global__ __launch_bounds__(1024) void rms_norm_weight_grad_kernel(const float* partials, int count, int cols, W* dw) {
    __shared__ float part[64][17];
    const int c = threadIdx.x & 15, g = threadIdx.x >> 4, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int col = blockIdx.x * 16; col < cols; col += DW_GROUPS * 16) {
        if (col >= DW_GROUPS * 16) __syncthreads();            // (the sums of the columns before have been read)
        const float* p = partials + min(col + c, cols - 1);
        float s = 0.f;
#pragma unroll 8
        for (int r = g; r < count; r += 64) s += p[(int64_t)r * cols];
        part[g][c] = s;
        __syncthreads();
        s = wave_sum(part[lane][wave]);
        if (lane == 0 && col + wave < cols) sgv_traits<W>::store(dw + col + wave, s);
    }
}

template <typename T, bool STREAM, bool DW, int WK>
struct backward_go {
    const bwd_args& p; int64_t blocks; hipStream_t stream;
    template <int TEAM, int NV> void go() const { hipLaunchKernelGGL((rms_norm_backward_kernel<T, STREAM, DW, WK, TEAM, NV>), dim3((unsigned)blocks), dim3(TEAM <= 64 ? 256 : TEAM), 0, stream, p); }
};
template <typename T, bool STREAM, bool DW>
static void launch_backward(const bwd_args& p, const shape& s, int64_t blocks, hipStream_t stream) {
    if (!p.weight) { if constexpr (!DW) for_shape<T>(s, backward_go<T, STREAM, DW, W_NONE>{p, blocks, stream}); }
    else if (io<T>::VEC == 8 && p.weight_f32) { if constexpr (io<T>::VEC == 8) for_shape<T>(s, backward_go<T, STREAM, DW, W_F32>{p, blocks, stream}); }
    else for_shape<T>(s, backward_go<T, STREAM, DW, W_ROWS>{p, blocks, stream});
}
template <typename T>
static void launch_backward(const bwd_args& p, const shape& s, int64_t blocks, hipStream_t stream) {
    if (s.elems == 0) hipLaunchKernelGGL((rms_norm_backward_long_kernel<T, 1024>), dim3((unsigned)blocks), dim3(1024), 0, stream, p);
    else if (p.partials) { if (p.stream) launch_backward<T, true, true>(p, s, blocks, stream); else launch_backward<T, false, true>(p, s, blocks, stream); }
    else { if (p.stream) launch_backward<T, true, false>(p, s, blocks, stream); else launch_backward<T, false, false>(p, s, blocks, stream); }
}

}  // namespace sgv_rn

extern "C" int64_t sgv_rms_norm_backward_workspace_bytes(int64_t rows, int32_t cols, int dtype) {
    if (rows < 1 || cols < 1 || !sgv_rn::row_dtype(dtype)) return 0;
    return sgv_rn::groups(rows, sgv_rn::row_shape(cols, dtype == SGV_F32 ? 4 : 8), true) * cols * 4;
}

extern "C" int sgv_rms_norm_backward(const sgv_rms_norm_backward_params* q, int dtype, void* stream_) {
    if (!q) return sgv_fail(SGV_ERR_INVALID_ARG, "rms_norm_backward: params is NULL");
    if (!sgv_rn::row_dtype(dtype)) return sgv_fail(SGV_ERR_UNSUPPORTED, "rms_norm_backward: rows are fp32, fp16 or bf16");
    if (q->rows < 1 || q->cols < 1) return sgv_fail(SGV_ERR_INVALID_ARG, "rms_norm_backward: rows and cols must be >= 1");
    if (q->cols > sgv_rn::MAX_COLS) return sgv_fail(SGV_ERR_TOO_LARGE, "rms_norm_backward: rows are too long");
    if (!q->dy || !q->h || !q->inv_rms || (!q->dx && !q->dweight)) return sgv_fail(SGV_ERR_INVALID_ARG, "rms_norm_backward: NULL pointer");
    if (q->dweight && !q->weight) return sgv_fail(SGV_ERR_INVALID_ARG, "rms_norm_backward: a gradient of no weight");
    if (q->dy_stride < 0 || q->h_stride < 0 || q->dh_stride < 0) return sgv_fail(SGV_ERR_INVALID_ARG, "rms_norm_backward: negative strides");
    const int vec = dtype == SGV_F32 ? 4 : 8;
    const sgv_rn::shape shape = sgv_rn::row_shape(q->cols, vec);
    const int64_t blocks = sgv_rn::groups(q->rows, shape, q->dweight != nullptr);
    if (q->dweight && (!q->workspace || q->workspace_bytes < blocks * q->cols * 4))
        return sgv_fail(SGV_ERR_INVALID_ARG, "rms_norm_backward: the weight gradient needs sgv_rms_norm_backward_workspace_bytes() of workspace");
    sgv_rn::bwd_args p{};
    p.dy = q->dy; p.h = q->h; p.dh = q->dh; p.weight = q->weight; p.inv_rms = q->inv_rms; p.dx = q->dx; p.partials = q->dweight ? (float*)q->workspace : nullptr;
    p.rows = q->rows; p.dy_stride = q->dy_stride; p.h_stride = q->h_stride; p.dh_stride = q->dh_stride; p.cols = q->cols; p.weight_f32 = q->weight_f32;
    hipStream_t stream = (hipStream_t)stream_;
    const double es = (double)sgv_dtype_size(dtype), n = (double)q->rows * q->cols;
    p.inv_cols = (float)(1.0 / q->cols);
    p.stream = sgv_rn::streams(n * es * (q->dh ? 4 : 3), dtype, q->cols, {{q->dy, q->dy_stride}, {q->h, q->h_stride}, {q->dh, q->dh_stride}, {q->dx, q->cols}});
    sgv_launch_scope scope(SGV_K_RMS_NORM, stream, n * es * (q->dh ? 4 : 3));
    sgv_note_variant(shape.elems == 0 ? SGV_V_rms_norm_backward_walked : p.stream ? SGV_V_rms_norm_backward_held_past_caches : SGV_V_rms_norm_backward_held);
    if (dtype == SGV_F32) sgv_rn::launch_backward<float>(p, shape, blocks, stream);
    else if (dtype == SGV_F16) sgv_rn::launch_backward<sgv_half_t>(p, shape, blocks, stream);
    else sgv_rn::launch_backward<sgv_bf16_t>(p, shape, blocks, stream);
    int rc = sgv_check_launch("rms_norm_backward_kernel");
    if (rc != SGV_OK || !q->dweight) return rc;
    const dim3 grid((unsigned)std::min((q->cols + 15) / 16, sgv_rn::DW_GROUPS));
    const float* part = (const float*)q->workspace;
    if (dtype == SGV_F32 || q->weight_f32) hipLaunchKernelGGL((sgv_rn::rms_norm_weight_grad_kernel<float>), grid, dim3(1024), 0, stream, part, (int)blocks, q->cols, (float*)q->dweight);
    else if (dtype == SGV_F16) hipLaunchKernelGGL((sgv_rn::rms_norm_weight_grad_kernel<sgv_half_t>), grid, dim3(1024), 0, stream, part, (int)blocks, q->cols, (sgv_half_t*)q->dweight);
    else hipLaunchKernelGGL((sgv_rn::rms_norm_weight_grad_kernel<sgv_bf16_t>), grid, dim3(1024), 0, stream, part, (int)blocks, q->cols, (sgv_bf16_t*)q->dweight);
    return sgv_check_launch("rms_norm_weight_grad_kernel");
}

