// Root-mean-square norm of rows, with the addition of a residual stream in front of it and an 8-bit output behind it (sgv_rms_norm), its gradient
// (sgv_rms_norm_backward), and the way back from 8 bits (sgv_dequantize_rows).
//
//   h = T(x + r)                                     r optional; T = rounding to the tensors' type: h is a tensor of its own, and the norm sees that tensor
//   y = h * inv * w        inv = rsqrt(mean_k h^2 + eps)       w optional, per column
//   8 bits: u = h * w,  q = rint_half_even(127 u / max|u|),  scale = max|y| / 127   (inv cancels out of q)
//   gradient, with g = dy * w and xh = h * inv:  dx = dr = inv * (g - xh * mean_k(g xh)) + dh,   dw = sum_rows dy * xh
//
// All of it is bound by memory (12 operations per element against 3..10 bytes): a row is read once into registers, 16 bytes per lane and load, and nothing is
// read again.  Rows of up to 4 vectors per lane of a wave are one wave's (no barrier at all), longer ones a 256-thread workgroup's, and rows beyond the registers of
// one take a kernel that walks the row three times (its second and third reads come from the L2).  16-byte accesses need no alignment on this chip, so odd
// lengths and strides take the same kernels; only a row's last, partial vector is read element by element.
//
// Statistics are fp32: a lane sums at most 64 squares before the tree.  A row whose squares leave fp32's range (|h| > 1e18, or tiny rows under a tiny eps) is
// summed again in fp64.  The 8-bit values are the correctly rounded ones: fp32 places a value to 2.3e-5 of a step, so a value within 3e-5 of a border
// between two steps is decided by the fp64 quotient; the row maximum is exact because the product of two 16-bit values is exact in fp32, and other products are
// taken in fp64.
#include "sgv_common.h"

#include <algorithm>

namespace sgv_rn {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct any_u32x4 { u32x4 v; } __attribute__((packed, aligned(2)));       // a 16-byte access at any element's address

template <typename T> struct io;
template <> struct io<float> {
    static constexpr int VEC = 4;
    static __device__ __forceinline__ void unpack(const u32x4& r, float* f) {
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = __uint_as_float(r[i]);        // (not __builtin_bit_cast: of a vector's element it takes the first one)
    }
    static __device__ __forceinline__ u32x4 pack(const float* f) {
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; i++) r[i] = __builtin_bit_cast(unsigned, f[i]);
        return r;
    }
};
template <> struct io<sgv_half_t> {
    static constexpr int VEC = 8;
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ void unpack(const u32x4& r, float* f) {
#pragma unroll
        for (int i = 0; i < 4; i++) { const unsigned u = r[i]; const h2 h = __builtin_bit_cast(h2, u); f[2 * i] = (float)h[0]; f[2 * i + 1] = (float)h[1]; }
    }
    static __device__ __forceinline__ u32x4 pack(const float* f) {
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; i++) { const h2 h = {(_Float16)f[2 * i], (_Float16)f[2 * i + 1]}; r[i] = __builtin_bit_cast(unsigned, h); }
        return r;
    }
};
template <> struct io<sgv_bf16_t> {
    static constexpr int VEC = 8;
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ void unpack(const u32x4& r, float* f) {
#pragma unroll
        for (int i = 0; i < 4; i++) { f[2 * i] = __uint_as_float(r[i] << 16); f[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u); }
    }
    static __device__ __forceinline__ u32x4 pack(const float* f) {
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; i++) { const b2 b = {(__bf16)f[2 * i], (__bf16)f[2 * i + 1]}; r[i] = __builtin_bit_cast(unsigned, b); }     // (v_cvt_pk_bf16_f32: to nearest even)
        return r;
    }
};

// The VEC elements of a row at column i; TAIL: a row's length is no multiple of VEC, and elements at or behind `cols` read as zero.
template <typename T, bool TAIL>
__device__ __forceinline__ u32x4 load_vec(const T* row, int i, int cols) {
    constexpr int VEC = io<T>::VEC;
    u32x4 r = {0u, 0u, 0u, 0u};
    if (!TAIL || i + VEC <= cols) {
        r = ((const any_u32x4*)(row + i))->v;
    } else {
        float f[VEC];
#pragma unroll
        for (int j = 0; j < VEC; j++) f[j] = i + j < cols ? (float)sgv_traits<T>::load(row + i + j) : 0.f;
        r = io<T>::pack(f);          // (exact: the values came from T)
    }
    return r;
}
template <typename T, bool TAIL>
__device__ __forceinline__ void store_vec(T* row, int i, int cols, const u32x4& v) {
    constexpr int VEC = io<T>::VEC;
    if (!TAIL || i + VEC <= cols) {
        ((any_u32x4*)(row + i))->v = v;
    } else {
        float f[VEC];
        io<T>::unpack(v, f);
#pragma unroll
        for (int j = 0; j < VEC; j++) if (i + j < cols) sgv_traits<T>::store(row + i + j, f[j]);
    }
}
// The weight of those columns as fp32 (ones without a weight); `f32`: the weight is kept in fp32 beside 16-bit rows.
template <typename T, bool TAIL>
__device__ __forceinline__ void load_weight(const void* w, bool f32, int i, int cols, float* f) {
    constexpr int VEC = io<T>::VEC;
    if (!w) {
#pragma unroll
        for (int j = 0; j < VEC; j++) f[j] = 1.f;
    } else if (f32 && VEC == 8) {
        io<float>::unpack(load_vec<float, TAIL>((const float*)w, i, cols), f);
        if (!TAIL || i + 4 < cols) io<float>::unpack(load_vec<float, TAIL>((const float*)w, i + 4, cols), f + 4);
        else {
#pragma unroll
            for (int j = 4; j < VEC; j++) f[j] = 0.f;
        }
    } else {
        io<T>::unpack(load_vec<T, TAIL>((const T*)w, i, cols), f);
    }
}

// Reductions over the threads of a row: a wave's by lane exchange, a workgroup's through LDS with one barrier.  Two slots in turn: a slot is written
// again only behind the barrier of the reduction in between, which every wave reaches after it has read the slot.
struct red_slots { double v[2][16]; };
template <int TEAM, typename V, typename F>
__device__ __forceinline__ V team_reduce(V v, red_slots& s, int& turn, F f) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = f(v, __shfl_xor(v, off, 64));
    if constexpr (TEAM > 64) {
        V* slot = (V*)s.v[turn];
        turn ^= 1;
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) slot[wave] = v;
        __syncthreads();
        v = slot[0];
#pragma unroll
        for (int w = 1; w < TEAM / 64; w++) v = f(v, slot[w]);
    }
    return v;
}
struct add_op { template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return a + b; } };
struct max_op { template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return a > b ? a : b; } };

__device__ __forceinline__ unsigned abs_bits(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }                       // orders magnitudes, NaN above infinity
__device__ __forceinline__ unsigned long long abs_bits(double v) { return __builtin_bit_cast(unsigned long long, v) & 0x7fffffffffffffffull; }

struct args {
    const void* x; const void* residual; const void* weight;
    void* y; void* h; float* inv_rms; int8_t* q; float* q_scale;
    int64_t rows, x_stride, residual_stride, q_stride;
    int cols, q_cols;            // q_cols: cols rounded up to 16 -- the 8-bit rows are written that far, with zeros
    int weight_f32, normalize, wide;     // wide: products h * w are not exact in fp32
    float eps;
};

// does fp32 hold the sum of squares?  (a sum below the range matters only where eps does not cover it)
__device__ __forceinline__ bool sum_in_range(float ss, float eps) { return ss < 1e37f && (ss > 1e-30f || eps > 1e-20f); }

// the 8-bit values of VEC columns, four to a word.  k = 127 / max|u|; u64(j) = the exact product.
template <int VEC, typename U>
__device__ __forceinline__ void quantise(const float* t, U u64, double amax, unsigned* word) {
#pragma unroll
    for (int w = 0; w < VEC / 4; w++) {
        unsigned b[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float v = t[4 * w + j];
            float r = __builtin_rintf(v);
            if (__builtin_fabsf(v - r) > 0.49997f) r = (float)__builtin_rint(u64(4 * w + j) * 127.0 / amax);
            b[j] = (unsigned)(int)r & 0xffu;
        }
        word[w] = b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24;
    }
}

// OUT 0: y; 1: q and its scale.  TEAM threads (64: a wave, four rows per workgroup; 256: the workgroup) hold a row as NV vectors each.
template <typename T, int OUT, int TEAM, int NV, bool TAIL>
__global__ __launch_bounds__(256) void rms_norm_kernel(const args p) {
    constexpr int VEC = io<T>::VEC, RPB = 256 / TEAM;
    __shared__ red_slots red;
    int turn = 0;
    const int t = threadIdx.x % TEAM;
    for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TEAM; row < p.rows; row += (int64_t)gridDim.x * RPB) {
        const T* x = (const T*)p.x + row * p.x_stride;
        const T* r = p.residual ? (const T*)p.residual + row * p.residual_stride : nullptr;
        float h[NV][VEC];
        u32x4 xv[NV], rv[NV];
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const int i = (v * TEAM + t) * VEC;
            xv[v] = u32x4{0u, 0u, 0u, 0u};
            rv[v] = u32x4{0u, 0u, 0u, 0u};
            if (i < p.cols) {
                xv[v] = load_vec<T, TAIL>(x, i, p.cols);
                if (r) rv[v] = load_vec<T, TAIL>(r, i, p.cols);
            }
        }
        float ss = 0.f;
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const int i = (v * TEAM + t) * VEC;
            io<T>::unpack(xv[v], h[v]);
            if (r) {
                float rf[VEC];
                io<T>::unpack(rv[v], rf);
#pragma unroll
                for (int j = 0; j < VEC; j++) h[v][j] += rf[j];
                const u32x4 hv = io<T>::pack(h[v]);
                io<T>::unpack(hv, h[v]);
                if (i < p.cols) store_vec<T, TAIL>((T*)p.h + row * p.cols, i, p.cols, hv);
            }
#pragma unroll
            for (int j = 0; j < VEC; j++) ss = __builtin_fmaf(h[v][j], h[v][j], ss);
        }
        float inv = 1.f;
        if (p.normalize) {
            ss = team_reduce<TEAM>(ss, red, turn, add_op());
            inv = 1.0f / __builtin_sqrtf(ss / (float)p.cols + p.eps);
            if (!sum_in_range(ss, p.eps)) {
                double s2 = 0.0;
#pragma unroll
                for (int v = 0; v < NV; v++)
#pragma unroll
                    for (int j = 0; j < VEC; j++) s2 += (double)h[v][j] * h[v][j];
                s2 = team_reduce<TEAM>(s2, red, turn, add_op());
                inv = (float)(1.0 / __builtin_sqrt(s2 / p.cols + p.eps));
            }
            if (p.inv_rms && t == 0) p.inv_rms[row] = inv;
        }
        if constexpr (OUT == 0) {
#pragma unroll
            for (int v = 0; v < NV; v++) {
                const int i = (v * TEAM + t) * VEC;
                if (i < p.cols) {
                    float w[VEC], y[VEC];
                    load_weight<T, TAIL>(p.weight, p.weight_f32, i, p.cols, w);
#pragma unroll
                    for (int j = 0; j < VEC; j++) y[j] = h[v][j] * inv * w[j];
                    store_vec<T, TAIL>((T*)p.y + row * p.cols, i, p.cols, io<T>::pack(y));
                }
            }
        } else {
            float w[NV][VEC];
            unsigned top = 0;
#pragma unroll
            for (int v = 0; v < NV; v++) {
                const int i = (v * TEAM + t) * VEC;
#pragma unroll
                for (int j = 0; j < VEC; j++) w[v][j] = 0.f;
                if (i < p.cols) load_weight<T, TAIL>(p.weight, p.weight_f32, i, p.cols, w[v]);
#pragma unroll
                for (int j = 0; j < VEC; j++) top = max(top, abs_bits(h[v][j] * w[v][j]));
            }
            top = team_reduce<TEAM>(top, red, turn, max_op());
            double amax = (double)__builtin_bit_cast(float, top);
            // (also rows whose products leave fp32's range or come near its end: among them the rows of zeros)
            const bool wide = p.wide || !(amax > 1e-30 && amax < 1e37);
            if (wide) {
                unsigned long long top64 = 0;
#pragma unroll
                for (int v = 0; v < NV; v++)
#pragma unroll
                    for (int j = 0; j < VEC; j++) top64 = max(top64, abs_bits((double)h[v][j] * w[v][j]));
                top64 = team_reduce<TEAM>(top64, red, turn, max_op());
                amax = __builtin_bit_cast(double, top64);
            }
            const bool fine = amax > 0.0 && amax < __builtin_inf();
            if (t == 0) p.q_scale[row] = fine || amax == 0.0 ? (float)(amax * inv / 127.0) : __builtin_nanf("");
            const double k64 = fine ? 127.0 / amax : 0.0;
            const float k = (float)k64;
#pragma unroll
            for (int v = 0; v < NV; v++) {
                const int i = (v * TEAM + t) * VEC;
                if (i < p.q_cols) {
                    float s[VEC];
                    unsigned word[VEC / 4];
#pragma unroll
                    for (int j = 0; j < VEC; j++) s[j] = wide ? (float)((double)h[v][j] * w[v][j] * k64) : h[v][j] * w[v][j] * k;
                    if (fine) quantise<VEC>(s, [&](int j) { return (double)h[v][j] * w[v][j]; }, amax, word);
                    else {
#pragma unroll
                        for (int e = 0; e < VEC / 4; e++) word[e] = 0u;
                    }
                    int8_t* q = p.q + row * p.q_stride + i;
                    if constexpr (VEC == 8) *(u32x2*)q = u32x2{word[0], word[1]};
                    else *(unsigned*)q = word[0];
                }
            }
        }
    }
}

// A row longer than the registers of a workgroup: 1024 threads walk it once per step.  With a residual, the later walks read the h that the same thread wrote.
template <typename T, int OUT>
__global__ __launch_bounds__(1024) void rms_norm_long_kernel(const args p) {
    constexpr int VEC = io<T>::VEC, TEAM = 1024;
    __shared__ red_slots red;
    int turn = 0;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = (const T*)p.x + row * p.x_stride;
        const T* r = p.residual ? (const T*)p.residual + row * p.residual_stride : nullptr;
        T* hout = r ? (T*)p.h + row * p.cols : nullptr;
        const T* again = r ? (const T*)hout : x;
        float ss = 0.f;
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
            for (int j = 0; j < VEC; j++) ss = __builtin_fmaf(h[j], h[j], ss);
        }
        float inv = 1.f;
        if (p.normalize) {
            ss = team_reduce<TEAM>(ss, red, turn, add_op());
            inv = 1.0f / __builtin_sqrtf(ss / (float)p.cols + p.eps);
            if (!sum_in_range(ss, p.eps)) {
                double s2 = 0.0;
                for (int i = threadIdx.x * VEC; i < p.cols; i += TEAM * VEC) {
                    float h[VEC];
                    io<T>::unpack(load_vec<T, true>(again, i, p.cols), h);
#pragma unroll
                    for (int j = 0; j < VEC; j++) s2 += (double)h[j] * h[j];
                }
                s2 = team_reduce<TEAM>(s2, red, turn, add_op());
                inv = (float)(1.0 / __builtin_sqrt(s2 / p.cols + p.eps));
            }
            if (p.inv_rms && threadIdx.x == 0) p.inv_rms[row] = inv;
        }
        if constexpr (OUT == 0) {
            for (int i = threadIdx.x * VEC; i < p.cols; i += TEAM * VEC) {
                float h[VEC], w[VEC];
                io<T>::unpack(load_vec<T, true>(again, i, p.cols), h);
                load_weight<T, true>(p.weight, p.weight_f32, i, p.cols, w);
#pragma unroll
                for (int j = 0; j < VEC; j++) h[j] = h[j] * inv * w[j];
                store_vec<T, true>((T*)p.y + row * p.cols, i, p.cols, io<T>::pack(h));
            }
        } else {
            unsigned long long top = 0;
            for (int i = threadIdx.x * VEC; i < p.cols; i += TEAM * VEC) {
                float h[VEC], w[VEC];
                io<T>::unpack(load_vec<T, true>(again, i, p.cols), h);
                load_weight<T, true>(p.weight, p.weight_f32, i, p.cols, w);
#pragma unroll
                for (int j = 0; j < VEC; j++) if (i + j < p.cols) top = max(top, abs_bits((double)h[j] * w[j]));
            }
            const double amax = __builtin_bit_cast(double, team_reduce<TEAM>(top, red, turn, max_op()));
            const bool fine = amax > 0.0 && amax < __builtin_inf();
            if (threadIdx.x == 0) p.q_scale[row] = fine || amax == 0.0 ? (float)(amax * inv / 127.0) : __builtin_nanf("");
            const double k64 = fine ? 127.0 / amax : 0.0;
            for (int i = threadIdx.x * VEC; i < p.q_cols; i += TEAM * VEC) {
                float h[VEC], w[VEC], s[VEC];
                unsigned word[VEC / 4];
#pragma unroll
                for (int j = 0; j < VEC; j++) h[j] = w[j] = 0.f;
                if (i < p.cols) {
                    io<T>::unpack(load_vec<T, true>(again, i, p.cols), h);
                    load_weight<T, true>(p.weight, p.weight_f32, i, p.cols, w);
                }
#pragma unroll
                for (int j = 0; j < VEC; j++) s[j] = (float)((double)h[j] * w[j] * k64);
                if (fine) quantise<VEC>(s, [&](int j) { return (double)h[j] * w[j]; }, amax, word);
                else {
#pragma unroll
                    for (int e = 0; e < VEC / 4; e++) word[e] = 0u;
                }
                int8_t* q = p.q + row * p.q_stride + i;
                if constexpr (VEC == 8) *(u32x2*)q = u32x2{word[0], word[1]};
                else *(unsigned*)q = word[0];
            }
        }
    }
}

struct bwd_args {
    const void* dy; const void* h; const void* dh; const void* weight; const float* inv_rms;
    void* dx; float* partials;       // partials [gridDim.x, cols]: sums of dy * xh over the rows of a workgroup (NULL: no weight gradient)
    int64_t rows, dy_stride, h_stride, dh_stride;
    int cols, weight_f32;
};

template <typename T, int TEAM, int NV, bool TAIL>
__global__ __launch_bounds__(256) void rms_norm_backward_kernel(const bwd_args p) {
    constexpr int VEC = io<T>::VEC, RPB = 256 / TEAM;
    __shared__ red_slots red;
    __shared__ float part[TEAM == 64 ? 3 * 64 * NV * VEC : 1];
    int turn = 0;
    const int t = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    float dw[NV][VEC];
#pragma unroll
    for (int v = 0; v < NV; v++)
#pragma unroll
        for (int j = 0; j < VEC; j++) dw[v][j] = 0.f;
    for (int64_t row = (int64_t)blockIdx.x * RPB + team; row < p.rows; row += (int64_t)gridDim.x * RPB) {
        const T* dy = (const T*)p.dy + row * p.dy_stride;
        const T* h = (const T*)p.h + row * p.h_stride;
        const T* dh = p.dh ? (const T*)p.dh + row * p.dh_stride : nullptr;
        const float inv = p.inv_rms[row];
        u32x4 gv[NV], hv[NV], ev[NV];
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const int i = (v * TEAM + t) * VEC;
            gv[v] = hv[v] = ev[v] = u32x4{0u, 0u, 0u, 0u};
            if (i < p.cols) {
                gv[v] = load_vec<T, TAIL>(dy, i, p.cols);
                hv[v] = load_vec<T, TAIL>(h, i, p.cols);
                if (dh) ev[v] = load_vec<T, TAIL>(dh, i, p.cols);
            }
        }
        float g[NV][VEC], xh[NV][VEC], c = 0.f;
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const int i = (v * TEAM + t) * VEC;
            float w[VEC];
#pragma unroll
            for (int j = 0; j < VEC; j++) w[j] = 0.f;
            if (i < p.cols) load_weight<T, TAIL>(p.weight, p.weight_f32, i, p.cols, w);
            io<T>::unpack(gv[v], g[v]);
            io<T>::unpack(hv[v], xh[v]);
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                xh[v][j] *= inv;
                dw[v][j] = __builtin_fmaf(g[v][j], xh[v][j], dw[v][j]);
                g[v][j] *= w[j];
                c = __builtin_fmaf(g[v][j], xh[v][j], c);
            }
        }
        c = team_reduce<TEAM>(c, red, turn, add_op()) / (float)p.cols;
        if (p.dx) {
#pragma unroll
            for (int v = 0; v < NV; v++) {
                const int i = (v * TEAM + t) * VEC;
                if (i < p.cols) {
                    float e[VEC], d[VEC];
                    io<T>::unpack(ev[v], e);
#pragma unroll
                    for (int j = 0; j < VEC; j++) d[j] = __builtin_fmaf(inv, __builtin_fmaf(-xh[v][j], c, g[v][j]), e[j]);
                    store_vec<T, TAIL>((T*)p.dx + row * p.cols, i, p.cols, io<T>::pack(d));
                }
            }
        }
    }
    if (!p.partials) return;
    if constexpr (TEAM == 64) {       // the four waves' sums, in the order of the waves
        if (team > 0) {
#pragma unroll
            for (int v = 0; v < NV; v++)
#pragma unroll
                for (int j = 0; j < VEC; j++) part[((team - 1) * NV + v) * 64 * VEC + j * 64 + t] = dw[v][j];
        }
        __syncthreads();
        if (team > 0) return;
#pragma unroll
        for (int w = 0; w < 3; w++)
#pragma unroll
            for (int v = 0; v < NV; v++)
#pragma unroll
                for (int j = 0; j < VEC; j++) dw[v][j] += part[(w * NV + v) * 64 * VEC + j * 64 + t];
    }
    float* out = p.partials + (int64_t)blockIdx.x * p.cols;
#pragma unroll
    for (int v = 0; v < NV; v++) {
        const int i = (v * TEAM + t) * VEC;
#pragma unroll
        for (int j = 0; j < VEC; j++) if (i + j < p.cols) out[i + j] = dw[v][j];
    }
}

// rows beyond the registers: two walks; a workgroup's weight-gradient sums live in its own row of `partials`
template <typename T>
__global__ __launch_bounds__(1024) void rms_norm_backward_long_kernel(const bwd_args p) {
    constexpr int VEC = io<T>::VEC, TEAM = 1024;
    __shared__ red_slots red;
    int turn = 0;
    float* out = p.partials ? p.partials + (int64_t)blockIdx.x * p.cols : nullptr;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* dy = (const T*)p.dy + row * p.dy_stride;
        const T* h = (const T*)p.h + row * p.h_stride;
        const T* dh = p.dh ? (const T*)p.dh + row * p.dh_stride : nullptr;
        const float inv = p.inv_rms[row];
        const bool first = row == (int64_t)blockIdx.x;
        float c = 0.f;
        for (int i = threadIdx.x * VEC; i < p.cols; i += TEAM * VEC) {
            float g[VEC], xh[VEC], w[VEC];
            io<T>::unpack(load_vec<T, true>(dy, i, p.cols), g);
            io<T>::unpack(load_vec<T, true>(h, i, p.cols), xh);
            load_weight<T, true>(p.weight, p.weight_f32, i, p.cols, w);
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                xh[j] *= inv;
                if (out && i + j < p.cols) out[i + j] = first ? g[j] * xh[j] : __builtin_fmaf(g[j], xh[j], out[i + j]);
                c = __builtin_fmaf(g[j] * w[j], xh[j], c);
            }
        }
        c = team_reduce<TEAM>(c, red, turn, add_op()) / (float)p.cols;
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

// dw[k] = sum of the workgroups' partial rows, 64 columns per workgroup of 16 waves; the order is fixed, so the result is too
template <typename W>
__global__ __launch_bounds__(1024) void rms_norm_weight_grad_kernel(const float* partials, int count, int cols, W* dw) {
    __shared__ float part[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = blockIdx.x * 64 + lane;
    float s = 0.f;
    if (col < cols)
        for (int g = wave; g < count; g += 16) s += partials[(int64_t)g * cols + col];
    part[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && col < cols) {
#pragma unroll
        for (int w = 1; w < 16; w++) s += part[w][lane];
        sgv_traits<W>::store(dw + col, s);
    }
}

template <typename T>
__global__ __launch_bounds__(256) void dequantize_rows_kernel(const int8_t* q, int64_t q_stride, const float* scale, T* out, int64_t rows, int cols) {
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const float s = scale[row];
        for (int i = threadIdx.x; i < cols; i += 256) sgv_traits<T>::store(out + row * cols + i, (float)q[row * q_stride + i] * s);
    }
}

// How a row of `cols` elements is held: vectors per lane of a wave (<= 4), or of a 256-thread workgroup (<= 8), or not at all.
struct shape { int team, nv; };
static inline shape row_shape(int cols, int vec) {
    const int vectors = (((cols + 15) / 16 * 16) + vec - 1) / vec;       // (the 8-bit rows are written to a multiple of 16)
    for (int nv = 1; nv <= 4; nv *= 2) if (vectors <= 64 * nv) return shape{64, nv};
    for (int nv = 2; nv <= 8; nv *= 2) if (vectors <= 256 * nv) return shape{256, nv};
    return shape{1024, 0};
}

// workgroups of a backward launch = rows of its partial sums: two per CU keep the memory busy, and the partial sums stay small beside the rows
static inline int backward_blocks(int64_t rows, int cols, int vec) {
    const shape s = row_shape(cols, vec);
    const int64_t teams = s.team == 64 ? (rows + 3) / 4 : rows;
    return (int)std::min<int64_t>(teams, 512);
}

template <typename T, int OUT, bool TAIL>
static void launch_forward(const args& p, hipStream_t stream) {
    const shape s = row_shape(p.cols, io<T>::VEC);
    const int64_t teams = s.team == 64 ? (p.rows + 3) / 4 : p.rows;
    const dim3 grid((unsigned)std::min<int64_t>(teams, 1 << 20));
#define SGV_RN_GO(TEAM, NV) hipLaunchKernelGGL((rms_norm_kernel<T, OUT, TEAM, NV, TAIL>), grid, dim3(256), 0, stream, p)
    if (s.team == 64) { if (s.nv == 1) SGV_RN_GO(64, 1); else if (s.nv == 2) SGV_RN_GO(64, 2); else SGV_RN_GO(64, 4); }
    else if (s.team == 256) { if (s.nv == 2) SGV_RN_GO(256, 2); else if (s.nv == 4) SGV_RN_GO(256, 4); else SGV_RN_GO(256, 8); }
    else hipLaunchKernelGGL((rms_norm_long_kernel<T, OUT>), grid, dim3(1024), 0, stream, p);
#undef SGV_RN_GO
}

template <typename T>
static void launch_forward(const args& p, hipStream_t stream) {
    const bool tail = p.cols % io<T>::VEC != 0;
    if (p.q) { if (tail) launch_forward<T, 1, true>(p, stream); else launch_forward<T, 1, false>(p, stream); }
    else { if (tail) launch_forward<T, 0, true>(p, stream); else launch_forward<T, 0, false>(p, stream); }
}

template <typename T, bool TAIL>
static void launch_backward(const bwd_args& p, int blocks, hipStream_t stream) {
    const shape s = row_shape(p.cols, io<T>::VEC);
    const dim3 grid((unsigned)blocks);
#define SGV_RN_GO(TEAM, NV) hipLaunchKernelGGL((rms_norm_backward_kernel<T, TEAM, NV, TAIL>), grid, dim3(256), 0, stream, p)
    if (s.team == 64) { if (s.nv == 1) SGV_RN_GO(64, 1); else if (s.nv == 2) SGV_RN_GO(64, 2); else SGV_RN_GO(64, 4); }
    else if (s.team == 256) { if (s.nv == 2) SGV_RN_GO(256, 2); else if (s.nv == 4) SGV_RN_GO(256, 4); else SGV_RN_GO(256, 8); }
    else hipLaunchKernelGGL((rms_norm_backward_long_kernel<T>), grid, dim3(1024), 0, stream, p);
#undef SGV_RN_GO
}

}  // namespace sgv_rn

static inline bool sgv_row_dtype(int dtype) { return dtype == SGV_F32 || dtype == SGV_F16 || dtype == SGV_BF16; }

extern "C" int sgv_rms_norm(const sgv_rms_norm_params* q, int dtype, void* stream_) {
    if (!q) return sgv_fail(SGV_ERR_INVALID_ARG, "rms_norm: params is NULL");
    if (!sgv_row_dtype(dtype)) return sgv_fail(SGV_ERR_UNSUPPORTED, "rms_norm: rows are fp32, fp16 or bf16");
    if (q->rows < 0 || q->cols < 1) return sgv_fail(SGV_ERR_INVALID_ARG, "rms_norm: rows must be >= 0 and cols >= 1");
    if (q->cols > 0x7fffffff - 16384) return sgv_fail(SGV_ERR_TOO_LARGE, "rms_norm: rows are too long");
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
    p.wide = q->weight != nullptr && (dtype == SGV_F32 || q->weight_f32);
    hipStream_t stream = (hipStream_t)stream_;
    const double es = (double)sgv_dtype_size(dtype), n = (double)q->rows * q->cols;
    sgv_launch_scope scope(SGV_K_RMS_NORM, stream, n * (es * (q->residual ? 3 : 1) + (q->q ? 1.0 : es)));
    if (dtype == SGV_F32) sgv_rn::launch_forward<float>(p, stream);
    else if (dtype == SGV_F16) sgv_rn::launch_forward<sgv_half_t>(p, stream);
    else sgv_rn::launch_forward<sgv_bf16_t>(p, stream);
    return sgv_check_launch("rms_norm_kernel");
}

extern "C" int64_t sgv_rms_norm_backward_workspace_bytes(int64_t rows, int32_t cols, int dtype) {
    if (rows < 1 || cols < 1 || !sgv_row_dtype(dtype)) return 0;
    return (int64_t)sgv_rn::backward_blocks(rows, cols, dtype == SGV_F32 ? 4 : 8) * cols * 4;
}

extern "C" int sgv_rms_norm_backward(const sgv_rms_norm_backward_params* q, int dtype, void* stream_) {
    if (!q) return sgv_fail(SGV_ERR_INVALID_ARG, "rms_norm_backward: params is NULL");
    if (!sgv_row_dtype(dtype)) return sgv_fail(SGV_ERR_UNSUPPORTED, "rms_norm_backward: rows are fp32, fp16 or bf16");
    if (q->rows < 1 || q->cols < 1) return sgv_fail(SGV_ERR_INVALID_ARG, "rms_norm_backward: rows and cols must be >= 1");
    if (q->cols > 0x7fffffff - 16384) return sgv_fail(SGV_ERR_TOO_LARGE, "rms_norm_backward: rows are too long");
    if (!q->dy || !q->h || !q->inv_rms || (!q->dx && !q->dweight)) return sgv_fail(SGV_ERR_INVALID_ARG, "rms_norm_backward: NULL pointer");
    if (q->dweight && !q->weight) return sgv_fail(SGV_ERR_INVALID_ARG, "rms_norm_backward: a gradient of no weight");
    if (q->dy_stride < 0 || q->h_stride < 0 || q->dh_stride < 0) return sgv_fail(SGV_ERR_INVALID_ARG, "rms_norm_backward: negative strides");
    const int vec = dtype == SGV_F32 ? 4 : 8;
    const int blocks = sgv_rn::backward_blocks(q->rows, q->cols, vec);
    if (q->dweight && (!q->workspace || q->workspace_bytes < (int64_t)blocks * q->cols * 4))
        return sgv_fail(SGV_ERR_INVALID_ARG, "rms_norm_backward: the weight gradient needs sgv_rms_norm_backward_workspace_bytes() of workspace");
    sgv_rn::bwd_args p{};
    p.dy = q->dy; p.h = q->h; p.dh = q->dh; p.weight = q->weight; p.inv_rms = q->inv_rms; p.dx = q->dx; p.partials = q->dweight ? (float*)q->workspace : nullptr;
    p.rows = q->rows; p.dy_stride = q->dy_stride; p.h_stride = q->h_stride; p.dh_stride = q->dh_stride; p.cols = q->cols; p.weight_f32 = q->weight_f32;
    hipStream_t stream = (hipStream_t)stream_;
    const double es = (double)sgv_dtype_size(dtype), n = (double)q->rows * q->cols;
    sgv_launch_scope scope(SGV_K_RMS_NORM, stream, n * es * (q->dh ? 4 : 3));
    const bool tail = q->cols % vec != 0;
    if (dtype == SGV_F32) { if (tail) sgv_rn::launch_backward<float, true>(p, blocks, stream); else sgv_rn::launch_backward<float, false>(p, blocks, stream); }
    else if (dtype == SGV_F16) { if (tail) sgv_rn::launch_backward<sgv_half_t, true>(p, blocks, stream); else sgv_rn::launch_backward<sgv_half_t, false>(p, blocks, stream); }
    else { if (tail) sgv_rn::launch_backward<sgv_bf16_t, true>(p, blocks, stream); else sgv_rn::launch_backward<sgv_bf16_t, false>(p, blocks, stream); }
    int rc = sgv_check_launch("rms_norm_backward_kernel");
    if (rc != SGV_OK || !q->dweight) return rc;
    const dim3 grid((unsigned)((q->cols + 63) / 64));
    const float* part = (const float*)q->workspace;
    if (dtype == SGV_F32 || q->weight_f32) hipLaunchKernelGGL((sgv_rn::rms_norm_weight_grad_kernel<float>), grid, dim3(1024), 0, stream, part, blocks, q->cols, (float*)q->dweight);
    else if (dtype == SGV_F16) hipLaunchKernelGGL((sgv_rn::rms_norm_weight_grad_kernel<sgv_half_t>), grid, dim3(1024), 0, stream, part, blocks, q->cols, (sgv_half_t*)q->dweight);
    else hipLaunchKernelGGL((sgv_rn::rms_norm_weight_grad_kernel<sgv_bf16_t>), grid, dim3(1024), 0, stream, part, blocks, q->cols, (sgv_bf16_t*)q->dweight);
    return sgv_check_launch("rms_norm_weight_grad_kernel");
}

extern "C" int sgv_dequantize_rows(const void* q, int64_t q_stride, const float* scale, void* out, int64_t rows, int32_t cols, int dtype, void* stream_) {
    if (!sgv_row_dtype(dtype)) return sgv_fail(SGV_ERR_UNSUPPORTED, "dequantize_rows: the output is fp32, fp16 or bf16");
    if (rows < 0 || cols < 1 || q_stride < 0) return sgv_fail(SGV_ERR_INVALID_ARG, "dequantize_rows: rows must be >= 0 and cols >= 1");
    if (cols > 0x7fffffff - 16384) return sgv_fail(SGV_ERR_TOO_LARGE, "dequantize_rows: rows are too long");
    if (rows == 0) return SGV_OK;
    if (!q || !scale || !out) return sgv_fail(SGV_ERR_INVALID_ARG, "dequantize_rows: NULL pointer");
    hipStream_t stream = (hipStream_t)stream_;
    sgv_launch_scope scope(SGV_K_RMS_NORM, stream, (double)rows * cols * (1.0 + sgv_dtype_size(dtype)));
    const dim3 grid((unsigned)std::min<int64_t>(rows, 1 << 20));
    const int8_t* in = (const int8_t*)q;
    if (dtype == SGV_F32) hipLaunchKernelGGL((sgv_rn::dequantize_rows_kernel<float>), grid, dim3(256), 0, stream, in, q_stride, scale, (float*)out, rows, cols);
    else if (dtype == SGV_F16) hipLaunchKernelGGL((sgv_rn::dequantize_rows_kernel<sgv_half_t>), grid, dim3(256), 0, stream, in, q_stride, scale, (sgv_half_t*)out, rows, cols);
    else hipLaunchKernelGGL((sgv_rn::dequantize_rows_kernel<sgv_bf16_t>), grid, dim3(256), 0, stream, in, q_stride, scale, (sgv_bf16_t*)out, rows, cols);
    return sgv_check_launch("dequantize_rows_kernel");
}
