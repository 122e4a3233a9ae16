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
struct any_bytes16 { u32x4 v; } __attribute__((packed, aligned(1)));
struct any_f32x4 { f32x4 v; } __attribute__((packed, aligned(4)));
struct any_u32x2 { u32x2 v; } __attribute__((packed, aligned(1)));
struct any_u32 { unsigned v; } __attribute__((packed, aligned(1)));

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

// The 8-bit values of VEC columns, four to a word.  v(j): the value in steps of the row, good to 2.3e-5 (|v| <= 127: three fp32 roundings); u64(j): the exact u.
// Adding 1.5 * 2^23 leaves the nearest whole number in the low bits.
template <int VEC, typename V, typename U>
__device__ __forceinline__ void quantise(V v, U u64, double amax, unsigned* word) {
    constexpr float MAGIC = 12582912.f;
    float x[VEC], far = 0.f;
#pragma unroll
    for (int j = 0; j < VEC; j++) {
        const float s = v(j);
        x[j] = s + MAGIC;
        far = __builtin_fmaxf(far, __builtin_fabsf(s - (x[j] - MAGIC)));
    }
    if (far > 0.49997f) {
#pragma unroll
        for (int j = 0; j < VEC; j++) x[j] = (float)__builtin_rint(u64(j) * 127.0 / amax) + MAGIC;
    }
#pragma unroll
    for (int w = 0; w < VEC / 4; w++) {
        const unsigned lo = __builtin_amdgcn_perm(__float_as_uint(x[4 * w + 1]), __float_as_uint(x[4 * w]), 0x0c0c0400u);
        const unsigned hi = __builtin_amdgcn_perm(__float_as_uint(x[4 * w + 3]), __float_as_uint(x[4 * w + 2]), 0x04000c0cu);
        word[w] = lo | hi;
    }
}
template <int VEC>
__device__ __forceinline__ void store_bytes(int8_t* q, const unsigned* word) {
    if constexpr (VEC == 8) ((any_u32x2*)q)->v = u32x2{word[0], word[1]};
    else ((any_u32*)q)->v = word[0];
}

// The vector v of thread t of a row: its first column, and how many of its columns the vector in front of it has too.  A row whose length is no multiple of VEC ends with
// a vector that is moved back to lie inside the row: both write the same values to the columns they share, and the sums leave them out once.
template <int TEAM, int VEC, bool TAIL>
__device__ __forceinline__ int vec_column(int v, int t, int cols, int& shared) {
    int i = (v * TEAM + t) * VEC;
    shared = 0;
    if (TAIL && i < cols && i + VEC > cols) { shared = i + VEC - cols; i = cols - VEC; }
    return i;
}

// OUT 0: y; 1: q and its scale, no weight; 2: q and its scale, with a weight.  TEAM threads (64: a wave, four rows per workgroup; else the workgroup) hold a row as NV vectors each.
template <typename T, int OUT, int TEAM, int NV, bool TAIL>
__global__ __launch_bounds__(TEAM == 64 ? 256 : TEAM) void rms_norm_kernel(const args p) {
    constexpr int VEC = io<T>::VEC, RPB = TEAM == 64 ? 4 : 1;
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
            int shared;
            const int i = vec_column<TEAM, VEC, TAIL>(v, t, p.cols, shared);
            xv[v] = u32x4{0u, 0u, 0u, 0u};
            rv[v] = u32x4{0u, 0u, 0u, 0u};
            if (i < p.cols) {
                xv[v] = load_vec<T, false>(x, i, p.cols);
                if (r) rv[v] = load_vec<T, false>(r, i, p.cols);
            }
        }
        float ss = 0.f;
#pragma unroll
        for (int v = 0; v < NV; v++) {
            int shared;
            const int i = vec_column<TEAM, VEC, TAIL>(v, t, p.cols, shared);
            io<T>::unpack(xv[v], h[v]);
            if (r) {
                float rf[VEC];
                io<T>::unpack(rv[v], rf);
#pragma unroll
                for (int j = 0; j < VEC; j++) h[v][j] += rf[j];
                const u32x4 hv = io<T>::pack(h[v]);
                io<T>::unpack(hv, h[v]);
                if (i < p.cols) store_vec<T, false>((T*)p.h + row * p.cols, i, p.cols, hv);
            }
            float part = ss;
#pragma unroll
            for (int j = 0; j < VEC; j++) part = __builtin_fmaf(h[v][j], h[v][j], part);
            if (TAIL && shared > 0) {
                part = ss;
#pragma unroll
                for (int j = 0; j < VEC; j++) part = j >= shared ? __builtin_fmaf(h[v][j], h[v][j], part) : part;
            }
            ss = part;
        }
        ss = team_reduce<TEAM>(ss, red, turn, add_op());
        float inv = 1.f;
        if (p.normalize) {
            inv = 1.0f / __builtin_sqrtf(ss / (float)p.cols + p.eps);
            if (!sum_in_range(ss, p.eps)) {
                double s2 = 0.0;
#pragma unroll
                for (int v = 0; v < NV; v++) {
                    int shared;
                    vec_column<TEAM, VEC, TAIL>(v, t, p.cols, shared);
#pragma unroll
                    for (int j = 0; j < VEC; j++) s2 += !TAIL || j >= shared ? (double)h[v][j] * h[v][j] : 0.0;
                }
                s2 = team_reduce<TEAM>(s2, red, turn, add_op());
                inv = (float)(1.0 / __builtin_sqrt(s2 / p.cols + p.eps));
            }
            if (p.inv_rms && t == 0) p.inv_rms[row] = inv;
        }
        if constexpr (OUT == 0) {
#pragma unroll
            for (int v = 0; v < NV; v++) {
                int shared;
                const int i = vec_column<TEAM, VEC, TAIL>(v, t, p.cols, shared);
                if (i < p.cols) {
                    float w[VEC], y[VEC];
                    load_weight<T, false>(p.weight, p.weight_f32, i, p.cols, w);
#pragma unroll
                    for (int j = 0; j < VEC; j++) y[j] = h[v][j] * inv * w[j];
                    store_vec<T, false>((T*)p.y + row * p.cols, i, p.cols, io<T>::pack(y));
                }
            }
        } else {
            double amax;
            bool wide = false;
            u32x4 wv[OUT == 2 ? NV : 1][2];          // the weight as it is kept: unpacked again below, where registers are free
            auto weight = [&](int v, float* w) {
                if (p.weight_f32 && VEC == 8) { io<float>::unpack(wv[v][0], w); io<float>::unpack(wv[v][1], w + 4); }
                else io<T>::unpack(wv[v][0], w);
            };
            if constexpr (OUT == 1) {
                // the largest magnitude of h; a NaN does not show in it, but in the sum of squares
                float top = 0.f;
#pragma unroll
                for (int v = 0; v < NV; v++)
#pragma unroll
                    for (int j = 0; j < VEC; j++) top = __builtin_fmaxf(top, __builtin_fabsf(h[v][j]));
                top = team_reduce<TEAM>(top, red, turn, max_op());
                amax = ss != ss ? (double)ss : (double)top;
            } else {
                unsigned top = 0;
#pragma unroll
                for (int v = 0; v < NV; v++) {
                    int shared;
                    const int i = vec_column<TEAM, VEC, TAIL>(v, t, p.cols, shared);
                    wv[v][0] = wv[v][1] = u32x4{0u, 0u, 0u, 0u};
                    if (i < p.cols) {
                        if (p.weight_f32 && VEC == 8) { wv[v][0] = load_vec<float, false>((const float*)p.weight, i, p.cols); wv[v][1] = load_vec<float, false>((const float*)p.weight, i + 4, p.cols); }
                        else wv[v][0] = load_vec<T, false>((const T*)p.weight, i, p.cols);
                    }
                    float w[VEC];
                    weight(v, w);
#pragma unroll
                    for (int j = 0; j < VEC; j++) top = max(top, abs_bits(h[v][j] * w[j]));
                }
                top = team_reduce<TEAM>(top, red, turn, max_op());
                amax = (double)__uint_as_float(top);
                // (also rows whose products leave fp32's range or come near its end: among them the rows of zeros)
                wide = p.wide || !(amax > 1e-30 && amax < 1e37);
                if (wide) {
                    unsigned long long top64 = 0;
#pragma unroll
                    for (int v = 0; v < NV; v++) {
                        float w[VEC];
                        weight(v, w);
#pragma unroll
                        for (int j = 0; j < VEC; j++) top64 = max(top64, abs_bits((double)h[v][j] * w[j]));
                    }
                    amax = __builtin_bit_cast(double, team_reduce<TEAM>(top64, red, turn, max_op()));
                }
            }
            const bool fine = amax > 0.0 && amax < __builtin_inf();
            if (t == 0) p.q_scale[row] = fine || amax == 0.0 ? (float)(amax * inv / 127.0) : __builtin_nanf("");
            const double k64 = fine ? 127.0 / amax : 0.0;
            // (tiny rows: 127 / max may not be an fp32 number; 2^100 times the value and 2^-100 times the factor are)
            const float up = OUT == 1 && amax < 1e-30 ? 0x1p100f : 1.f, k = (float)(k64 / up);
            int8_t* q = p.q + row * p.q_stride;
#pragma unroll
            for (int v = 0; v < NV; v++) {
                int shared;
                const int i = vec_column<TEAM, VEC, TAIL>(v, t, p.cols, shared);
                if (i < p.cols) {
                    unsigned word[VEC / 4];
                    if constexpr (OUT == 1) {
                        if (fine) quantise<VEC>([&](int j) { return h[v][j] * up * k; }, [&](int j) { return (double)h[v][j]; }, amax, word);
                    } else {
                        float w[VEC];
                        weight(v, w);
                        if (fine && wide) quantise<VEC>([&](int j) { return (float)((double)h[v][j] * w[j] * k64); }, [&](int j) { return (double)h[v][j] * w[j]; }, amax, word);
                        else if (fine) quantise<VEC>([&](int j) { return h[v][j] * w[j] * k; }, [&](int j) { return (double)h[v][j] * w[j]; }, amax, word);
                    }
                    if (!fine) {
#pragma unroll
                        for (int e = 0; e < VEC / 4; e++) word[e] = 0u;
                    }
                    store_bytes<VEC>(q + i, word);
                }
            }
            if (t < p.q_cols - p.cols) q[p.cols + t] = 0;
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
                float h[VEC], w[VEC];
                unsigned word[VEC / 4];
#pragma unroll
                for (int j = 0; j < VEC; j++) h[j] = w[j] = 0.f;
                if (i < p.cols) {
                    io<T>::unpack(load_vec<T, true>(again, i, p.cols), h);
                    load_weight<T, true>(p.weight, p.weight_f32, i, p.cols, w);
                }
                if (fine) quantise<VEC>([&](int j) { return i + j < p.cols ? (float)((double)h[j] * w[j] * k64) : 0.f; }, [&](int j) { return i + j < p.cols ? (double)h[j] * w[j] : 0.0; }, amax, word);
                else {
#pragma unroll
                    for (int e = 0; e < VEC / 4; e++) word[e] = 0u;
                }
                store_bytes<VEC>(p.q + row * p.q_stride + i, word);
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

template <typename T, bool DW, int TEAM, int NV, bool TAIL>
__global__ __launch_bounds__(TEAM == 64 ? 256 : TEAM) void rms_norm_backward_kernel(const bwd_args p) {
    constexpr int VEC = io<T>::VEC, RPB = TEAM == 64 ? 4 : 1;
    __shared__ red_slots red;
    __shared__ float part[DW && TEAM == 64 ? 3 * 64 * NV * VEC : 1];
    int turn = 0;
    const int t = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    float dw[DW ? NV : 1][VEC];
    if constexpr (DW) {
#pragma unroll
        for (int v = 0; v < NV; v++)
#pragma unroll
            for (int j = 0; j < VEC; j++) dw[v][j] = 0.f;
    }
    for (int64_t row = (int64_t)blockIdx.x * RPB + team; row < p.rows; row += (int64_t)gridDim.x * RPB) {
        const T* dy = (const T*)p.dy + row * p.dy_stride;
        const T* h = (const T*)p.h + row * p.h_stride;
        const T* dh = p.dh ? (const T*)p.dh + row * p.dh_stride : nullptr;
        u32x4 gv[NV], hv[NV], ev[NV];
#pragma unroll
        for (int v = 0; v < NV; v++) {
            int shared;
            const int i = vec_column<TEAM, VEC, TAIL>(v, t, p.cols, shared);
            gv[v] = hv[v] = ev[v] = u32x4{0u, 0u, 0u, 0u};
            if (i < p.cols) {
                gv[v] = load_vec<T, false>(dy, i, p.cols);
                hv[v] = load_vec<T, false>(h, i, p.cols);
                if (dh) ev[v] = load_vec<T, false>(dh, i, p.cols);
            }
        }
        const float inv = p.inv_rms[row];
        float c = 0.f;
        // g = dy * w and xh = h * inv of vector v: made twice, in front of the sum and behind it, where holding them would cost the registers of two more rows in flight
        auto terms = [&](int v, float* g, float* xh) {
            int shared;
            const int i = vec_column<TEAM, VEC, TAIL>(v, t, p.cols, shared);
            io<T>::unpack(gv[v], g);
            io<T>::unpack(hv[v], xh);
#pragma unroll
            for (int j = 0; j < VEC; j++) xh[j] *= inv;
            if (p.weight && i < p.cols) {
                float w[VEC];
                load_weight<T, false>(p.weight, p.weight_f32, i, p.cols, w);
#pragma unroll
                for (int j = 0; j < VEC; j++) g[j] *= w[j];
            }
            return shared;
        };
#pragma unroll
        for (int v = 0; v < NV; v++) {
            float g[VEC], xh[VEC];
            const int shared = terms(v, g, xh);
            if constexpr (DW) {
                float d[VEC];
                io<T>::unpack(gv[v], d);
#pragma unroll
                for (int j = 0; j < VEC; j++) dw[v][j] = __builtin_fmaf(d[j], xh[j], dw[v][j]);
            }
            float sum = c;
#pragma unroll
            for (int j = 0; j < VEC; j++) sum = __builtin_fmaf(g[j], xh[j], sum);
            if (TAIL && shared > 0) {
                sum = c;
#pragma unroll
                for (int j = 0; j < VEC; j++) sum = j >= shared ? __builtin_fmaf(g[j], xh[j], sum) : sum;
            }
            c = sum;
        }
        c = team_reduce<TEAM>(c, red, turn, add_op()) / (float)p.cols;
        if (p.dx) {
#pragma unroll
            for (int v = 0; v < NV; v++) {
                int shared;
                const int i = vec_column<TEAM, VEC, TAIL>(v, t, p.cols, shared);
                if (i < p.cols) {
                    float g[VEC], xh[VEC], d[VEC];
                    terms(v, g, xh);
                    io<T>::unpack(ev[v], d);
#pragma unroll
                    for (int j = 0; j < VEC; j++) d[j] = __builtin_fmaf(inv, __builtin_fmaf(-xh[j], c, g[j]), d[j]);
                    store_vec<T, false>((T*)p.dx + row * p.cols, i, p.cols, io<T>::pack(d));
                }
            }
        }
    }
    if constexpr (DW) {
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
            int shared;
            const int i = vec_column<TEAM, VEC, TAIL>(v, t, p.cols, shared);
            if (i < p.cols) {
#pragma unroll
                for (int q = 0; q < VEC / 4; q++) ((any_f32x4*)(out + i + 4 * q))->v = f32x4{dw[v][4 * q], dw[v][4 * q + 1], dw[v][4 * q + 2], dw[v][4 * q + 3]};
            }
        }
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

// dw[k] = sum of the workgroups' partial rows: 32 columns per workgroup, 32 threads to a column; the order is fixed, so the result is too
template <typename W>
__global__ __launch_bounds__(1024) void rms_norm_weight_grad_kernel(const float* partials, int count, int cols, W* dw) {
    __shared__ float part[32][33];
    const int c = threadIdx.x & 31, g = threadIdx.x >> 5, col = min((int)blockIdx.x * 32 + c, cols - 1);
    float s = 0.f;
#pragma unroll 8
    for (int r = g; r < count; r += 32) s += partials[(int64_t)r * cols + col];
    part[g][c] = s;
    __syncthreads();
    s = part[c][g];                      // (now the 32 sums of one column lie in one half of a wave)
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor(s, off, 32);
    if (c == 0 && (int)blockIdx.x * 32 + g < cols) sgv_traits<W>::store(dw + blockIdx.x * 32 + g, s);
}

// 16 columns to a thread: one load, and stores of 16 bytes
template <typename T>
__global__ __launch_bounds__(256) void dequantize_rows_kernel(const int8_t* q, int64_t q_stride, const float* scale, T* out, int64_t rows, int cols) {
    const int pieces = (cols + 15) / 16;
    for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < rows * pieces; x += (int64_t)gridDim.x * 256) {
        const int64_t row = x / pieces;
        const int i = (int)(x - row * pieces) * 16;
        const float s = scale[row];
        const int8_t* src = q + row * q_stride + i;
        T* dst = out + row * cols + i;
        if (i + 16 <= cols) {
            const u32x4 b = ((const any_bytes16*)src)->v;
            float f[16];
#pragma unroll
            for (int e = 0; e < 16; e++) f[e] = (float)(int8_t)(b[e >> 2] >> (8 * (e & 3))) * s;
#pragma unroll
            for (int e = 0; e < 16; e += io<T>::VEC) store_vec<T, false>(dst, e, cols, io<T>::pack(f + e));
        } else {
            for (int e = 0; i + e < cols; e++) sgv_traits<T>::store(dst + e, (float)src[e] * s);
        }
    }
}

// How a row is held: TEAM threads with NV vectors each, or not at all (nv = 0: rows beyond 1024 x 4 vectors, and rows shorter than a vector)
struct shape { int team, nv; };
static inline shape row_shape(int cols, int vec) {
    static const shape held[] = {{64, 1}, {64, 2}, {64, 4}, {256, 2}, {512, 2}, {512, 4}, {1024, 4}};
    if (cols >= vec)
        for (const shape& s : held) if (cols <= s.team * s.nv * vec) return s;
    return shape{1024, 0};
}

// Workgroups of a backward launch.  With a weight gradient they are the rows of its partial sums: two per CU keep the memory busy, and the partial sums stay small
// beside the rows.
static inline int backward_blocks(int64_t rows, int cols, int vec, bool dw) {
    const shape s = row_shape(cols, vec);
    const int64_t teams = s.team == 64 ? (rows + 3) / 4 : rows;
    return (int)std::min<int64_t>(teams, dw ? 512 : 1 << 20);
}

#define SGV_RN_SHAPES(GO) \
    if (s.team == 64) { if (s.nv == 1) GO(64, 1); else if (s.nv == 2) GO(64, 2); else GO(64, 4); } \
    else if (s.team == 256) GO(256, 2); \
    else if (s.team == 512) { if (s.nv == 2) GO(512, 2); else GO(512, 4); } \
    else GO(1024, 4);

template <typename T, int OUT, bool TAIL>
static void launch_forward(const args& p, hipStream_t stream) {
    const shape s = row_shape(p.cols, io<T>::VEC);
    const int64_t teams = s.team == 64 ? (p.rows + 3) / 4 : p.rows;
    const dim3 grid((unsigned)std::min<int64_t>(teams, 1 << 20));
#define SGV_RN_GO(TEAM, NV) hipLaunchKernelGGL((rms_norm_kernel<T, OUT, TEAM, NV, TAIL>), grid, dim3(TEAM == 64 ? 256 : TEAM), 0, stream, p)
    if (s.nv == 0) hipLaunchKernelGGL((rms_norm_long_kernel<T, (OUT > 0)>), grid, dim3(1024), 0, stream, p);
    else { SGV_RN_SHAPES(SGV_RN_GO) }
#undef SGV_RN_GO
}

template <typename T>
static void launch_forward(const args& p, hipStream_t stream) {
    const bool tail = p.cols % io<T>::VEC != 0;
    if (p.q && p.weight) { if (tail) launch_forward<T, 2, true>(p, stream); else launch_forward<T, 2, false>(p, stream); }
    else if (p.q) { if (tail) launch_forward<T, 1, true>(p, stream); else launch_forward<T, 1, false>(p, stream); }
    else { if (tail) launch_forward<T, 0, true>(p, stream); else launch_forward<T, 0, false>(p, stream); }
}

template <typename T, bool DW, bool TAIL>
static void launch_backward(const bwd_args& p, int blocks, hipStream_t stream) {
    const shape s = row_shape(p.cols, io<T>::VEC);
    const dim3 grid((unsigned)blocks);
#define SGV_RN_GO(TEAM, NV) hipLaunchKernelGGL((rms_norm_backward_kernel<T, DW, TEAM, NV, TAIL>), grid, dim3(TEAM == 64 ? 256 : TEAM), 0, stream, p)
    if (s.nv == 0) hipLaunchKernelGGL((rms_norm_backward_long_kernel<T>), grid, dim3(1024), 0, stream, p);
    else { SGV_RN_SHAPES(SGV_RN_GO) }
#undef SGV_RN_GO
}

template <typename T>
static void launch_backward(const bwd_args& p, int blocks, hipStream_t stream) {
    const bool tail = p.cols % io<T>::VEC != 0;
    if (p.partials) { if (tail) launch_backward<T, true, true>(p, blocks, stream); else launch_backward<T, true, false>(p, blocks, stream); }
    else { if (tail) launch_backward<T, false, true>(p, blocks, stream); else launch_backward<T, false, false>(p, blocks, stream); }
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
    return (int64_t)sgv_rn::backward_blocks(rows, cols, dtype == SGV_F32 ? 4 : 8, true) * cols * 4;
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
    const int blocks = sgv_rn::backward_blocks(q->rows, q->cols, vec, q->dweight != nullptr);
    if (q->dweight && (!q->workspace || q->workspace_bytes < (int64_t)blocks * q->cols * 4))
        return sgv_fail(SGV_ERR_INVALID_ARG, "rms_norm_backward: the weight gradient needs sgv_rms_norm_backward_workspace_bytes() of workspace");
    sgv_rn::bwd_args p{};
    p.dy = q->dy; p.h = q->h; p.dh = q->dh; p.weight = q->weight; p.inv_rms = q->inv_rms; p.dx = q->dx; p.partials = q->dweight ? (float*)q->workspace : nullptr;
    p.rows = q->rows; p.dy_stride = q->dy_stride; p.h_stride = q->h_stride; p.dh_stride = q->dh_stride; p.cols = q->cols; p.weight_f32 = q->weight_f32;
    hipStream_t stream = (hipStream_t)stream_;
    const double es = (double)sgv_dtype_size(dtype), n = (double)q->rows * q->cols;
    sgv_launch_scope scope(SGV_K_RMS_NORM, stream, n * es * (q->dh ? 4 : 3));
    if (dtype == SGV_F32) sgv_rn::launch_backward<float>(p, blocks, stream);
    else if (dtype == SGV_F16) sgv_rn::launch_backward<sgv_half_t>(p, blocks, stream);
    else sgv_rn::launch_backward<sgv_bf16_t>(p, blocks, stream);
    int rc = sgv_check_launch("rms_norm_backward_kernel");
    if (rc != SGV_OK || !q->dweight) return rc;
    const dim3 grid((unsigned)((q->cols + 31) / 32));
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
    const dim3 grid((unsigned)std::min<int64_t>((rows * ((cols + 15) / 16) + 255) / 256, 1 << 20));
    const int8_t* in = (const int8_t*)q;
    if (dtype == SGV_F32) hipLaunchKernelGGL((sgv_rn::dequantize_rows_kernel<float>), grid, dim3(256), 0, stream, in, q_stride, scale, (float*)out, rows, cols);
    else if (dtype == SGV_F16) hipLaunchKernelGGL((sgv_rn::dequantize_rows_kernel<sgv_half_t>), grid, dim3(256), 0, stream, in, q_stride, scale, (sgv_half_t*)out, rows, cols);
    else hipLaunchKernelGGL((sgv_rn::dequantize_rows_kernel<sgv_bf16_t>), grid, dim3(256), 0, stream, in, q_stride, scale, (sgv_bf16_t*)out, rows, cols);
    return sgv_check_launch("dequantize_rows_kernel");
}
