// Root-mean-square norm of rows, with the addition of a residual stream in front of it and an 8-bit output behind it (sgv_rms_norm), its gradient
// (sgv_rms_norm_backward), and the way back from 8 bits (sgv_dequantize_rows).
//
//   h = T(x + r)                                     r optional; T = rounding to the tensors' type: h is a tensor of its own, and the norm sees that tensor
//   y = h * inv * w        inv = rsqrt(mean_k h^2 + eps)       w optional, per column
//   8 bits: u = h * w,  q = rint_half_even(127 u / max|u|),  scale = max|y| / 127   (inv cancels out of q)
//   gradient, with g = dy * w and xh = h * inv:  dx = dr = inv * (g - xh * mean_k(g xh)) + dh,   dw = sum_rows dy * xh
//
// All of it is bound by memory (12 operations per element against 3..10 bytes): a row is read once into registers, 16 bytes per lane and load, at most 16 elements to a
// thread, and nothing is read again.  Rows of up to 1024 elements are one wave's or share one (no barrier at all), longer ones a workgroup's of 128..1024 threads;
// workgroups walk over rows with the next row's loads in flight while one is reduced and written, and hold the weight in registers.  Rows beyond 16384 elements are walked
// over three times (the later reads come from the L2).  16-byte accesses need no alignment on this chip, so odd lengths and strides take the same kernels: a row's last,
// partial vector is moved back to end with the row.  Calls that move more than the caches hold go past them.
// Measured with a weight (a 1 GB copy: 5.2 TB/s): [16384, 4096] bf16 forward 41 us = 6.5 TB/s, with a residual 92 us = 5.9, to 8 bits 39 us = 5.2 (half of it instructions:
// 16 an element), with a residual 75 us = 6.3, backward with all gradients 89 us = 6.0; [30000, 1111] fp16 forward 27 us = 5.0, backward with all gradients 73 us = 3.6 (few
// waves in flight: the workgroups are held down by the partial sums below, and eleven of 128 threads have a second vector).
//
// Statistics are fp32: a lane sums at most 16 squares before the tree (fp64 in the walking kernels).  A row whose squares leave fp32's range (|h| > 1e18, or tiny rows under a
// tiny eps) is summed again in fp64.  The 8-bit values are the correctly rounded ones: fp32 places a value to 5.4e-5 of a step, so a value within 6e-5 of a border
// between two steps is decided in fp64; the row maximum is exact because the product of two 16-bit values is exact in fp32, and other products are taken in fp64 by the
// lanes that hold the maximum.
#pragma once

#include "sgv_common.h"

#include <algorithm>
#include <initializer_list>

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

// 16 bytes past the caches (aligned rows only: partial lines are written twice that way)
template <typename T> __device__ __forceinline__ u32x4 stream_vec(const T* row, int i) { return __builtin_nontemporal_load((const u32x4*)(row + i)); }
template <typename T> __device__ __forceinline__ void stream_vec(T* row, int i, const u32x4& v) { __builtin_nontemporal_store(v, (u32x4*)(row + i)); }
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

// Reductions over the threads of a row.  A wave's fp32 sum and 32-bit maximum go through the DPP lanes shifts (six dependent VALU operations; the same tree through
// LDS permutes costs six trips of ~60 clocks) and come back as scalars; a workgroup's waves meet in LDS with one barrier.  Two slots in turn: a slot is written again
// only behind the barrier of the reduction in between, which every wave reaches after it has read the slot.
template <int CTRL, int ROWS> __device__ __forceinline__ unsigned dpp(unsigned v) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false); }
__device__ __forceinline__ float wave_sum(float v) {
#define SGV_RN_STEP(CTRL, ROWS) v += __uint_as_float(dpp<CTRL, ROWS>(__float_as_uint(v)))
    SGV_RN_STEP(0x111, 0xf); SGV_RN_STEP(0x112, 0xf); SGV_RN_STEP(0x114, 0xf); SGV_RN_STEP(0x118, 0xf);      // row_shr 1, 2, 4, 8: lane 15 of every row of 16 holds its sum
    SGV_RN_STEP(0x142, 0xa); SGV_RN_STEP(0x143, 0xc);                                                          // row_bcast 15, 31: lane 63 holds the wave's
#undef SGV_RN_STEP
    return __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(v), 63));
}
__device__ __forceinline__ unsigned wave_max(unsigned v) {
#define SGV_RN_STEP(CTRL, ROWS) v = max(v, dpp<CTRL, ROWS>(v))
    SGV_RN_STEP(0x111, 0xf); SGV_RN_STEP(0x112, 0xf); SGV_RN_STEP(0x114, 0xf); SGV_RN_STEP(0x118, 0xf); SGV_RN_STEP(0x142, 0xa); SGV_RN_STEP(0x143, 0xc);
#undef SGV_RN_STEP
    return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}
// Rows of 8, 16 or 32 lanes, several to a wave: quad_perm 1, 2, half mirror, mirror and a swizzle; every lane ends with the same bits, sums being of equal pairs.
__device__ __forceinline__ unsigned swap16(unsigned v) { return (unsigned)__builtin_amdgcn_ds_swizzle((int)v, 0x401f); }
template <int TEAM> __device__ __forceinline__ float lanes_sum(float v) {
    if constexpr (TEAM >= 8) {
        v += __uint_as_float(dpp<0xb1, 0xf>(__float_as_uint(v)));
        v += __uint_as_float(dpp<0x4e, 0xf>(__float_as_uint(v)));
        v += __uint_as_float(dpp<0x141, 0xf>(__float_as_uint(v)));
    }
    if constexpr (TEAM >= 16) v += __uint_as_float(dpp<0x140, 0xf>(__float_as_uint(v)));
    if constexpr (TEAM >= 32) v += __uint_as_float(swap16(__float_as_uint(v)));
    return v;
}
template <int TEAM> __device__ __forceinline__ unsigned lanes_max(unsigned v) {
    if constexpr (TEAM >= 8) { v = max(v, dpp<0xb1, 0xf>(v)); v = max(v, dpp<0x4e, 0xf>(v)); v = max(v, dpp<0x141, 0xf>(v)); }
    if constexpr (TEAM >= 16) v = max(v, dpp<0x140, 0xf>(v));
    if constexpr (TEAM >= 32) v = max(v, swap16(v));
    return v;
}
struct red_slots { float sum[2][16]; unsigned top[2][16]; double wide[2][16]; };
// sum and maximum of a row together (MAX false: the sum alone)
template <int TEAM, bool MAX>
__device__ __forceinline__ void team_reduce(float& sum, unsigned& top, red_slots& s, int& turn) {
    if constexpr (TEAM < 64) {
        sum = lanes_sum<TEAM>(sum);
        if constexpr (MAX) top = lanes_max<TEAM>(top);
        return;
    }
    sum = wave_sum(sum);
    if constexpr (MAX) top = wave_max(top);
    if constexpr (TEAM > 64) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) { s.sum[turn][wave] = sum; if constexpr (MAX) s.top[turn][wave] = top; }
        __syncthreads();
        sum = 0.f;
        top = 0;
#pragma unroll
        for (int w = 0; w < TEAM / 64; w++) { sum += s.sum[turn][w]; if constexpr (MAX) top = max(top, s.top[turn][w]); }
        turn ^= 1;
    }
}
template <int TEAM>
__device__ __forceinline__ float team_sum(float v, red_slots& s, int& turn) {
    unsigned none = 0;
    team_reduce<TEAM, false>(v, none, s, turn);
    return v;
}
// the rare fp64 ones (values out of fp32's range)
template <int TEAM, typename F>
__device__ __forceinline__ double team_wide(double v, red_slots& s, int& turn, F f) {
#pragma unroll
    for (int off = TEAM < 64 ? TEAM / 2 : 32; off > 0; off >>= 1) v = f(v, __shfl_xor(v, off, 64));
    if constexpr (TEAM > 64) {
        if ((threadIdx.x & 63) == 0) s.wide[turn][threadIdx.x >> 6] = v;
        __syncthreads();
        v = s.wide[turn][0];
#pragma unroll
        for (int w = 1; w < TEAM / 64; w++) v = f(v, s.wide[turn][w]);
        turn ^= 1;
    }
    return v;
}
struct add_op { __device__ __forceinline__ double operator()(double a, double b) const { return a + b; } };
struct max_op { __device__ __forceinline__ double operator()(double a, double b) const { return a > b ? a : b; } };      // (of numbers; NaN is looked for elsewhere)
// The maximum of v (not below zero) over the lanes where `any` -- few -- of the threads of a row
template <int TEAM>
__device__ __forceinline__ double team_top(double v, bool any, red_slots& s, int& turn) {
    if constexpr (TEAM < 64) return team_wide<TEAM>(v, s, turn, max_op());
    double m = 0.0;
    for (uint64_t lanes = __ballot(any); lanes; lanes &= lanes - 1) {
        const int lane = __builtin_ctzll(lanes);
        const uint64_t b = (uint64_t)__double_as_longlong(v);
        const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)b, lane), hi = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)(b >> 32), lane);
        const double x = __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
        m = x > m ? x : m;
    }
    if constexpr (TEAM > 64) {
        if ((threadIdx.x & 63) == 0) s.wide[turn][threadIdx.x >> 6] = m;
        __syncthreads();
        m = s.wide[turn][0];
#pragma unroll
        for (int w = 1; w < TEAM / 64; w++) m = s.wide[turn][w] > m ? s.wide[turn][w] : m;
        turn ^= 1;
    }
    return m;
}

__device__ __forceinline__ unsigned abs_bits(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }                       // orders magnitudes, NaN above infinity
// the largest magnitude so far and two more values (one instruction; a NaN is passed over).  In assembly: of __builtin_fmaxf each argument is made canonical first.
__device__ __forceinline__ unsigned max3_abs(unsigned top, float a, float b) {
    unsigned r;
    asm("v_max3_f32 %0, %1, |%2|, |%3|" : "=v"(r) : "v"(top), "v"(a), "v"(b));
    return r;
}

// The vector v of thread t of a row: its first column, and how many of its columns the vector in front of it has too.  A row whose length is no multiple of VEC ends with
// a vector that is moved back to lie inside the row: both write the same values to the columns they share, and the sums leave them out once.  A row shorter than a vector is
// one thread's (TEAM = 1), whose vector ends with zeros.
template <int TEAM, int VEC>
__device__ __forceinline__ int vec_column(int v, int t, int cols, int& shared) {
    int i = (v * TEAM + t) * VEC;
    shared = 0;
    if (TEAM > 1 && i < cols && i + VEC > cols) { shared = i + VEC - cols; i = cols - VEC; }
    return i;
}

template <typename T, bool STREAM, bool TAIL, int NV>
__device__ __forceinline__ void load_row(const T* row, const int* col, int cols, u32x4* out) {
#pragma unroll
    for (int v = 0; v < NV; v++) {
        out[v] = u32x4{0u, 0u, 0u, 0u};
        if (col[v] < cols) out[v] = STREAM ? stream_vec(row, col[v]) : load_vec<T, TAIL>(row, col[v], cols);
    }
}
template <typename T, bool STREAM, bool TAIL>
__device__ __forceinline__ void put_vec(T* row, int i, int cols, const u32x4& v) {
    if (i >= cols) return;
    if (STREAM) stream_vec(row, i, v); else store_vec<T, TAIL>(row, i, cols, v);
}

// How the weight is kept: not at all, in the rows' type, in fp32 beside 16-bit rows.
enum weight_kind { W_NONE, W_ROWS, W_F32 };
// The weight of a thread's columns: loaded once per workgroup, kept as it is stored.
template <typename T, int WK, bool TAIL, int NV>
struct held_weight {
    static constexpr int VEC = io<T>::VEC;
    u32x4 raw[WK == W_NONE ? 1 : NV][WK == W_F32 ? 2 : 1];
    __device__ __forceinline__ void load(const void* w, int v, int i, int cols) {
        if constexpr (WK == W_ROWS) raw[v][0] = i < cols ? load_vec<T, TAIL>((const T*)w, i, cols) : u32x4{0u, 0u, 0u, 0u};
        if constexpr (WK == W_F32) {
            raw[v][0] = i < cols ? load_vec<float, TAIL>((const float*)w, i, cols) : u32x4{0u, 0u, 0u, 0u};
            raw[v][1] = i < cols ? load_vec<float, TAIL>((const float*)w, i + 4, cols) : u32x4{0u, 0u, 0u, 0u};
        }
    }
    // once per row: keeps the compiler from holding the unpacked weight (and its fp64 form) over the rows, which takes twice the registers
    __device__ __forceinline__ void fresh() {
        if constexpr (WK != W_NONE) {
#pragma unroll
            for (int v = 0; v < NV; v++)
#pragma unroll
                for (int i = 0; i < (WK == W_F32 ? 2 : 1); i++) asm volatile("" : "+v"(raw[v][i]));
        }
    }
    __device__ __forceinline__ void get(int v, float* f) const {
        if constexpr (WK == W_NONE) {
#pragma unroll
            for (int j = 0; j < VEC; j++) f[j] = 1.f;
        }
        if constexpr (WK == W_ROWS) io<T>::unpack(raw[v][0], f);
        if constexpr (WK == W_F32) { io<float>::unpack(raw[v][0], f); io<float>::unpack(raw[v][1], f + 4); }
    }
};

// How a row is held: TEAM threads with at most 16 elements each, or not at all (elems = 0, the walking kernels: 1024 threads for rows beyond 16384 elements).  Rows of
// up to 64 vectors have as many lanes as vectors, up to a power of two ([262144, 128] bf16: a wave to a row 34 us forward, 56 to 8 bits, 100 backward with the weight's
// gradient; 16 lanes 20, 20 and 40), rows shorter than a vector one ([1000000, 5] bf16: a wave 593 us forward, 5.0 ms backward as it was first built; a thread 10 and 21 us).
// 16 elements are what leaves registers for the next row's loads, the weight and its gradient's sums; rows beyond 16384 elements are walked over for it (forward 3.7 TB/s,
// 1.4 to 1.5 to 8 bits or with the weight's gradient: [2048, 32768] bf16).
struct shape { int team, elems; };
static inline shape row_shape(int cols, int vec) {
    static const shape held[] = {{8, 4}, {16, 4}, {32, 4}, {64, 4}, {8, 8}, {16, 8}, {32, 8}, {64, 8}, {64, 16}, {128, 16}, {256, 16}, {512, 16}, {1024, 16}};
    if (cols < vec) return shape{1, vec};
    for (const shape& s : held) if (s.elems >= vec && cols <= s.team * s.elems) return s;
    return shape{1024, 0};
}
constexpr int MAX_COLS = (1 << 26) - 1;

// Workgroups of a launch, which walk over the rows: twice as many as 2048 threads to a CU, where rows are short; as many as the registers let a CU hold, 1024 threads, where
// a row takes 512 threads or more ([4096, 16384] bf16 forward 40.8 us, four times as many 43.1; to 8 bits with a weight 44.6 and 49.5).  With a weight gradient they are the
// rows of its partial sums, which should stay small beside the rows: one to a CU where a row takes 256 threads or more ([16384, 4096] bf16 with all gradients 89 us, two 92, four 107;
// [4096, 16384] with the weight's 80, 89, 104), four to a CU of 128 threads ([30000, 1111] fp16: 59 us, two 74, one 104), two of four short rows ([65536, 512] bf16: 40 us, one
// 57, four 43); four rows to each at least ([2049, 1111] fp16: 10.5 us, one workgroup to a CU 12.8, two rows to each 10.6).
static inline int64_t groups(int64_t rows, const shape& s, bool dw) {
    const int threads = std::max(s.team, 256 * (s.team <= 64)), rpb = threads / s.team;
    const int64_t teams = (rows + rpb - 1) / rpb;
    const int64_t most = dw ? std::min<int64_t>(rpb > 1 ? 512 : threads <= 128 ? 1024 : 256, std::max<int64_t>(256, rows / 4)) : threads >= 512 ? 262144 / threads : 512 * (2048 / threads);
    return std::min(teams, most);
}

// the kernel for a shape: F<team, vectors>
template <typename T, typename F>
static void for_shape(const shape& s, F f) {
    constexpr int VEC = io<T>::VEC;
    if (s.team == 1) f.template go<1, 1>();
    else if (s.team == 8) f.template go<8, 1>();
    else if (s.team == 16) f.template go<16, 1>();
    else if (s.team == 32) f.template go<32, 1>();
    else if (s.team == 64) {
        if constexpr (VEC == 4) { if (s.elems == 4) { f.template go<64, 1>(); return; } }
        if (s.elems == 8) f.template go<64, 8 / VEC>(); else f.template go<64, 16 / VEC>();
    } else if (s.team == 128) f.template go<128, 16 / VEC>();
    else if (s.team == 256) f.template go<256, 16 / VEC>();
    else if (s.team == 512) f.template go<512, 16 / VEC>();
    else f.template go<1024, 16 / VEC>();
}

// Past the caches: calls that move more than 1.5 times the 256 MB Infinity Cache, over rows of whole aligned vectors ([16384, 4096] bf16 with a residual forward 98 -> 92 us,
// backward 97 -> 89; the forward alone, 268 MB, would go from 41 to 44).
struct rows_at { const void* p; int64_t stride; };
static bool streams(double bytes, int dtype, int cols, std::initializer_list<rows_at> all) {
    const int64_t es = (int64_t)sgv_dtype_size(dtype);
    if (bytes < 384e6 || cols * es % 16) return false;
    for (const rows_at& r : all) if ((uintptr_t)r.p % 16 || r.stride * es % 16) return false;
    return true;
}

static inline bool row_dtype(int dtype) { return dtype == SGV_F32 || dtype == SGV_F16 || dtype == SGV_BF16; }

}  // namespace sgv_rn
