// Matrix product in 8-bit integers with one scale per row of either operand (sgv_int8_gemm):
//
//   C[m,n] = act( (sum_k A[m,k] B[n,k]) * a_scale[m] * b_scale[n] + bias[n] ) * gain        A [M,K], B [N,K] signed bytes, sums in 32-bit integers
//
// Both operands are contiguous along k, which is how the matrix instruction wants them: a lane of v_mfma_i32_16x16x64_i8 holds 16 consecutive bytes of one row
// (row = lane & 15, bytes 16 (lane >> 4) ..+15 of 64).  The integer sums are exact whatever their order, so K is split freely -- over the waves of a workgroup, over
// workgroups -- and the result depends neither on the split nor on the other rows of a batch.
//
// Three forms, chosen in sgv_int8_gemm by how many workgroups they make and what each has to read:
//   int8_rows_kernel   few rows: bound by reading B once
//   int8_tile_kernel   tiles of C through LDS: bound by the matrix pipe (large) or by the latency of a tile's K loop (few tiles)
//   ... with K split over workgroups into 32-bit partial tiles, and int8_sum_kernel behind it
#include "sgv_common.h"

#include <algorithm>

namespace sgv_i8 {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
struct any_i32x4 { i32x4 v; } __attribute__((packed, aligned(2)));       // a 16-byte access at any element's address

struct args {
    const int8_t* a; const int8_t* b; const float* a_scale; const float* b_scale; const float* bias; void* c;
    int64_t lda, ldb, ldc;
    int m, n, k;
    int lrelu;
    float alpha, gain;
    int tiles_m, tiles_n;
    int slice;               // k per workgroup (a multiple of 128; the whole of k: no split); slice z writes its sums at c + z * m * ldc
};

// 16 bytes of a row, `left` of them in front of K: the others are cleared (in one operand: 0 times anything is 0)
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

// ---------------------------------------------------------------------------------------------------------------------------------------
// Few rows: a workgroup owns 16 MT rows x 16 columns, its waves split K, the partial sums meet in LDS.  Operands go from memory to registers: B is used MT times per
// wave, there is nothing to share.  U steps of 64 k are loaded together.
template <typename T, int MT, int U>
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
    const int steps = (p.k + 63) / 64, per = (steps + waves - 1) / waves;
    const int first = min(wave * per, steps), last = min(first + per, steps);           // a wave's steps are consecutive: whole cache lines
    int s = first;
    for (; s + U <= last && (s + U) * 64 <= p.k; s += U) {
        i32x4 av[U][MT], bv[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            bv[u] = *(const i32x4*)(b + (s + u) * 64);
#pragma unroll
            for (int t = 0; t < MT; t++) av[u][t] = *(const i32x4*)(a[t] + (s + u) * 64);
        }
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int t = 0; t < MT; t++) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(av[u][t], bv[u], acc[t], 0, 0, 0);
    }
    for (; s < last; s++) {
        const int left = p.k - s * 64 - kq;
        const bool ok = left > 0;
        const i32x4 bv = mask_tail(ok ? *(const i32x4*)(b + s * 64) : i32x4{0, 0, 0, 0}, left);
#pragma unroll
        for (int t = 0; t < MT; t++) {
            const i32x4 av = ok ? *(const i32x4*)(a[t] + s * 64) : i32x4{0, 0, 0, 0};
            acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(av, bv, acc[t], 0, 0, 0);
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
        int sum = red[i];
        for (int w = 1; w < waves; w++) sum += red[w * (MT * 256) + i];
        sgv_traits<T>::store((T*)p.c + (int64_t)m * p.ldc + n, finish(p, sum, p.a_scale[m], p.b_scale[n], p.bias ? p.bias[n] : 0.f));
    }
}

// ---------------------------------------------------------------------------------------------------------------------------------------
// Tiles of C.  K is walked in stages of 128 bytes per row -- a cache line -- that go from memory straight into LDS (buffer_load ... lds: no registers, no instructions
// to store them), S stages in a ring.  A stage's 16-byte chunks lie at position chunk ^ ((row >> 1) & 7) of their row, which makes the fragment reads below free of
// bank conflicts.  A wave holds the fragments of one step of 64 k in registers and replaces each as soon as its last product is issued, so that the matrix pipe finds
// the next step's fragments there; one barrier per stage.  Rows beyond the matrix and bytes beyond its end are outside the buffers' bounds and read as zero.

__device__ __forceinline__ i32x4 make_rsrc(const void* base, int64_t bytes) {
    const uint64_t b = (uint64_t)base;
    return i32x4{(int)(unsigned)b, (int)((unsigned)(b >> 32) & 0xffffu), (int)(unsigned)(bytes > 0xffffffffll ? 0xffffffffll : bytes), 0x00020000};
}
// 16 bytes per lane from rsrc + voff + soff to LDS at lds + 16 lane.  In inline assembly because the compiler waits for ALL outstanding loads in front of any LDS read behind
// the builtin; nothing lands in a register, and the kernel counts these loads itself (s_waitcnt vmcnt).
__device__ __forceinline__ void dma16(i32x4 rsrc, unsigned lds, unsigned voff, int soff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" :: "s"(lds), "v"(voff), "s"(rsrc), "s"(soff) : "memory");
}

// four consecutive columns as they are stored
template <typename T> struct quad;
template <> struct quad<int> {
    typedef i32x4 type;
    static __device__ __forceinline__ type make(const args&, const i32x4& acc, float, const f32x4&, const f32x4&) { return acc; }
};
__device__ __forceinline__ f32x4 finish4(const args& p, const i32x4& acc, float sa, const f32x4& sb, const f32x4& bias) {
    return f32x4{finish(p, acc[0], sa, sb[0], bias[0]), finish(p, acc[1], sa, sb[1], bias[1]), finish(p, acc[2], sa, sb[2], bias[2]), finish(p, acc[3], sa, sb[3], bias[3])};
}
template <> struct quad<float> {
    typedef f32x4 type;
    static __device__ __forceinline__ type make(const args& p, const i32x4& acc, float sa, const f32x4& sb, const f32x4& bias) { return finish4(p, acc, sa, sb, bias); }
};
template <> struct quad<sgv_half_t> {
    typedef i32x2 type;
    static __device__ __forceinline__ type make(const args& p, const i32x4& acc, float sa, const f32x4& sb, const f32x4& bias) {
        typedef _Float16 h4 __attribute__((ext_vector_type(4)));
        return __builtin_bit_cast(i32x2, __builtin_convertvector(finish4(p, acc, sa, sb, bias), h4));
    }
};
template <> struct quad<sgv_bf16_t> {
    typedef i32x2 type;
    static __device__ __forceinline__ type make(const args& p, const i32x4& acc, float sa, const f32x4& sb, const f32x4& bias) {
        typedef __bf16 b4 __attribute__((ext_vector_type(4)));
        return __builtin_bit_cast(i32x2, __builtin_convertvector(finish4(p, acc, sa, sb, bias), b4));
    }
};

// WGM x WGN waves; LEAD: rows of products between a stage's wait and the reads it allows
template <typename T, int BM, int BN, int WGM, int WGN, int S, int LEAD>
__global__ __launch_bounds__(64 * WGM * WGN) void int8_tile_kernel(const args p) {
    constexpr int BK = 128, CPR = BK / 16, RPI = 64 / CPR;                // chunks per row, rows per DMA instruction
    constexpr int WAVES = WGM * WGN, TM = BM / WGM / 16, TN = BN / WGN / 16, STAGE = (BM + BN) * BK, LA = BM / RPI / WAVES, LB = BN / RPI / WAVES, LPS = LA + LB;
    constexpr bool PARTIAL = sizeof(T) == 4 && __is_same(T, int);
    __shared__ __attribute__((aligned(128))) int8_t lds[S * STAGE];
    __shared__ __attribute__((aligned(16))) float sb_lds[BN], bias_lds[BN];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // workgroups go to the eight XCDs in turn: each XCD takes a consecutive run of tiles, in columns of eight tile rows, so that its L2 holds what its CUs share
    int id = blockIdx.x;
    {
        const int total = p.tiles_m * p.tiles_n, xcd = id & 7, q = total >> 3, extra = total & 7;
        id = xcd * q + min(xcd, extra) + (id >> 3);
    }
    const int per = 8 * p.tiles_n, first = id / per * 8, rows8 = min(p.tiles_m - first, 8);
    const int m0 = (first + (id % per) % rows8) * BM, n0 = ((id % per) / rows8) * BN;
    const int kbase = blockIdx.y * p.slice, k = min(p.k - kbase, p.slice), k16 = (k + 15) & ~15;
    const i32x4 ra = make_rsrc(p.a + (int64_t)m0 * p.lda + kbase, (int64_t)(p.m - 1 - m0) * p.lda + k16);
    const i32x4 rb = make_rsrc(p.b + (int64_t)n0 * p.ldb + kbase, (int64_t)(p.n - 1 - n0) * p.ldb + k16);
    const i32x4 none = make_rsrc(p.a, 0);                                // (stages behind the last one: nothing is fetched, and the count of loads stays the same)
    unsigned va[LA], vb[LB];
    auto swizzle = [](int row) { return (row >> 1) & 7; };
#pragma unroll
    for (int i = 0; i < LA; i++) { const int row = (wave * LA + i) * RPI + lane / CPR; va[i] = row * (unsigned)p.lda + ((lane % CPR) ^ swizzle(row)) * 16; }
#pragma unroll
    for (int i = 0; i < LB; i++) { const int row = (wave * LB + i) * RPI + lane / CPR; vb[i] = row * (unsigned)p.ldb + ((lane % CPR) ^ swizzle(row)) * 16; }
    const int nst = (k + BK - 1) / BK;
    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) int8_t*)lds;
    auto piece = [&](int t, int slot, int q) {
        const unsigned s = lds0 + slot * STAGE;
        const int k0 = t < nst ? t * BK : 0;
        if (q < LA) dma16(t < nst ? ra : none, s + (wave * LA + q) * 1024, va[q], k0);
        else dma16(t < nst ? rb : none, s + BM * BK + (wave * LB + q - LA) * 1024, vb[q - LA], k0);
    };
#pragma unroll
    for (int t = 0; t < S; t++)
#pragma unroll
        for (int q = 0; q < LPS; q++) piece(t, t, q);
    const int wm = wave / WGN, wn = wave % WGN, quarter = lane >> 4, r = lane & 15;
    // the scales of the tile: in flight beside the first stages
    constexpr int PER = (BN + 64 * WAVES - 1) / (64 * WAVES);
    float sa[TM], sbv[PER], biv[PER];
    if constexpr (!PARTIAL) {
#pragma unroll
        for (int i = 0; i < TM; i++) { const int m = m0 + (wm * TM + i) * 16 + r; sa[i] = m < p.m ? p.a_scale[m] : 0.f; }
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int x = i * 64 * WAVES + threadIdx.x, n = n0 + x;
            const bool ok = x < BN && n < p.n;
            sbv[i] = ok ? p.b_scale[n] : 0.f;
            biv[i] = ok && p.bias ? p.bias[n] : 0.f;
        }
    }
    i32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = i32x4{0, 0, 0, 0};
    const int ck[2] = {(quarter ^ swizzle(r)) * 16, ((4 + quarter) ^ swizzle(r)) * 16};
    const int abase = (wm * TM * 16 + r) * BK, bbase = BM * BK + (wn * TN * 16 + r) * BK;
    i32x4 fa[TM], fb[TN], fn[TN];
    // (the operands change places: D's rows are columns of C, so that a lane ends with four consecutive columns of one row)
    auto row = [&](int i) {
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[j], fa[i], acc[i][j], 0, 0, 0);
    };
    // One step of 64 k on the fragments in registers, which are replaced by those at s + c.  cross: they are the next stage's.  Its loads are the oldest of S - 1 stages'
    // in flight; behind the barrier every wave has the whole of stage t in registers, and its slot takes stage t + S, one instruction between the rows of products at a
    // time (all of them at once hold the wave up at the full queue: 8192^3 5 % slower).
    auto step = [&](const int8_t* s, int c, bool cross, int t, int slot) {
#pragma unroll
        for (int i = 0; i < LEAD; i++) row(i);
        __builtin_amdgcn_sched_barrier(0);
        if (cross) {
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"((S - 2) * LPS) : "memory");
            __builtin_amdgcn_s_barrier();
        }
#pragma unroll
        for (int i = 0; i < LEAD; i++) fa[i] = *(const i32x4*)(s + abase + i * 16 * BK + c);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = LEAD; i < TM; i++) {
            row(i);
            if (cross) {
#pragma unroll
                for (int q = 0; q < LPS; q++) if (LEAD + q * (TM - LEAD) / LPS == i) piece(t + S, slot, q);
            }
            fa[i] = *(const i32x4*)(s + abase + i * 16 * BK + c);
#pragma unroll
            for (int j = 0; j < TN; j++) if (LEAD + j * (TM - LEAD) / TN == i) fn[j] = *(const i32x4*)(s + bbase + j * 16 * BK + c);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int j = 0; j < TN; j++) fb[j] = fn[j];
    };
    asm volatile("s_waitcnt vmcnt(%0)" :: "n"((S - 1) * LPS) : "memory");
    __builtin_amdgcn_s_barrier();
#pragma unroll
    for (int j = 0; j < TN; j++) fb[j] = *(const i32x4*)(lds + bbase + j * 16 * BK + ck[0]);
#pragma unroll
    for (int i = 0; i < TM; i++) fa[i] = *(const i32x4*)(lds + abase + i * 16 * BK + ck[0]);
    int slot = 0;
    for (int t = 0; t < nst - 1; t++) {
        const int next = slot + 1 == S ? 0 : slot + 1;
        step(lds + slot * STAGE, ck[1], false, t, slot);
        step(lds + next * STAGE, ck[0], true, t, slot);
        slot = next;
    }
    int left = k - (nst - 1) * BK;
    if (left > 64) { step(lds + slot * STAGE, ck[1], false, 0, 0); left -= 64; }
    if (left < 64) {
#pragma unroll
        for (int j = 0; j < TN; j++) fb[j] = mask_tail(fb[j], left - quarter * 16);
    }
#pragma unroll
    for (int i = 0; i < TM; i++) row(i);

    // Strips of 16 rows go through a wave's own piece of LDS, so that rows of C leave in 16-byte pieces.
    constexpr int ES = sizeof(T), PITCH = TN * 16 * ES + 16, CH = TN * ES, PCS = 16 / ES;
    static_assert(WAVES * 16 * PITCH <= S * STAGE && (16 * CH) % 64 == 0, "");
    if constexpr (!PARTIAL) {
#pragma unroll
        for (int i = 0; i < PER; i++) { const int x = i * 64 * WAVES + threadIdx.x; if (x < BN) { sb_lds[x] = sbv[i]; bias_lds[x] = biv[i]; } }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");            // (every load into LDS has landed, the empty ones too: the ring may be written over)
    __builtin_amdgcn_s_barrier();
    int8_t* buf = lds + wave * 16 * PITCH;
    const int nb = n0 + wn * TN * 16, ncols = PARTIAL ? (int)p.ldc : p.n;
    const bool whole = m0 + BM <= p.m && n0 + BN <= ncols;
    T* out = (T*)p.c + (PARTIAL ? (int64_t)blockIdx.y * p.m * p.ldc : 0);
#pragma unroll
    for (int i = 0; i < TM; i++) {
#pragma unroll
        for (int j = 0; j < TN; j++) {
            const int x = j * 16 + 4 * quarter;
            f32x4 s4 = {0.f, 0.f, 0.f, 0.f}, b4 = {0.f, 0.f, 0.f, 0.f};
            if constexpr (!PARTIAL) { s4 = *(const f32x4*)(sb_lds + wn * TN * 16 + x); b4 = *(const f32x4*)(bias_lds + wn * TN * 16 + x); }
            *(typename quad<T>::type*)(buf + r * PITCH + x * ES) = quad<T>::make(p, acc[i][j], PARTIAL ? 0.f : sa[i], s4, b4);
        }
        const int mb = m0 + (wm * TM + i) * 16;
#pragma unroll
        for (int q = 0; q < 16 * CH / 64; q++) {
            const int idx = q * 64 + lane, rr = idx / CH, ch = idx % CH, n = nb + ch * PCS;
            T* o = out + (int64_t)(mb + rr) * p.ldc + n;
            const i32x4 v = *(const i32x4*)(buf + rr * PITCH + ch * 16);
            if (whole || (mb + rr < p.m && n + PCS <= ncols)) ((any_i32x4*)o)->v = v;
            else if (mb + rr < p.m)
                for (int x = 0; n + x < ncols; x++) o[x] = ((const T*)(buf + rr * PITCH + ch * 16))[x];
        }
    }
}

// C from the partial sums [slices][m][ldp] of a product whose K was split; ldp is a multiple of 4, a thread takes four columns
template <typename T>
__global__ __launch_bounds__(256) void int8_sum_kernel(const args p, const int* part, int64_t ldp, int slices) {
    const int64_t quads = ldp / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= quads * p.m) return;
    const int m = (int)(i / quads), n = (int)(i % quads) * 4;
    const int* src = part + (int64_t)m * ldp + n;
    i32x4 acc = *(const i32x4*)src;
#pragma unroll 4
    for (int z = 1; z < slices; z++) acc += *(const i32x4*)(src + (int64_t)z * p.m * ldp);
    const float sa = p.a_scale[m];
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (n + e < p.n) sgv_traits<T>::store((T*)p.c + (int64_t)m * p.ldc + n + e, finish(p, acc[e], sa, p.b_scale[n + e], p.bias ? p.bias[n + e] : 0.f));
}

// ---------------------------------------------------------------------------------------------------------------------------------------
enum form { ROWS, TILE64, TILE128, TILE256 };
struct plan { form f; int slices, slice; };

static inline int64_t tiles(int m, int n, int edge) { return ((int64_t)(m + edge - 1) / edge) * ((n + edge - 1) / edge); }

static plan choose(int m, int n, int k, int64_t lda, int64_t ldb) {
    const int whole = (k + 127) / 128 * 128;
    const bool near = lda < (1 << 23) && ldb < (1 << 23);           // the offsets inside a tile fit 32 bits
    if (m <= 64 || !near) return plan{ROWS, 1, whole};
    if (tiles(m, n, 256) >= 200) return plan{TILE256, 1, whole};
    if (tiles(m, n, 128) >= 200) return plan{TILE128, 1, whole};
    const int64_t t64 = tiles(m, n, 64);
    const int slices = (int)std::min<int64_t>(256 / t64, whole / 512);
    if (slices >= 2) {
        const int slice = (whole / 128 + slices - 1) / slices * 128;
        return plan{TILE64, (whole + slice - 1) / slice, slice};
    }
    return plan{TILE64, 1, whole};
}

static inline int64_t partial_pitch(int n) { return ((int64_t)n + 3) / 4 * 4; }

template <typename T, int BM, int BN, int WGM, int WGN, int S, int LEAD>
static void launch_tile(args p, int slices, hipStream_t stream) {
    p.tiles_m = (p.m + BM - 1) / BM;
    p.tiles_n = (p.n + BN - 1) / BN;
    hipLaunchKernelGGL((int8_tile_kernel<T, BM, BN, WGM, WGN, S, LEAD>), dim3((unsigned)(p.tiles_m * p.tiles_n), (unsigned)slices), dim3(64 * WGM * WGN), 0, stream, p);
}

template <typename T>
static void launch(args p, const plan& pl, void* workspace, hipStream_t stream) {
    p.slice = pl.slice;
    if (pl.f == ROWS) {
        const int mt = p.m <= 16 ? 1 : p.m <= 32 ? 2 : 4;
        const int steps = (p.k + 63) / 64;
        const int waves = std::max(1, std::min(mt == 4 ? 8 : 16, steps));
        const dim3 grid((unsigned)((p.n + 15) / 16), (unsigned)((p.m + 16 * mt - 1) / (16 * mt))), block(64 * waves);
        const size_t lds = (size_t)waves * mt * 1024;
        if (mt == 1) hipLaunchKernelGGL((int8_rows_kernel<T, 1, 8>), grid, block, lds, stream, p);
        else if (mt == 2) hipLaunchKernelGGL((int8_rows_kernel<T, 2, 4>), grid, block, lds, stream, p);
        else hipLaunchKernelGGL((int8_rows_kernel<T, 4, 4>), grid, block, lds, stream, p);
    } else if (pl.slices > 1) {
        args q = p;
        q.c = workspace;
        q.ldc = partial_pitch(p.n);
        launch_tile<int, 64, 64, 2, 2, 4, 1>(q, pl.slices, stream);
        const int64_t quads = q.ldc / 4 * p.m;
        hipLaunchKernelGGL((int8_sum_kernel<T>), dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, stream, p, (const int*)workspace, q.ldc, pl.slices);
    } else if (pl.f == TILE256) launch_tile<T, 256, 256, 2, 4, 2, 2>(p, 1, stream);
    else if (pl.f == TILE128) launch_tile<T, 128, 128, 2, 4, 4, 1>(p, 1, stream);
    else launch_tile<T, 64, 64, 2, 2, 4, 1>(p, 1, stream);
}

}  // namespace sgv_i8

extern "C" int64_t sgv_int8_gemm_workspace_bytes(int32_t m, int32_t n, int32_t k, int64_t lda, int64_t ldb) {
    if (m < 1 || n < 1 || k < 1 || k > 131071) return 0;
    const sgv_i8::plan pl = sgv_i8::choose(m, n, k, lda, ldb);
    return pl.slices > 1 ? (int64_t)pl.slices * m * sgv_i8::partial_pitch(n) * 4 : 0;
}

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
    const sgv_i8::plan pl = sgv_i8::choose(q->m, q->n, q->k, q->lda, q->ldb);
    if (pl.f == sgv_i8::ROWS && ((int64_t)q->m + 63) / 64 > 65535) return sgv_fail(SGV_ERR_TOO_LARGE, "int8_gemm: too many rows");
    if (sgv_i8::tiles(q->m, q->n, pl.f == sgv_i8::TILE256 ? 256 : pl.f == sgv_i8::TILE128 ? 128 : 64) > 0x7fffffff) return sgv_fail(SGV_ERR_TOO_LARGE, "int8_gemm: too many tiles");
    if (q->workspace_bytes < sgv_int8_gemm_workspace_bytes(q->m, q->n, q->k, q->lda, q->ldb) || (pl.slices > 1 && !q->workspace))
        return sgv_fail(SGV_ERR_INVALID_ARG, "int8_gemm: this size needs sgv_int8_gemm_workspace_bytes() of workspace");
    sgv_i8::args p{};
    p.a = (const int8_t*)q->a; p.b = (const int8_t*)q->b; p.a_scale = q->a_scale; p.b_scale = q->b_scale; p.bias = q->bias; p.c = q->c;
    p.lda = q->lda; p.ldb = q->ldb; p.ldc = q->ldc; p.m = q->m; p.n = q->n; p.k = q->k;
    p.lrelu = q->act == 3; p.alpha = q->alpha; p.gain = q->gain;
    hipStream_t stream = (hipStream_t)stream_;
    const double m = q->m, n = q->n, k = q->k;
    sgv_launch_scope scope(SGV_K_INT8_GEMM, stream, m * k + n * k + m * n * (double)sgv_dtype_size(dtype), 2.0 * m * n * k);
    if (dtype == SGV_F32) sgv_i8::launch<float>(p, pl, q->workspace, stream);
    else if (dtype == SGV_F16) sgv_i8::launch<sgv_half_t>(p, pl, q->workspace, stream);
    else sgv_i8::launch<sgv_bf16_t>(p, pl, q->workspace, stream);
    return sgv_check_launch("int8_gemm kernel");
}
