// Matrix product in 8-bit integers with one scale per row of either operand (sgv_int8_gemm):
//
//   C[m,n] = act( (sum_k A[m,k] B[n,k]) * a_scale[m] * b_scale[n] + bias[n] ) * gain        A [M,K], B [N,K] signed bytes, sums in 32-bit integers
//
// Both operands are contiguous along k, which is how the matrix instruction wants them: a lane of v_mfma_i32_16x16x64_i8 holds 16 consecutive bytes of one row
// (row = lane & 15, bytes 16 (lane >> 4) ..+15 of 64).  The integer sums are exact whatever their order, so K is split freely over the waves of a workgroup, and the result
// depends neither on the split nor on the other rows of a batch.
//
// Two kernels: int8_rows_kernel for few rows (bound by reading B once: 1 x 8192 x 8192 12.3 us = 5.4 TB/s) and few tiles, int8_tile_kernel for the rest (bound by the matrix
// pipe and its power: 8192^3 takes 750 to 800 thousand clocks, 0.65 to 0.70 of the issue slots busy; 413 us = 2,660 TOP/s on a cool chip at 1.85 GHz, 490 us = 2,240 where
// ten launches in a row have brought it down to 1.53 GHz, 420 us in the long run).  The table at choose() below has both sides of every border.
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

// (the scale of B first: a weight's is moderate, and rows of any size then leave fp32's range only where the result does)
__device__ __forceinline__ float finish(const args& p, int acc, float sa, float sb, float bias) {
    float v = __builtin_fmaf((float)acc * sb, sa, bias);
    if (p.lrelu) v = v > 0.f ? v : v * p.alpha;
    return v * p.gain;
}

// ---------------------------------------------------------------------------------------------------------------------------------------
// Tiles of C.  K is walked in stages of 128 bytes per row -- a cache line -- that go from memory straight into LDS (buffer_load ... lds: no registers, no instructions
// to store them), S stages in a ring.  A stage's 16-byte chunks lie at position chunk ^ ((row >> 1) & 7) of their row, which makes the fragment reads below free of
// bank conflicts.  A wave holds the fragments of one step of 64 k in registers and replaces each as soon as its last product is issued, so that the matrix pipe finds
// the next step's fragments there; one barrier per stage.  (16x16x64 rather than 32x32x32 products: half the accumulator traffic for the same work, 5 % of the time at
// 8192^3, where time is energy.  128 bytes of K per stage rather than 64: whole cache lines, another 5 %.)  Rows beyond the matrix and bytes beyond its end are outside the buffers' bounds and read as zero.

__device__ __forceinline__ i32x4 make_rsrc(const void* base, int64_t bytes) {
    const uint64_t b = (uint64_t)base;
    return i32x4{(int)(unsigned)b, (int)((unsigned)(b >> 32) & 0xffffu), (int)(unsigned)(bytes > 0xffffffffll ? 0xffffffffll : bytes), 0x00020000};
}
// 16 bytes per lane from rsrc + voff + soff to LDS at lds + 16 lane.  In inline assembly because the compiler waits for ALL outstanding loads in front of any LDS read behind
// the builtin; nothing lands in a register, and the kernel counts these loads itself (s_waitcnt vmcnt).
__device__ __forceinline__ void dma16(i32x4 rsrc, unsigned lds, unsigned voff, int soff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" :: "s"(lds), "v"(voff), "s"(rsrc), "s"(soff) : "memory");
}

// ---------------------------------------------------------------------------------------------------------------------------------------
// Few tiles: every wave of a workgroup computes the whole 16 MT x 16 NT tile over its own stages of K (128 bytes per row; wave w takes stages w, w + waves, ...), in a
// ring of S stages of LDS of its own -- no barrier in the loop --, and the waves' sums meet in LDS.  Through LDS because the matrix instruction wants 16 rows side by side:
// read straight into registers, 16 neighbouring lanes touch 16 cache lines, and a CU gets 16 bytes a clock instead of 64 (32 x 512 x 8192: 13.0 us against 5.6).
template <typename T, int MT, int NT, int S>
__global__ __launch_bounds__(512) void int8_rows_kernel(const args p) {
    extern __shared__ __attribute__((aligned(128))) int8_t ring[];          // [waves][S][(MT + NT) * 16 rows][128], then [waves][MT * NT * 256] sums
    constexpr int STAGE = (MT + NT) * 2048, LPS = 2 * (MT + NT);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int n0 = blockIdx.x * (16 * NT), m0 = blockIdx.y * (16 * MT), k16 = (p.k + 15) & ~15;
    const int quarter = lane >> 4, r = lane & 15;
    const i32x4 ra = make_rsrc(p.a + (int64_t)m0 * p.lda, (int64_t)(p.m - 1 - m0) * p.lda + k16);
    const i32x4 rb = make_rsrc(p.b + (int64_t)n0 * p.ldb, (int64_t)(p.n - 1 - n0) * p.ldb + k16);
    const i32x4 none = make_rsrc(p.a, 0);
    unsigned va[2 * MT], vb[2 * NT];
#pragma unroll
    for (int i = 0; i < 2 * MT; i++) { const int row = i * 8 + (lane >> 3); va[i] = row * (unsigned)p.lda + ((lane & 7) ^ ((row >> 1) & 7)) * 16; }
#pragma unroll
    for (int i = 0; i < 2 * NT; i++) { const int row = i * 8 + (lane >> 3); vb[i] = row * (unsigned)p.ldb + ((lane & 7) ^ ((row >> 1) & 7)) * 16; }
    const int nst = (p.k + 127) / 128;
    int8_t* mine = ring + wave * S * STAGE;
    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) int8_t*)mine;
    auto issue = [&](int t, int slot) {
        const unsigned s = lds0 + slot * STAGE;
        const int k0 = t < nst ? t * 128 : 0;
        const i32x4 xa = t < nst ? ra : none, xb = t < nst ? rb : none;
#pragma unroll
        for (int i = 0; i < 2 * NT; i++) dma16(xb, s + i * 1024, vb[i], k0);
#pragma unroll
        for (int i = 0; i < 2 * MT; i++) dma16(xa, s + NT * 2048 + i * 1024, va[i], k0);
    };
    i32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) acc[i][j] = i32x4{0, 0, 0, 0};
#pragma unroll
    for (int u = 0; u < S; u++) issue(wave + u * waves, u);
    const int base = r * 128, c0 = (quarter ^ ((r >> 1) & 7)) * 16, c1 = ((4 + quarter) ^ ((r >> 1) & 7)) * 16;
    int slot = 0;
    for (int t = wave; t < nst; t += waves) {
        asm volatile("s_waitcnt vmcnt(%0)" :: "n"((S - 1) * LPS) : "memory");
        const int8_t* s = mine + slot * STAGE + base;
        i32x4 f[2][MT + NT];
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < MT + NT; i++) f[h][i] = *(const i32x4*)(s + i * 2048 + (h ? c1 : c0));
        const int left = p.k - t * 128;
        if (left < 128) {
#pragma unroll
            for (int j = 0; j < NT; j++) { f[0][j] = mask_tail(f[0][j], left - quarter * 16); f[1][j] = mask_tail(f[1][j], left - 64 - quarter * 16); }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                // (the stage is in registers: its slot may be written over)
        issue(t + S * waves, slot);
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int j = 0; j < NT; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[h][NT + i], f[h][j], acc[i][j], 0, 0, 0);
        slot = slot + 1 == S ? 0 : slot + 1;
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __syncthreads();
    // D layout of the instruction: column = lane & 15, row = 4 * (lane >> 4) + e
    int* red = (int*)ring;
    constexpr int TILE = MT * NT * 256;
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) red[wave * TILE + (i * 16 + quarter * 4 + e) * (NT * 16) + j * 16 + r] = acc[i][j][e];
    __syncthreads();
    for (int x = threadIdx.x; x < TILE; x += blockDim.x) {
        const int m = m0 + x / (NT * 16), n = n0 + x % (NT * 16);
        if (m >= p.m || n >= p.n) continue;
        int sum = red[x];
        for (int w = 1; w < waves; w++) sum += red[w * TILE + x];
        sgv_traits<T>::store((T*)p.c + (int64_t)m * p.ldc + n, finish(p, sum, p.a_scale[m], p.b_scale[n], p.bias ? p.bias[n] : 0.f));
    }
}

// four consecutive columns as they are stored
template <typename T> struct quad;
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
    const int k = p.k, k16 = (k + 15) & ~15;
    const i32x4 ra = make_rsrc(p.a + (int64_t)m0 * p.lda, (int64_t)(p.m - 1 - m0) * p.lda + k16);
    const i32x4 rb = make_rsrc(p.b + (int64_t)n0 * p.ldb, (int64_t)(p.n - 1 - n0) * p.ldb + k16);
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
#pragma unroll
    for (int i = 0; i < TM; i++) { const int m = m0 + (wm * TM + i) * 16 + r; sa[i] = m < p.m ? p.a_scale[m] : 0.f; }
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int x = i * 64 * WAVES + threadIdx.x, n = n0 + x;
        const bool ok = x < BN && n < p.n;
        sbv[i] = ok ? p.b_scale[n] : 0.f;
        biv[i] = ok && p.bias ? p.bias[n] : 0.f;
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
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"((S - 2) * LPS) : "memory");
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
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" :: "n"((S - 1) * LPS) : "memory");
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
#pragma unroll
    for (int i = 0; i < PER; i++) { const int x = i * 64 * WAVES + threadIdx.x; if (x < BN) { sb_lds[x] = sbv[i]; bias_lds[x] = biv[i]; } }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");      // (every load into LDS has landed, the empty ones too: the ring may be written over)
    int8_t* buf = lds + wave * 16 * PITCH;
    const int nb = n0 + wn * TN * 16;
    const bool whole = m0 + BM <= p.m && n0 + BN <= p.n;
#pragma unroll
    for (int i = 0; i < TM; i++) {
#pragma unroll
        for (int j = 0; j < TN; j++) {
            const int x = j * 16 + 4 * quarter;
            const f32x4 s4 = *(const f32x4*)(sb_lds + wn * TN * 16 + x), b4 = *(const f32x4*)(bias_lds + wn * TN * 16 + x);
            *(typename quad<T>::type*)(buf + r * PITCH + x * ES) = quad<T>::make(p, acc[i][j], sa[i], s4, b4);
        }
        const int mb = m0 + (wm * TM + i) * 16;
#pragma unroll
        for (int q = 0; q < 16 * CH / 64; q++) {
            const int idx = q * 64 + lane, rr = idx / CH, ch = idx % CH, n = nb + ch * PCS;
            T* o = (T*)p.c + (int64_t)(mb + rr) * p.ldc + n;
            const i32x4 v = *(const i32x4*)(buf + rr * PITCH + ch * 16);
            if (whole || (mb + rr < p.m && n + PCS <= p.n)) ((any_i32x4*)o)->v = v;
            else if (mb + rr < p.m)
                for (int x = 0; n + x < p.n; x++) o[x] = ((const T*)(buf + rr * PITCH + ch * 16))[x];
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------------------------
// Which form serves a product (microseconds in a replayed graph, operands rotating through 3 sets, bf16 out):
//                            m x n x k           rows kernel   64^2 tiles   128^2    256^2
//   few rows                 32 x 512 x 8192         5.6           -          -        -        16 x 8192 x 8192: 13.4 (5.1 TB/s), 1 x 8192 x 8192: 12.3 (5.4 TB/s)
//   few tiles, a long k     100 x 512 x 2048         4.7          6.2         9.1     24.3
//                           512 x 512 x 2048         4.9          6.4         9.3     24.1
//   ... a short k           256 x 512 x 512          4.0          3.7         5.1     11.7
//   some tiles              777 x 1001 x 1030       14.0          5.4         8.0     19.7
//                           128 x 4096 x 4096       13.1          9.9        22.3     41.2
//   about a tile per CU    1500 x 1500 x 1500       37.1         13.4        13.3     27.1
//                          2048 x 2048 x 2048       65.3         17.5        14.6     26.2
//   many                  10007 x 512 x 512         38.4         11.4         8.8     13.7
//                          4096 x 4096 x 4096         -          106          69       56
//                          8192 x 8192 x 8192         -          850         535      420      (2,615 TOP/s)
enum form { ROWS11, ROWS21, ROWS22, TILE64, TILE128, TILE256 };      // (in the order of their names in SGV_VARIANTS)

static inline int64_t tiles(int m, int n, int em, int en) { return ((int64_t)(m + em - 1) / em) * ((n + en - 1) / en); }

static form choose(int m, int n, int k) {
    // few rows: B is read once by as many workgroups as there are; 32 rows take 32 columns where 16 would mean more than one workgroup per CU
    if (m <= 16) return ROWS11;
    if (m <= 32) return tiles(m, n, 32, 16) <= 256 ? ROWS21 : ROWS22;
    // few tiles: the time is the K loop of one of them, which eight waves split
    if (tiles(m, n, 32, 32) <= 256 && k >= 1024) return ROWS22;
    // 256 CUs hold two 128^2 tiles each, or one 256^2 tile at 1.6 times the time of two
    const int64_t t128 = tiles(m, n, 128, 128), t256 = tiles(m, n, 256, 256);
    if (t128 < 150) return TILE64;
    return (t256 + 255) / 256 * 1.6 <= (double)((t128 + 511) / 512) ? TILE256 : TILE128;
}

template <typename T, int MT, int NT, int S>
static void launch_rows(const args& p, int waves, hipStream_t stream) {
    const dim3 grid((unsigned)((p.n + 16 * NT - 1) / (16 * NT)), (unsigned)((p.m + 16 * MT - 1) / (16 * MT))), block(64 * waves);
    const size_t lds = (size_t)waves * std::max(S * (MT + NT) * 2048, MT * NT * 1024);
    hipLaunchKernelGGL((int8_rows_kernel<T, MT, NT, S>), grid, block, lds, stream, p);
}

template <typename T, int BM, int BN, int WGM, int WGN, int S, int LEAD>
static void launch_tile(args p, hipStream_t stream) {
    p.tiles_m = (p.m + BM - 1) / BM;
    p.tiles_n = (p.n + BN - 1) / BN;
    hipLaunchKernelGGL((int8_tile_kernel<T, BM, BN, WGM, WGN, S, LEAD>), dim3((unsigned)(p.tiles_m * p.tiles_n)), dim3(64 * WGM * WGN), 0, stream, p);
}

template <typename T>
static void launch(const args& p, form f, hipStream_t stream) {
    switch (f) {
        case ROWS11: launch_rows<T, 1, 1, 2>(p, std::min(4, (p.k + 127) / 128), stream); break;
        case ROWS21: launch_rows<T, 2, 1, 2>(p, std::min(8, (p.k + 127) / 128), stream); break;
        case ROWS22: launch_rows<T, 2, 2, 2>(p, std::min(8, (p.k + 127) / 128), stream); break;
        case TILE64: launch_tile<T, 64, 64, 2, 2, 4, 1>(p, stream); break;
        case TILE128: launch_tile<T, 128, 128, 2, 4, 2, 1>(p, stream); break;
        case TILE256: launch_tile<T, 256, 256, 2, 4, 2, 2>(p, stream); break;
    }
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
    if (q->lda >= 1 << 23 || q->ldb >= 1 << 23) return sgv_fail(SGV_ERR_TOO_LARGE, "int8_gemm: rows are at most 8 MB apart (offsets inside a tile are 32 bits)");
    const sgv_i8::form f = sgv_i8::choose(q->m, q->n, q->k);
    // (a launch has fewer than 2^32 threads)
    const int64_t threads = f == sgv_i8::ROWS11 ? sgv_i8::tiles(q->m, q->n, 16, 16) * 256 : f <= sgv_i8::ROWS22 ? sgv_i8::tiles(q->m, q->n, 32, 16) * 512
                          : f == sgv_i8::TILE64 ? sgv_i8::tiles(q->m, q->n, 64, 64) * 256 : sgv_i8::tiles(q->m, q->n, f == sgv_i8::TILE128 ? 128 : 256, f == sgv_i8::TILE128 ? 128 : 256) * 512;
    if (threads >= 1ll << 32) return sgv_fail(SGV_ERR_TOO_LARGE, "int8_gemm: too many tiles");
    sgv_i8::args p{};
    p.a = (const int8_t*)q->a; p.b = (const int8_t*)q->b; p.a_scale = q->a_scale; p.b_scale = q->b_scale; p.bias = q->bias; p.c = q->c;
    p.lda = q->lda; p.ldb = q->ldb; p.ldc = q->ldc; p.m = q->m; p.n = q->n; p.k = q->k;
    p.lrelu = q->act == 3; p.alpha = q->alpha; p.gain = q->gain;
    hipStream_t stream = (hipStream_t)stream_;
    const double m = q->m, n = q->n, k = q->k;
    sgv_launch_scope scope(SGV_K_INT8_GEMM, stream, m * k + n * k + m * n * (double)sgv_dtype_size(dtype), 2.0 * m * n * k);
    sgv_note_variant(SGV_V_int8_rows_16x16 + f);
    if (dtype == SGV_F32) sgv_i8::launch<float>(p, f, stream);
    else if (dtype == SGV_F16) sgv_i8::launch<sgv_half_t>(p, f, stream);
    else sgv_i8::launch<sgv_bf16_t>(p, f, stream);
    return sgv_check_launch("int8_gemm kernel");
}
