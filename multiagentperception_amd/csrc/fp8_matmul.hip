// Matrix product of e4m3 codes with a power-of-two (e8m0) scale per 128 elements of the reduction, and the quantiser that makes them.
//
//   C[m][n] = sum_k  a[m][k] 2^ea(m, k / 128)  b[n][k] 2^eb(n, k / 128)  (+ bias[n])
//
// Rows are stored padded with zero codes to a multiple of 128.  A scale belongs to one row's 128 (activations, gradients) or to a 128 x 128 tile
// (weights: the transposed weights then have the same codes and scales).  Within a block of 128 the order of k is free as long as both
// operands agree, since its scale is one.
//
// Products are summed in 32 bits: a code times its scale is a bf16 number exactly (one conversion instruction per pair does both; beyond f32's range it is
// infinite, below 2^-126 a multiple of 2^-133), and the bf16 matrix instructions add exact products of those to an f32 accumulator: 4e-8 of the
// result's norm, 8192^3 to bf16 in 769 us = 1.43 PFLOP/s (FAST: 1.5e-5, 459 us).
// FAST, for outputs of 16 bits and callers that ask for it, feeds the codes to gfx950's scaled matrix instructions, which multiply by both e8m0
// scales themselves at twice the rate.  They line the products of 8 neighbouring k up to the largest of them and keep 13 bits below it (measured: a
// product 2^-14 of the largest is lost, in the next group of 8 it is not).  On normal data that is about 1.5e-5 of the result's norm, and
// an element whose sum cancels can lose all its digits.
//
//   tile kernels   at least 25 rows: TM x TN tiles, both operands by LDS-DMA into a ring of four stages of 64 k
//   row kernel     up to 24 rows (tokens being decoded): bound by reading b once; no LDS for operands, the waves of a block split k
#include "lm_common.h"

namespace {

typedef unsigned char u8;
constexpr int KT = 128;                       // elements of the reduction per scale
// The longest reduction is the most rows that the quantiser takes (its tiles of rows are a grid's second dimension): a gradient of weights sums over them.
// 256 rows of it are 2^31 bytes at most, within a descriptor and its 32-bit offsets.
constexpr int ROW_TILES = 65535, K_MOST = ROW_TILES * KT;
// The row kernel reads all of a once per 16 columns, the tile kernels multiply 128 rows whatever there are.  us to bf16, row / tile kernels: 16384 x 8192
// weights with 16 rows 35.6 / 40.2, 20 41.4 / 38.4, 24 44.8 / 38.9, 32 50.8 / 39.3; 1024 x 8192 with 16 10.2 / 12.0, 24 13.0 / 12.2, 32 14.5 / 12.2; 4096 x 4096
// with 16 9.2 / 11.3, 24 10.7 / 11.5, 32 11.8 / 11.9.
constexpr int ROWS_MOST = 24;

// four scale bytes (k blocks kb .. kb + 3) of a row; bytes past the row's end are not read, and not used
__device__ __forceinline__ uint32_t scales4(const u8* p, int kb, int KB) {
    uint32_t v = 0;
    if (KB >= 4) {
        const int k = kb < KB - 4 ? kb : KB - 4;
        __builtin_memcpy(&v, p + k, 4);
        return v >> (8 * (kb - k));
    }
    for (int i = kb; i < KB; ++i) v |= (uint32_t)p[i] << (8 * (i - kb));
    return v;
}

struct Product {
    const u8 *a, *sa, *b, *sb;
    const float* bias;
    void* c;
    int M, N, K;                              // K: padded to 128
    int parts;                                // > 1: the reduction is cut into that many parts of whole groups of four blocks (blockIdx.y)
    float* part;                              // [parts][M][N] of them, added up by sum_splits_kernel
    int a_shift, b_shift;                     // row of the scales = row >> shift: 0 or 7
};

__device__ __forceinline__ void dma16(unsigned dst, unsigned voff, u32x4_t srd, unsigned soff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(dst), "v"(voff), "s"(srd), "s"(soff) : "memory", "m0");
}
__device__ __forceinline__ u32x4_t descriptor(const u8* p, unsigned bytes) {       // reads past `bytes` give 0
    const unsigned long long a = reinterpret_cast<unsigned long long>(p);
    return u32x4_t{(unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)a), (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(a >> 32)),
                   (unsigned)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
}

// 16 codes of a row (four bytes each of w), scaled: two operands of the bf16 instructions (8 k each).  The conversion takes the scale's
// exponent field as it is, so a scale byte in that place needs no more than a shift.
__device__ __forceinline__ bf16x8_t scaled8(uint32_t lo, uint32_t hi, float s) {
    const w2c_bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true);
    const w2c_bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true);
    return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ void dma4(unsigned dst, unsigned voff, u32x4_t srd, unsigned soff) {       // a dword per lane
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds" ::"s"(dst), "v"(voff), "s"(srd), "s"(soff) : "memory", "m0");
}
__device__ __forceinline__ void dma1(unsigned dst, unsigned voff, u32x4_t srd, unsigned soff) {       // a byte per lane, into a dword of LDS
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_ubyte %1, %2, %3 offen lds" ::"s"(dst), "v"(voff), "s"(srd), "s"(soff) : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void wait_pieces() {               // at most N of this wave's LDS-DMA pieces are still under way; its LDS reads are done
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// A ring of four stages of 64 k.  Step t multiplies stage t, whose operands are in registers already, reads stage t + 1's from LDS and sends for stage
// t + 4, into the buffer of stage t (its reads were done before the barrier at the top of step t).  So a stage has three steps to arrive, and neither
// its arrival nor an LDS read stands between the matrix instructions of two steps.  The scales of a block of 128 come with its first stage, into a
// dword of LDS per row: four blocks' together where rows of scales are whole dwords (every row is a cache line of its own to the address unit:
// 8192^3 FAST to bf16 523 us with a byte per block, 512 with a dword per four; the bf16 instructions, at half the rate, lose 4 % by the branch and do without).
// Stage image: row r (64 bytes) at 64 r, its 16-byte chunk c in slot c ^ ((r >> 2) & 3): 16 neighbouring rows' same chunk then cover all 64 banks once.
// A piece of LDS-DMA is 16 rows (64 lanes x 16 bytes, contiguous in LDS); the swizzle is in the source address.
template <typename T, bool FAST, int TM, int TN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64, 1) void matmul_tile_kernel(Product p, int tiles_m, int tiles_n) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int NW = WM * WN, MI = TM / WM / 32, NI = TN / WN / 32, PA = TM / 16 / NW, PB = TN / 16 / NW, HALF = KT / 2;
    constexpr int PS = ((TM + TN) / 64 + NW - 1) / NW;         // pieces of 64 rows of scales, at most, of a wave
    constexpr unsigned STAGE = (TM + TN) * HALF, SCALES = 4 * STAGE, SBUF = (TM + TN) * 4;
    extern __shared__ __attribute__((aligned(1024))) u8 smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l31 = lane & 31, lhi = lane >> 5;
    // tiles in groups of 8 tile rows, walked column by column: the 32 tiles in flight on an XCD share 8 row panels and 4 column panels
    int m0, n0;
    {
        const int id = xcd_remap(blockIdx.x, tiles_m * tiles_n), per = 8 * tiles_n, g = id / per, r = id - g * per;
        const int rows = tiles_m - 8 * g < 8 ? tiles_m - 8 * g : 8;
        m0 = (8 * g + r % rows) * TM;
        n0 = (r / rows) * TN;
    }
    const int ml = p.M - m0 < TM ? p.M - m0 : TM, nl = p.N - n0 < TN ? p.N - n0 : TN, KB = p.K / KT;
    const int k0 = p.parts > 1 ? (KB + 3) / 4 * (int)blockIdx.y / p.parts * 4 : 0;
    const int k1 = p.parts > 1 && (int)blockIdx.y + 1 < p.parts ? (KB + 3) / 4 * ((int)blockIdx.y + 1) / p.parts * 4 : KB, steps = 2 * (k1 - k0);
    const u32x4_t srd_a = descriptor(p.a + (long long)m0 * p.K, (unsigned)ml * (unsigned)p.K);
    const u32x4_t srd_b = descriptor(p.b + (long long)n0 * p.K, (unsigned)nl * (unsigned)p.K);
    const unsigned lds = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(size_t)W2C_LPTR(smem));
    const int prow = wave * 16 + (lane >> 2), pchunk = (lane & 3) ^ ((lane >> 4) & 3);
    const unsigned voff = (unsigned)prow * (unsigned)p.K + (unsigned)pchunk * 16u, vstep = (unsigned)(NW * 16) * (unsigned)p.K;
    u32x4_t srd_s[PS];
    unsigned svoff[PS];
#pragma unroll
    for (int i = 0; i < PS; ++i) {                            // a piece's 64 rows are rows of a or of b; rows past the last repeat it
        const int q = wave + NW * i;
        const bool of_a = q < TM / 64;
        const int row = (of_a ? m0 : n0 - TM) + q * 64 + lane, last = (of_a ? p.M : p.N) - 1, shift = of_a ? p.a_shift : p.b_shift;
        const int first = (of_a ? m0 : n0) >> shift, count = (last >> shift) + 1 - first;
        srd_s[i] = descriptor((of_a ? p.sa : p.sb) + (long long)first * KB, (unsigned)(count < TM + TN ? count : TM + TN) * (unsigned)KB);
        svoff[i] = (unsigned)(((row < last ? row : last) >> shift) - first) * (unsigned)KB;
    }
    const bool packed = FAST && (KB & 3) == 0 && ((reinterpret_cast<uintptr_t>(p.sa) | reinterpret_cast<uintptr_t>(p.sb)) & 3) == 0;
    // piece i of stage t: scales first (a stage pair's come with its even one), then a's rows, then b's.  Behind the last stage the last is sent
    // again, into buffers that nothing reads any more: every step then has the same pieces to wait for.
    auto send = [&](int t, int i, bool with_scales) {
        const int u = t < steps ? t : steps - 1;
        const unsigned dst = lds + (unsigned)(t & 3) * STAGE + (unsigned)wave * 1024u, soff = (unsigned)(k0 * 2 + u) * HALF;
        if (with_scales) {
            if (i < PS) {
                if constexpr ((TM + TN) / 64 % NW != 0)
                    if (wave + NW * i >= (TM + TN) / 64) return;
                const unsigned to = lds + SCALES + (unsigned)(wave + NW * i) * 256u;
                if (!packed) dma1(to + (unsigned)((t >> 1) & 1) * SBUF, svoff[i], srd_s[i], (unsigned)(k0 + (u >> 1)));
                else if (!(t & 7)) dma4(to + (unsigned)((t >> 3) & 1) * SBUF, svoff[i], srd_s[i], (unsigned)(k0 + (u >> 1)) & ~3u);
                return;
            }
            i -= PS;
        }
        if (i < PA) dma16(dst + i * NW * 1024u, voff + i * vstep, srd_a, soff);
        else dma16(dst + TM * HALF + (i - PA) * NW * 1024u, voff + (i - PA) * vstep, srd_b, soff);
    };
    constexpr int EACH = PA + PB, TWO = 2 * EACH + (FAST ? 0 : (TM + TN) / 64 / NW);      // pieces of a stage, and what two neighbours have at least
    const int wm = (wave % WM) * (TM / WM), wn = (wave / WM) * (TN / WN);
    // a lane's 32 bytes of a stage: chunks 2 lhi, 2 lhi + 1 of rows l31 of its fragments
    const int key = (l31 >> 2) & 3, s0 = (((2 * lhi) ^ key) << 4), s1 = (((2 * lhi + 1) ^ key) << 4);
    const u8* ra = smem + (wm + l31) * HALF;
    const u8* rb = smem + (TM + wn + l31) * HALF;
    struct Operands {
        u32x4_t a[MI][2], b[NI][2];
    };
    constexpr int READS = 2 * (MI + NI), SREADS = MI + NI, QUARTERS = FAST ? 1 : 4, MULTS = MI * NI * QUARTERS;
    auto read = [&](Operands& f, unsigned buf, int i) {       // one of READS: b's fragments first
        const int k = i >> 1, h = i & 1;
        if (k < NI) f.b[k][h] = *reinterpret_cast<const u32x4_t*>(rb + buf + (h ? s1 : s0) + k * 32 * HALF);
        else f.a[k - NI][h] = *reinterpret_cast<const u32x4_t*>(ra + buf + (h ? s1 : s0) + (k - NI) * 32 * HALF);
    };
    struct Scales {
        int a[MI], b[NI];
    };
    auto read_scales = [&](Scales& x, int kb, int i) {
        const int* s = reinterpret_cast<const int*>(smem + SCALES + ((packed ? kb >> 2 : kb) & 1) * SBUF) + l31;
        int v = s[i < NI ? TM + wn + i * 32 : wm + (i - NI) * 32] >> (packed ? 8 * (kb & 3) : 0);      // the scaled instructions take the lowest byte,
        if constexpr (!FAST) v = (v & 255) << 23;                                                   // the conversion a float's exponent field
        if (i < NI) x.b[i] = v;
        else x.a[i - NI] = v;
    };
    f32x16_t acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    auto multiply = [&](const Operands& f, const Scales& x, int q, int i, int j) {
        if constexpr (!FAST) {                                // 16 k: a quarter of the stage
            const bf16x8_t fb = scaled8(f.b[j][q >> 1][2 * (q & 1)], f.b[j][q >> 1][2 * (q & 1) + 1], __int_as_float(x.b[j]));
            const bf16x8_t fa = scaled8(f.a[i][q >> 1][2 * (q & 1)], f.a[i][q >> 1][2 * (q & 1) + 1], __int_as_float(x.a[i]));
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fb, fa, acc[i][j], 0, 0, 0);
        } else
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(cat_i32x8(f.b[j][0], f.b[j][1]), cat_i32x8(f.a[i][0], f.a[i][1]), acc[i][j], 0, 0, 0,
                                                                        x.b[j], 0, x.a[i]);
    };
    // step t: multiply `now`, read stage t + 1 into `next`, send stage t + 4.  Reads and pieces are spread between the matrix instructions: in one go they
    // would hold up the only wave of the SIMD for as long as the LDS and the address unit take for all four waves' (8192^3 FAST to bf16: 721 us against 603).
    // What is left of FAST is bound by power: the same product of zeros takes 360 us, of random codes 515; matrix instructions alone reach 3.7 PFLOP/s on
    // random codes.
    auto step = [&](const Operands& now, Operands& next, const Scales& x, Scales& x_next, int t, bool second) {
        const unsigned buf = (unsigned)((t + 1) & 3) * STAGE;
        const int pieces = EACH + (second ? 0 : PS), reads = READS + (second ? SREADS : 0);
#pragma unroll
        for (int q = 0; q < QUARTERS; ++q)
#pragma unroll
        for (int ij = 0; ij < MI * NI; ++ij) {
            const int m = q * MI * NI + ij;
#pragma unroll
            for (int i = m * reads / MULTS; i < (m + 1) * reads / MULTS; ++i) {
                if (i < READS) read(next, buf, i);
                else read_scales(x_next, (t + 1) >> 1, i - READS);
            }
#pragma unroll
            for (int i = m * pieces / MULTS; i < (m + 1) * pieces / MULTS; ++i) send(t + 4, i, !second);
            multiply(now, x, q, ij / NI, ij % NI);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < EACH + (t & 1 ? 0 : PS); ++i) send(t, i, !(t & 1));
    wait_pieces<EACH + TWO>();
    Operands even, odd;
    Scales x, x_next;
#pragma unroll
    for (int i = 0; i < READS; ++i) read(even, 0, i);
#pragma unroll
    for (int i = 0; i < SREADS; ++i) read_scales(x, 0, i);
    for (int t = 0; t < steps; t += 2) {
        wait_pieces<TWO>();                                   // stage t + 1 has landed everywhere
        step(even, odd, x, x_next, t, false);
        wait_pieces<TWO>();                                   // stage t + 2
        step(odd, even, x, x_next, t + 1, true);
        x = x_next;
    }
    // The accumulators of a fragment row (32 rows of the wave's part) go through LDS, f32, so that whole lines of c are written: stored as they lie,
    // 8 bytes of each of 32 rows at a time, the epilogue took 28 us a tile.  Accumulator e of a lane: column (e & 3) + 8 (e >> 2) + 4 lhi, row l31 of its
    // 32 x 32.  (The ring's last pieces are waited for: they may not land in this.)
    wait_pieces<0>();
    constexpr int COLS = TN / WN, PITCH = COLS + 4, VEC = ElemOf<T>::VEC, LANES = COLS / VEC, ROWS = 64 / LANES;
    static_assert(NW * 32 * PITCH * 4 <= 4 * STAGE, "the epilogue fits the ring");
    float* mine = reinterpret_cast<float*>(smem) + wave * 32 * PITCH;
    const int col = lane % LANES * VEC, n = n0 + wn + col, left = p.N - n;
    const bool whole = m0 + TM <= p.M && n0 + TN <= p.N;
    float bias[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) bias[e] = p.bias && p.parts == 1 && e < left ? p.bias[n + e] : 0.f;
    T* C = (T*)p.c;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<f32x4_t*>(mine + l31 * PITCH + j * 32 + 8 * q + 4 * lhi) =
                    f32x4_t{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");    // the wave's own: nobody else reads or writes them
#pragma unroll
        for (int r = 0; r < 32; r += ROWS) {
            const int row = r + lane / LANES, m = m0 + wm + i * 32 + row;
            float v[VEC];
#pragma unroll
            for (int e = 0; e < VEC; e += 4) {
                const f32x4_t w = *reinterpret_cast<const f32x4_t*>(mine + row * PITCH + col + e);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[e + k] = w[k] + bias[e + k];
            }
            const long long at = (long long)m * p.N + n;
            if (p.parts > 1) {
                if (m < p.M) store_part<float, VEC>(p.part + (long long)blockIdx.y * p.M * p.N + at, left, v);
            } else if (whole) store_n<T, VEC>(C + at, v);
            else if (m < p.M) store_part<T, VEC>(C + at, left, v);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
#endif
}

// c = the parts' sum, in part order, + bias; four columns of a row per thread
template <typename T>
__global__ __launch_bounds__(256) void sum_splits_kernel(Product p) {
    const long long groups = (p.N + 3) / 4, i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= groups * p.M) return;
    const long long m = i / groups;
    const int n = (int)(i - m * groups) * 4, left = p.N - n;
    const float* q = p.part + m * p.N + n;
    float v[4], w[4];
    load_part<float, 4>(q, left, v);
    for (int k = 1; k < p.parts; ++k) {
        load_part<float, 4>(q + (long long)k * p.M * p.N, left, w);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += w[e];
    }
    if (p.bias) {
        load_part<float, 4>(p.bias + n, left, w);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += w[e];
    }
    store_part<T, 4>((T*)p.c + m * p.N + n, left, v);
}

// At most 16 MT rows of a against 16 rows of b per block; wave w takes its share of the k blocks, the partial tiles are added in wave order.
template <typename T, bool FAST, int MT, int NW>
__global__ __launch_bounds__(NW * 64) void matmul_rows_kernel(Product p) {
#if defined(__HIP_DEVICE_COMPILE__)
    __shared__ float part[NW][MT][256];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, grp = lane >> 4, KB = p.K / KT;
    const int n0 = blockIdx.x * 16, n = n0 + r16 < p.N ? n0 + r16 : p.N - 1;
    const int lo = (int)((long long)KB * wave / NW), hi = (int)((long long)KB * (wave + 1) / NW);
    const u8* pb = p.b + (long long)n * p.K + grp * 16;               // a lane's 32 bytes of a block: chunks grp and grp + 4
    const u8* psb = p.sb + (long long)(n >> p.b_shift) * KB;
    f32x4_t acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    const u8 *pa[MT], *psa[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int m = t * 16 + r16 < p.M ? t * 16 + r16 : p.M - 1;    // rows past the last repeat it; their results are not stored
        pa[t] = p.a + (long long)m * p.K + grp * 16;
        psa[t] = p.sa + (long long)(m >> p.a_shift) * KB;
    }
    for (int k0 = lo; k0 < hi; k0 += 4) {
        const int kn = hi - k0 < 4 ? hi - k0 : 4;
        u32x4_t b0[4], b1[4];
        uint32_t sb = scales4(psb, k0, KB), sa[MT];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const long long o = (long long)(k0 + (u < kn ? u : 0)) * KT;
            b0[u] = *reinterpret_cast<const u32x4_t*>(pb + o);
            b1[u] = *reinterpret_cast<const u32x4_t*>(pb + o + 64);
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) sa[t] = scales4(psa[t], k0, KB);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (u >= kn) break;
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const u8* q = pa[t] + (long long)(k0 + u) * KT;
                const u32x4_t a0 = *reinterpret_cast<const u32x4_t*>(q), a1 = *reinterpret_cast<const u32x4_t*>(q + 64);
                if constexpr (!FAST) {
                    const float xa = __uint_as_float((sa[t] >> (8 * u) & 255u) << 23), xb = __uint_as_float((sb >> (8 * u) & 255u) << 23);
                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(scaled8(b0[u][0], b0[u][1], xb), scaled8(a0[0], a0[1], xa), acc[t], 0, 0, 0);
                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(scaled8(b0[u][2], b0[u][3], xb), scaled8(a0[2], a0[3], xa), acc[t], 0, 0, 0);
                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(scaled8(b1[u][0], b1[u][1], xb), scaled8(a1[0], a1[1], xa), acc[t], 0, 0, 0);
                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(scaled8(b1[u][2], b1[u][3], xb), scaled8(a1[2], a1[3], xa), acc[t], 0, 0, 0);
                } else
                    acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(cat_i32x8(b0[u], b1[u]), cat_i32x8(a0, a1), acc[t], 0, 0, 0,
                                                                             (int)(sb >> (8 * u)), 0, (int)(sa[t] >> (8 * u)));
            }
        }
    }
    // lane: row m = r16 of a, columns n0 + 4 grp + e
#pragma unroll
    for (int t = 0; t < MT; ++t) *reinterpret_cast<f32x4_t*>(&part[wave][t][lane * 4]) = acc[t];
    __syncthreads();
    T* C = (T*)p.c;
    for (int t = wave; t < MT; t += NW) {
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += part[w][t][lane * 4 + e];
        const int m = t * 16 + r16, c = n0 + 4 * grp, left = p.N - c;
        if (m >= p.M) continue;
        if (p.bias) {
            float bias[4];
            load_part<float, 4>(p.bias + c, left, bias);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += bias[e];
        }
        store_part<T, 4>(C + (long long)m * p.N + c, left, v);
    }
#endif
}

// ---- the quantiser: a block reads a 128 x 128 tile of x once and writes its codes by rows, by columns, or both, and the tile's column sums ----
struct Quantize {
    const void* x;
    long long rows, cols, stride;
    int tile;                                 // 1: a scale per row of 128 (and per column of 128 rows); 128: one for the tile
    u8 *codes, *scale, *codes_t, *scale_t;    // [rows][cp], [rows or tiles][cp / 128]; [cols][rp], [cols or tiles][rp / 128]; NULL: not wanted
    float* sums;                              // [tiles of rows][cols]
};
// The tile stays in registers between its read and its two ways out, and the column reductions share their LDS with the transposed image.
// HBM-bound: 8192 x 4096 bf16 both ways, 134 MB, 32 us = 4.2 TB/s (36 with column sums); three blocks a CU by their registers.  Held to fewer
// registers the compiler spills the tile (100 us).
template <typename T>
__global__ __launch_bounds__(256) void quantize_kernel(Quantize q) {
    constexpr int PITCH = 136, VEC = ElemOf<T>::VEC, ACC = 8 / VEC;      // bytes of a column in the transposed image
    union Shared {
        struct {
            float amax[16][128], sum[16][128];
        } col;
        u8 image[128 * PITCH];
    };
    __shared__ __attribute__((aligned(16))) Shared sh;
    __shared__ float col_scale[128];
    __shared__ float tile_amax[4];
    const T* x = (const T*)q.x;
    const int tid = threadIdx.x, g = tid >> 4, l = tid & 15;   // rows 8 g .. + 7, columns 8 l .. + 7 of the tile
    const long long tr = blockIdx.y, tc = blockIdx.x, r0 = tr * 128 + g * 8, c0 = tc * 128 + l * 8;
    const long long kc = (q.cols + 127) / 128, kr = (q.rows + 127) / 128;
    u32x4_t raw[8][ACC];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const T* src = x + (r0 + i) * q.stride + c0;
#pragma unroll
        for (int k = 0; k < ACC; ++k) {
            const long long left = r0 + i < q.rows ? q.cols - c0 - k * VEC : 0;
            raw[i][k] = load_raw_part<T>(src + k * VEC, left);
        }
    }
    auto row_of = [&](int i, float (&v)[8]) {
#pragma unroll
        for (int k = 0; k < ACC; ++k) {
            float w[VEC];
            widen<T>(raw[i][k], w);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[k * VEC + e] = w[e];
        }
    };
    const bool columns = q.codes_t || q.sums;
    float ca[8], cs[8], ra[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) ca[e] = cs[e] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float v[8], a = 0.f;
        row_of(i, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float m = __builtin_fabsf(v[e]) < INFINITY ? __builtin_fabsf(v[e]) : 0.f;            // of the finite values
            a = __builtin_fmaxf(a, m);
            ca[e] = __builtin_fmaxf(ca[e], m);
            cs[e] += v[e];
        }
        ra[i] = a;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) ra[i] = __builtin_fmaxf(ra[i], __shfl_xor(ra[i], o, 16));
    int e_tile = 0;
    if (q.tile == 128) {
        float a = ra[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) a = __builtin_fmaxf(a, ra[i]);
        a = wave_max(a);
        if ((tid & 63) == 0) tile_amax[tid >> 6] = a;
        __syncthreads();
        e_tile = scale_exponent(__builtin_fmaxf(__builtin_fmaxf(tile_amax[0], tile_amax[1]), __builtin_fmaxf(tile_amax[2], tile_amax[3])));
        if (tid == 0) {
            if (q.codes) q.scale[tr * kc + tc] = (u8)(e_tile + 127);
            if (q.codes_t) q.scale_t[tc * kr + tr] = (u8)(e_tile + 127);
        }
    }
    // no value is beyond 448 times its scale but infinities, and those and NaN become the NaN code
    if (q.codes) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (r0 + i >= q.rows) break;
            const int e = q.tile == 128 ? e_tile : scale_exponent(ra[i]);
            const float s = pow2f(-e);
            float v[8];
            row_of(i, v);
            uint32_t w[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int t = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * k] * s, v[4 * k + 1] * s, 0, false);
                w[k] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * k + 2] * s, v[4 * k + 3] * s, t, true);
            }
            __builtin_memcpy(q.codes + (r0 + i) * kc * 128 + c0, w, 8);
            if (q.tile == 1 && l == 0) q.scale[(r0 + i) * kc + tc] = (u8)(e + 127);
        }
    }
    if (!columns) return;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        *reinterpret_cast<f32x4_t*>(&sh.col.amax[g][l * 8 + 4 * k]) = f32x4_t{ca[4 * k], ca[4 * k + 1], ca[4 * k + 2], ca[4 * k + 3]};
        *reinterpret_cast<f32x4_t*>(&sh.col.sum[g][l * 8 + 4 * k]) = f32x4_t{cs[4 * k], cs[4 * k + 1], cs[4 * k + 2], cs[4 * k + 3]};
    }
    __syncthreads();
    if (tid < 128) {
        const long long c = tc * 128 + tid;
        float a = sh.col.amax[0][tid];
#pragma unroll
        for (int k = 1; k < 16; ++k) a = __builtin_fmaxf(a, sh.col.amax[k][tid]);
        const int e = q.tile == 128 ? e_tile : scale_exponent(a);
        col_scale[tid] = pow2f(-e);
        if (c < q.cols && q.codes_t && q.tile == 1) q.scale_t[c * kr + tr] = (u8)(e + 127);
    } else if (q.sums) {
        const long long c = tc * 128 + tid - 128;
        float s = sh.col.sum[0][tid - 128];
#pragma unroll
        for (int k = 1; k < 16; ++k) s += sh.col.sum[k][tid - 128];
        if (c < q.cols) q.sums[tr * q.cols + c] = s;
    }
    if (!q.codes_t) return;
    __syncthreads();                                          // (the image overlays the reductions)
    float s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = col_scale[l * 8 + e];
    uint32_t w[8][2];                                         // a column's eight rows are eight neighbouring bytes of the transposed image
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        float v0[8], v1[8];
        row_of(4 * k, v0);
        row_of(4 * k + 1, v1);
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e][k] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v0[e] * s[e], v1[e] * s[e], 0, false);
        row_of(4 * k + 2, v0);
        row_of(4 * k + 3, v1);
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e][k] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v0[e] * s[e], v1[e] * s[e], (int)w[e][k], true);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) *reinterpret_cast<uint64_t*>(sh.image + (l * 8 + e) * PITCH + g * 8) = (uint64_t)w[e][1] << 32 | w[e][0];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {                             // 8 lanes write a column's 128 bytes
        const int cc = i * 32 + (tid >> 3), part = tid & 7;
        const long long c = tc * 128 + cc;
        if (c < q.cols) {
            const uint64_t lo = *reinterpret_cast<const uint64_t*>(sh.image + cc * PITCH + part * 16), hi = *reinterpret_cast<const uint64_t*>(sh.image + cc * PITCH + part * 16 + 8);
            *reinterpret_cast<u32x4_t*>(q.codes_t + c * kr * 128 + tr * 128 + part * 16) = u32x4_t{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
        }
    }
}

// out[c] = sum over the parts in order within 16 strips, then in strip order
__global__ __launch_bounds__(1024) void sum_parts_kernel(const float* __restrict__ parts, long long n, long long cols, long long from, float* __restrict__ out) {
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, strip = threadIdx.x >> 6;
    const long long c = from + (long long)blockIdx.x * 64 + lane;
    float s = 0.f;
    if (c < cols)
        for (long long k = strip; k < n; k += 16) s += parts[k * cols + c];
    red[strip][lane] = s;
    __syncthreads();
    if (strip == 0 && c < cols) {
#pragma unroll
        for (int k = 1; k < 16; ++k) s += red[k][lane];
        out[c] = s;
    }
}

template <typename T, bool FAST, int TM, int TN, int WM, int WN>
int launch_tile(const Product& p, hipStream_t st) {
    const int tm = (p.M + TM - 1) / TM, tn = (p.N + TN - 1) / TN;
    constexpr int lds = 4 * (TM + TN) * (KT / 2) + 2 * (TM + TN) * 4;
    static std::atomic<bool> big[64] = {};                    // per device: the kernel may use more than 64 KiB of LDS
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return w2c_launch_status();
    if (!big[dev].load(std::memory_order_acquire)) {
        if (hipFuncSetAttribute(reinterpret_cast<const void*>(&matmul_tile_kernel<T, FAST, TM, TN, WM, WN>), hipFuncAttributeMaxDynamicSharedMemorySize, lds) !=
            hipSuccess)
            return w2c_launch_status();
        big[dev].store(true, std::memory_order_release);
    }
    hipLaunchKernelGGL((matmul_tile_kernel<T, FAST, TM, TN, WM, WN>), dim3(tm * tn, p.parts), dim3(WM * WN * 64), lds, st, p, tm, tn);
    if (p.parts > 1)
        hipLaunchKernelGGL((sum_splits_kernel<T>), dim3((unsigned)(((long long)((p.N + 3) / 4) * p.M + 255) / 256)), dim3(256), 0, st, p);
    return w2c_launch_status();
}

long long tiles(int M, int N, int tm, int tn) { return (long long)((M + tm - 1) / tm) * ((N + tn - 1) / tn); }
// What a product of the tile kernels is cut into: the largest tiles of which there are enough for the 256 CUs (a larger tile reads less per product),
// and where there are at most half as many of the smallest, parts of the reduction: about 256 in all, none shorter than 8 blocks of 128 (16 with more
// than 64 tiles), to be worth the sum of the parts.  us to bf16, default / FAST:
//   256 x 256 or 128 x 128 tiles  3200 x 3200 x 4096 (169 of the former) 85 or 83; 3584 x 3584 x 4096 (196) 90 or 107 / 55 or 73
//   128 x 128 or 128 x 64 tiles   1536 x 1920 x 4096 (180) 34 or 34 / 21 or 28; 1664 x 2048 x 4096 (208) 36 or 38 / 22 or 30
//   1 or 2 parts, up to 64 tiles  512 x 512 x 1152 8.5 or 9.7 / 7.0 or 8.9; 256 x 256 x 1920 (15 blocks) 11.5 or 10.4 / 9.0 either way
//   ... with more                 1024 x 1024 x 2176 12.8 or 16.6 / 9.8 or 14.8; 1024 x 1024 x 4096 21.6 or 19.4
//   about 256 parts, or twice     64 x 4096 x 4096 13.1 or 16.3, 512 x 512 x 8192 15.5 or 20.3
struct Cut {
    int tm, tn, parts;
};
Cut product_cut(int M, int N, int K) {
    if (tiles(M, N, 256, 256) >= 160) return {256, 256, 1};
    if (tiles(M, N, 128, 128) >= 180) return {128, 128, 1};
    const long long t = tiles(M, N, 128, 64);
    long long parts = t > 128 ? 1 : 256 / t;
    const int least = t > 64 ? 16 : 8, most = K / KT / least;
    if (parts > most) parts = most > 1 ? most : 1;
    if (parts > 16) parts = 16;
    return {128, 64, (int)parts};
}

long long product_blocks(int M, int N, int K) {
    const Cut cut = product_cut(M, N, K);
    return tiles(M, N, cut.tm, cut.tn);
}

template <typename T, bool FAST>
int launch_product(const Product& p, hipStream_t st) {
    if (p.M <= ROWS_MOST) {
        const dim3 grid((p.N + 15) / 16);
        // 16 waves to a block of 16 columns where there is at most one block for a CU and each of the waves still gets a few k blocks to keep on their
        // way; they pay for their larger sum.  4 / 16 waves, us, bf16, with 1 row: 4096 x 6144 7.9 / 7.6, 4096 x 8192 11.9 / 8.7, 512 x 16384 16.3 / 12.2, but
        // 4096 x 4096 7.0 / 7.9, 8192 x 4096 8.9 / 12.8, 6144 x 12288 22.5 / 24.4; with 16 rows: 4096 x 6144 8.8 / 9.5, 4096 x 7168 12.0 / 10.3,
        // 4096 x 8192 12.8 / 11.2, 6144 x 7168 18.3 / 18.6, and the worst on this side, 512 x 12288 14.5 / 16.2.
        const bool few = p.N <= 16 * 256 && p.K >= 56 * KT;
#define MATMUL_ROWS(MT)                                                                                                             \
    do {                                                                                                                            \
        if (few) hipLaunchKernelGGL((matmul_rows_kernel<T, FAST, MT, 16>), grid, dim3(1024), 0, st, p);                                    \
        else hipLaunchKernelGGL((matmul_rows_kernel<T, FAST, MT, 4>), grid, dim3(256), 0, st, p);                                          \
    } while (0)
        if (p.M <= 16) MATMUL_ROWS(1);
        else MATMUL_ROWS(2);
#undef MATMUL_ROWS
        return w2c_launch_status();
    }
    const Cut cut = product_cut(p.M, p.N, p.K);
    if (cut.tm == 256) return launch_tile<T, FAST, 256, 256, 2, 2>(p, st);
    if (cut.tn == 128) return launch_tile<T, FAST, 128, 128, 2, 2>(p, st);
    return launch_tile<T, FAST, 128, 64, 2, 2>(p, st);
}

long long workspace_bytes_of(int M, int N, int K) {
    if (M < 1 || N < 1 || K < KT || K % KT || M > 0x7FFFFFFF - 255 || N > 0x7FFFFFFF - 255) return W2C_E_ARG;
    const int parts = M <= ROWS_MOST ? 1 : product_cut(M, N, K).parts;
    return parts > 1 ? (long long)parts * M * N * (long long)sizeof(float) : 0;
}

int product(bool fast, const void* a, const void* a_scale, int a_tile, const void* b, const void* b_scale, int b_tile, int M, int N, int K,
            const float* bias, void* c, int dtype, void* workspace, long long workspace_bytes, void* stream) {
    if (!a || !a_scale || !b || !b_scale || !c || M < 1 || N < 1 || K < KT || K % KT || K > K_MOST || dtype < W2C_F32 || dtype > W2C_F16) return W2C_E_ARG;
    if (M > 0x7FFFFFFF - 255 || N > 0x7FFFFFFF - 255) return W2C_E_ARG;                       // (sizes are rounded up to tiles)
    if ((a_tile != 1 && a_tile != 128) || (b_tile != 1 && b_tile != 128) || (long long)M * N > (1ll << 40)) return W2C_E_ARG;
    if ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) return W2C_E_ARG;
    if (M <= ROWS_MOST ? tiles(1, N, 1, 16) > most_blocks(256) : product_blocks(M, N, K) > most_blocks(256)) return W2C_E_ARG;      // (one launch)
    w2c_clear_error();
    const long long need = workspace_bytes_of(M, N, K);
    if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15))) return W2C_E_ARG;
    const Product p{(const u8*)a, (const u8*)a_scale, (const u8*)b, (const u8*)b_scale, bias, c, M, N, K,
                    M <= ROWS_MOST ? 1 : product_cut(M, N, K).parts, (float*)workspace, a_tile == 128 ? 7 : 0, b_tile == 128 ? 7 : 0};
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == W2C_F32) return fast ? W2C_E_ARG : launch_product<float, false>(p, st);
    if (dtype == W2C_BF16) return fast ? launch_product<bf16_t, true>(p, st) : launch_product<bf16_t, false>(p, st);
    return fast ? launch_product<f16_t, true>(p, st) : launch_product<f16_t, false>(p, st);
}

}  // namespace

extern "C" long long w2c_matmul_fp8_workspace_bytes(int M, int N, int K) { return workspace_bytes_of(M, N, K); }

extern "C" int w2c_matmul_fp8(const void* a, const void* a_scale, int a_tile, const void* b, const void* b_scale, int b_tile, int M, int N, int K,
                              const float* bias, void* c, int dtype, void* workspace, long long workspace_bytes, void* stream) {
    return product(false, a, a_scale, a_tile, b, b_scale, b_tile, M, N, K, bias, c, dtype, workspace, workspace_bytes, stream);
}

extern "C" int w2c_matmul_fp8_fast(const void* a, const void* a_scale, int a_tile, const void* b, const void* b_scale, int b_tile, int M, int N, int K,
                                   const float* bias, void* c, int dtype, void* workspace, long long workspace_bytes, void* stream) {
    return product(true, a, a_scale, a_tile, b, b_scale, b_tile, M, N, K, bias, c, dtype, workspace, workspace_bytes, stream);
}

extern "C" long long w2c_quantize_fp8_workspace_bytes(long long rows, long long cols) {
    return rows < 1 || cols < 1 ? W2C_E_ARG : rows <= 128 ? 0 : (rows + 127) / 128 * cols * (long long)sizeof(float);      // (one tile's sums are the sums)
}

extern "C" int w2c_quantize_fp8(const void* x, int dtype, long long rows, long long cols, long long stride, int tile, void* codes, void* scale,
                                void* codes_t, void* scale_t, float* column_sums, void* workspace, long long workspace_bytes, void* stream) {
    if (!x || dtype < W2C_F32 || dtype > W2C_F16 || rows < 1 || cols < 1 || stride < cols || (tile != 1 && tile != 128)) return W2C_E_ARG;
    if ((!codes && !codes_t && !column_sums) || (codes && !scale) || (codes_t && !scale_t) || rows > K_MOST || cols > 128 * most_blocks(256)) return W2C_E_ARG;
    if (codes_t && (reinterpret_cast<uintptr_t>(codes_t) & 15)) return W2C_E_ARG;
    const bool parts = column_sums && w2c_quantize_fp8_workspace_bytes(rows, cols) > 0;
    if (parts && (!workspace || workspace_bytes < w2c_quantize_fp8_workspace_bytes(rows, cols))) return W2C_E_ARG;
    w2c_clear_error();
    const hipStream_t st = (hipStream_t)stream;
    const Quantize q{x, rows, cols, stride, tile, (u8*)codes, (u8*)scale, (u8*)codes_t, (u8*)scale_t, parts ? (float*)workspace : column_sums};
    const dim3 grid((unsigned)((cols + 127) / 128), (unsigned)((rows + 127) / 128));
    if (dtype == W2C_F32) hipLaunchKernelGGL((quantize_kernel<float>), grid, dim3(256), 0, st, q);
    else if (dtype == W2C_BF16) hipLaunchKernelGGL((quantize_kernel<bf16_t>), grid, dim3(256), 0, st, q);
    else hipLaunchKernelGGL((quantize_kernel<f16_t>), grid, dim3(256), 0, st, q);
    if (parts)
        for (long long from = 0; from < cols; from += 64 * most_blocks(1024)) {
            const long long blocks = (cols - from + 63) / 64;
            hipLaunchKernelGGL(sum_parts_kernel, dim3((unsigned)(blocks < most_blocks(1024) ? blocks : most_blocks(1024))), dim3(1024), 0, st,
                               (const float*)workspace, (rows + 127) / 128, cols, from, column_sums);
        }
    return w2c_launch_status();
}
