// Matrix product of e4m3 codes with a power-of-two (e8m0) scale per 128 elements of the reduction, and the quantiser that makes them.
//
//   C[m][n] = sum_k  a[m][k] 2^ea(m, k / 128)  b[n][k] 2^eb(n, k / 128)  (+ bias[n])
//
// Rows are stored padded with zero codes to a multiple of 128.  A scale belongs to one row's 128 (activations, gradients) or to a 128 x 128 tile
// (weights: the transposed weights then have the same codes and scales).  gfx950's scaled matrix instructions multiply by both e8m0 scales
// themselves, so one f32 accumulator runs through the whole reduction and no vector instruction touches the products.  Within a block of 128
// the order of k is free as long as both operands agree, since its scale is one.
//
// The scaled instructions line the products of 8 neighbouring k up to the largest of them and keep 13 bits below it (measured: a product 2^-14 of the
// largest is lost, in the next group of 8 it is not): about 1.5e-5 of the result's norm, far below a bf16 or f16 output's own rounding
// but not below an f32 one's.  An f32 output therefore goes through the bf16 instructions, which keep 23: a code times its scale is a bf16
// number exactly (one conversion instruction per pair does both), at half the rate.
//
//   tile kernels   at least 65 rows: TM x TN tiles, both operands by LDS-DMA into two stages of 128 k, one barrier per stage
//   row kernel     up to 64 rows (tokens being decoded): bound by reading b once; no LDS for operands, the waves of a block split k
#include "lm_common.h"

namespace {

typedef unsigned char u8;
constexpr int KT = 128;                       // elements of the reduction per scale, and per stage

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

// Stage image: row r (128 bytes) at r * 128, its 16-byte chunk c in slot c ^ ((r >> 1) & 7): 16 neighbouring rows' same chunk then cover all 64
// banks once.  A piece of LDS-DMA is 8 rows (64 lanes x 16 bytes, contiguous in LDS); the swizzle is in the source address.
template <typename T, int TM, int TN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64, 1) void matmul_tile_kernel(Product p, int tiles_m, int tiles_n) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int NW = WM * WN, MI = TM / WM / 32, NI = TN / WN / 32, PA = TM / 8 / NW, PB = TN / 8 / NW;
    constexpr unsigned STAGE = (TM + TN) * KT;
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
    const u32x4_t srd_a = descriptor(p.a + (long long)m0 * p.K, (unsigned)ml * (unsigned)p.K);
    const u32x4_t srd_b = descriptor(p.b + (long long)n0 * p.K, (unsigned)nl * (unsigned)p.K);
    const unsigned lds = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(size_t)W2C_LPTR(smem));
    const int prow = wave * 8 + (lane >> 3), pchunk = (lane & 7) ^ ((prow >> 1) & 7);
    const unsigned voff = (unsigned)prow * (unsigned)p.K + (unsigned)pchunk * 16u, vstep = (unsigned)(NW * 8) * (unsigned)p.K;
    auto stage = [&](int kb) {
        const unsigned dst = lds + (unsigned)(kb & 1) * STAGE + (unsigned)wave * 1024u, soff = (unsigned)kb * KT;
#pragma unroll
        for (int i = 0; i < PA; ++i) dma16(dst + i * NW * 1024u, voff + i * vstep, srd_a, soff);
#pragma unroll
        for (int i = 0; i < PB; ++i) dma16(dst + TM * KT + i * NW * 1024u, voff + i * vstep, srd_b, soff);
    };
    const int wm = (wave % WM) * (TM / WM), wn = (wave / WM) * (TN / WN);
    const u8 *psa[MI], *psb[NI];
    int sa[MI], sb[NI], sa_next[MI], sb_next[NI];
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        const int r = m0 + wm + i * 32 + l31;
        psa[i] = p.sa + (long long)((r < p.M ? r : p.M - 1) >> p.a_shift) * KB;
        sa_next[i] = *psa[i];
    }
#pragma unroll
    for (int j = 0; j < NI; ++j) {
        const int r = n0 + wn + j * 32 + l31;
        psb[j] = p.sb + (long long)((r < p.N ? r : p.N - 1) >> p.b_shift) * KB;
        sb_next[j] = *psb[j];
    }
    f32x16_t acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    // a lane's 32 bytes of k half h: chunks 4 h + 2 lhi, + 1
    const int key = (l31 >> 1) & 7;
    const u8* ra = smem + (wm + l31) * KT;
    const u8* rb = smem + (TM + wn + l31) * KT;
    int slot[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) slot[q] = ((((q >> 1) * 4 + 2 * lhi + (q & 1)) ^ key) << 4);
    stage(0);
    for (int kb = 0; kb < KB; ++kb) {
        // this wave's pieces of stage kb have landed and its reads of stage kb - 1 are done; behind the barrier everyone's are
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        // the scales of this stage came with it; they are taken here, before the next stage's loads are issued, so that no wait for them
        // can end up behind those
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            asm volatile("" : "+v"(sa_next[i]));
            sa[i] = sa_next[i];
        }
#pragma unroll
        for (int j = 0; j < NI; ++j) {
            asm volatile("" : "+v"(sb_next[j]));
            sb[j] = sb_next[j];
        }
        if (kb + 1 < KB) {
            stage(kb + 1);
#pragma unroll
            for (int i = 0; i < MI; ++i) sa_next[i] = psa[i][kb + 1];
#pragma unroll
            for (int j = 0; j < NI; ++j) sb_next[j] = psb[j][kb + 1];
        }
        const unsigned buf = (unsigned)(kb & 1) * STAGE;
        if constexpr (sizeof(T) == 4) {
            float xa[MI], xb[NI];
#pragma unroll
            for (int i = 0; i < MI; ++i) xa[i] = __uint_as_float((uint32_t)sa[i] << 23);
#pragma unroll
            for (int j = 0; j < NI; ++j) xb[j] = __uint_as_float((uint32_t)sb[j] << 23);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                u32x4_t ca[MI], cb[NI];
#pragma unroll
                for (int j = 0; j < NI; ++j) cb[j] = *reinterpret_cast<const u32x4_t*>(rb + buf + j * 32 * KT + slot[q]);
#pragma unroll
                for (int i = 0; i < MI; ++i) ca[i] = *reinterpret_cast<const u32x4_t*>(ra + buf + i * 32 * KT + slot[q]);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    bf16x8_t fb[NI];
#pragma unroll
                    for (int j = 0; j < NI; ++j) fb[j] = scaled8(cb[j][2 * h], cb[j][2 * h + 1], xb[j]);
#pragma unroll
                    for (int i = 0; i < MI; ++i) {
                        const bf16x8_t fa = scaled8(ca[i][2 * h], ca[i][2 * h + 1], xa[i]);
#pragma unroll
                        for (int j = 0; j < NI; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fb[j], fa, acc[i][j], 0, 0, 0);
                    }
                }
            }
        } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            i32x8_t fa[MI], fb[NI];
#pragma unroll
            for (int j = 0; j < NI; ++j)
                fb[j] = cat_i32x8(*reinterpret_cast<const u32x4_t*>(rb + buf + j * 32 * KT + slot[2 * h]),
                                  *reinterpret_cast<const u32x4_t*>(rb + buf + j * 32 * KT + slot[2 * h + 1]));
#pragma unroll
            for (int i = 0; i < MI; ++i)
                fa[i] = cat_i32x8(*reinterpret_cast<const u32x4_t*>(ra + buf + i * 32 * KT + slot[2 * h]),
                                  *reinterpret_cast<const u32x4_t*>(ra + buf + i * 32 * KT + slot[2 * h + 1]));
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[j], fa[i], acc[i][j], 0, 0, 0, sb[j], 0, sa[i]);
        }
        }
    }
    // accumulator e of a lane: column n = (e & 3) + 8 (e >> 2) + 4 lhi, row m = l31 of its 32 x 32 tile
    T* C = (T*)p.c;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        const int m = m0 + wm + i * 32 + l31;
        if (m >= p.M) continue;
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int n = n0 + wn + j * 32 + 8 * q + 4 * lhi, left = p.N - n;
                float v[4] = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                if (p.bias) {
                    float bias[4];
                    load_part<float, 4>(p.bias + n, left, bias);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] += bias[e];
                }
                store_part<T, 4>(C + (long long)m * p.N + n, left, v);
            }
    }
#endif
}

// Up to 16 MT rows of a against 16 rows of b per block; wave w takes its share of the k blocks, the partial tiles are added in wave order.
template <typename T, int MT, int NW>
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
                if constexpr (sizeof(T) == 4) {
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
template <typename T>
__global__ __launch_bounds__(256) void quantize_kernel(Quantize q) {
    constexpr int PITCH = 144;                                 // bytes of a column in the transposed image
    __shared__ float col_amax[16][128];
    __shared__ float col_sum[16][128];
    __shared__ int col_e[128];
    __shared__ float tile_amax[4];
    __shared__ __attribute__((aligned(16))) u8 image[128 * PITCH];
    const T* x = (const T*)q.x;
    const int tid = threadIdx.x, g = tid >> 4, l = tid & 15;   // rows 8 g .. + 7, columns 8 l .. + 7 of the tile
    const long long tr = blockIdx.y, tc = blockIdx.x, r0 = tr * 128 + g * 8, c0 = tc * 128 + l * 8;
    const long long kc = (q.cols + 127) / 128, kr = (q.rows + 127) / 128;
    float v[8][8], ca[8], cs[8], ra[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) ca[e] = cs[e] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long long left = r0 + i < q.rows ? q.cols - c0 : 0;
        const T* src = x + (r0 + i) * q.stride + c0;
        if constexpr (sizeof(T) == 4) {
            float lo[4], hi[4];
            load_part<T, 4>(src, left, lo);
            load_part<T, 4>(src + 4, left - 4, hi);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[i][e] = lo[e];
                v[i][4 + e] = hi[e];
            }
        } else load_part<T, 8>(src, left, v[i]);
        float a = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float m = __builtin_fabsf(v[i][e]) < INFINITY ? __builtin_fabsf(v[i][e]) : 0.f;      // of the finite values
            a = __builtin_fmaxf(a, m);
            ca[e] = __builtin_fmaxf(ca[e], m);
            cs[e] += v[i][e];
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) a = __builtin_fmaxf(a, __shfl_xor(a, o, 16));
        ra[i] = a;
    }
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
    if (q.codes) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (r0 + i >= q.rows) break;
            const int e = q.tile == 128 ? e_tile : scale_exponent(ra[i]);
            const float s = pow2f(-e);
            uint32_t w[2] = {0, 0};
#pragma unroll
            for (int k = 0; k < 2; ++k) {                     // no value is beyond 448 but infinities, and those and NaN become the NaN code
                int t = __builtin_amdgcn_cvt_pk_fp8_f32(v[i][4 * k] * s, v[i][4 * k + 1] * s, 0, false);
                w[k] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[i][4 * k + 2] * s, v[i][4 * k + 3] * s, t, true);
            }
            __builtin_memcpy(q.codes + (r0 + i) * kc * 128 + c0, w, 8);
            if (q.tile == 1 && l == 0) q.scale[(r0 + i) * kc + tc] = (u8)(e + 127);
        }
    }
    if (!q.codes_t && !q.sums) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        col_amax[g][l * 8 + e] = ca[e];
        col_sum[g][l * 8 + e] = cs[e];
    }
    __syncthreads();
    if (tid < 128) {
        const long long c = tc * 128 + tid;
        float a = col_amax[0][tid], s = col_sum[0][tid];
#pragma unroll
        for (int k = 1; k < 16; ++k) {
            a = __builtin_fmaxf(a, col_amax[k][tid]);
            s += col_sum[k][tid];
        }
        col_e[tid] = q.tile == 128 ? e_tile : scale_exponent(a);
        if (c < q.cols) {
            if (q.sums) q.sums[tr * q.cols + c] = s;
            if (q.codes_t && q.tile == 1) q.scale_t[c * kr + tr] = (u8)(col_e[tid] + 127);
        }
    }
    if (!q.codes_t) return;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) {                             // a column's eight rows are eight neighbouring bytes of the transposed image
        const float s = pow2f(-col_e[l * 8 + e]);
        uint32_t w[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            int t = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * k][e] * s, v[4 * k + 1][e] * s, 0, false);
            w[k] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * k + 2][e] * s, v[4 * k + 3][e] * s, t, true);
        }
        *reinterpret_cast<uint64_t*>(image + (l * 8 + e) * PITCH + g * 8) = (uint64_t)w[1] << 32 | w[0];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {                             // 8 lanes write a column's 128 bytes
        const int cc = i * 32 + (tid >> 3), part = tid & 7;
        const long long c = tc * 128 + cc;
        if (c < q.cols)
            *reinterpret_cast<u32x4_t*>(q.codes_t + c * kr * 128 + tr * 128 + part * 16) = *reinterpret_cast<const u32x4_t*>(image + cc * PITCH + part * 16);
    }
}

// out[c] = sum over the parts in order within 16 strips, then in strip order
__global__ __launch_bounds__(1024) void sum_parts_kernel(const float* __restrict__ parts, long long n, long long cols, float* __restrict__ out) {
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, strip = threadIdx.x >> 6;
    const long long c = (long long)blockIdx.x * 64 + lane;
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

template <typename T, int TM, int TN, int WM, int WN>
int launch_tile(const Product& p, hipStream_t st) {
    const int tm = (p.M + TM - 1) / TM, tn = (p.N + TN - 1) / TN;
    constexpr int lds = 2 * (TM + TN) * KT;
    static std::atomic<bool> big[64] = {};                    // per device: the kernel may use more than 64 KiB of LDS
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return w2c_launch_status();
    if (!big[dev].load(std::memory_order_acquire)) {
        if (hipFuncSetAttribute(reinterpret_cast<const void*>(&matmul_tile_kernel<T, TM, TN, WM, WN>), hipFuncAttributeMaxDynamicSharedMemorySize, lds) !=
            hipSuccess)
            return w2c_launch_status();
        big[dev].store(true, std::memory_order_release);
    }
    hipLaunchKernelGGL((matmul_tile_kernel<T, TM, TN, WM, WN>), dim3(tm * tn), dim3(WM * WN * 64), lds, st, p, tm, tn);
    return w2c_launch_status();
}

template <typename T>
int launch_product(const Product& p, hipStream_t st) {
    if (p.M <= 64) {
        const dim3 grid((p.N + 15) / 16);
        if (p.M <= 16) hipLaunchKernelGGL((matmul_rows_kernel<T, 1, 4>), grid, dim3(256), 0, st, p);
        else if (p.M <= 32) hipLaunchKernelGGL((matmul_rows_kernel<T, 2, 4>), grid, dim3(256), 0, st, p);
        else hipLaunchKernelGGL((matmul_rows_kernel<T, 4, 4>), grid, dim3(256), 0, st, p);
        return w2c_launch_status();
    }
    // the large tile halves the traffic per product, but only where there are tiles for most of the 256 CUs
    if ((long long)((p.M + 255) / 256) * ((p.N + 255) / 256) >= 160) return launch_tile<T, 256, 256, 2, 4>(p, st);
    return launch_tile<T, 128, 128, 2, 2>(p, st);
}

}  // namespace

extern "C" int w2c_matmul_fp8(const void* a, const void* a_scale, int a_tile, const void* b, const void* b_scale, int b_tile, int M, int N, int K,
                              const float* bias, void* c, int dtype, void* stream) {
    if (!a || !a_scale || !b || !b_scale || !c || M < 1 || N < 1 || K < KT || K % KT || K > (1 << 22) || dtype < W2C_F32 || dtype > W2C_F16) return W2C_E_ARG;
    if ((a_tile != 1 && a_tile != 128) || (b_tile != 1 && b_tile != 128) || (long long)M * N > (1ll << 40)) return W2C_E_ARG;
    if ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) return W2C_E_ARG;
    if ((long long)((M + 127) / 128) * ((N + 127) / 128) > 0x7FFFFFFF) return W2C_E_ARG;
    w2c_clear_error();
    const Product p{(const u8*)a, (const u8*)a_scale, (const u8*)b, (const u8*)b_scale, bias, c, M, N, K, a_tile == 128 ? 7 : 0, b_tile == 128 ? 7 : 0};
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == W2C_F32) return launch_product<float>(p, st);
    if (dtype == W2C_BF16) return launch_product<bf16_t>(p, st);
    return launch_product<f16_t>(p, st);
}

extern "C" long long w2c_quantize_fp8_workspace_bytes(long long rows, long long cols) {
    return rows < 1 || cols < 1 ? W2C_E_ARG : (rows + 127) / 128 * cols * (long long)sizeof(float);
}

extern "C" int w2c_quantize_fp8(const void* x, int dtype, long long rows, long long cols, long long stride, int tile, void* codes, void* scale,
                                void* codes_t, void* scale_t, float* column_sums, void* workspace, long long workspace_bytes, void* stream) {
    if (!x || dtype < W2C_F32 || dtype > W2C_F16 || rows < 1 || cols < 1 || stride < cols || (tile != 1 && tile != 128)) return W2C_E_ARG;
    if ((!codes && !codes_t && !column_sums) || (codes && !scale) || (codes_t && !scale_t) || rows > 65535ll * 128 || cols > (1ll << 31)) return W2C_E_ARG;
    if (codes_t && (reinterpret_cast<uintptr_t>(codes_t) & 15)) return W2C_E_ARG;
    if (column_sums && (!workspace || workspace_bytes < w2c_quantize_fp8_workspace_bytes(rows, cols))) return W2C_E_ARG;
    w2c_clear_error();
    const hipStream_t st = (hipStream_t)stream;
    const Quantize q{x, rows, cols, stride, tile, (u8*)codes, (u8*)scale, (u8*)codes_t, (u8*)scale_t, column_sums ? (float*)workspace : nullptr};
    const dim3 grid((unsigned)((cols + 127) / 128), (unsigned)((rows + 127) / 128));
    if (dtype == W2C_F32) hipLaunchKernelGGL((quantize_kernel<float>), grid, dim3(256), 0, st, q);
    else if (dtype == W2C_BF16) hipLaunchKernelGGL((quantize_kernel<bf16_t>), grid, dim3(256), 0, st, q);
    else hipLaunchKernelGGL((quantize_kernel<f16_t>), grid, dim3(256), 0, st, q);
    if (column_sums)
        hipLaunchKernelGGL(sum_parts_kernel, dim3((unsigned)((cols + 63) / 64)), dim3(1024), 0, st, (const float*)workspace, (rows + 127) / 128, cols,
                           column_sums);
    return w2c_launch_status();
}
