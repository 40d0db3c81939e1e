// Layer norm over the last dimension, forward and backward, with the residual add in front of it.
//
//   h = x + r (rounded to the tensors' type: the h that is returned is the h that is normalised; without r, h = x)
//   y = n w + b,   n = (h - mean) rstd,   rstd = 1 / sqrt(mean((h - mean)^2) + eps)
//   dx = rstd (g - mean(g) - n mean(g n)) + dh,   g = dy w;      dw = sum_rows dy n,   db = sum_rows dy
//
// HBM-bound both ways (a dozen operations per element).  A row lives in registers between its one read and its one write, so the variance is
// the mean of squared DIFFERENCES (no cancellation); sums are f32.  One to 16 waves own a row; rows longer than that are walked three times (their
// second and third walks hit the caches).  Two kernels spill: the forward of 16 waves with four accesses of a 16-bit type (rows of 16 385 to 32 768 columns: 1.3
// to 1.7 TB/s where 16 384 columns reach 4.6) and, 52 bytes a lane, the f32 backward of 8 193 to 16 384 columns (5 TB/s all the same).
#include "lm_common.h"

namespace {

// sum of one value over the row's NW waves; every lane gets it.  `slot`: NW floats that no other reduction in flight uses.
template <int NW>
__device__ __forceinline__ float row_sum(float v, float* slot) {
    v = wave_sum(v);
    if constexpr (NW == 1) return v;
    if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) s += slot[i];
    return s;
}

template <int NW> constexpr int block_threads() { return NW == 1 ? 256 : NW * 64; }

// A block walks every gridDim.x-th row (group): its weights stay in registers, and the next row is on its way while this one is reduced.
template <typename T, typename W, int NW, int NV>
__global__ __launch_bounds__(block_threads<NW>()) void ln_forward_kernel(const T* __restrict__ x, const T* __restrict__ res, long long rows,
                                                                          int D, const W* __restrict__ w, const W* __restrict__ b, float eps,
                                                                          T* __restrict__ y, T* __restrict__ h, float* __restrict__ mean,
                                                                          float* __restrict__ rstd) {
    constexpr int VEC = ElemOf<T>::VEC, TPR = NW * 64, ROWS = NW == 1 ? 4 : 1, WV = ElemOf<W>::VEC, WN = VEC / WV;
    constexpr bool AHEAD = NV <= 2;                            // (1024 threads of four accesses have no registers for it)
    __shared__ float slots[2][NW];
    const int t = NW == 1 ? (threadIdx.x & 63) : threadIdx.x;
    const long long first = (long long)blockIdx.x * ROWS + (NW == 1 ? threadIdx.x >> 6 : 0), stride = (long long)gridDim.x * ROWS;
    if (first >= rows) return;                                 // whole waves, and only where no barrier follows (NW == 1)
    u32x4_t next_x[NV], next_r[NV], kw[NV][WN], kb[NV][WN];
    auto fetch = [&](long long row) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * TPR + t) * VEC;
            next_x[i] = load_raw_part<T>(x + row * D + c, D - c);
            if (res) next_r[i] = load_raw_part<T>(res + row * D + c, D - c);
        }
    };
    auto weights = [&](int i) {
#pragma unroll
        for (int k = 0; k < WN; ++k) {
            const int c = (i * TPR + t) * VEC + k * WV;
            if (w) kw[i][k] = load_raw_part<W>(w + c, D - c);
            if (b) kb[i][k] = load_raw_part<W>(b + c, D - c);
        }
    };
    if constexpr (AHEAD) {
        fetch(first);
#pragma unroll
        for (int i = 0; i < NV; ++i) weights(i);
    }
    for (long long row = first; row < rows; row += stride) {
        const long long base = row * D;
        float v[NV][VEC], s = 0.f;
        if constexpr (!AHEAD) fetch(row);
#pragma unroll
        for (int i = 0; i < NV; ++i) widen<T>(next_x[i], v[i]);
        if (res) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * TPR + t) * VEC;
                float r[VEC];
                widen<T>(next_r[i], r);
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[i][j] = to_f32(from_f32<T>(v[i][j] + r[j]));
                store_part<T, VEC>(h + base + c, D - c, v[i]);
            }
        }
        if (AHEAD && row + stride < rows) fetch(row + stride);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) s += v[i][j];
        const float mu = row_sum<NW>(s, slots[0]) / (float)D;
        s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * TPR + t) * VEC;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float d = c + j < D ? v[i][j] - mu : 0.f;
                v[i][j] = d;
                s = fmaf(d, d, s);
            }
        }
        const float rs = 1.f / sqrtf(row_sum<NW>(s, slots[1]) / (float)D + eps);
        if (t == 0) {
            mean[row] = mu;
            rstd[row] = rs;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * TPR + t) * VEC;
            if constexpr (!AHEAD) weights(i);
#pragma unroll
            for (int k = 0; k < WN; ++k) {
                float g[WV], o[WV];
                if (w) widen<W>(kw[i][k], g);
                if (b) widen<W>(kb[i][k], o);
#pragma unroll
                for (int j = 0; j < WV; ++j) {
                    float r = v[i][k * WV + j] * rs;
                    if (w) r *= g[j];
                    if (b) r += o[j];
                    v[i][k * WV + j] = r;
                }
            }
            store_part<T, VEC>(y + base + c, D - c, v[i]);
        }
    }
}

// rows that do not fit the registers of 16 waves: mean, squared differences and output in three walks
template <typename T, typename W>
__global__ __launch_bounds__(1024) void ln_forward_long_kernel(const T* __restrict__ x, const T* __restrict__ res, int D, const W* __restrict__ w,
                                                               const W* __restrict__ b, float eps, T* __restrict__ y, T* __restrict__ h,
                                                               float* __restrict__ mean, float* __restrict__ rstd) {
    constexpr int VEC = ElemOf<T>::VEC;
    __shared__ float slots[2][16];
    const long long row = blockIdx.x, base = row * D;
    const T* src = res ? h : x;
    float s = 0.f;
    for (long long c = threadIdx.x * VEC; c < D; c += 1024 * VEC) {
        float v[VEC];
        load_part<T, VEC>(x + base + c, D - c, v);
        if (res) {                                             // each thread re-reads only what it wrote itself
            float r[VEC];
            load_part<T, VEC>(res + base + c, D - c, r);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = to_f32(from_f32<T>(v[j] + r[j]));
            store_part<T, VEC>(h + base + c, D - c, v);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) s += v[j];
    }
    const float mu = row_sum<16>(s, slots[0]) / (float)D;
    s = 0.f;
    for (long long c = threadIdx.x * VEC; c < D; c += 1024 * VEC) {
        float v[VEC];
        load_part<T, VEC>(src + base + c, D - c, v, mu);
#pragma unroll
        for (int j = 0; j < VEC; ++j) s = fmaf(v[j] - mu, v[j] - mu, s);
    }
    const float rs = 1.f / sqrtf(row_sum<16>(s, slots[1]) / (float)D + eps);
    if (threadIdx.x == 0) {
        mean[row] = mu;
        rstd[row] = rs;
    }
    for (long long c = threadIdx.x * VEC; c < D; c += 1024 * VEC) {
        float v[VEC], g[VEC], o[VEC];
        load_part<T, VEC>(src + base + c, D - c, v);
        if (w) load_part<W, VEC>(w + c, D - c, g);
        if (b) load_part<W, VEC>(b + c, D - c, o);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            v[j] = (v[j] - mu) * rs;
            if (w) v[j] *= g[j];
            if (b) v[j] += o[j];
        }
        store_part<T, VEC>(y + base + c, D - c, v);
    }
}

// dx, and the block's sums of dy n and dy over its rows (every gridDim.x-th row group) into parts[block][2][D].  A thread owns the same 8 columns (16 of the
// longest rows) in every row, so the two sums and the weights stay in its registers, and the next row is on its way while this one is reduced; no
// atomics: the parts are added in block order by ln_sum_parts_kernel.  (16 columns a thread everywhere leave 2 to 4 waves on a SIMD:
// 16384 x 4096 bf16 with dh 136 us against 108.)
template <typename T, typename W, int NW, int NV>
__global__ __launch_bounds__(block_threads<NW>()) void ln_backward_kernel(const T* __restrict__ dy, const T* __restrict__ h, const T* __restrict__ dh,
                                                                           long long rows, int D, const W* __restrict__ w,
                                                                           const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                           T* __restrict__ dx, float* __restrict__ parts) {
    constexpr int VEC = ElemOf<T>::VEC, TPR = NW * 64, ROWS = NW == 1 ? 4 : 1;
    constexpr bool AHEAD = NV * VEC <= 8;
    __shared__ float slots[2][2][NW];                          // [row parity][sum][wave]: one barrier per row is enough
    const int t = NW == 1 ? (threadIdx.x & 63) : threadIdx.x, wave = threadIdx.x >> 6;
    float sw[NV][VEC], sb[NV][VEC], k[NV][VEC];
    auto weights = [&](int i) {
        const int c = (i * TPR + t) * VEC;
#pragma unroll
        for (int j = 0; j < VEC; ++j) k[i][j] = 1.f;
        if (w) load_part<W, VEC>(w + c, D - c, k[i]);
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if constexpr (AHEAD) weights(i);
#pragma unroll
        for (int j = 0; j < VEC; ++j) sw[i][j] = sb[i][j] = 0.f;
    }
    u32x4_t next_h[NV], next_dy[NV], next_dh[NV];
    float next_mu = 0.f, next_rs = 0.f;
    auto fetch = [&](long long row) {
        next_mu = mean[row];
        next_rs = rstd[row];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * TPR + t) * VEC;
            next_h[i] = load_raw_part<T>(h + row * D + c, D - c);
            next_dy[i] = load_raw_part<T>(dy + row * D + c, D - c);
            if (dh) next_dh[i] = load_raw_part<T>(dh + row * D + c, D - c);
        }
    };
    const long long first = (long long)blockIdx.x * ROWS + (NW == 1 ? wave : 0), stride = (long long)gridDim.x * ROWS;
    if (AHEAD && first < rows) fetch(first);
    int odd = 0;
    for (long long row = first; row < rows; row += stride, odd ^= 1) {
        const long long base = row * D;
        if constexpr (!AHEAD) fetch(row);
        const float mu = next_mu, rs = next_rs;
        float n[NV][VEC], g[NV][VEC], s1 = 0.f, s2 = 0.f;
        u32x4_t more[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            widen<T>(next_h[i], n[i]);
            widen<T>(next_dy[i], g[i]);
            more[i] = next_dh[i];
        }
        if (AHEAD && row + stride < rows) fetch(row + stride);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if constexpr (!AHEAD) weights(i);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                n[i][j] = (n[i][j] - mu) * rs;                 // (an absent column has dy = 0 and is not stored)
                sw[i][j] = fmaf(g[i][j], n[i][j], sw[i][j]);
                sb[i][j] += g[i][j];
                g[i][j] *= k[i][j];
                const bool there = (i * TPR + t) * VEC + j < D;
                s1 += there ? g[i][j] : 0.f;
                s2 += there ? g[i][j] * n[i][j] : 0.f;
            }
        }
        s1 = wave_sum(s1);
        s2 = wave_sum(s2);
        if constexpr (NW > 1) {
            if ((threadIdx.x & 63) == 0) {
                slots[odd][0][wave] = s1;
                slots[odd][1][wave] = s2;
            }
            __syncthreads();
            s1 = s2 = 0.f;
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                s1 += slots[odd][0][i];
                s2 += slots[odd][1][i];
            }
        }
        s1 /= (float)D;
        s2 /= (float)D;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * TPR + t) * VEC;
            if (c >= D) continue;
            float e[VEC];
            if (dh) widen<T>(more[i], e);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                float d = rs * (g[i][j] - s1 - n[i][j] * s2);
                if (dh) d += e[j];
                g[i][j] = d;
            }
            store_part<T, VEC>(dx + base + c, D - c, g[i]);
        }
    }
    if (!parts) return;
    float* out = parts + (long long)blockIdx.x * 2 * D;
    if constexpr (NW == 1) {                                   // the block's four waves walked different rows: add them in wave order
        __shared__ float red[3][64 * VEC];
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const float (&a)[VEC] = q ? sb[i] : sw[i];
                __syncthreads();
                if (wave)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) red[wave - 1][j * 64 + t] = a[j];
                __syncthreads();
                if (!wave) {
                    float v[VEC];
#pragma unroll
                    for (int j = 0; j < VEC; ++j) v[j] = ((a[j] + red[0][j * 64 + t]) + red[1][j * 64 + t]) + red[2][j * 64 + t];
                    const int c = (i * TPR + t) * VEC;
                    store_part<float, VEC>(out + (long long)q * D + c, D - c, v);
                }
            }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * TPR + t) * VEC;
            store_part<float, VEC>(out + c, D - c, sw[i]);
            store_part<float, VEC>(out + D + c, D - c, sb[i]);
        }
    }
}

// long rows: dx in two walks of the row
template <typename T, typename W>
__global__ __launch_bounds__(1024) void ln_backward_long_kernel(const T* __restrict__ dy, const T* __restrict__ h, const T* __restrict__ dh, int D,
                                                                const W* __restrict__ w, const float* __restrict__ mean,
                                                                const float* __restrict__ rstd, T* __restrict__ dx) {
    constexpr int VEC = ElemOf<T>::VEC;
    __shared__ float slots[2][16];
    const long long row = blockIdx.x, base = row * D;
    const float mu = mean[row], rs = rstd[row];
    float s1 = 0.f, s2 = 0.f;
    for (int walk = 0; walk < 2; ++walk) {
        for (long long c = threadIdx.x * VEC; c < D; c += 1024 * VEC) {
            float n[VEC], g[VEC], k[VEC], e[VEC];
            load_part<T, VEC>(h + base + c, D - c, n, mu);
            load_part<T, VEC>(dy + base + c, D - c, g);
            if (w) load_part<W, VEC>(w + c, D - c, k);
            if (walk && dh) load_part<T, VEC>(dh + base + c, D - c, e);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                n[j] = (n[j] - mu) * rs;
                if (w) g[j] *= k[j];
                if (!walk) {
                    s1 += g[j];
                    s2 = fmaf(g[j], n[j], s2);
                } else {
                    g[j] = rs * (g[j] - s1 - n[j] * s2);
                    if (dh) g[j] += e[j];
                }
            }
            if (walk) store_part<T, VEC>(dx + base + c, D - c, g);
        }
        if (!walk) {
            s1 = row_sum<16>(s1, slots[0]) / (float)D;
            s2 = row_sum<16>(s2, slots[1]) / (float)D;
        }
    }
}

// long rows: the sums over rows; a block owns 256 columns and every gridDim.y-th row
template <typename T>
__global__ __launch_bounds__(256) void ln_columns_kernel(const T* __restrict__ dy, const T* __restrict__ h, long long rows, int D,
                                                         const float* __restrict__ mean, const float* __restrict__ rstd, float* __restrict__ parts) {
    const long long c = (long long)blockIdx.x * 256 + threadIdx.x;
    if (c >= D) return;
    float sw = 0.f, sb = 0.f;
    for (long long r = blockIdx.y; r < rows; r += gridDim.y) {
        const float g = to_f32(dy[r * D + c]);
        sw = fmaf(g, (to_f32(h[r * D + c]) - mean[r]) * rstd[r], sw);
        sb += g;
    }
    parts[(long long)blockIdx.y * 2 * D + c] = sw;
    parts[(long long)blockIdx.y * 2 * D + D + c] = sb;
}

// dw[c] = sum over the parts, in part order within each of 16 strips and then strip order (a fixed tree).  blockIdx.y: 0 = dw, 1 = db
template <typename W>
__global__ __launch_bounds__(1024) void ln_sum_parts_kernel(const float* __restrict__ parts, int n_parts, int D, int from, W* __restrict__ dw, W* __restrict__ db) {
    __shared__ float red[16][64];
    W* out = blockIdx.y ? db : dw;
    const int lane = threadIdx.x & 63, strip = threadIdx.x >> 6, c = from + blockIdx.x * 64 + lane;
    float s = 0.f;
    if (out && c < D) {
        const float* p = parts + (long long)blockIdx.y * D + c;
#pragma unroll 8
        for (int k = strip; k < n_parts; k += 16) s += p[(long long)k * 2 * D];
    }
    red[strip][lane] = s;
    __syncthreads();
    if (strip == 0 && out && c < D) {
#pragma unroll
        for (int k = 1; k < 16; ++k) s += red[k][lane];
        out[c] = from_f32<W>(s);
    }
}

// A row is read in accesses of 16 bytes, NV of them per lane of its NW waves.  More waves are taken before more than two accesses per lane: with four, the
// registers of a 16-bit row leave two waves on a SIMD (4096 x 8192 bf16 with 4 waves of 4 accesses: forward 45 us, backward 77 to 120).
// Returns NW * 16 + NV, or 0 for a row that is too long.
int ln_forward_shape(int D, int vec) {
    const long long acc = ((long long)D + vec - 1) / vec;
    return acc <= 64 ? 17 : acc <= 128 ? 18 : acc <= 256 ? 34 : acc <= 512 ? 66 : acc <= 1024 ? 130 : acc <= 2048 ? 258 : acc <= 4096 ? 260 : 0;
}
// as many waves as the card holds at a time (20 on a CU), and each row (four for blocks of single waves) a block of its own below that
int ln_forward_blocks(long long rows, int nw) {
    const long long groups = nw == 1 ? (rows + 3) / 4 : rows, most = nw == 1 ? 256 * 5 : nw == 16 ? 256 : 256 * (20 / nw);
    return (int)(groups < most ? groups : most);
}
// waves to a row of the backward kernel, 8 columns a lane; 32: 16 waves with 16 columns; 0: too long
int ln_backward_waves(int D) { return D <= 512 ? 1 : D <= 1024 ? 2 : D <= 2048 ? 4 : D <= 4096 ? 8 : D <= 8192 ? 16 : D <= 16384 ? 32 : 0; }
// As many blocks as the card holds at a time (16 waves on a CU), of at least four rows where that leaves a block for every CU: a block's sums are
// written and read again.
int ln_backward_blocks(long long rows, int D) {
    const int nw = ln_backward_waves(D);
    const long long groups = nw == 1 ? (rows + 3) / 4 : rows, most = nw == 1 ? 1024 : nw == 0 || nw >= 16 ? 256 : 256 * (16 / nw);
    long long n = nw == 1 ? groups : (groups + 3) / 4;
    if (n < 256) n = groups < 256 ? groups : 256;
    return (int)(n < most ? n : most);
}

template <typename T, typename W>
int ln_forward(const void* x, const void* res, long long rows, int D, const void* w, const void* b, float eps, void* y, void* h, float* mean,
               float* rstd, hipStream_t st) {
    const int shape = ln_forward_shape(D, ElemOf<T>::VEC);
#define LN_FWD(NW, NV)                                                                                                                          \
    case NW * 16 + NV:                                                                                                                          \
        hipLaunchKernelGGL((ln_forward_kernel<T, W, NW, NV>), dim3(ln_forward_blocks(rows, NW)), dim3(block_threads<NW>()), 0, st, \
                           (const T*)x, (const T*)res, rows, D, (const W*)w, (const W*)b, eps, (T*)y, (T*)h, mean, rstd);                       \
        break;
    switch (shape) {
        LN_FWD(1, 1) LN_FWD(1, 2) LN_FWD(2, 2) LN_FWD(4, 2) LN_FWD(8, 2) LN_FWD(16, 2) LN_FWD(16, 4)
    default:
        hipLaunchKernelGGL((ln_forward_long_kernel<T, W>), dim3((unsigned)rows), dim3(1024), 0, st, (const T*)x, (const T*)res, D, (const W*)w,
                           (const W*)b, eps, (T*)y, (T*)h, mean, rstd);
    }
#undef LN_FWD
    return w2c_launch_status();
}

template <typename T, typename W>
int ln_backward(const void* dy, const void* h, const void* dh, long long rows, int D, const void* w, const float* mean, const float* rstd, void* dx,
                void* dw, void* db, float* parts, hipStream_t st) {
    constexpr int EIGHT = 8 / ElemOf<T>::VEC;
    const int nb = ln_backward_blocks(rows, D);
    if (!dw && !db) parts = nullptr;
#define LN_BWD(WAVES, NW, NV)                                                                                                                \
    case WAVES:                                                                                                                              \
        hipLaunchKernelGGL((ln_backward_kernel<T, W, NW, NV>), dim3(nb), dim3(block_threads<NW>()), 0, st, (const T*)dy, (const T*)h,         \
                           (const T*)dh, rows, D, (const W*)w, mean, rstd, (T*)dx, parts);                                                   \
        break;
    switch (ln_backward_waves(D)) {
        LN_BWD(1, 1, EIGHT) LN_BWD(2, 2, EIGHT) LN_BWD(4, 4, EIGHT) LN_BWD(8, 8, EIGHT) LN_BWD(16, 16, EIGHT) LN_BWD(32, 16, 2 * EIGHT)
    default:
        hipLaunchKernelGGL((ln_backward_long_kernel<T, W>), dim3((unsigned)rows), dim3(1024), 0, st, (const T*)dy, (const T*)h, (const T*)dh, D,
                           (const W*)w, mean, rstd, (T*)dx);
        if (parts)
            hipLaunchKernelGGL((ln_columns_kernel<T>), dim3((D + 255) / 256, nb), dim3(256), 0, st, (const T*)dy, (const T*)h, rows, D, mean, rstd,
                               parts);
    }
#undef LN_BWD
    constexpr int MOST = (int)most_blocks(1024);
    for (int from = 0; parts && from < D; from += 64 * MOST) {
        const int blocks = (D - from + 63) / 64;
        hipLaunchKernelGGL((ln_sum_parts_kernel<W>), dim3(blocks < MOST ? blocks : MOST, 2), dim3(1024), 0, st, (const float*)parts, nb, D, from, (W*)dw,
                           (W*)db);
    }
    return w2c_launch_status();
}

// rows of more than 16 384 columns take a block of 1024 threads each, in one launch
bool ln_shape_ok(long long rows, int cols) {
    return rows >= 1 && rows <= 0x7FFFFFFF && cols >= 1 && cols <= (1 << 30) && (cols <= 16384 || rows <= most_blocks(1024));
}
bool ln_types_ok(int dtype, int wtype) { return dtype >= W2C_F32 && dtype <= W2C_F16 && (wtype == W2C_F32 || wtype == dtype); }

}  // namespace

extern "C" int w2c_layer_norm_forward(const void* x, const void* residual, int dtype, long long rows, int cols, const void* weight, const void* bias,
                                      int wtype, float eps, void* y, void* h, float* mean, float* rstd, void* stream) {
    if (!x || !y || !mean || !rstd || (residual && !h) || !ln_types_ok(dtype, wtype)) return W2C_E_ARG;
    if (!ln_shape_ok(rows, cols)) return W2C_E_ARG;
    w2c_clear_error();
    const hipStream_t st = (hipStream_t)stream;
#define LN_CALL(T, W) return ln_forward<T, W>(x, residual, rows, cols, weight, bias, eps, y, h, mean, rstd, st)
    if (dtype == W2C_F32) LN_CALL(float, float);
    if (dtype == W2C_BF16) {
        if (wtype == W2C_F32) LN_CALL(bf16_t, float);
        LN_CALL(bf16_t, bf16_t);
    }
    if (wtype == W2C_F32) LN_CALL(f16_t, float);
    LN_CALL(f16_t, f16_t);
#undef LN_CALL
}

extern "C" long long w2c_layer_norm_workspace_bytes(long long rows, int cols, int dtype) {
    if (!ln_shape_ok(rows, cols) || dtype < W2C_F32 || dtype > W2C_F16) return W2C_E_ARG;
    return (long long)ln_backward_blocks(rows, cols) * 2 * cols * (long long)sizeof(float);
}

extern "C" int w2c_layer_norm_backward(const void* dy, const void* h, const void* dh, int dtype, long long rows, int cols, const void* weight,
                                       int wtype, const float* mean, const float* rstd, void* dx, void* dweight, void* dbias, void* workspace,
                                       long long workspace_bytes, void* stream) {
    if (!dy || !h || !mean || !rstd || !dx || !ln_types_ok(dtype, wtype)) return W2C_E_ARG;
    if (!ln_shape_ok(rows, cols)) return W2C_E_ARG;
    if ((dweight || dbias) && (!workspace || workspace_bytes < w2c_layer_norm_workspace_bytes(rows, cols, dtype))) return W2C_E_ARG;
    w2c_clear_error();
    const hipStream_t st = (hipStream_t)stream;
#define LN_CALL(T, W) return ln_backward<T, W>(dy, h, dh, rows, cols, weight, mean, rstd, dx, dweight, dbias, (float*)workspace, st)
    if (dtype == W2C_F32) LN_CALL(float, float);
    if (dtype == W2C_BF16) {
        if (wtype == W2C_F32) LN_CALL(bf16_t, float);
        LN_CALL(bf16_t, bf16_t);
    }
    if (wtype == W2C_F32) LN_CALL(f16_t, float);
    LN_CALL(f16_t, f16_t);
#undef LN_CALL
}
