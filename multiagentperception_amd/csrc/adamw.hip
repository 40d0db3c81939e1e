// One AdamW step over many tensors, with the two moments in 32 or in 8 bits, and the gradients' total norm.
//
//   t += 1;   g <- g * min(1, max_norm / (|all g| + 1e-6))
//   m = b1 m + (1 - b1) g;   v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)            in f32, rounded once to p's type
//
// HBM-bound: f32 parameters move 28 bytes an element with 32-bit moments, 16 with 8-bit ones.  Tensors travel as tables in the kernel
// arguments (60 to 190 a launch), so nothing is copied to the device, nothing is kept between calls and a captured step replays as it is; a
// block finds its tensor by bisecting the table's prefix of chunks.  The step counters live on the device: one small launch advances them and
// leaves each tensor's factors for the launches behind it.
//
// 8-bit moments: m and r = sqrt(v) (the root halves the range to cover) as e4m3 codes, 256 elements to a power-of-two scale.  b2 = 0.999 moves v by
// a thousandth of itself per step, far less than half a step of any 8-bit code: rounded to nearest, v would never decay.  So both are
// rounded up or down at random with the distance as the chance (the mean of m and of the root is kept, v's grows by the root's variance: some per cent of
// what b2 = 0.999 takes off it in a step; a value that did not move keeps its code).  The random bits are a hash of (seed, t, place), so a step
// gives the same bits every time, and tensors of one call are rounded alike at the same place.  A root above 0 keeps a code above 0: m / r stays bounded.  The step
// itself uses m and v before they are rounded.  Codes of values that are not finite are NaN; the scale comes from the others.
#include "lm_common.h"

namespace {

// tensors of a launch's table, by the 4 KiB that kernel arguments may take: 48 bytes a tensor with 32-bit moments, 64 with 8-bit ones, 20 for the norm
constexpr int AW_TENSORS32 = 80, AW_TENSORS8 = 60, SQ_TENSORS = 190;
constexpr int AW_STEPS = 256;             // step counters per launch
constexpr int AW_STATE = 256;             // elements per 8-bit scale
constexpr int AW_FIELDS = 9;              // of a tensor's row in the C ABI: p, g, m, v, m_scale, v_scale, step, n, dtype
constexpr int AW_CHUNK = 4096;            // elements per block
constexpr int SQ_CHUNK = 16384, SQ_MOST = 1024;
constexpr long long AW_BLOCKS = most_blocks(256), AW_ELEMENTS = AW_BLOCKS * AW_CHUNK;      // of a launch; of a tensor: its blocks fit one launch

template <int TENSORS>
struct Table32 {
    void* p[TENSORS];
    const void* g[TENSORS];
    void* m[TENSORS];
    void* v[TENSORS];
    long long n[TENSORS];
    int first[TENSORS];                   // the tensor's first block in this launch
    int factors[TENSORS];                 // its row of factors
    int tensors;
};
struct Table8 : Table32<AW_TENSORS8> {
    uint8_t* ms[AW_TENSORS8];
    uint8_t* vs[AW_TENSORS8];
};
static_assert(sizeof(Table32<AW_TENSORS32>) <= 4000 && sizeof(Table8) <= 4000, "a table and the other arguments");
struct Factors {                          // of one tensor in this step
    float step_size, root_scale, decay, clip;
    uint32_t key, pad[3];
};
struct StepTable {
    float* step[AW_STEPS];
    int count, first;
};

__device__ __forceinline__ int find_tensor(const int* first, int tensors, int block) {
    int lo = 0, hi = tensors - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= block) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// one block: the norm from the partial sums of squares, then a thread per tensor
__global__ __launch_bounds__(256) void adamw_begin_kernel(StepTable s, const double* __restrict__ squares, int n_squares, double max_norm,
                                                          float* __restrict__ norm_out, double lr, const float* __restrict__ lr_dev, double b1,
                                                          double b2, double wd, uint32_t seed, Factors* __restrict__ out) {
    float clip = 1.f;
    if (n_squares) {
        __shared__ double red[4];
        double a = 0.0;
        for (int i = threadIdx.x; i < n_squares; i += 256) a += squares[i];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) a += __shfl_xor(a, o, 64);
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
        __syncthreads();
        const double norm = sqrt((red[0] + red[1]) + (red[2] + red[3]));
        const double f = max_norm / (norm + 1e-6);
        clip = f > 1.0 ? 1.f : (float)f;                     // a norm that is NaN stays NaN
        if (threadIdx.x == 0 && norm_out) *norm_out = (float)norm;
    }
    const int i = threadIdx.x;
    if (i >= s.count) return;
    const float t = *s.step[i] + 1.f;
    *s.step[i] = t;
    if (lr_dev) lr = (double)*lr_dev;
    Factors f;
    f.step_size = (float)(lr / (1.0 - pow(b1, (double)t)));
    f.root_scale = (float)(1.0 / sqrt(1.0 - pow(b2, (double)t)));
    f.decay = (float)(1.0 - lr * wd);
    f.clip = clip;
    f.key = seed * 0x9E3779B1u + (uint32_t)(long long)t * 0x85EBCA6Bu;
    f.pad[0] = f.pad[1] = f.pad[2] = 0;
    out[s.first + i] = f;
}

struct Rates {
    float b1, c1, b2, c2, eps;            // c = 1 - b, formed in 64 bits
};
// (p, m, v) of one element -> the next; r = sqrt(v).  An element whose root and eps are both 0 (no gradient yet, or one whose square is below f32) has no
// direction: it is decayed and else left as it is.  HARDWARE: the root and reciprocal instructions, each within a step of f32 (the root's input
// lifted out of the subnormals, which it takes for 0), for 8-bit moments, whose step is bound by instructions as much as by memory and which are
// rounded at random to a few bits behind it.  (134 M elements, with the instructions as they are / lifted and guarded: 8 bits f32 429 / 430 us, bf16
// 278 / 287; 32 bits exact 708, 615, as before)
template <bool HARDWARE>
__device__ __forceinline__ void adamw_element(const Rates& k, const Factors& f, float g, float& p, float& m, float& v, float& r) {
    constexpr float LEAST = 0x1p-126f;
    g *= f.clip;
    m = k.b1 * m + k.c1 * g;
    v = k.b2 * v + k.c2 * (g * g);
    if constexpr (HARDWARE) {
        const bool low = v < LEAST;
        r = __builtin_amdgcn_sqrtf(low ? v * 0x1p64f : v);
        r = low ? r * 0x1p-32f : r;
    } else
        r = sqrtf(v);
    const float d = r * f.root_scale + k.eps;
    if constexpr (HARDWARE) p = p * f.decay - f.step_size * (m * (d < LEAST ? 0.f : __builtin_amdgcn_rcpf(d)));
    else p = p * f.decay - f.step_size * (d < LEAST ? 0.f : m / d);
}

template <typename T>
__global__ __launch_bounds__(256) void adamw32_kernel(Table32<AW_TENSORS32> t, const Factors* __restrict__ factors, Rates k) {
    constexpr int VEC = ElemOf<T>::VEC;
    const int i = find_tensor(t.first, t.tensors, blockIdx.x);
    const long long base = (long long)(blockIdx.x - t.first[i]) * AW_CHUNK, n = t.n[i];
    const Factors f = factors[t.factors[i]];
    T* P = (T*)t.p[i];
    const T* G = (const T*)t.g[i];
    float *M = (float*)t.m[i], *V = (float*)t.v[i];
#pragma unroll
    for (int it = 0; it < AW_CHUNK / (256 * VEC); ++it) {
        const long long c = base + (it * 256 + threadIdx.x) * VEC;
        float p[VEC], g[VEC], m[VEC], v[VEC], r;
        load_part<T, VEC>(P + c, n - c, p);
        load_part<T, VEC>(G + c, n - c, g);
        load_part<float, VEC>(M + c, n - c, m);
        load_part<float, VEC>(V + c, n - c, v);
#pragma unroll
        for (int j = 0; j < VEC; ++j) adamw_element<false>(k, f, g[j], p[j], m[j], v[j], r);
        store_part<T, VEC>(P + c, n - c, p);
        store_part<float, VEC>(M + c, n - c, m);
        store_part<float, VEC>(V + c, n - c, v);
    }
}

// the bits of a place: `x` = place * 0xA3D8F62B + (place >> 32) * 0xC2B2AE35 + key
__device__ __forceinline__ uint32_t random_bits(uint32_t x) {
    x = (x ^ (x >> 15)) * 0xC58B3E95u;
    x = (x ^ (x >> 13)) * 0x9E3779B1u;
    return x ^ (x >> 16);
}
__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u; }
// The e4m3 code of |x| <= 448 2^e, sign aside.  x * 2^(-e - 120) puts e4m3's exponent and mantissa fields (subnormals too) into bits 20.. of the f32: 20
// random bits below them and a cut round up with the cut-off part's share of a step as the chance.
__device__ __forceinline__ uint32_t code_of(float x, int e, uint32_t noise20) {
    return ((__float_as_uint(__builtin_amdgcn_ldexpf(x, -120 - e)) & 0x7FFFFFFFu) + noise20) >> 20;
}

// one block of 256 of a tensor: WHOLE, or its last `left` (counted from this lane's first element)
template <typename T, bool WHOLE>
__device__ __forceinline__ void adamw8_block(const Factors& f, const Rates& k, T* P, const T* G, uint8_t* M, uint8_t* V, uint8_t* ms, uint8_t* vs,
                                             long long place, long long left, int lane) {
    constexpr int VEC = 4;                                    // elements per lane
    float p[VEC], g[VEC], m[VEC], r[VEC];
    uint32_t mc = 0, vc = 0;
    if constexpr (WHOLE) {
        load_n<T, VEC>(P, p);
        load_n<T, VEC>(G, g);
        __builtin_memcpy(&mc, M, 4);
        __builtin_memcpy(&vc, V, 4);
    } else {
        load_part<T, VEC>(P, left, p);
        load_part<T, VEC>(G, left, g);
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if (j < left) {
                mc |= (uint32_t)M[j] << (8 * j);
                vc |= (uint32_t)V[j] << (8 * j);
            }
    }
    const float sm = pow2f((int)*ms - 127), sv = pow2f((int)*vs - 127);
    m[0] = __builtin_amdgcn_cvt_f32_fp8(mc, 0) * sm;
    m[1] = __builtin_amdgcn_cvt_f32_fp8(mc, 1) * sm;
    m[2] = __builtin_amdgcn_cvt_f32_fp8(mc, 2) * sm;
    m[3] = __builtin_amdgcn_cvt_f32_fp8(mc, 3) * sm;
    r[0] = __builtin_amdgcn_cvt_f32_fp8(vc, 0) * sv;
    r[1] = __builtin_amdgcn_cvt_f32_fp8(vc, 1) * sv;
    r[2] = __builtin_amdgcn_cvt_f32_fp8(vc, 2) * sv;
    r[3] = __builtin_amdgcn_cvt_f32_fp8(vc, 3) * sv;
    float am = 0.f, ar = 0.f, odd = 0.f;                      // odd: NaN where a value is not finite
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        float v = r[j] * r[j];
        adamw_element<true>(k, f, g[j], p[j], m[j], v, r[j]);
        if (!WHOLE && j >= left) m[j] = r[j] = 0.f;
        am = __builtin_fmaxf(am, __builtin_fabsf(m[j]));
        ar = __builtin_fmaxf(ar, r[j]);
        odd = fmaf(m[j], 0.f, fmaf(r[j], 0.f, odd));
    }
    if constexpr (WHOLE) store_n<T, VEC>(P, p);
    else store_part<T, VEC>(P, left, p);
    const bool any_odd = __any(odd != 0.f);                   // (NaN != 0)
    if (any_odd) {                                            // rare: the scale comes from the finite values
        am = ar = 0.f;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            if (finite(m[j])) am = __builtin_fmaxf(am, __builtin_fabsf(m[j]));
            if (finite(r[j])) ar = __builtin_fmaxf(ar, r[j]);
        }
    }
    const int em = scale_exponent(wave_max(am)), ev = scale_exponent(wave_max(ar));
    const uint32_t seed = (uint32_t)place * 0xA3D8F62Bu + (uint32_t)(place >> 32) * 0xC2B2AE35u + f.key;
    mc = vc = 0;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        // (a block's places share their upper half: 256 divides 2^32)
        const uint32_t x = random_bits(seed + (uint32_t)j * 0xA3D8F62Bu);
        uint32_t cm = code_of(m[j], em, (x << 4 & 0xFFFF0u) + 8u) | (__float_as_uint(m[j]) >> 24 & 0x80u);
        uint32_t cv = code_of(r[j], ev, (x >> 16 << 4) + 8u);
        const uint32_t least = __float_as_uint(r[j]) < 1u ? __float_as_uint(r[j]) : 1u;        // a root above 0 keeps a code above 0
        cv = cv < least ? least : cv;
        if (any_odd) {
            cm = finite(m[j]) ? cm : 0x7Fu;
            cv = finite(r[j]) ? cv : 0x7Fu;
        }
        mc |= cm << (8 * j);
        vc |= cv << (8 * j);
    }
    if constexpr (WHOLE) {
        __builtin_memcpy(M, &mc, 4);
        __builtin_memcpy(V, &vc, 4);
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if (j < left) {
                M[j] = (uint8_t)(mc >> (8 * j));
                V[j] = (uint8_t)(vc >> (8 * j));
            }
    }
    if (lane == 0) {
        *ms = (uint8_t)(em + 127);
        *vs = (uint8_t)(ev + 127);
    }
}

// a wave per block of 256; nothing is shared between waves
template <typename T>
__global__ __launch_bounds__(256) void adamw8_kernel(Table8 t, const Factors* __restrict__ factors, Rates k) {
    const int i = find_tensor(t.first, t.tensors, blockIdx.x);
    const long long n = t.n[i];
    const Factors f = factors[t.factors[i]];
    T* P = (T*)t.p[i];
    const T* G = (const T*)t.g[i];
    uint8_t *M = (uint8_t*)t.m[i], *V = (uint8_t*)t.v[i];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    long long s = (long long)(blockIdx.x - t.first[i]) * (AW_CHUNK / AW_STATE) + wave;
    for (int it = 0; it < AW_CHUNK / AW_STATE / 4; ++it, s += 4) {
        const long long first = s * AW_STATE, c = first + lane * 4;
        if (first >= n) return;
        if (first + AW_STATE <= n) adamw8_block<T, true>(f, k, P + c, G + c, M + c, V + c, t.ms[i] + s, t.vs[i] + s, c, 0, lane);
        else adamw8_block<T, false>(f, k, P + c, G + c, M + c, V + c, t.ms[i] + s, t.vs[i] + s, c, n - c, lane);
    }
}

struct SquareTable {
    const void* g[SQ_TENSORS];
    long long n[SQ_TENSORS];
    int first[SQ_TENSORS];                // the tensor's first chunk of SQ_CHUNK
    int tensors, chunks;
};
static_assert(sizeof(SquareTable) <= 4000, "a table and the other arguments");
// a block's sum of squares over every gridDim.x-th chunk, in 64 bits (an f32 square overflows at 1.8e19)
template <typename T>
__global__ __launch_bounds__(256) void grad_squares_kernel(SquareTable t, double* __restrict__ out) {
    constexpr int VEC = ElemOf<T>::VEC;
    __shared__ double red[4];
    double a = 0.0;
    for (int q = blockIdx.x; q < t.chunks; q += gridDim.x) {
        const int i = find_tensor(t.first, t.tensors, q);
        const long long base = (long long)(q - t.first[i]) * SQ_CHUNK, n = t.n[i];
        const T* G = (const T*)t.g[i];
        for (int it = 0; it < SQ_CHUNK / (256 * VEC); ++it) {
            const long long c = base + (it * 256 + threadIdx.x) * VEC;
            if (c >= n) break;
            float g[VEC];
            load_part<T, VEC>(G + c, n - c, g);
#pragma unroll
            for (int j = 0; j < VEC; ++j) a = fma((double)g[j], (double)g[j], a);
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) a += __shfl_xor(a, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
    __syncthreads();
    if (threadIdx.x == 0) out[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

const long long* row(const long long* tensors, int i) { return tensors + (long long)i * AW_FIELDS; }
bool aw_rows_ok(const long long* tensors, int n) {
    if (!tensors || n < 1) return false;
    for (int i = 0; i < n; ++i) {
        const long long* r = row(tensors, i);
        if (r[7] < 0 || r[7] > AW_ELEMENTS || r[8] < W2C_F32 || r[8] > W2C_F16 || (r[7] && !r[1])) return false;
    }
    return true;
}

// walks the tensors of one element type in launches of at most `most` tensors and AW_BLOCKS blocks; add(row, index, first block, blocks), flush(blocks)
template <typename Add, typename Flush>
bool aw_batches(const long long* tensors, int n, int dtype, int most, long long chunk, Add add, Flush flush) {
    int count = 0;
    long long blocks = 0;
    for (int i = 0; i < n; ++i) {
        const long long* r = row(tensors, i);
        if (r[8] != dtype || r[7] == 0) continue;
        const long long need = (r[7] + chunk - 1) / chunk;
        if (count && (count == most || blocks + need > AW_BLOCKS)) {
            if (!flush(count, (int)blocks)) return false;
            count = 0;
            blocks = 0;
        }
        add(r, i, count++, (int)blocks);
        blocks += need;
    }
    return !count || flush(count, (int)blocks);
}

int squares_blocks(const long long* tensors, int n, double* out, hipStream_t st, bool launch, int* status) {
    int total = 0;
    for (int dtype = W2C_F32; dtype <= W2C_F16; ++dtype) {
        SquareTable t;
        aw_batches(
            tensors, n, dtype, SQ_TENSORS, SQ_CHUNK,
            [&](const long long* r, int, int at, int first) {
                t.g[at] = (const void*)r[1];
                t.n[at] = r[7];
                t.first[at] = first;
            },
            [&](int count, int chunks) {
                t.tensors = count;
                t.chunks = chunks;
                const int blocks = chunks < SQ_MOST ? chunks : SQ_MOST;
                if (launch) {
                    if (dtype == W2C_F32) hipLaunchKernelGGL((grad_squares_kernel<float>), dim3(blocks), dim3(256), 0, st, t, out + total);
                    else if (dtype == W2C_BF16) hipLaunchKernelGGL((grad_squares_kernel<bf16_t>), dim3(blocks), dim3(256), 0, st, t, out + total);
                    else hipLaunchKernelGGL((grad_squares_kernel<f16_t>), dim3(blocks), dim3(256), 0, st, t, out + total);
                    *status = w2c_launch_status();
                }
                total += blocks;
                return !launch || *status == W2C_OK;
            });
        if (launch && *status != W2C_OK) return -1;
    }
    return total;
}

}  // namespace

extern "C" int w2c_grad_squares_count(const long long* tensors, int n) {
    return aw_rows_ok(tensors, n) ? squares_blocks(tensors, n, nullptr, nullptr, false, nullptr) : W2C_E_ARG;
}

extern "C" int w2c_grad_squares(const long long* tensors, int n, double* squares, int count, void* stream) {
    if (!aw_rows_ok(tensors, n) || !squares || count < w2c_grad_squares_count(tensors, n)) return W2C_E_ARG;
    w2c_clear_error();
    int status = W2C_OK;
    squares_blocks(tensors, n, squares, (hipStream_t)stream, true, &status);
    return status;
}

extern "C" long long w2c_adamw_workspace_bytes(int n) { return n < 1 ? W2C_E_ARG : (long long)n * (long long)sizeof(Factors); }

extern "C" int w2c_adamw_step(const long long* tensors, int n, int state_bits, double lr, const float* lr_dev, double beta1, double beta2, double eps,
                              double weight_decay, const double* squares, int n_squares, double max_norm, float* norm, unsigned seed, void* workspace,
                              long long workspace_bytes, void* stream) {
    if (!aw_rows_ok(tensors, n) || (state_bits != 8 && state_bits != 32) || !workspace || workspace_bytes < w2c_adamw_workspace_bytes(n)) return W2C_E_ARG;
    if ((reinterpret_cast<uintptr_t>(workspace) & 15) || n_squares < 0 || (n_squares && !squares)) return W2C_E_ARG;
    for (int i = 0; i < n; ++i) {
        const long long* r = row(tensors, i);
        if (!r[6] || (r[7] && (!r[0] || !r[2] || !r[3] || (state_bits == 8 && (!r[4] || !r[5]))))) return W2C_E_ARG;
    }
    w2c_clear_error();
    const hipStream_t st = (hipStream_t)stream;
    Factors* factors = (Factors*)workspace;
    for (int first = 0; first < n; first += AW_STEPS) {
        StepTable s;
        s.first = first;
        s.count = n - first < AW_STEPS ? n - first : AW_STEPS;
        for (int i = 0; i < s.count; ++i) s.step[i] = (float*)row(tensors, first + i)[6];
        hipLaunchKernelGGL(adamw_begin_kernel, dim3(1), dim3(256), 0, st, s, squares, n_squares, max_norm, norm, lr, lr_dev, beta1, beta2,
                           weight_decay, seed, factors);
        const int status = w2c_launch_status();
        if (status != W2C_OK) return status;
    }
    const Rates k{(float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps};
    int status = W2C_OK;
    auto fill = [](auto& t, const long long* r, int i, int at, int first) {
        t.p[at] = (void*)r[0];
        t.g[at] = (const void*)r[1];
        t.m[at] = (void*)r[2];
        t.v[at] = (void*)r[3];
        t.n[at] = r[7];
        t.first[at] = first;
        t.factors[at] = i;
    };
#define AW_LAUNCH(KERNEL, T) hipLaunchKernelGGL((KERNEL<T>), dim3(blocks), dim3(256), 0, st, t, (const Factors*)factors, k)
#define AW_FLUSH(KERNEL)                                      \
    [&](int count, int blocks) {                              \
        t.tensors = count;                                    \
        if (dtype == W2C_F32) AW_LAUNCH(KERNEL, float);       \
        else if (dtype == W2C_BF16) AW_LAUNCH(KERNEL, bf16_t); \
        else AW_LAUNCH(KERNEL, f16_t);                        \
        status = w2c_launch_status();                         \
        return status == W2C_OK;                              \
    }
    for (int dtype = W2C_F32; dtype <= W2C_F16; ++dtype) {
        if (state_bits == 32) {
            Table32<AW_TENSORS32> t;
            aw_batches(
                tensors, n, dtype, AW_TENSORS32, AW_CHUNK, [&](const long long* r, int i, int at, int first) { fill(t, r, i, at, first); },
                AW_FLUSH(adamw32_kernel));
        } else {
            Table8 t;
            aw_batches(
                tensors, n, dtype, AW_TENSORS8, AW_CHUNK,
                [&](const long long* r, int i, int at, int first) {
                    fill(t, r, i, at, first);
                    t.ms[at] = (uint8_t*)r[4];
                    t.vs[at] = (uint8_t*)r[5];
                },
                AW_FLUSH(adamw8_kernel));
        }
        if (status != W2C_OK) return status;
    }
#undef AW_FLUSH
#undef AW_LAUNCH
    return W2C_OK;
}
