// Log probabilities of given classes, with the entropy and the top alternatives of every row, and the gradient to the logits.
//
//   m = max_j x_j,  s = sum_j exp(x_j - m),  u = sum_j exp(x_j - m) (x_j - m)          one walk: (m, s, u) is rescaled when m grows
//   log p_j = (x_j - m) - log s,   H = log s - u / s,   alternatives: the largest x_j, equal ones by the lower index
//   dx_j = a_t [j = t] + sum_i b_i [j = top_i] - p_j (a_t + sum_i b_i + c (log p_j + H))       a, b, c: gradients of log p_t, log p_top, H
//
// (m, log s) are kept apart for the backward: their sum would cost the last digits of p where the logits are large.  A masked class is -inf
// (p = 0, no gradient); a row without any other class answers -inf, H = 0 and no gradient.  NaN or +inf make the row's answers NaN.  A target
// outside [0, C) that is not ignore_index answers NaN.
//
// HBM-bound: one read forward, one read and one write backward.  Three shapes of work:
//   lane per row   class dimension strided (label maps) or at most 64 classes: 64 neighbouring rows per wave, alternatives in registers
//   wave per row   up to 2 048 contiguous classes; a wave for one or two rows that fit its registers (about 500 classes)
//   block per row or per part of a row   longer; few long rows are split over blocks and joined by a second launch
// Alternatives of the last two: every thread keeps the largest (value, index) of what it read; the k-th largest of those is a bound that
// at most k threads reach, and only their values are looked through again.
#include "lm_common.h"

namespace {

constexpr float LP_L2E = 1.44269504088896340736f;
constexpr float LP_FLOOR = -200.f;            // exp(-200) is 0 in f32: stands for -inf where 0 * -inf would be NaN
constexpr int LP_TOP_MOST = 32, LP_SPLIT_MOST = 64;
constexpr int LP_LANE_MOST = 64, LP_WAVE_MOST = 2048;      // classes

// exp(d): the hardware's 2^x of the rounded d log2(e).  That rounding is half a step of f32 of the argument, |d| 2^-24 of the result, beside the
// instruction's own step: d = 10 below the row's largest, a term is off by 6e-7 of itself and adds 3e-11 of the sum.
__device__ __forceinline__ float exp_d(float d) { return __builtin_amdgcn_exp2f(d * LP_L2E); }

struct Run {                                  // of the values seen so far
    float m, s, u;
};
// max first, then the sums against it; m = -inf (nothing but masked values) counts from 0
__device__ __forceinline__ void run_raise(Run& r, float m) {
    if (m > r.m) {
        const float d = r.m - m, f = exp_d(d);
        r.u = f * (r.u + r.s * __builtin_fmaxf(d, LP_FLOOR));
        r.s *= f;
        r.m = m;
    }
}
template <int N>
__device__ __forceinline__ float max_of(const float (&x)[N]) {
    float m = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = __builtin_fmaxf(m, x[i]);
    return m;
}
template <int N>
__device__ __forceinline__ void run_add(Run& r, const float (&x)[N], float chunk_max) {
    run_raise(r, chunk_max);
    const float base = r.m == -INFINITY ? 0.f : r.m;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float d = x[i] - base, e = exp_d(d);
        r.s += e;
        r.u = fmaf(e, __builtin_fmaxf(d, LP_FLOOR), r.u);
    }
}
__device__ __forceinline__ void run_to(Run& r, float m) {           // restate against a larger (or equal) maximum
    run_raise(r, m);
}
__device__ __forceinline__ Run wave_join(Run r) {
    run_to(r, wave_max(r.m));
    r.s = wave_sum(r.s);
    r.u = wave_sum(r.u);
    return r;
}

// order of the alternatives: larger value first, then lower index; NaN ranks as -inf.  0 = none
typedef unsigned long long key_t;
__device__ __forceinline__ uint32_t ordered(float v) {               // not below 2^22: -inf is 0x007FFFFF
    const uint32_t b = __float_as_uint(__builtin_fmaxf(v, -INFINITY) + 0.f);               // NaN to -inf, -0 to +0
    return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o); }
__device__ __forceinline__ key_t key_of(float v, int index) { return (key_t)ordered(v) << 32 | (uint32_t)~index; }
__device__ __forceinline__ int key_index(key_t k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ float key_value(key_t k) { return unordered((uint32_t)(k >> 32)); }
__device__ __forceinline__ uint32_t wave_max_bits(uint32_t v) {
    return wave_reduce(v, [](uint32_t a, auto ctrl, auto rows) {
        const uint32_t p = dpp<decltype(ctrl)::value, decltype(rows)::value>(0u, a);
        return p > a ? p : a;
    });
}
// of all 64 lanes: the largest value, then the lowest index of the lanes that have it (mostly one)
__device__ __forceinline__ key_t wave_max_key(key_t k) {
    const uint32_t value = (uint32_t)(k >> 32), best = wave_max_bits(value);
    const unsigned long long have = __ballot(value == best);
    const uint32_t index = have & (have - 1) ? wave_max_bits(value == best ? (uint32_t)k : 0u)
                                             : (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)k, __builtin_ctzll(have));
    return (key_t)best << 32 | index;
}

// bf16 and f16 values leave 13 bits of an ordered f32 unused, and the class fits there where there are at most 8 192
constexpr int LP_PACKED_CLASSES = 8192;
constexpr uint32_t LP_PACKED = LP_PACKED_CLASSES - 1;
__device__ __forceinline__ uint32_t packed_key(float v, int index) { return (ordered(v) & ~LP_PACKED) | (~(uint32_t)index & LP_PACKED); }
__device__ __forceinline__ int key_index(uint32_t k) { return (int)(LP_PACKED - (k & LP_PACKED)); }
__device__ __forceinline__ float key_value(uint32_t k) { return unordered(k & 0x80000000u ? k & ~LP_PACKED : k | LP_PACKED); }
__device__ __forceinline__ uint32_t wave_max_key(uint32_t k) { return wave_max_bits(k); }

struct Out {                                  // where a row's answers go
    const long long* target;
    long long ignore;
    int top;
    float *logp, *entropy, *top_logp;
    long long* top_index;
    float* stats;
};
struct Stat {
    float m, logs;
};
// t, xt: the row's target and its logit
__device__ __forceinline__ Stat row_answer(const Run& r, const Out& o, long long row, int C, long long t, float xt) {
    const bool empty = r.m == -INFINITY && r.s == 0.f;
    const float m = r.m == -INFINITY ? 0.f : r.m, logs = empty ? INFINITY : logf(r.s);
    o.stats[2 * row] = m;
    o.stats[2 * row + 1] = logs;
    o.entropy[row] = empty ? 0.f : logs - r.u / r.s;
    if (o.logp) o.logp[row] = t == o.ignore ? 0.f : t < 0 || t >= C ? __builtin_nanf("") : (xt - m) - logs;
    return Stat{m, logs};
}

// ---- lane per row ------------------------------------------------------------------------------------------------------------------------
// The K largest of the classes a lane has walked, largest first; classes come in ascending order, so an equal one goes behind those before it.  A new
// value x moves place k to the middle one of (place k - 1, x, place k): no chain from place to place, and two instructions a place for packed keys where
// f32 values take five.  64 maps of 19 x 128 x 256, bf16 / f32, with 2, 5 and 16 alternatives: 46 / 52, 71 / 89 and 172 / 259 us (without any 31 / 39).
template <typename T, int K>
struct Largest {
    static constexpr bool ONE = sizeof(T) == 2;
    uint32_t v[K];
    int at[ONE ? 1 : K];
    __device__ __forceinline__ Largest() {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            v[k] = 0;
            if constexpr (!ONE) at[k] = 0;
        }
    }
    __device__ __forceinline__ void add(float value, int j, bool there) {
        const uint32_t x = !there ? 0 : ONE ? packed_key(value, j) : ordered(value);
#pragma unroll
        for (int k = K - 1; k >= 0; --k) {
            if constexpr (!ONE) {
                const int moved = k && x > v[k ? k - 1 : 0] ? +at[k ? k - 1 : 0] : j;
                at[k] = x > v[k] ? +moved : +at[k];
            }
            const uint32_t low = k && v[k ? k - 1 : 0] < x ? +v[k ? k - 1 : 0] : +x;
            v[k] = low > v[k] ? +low : +v[k];
        }
    }
    __device__ __forceinline__ int index(int k) const {
        if constexpr (ONE) return key_index(v[k]);
        else return at[k];
    }
    __device__ __forceinline__ float value(int k) const {
        if constexpr (ONE) return key_value(v[k]);
        else return unordered(v[k]);
    }
};

// row i of block row n: classes at x[n * outer_stride + i * row_stride + j * class_stride]
template <typename T, int KMAX>
__global__ __launch_bounds__(256) void lp_lane_forward_kernel(const T* __restrict__ x, long long P, long long outer, int C, long long outer_stride,
                                                              long long row_stride, long long class_stride, Out o) {
    constexpr int N = 8;
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= P) return;
    for (long long n = blockIdx.y; n < outer; n += gridDim.y) {
        const long long row = n * P + i;
        const T* p = x + n * outer_stride + i * row_stride;
        const long long t = o.logp ? o.target[row] : -1;
        const float xt = t >= 0 && t < C ? to_f32(p[t * class_stride]) : 0.f;
        Run r{-INFINITY, 0.f, 0.f};
        Largest<T, (KMAX > 0 ? KMAX : 1)> best;
        T next[N];
        auto fetch = [&](int j) {
#pragma unroll
            for (int e = 0; e < N; ++e) next[e] = j + e < C ? p[(long long)(j + e) * class_stride] : from_f32<T>(-INFINITY);
        };
        fetch(0);
        for (int j = 0; j < C; j += N) {
            float v[N];
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = to_f32(next[e]);
            if (j + N < C) fetch(j + N);                       // on its way while this one is added up
            run_add<N>(r, v, max_of<N>(v));
            if constexpr (KMAX > 0) {
#pragma unroll
                for (int e = 0; e < N; ++e) best.add(v[e], j + e, j + e < C);
            }
        }
        const Stat s = row_answer(r, o, row, C, t, xt);
        if constexpr (KMAX > 0 && KMAX <= 4) {
#pragma unroll
            for (int k = 0; k < KMAX; ++k)
                if (k < o.top) {
                    o.top_logp[row * o.top + k] = (best.value(k) - s.m) - s.logs;
                    o.top_index[row * o.top + k] = best.index(k);
                }
        }
        if constexpr (KMAX > 4) {
            // the wave's rows' answers lie one behind the other: through LDS (rows an odd number of dwords apart) each store covers whole lines
            // (64 x 19 x 128 x 256 bf16 with 8 alternatives 145 -> 87 us; up to 4 are stored as they are: 2 of them took 58 us this way, 51 directly)
            extern __shared__ uint32_t staged[];
            const int lane = threadIdx.x & 63, pitch = o.top | 1, there = P - (i - lane) < 64 ? (int)(P - (i - lane)) : 64;
            uint32_t* mine = staged + (threadIdx.x >> 6) * 64 * pitch;
            const uint32_t inverse = 0xFFFFFFFFu / (uint32_t)o.top + 1u;                   // q / top = umulhi(q, inverse) for q < 2^16
            const long long first = (row - lane) * o.top;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
#pragma unroll
                for (int k = 0; k < KMAX; ++k)
                    if (k < o.top) mine[lane * pitch + k] = half ? (uint32_t)best.index(k) : __float_as_uint((best.value(k) - s.m) - s.logs);
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
                for (int q = lane; q < there * o.top; q += there) {
                    const int of = (int)__umulhi((uint32_t)q, inverse);
                    const uint32_t v = mine[of * pitch + q - of * o.top];
                    if (half) o.top_index[first + q] = (int)v;
                    else o.top_logp[first + q] = __uint_as_float(v);
                }
                __builtin_amdgcn_wave_barrier();
            }
        }
    }
}

// ---- one or two short rows per wave ------------------------------------------------------------------------------------------------------
template <typename K>
__device__ __forceinline__ void order_pair(K& a, K& b) {
    const K x = a, y = b;
    a = x > y ? +x : +y;
    b = x > y ? +y : +x;
}
template <typename K>
__device__ __forceinline__ void sort_down(K (&k)[4]) {
    order_pair(k[0], k[1]), order_pair(k[2], k[3]), order_pair(k[0], k[2]), order_pair(k[1], k[3]), order_pair(k[1], k[2]);
}
template <typename K>
__device__ __forceinline__ void sort_down(K (&k)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i += 4) order_pair(k[i], k[i + 1]), order_pair(k[i + 2], k[i + 3]), order_pair(k[i], k[i + 2]), order_pair(k[i + 1], k[i + 3]), order_pair(k[i + 1], k[i + 2]);
    order_pair(k[0], k[4]), order_pair(k[1], k[5]), order_pair(k[2], k[6]), order_pair(k[3], k[7]);
    order_pair(k[2], k[4]), order_pair(k[3], k[5]), order_pair(k[1], k[2]), order_pair(k[3], k[4]), order_pair(k[5], k[6]);
}
// Rows of at most A accesses of 16 bytes a lane stay in registers, and `per` of them (one or two) share a wave: their loads are in flight together, and the
// closing arithmetic of each is done by a lane of its own, at once.  Alternatives: every lane sorts its values, the largest of the lanes' first ones is
// taken k times.  Bound by instructions: 65536 x 500 bf16 without alternatives, with 2, 8 and 20: 24, 38, 49 and 72 us, where a wave per row that is
// walked like longer ones takes 32, 63, 83 and 124.
template <typename T, int A>
__global__ __launch_bounds__(256) void lp_short_forward_kernel(const T* __restrict__ x, long long from, long long rows, int C, long long row_stride, int per,
                                                               Out o) {
    constexpr int VEC = ElemOf<T>::VEC, E = A * VEC, RW = 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), k = o.top;
    const long long row0 = from + ((long long)blockIdx.x * 4 + wave) * per, row = row0 + lane;
    if (row0 >= rows) return;                            // whole waves
    const int n = rows - row0 < per ? (int)(rows - row0) : per;
    u32x4_t raw[RW][A];
#pragma unroll
    for (int r = 0; r < RW; ++r)
        if (r < n) {
            const T* p = x + (row0 + r) * row_stride;
#pragma unroll
            for (int a = 0; a < A; ++a) raw[r][a] = load_raw_range<T>(p, (a * 64 + lane) * VEC - misaligned(p), 0, C, -INFINITY);
        }
    const long long target = lane < n && o.logp ? o.target[row] : -1;
    const float xt = target >= 0 && target < C ? to_f32(x[row * row_stride + target]) : 0.f;
    auto values = [&](int r, float (&v)[E]) {
#pragma unroll
        for (int a = 0; a < A; ++a) {
            float w[VEC];
            widen<T>(raw[r][a], w);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[a * VEC + e] = w[e];
        }
    };
    Run mine{0.f, 1.f, 0.f};
#pragma unroll
    for (int r = 0; r < RW; ++r)
        if (r < n) {
            float v[E], s = 0.f, u = 0.f;
            values(r, v);
            const float m = wave_max(max_of<E>(v)), base = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float d = v[e] - base, f = exp_d(d);
                s += f;
                u = fmaf(f, __builtin_fmaxf(d, LP_FLOOR), u);
            }
            s = wave_sum(s);
            u = wave_sum(u);
            if (lane == r) mine = Run{m, s, u};
        }
    Stat st{0.f, 0.f};
    if (lane < n) st = row_answer(mine, o, row, C, target, xt);
    if (!k) return;
#pragma unroll
    for (int r = 0; r < RW; ++r)
        if (r < n) {
            typedef std::conditional_t<sizeof(T) == 2, uint32_t, key_t> K;
            const T* p = x + (row0 + r) * row_stride;
            float v[E];
            K key[E], answer = 0;
            values(r, v);
#pragma unroll
            for (int a = 0; a < A; ++a)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {          // (what is absent is -inf and ranks behind what is there: places from C on, and below 0 as if from above)
                    const int c = (a * 64 + lane) * VEC - misaligned(p) + e;
                    if constexpr (sizeof(T) == 2) key[a * VEC + e] = packed_key(v[a * VEC + e], c);
                    else key[a * VEC + e] = key_of(v[a * VEC + e], c);
                }
            sort_down(key);
            for (int i = 0; i < k; ++i) {
                const K best = wave_max_key(key[0]);
                if (lane == i) answer = best;
                uint32_t taken = key[0] == best ? ~0u : 0u;           // (bits: of a condition the compiler makes a choice of the index)
                asm volatile("" : "+v"(taken));
                const K move = sizeof(K) == 8 ? (K)((key_t)taken << 32 | taken) : (K)taken;
#pragma unroll
                for (int e = 0; e < E; ++e) key[e] = (move & (e + 1 < E ? +key[e + 1 < E ? e + 1 : e] : K(0))) | (~move & key[e]);
            }
            const float m = __shfl(st.m, r, 64), logs = __shfl(st.logs, r, 64);
            if (lane < k) {
                o.top_logp[(row0 + r) * k + lane] = (key_value(answer) - m) - logs;
                o.top_index[(row0 + r) * k + lane] = key_index(answer);
            }
        }
}

// ---- wave or block per (part of a) row -----------------------------------------------------------------------------------------------------
// what top_keys keeps in shared memory for a row: candidates or lists | (NW > 1: every wave's k first keys) | the threads that look again | counts
constexpr int LP_CANDIDATES = 128;
template <int NW> __host__ __device__ constexpr int top_keys_words(int k) {
    return (k * k > LP_CANDIDATES ? k * k : LP_CANDIDATES) + (NW > 1 ? NW * k : 0) + k / 2 + 2;
}
template <int NW>
__device__ __forceinline__ void row_barrier() {
    if constexpr (NW > 1) __syncthreads();
    else {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
}
// Lane l < k of the FIRST wave gets the l-th largest of the part's elements; `mine`: the largest key of what this thread read, with the first place
// of its access in place of its own.  The k-th largest of those is a bound (accesses do not overlap, so these keys come in the order of places, and each of
// the k largest threads has an element in front of any element of the others); the elements of these k threads from the bound on are
// gathered by all threads, and their k largest taken by rounds.  Should more than 128 qualify (ascending rows), each of the k threads makes a
// list of its own k largest instead.
template <typename T, int NW>
__device__ __forceinline__ key_t top_keys(const T* __restrict__ p, int lo, int hi, int origin, key_t mine, int k, key_t* lists) {
    constexpr int VEC = ElemOf<T>::VEC, TPR = NW * 64;
    const int lane = threadIdx.x & 63, wave = NW == 1 ? 0 : threadIdx.x >> 6, t = NW == 1 ? lane : threadIdx.x;
    key_t* firsts = lists + (k * k > LP_CANDIDATES ? k * k : LP_CANDIDATES);
    int* chosen = (int*)(firsts + (NW > 1 ? NW * k : 0));
    int* counts = chosen + (k / 2) * 2 + 2;              // [0] threads, [1] elements
    key_t left = mine, bound = 0;
    for (int r = 0; r < k; ++r) {                        // this wave's k largest thread keys
        bound = wave_max_key(left);
        if (left == bound) left = 0;                     // keys differ (the index is in them), 0 aside
        if constexpr (NW > 1)
            if (lane == 0) firsts[wave * k + r] = bound;
    }
    if (t == 0) counts[0] = counts[1] = 0;
    row_barrier<NW>();
    if constexpr (NW > 1) {                              // the k-th largest of all of them
        static_assert(NW == 4 && LP_TOP_MOST <= 32, "two keys a lane");
        if (wave == 0) {
            key_t a = lane < NW * k ? firsts[lane] : 0, b = lane + 64 < NW * k ? firsts[lane + 64] : 0;
            order_pair(a, b);
            for (int r = 0; r < k; ++r) {
                bound = wave_max_key(a);
                if (a == bound) {
                    a = b;
                    b = 0;
                }
            }
            if (lane == 0) firsts[0] = bound;            // (read by this wave only, above)
        }
        __syncthreads();
        bound = firsts[0];
    }
    const bool again = mine && mine >= bound;            // at most k threads
    if (again) chosen[atomicAdd(&counts[0], 1)] = t;
    bound -= bound ? VEC - 1 : 0;                        // elements count from the end of the bound's access
    row_barrier<NW>();
    const int threads = counts[0], each = (hi - origin + TPR * VEC - 1) / (TPR * VEC);
    for (int w = t; w < threads * each; w += TPR) {
        const int turn = w / threads, c = origin + (turn * TPR + chosen[w - turn * threads]) * VEC;
        float v[VEC];
        load_range<T, VEC>(p, c, lo, hi, v, 0.f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const key_t q = c + e >= lo && c + e < hi ? key_of(v[e], c + e) : 0;
            if (q && q >= bound) {
                const int at = atomicAdd(&counts[1], 1);
                if (at < LP_CANDIDATES) lists[at] = q;
            }
        }
    }
    row_barrier<NW>();
    key_t answer = 0;
    const int found = counts[1];
    if (found <= LP_CANDIDATES) {
        if (wave == 0) {
            key_t a = lane < found ? lists[lane] : 0, b = lane + 64 < found ? lists[lane + 64] : 0;
            order_pair(a, b);
            for (int r = 0; r < k; ++r) {
                const key_t best = wave_max_key(a);
                if (lane == r) answer = best;
                if (a == best) {
                    a = b;
                    b = 0;
                }
            }
        }
        return answer;
    }
    row_barrier<NW>();                                   // (the lists overlay the candidates)
    if (again) {
        int which = 0;
        while (chosen[which] != t) ++which;
        key_t* list = lists + which * k;
        int n = 0;
        for (int c = origin + t * VEC; c < hi; c += TPR * VEC) {
            float v[VEC];
            load_range<T, VEC>(p, c, lo, hi, v, 0.f);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const key_t q = c + e >= lo && c + e < hi ? key_of(v[e], c + e) : 0;
                if (q >= bound && q && (n < k || q > list[n - 1])) {
                    int at = n < k ? n++ : n - 1;
                    for (; at > 0 && list[at - 1] < q; --at) list[at] = list[at - 1];
                    list[at] = q;
                }
            }
        }
        for (; n < k; ++n) list[n] = 0;
    }
    row_barrier<NW>();
    if (wave == 0) {
        int at = 0;
        for (int r = 0; r < k; ++r) {
            const key_t head = lane < threads && at < k ? lists[lane * k + at] : 0;
            const key_t best = wave_max_key(head);
            if (head == best && head) ++at;
            if (lane == r) answer = best;
        }
    }
    return answer;
}

// The elements [lo, hi) of a row by a block's (or wave's) threads, groups of four accesses in flight; then each with f(raw, its first place).  Which accesses
// there are goes by the row, not by the lane, so that the first and last ones, part of which is not there, cost no walk of their own.
template <typename T, int NW, typename F>
__device__ __forceinline__ void walk_row(const T* __restrict__ p, int origin, int lo, int hi, int t, float fill, F f) {
    constexpr int EACH = NW * 64 * ElemOf<T>::VEC;
    for (int g = origin; g < hi; g += 4 * EACH) {
        const bool whole = g >= lo && hi - g >= 4 * EACH;
        u32x4_t raw[4];
        if (whole) {
#pragma unroll
            for (int i = 0; i < 4; ++i) raw[i] = load_raw<T>(p + g + i * EACH + t * ElemOf<T>::VEC);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (g + i * EACH < hi) raw[i] = load_raw_range<T>(p, g + i * EACH + t * ElemOf<T>::VEC, lo, hi, fill);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (whole || g + i * EACH < hi) f(raw[i], g + i * EACH + t * ElemOf<T>::VEC, whole);
    }
}

// parts == nullptr: the whole row is here.  Otherwise part blockIdx.y of it, and its (m, s, u) and k keys go to parts / part_keys
// [row][part] for lp_join_kernel.
template <typename T, int NW>
__global__ __launch_bounds__(256) void lp_row_forward_kernel(const T* __restrict__ x, long long from, long long rows, int C, long long row_stride,
                                                             int part_len, Out o, float* __restrict__ parts, key_t* __restrict__ part_keys) {
    constexpr int VEC = ElemOf<T>::VEC, TPR = NW * 64, ROWS = 256 / TPR;
    extern __shared__ key_t shared[];                    // top_keys_words per row
    __shared__ float slots[3][NW];
    const int t = NW == 1 ? threadIdx.x & 63 : threadIdx.x, wave = threadIdx.x >> 6, k = o.top;
    const long long row = from + (long long)blockIdx.x * ROWS + (NW == 1 ? wave : 0);
    if (row >= rows) return;                             // whole waves, and only where no barrier follows
    const T* p = x + row * row_stride;
    const int lo = blockIdx.y * part_len, hi = C - lo < part_len ? C : lo + part_len;
    const long long target = o.logp && !parts ? o.target[row] : -1;     // (here, not behind the sums: two trips to memory, one behind the other)
    const float xt = target >= 0 && target < C ? to_f32(p[target]) : 0.f;
    Run r{-INFINITY, 0.f, 0.f};
    const int origin = lo - misaligned(p + lo), first = origin + t * VEC;
    float best = -INFINITY;
    int at = first;                                      // the access that brought it first
    walk_row<T, NW>(p, origin, lo, hi, t, -INFINITY, [&](u32x4_t raw, int c, bool) {
        float v[VEC];
        widen<T>(raw, v);
        const float cm = max_of<VEC>(v);
        if (k) {
            at = cm > best ? c : at;
            best = __builtin_fmaxf(cm, best);
        }
        run_add<VEC>(r, v, cm);
    });
    r = wave_join(r);
    if constexpr (NW > 1) {
        if ((threadIdx.x & 63) == 0) {
            slots[0][wave] = r.m;
            slots[1][wave] = r.s;
            slots[2][wave] = r.u;
        }
        __syncthreads();
        Run a{slots[0][0], slots[1][0], slots[2][0]};
#pragma unroll
        for (int i = 1; i < NW; ++i) {
            Run b{slots[0][i], slots[1][i], slots[2][i]};
            run_to(a, b.m);
            run_to(b, a.m);
            a.s += b.s;
            a.u += b.u;
        }
        r = a;
    }
    Stat s{0.f, 0.f};
    if (t == 0) {
        if (parts) {
            float* q = parts + (row * gridDim.y + blockIdx.y) * 3;
            q[0] = r.m;
            q[1] = r.s;
            q[2] = r.u;
        } else s = row_answer(r, o, row, C, target, xt);
    }
    if (!k) return;
    key_t* mem = shared + (NW == 1 ? wave * top_keys_words<NW>(k) : 0);
    const key_t mine = first < hi ? key_of(best, at < lo ? lo : at) : 0;
    const key_t q = top_keys<T, NW>(p, lo, hi, origin, mine, k, mem);
    if (wave == 0 || NW == 1) {
        s.m = __shfl(s.m, 0, 64);
        s.logs = __shfl(s.logs, 0, 64);
        if (t < k) {
            if (parts) part_keys[(row * gridDim.y + blockIdx.y) * k + t] = q;
            else {
                o.top_logp[row * k + t] = (key_value(q) - s.m) - s.logs;
                o.top_index[row * k + t] = key_index(q);
            }
        }
    }
}

// one wave per row: lane l joins part l
template <typename T>
__global__ __launch_bounds__(256) void lp_join_kernel(const T* __restrict__ x, long long rows, int C, long long row_stride, int n_parts, Out o,
                                                      const float* __restrict__ parts, const key_t* __restrict__ part_keys) {
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, k = o.top;
    if (row >= rows) return;
    const long long target = o.logp ? o.target[row] : -1;
    const float xt = target >= 0 && target < C ? to_f32(x[row * row_stride + target]) : 0.f;
    Run r{-INFINITY, 0.f, 0.f};
    if (lane < n_parts) {
        const float* q = parts + (row * n_parts + lane) * 3;
        r = Run{q[0], q[1], q[2]};
    }
    r = wave_join(r);
    Stat s{0.f, 0.f};
    if (lane == 0) s = row_answer(r, o, row, C, target, xt);
    if (!k) return;
    s.m = __shfl(s.m, 0, 64);
    s.logs = __shfl(s.logs, 0, 64);
    int at = 0;
    key_t answer = 0;
    for (int i = 0; i < k; ++i) {
        const key_t head = lane < n_parts && at < k ? part_keys[(row * n_parts + lane) * k + at] : 0;
        const key_t best = wave_max_key(head);
        if (head == best && head) ++at;
        if (lane == i) answer = best;
    }
    if (lane < k) {
        o.top_logp[row * k + lane] = (key_value(answer) - s.m) - s.logs;
        o.top_index[row * k + lane] = key_index(answer);
    }
}

// ---- backward ------------------------------------------------------------------------------------------------------------------------------
struct Grad {
    const long long* target;
    long long ignore;
    const float *stats, *entropy, *g_logp, *g_entropy, *g_top;
    const long long* top_index;
    int top;
};
// dx_j = p_j (c1 l_j + c0) with l_j = log p_j, plus a at the target and b_i at the alternatives
struct RowGrad {
    float m, logs, a, c0, c1;
    int t;                                    // -1: none
};
__device__ __forceinline__ RowGrad row_grad(const Grad& g, long long row, int C, float sum_of_top) {
    RowGrad r;
    r.m = g.stats[2 * row];
    r.logs = g.stats[2 * row + 1];
    r.t = -1;
    r.a = 0.f;
    if (g.g_logp) {
        const long long t = g.target[row];
        if (t != g.ignore) {
            const bool in = t >= 0 && t < C;
            r.a = in ? g.g_logp[row] : __builtin_nanf("");
            r.t = in ? (int)t : -1;
        }
    }
    const float whole = r.a + sum_of_top;
    const float c = g.g_entropy ? g.g_entropy[row] : 0.f;
    r.c1 = -c;
    r.c0 = -fmaf(c, g.entropy[row], whole);
    if (r.logs == INFINITY) r.t = -1;         // a row of masked classes: p = 0 everywhere
    return r;
}
__device__ __forceinline__ float class_grad(const RowGrad& r, float x) {
    const float l = (x - r.m) - r.logs;
    return exp_d(l) * fmaf(r.c1, __builtin_fmaxf(l, LP_FLOOR), r.c0);
}
__device__ __forceinline__ uint32_t class_or_none(long long j, int C) { return j >= 0 && j < C ? (uint32_t)j : 0xFFFFFFFFu; }
// KMAX alternatives in registers, their places compared with every class.  More than 4 come through LDS, so that whole lines are read (as in the
// forward kernel).  The next classes are on their way while these are stored: a store could alias them, so the compiler would not do it.
// (64 maps of 19 x 128 x 256, bf16 / f32: 40 / 69 us without alternatives, 51 / 79 with 2, 111 / 116 with 5, 300 / 308 with 16)
template <typename T, int KMAX>
__global__ __launch_bounds__(256) void lp_lane_backward_kernel(const T* __restrict__ x, long long P, long long outer, int C, long long outer_stride,
                                                               long long row_stride, long long class_stride, Grad g, T* __restrict__ dx,
                                                               long long dx_outer_stride, long long dx_row_stride) {
    constexpr int N = 8;
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= P) return;
    for (long long n = blockIdx.y; n < outer; n += gridDim.y) {
        const long long row = n * P + i;
        const T* p = x + n * outer_stride + i * row_stride;
        T* d = dx + n * dx_outer_stride + i * dx_row_stride;
        T next[N];
        auto fetch = [&](int j) {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (j + e < C) next[e] = p[(long long)(j + e) * class_stride];
        };
        fetch(0);
        float b[KMAX > 0 ? KMAX : 1], sum = 0.f;
        int at[KMAX > 0 ? KMAX : 1];
        if constexpr (KMAX > 4) {
            extern __shared__ uint32_t staged[];
            const int lane = threadIdx.x & 63, pitch = g.top | 1, there = P - (i - lane) < 64 ? (int)(P - (i - lane)) : 64;
            uint32_t* mine = staged + (threadIdx.x >> 6) * 64 * pitch;
            const uint32_t inverse = 0xFFFFFFFFu / (uint32_t)g.top + 1u;
            const long long first = (row - lane) * g.top;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                for (int q = lane; q < there * g.top; q += there) {
                    const int of = (int)__umulhi((uint32_t)q, inverse);
                    mine[of * pitch + q - of * g.top] = half ? class_or_none(g.top_index[first + q], C) : __float_as_uint(g.g_top[first + q]);
                }
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
                for (int k = 0; k < KMAX; ++k) {
                    const uint32_t v = k < g.top ? mine[lane * pitch + k] : 0u;
                    if (half) at[k] = k < g.top ? (int)v : -1;
                    else b[k] = __uint_as_float(v);
                }
                __builtin_amdgcn_wave_barrier();
            }
        } else {
#pragma unroll
            for (int k = 0; k < KMAX; ++k) {
                at[k] = k < g.top ? (int)class_or_none(g.top_index[row * g.top + k], C) : -1;
                b[k] = k < g.top ? g.g_top[row * g.top + k] : 0.f;
            }
        }
#pragma unroll
        for (int k = 0; k < KMAX; ++k) sum += b[k];
        const RowGrad r = row_grad(g, row, C, sum);
        if (r.logs == INFINITY) {                              // a row of masked classes has no gradient
#pragma unroll
            for (int k = 0; k < KMAX; ++k) b[k] = 0.f;
        }
        for (int j = 0; j < C; j += N) {
            float v[N];
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = to_f32(next[e]);
            if (j + N < C) fetch(j + N);
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (j + e < C) {
                    float w = class_grad(r, v[e]) + (j + e == r.t ? r.a : 0.f);
#pragma unroll
                    for (int k = 0; k < KMAX; ++k) w += j + e == at[k] ? b[k] : 0.f;
                    d[(long long)(j + e) * class_stride] = from_f32<T>(w);
                }
        }
    }
}

// a block (NW = 4) or a wave (NW = 1) per part of a row; the places of the target and of the alternatives get more than that, and are written again
// by the first wave of the block that wrote them
template <typename T, int NW>
__global__ __launch_bounds__(256) void lp_row_backward_kernel(const T* __restrict__ x, long long from, long long rows, int C, long long row_stride,
                                                              int part_len, Grad g, T* __restrict__ dx) {
    constexpr int VEC = ElemOf<T>::VEC, TPR = NW * 64, ROWS = 256 / TPR;
    const int t = NW == 1 ? threadIdx.x & 63 : threadIdx.x;
    const long long row = from + (long long)blockIdx.x * ROWS + (NW == 1 ? threadIdx.x >> 6 : 0);
    if (row >= rows) return;
    const T* p = x + row * row_stride;
    T* d = dx + row * C;
    const int lo = blockIdx.y * part_len, hi = C - lo < part_len ? C : lo + part_len;
    const int lane = threadIdx.x & 63, top = g.g_top ? g.top : 0;      // lane 1 + i has alternative i
    const bool mine = lane > 0 && lane <= top;
    const int at = mine ? (int)class_or_none(g.top_index[row * top + lane - 1], C) : -1;
    const float b = mine ? g.g_top[row * top + lane - 1] : 0.f;
    const RowGrad r = row_grad(g, row, C, top ? wave_sum(b) : 0.f);
    const int j = lane ? at : r.t;
    const bool here = lane <= top && j >= lo && j < hi;
    const float xj = here ? to_f32(p[j]) : 0.f;
    walk_row<T, NW>(p, lo - misaligned(p + lo), lo, hi, t, 0.f, [&](u32x4_t raw, int c, bool whole) {
        float v[VEC];
        widen<T>(raw, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = class_grad(r, v[e]);
        if (whole) store_n<T, VEC>(d + c, v);
        else store_range<T, VEC>(d, c, lo, hi, v);
    });
    // (behind the block's stores to these places)
    if constexpr (NW > 1) __syncthreads();
    else __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "workgroup");
    if (t > 63 || r.logs == INFINITY) return;
    float v = class_grad(r, xj) + (j == r.t ? r.a : 0.f);
    for (int i = 1; i <= top; ++i) {
        const int ai = __builtin_amdgcn_readlane(at, i);
        const float bi = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(b), i));
        v += ai == j ? bi : 0.f;
    }
    if (here) d[j] = from_f32<T>(v);                                   // (the same place: the same value)
}

// few long rows: enough parts for about four blocks on every CU, of at least 1 024 classes (2 049 make two parts: 8 rows 5.7 us, of 4 096 5.5)
int lp_parts(long long rows, int C) {
    if (C <= LP_WAVE_MOST) return 1;
    long long n = (1024 + rows - 1) / rows;
    const long long most = (C + 2047) / 2048;
    if (n > most) n = most;
    return (int)(n > LP_SPLIT_MOST ? LP_SPLIT_MOST : n < 1 ? 1 : n);
}
int lp_part_len(int C, int n) {                // a multiple of 8 elements
    const long long len = ((long long)C + n - 1) / n;
    return (int)((len + 7) / 8 * 8);
}
// launch(first row, blocks) over all rows, in as many launches as the limit on a launch's work-items makes of them
template <typename F>
void lp_launches(long long rows, int per_block, F launch) {
    const long long most = most_blocks(256) * per_block;
    for (long long from = 0; from < rows; from += most) {
        const long long n = rows - from < most ? rows - from : most;
        launch(from, (unsigned)((n + per_block - 1) / per_block));
    }
}
bool lp_lane(int C, long long inner) { return inner > 1 || C <= LP_LANE_MOST; }

struct LaneGrid {
    long long P, outer, outer_stride, row_stride, class_stride;
    dim3 grid, block;
};
LaneGrid lane_grid(long long outer, int C, long long inner, long long row_stride) {
    LaneGrid g;
    if (inner > 1) g = {inner, outer, (long long)C * inner, 1, inner};
    else g = {outer, 1, 0, row_stride, 1};
    const int threads = g.P <= 64 ? 64 : 256;
    g.block = dim3(threads);
    g.grid = dim3((unsigned)((g.P + threads - 1) / threads), (unsigned)(g.outer < 65535 ? g.outer : 65535));
    return g;
}

template <typename T>
int lp_forward(const void* x, long long outer, int C, long long inner, long long row_stride, const Out& o, void* ws, hipStream_t st) {
    if (lp_lane(C, inner)) {
        const LaneGrid g = lane_grid(outer, C, inner, row_stride);
        const size_t lds = o.top > 4 ? (size_t)g.block.x * (o.top | 1) * sizeof(uint32_t) : 0;
#define LP_LANE(K) hipLaunchKernelGGL((lp_lane_forward_kernel<T, K>), g.grid, g.block, lds, st, (const T*)x, g.P, g.outer, C, g.outer_stride, g.row_stride, g.class_stride, o)
        if (o.top == 0) LP_LANE(0);
        else if (o.top <= 2) LP_LANE(2);
        else if (o.top <= 4) LP_LANE(4);
        else if (o.top <= 8) LP_LANE(8);
        else LP_LANE(32);
#undef LP_LANE
        return w2c_launch_status();
    }
    const int k = o.top;
    constexpr int VEC = ElemOf<T>::VEC, MOST = 8 / VEC;                  // eight values a lane
    if (C + VEC - 1 <= 64 * VEC * MOST) {
        const int per = outer >= 8192 ? 2 : 1;
        // (the card holds 8 192 waves.  1 / 2 rows to a wave, us, bf16, without / with 8 alternatives: 4096 x 250 4.2 or 4.4 / 6.2 or 7.0, 8192 x 250 5.5 or 5.2 /
        // 9.3 or 9.6, 16384 x 250 7.8 or 6.9 / 14.9 either way, 65536 x 500 23.4 or 22.5 / 47.7 or 48.0; with four 22.9 / 50.0)
        lp_launches(outer, 4 * per, [&](long long from, unsigned blocks) {
            if (C + VEC - 1 <= 64 * VEC)
                hipLaunchKernelGGL((lp_short_forward_kernel<T, 1>), dim3(blocks), dim3(256), 0, st, (const T*)x, from, outer, C, row_stride, per, o);
            else
                hipLaunchKernelGGL((lp_short_forward_kernel<T, MOST>), dim3(blocks), dim3(256), 0, st, (const T*)x, from, outer, C, row_stride, per, o);
        });
        return w2c_launch_status();
    }
    if (C <= LP_WAVE_MOST) {
        lp_launches(outer, 4, [&](long long from, unsigned blocks) {
            hipLaunchKernelGGL((lp_row_forward_kernel<T, 1>), dim3(blocks), dim3(256), (size_t)(k ? 4 * top_keys_words<1>(k) * sizeof(key_t) : 0), st,
                               (const T*)x, from, outer, C, row_stride, C, o, (float*)nullptr, (key_t*)nullptr);
        });
        return w2c_launch_status();
    }
    const int n = lp_parts(outer, C);
    const int len = n > 1 ? lp_part_len(C, n) : C, used = (int)(((long long)C + len - 1) / len);
    key_t* keys = n > 1 ? (key_t*)ws : nullptr;
    float* parts = n > 1 ? (float*)(keys + (long long)outer * n * k) : nullptr;
    lp_launches(outer, 1, [&](long long from, unsigned blocks) {
        hipLaunchKernelGGL((lp_row_forward_kernel<T, 4>), dim3(blocks, used), dim3(256), (size_t)(k ? top_keys_words<4>(k) * sizeof(key_t) : 0), st,
                           (const T*)x, from, outer, C, row_stride, len, o, parts, keys);
    });
    if (n > 1)
        hipLaunchKernelGGL((lp_join_kernel<T>), dim3((unsigned)((outer + 3) / 4)), dim3(256), 0, st, (const T*)x, outer, C, row_stride, used, o,
                           (const float*)parts, (const key_t*)keys);
    return w2c_launch_status();
}

template <typename T>
int lp_backward(const void* x, long long outer, int C, long long inner, long long row_stride, const Grad& g, void* dx, hipStream_t st) {
    if (lp_lane(C, inner)) {
        const LaneGrid l = lane_grid(outer, C, inner, row_stride);
        const int top = g.g_top ? g.top : 0;
        const size_t lds = top > 4 ? (size_t)l.block.x * (top | 1) * sizeof(uint32_t) : 0;
#define LP_LANE(K)                                                                                                                                \
    hipLaunchKernelGGL((lp_lane_backward_kernel<T, K>), l.grid, l.block, lds, st, (const T*)x, l.P, l.outer, C, l.outer_stride, l.row_stride,          \
                       l.class_stride, g, (T*)dx, l.outer_stride, inner > 1 ? 1ll : (long long)C)
        if (top == 0) LP_LANE(0);
        else if (top <= 2) LP_LANE(2);
        else if (top <= 4) LP_LANE(4);
        else if (top <= 8) LP_LANE(8);
        else LP_LANE(32);
#undef LP_LANE
        return w2c_launch_status();
    }
    if (C <= LP_WAVE_MOST) {
        lp_launches(outer, 4, [&](long long from, unsigned blocks) {
            hipLaunchKernelGGL((lp_row_backward_kernel<T, 1>), dim3(blocks), dim3(256), 0, st, (const T*)x, from, outer, C, row_stride, C, g, (T*)dx);
        });
        return w2c_launch_status();
    }
    // a block per row, or per part of one where there are not rows enough for two rounds of blocks; more than two accesses per lane
    long long n = (4096 + outer - 1) / outer;
    const long long most = (C + 256 * ElemOf<T>::VEC * 4 - 1) / (256 * ElemOf<T>::VEC * 4);
    if (n > most) n = most;
    const int len = lp_part_len(C, (int)n);
    lp_launches(outer, 1, [&](long long from, unsigned blocks) {
        hipLaunchKernelGGL((lp_row_backward_kernel<T, 4>), dim3(blocks, (C - 1) / len + 1), dim3(256), 0, st, (const T*)x, from, outer, C, row_stride,
                           len, g, (T*)dx);
    });
    return w2c_launch_status();
}

bool lp_shape_ok(int dtype, long long outer, int C, long long inner, long long row_stride) {
    return dtype >= W2C_F32 && dtype <= W2C_F16 && outer >= 1 && outer <= 0x7FFFFFFF && C >= 1 && C <= (1 << 28) && inner >= 1 &&
           inner <= 0x7FFFFFFF && (inner == 1 || C <= LP_PACKED_CLASSES) && (inner > 1 ? row_stride == (long long)C * inner : row_stride >= C);
}

}  // namespace

extern "C" long long w2c_log_probs_workspace_bytes(long long outer, int classes, long long inner, int top) {
    if (!lp_shape_ok(W2C_F32, outer, classes, inner, (long long)classes * inner) || top < 0 || top > LP_TOP_MOST) return W2C_E_ARG;
    const int n = lp_lane(classes, inner) ? 1 : lp_parts(outer, classes);
    return n > 1 ? outer * n * ((long long)top * 8 + 12) : 0;
}

extern "C" int w2c_log_probs_forward(const void* x, int dtype, long long outer, int classes, long long inner, long long row_stride,
                                     const long long* target, long long ignore_index, int top, float* logp, float* entropy, float* top_logp,
                                     long long* top_index, float* stats, void* workspace, long long workspace_bytes, void* stream) {
    if (!x || !entropy || !stats || !lp_shape_ok(dtype, outer, classes, inner, row_stride)) return W2C_E_ARG;
    if ((target == nullptr) != (logp == nullptr) || top < 0 || top > LP_TOP_MOST || top > classes || (top && (!top_logp || !top_index))) return W2C_E_ARG;
    const long long need = w2c_log_probs_workspace_bytes(outer, classes, inner, top);
    if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 7))) return W2C_E_ARG;
    w2c_clear_error();
    const Out o{target, ignore_index, top, logp, entropy, top_logp, top_index, stats};
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == W2C_F32) return lp_forward<float>(x, outer, classes, inner, row_stride, o, workspace, st);
    if (dtype == W2C_BF16) return lp_forward<bf16_t>(x, outer, classes, inner, row_stride, o, workspace, st);
    return lp_forward<f16_t>(x, outer, classes, inner, row_stride, o, workspace, st);
}

extern "C" int w2c_log_probs_backward(const void* x, int dtype, long long outer, int classes, long long inner, long long row_stride,
                                      const long long* target, long long ignore_index, const float* stats, const float* entropy, int top,
                                      const long long* top_index, const float* g_logp, const float* g_entropy, const float* g_top, void* dx,
                                      void* stream) {
    if (!x || !stats || !entropy || !dx || !lp_shape_ok(dtype, outer, classes, inner, row_stride)) return W2C_E_ARG;
    if ((g_logp && !target) || top < 0 || top > LP_TOP_MOST || top > classes || (g_top && (!top || !top_index))) return W2C_E_ARG;
    w2c_clear_error();
    const Grad g{target, ignore_index, stats, entropy, g_logp, g_entropy, g_top, top_index, top};
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == W2C_F32) return lp_backward<float>(x, outer, classes, inner, row_stride, g, dx, st);
    if (dtype == W2C_BF16) return lp_backward<bf16_t>(x, outer, classes, inner, row_stride, g, dx, st);
    return lp_backward<f16_t>(x, outer, classes, inner, row_stride, g, dx, st);
}
