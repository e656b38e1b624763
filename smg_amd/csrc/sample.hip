// Sampling with temperature, top-k, top-p and min-p from given random numbers — gfx950.
//
// Per row of V logits, in the order (logit falling, index rising), with the
// weights w_i = exp((x_i - max x) / temperature):
//   top-k   keeps the first k tokens of the order;
//   top-p   keeps of those the ones whose predecessors weigh less than
//           p * (what top-k kept weighs): the first always;
//   min-p   keeps of those the ones with w_i >= min_p (the largest w is 1).
// The answer is the first token, by index, at which the kept weights add up to
// more than u times their sum.  Temperature 0 takes the first token of the order.
//
// A token is right or wrong, so sums have to be exact and of no particular
// order: a weight is exp in 64 bits, rounded to a multiple of 2^-S and summed as
// a 64-bit integer, S = min(50, 62 - ceil(log2 V)).  Integer atomics give the
// same sums in every order.  (In 32 bits the sums of 32768 weights are off by
// about 1e-7, which moves one row in 300 to another token.)
//
// Both cuts are one search: the shortest prefix of the order whose measure (a
// count, or a weight) reaches a number.  It runs over a histogram of NB equal
// steps of the logit below the largest, which LDS atomics fill; the step in
// which the number is reached is divided again, until it holds one value, and
// equal values go by index.  Nothing is sorted.
//
// A workgroup has a row, and each wave a run of it, 512 tokens at a time, 8 a
// lane, so that index order is (wave, iteration, lane, element).
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>

#include <cstdint>

#define WAVE 64
#define THREADS 1024
#define WAVES (THREADS / WAVE)
#define NB 2048             // steps of a histogram; also the most blocks
#define BLOCK 512           // tokens of a wave's iteration
#define HELD_ITS 4          // iterations that stay in registers: V <= 32768
#define MAX_V (NB * BLOCK)

namespace {

typedef unsigned long long u64;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;

struct SampleArgs {
    const void* logits;  // [R, V] bf16 or f32
    long long stride;
    const float* u;            // [R]
    const float* temperature;  // [R]
    const int* top_k;          // [R] or null
    const float* top_p;        // [R] or null
    const float* min_p;        // [R] or null
    long long* out;            // [R]
    int R, V;
};

struct Shared {
    u64 hist[NB];
    double pow2[64];  // 2^(i/64)
    u64 part[WAVES];
    float lo[WAVES], hi[WAVES];
    u64 above, total;
    int bin, index;
};

template <typename T>
__device__ __forceinline__ T wave_scan(T x) {  // inclusive
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) {
        const T up = __shfl_up(x, o, WAVE);
        if (lane >= o) x += up;
    }
    return x;
}

// Sums the NB counters of sh.hist; sh.bin and sh.above get the first at which
// the sum reaches `want` and the sum before it (bin NB if it never does).
__device__ __forceinline__ void locate(Shared& sh, u64 want) {
    const int t = threadIdx.x, wave = t / WAVE;
    __syncthreads();
    const u64 a = sh.hist[2 * t], s = a + sh.hist[2 * t + 1];
    const u64 run = wave_scan(s);
    if ((t & 63) == 63) sh.part[wave] = run;
    if (t == 0) sh.bin = NB;
    __syncthreads();
    u64 before = run - s;
    for (int w = 0; w < wave; ++w) before += sh.part[w];
    if (before < want && before + s >= want) {
        const bool second = before + a < want;
        sh.bin = 2 * t + second;
        sh.above = before + (second ? a : 0);
    }
    if (t == THREADS - 1) sh.total = before + s;
    __syncthreads();
}

// the order's tokens up to the value x, of those equal to x up to index i
struct Prefix {
    float x;
    int i;
    __device__ __forceinline__ bool has(float y, int j) const { return y > x || (y == x && j <= i); }
};

// exp((x - top) / t) in 64 bits: 2^(n/64) from a table times a polynomial of
// 2^r, |r| <= 1/128 (off by 4e-14 at most)
struct Weigh {
    const double* pow2;
    double top, c, magic;
    int S;
    __device__ __forceinline__ void init(Shared& sh, float largest, float t, int V) {
        pow2 = sh.pow2;
        top = (double)largest;
        c = 64. * 1.44269504088896340736 / (double)t;
        S = min(50, 62 - (V > 1 ? 32 - __clz(V - 1) : 0));
    }
    __device__ __forceinline__ double mantissa(float x, int& e) const {
        // -inf and NaN: weight 0
        const double y = fmax(((double)x - top) * c, -1e9);
        const double n = rint(y), r = y - n;
        const int k = (int)n;
        constexpr double q = 0.6931471805599453094 / 64;
        double p = fma(r, q * q * q * q / 24, q * q * q / 6);
        p = fma(r, p, q * q / 2);
        p = fma(r, p, q);
        p = fma(r, p, 1.);
        e = k >> 6;
        return p * pow2[k & 63];
    }
    __device__ __forceinline__ double value(float x) const {
        int e;
        const double m = mantissa(x, e);
        return ldexp(m, e);
    }
    __device__ __forceinline__ u64 fixed(float x) const {
        int e;
        const double m = mantissa(x, e);
        return (u64)__double_as_longlong(ldexp(m, e + S) + 4503599627370496.) & 0xfffffffffffffull;
    }
};

// A row's tokens: `f(i, x)` for each of the thread's, in index order.
template <bool F32, bool HELD>
struct Row {
    const char* at;
    int V, start, its, lane;
    bool infinite;  // the largest is +inf: those weigh 1, all others nothing
    u32x4 raw[HELD ? HELD_ITS * (F32 ? 2 : 1) : 1];

    __device__ __forceinline__ void load8(int it, u32x4* r) const {
        const int i = start + it * BLOCK + lane * 8;
        if (i + 8 <= V) {
            // rows may start anywhere: the hardware takes wide loads at any element
            __builtin_memcpy(r, at + (size_t)i * (F32 ? 4 : 2), F32 ? 32 : 16);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (F32)
                    r[e / 4][e % 4] = i + e < V ? ((const unsigned*)at)[i + e] : 0x7fc00000u;
                else {
                    const unsigned h = i + e < V ? ((const unsigned short*)at)[i + e] : 0x7fc0u;
                    r[0][e / 2] = e % 2 ? r[0][e / 2] | h << 16 : h;
                }
            }
        }
    }
    __device__ __forceinline__ void init(const SampleArgs& a) {
        lane = threadIdx.x & 63;
        V = a.V;
        at = (const char*)a.logits + blockIdx.x * a.stride * (F32 ? 4 : 2);
        its = (V + WAVES * BLOCK - 1) / (WAVES * BLOCK);
        start = threadIdx.x / WAVE * its * BLOCK;
        infinite = false;
        if constexpr (HELD) {
#pragma unroll
            for (int it = 0; it < HELD_ITS; ++it) load8(it, raw + it * (F32 ? 2 : 1));
        }
    }
    template <typename F>
    __device__ __forceinline__ void each8(int it, F&& f) const {
        u32x4 tmp[F32 ? 2 : 1];
        const u32x4* r = tmp;
        if constexpr (HELD)
            r = raw + it * (F32 ? 2 : 1);
        else
            load8(it, tmp);
        const int i = start + it * BLOCK + lane * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float x = __uint_as_float(F32 ? r[e / 4][e % 4] : e % 2 ? r[0][e / 2] & 0xffff0000u : r[0][e / 2] << 16);
            if (infinite) x = x == INFINITY ? 0.f : -INFINITY;
            f(i + e, x);
        }
    }
    template <typename F>
    __device__ __forceinline__ void each(F&& f) const {
        if constexpr (HELD) {
#pragma unroll
            for (int it = 0; it < HELD_ITS; ++it)
                if (it < its) each8(it, f);
        } else {
            for (int it = 0; it < its; ++it) each8(it, f);
        }
    }
    // f(it, first index of the iteration)
    template <typename F>
    __device__ __forceinline__ void blocks(F&& f) const {
        if constexpr (HELD) {
#pragma unroll
            for (int it = 0; it < HELD_ITS; ++it)
                if (it < its) f(it);
        } else {
            for (int it = 0; it < its; ++it) f(it);
        }
    }
};

__device__ __forceinline__ void clear(Shared& sh) {
    __syncthreads();
    sh.hist[threadIdx.x] = sh.hist[threadIdx.x + THREADS] = 0;
    __syncthreads();
}

__device__ __forceinline__ float2 range_of(Shared& sh, float lo, float hi) {
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) {
        lo = fminf(lo, __shfl_xor(lo, o, WAVE));
        hi = fmaxf(hi, __shfl_xor(hi, o, WAVE));
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.lo[threadIdx.x / WAVE] = lo, sh.hi[threadIdx.x / WAVE] = hi;
    __syncthreads();
    for (int w = 0; w < WAVES; ++w) lo = fminf(lo, sh.lo[w]), hi = fmaxf(hi, sh.hi[w]);
    return make_float2(lo, hi);
}

// The first index at which the sums of measure(i, x), by index, reach `want`
// (>= 1, at most all of them).
template <typename R, typename M>
__device__ __forceinline__ int find_by_index(Shared& sh, const R& row, u64 want, M&& measure) {
    clear(sh);
    row.blocks([&](int it) {
        u64 s = 0;
        row.each8(it, [&](int i, float x) { s += measure(i, x); });
#pragma unroll
        for (int o = 1; o < WAVE; o <<= 1) s += __shfl_xor(s, o, WAVE);
        if (row.lane == 0) sh.hist[row.start / BLOCK + it] = s;
    });
    locate(sh, want);
    const int block = sh.bin;
    want -= sh.above;
    row.blocks([&](int it) {
        if (row.start / BLOCK + it != block) return;
        u64 s = 0;
        row.each8(it, [&](int i, float x) { s += measure(i, x); });
        u64 run = wave_scan(s) - s;
        if (run < want && run + s >= want) {
            int found = 0x7fffffff;
            row.each8(it, [&](int i, float x) {
                const u64 w = measure(i, x);
                if (run < want && run + w >= want) found = i;
                run += w;
            });
            sh.index = found;
        }
    });
    __syncthreads();
    return sh.index;
}

// The shortest prefix of the order whose measure reaches `want` (>= 1): sh.hist
// holds the first division of the measure, by step(x).  all: that is no prefix
// but everything.  Tokens take part where measure(i, x) is not 0.
template <typename R, typename M, typename Step>
__device__ __forceinline__ Prefix shortest(Shared& sh, const R& row, u64 want, Prefix all, M&& measure, Step&& step) {
    locate(sh, want);
    if (sh.bin >= NB - 1) return all;  // the last step's tokens weigh nothing
    int bin = sh.bin;
    float lo = INFINITY, hi = -INFINITY;
    row.each([&](int i, float x) {
        if (step(x) == bin && all.has(x, i)) lo = fminf(lo, x), hi = fmaxf(hi, x);
    });
    want -= sh.above;
    float2 r = range_of(sh, lo, hi);
    while (r.x < r.y) {
        // the ends fall into different steps, so this ends
        const double top = (double)r.y, c = (NB - 1) / (top - (double)r.x);
        auto finer = [&](float x) { return min(NB - 1, (int)((top - (double)x) * c)); };
        clear(sh);
        row.each([&](int i, float x) {
            if (x >= r.x && x <= r.y) {
                const u64 w = measure(i, x);
                if (w) atomicAdd(&sh.hist[finer(x)], w);
            }
        });
        locate(sh, want);
        bin = sh.bin;
        want -= sh.above;
        lo = INFINITY, hi = -INFINITY;
        row.each([&](int i, float x) {
            if (x >= r.x && x <= r.y && finer(x) == bin && all.has(x, i)) lo = fminf(lo, x), hi = fmaxf(hi, x);
        });
        r = range_of(sh, lo, hi);
    }
    const float x0 = r.x;
    return {x0, find_by_index(sh, row, want, [&](int i, float x) { return x == x0 ? measure(i, x) : 0ull; })};
}

template <bool F32, bool HELD>
__global__ void __launch_bounds__(THREADS) smg_sample_t(SampleArgs a) {
    __shared__ Shared sh;
    const int r = blockIdx.x, tid = threadIdx.x;
    Row<F32, HELD> row;
    row.init(a);
    if (tid < 64) sh.pow2[tid] = exp2((double)tid / 64);

    float lo = INFINITY, hi = -INFINITY;
    row.each([&](int, float x) {
        hi = fmaxf(hi, x);  // NaN is passed over
        if (x > -INFINITY) lo = fminf(lo, x);
    });
    float2 ends = range_of(sh, lo, hi);
    const float t = a.temperature[r];
    if (ends.y == -INFINITY) {
        if (tid == 0) a.out[r] = -1;
        return;
    }
    if (!(t > 0.f)) {
        int first = 0x7fffffff;
        row.each([&](int i, float x) { if (x == ends.y) first = min(first, i); });
        if (tid == 0) sh.index = 0x7fffffff;
        __syncthreads();
        if (first != 0x7fffffff) atomicMin(&sh.index, first);
        __syncthreads();
        if (tid == 0) a.out[r] = sh.index;
        return;
    }
    row.infinite = ends.y == INFINITY;
    if (row.infinite) ends = make_float2(0.f, 0.f);
    Weigh weigh;
    weigh.init(sh, ends.y, t, a.V);

    // steps down from the largest: to the smallest, or to where weights are 0
    // (below 2^-51), whose tokens the last step takes
    const float depth = fminf(ends.y - ends.x, 51.f * 0.69314718f * t);
    const float per = depth > 1e-30f ? (NB - 2) / depth : 0.f;
    auto step = [&](float x) { return (int)fminf((ends.y - x) * per, NB - 1.f); };

    Prefix kept = {-INFINITY, -1};
    const int k = a.top_k ? a.top_k[r] : 0;
    const bool cut = k > 0 && k < a.V;
    if (cut) {
        clear(sh);
        row.each([&](int, float x) {
            if (x > -INFINITY) atomicAdd(&sh.hist[step(x)], 1ull);
        });
        kept = shortest(sh, row, (u64)k, kept, [](int, float x) { return (u64)(x > -INFINITY); }, step);
    }
    const float p = a.top_p ? a.top_p[r] : 1.f;
    if (p < 1.f) {
        auto mass = [&](int i, float x) { return kept.has(x, i) ? weigh.fixed(x) : 0ull; };
        clear(sh);
        row.each([&](int i, float x) {
            const u64 w = mass(i, x);
            if (w) atomicAdd(&sh.hist[step(x)], w);
        });
        locate(sh, 1);
        const double want = ceil((double)p * (double)sh.total);
        const Prefix all = kept;
        kept = shortest(sh, row, want >= 1. ? (u64)want : 1, all, mass, step);
    }
    const float mp = a.min_p ? a.min_p[r] : 0.f;
    const double least = mp > 0.f ? fmin((double)mp, 1.) : 0.;
    auto last = [&](int i, float x) {
        if (!kept.has(x, i)) return 0ull;
        if (least > 0. && weigh.value(x) < least) return 0ull;
        return weigh.fixed(x);
    };
    u64 s = 0;
    row.each([&](int i, float x) { s += last(i, x); });
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) s += __shfl_xor(s, o, WAVE);
    __syncthreads();
    if ((tid & 63) == 0) sh.part[tid / WAVE] = s;
    __syncthreads();
    u64 all = 0;
    for (int w = 0; w < WAVES; ++w) all += sh.part[w];
    const float u = a.u[r];
    const double aim = u > 0.f ? (double)u * (double)all : 0.;
    const u64 want = aim < (double)all ? (u64)aim + 1 : all;  // the first sum above it
    const int found = find_by_index(sh, row, want, last);
    if (tid == 0) a.out[r] = found;
}

template <bool F32>
void launch(const SampleArgs& a, hipStream_t s) {
    if (false)
        hipLaunchKernelGGL((smg_sample_t<F32, true>), dim3(a.R), dim3(THREADS), 0, s, a);
    else
        hipLaunchKernelGGL((smg_sample_t<F32, false>), dim3(a.R), dim3(THREADS), 0, s, a);
}

}  // namespace

extern "C" int smg_sample_launch(const void* logits, const void* u, const void* temperature,
                                 const void* top_k, const void* top_p, const void* min_p, void* out,
                                 long long stride, int R, int V, int f32, void* stream) {
    if (V < 1 || V > MAX_V) return -1;
    if (R < 1) return 0;
    SampleArgs a = {logits, stride, (const float*)u, (const float*)temperature, (const int*)top_k,
                    (const float*)top_p, (const float*)min_p, (long long*)out, R, V};
    if (f32)
        launch<true>(a, (hipStream_t)stream);
    else
        launch<false>(a, (hipStream_t)stream);
    return hipGetLastError() == hipSuccess ? 0 : -2;
}
