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
// a 64-bit integer, S = 62 - ceil(log2 V) (2^-47 at 32768 tokens).  Integer
// atomics give the same sums in every order.
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>

#include <cstdint>

#define WAVE 64
#define THREADS 1024
#define WAVES (THREADS / WAVE)

namespace {

typedef unsigned long long u64;

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

// a key in the order of the values; 0 for NaN, which is never taken
__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned bits = __float_as_uint(x + 0.f);  // -0 is 0
    return x != x ? 0u : bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
#define KEY_NEG_INF 0x007fffffu

template <typename T>
__device__ __forceinline__ T wave_sum(T x) {
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) x += __shfl_xor(x, o, WAVE);
    return x;
}

template <bool F32>
struct Row {
    const char* at;
    float top;      // the largest logit
    double inv_t;   // 1 / temperature
    double unit;    // 2^S
    __device__ __forceinline__ unsigned key(int i) const {
        return key_of(F32 ? ((const float*)at)[i] : (float)((const __hip_bfloat16*)at)[i]);
    }
    __device__ __forceinline__ double weight(unsigned k) const {
        const float x = value_of(k);
        if (k <= KEY_NEG_INF) return 0.;
        if (top == INFINITY) return x == INFINITY ? 1. : 0.;
        return exp(((double)x - (double)top) * inv_t);
    }
    __device__ __forceinline__ u64 fixed(double w) const { return (u64)(w * unit + 0.5); }
};

// the tokens up to (key, last) in the order
struct Prefix {
    unsigned key;
    int last;
    __device__ __forceinline__ bool has(unsigned k, int i) const { return k > key || (k == key && i <= last); }
};

struct Shared {
    u64 hist[256];
    u64 part[WAVES];
    u64 above;
    unsigned bin;
    int index;
};

template <typename F>
__device__ __forceinline__ u64 block_sum(Shared& sh, F&& f, int v0, int v1) {
    u64 s = 0;
    for (int i = v0 + (threadIdx.x & 63); i < v1; i += WAVE) s += f(i);
    s = wave_sum(s);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.part[threadIdx.x / WAVE] = s;
    __syncthreads();
    u64 all = 0;
    for (int w = 0; w < WAVES; ++w) all += sh.part[w];
    return all;
}

// The shortest prefix of the order whose measure reaches `want` (>= 1, at most
// the measure of all): measure(i, key) is 1 or a weight.  Four digits of the key,
// the largest first, then the index among equal keys.
template <bool F32, typename M>
__device__ Prefix select(Shared& sh, const Row<F32>& row, int v0, int v1, u64 want, M&& measure) {
    unsigned found = 0;
    u64 each = 1;
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (threadIdx.x < 256) sh.hist[threadIdx.x] = 0;
        __syncthreads();
        for (int i = v0 + (threadIdx.x & 63); i < v1; i += WAVE) {
            const unsigned k = row.key(i);
            if (shift == 24 || k >> (shift + 8) == found) {
                const u64 w = measure(i, k);
                if (w) atomicAdd(&sh.hist[k >> shift & 255], w);
            }
        }
        __syncthreads();
        if (threadIdx.x < WAVE) {
            // from the top: lane l holds the bins 255-4l .. 252-4l
            const int b0 = 255 - 4 * (int)threadIdx.x;
            u64 s = sh.hist[b0] + sh.hist[b0 - 1] + sh.hist[b0 - 2] + sh.hist[b0 - 3];
            u64 sum = s;
#pragma unroll
            for (int o = 1; o < WAVE; o <<= 1) {
                const u64 up = __shfl_up(sum, o, WAVE);
                if ((int)threadIdx.x >= o) sum += up;
            }
            const u64 reach = __ballot(sum >= want);
            const int l = reach ? __ffsll((long long)reach) - 1 : WAVE - 1;
            if ((int)threadIdx.x == l) {
                u64 above = sum - s;
                int bin = b0;
                while (bin > b0 - 3 && above + sh.hist[bin] < want) above += sh.hist[bin--];
                sh.above = above;
                sh.bin = bin;
            }
        }
        __syncthreads();
        want -= sh.above;
        found = found << 8 | sh.bin;
        each = sh.hist[sh.bin];
        __syncthreads();
    }
    // equal keys weigh the same: the first `rank` of them by index
    const u64 ties = block_sum(sh, [&](int i) { return (u64)(row.key(i) == found && measure(i, found)); }, v0, v1);
    const u64 w = ties ? each / ties : 1;
    u64 rank = w ? (want + w - 1) / w : 1;
    if (rank > ties) rank = ties;
    const int wave = threadIdx.x / WAVE, lane = threadIdx.x & 63;
    u64 before = 0;
    for (int q = 0; q < wave; ++q) before += sh.part[q];
    if (threadIdx.x == 0) sh.index = 0x7fffffff;
    __syncthreads();
    if (before < rank && before + sh.part[wave] >= rank) {
        for (int i0 = v0; i0 < v1; i0 += WAVE) {
            const int i = i0 + lane;
            const bool tie = i < v1 && row.key(i) == found && measure(i, found);
            const u64 m = __ballot(tie);
            const int n = __popcll(m);
            if (before + n >= rank) {
                if (tie && before + __popcll(m & ((1ull << lane) - 1)) + 1 == rank) sh.index = i;
                break;
            }
            before += n;
        }
    }
    __syncthreads();
    const int last = sh.index;
    __syncthreads();
    return {found, last};
}

template <bool F32>
__global__ void __launch_bounds__(THREADS) smg_sample_t(SampleArgs a) {
    __shared__ Shared sh;
    const int r = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x / WAVE;
    Row<F32> row;
    row.at = (const char*)a.logits + r * a.stride * (F32 ? 4 : 2);
    // a wave has a run of the row of its own, so that waves are in index order
    const int per = ((a.V + WAVES - 1) / WAVES + WAVE - 1) / WAVE * WAVE;
    const int v0 = min(a.V, wave * per), v1 = min(a.V, v0 + per);

    // the largest key, and the first index that has it
    u64 best = 0;
    for (int i = v0 + lane; i < v1; i += WAVE) {
        const u64 k = (u64)row.key(i) << 32 | (0xffffffffu - i);
        best = k > best ? k : best;
    }
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) {
        const u64 x = __shfl_xor(best, o, WAVE);
        best = x > best ? x : best;
    }
    if (lane == 0) sh.part[wave] = best;
    __syncthreads();
    for (int w = 0; w < WAVES; ++w) best = sh.part[w] > best ? sh.part[w] : best;
    const unsigned top = (unsigned)(best >> 32);
    const float t = a.temperature[r];
    if (top <= KEY_NEG_INF || !(t > 0.f)) {
        // nothing to take, or the first of the largest
        if (threadIdx.x == 0) a.out[r] = top <= KEY_NEG_INF ? -1 : (long long)(0xffffffffu - (unsigned)best);
        return;
    }
    row.top = value_of(top);
    row.inv_t = 1. / (double)t;
    row.unit = (double)(1ull << (62 - (a.V > 1 ? 32 - __clz(a.V - 1) : 0)));

    Prefix kept = {KEY_NEG_INF, -1};  // everything above -inf
    const int k = a.top_k ? a.top_k[r] : 0;
    if (k > 0) {
        const u64 live = block_sum(sh, [&](int i) { return (u64)(row.key(i) > KEY_NEG_INF); }, v0, v1);
        if ((u64)k < live)
            kept = select(sh, row, v0, v1, (u64)k, [&](int, unsigned key) { return (u64)(key > KEY_NEG_INF); });
    }
    auto mass = [&](int i, unsigned key) { return kept.has(key, i) ? row.fixed(row.weight(key)) : 0ull; };
    const float p = a.top_p ? a.top_p[r] : 1.f;
    if (p < 1.f) {
        const u64 all = block_sum(sh, [&](int i) { return mass(i, row.key(i)); }, v0, v1);
        const double want = ceil((double)p * (double)all);
        const u64 w = want >= 1. ? (u64)want : 1;
        const Prefix cut = select(sh, row, v0, v1, w < all ? w : all, mass);
        kept = cut;
    }
    const float mp = a.min_p ? a.min_p[r] : 0.f;
    const double least = mp > 0.f ? fmin((double)mp, 1.) : 0.;
    auto final = [&](int i) {
        const unsigned key = row.key(i);
        if (!kept.has(key, i)) return 0ull;
        const double w = row.weight(key);
        return w >= least ? row.fixed(w) : 0ull;
    };
    const u64 all = block_sum(sh, [&](int i) { return i < v1 ? final(i) : 0ull; }, v0, v1);
    const float u = a.u[r];
    const double aim = u > 0.f ? (double)u * (double)all : 0.;
    const u64 want = aim < (double)all ? (u64)aim : all - 1;  // the first sum above it
    u64 before = 0;
    for (int w = 0; w < wave; ++w) before += sh.part[w];
    if (before <= want && want < before + sh.part[wave]) {
        for (int i0 = v0; i0 < v1; i0 += WAVE) {
            const int i = i0 + lane;
            const u64 w = i < v1 ? final(i) : 0;
            u64 sum = w;
#pragma unroll
            for (int o = 1; o < WAVE; o <<= 1) {
                const u64 up = __shfl_up(sum, o, WAVE);
                if (lane >= o) sum += up;
            }
            const u64 reach = __ballot(before + sum > want);
            if (reach) {
                if (lane == 0) a.out[r] = i0 + __ffsll((long long)reach) - 1;
                break;
            }
            before += __shfl(sum, WAVE - 1, WAVE);
        }
    }
}

}  // namespace

extern "C" int smg_sample_launch(const void* logits, const void* u, const void* temperature,
                                 const void* top_k, const void* top_p, const void* min_p, void* out,
                                 long long stride, int R, int V, int f32, void* stream) {
    if (V < 1) return -1;
    if (R < 1) return 0;
    SampleArgs a = {logits, stride, (const float*)u, (const float*)temperature, (const int*)top_k,
                    (const float*)top_p, (const float*)min_p, (long long*)out, R, V};
    if (f32)
        hipLaunchKernelGGL(smg_sample_t<true>, dim3(R), dim3(THREADS), 0, (hipStream_t)stream, a);
    else
        hipLaunchKernelGGL(smg_sample_t<false>, dim3(R), dim3(THREADS), 0, (hipStream_t)stream, a);
    return hipGetLastError() == hipSuccess ? 0 : -2;
}
