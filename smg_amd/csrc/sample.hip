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
// steps of the logit below the largest, which LDS atomics fill (for a small top-k
// each thread's largest token alone: they bound the k-th of all).  The tokens down to
// the step in which the number is reached are listed in index order, if they fit,
// and all that follows runs over the list.  The tokens of that step are compared with
// each other; where they are more than CAND, the step is divided again, until it
// holds few tokens or one value, and equal values go by index.  Nothing is sorted.
//
// A workgroup has a row, and each wave a run of it, 512 tokens at a time, 8 a
// lane, so that index order is (wave, iteration, lane, element).
//
// What bounds it: a pass that weighs every token, about 45 vector instructions each, half
// of them in 64 bits; without a cut that is one pass (512 rows of 32768 in bf16 on an
// MI355X: 25 us, the memory's part 7), with a top-p the one that fills the histogram, and
// the list after it (44 us), or another pass where the list does not hold what is kept
// (61 us).  A top-k of 50 weighs only the list (19 us), temperature 0 nothing (10 us).
// One row of 2048 with a top-p: 8.2 us, most of it barriers and latency.
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>

#include <cstdint>

#define WAVE 64
#define NB 2048             // steps of a histogram; also the most blocks
#define BLOCK 512           // tokens of a wave's iteration
#define MAX_V (NB * BLOCK)
#define DEEP 2              // loads of a wave on their way in a pass that computes
#define LIGHT 4             // and in one that only compares
#define MAX_PARTS 16        // workgroups of a row
#define NONE 0x7fffffff

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
    u64* work;                 // split rows: [R] of Work
    int parts;                 // workgroups that share a row (1: none do)
};

// What the workgroups of a row leave for each other.
struct Work {
    u64 hist[NB];        // of the first cut's measure
    u64 blocks[NB];      // sums of weights, 512 tokens each
    float lo[MAX_PARTS], hi[MAX_PARTS];
    int first[MAX_PARTS];  // the first index of each part's largest
    float x;             // what the cuts keep, if `open`
    int i;
    int open;            // whether the row still needs its answer
    int pad;
};

// ---- a wave's scans, by lane moves within the vector unit ---------------------
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned moved(unsigned x, unsigned none) {
    return (unsigned)__builtin_amdgcn_update_dpp((int)none, (int)x, CTRL, ROWS, 0xf, false);
}
// x of the lanes 1, 2, 4, 8 before within 16, then of lane 15 and lane 31 of the
// 16s before: the six steps of an inclusive scan over 64 lanes
#define SCAN_STEPS(STEP) STEP(0x111, 0xf) STEP(0x112, 0xf) STEP(0x114, 0xf) STEP(0x118, 0xf) STEP(0x142, 0xa) STEP(0x143, 0xc)

__device__ __forceinline__ u64 wave_scan(u64 x) {
#define STEP(CTRL, ROWS)                                                       \
    x += (u64)moved<CTRL, ROWS>((unsigned)(x >> 32), 0) << 32 | moved<CTRL, ROWS>((unsigned)x, 0);
    SCAN_STEPS(STEP)
#undef STEP
    return x;
}
__device__ __forceinline__ int wave_scan(int x) {
#define STEP(CTRL, ROWS) x += (int)moved<CTRL, ROWS>((unsigned)x, 0);
    SCAN_STEPS(STEP)
#undef STEP
    return x;
}
__device__ __forceinline__ float wave_max(float x) {
#define STEP(CTRL, ROWS) \
    x = fmaxf(x, __uint_as_float(moved<CTRL, ROWS>(__float_as_uint(x), 0xff800000u)));
    SCAN_STEPS(STEP)
#undef STEP
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), 63));
}
__device__ __forceinline__ u64 at_lane(u64 x, int lane) {
    return (u64)(unsigned)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32 |
           (unsigned)__builtin_amdgcn_readlane((int)x, lane);
}
__device__ __forceinline__ u64 wave_sum(u64 x) { return at_lane(wave_scan(x), 63); }

// What a workgroup of THREADS does, with up to LIST listed tokens, and CAND that are
// compared with each other.
template <int THREADS, int LIST, int CAND = 128>
struct Sampler {
    static constexpr int WAVES = THREADS / WAVE;

    struct Shared {
        u64 hist[NB];
        float list_x[LIST];
        int list_i[LIST];
        double pow2[64];  // 2^(i/64 + S)
        u64 part[WAVES];
        float lo[WAVES], hi[WAVES];
        int ints[WAVES];
        u64 cand_m[CAND], cand_before[CAND];
        float cand_x[CAND];
        int cand_i[CAND];
        u64 above;
        float px;
        int pi, bin, count, index;
    };

    // (lowest, highest) over the workgroup
    static __device__ __forceinline__ float2 block_range(Shared& sh, float lo, float hi) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x / WAVE;
        lo = wave_max(-lo), hi = wave_max(hi);
        __syncthreads();
        if (lane == 0) sh.lo[wave] = lo, sh.hi[wave] = hi;
        __syncthreads();
        lo = sh.lo[lane & (WAVES - 1)], hi = sh.hi[lane & (WAVES - 1)];
        return make_float2(-wave_max(lo), wave_max(hi));
    }
    // the sum over the waves before this one of what each has in v[wave]
    template <typename T>
    static __device__ __forceinline__ T before_wave(const T* v, T* all) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
        const T run = wave_scan(lane < WAVES ? v[lane] : (T)0);
        if constexpr (sizeof(T) == 8) {
            *all = at_lane(run, WAVES - 1);
            return wave ? at_lane(run, wave - 1) : 0;
        } else {
            *all = __builtin_amdgcn_readlane(run, WAVES - 1);
            return wave ? __builtin_amdgcn_readlane(run, wave - 1) : 0;
        }
    }

    static __device__ __forceinline__ void clear(Shared& sh) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NB / THREADS; ++i) sh.hist[threadIdx.x + i * THREADS] = 0;
        __syncthreads();
    }

    static __device__ __forceinline__ void load(Shared& sh, const u64* from, int n) {
        __syncthreads();
#pragma unroll
        for (int i = threadIdx.x; i < NB; i += THREADS) sh.hist[i] = i < n ? from[i] : 0;
    }

    // Adds numbers up, of which thread t has the sums sum[] of the first 1, 2, .. of its own,
    // number `own` * t and so on: sh.bin and sh.above get the first number at which the sum
    // reaches want(sum of all) and the sum before it (bin NONE if it never does).  Returns
    // that want.
    template <int OWN, typename W>
    static __device__ __forceinline__ u64 locate(Shared& sh, const u64 (&sum)[OWN], int own, W&& want_of) {
        const int t = threadIdx.x;
        const u64 run = wave_scan(sum[OWN - 1]);
        if ((t & 63) == 63) sh.part[t / WAVE] = run;
        if (t == 0) sh.bin = NONE;
        __syncthreads();
        u64 all;
        const u64 before = before_wave(sh.part, &all) + run - sum[OWN - 1];
        const u64 want = want_of(all);
        if (before < want && before + sum[OWN - 1] >= want) {
            int n = 0;
            u64 above = before;
#pragma unroll
            for (int i = 0; i < OWN - 1; ++i)
                if (before + sum[i] < want) n = i + 1, above = before + sum[i];
            sh.bin = own * t + n;
            sh.above = above;
        }
        __syncthreads();
        return want;
    }
    // the same of the NB counters of sh.hist
    template <typename W>
    static __device__ __forceinline__ u64 locate(Shared& sh, W&& want_of) {
        constexpr int OWN = NB / THREADS;
        __syncthreads();
        u64 sum[OWN];
#pragma unroll
        for (int i = 0; i < OWN; ++i) sum[i] = sh.hist[OWN * threadIdx.x + i] + (i ? sum[i - 1] : 0);
        return locate(sh, sum, OWN, want_of);
    }

    // the order's tokens up to the value x, of those equal to x up to index i
    struct Prefix {
        float x;
        int i;
        __device__ __forceinline__ bool has(float y, int j) const { return (y > x) | ((y == x) & (j <= i)); }
    };

    // exp((x - top) / t) in 64 bits: 2^(n/64) from a table times a polynomial of
    // 2^r, |r| <= 1/128 (off by 4e-14 at most), as a multiple of 2^-S
    struct Weigh {
        const double* pow2;
        double top, c, units;
        float floor, cap;  // below the floor weights are 0; +inf weighs as the cap
        __device__ __forceinline__ void init(Shared& sh, float largest, float t, int V) {
            const int S = min(50, 62 - (V > 1 ? 32 - __clz(V - 1) : 0));
            units = (double)(1ull << S);
            pow2 = sh.pow2;
            // where the largest is +inf, only that weighs anything
            cap = fminf(largest, 3.40282347e38f);
            top = (double)cap;
            c = 64. * 1.44269504088896340736 / (double)t;
            floor = largest == INFINITY ? INFINITY : fmaxf(largest - 45.f * t, -3.40282347e38f);  // 2^-64
            if (threadIdx.x < 64) sh.pow2[threadIdx.x] = exp2((double)threadIdx.x / 64) * units;
        }
        __device__ __forceinline__ double scaled(float x) const {  // weight * 2^S
            constexpr double magic = 6755399441055744., q = 0.6931471805599453094 / 64;
            const double d = (double)fminf(fmaxf(x, floor), cap) - top;  // NaN goes to the floor
            const double n = fma(d, c, magic);                           // the nearest integer in its low bits
            const double r = fma(d, c, magic - n);
            double p = fma(r, q * q * q * q / 24, q * q * q / 6);
            p = fma(r, p, q * q / 2);
            p = fma(r, p, q);
            p = fma(r, p, 1.);
            const int k = (int)__double_as_longlong(n);
            const long long bits = __double_as_longlong(p * pow2[k & 63]);
            // times 2^(k/64): to the exponent, which stays in range (above 2^-66)
            return __longlong_as_double(bits + ((long long)(k & ~63) << 46));
        }
        __device__ __forceinline__ u64 rounded(double scaled) const {
            return (u64)__double_as_longlong(scaled + 4503599627370496.) & 0xfffffffffffffull;
        }
        __device__ __forceinline__ u64 fixed(float x, bool live) const {
            const u64 w = rounded(scaled(x));
            return live & (x >= floor) ? w : 0;
        }
    };

    // ---- the tokens: f(i, x) for each of the thread's, in index order ---------------
    // FEW: V < 8, where 8 tokens cannot be loaded at once.
    template <bool F32, bool FEW>
    struct Row {
        static constexpr bool LISTED = false;
        const char* at;
        int V, start, end, its, lane;  // this wave's run, in `its` iterations at most

        struct Raw {
            u32x4 w[F32 ? 2 : 1];
            __device__ __forceinline__ float operator[](int e) const {
                return __uint_as_float(F32 ? w[e / 4][e % 4] : e % 2 ? w[0][e / 2] & 0xffff0000u : w[0][e / 2] << 16);
            }
            __device__ __forceinline__ void drop(int e) {
                if (F32)
                    w[e / 4][e % 4] = 0x7fc00000u;
                else
                    w[0][e / 2] = e % 2 ? (w[0][e / 2] & 0xffffu) | 0x7fc00000u : (w[0][e / 2] & 0xffff0000u) | 0x7fc0u;
            }
        };
        // the first of an iteration's 8 tokens, and the first that is in memory: at the
        // row's end a lane reads the last 8 and drops those before its own
        __device__ __forceinline__ int first(int it) const { return start + it * BLOCK + lane * 8; }
        __device__ __forceinline__ int base(int it) const { return FEW ? first(it) : min(first(it), V - 8); }
        __device__ __forceinline__ Raw load8(int it) const {
            const int i = first(it), b = base(it);
            Raw r = {};
            if constexpr (FEW) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    r.drop(e);
                    if (i + e >= V) continue;
                    if (F32)
                        r.w[e / 4][e % 4] = ((const unsigned*)at)[i + e];
                    else
                        r.w[0][e / 2] = (r.w[0][e / 2] & (e % 2 ? 0xffffu : 0xffff0000u)) | (unsigned)((const unsigned short*)at)[i + e] << (e % 2 * 16);
                }
            } else {
                // rows may start anywhere: the hardware takes wide loads at any element
                __builtin_memcpy(&r, at + (size_t)b * (F32 ? 4 : 2), F32 ? 32 : 16);
                if (b < i) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (b + e < i) r.drop(e);
                }
            }
            return r;
        }
        __device__ __forceinline__ float value(int i) const {
            return __uint_as_float(F32 ? ((const unsigned*)at)[i] : (unsigned)((const unsigned short*)at)[i] << 16);
        }
        // row r, or part `part` of `parts` of it
        __device__ __forceinline__ void init(const SampleArgs& a, int r, int part = 0, int parts = 1) {
            lane = threadIdx.x & 63;
            V = a.V;
            at = (const char*)a.logits + r * a.stride * (F32 ? 4 : 2);
            const int blocks = (V + BLOCK - 1) / BLOCK, mine = (blocks + parts - 1) / parts;
            its = (mine + WAVES - 1) / WAVES;
            end = min(V, (part + 1) * mine * BLOCK);
            start = part * mine * BLOCK + __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE) * its * BLOCK;
        }
        template <typename F>
        __device__ __forceinline__ void each8(int it, const Raw& r, F&& f) const {
            const int b = base(it);
#pragma unroll
            for (int e = 0; e < 8; ++e) f(b + e, r[e]);
        }
        // g(it, raw) for each iteration that has tokens: ON_WAY loads at once
        template <int ON_WAY = DEEP, typename G>
        __device__ __forceinline__ void blocks(G&& g) const {
            const int n = min(its, (end - start + BLOCK - 1) / BLOCK);
            for (int i0 = 0; i0 < n; i0 += ON_WAY) {
                Raw r[ON_WAY];
#pragma unroll
                for (int i = 0; i < ON_WAY; ++i)
                    if (i0 + i < n) r[i] = load8(i0 + i);
#pragma unroll
                for (int i = 0; i < ON_WAY; ++i)
                    if (i0 + i < n) g(i0 + i, r[i]);
            }
        }
        template <int ON_WAY = DEEP, typename F>
        __device__ __forceinline__ void each(F&& f) const {
            blocks<ON_WAY>([&](int it, const Raw& r) { each8(it, r, f); });
        }
        // f(x, measure(i, x)) where that is not 0; the measures of 8 tokens side by side
        template <typename M, typename F>
        __device__ __forceinline__ void weighed(M&& measure, F&& f) const {
            blocks([&](int it, const Raw& r) {
                u64 w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = measure(base(it) + e, r[e]);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (w[e]) f(r[e], w[e]);
            });
        }
        // Sums of measure(i, x) over 512 tokens each.
        template <typename M>
        __device__ __forceinline__ void sums(u64* to, M&& measure) const {
            blocks([&](int it, const Raw& r) {
                u64 s = 0;
                each8(it, r, [&](int i, float x) { s += measure(i, x); });
                s = wave_sum(s);
                if (lane == 0) to[start / BLOCK + it] = s;
            });
        }
        // The first index at which the sums of measure(i, x), by index, reach
        // want(sum of all), which is at least 1 and at most that.  `given`: those sums.
        template <typename W, typename M>
        __device__ __forceinline__ int find(Shared& sh, W&& want_of, M&& measure, const u64* given = nullptr) const {
            if (given) {
                load(sh, given, (V + BLOCK - 1) / BLOCK);
            } else {
                clear(sh);
                sums(sh.hist, measure);
            }
            u64 want = locate(sh, want_of);
            const int it = sh.bin - start / BLOCK;
            if (it >= 0 && it < its) {
                want -= sh.above;
                const Raw r = load8(it);
                u64 s[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) s[e] = measure(base(it) + e, r[e]) + (e ? s[e - 1] : 0);
                const u64 before = wave_scan(s[7]) - s[7];
                if (before < want && before + s[7] >= want) {
                    int n = 0;
#pragma unroll
                    for (int j = 0; j < 7; ++j) n += before + s[j] < want;
                    sh.index = base(it) + n;
                }
            }
            __syncthreads();
            return sh.index;
        }
        // f(i, x) for the tokens that `rare`, a comparison that few pass
        template <typename P, typename F>
        __device__ __forceinline__ void some(P&& rare, F&& f) const {
            blocks<LIGHT>([&](int it, const Raw& r) {
                for (unsigned hits = these(it, r, [&](int, float x) { return rare(x); }); hits; hits &= hits - 1) {
                    const int i = base(it) + __ffs(hits) - 1;
                    f(i, value(i));
                }
            });
        }
        // a bit for each of an iteration's 8 tokens that `has`
        template <typename H>
        __device__ __forceinline__ unsigned these(int it, const Raw& r, H&& has) const {
            unsigned hits = 0;
            const int b = base(it);
#pragma unroll
            for (int e = 0; e < 8; ++e) hits |= has(b + e, r[e]) ? 1u << e : 0u;
            return hits;
        }
        // Lists the tokens that `has` in index order, if they fit; their number.
        template <typename H>
        __device__ __forceinline__ int list(Shared& sh, H&& has) const {
            int c = 0;
            each<LIGHT>([&](int i, float x) { c += has(i, x); });
            c = __builtin_amdgcn_readlane(wave_scan(c), 63);
            __syncthreads();
            if (lane == 0) sh.ints[threadIdx.x / WAVE] = c;
            __syncthreads();
            int all, at = before_wave(sh.ints, &all);
            if (all > LIST) {
                __syncthreads();
                return all;
            }
            if (c) blocks<LIGHT>([&](int it, const Raw& r) {
                unsigned hits = these(it, r, has);
                const int n = __popc(hits), run = wave_scan(n);
                int to = at + run - n;
                at += __builtin_amdgcn_readlane(run, 63);
                for (; hits; hits &= hits - 1) sh.list_i[to++] = base(it) + __ffs(hits) - 1;
            });
            __syncthreads();
            for (int i = threadIdx.x; i < all; i += THREADS) sh.list_x[i] = value(sh.list_i[i]);
            __syncthreads();
            return all;
        }
    };

    // The tokens that a cut left: i is their place in the list.
    struct List {
        static constexpr bool LISTED = true;
        static constexpr int MOST = LIST / THREADS;  // tokens of a thread
        Shared* sh;
        int n, own;
        __device__ __forceinline__ void set(int tokens) { n = tokens, own = (n + THREADS - 1) / THREADS; }
        __device__ __forceinline__ bool fits() const { return n <= LIST; }
        template <typename F>
        __device__ __forceinline__ void each(F&& f) const {
            for (int i = own * threadIdx.x, end = min(n, i + own); i < end; ++i) f(i, sh->list_x[i]);
        }
        template <typename P, typename F>
        __device__ __forceinline__ void some(P&& rare, F&& f) const {
            each([&](int i, float x) {
                if (rare(x)) f(i, x);
            });
        }
        template <typename M, typename F>
        __device__ __forceinline__ void weighed(M&& measure, F&& f) const {
            each([&](int i, float x) {
                const u64 w = measure(i, x);
                if (w) f(x, w);
            });
        }
        template <typename W, typename M>
        __device__ __forceinline__ int find(Shared& s, W&& want_of, M&& measure) const {
            u64 sum[MOST];
#pragma unroll
            for (int e = 0; e < MOST; ++e) {
                const int i = own * threadIdx.x + e;
                sum[e] = e ? sum[e - 1] : 0;
                if (e < own && i < n) sum[e] += measure(i, s.list_x[i]);
            }
            __syncthreads();
            locate(s, sum, own, want_of);
            return s.bin;
        }
    };

    // Finds the shortest prefix of the order whose measure reaches a number: counts, or
    // weights, of the tokens that `from` has.
    template <typename T, typename Step>
    struct Search {
        Shared& sh;
        const T& tokens;
        const Weigh& weigh;
        Step step;  // NB falling steps of the logit; the last one's tokens weigh nothing
        bool counting;
        Prefix from;

        __device__ __forceinline__ u64 measure(int i, float x) const {
            if (counting) return (u64)from.has(x, i);
            return weigh.fixed(x, from.has(x, i));
        }
        // The measure of each step, into sh.hist.
        __device__ __forceinline__ void fill() const {
            clear(sh);
            if (counting)
                tokens.each([&](int i, float x) {
                    if (from.has(x, i)) atomicAdd(&sh.hist[step(x)], 1ull);
                });
            else
                tokens.weighed([&](int i, float x) { return weigh.fixed(x, from.has(x, i)); },
                               [&](float x, u64 w) { atomicAdd(&sh.hist[step(x)], w); });
        }
        // The step in which want(sum of all) is reached, NB - 1 or more if it never is.
        template <typename W>
        __device__ __forceinline__ u64 divide(W&& want_of, const u64* given = nullptr) const {
            if (given)
                load(sh, given, NB);
            else
                fill();
            return locate(sh, want_of);
        }
        // The prefix, from the step `bin` in which `want` is reached and the measure
        // `above` it.
        __device__ __forceinline__ Prefix within(int bin, u64 above, u64 want) const {
            float top = step.highest(bin), bottom = step.lowest(bin);  // `again`: of the last division
            double c = 0.;
            bool again = false;
            for (;;) {
                want -= above;
                if (threadIdx.x == 0) sh.count = 0;
                if (threadIdx.x < CAND) sh.cand_before[threadIdx.x] = 0;
                __syncthreads();
                float lo = INFINITY, hi = -INFINITY;
                tokens.some([&](float x) { return (x >= bottom) & (x <= top); }, [&](int i, float x) {
                    if ((again ? min(NB - 1, (int)(((double)top - (double)x) * c)) : step(x)) != bin) return;
                    const u64 w = measure(i, x);
                    if (!w) return;
                    lo = fminf(lo, x), hi = fmaxf(hi, x);
                    const int at = atomicAdd(&sh.count, 1);
                    if (at < CAND) sh.cand_x[at] = x, sh.cand_i[at] = i, sh.cand_m[at] = w;
                });
                __syncthreads();
                const int n = sh.count;
                if (n <= CAND) {
                    // some of the candidates, from this thread's first on, that come before
                    // this thread's own
                    const int me = threadIdx.x & (CAND - 1), first = threadIdx.x / CAND;
                    const float x = sh.cand_x[me];
                    const int i = sh.cand_i[me];
                    if (me < n) {
                        u64 s = 0;
                        for (int j = first; j < n; j += THREADS / CAND) {
                            const float y = sh.cand_x[j];
                            if (y > x || (y == x && sh.cand_i[j] < i)) s += sh.cand_m[j];
                        }
                        if (s) atomicAdd(&sh.cand_before[me], s);
                    }
                    __syncthreads();
                    if (threadIdx.x < n) {
                        const u64 s = sh.cand_before[me];
                        if (s < want && s + sh.cand_m[me] >= want) sh.px = x, sh.pi = i;
                    }
                    __syncthreads();
                    return {sh.px, sh.pi};
                }
                const float2 r = block_range(sh, lo, hi);
                if (r.x == r.y) {
                    const float x0 = r.x;
                    return {x0, tokens.find(sh, [&](u64) { return want; }, [&](int i, float x) { return x == x0 ? measure(i, x) : 0ull; })};
                }
                // the ends fall into different steps, so this ends
                again = true;
                bottom = r.x, top = r.y;
                c = (NB - 1) / ((double)top - (double)bottom);
                clear(sh);
                tokens.each([&](int i, float x) {
                    if (!(x >= bottom && x <= top)) return;
                    const u64 w = measure(i, x);
                    if (w) atomicAdd(&sh.hist[min(NB - 1, (int)(((double)top - (double)x) * c))], w);
                });
                locate(sh, [&](u64) { return want; });
                bin = sh.bin, above = sh.above;
            }
        }
        template <typename W>
        __device__ __forceinline__ Prefix operator()(W&& want_of, const u64* given = nullptr) const {
            const u64 want = divide(want_of, given);
            return sh.bin >= NB - 1 ? from : within(sh.bin, sh.above, want);
        }
    };

    static __device__ __forceinline__ u64 share(float p, u64 all) {  // the measure that top-p asks for
        const double want = ceil((double)p * (double)all);
        return want >= 1. ? (u64)want : 1;
    }

    struct Step {
        float cap, half, per;  // halves, whose differences stay in range
        __device__ __forceinline__ int operator()(float x) const { return (int)fminf(fmaf(fminf(x, cap), -.5f, half) * per, NB - 1.f); }
        // values above -inf between which the tokens of the steps up to `bin`, or from it on,
        // lie, and few others
        __device__ __forceinline__ float lowest(int bin) const {
            const double x = (double)cap - 2. * (bin + 1) / (double)per * (1. + 1e-6);
            return fmaxf((float)(x - fabs(x) * 1e-6), -3.40282347e38f);
        }
        __device__ __forceinline__ float highest(int bin) const {
            if (bin == 0) return INFINITY;
            const double x = (double)cap - 2. * bin / (double)per * (1. - 1e-6);
            return fmaxf((float)(x + fabs(x) * 1e-6), -3.40282347e38f);
        }
    };

    // A row's settings, and what follows from its largest and smallest logit.
    struct Plan {
        Weigh weigh;
        Step step;
        Prefix all;  // everything above -inf, or the +inf
        int k;
        float p, u, t;
        double least;  // the smallest weight that min-p keeps, in units
        bool by_count, by_mass;

        __device__ __forceinline__ Plan(const SampleArgs& a, int r) {
            t = a.temperature[r];
            k = a.top_k ? a.top_k[r] : 0;
            p = a.top_p ? a.top_p[r] : 1.f;
            u = a.u[r];
            by_count = k > 0 && k < a.V;
            by_mass = p < 1.f;
        }
        __device__ __forceinline__ void init(Shared& sh, const SampleArgs& a, int r, float2 ends) {
            weigh.init(sh, ends.y, t, a.V);
            // steps down from the largest: to the smallest, or to where weights are 0
            // (below 2^-51), whose tokens the last step takes
            const float half = .5f * weigh.cap, depth = fminf(fmaf(ends.x, -.5f, half), .5f * 51.f * 0.69314718f * t);
            step = {weigh.cap, half, depth > 1e-30f ? (NB - 2) / depth : 0.f};
            all = {ends.y == INFINITY ? weigh.cap : -INFINITY, -1};
            const float mp = a.min_p ? a.min_p[r] : 0.f;
            least = mp > 0.f ? fmin((double)mp, 1.) * weigh.units : 0.;
        }
        // what the tokens of the steps up to `bin` reach
        __device__ __forceinline__ float lowest(int bin) const { return all.x >= weigh.cap ? INFINITY : step.lowest(bin); }
        // the weights that `kept` and min-p leave
        template <bool CUT>
        __device__ __forceinline__ u64 left(Prefix kept, int i, float x) const {
            const double w = weigh.scaled(x);
            const bool live = (x >= weigh.floor) & (w >= least);
            return (CUT ? live & kept.has(x, i) : live) ? weigh.rounded(w) : 0ull;
        }
        // the first token by index at which they reach more than u of their sum
        template <bool CUT, typename T>
        __device__ __forceinline__ int draw(Shared& sh, const T& tokens, Prefix kept, const u64* given = nullptr) const {
            auto want_of = [&](u64 sum) {
                const double aim = u > 0.f ? (double)u * (double)sum : 0.;
                return aim < (double)sum ? (u64)aim + 1 : sum;
            };
            auto measure = [&](int i, float x) { return left<CUT>(kept, i, x); };
            if constexpr (T::LISTED)
                return tokens.find(sh, want_of, measure);
            else
                return tokens.find(sh, want_of, measure, given);
        }
    };

    // Top-k, then top-p: what they keep, as a prefix of the list if that holds it
    // (list.fits()), else of the row.  hi: the largest of this thread's tokens; given: the
    // first cut's measures of the steps, by other workgroups.
    template <typename R>
    static __device__ __forceinline__ Prefix cut(Shared& sh, const R& row, const Plan& plan, List& list, float hi, const u64* given) {
        const Prefix all = plan.all;
        Prefix kept = all;
        if (plan.by_count) {
            const Search<R, Step> search = {sh, row, plan.weigh, plan.step, true, all};
            auto want_of = [&](u64) { return (u64)plan.k; };
            const bool few = !given && plan.k <= THREADS / 2;
            if (few) {
                // the threads' largest tokens alone bound the k-th of all: what lies in
                // their k-th's step or above is few
                clear(sh);
                if (hi > all.x) atomicAdd(&sh.hist[plan.step(hi)], 1ull);
                locate(sh, want_of);
            } else {
                search.divide(want_of, given);
            }
            const int bin = sh.bin;
            const u64 above = sh.above;
            const float low = plan.lowest(bin);
            if (bin < NB - 1 && plan.k <= LIST) list.set(row.list(sh, [&](int, float x) { return x >= low; }));
            if (list.fits()) {
                const Search<List, Step> among = {sh, list, plan.weigh, plan.step, true, all};
                kept = few ? among(want_of) : among.within(bin, above, plan.k);
            } else {
                kept = few ? search(want_of) : bin < NB - 1 ? search.within(bin, above, plan.k) : all;
                list.set(row.list(sh, [&](int i, float x) { return kept.has(x, i); }));
                if (list.fits()) kept = all;
            }
        }
        if (plan.by_mass) {
            auto want_of = [&](u64 sum) { return share(plan.p, sum); };
            if (!list.fits()) {
                const Search<R, Step> search = {sh, row, plan.weigh, plan.step, false, kept};
                const u64 want = search.divide(want_of, plan.by_count ? nullptr : given);
                const int bin = sh.bin;
                const u64 above = sh.above;
                if (bin < NB - 1) {
                    const float low = plan.lowest(bin);
                    if (plan.by_count)
                        list.set(row.list(sh, [&](int i, float x) { return (x >= low) & kept.has(x, i); }));
                    else
                        list.set(row.list(sh, [&](int, float x) { return x >= low; }));
                    if (list.fits()) {
                        const Search<List, Step> among = {sh, list, plan.weigh, plan.step, false, all};
                        kept = among.within(bin, above, want);
                    } else {
                        kept = search.within(bin, above, want);
                    }
                }
            } else {
                const Search<List, Step> among = {sh, list, plan.weigh, plan.step, false, kept};
                kept = among(want_of);
            }
        }
        return kept;
    }

    // (smallest above -inf, largest) of the tokens, over the workgroup; hi: this thread's
    template <typename R>
    static __device__ __forceinline__ float2 ends_of(Shared& sh, const R& row, float& hi) {
        float lo = INFINITY;
        hi = -INFINITY;
        row.template each<LIGHT>([&](int, float x) {
            hi = fmaxf(hi, x);  // NaN is passed over
            lo = fminf(lo, x > -INFINITY ? x : lo);
        });
        return block_range(sh, lo, hi);
    }
    template <typename R>
    static __device__ __forceinline__ int first_of(Shared& sh, const R& row, float largest) {
        int first = 0x7fffffff;
        if (threadIdx.x == 0) sh.index = 0x7fffffff;
        row.template each<LIGHT>([&](int i, float x) { first = min(first, x == largest ? i : 0x7fffffff); });
        __syncthreads();
        if (first != 0x7fffffff) atomicMin(&sh.index, first);
        __syncthreads();
        return sh.index;
    }
};

template <int THREADS, int LIST, bool F32, bool FEW>
__global__ void __launch_bounds__(THREADS) smg_sample_t(SampleArgs a) {
    using Z = Sampler<THREADS, LIST>;
    __shared__ typename Z::Shared sh;
    const int r = blockIdx.x;
    typename Z::template Row<F32, FEW> row;
    row.init(a, r);
    float hi;
    const float2 ends = Z::ends_of(sh, row, hi);
    typename Z::Plan plan(a, r);
    int found = -1;
    if (ends.y > -INFINITY && !(plan.t > 0.f)) {
        found = Z::first_of(sh, row, ends.y);
    } else if (ends.y > -INFINITY) {
        plan.init(sh, a, r, ends);
        typename Z::List list = {&sh, NONE, 0};
        const typename Z::Prefix kept = Z::cut(sh, row, plan, list, hi, nullptr);
        if (list.fits())
            found = sh.list_i[plan.template draw<true>(sh, list, kept)];
        else if (plan.by_count || plan.by_mass)
            found = plan.template draw<true>(sh, row, kept);
        else
            found = plan.template draw<false>(sh, row, kept);
    }
    if (threadIdx.x == 0) a.out[r] = found;
}

// ---- few long rows: workgroups share a row, in five launches ---------------------
// Each of the passes over a row that cost the most (the largest logit, the first cut's
// measures, the last sums) has `parts` workgroups a row; the searches between them have
// one.  Integer sums make the answer the same.
// Their steps hold more tokens: 64 rows of 131071 take 71 us where 256 are compared, 82 with
// 128 and another division; 512 shorter rows 58 and 56.
using Wide = Sampler<1024, 8192, 256>;
using Slim = Sampler<1024, 1024>;  // where nothing is listed: more workgroups fit a compute unit
__device__ __forceinline__ float2 ends_of(const Work& w, int parts) {
    const int lane = threadIdx.x & 63;
    const float lo = lane < parts ? w.lo[lane] : INFINITY, hi = lane < parts ? w.hi[lane] : -INFINITY;
    return make_float2(-wave_max(-lo), wave_max(hi));
}

template <bool F32>
__global__ void __launch_bounds__(1024) smg_sample_ends_t(SampleArgs a) {
    __shared__ Slim::Shared sh;
    const int part = blockIdx.x, r = blockIdx.y;
    Work& w = ((Work*)a.work)[r];
    Slim::Row<F32, false> row;
    row.init(a, r, part, a.parts);
    for (int i = part * 1024 + threadIdx.x; i < NB; i += a.parts * 1024) w.hist[i] = 0;
    float hi;
    const float2 ends = Slim::ends_of(sh, row, hi);
    const int first = a.temperature[r] > 0.f ? 0 : Slim::first_of(sh, row, ends.y);
    if (threadIdx.x == 0) w.lo[part] = ends.x, w.hi[part] = ends.y, w.first[part] = first;
}

// the first cut's measures, or without a cut the last sums
template <bool F32>
__global__ void __launch_bounds__(1024) smg_sample_measure_t(SampleArgs a) {
    __shared__ Slim::Shared sh;
    const int part = blockIdx.x, r = blockIdx.y;
    Work& w = ((Work*)a.work)[r];
    const float2 ends = ends_of(w, a.parts);
    Slim::Plan plan(a, r);
    if (ends.y == -INFINITY || !(plan.t > 0.f)) return;
    plan.init(sh, a, r, ends);
    Slim::Row<F32, false> row;
    row.init(a, r, part, a.parts);
    if (!plan.by_count && !plan.by_mass) {
        __syncthreads();
        row.sums(w.blocks, [&](int i, float x) { return plan.template left<false>(plan.all, i, x); });
        return;
    }
    const Slim::Search<Slim::Row<F32, false>, Slim::Step> search = {sh, row, plan.weigh, plan.step, plan.by_count, plan.all};
    search.fill();
    __syncthreads();
    for (int i = threadIdx.x; i < NB; i += 1024)
        if (sh.hist[i]) atomicAdd(&w.hist[i], sh.hist[i]);
}

template <bool F32>
__global__ void __launch_bounds__(1024) smg_sample_cut_t(SampleArgs a) {
    __shared__ Wide::Shared sh;
    const int r = blockIdx.x;
    Work& w = ((Work*)a.work)[r];
    const float2 ends = ends_of(w, a.parts);
    Wide::Plan plan(a, r);
    Wide::Row<F32, false> row;
    row.init(a, r);
    int found = -1;
    bool open = false;
    if (ends.y > -INFINITY && !(plan.t > 0.f)) {
        for (int part = a.parts - 1; part >= 0; --part)
            if (w.hi[part] == ends.y) found = w.first[part];
    } else if (ends.y > -INFINITY) {
        plan.init(sh, a, r, ends);
        if (!plan.by_count && !plan.by_mass) {
            found = plan.draw<false>(sh, row, plan.all, w.blocks);
        } else {
            Wide::List list = {&sh, NONE, 0};
            const Wide::Prefix kept = Wide::cut(sh, row, plan, list, 0.f, w.hist);
            open = !list.fits();
            if (open)
                w.x = kept.x, w.i = kept.i;
            else
                found = sh.list_i[plan.draw<true>(sh, list, kept)];
        }
    }
    if (threadIdx.x == 0) {
        w.open = open;
        a.out[r] = found;
    }
}

// the last sums of the rows that are still open
template <bool F32>
__global__ void __launch_bounds__(1024) smg_sample_sums_t(SampleArgs a) {
    __shared__ Slim::Shared sh;
    const int part = blockIdx.x, r = blockIdx.y;
    Work& w = ((Work*)a.work)[r];
    if (!w.open) return;
    Slim::Plan plan(a, r);
    plan.init(sh, a, r, ends_of(w, a.parts));
    __syncthreads();
    Slim::Row<F32, false> row;
    row.init(a, r, part, a.parts);
    const Slim::Prefix kept = {w.x, w.i};
    row.sums(w.blocks, [&](int i, float x) { return plan.template left<true>(kept, i, x); });
}

template <bool F32>
__global__ void __launch_bounds__(1024) smg_sample_pick_t(SampleArgs a) {
    __shared__ Wide::Shared sh;
    const int r = blockIdx.x;
    Work& w = ((Work*)a.work)[r];
    if (!w.open) return;
    Wide::Plan plan(a, r);
    plan.init(sh, a, r, ends_of(w, a.parts));
    Wide::Row<F32, false> row;
    row.init(a, r);
    const int found = plan.draw<true>(sh, row, {w.x, w.i}, w.blocks);
    if (threadIdx.x == 0) a.out[r] = found;
}

template <bool F32>
void launch(const SampleArgs& a, hipStream_t s) {
    // 512 threads a row where there are more rows than compute units, which then take two
    // each, one computing while the other waits (512 rows of 32768, top-p: 44 us, 52 with
    // 1024), or where a row is short (512 rows of 2048: 14.7 and 25 us; one of 8192: 11.1
    // and 11.7); 1024 otherwise (128 rows of 32768: 27.7 and 24.3 us)
    if (a.V < 8) {
        hipLaunchKernelGGL((smg_sample_t<512, 4096, F32, true>), dim3(a.R), dim3(512), 0, s, a);
    } else if (a.parts == 1 && (a.R > 256 || a.V <= 8192)) {
        hipLaunchKernelGGL((smg_sample_t<512, 4096, F32, false>), dim3(a.R), dim3(512), 0, s, a);
    } else if (a.parts == 1) {
        hipLaunchKernelGGL((smg_sample_t<1024, 8192, F32, false>), dim3(a.R), dim3(1024), 0, s, a);
    } else {
        const dim3 all(a.parts, a.R);
        hipLaunchKernelGGL(smg_sample_ends_t<F32>, all, dim3(1024), 0, s, a);
        hipLaunchKernelGGL(smg_sample_measure_t<F32>, all, dim3(1024), 0, s, a);
        hipLaunchKernelGGL(smg_sample_cut_t<F32>, dim3(a.R), dim3(1024), 0, s, a);
        if (a.top_k || a.top_p) {
            hipLaunchKernelGGL(smg_sample_sums_t<F32>, all, dim3(1024), 0, s, a);
            hipLaunchKernelGGL(smg_sample_pick_t<F32>, dim3(a.R), dim3(1024), 0, s, a);
        }
    }
}

}  // namespace

// bytes of workspace that a row takes where workgroups share it
extern "C" long long smg_sample_work_bytes() { return (long long)sizeof(Work); }

extern "C" int smg_sample_launch(const void* logits, const void* u, const void* temperature,
                                 const void* top_k, const void* top_p, const void* min_p, void* out,
                                 void* work, long long stride, int R, int V, int parts, int f32, void* stream) {
    if (V < 1 || V > MAX_V || parts < 1 || parts > MAX_PARTS || (parts > 1 && (!work || R > 65535))) return -1;
    if (R < 1) return 0;
    SampleArgs a = {logits, stride, (const float*)u, (const float*)temperature, (const int*)top_k,
                    (const float*)top_p, (const float*)min_p, (long long*)out, R, V, (u64*)work, parts};
    if (f32)
        launch<true>(a, (hipStream_t)stream);
    else
        launch<false>(a, (hipStream_t)stream);
    return hipGetLastError() == hipSuccess ? 0 : -2;
}
