// Attention of many new tokens over the engine's slot cache — gfx950 MFMA.
//
//   attn_prefill: packed prompts (or prompt chunks) of different lengths.
//     Token i of sequence b sees the cache rows 0 .. start[b]+i of its slot:
//     its history, the chunk's earlier tokens and itself (their K/V are in the
//     cache already).
//   attn_tree: N drafted tokens per sequence.  Node i sees the whole context
//     (cache rows 0 .. ctx[b]-1) and, of the drafted nodes, its ancestors and
//     itself; the drafts' K/V come in tensors of their own.
//
// Mathematics: out = softmax(scale * q K^T) V per (token, head), in one pass
// over K/V with a running maximum m and sum l (both f32):
//     m' = max(m, max_j s_j);  p_j = 2^((s_j - m') c),  c = scale * log2(e)
//     l = l 2^((m-m') c) + sum p_j;  O = O 2^((m-m') c) + sum p_j v_j
//
// Layout: the G = heads / kv heads query heads of a kv head are packed with
// the tokens into rows r = token * G + g, so K/V is read once per group.  Both
// products run transposed on v_mfma_f32_32x32x16_bf16: S^T = K Q^T leaves lane
// (h = lane/32, c = lane%32) with 16 scores of query row c, at key rows
// 8b + 4h + i (b, i < 4).  The sum over keys in O^T = V^T P^T may run in any
// order that both operands share, so these registers, rounded to bf16, ARE the
// second product's B operand, and V^T is read from LDS to match
// (ds_read_b64_tr_b16 gives a lane 4 consecutive key rows of one column).  P
// never leaves the registers, and m, l and the rescaling are per lane.  P is
// rounded to bf16 because the matrix cores take no wider second operand at
// this rate: at most 2^-8 relative a weight, while l sums the f32 values.
// 8-bit K/V become bf16, exactly, on their way through LDS: products in 8 bits
// would round Q and P to 4 bits.
//
// What bounds it, and what it measures on an MI355X (2.4 GHz, 1.37 PF/s in a
// large bf16 product, 4.6 TB/s in a large copy):
//   16384 tokens, 16 over 4 heads of 128: 1.10 ms, 1.00 PF/s.  Matrix cores
//     are busy 54% of the cycles and the vector unit, with exp and the
//     roundings, 56%; under both the clock falls to 1.9 GHz.
//   two chunks of 1900 tokens over 5900 8-bit rows, 16 heads: 270 us, 0.80 PF/s.
//     One workgroup of 8 waves a compute unit where 16 bits have two of 4, and
//     7% for the widening.
//   32 prompts of about 75 over 460 rows: 30 us; 104 of the units have two
//     workgroups and 152 one, and 19% of the rows computed are padding.
//   64 trees of 16 nodes over 250 to 2000 rows: 51 us, 3.2 TB/s of K/V, 38 where
//     the caches hold them.  Each unit has one workgroup and its whole sequence:
//     the longest take 17 tiles of keys, the mean one 10.6.
//   4 trees of 61 over 35000 8-bit rows: 106 us, of which joining takes 10.
//   one prompt of a token, or a tree of 5: 6.5 and 7.5 us, latency alone.
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>

#include <atomic>
#include <cstdint>
#include <type_traits>

#define WAVE 64
#define LOG2E 1.44269504088896340736f

namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;

struct AttnArgs {
    const __hip_bfloat16* q;     // prefill [N, H, D]; tree [B, N, H, D]
    __hip_bfloat16* out;         // as q
    const void* k;               // [S, KVH, T, D] bf16 or e4m3
    const void* v;
    const __hip_bfloat16* k_new;  // tree: [B, N, KVH, D]
    const __hip_bfloat16* v_new;
    const int* slots;            // [B]
    const int* ctx;              // [B] rows in the cache before the new tokens
    const int* cu;               // prefill: [B + 1] first packed row of each sequence
    const int* parents;          // tree: [B, N]
    float* part_o;               // n_split > 1: [units, KVH, part_rows, D], unnormalised
    float* part_ml;              // n_split > 1: [units, KVH, part_rows, 2]
    long long q_sb, q_st, q_sh, o_sb, o_st, o_sh;        // strides in elements
    long long k_ss, k_sh, k_st, v_ss, v_sh, v_st;
    long long kn_sb, kn_st, kn_sh, vn_sb, vn_st, vn_sh;
    int B, N, H, KVH, S, T;
    int n_split;                 // most runs that a row's keys are split into
    int share;                   // workgroups that the card takes at once, for each kv head
    int units;                   // of a kv head: tiles of rows, or with n_split > 1 their runs at most
    int part_rows;               // of a tile: BM, or all there are if fewer
    float scale;
};

__device__ __forceinline__ int context(const AttnArgs& a, int b, bool tree) {
    return min(max(a.ctx[b], tree ? 0 : -a.N), a.T);
}
// cache rows that the query rows up to `last_row` of a sequence see
__device__ __forceinline__ int keys_of(const AttnArgs& a, int ctx, int last_row, int G, bool tree) {
    return tree ? ctx : max(0, min(ctx + last_row / G + 1, a.T));
}

// Where a sequence's rows lie, its tiles of rows, and the key tiles of the last of them
// (0 tiles of rows for a padding entry whose keys are split: it is left to run 0).
struct Seq {
    int base, rows, row_tiles, key_tiles;
    __device__ __forceinline__ Seq(const AttnArgs& a, int b, int G, int BM, int BN, bool tree) {
        base = 0;
        int len = a.N;
        if (!tree) {
            base = min(max(a.cu[b], 0), a.N);
            len = min(max(a.cu[b + 1], base), a.N) - base;
        }
        rows = len * G;
        row_tiles = (rows + BM - 1) / BM;
        const int slot = a.slots[b];
        key_tiles = 0;
        if (slot >= 0 && slot < a.S && rows)
            key_tiles = (keys_of(a, context(a, b, tree), rows - 1, G, tree) + BN - 1) / BN + (tree ? (a.N + BN - 1) / BN : 0);
    }
};

// The keys of a tile of rows are split into runs of tiles, which workgroups take side by
// side.  A run is as long as the tiles of all rows over the workgroups that the card
// takes at once (less one for each tile of rows, whose last run is a part): then long
// sequences have many runs and short ones one, which writes its result itself.  Every
// wave of both kernels computes the same.  mine: a lane's (row tiles, key tiles) of its
// sequence among the first 64.
__device__ __forceinline__ int run_length(const AttnArgs& a, int BM, int BN, bool tree, int2* mine = nullptr) {
    if (a.n_split == 1) return 0x7fffffff;
    const int lane = threadIdx.x & 63, G = a.H / a.KVH;
    float tiles = 0.f, rows = 0.f;
    for (int b = lane; b < a.B; b += WAVE) {
        const Seq s(a, b, G, BM, BN, tree);
        if (mine && b == lane) *mine = make_int2(s.row_tiles, s.key_tiles);
        tiles += (float)s.row_tiles * (float)s.key_tiles;
        rows += (float)s.row_tiles;
    }
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) tiles += __shfl_xor(tiles, o, WAVE), rows += __shfl_xor(rows, o, WAVE);
    const int per = (int)ceilf(tiles / fmaxf(1.f, (float)a.share - rows));
    return __builtin_amdgcn_readfirstlane(max(per, 256 / BN));
}

// tiles of a run in a sequence whose last tile of rows has `most` key tiles
__device__ __forceinline__ int run_of(const AttnArgs& a, int most, int length) {
    return max(1, max(min(length, most), (most + a.n_split - 1) / a.n_split));
}
// and the runs that each of its tiles of rows has
__device__ __forceinline__ int runs_of(const AttnArgs& a, int most, int length) {
    const int per = run_of(a, most, length);
    return max(1, (most + per - 1) / per);
}

// max and sum over the two halves of a wave (lane and lane ^ 32)
__device__ __forceinline__ float max_halves(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ unsigned fp8x2_to_bf16x2(unsigned w, bool hi) {
    // e4m3 values are bf16 values: exact
    bf16x2 r = hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true)
                  : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false);
    return __builtin_bit_cast(unsigned, r);
}

// Values of V that are not finite: all, +inf, -inf, NaN.
enum Kind { BAD, PLUS, MINUS, NOT };
// two bf16 in a word: all ones in the halves that hold that kind
template <Kind K>
__device__ __forceinline__ unsigned halves_where(unsigned w) {
    const unsigned lo = w & 0xffffu, hi = w >> 16;
    auto is = [](unsigned x) {
        return K == BAD ? (x & 0x7f80u) == 0x7f80u : K == PLUS ? x == 0x7f80u : K == MINUS ? x == 0xff80u : (x & 0x7fffu) > 0x7f80u;
    };
    return (is(lo) ? 0xffffu : 0u) | (is(hi) ? 0xffff0000u : 0u);
}
// adds `value` to the accumulators whose row has a weight on a V of that kind
template <Kind K>
__device__ __forceinline__ f32x16 hits(u32x4 v, bf16x8 p) {
    u32x4 one;
#pragma unroll
    for (int i = 0; i < 4; ++i) one[i] = halves_where<K>(v[i]) & 0x3f803f80u;
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, one), p, (f32x16)0.f, 0, 0, 0);
}
template <Kind K>
__device__ __forceinline__ void add_where(f32x16& acc, u32x4 v, bf16x8 p, float value) {
    const f32x16 hit = hits<K>(v, p);
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (!(hit[i] == 0.f)) acc[i] += value;
}

// Tiles hold D bf16 a row in 16-byte chunks, permuted within the row so that
// neighbouring lanes read different banks: 8 lanes one chunk column of 8 key
// rows (K), and 4 rows of 32 bytes, a pair of chunks (V).  The counters still
// have 33% of the LDS cycles as conflicts (36% in 8 bits); which of the reads or
// DMA writes they come from has not been told apart.
template <int D>
__device__ __forceinline__ int k_chunk(int row, int c) {
    return row * (D / 8) + (c ^ (row & (D / 8 - 1)));
}
template <int D>
__device__ __forceinline__ int v_swap(int row) {
    return D == 128 ? (row & 7) << 1 : ((row >> 1) & 3) << 1;
}
template <int D>
__device__ __forceinline__ int v_chunk(int row, int c) {
    return row * (D / 8) + (c ^ v_swap<D>(row));
}

// 64 lanes' 16 bytes each straight to 1 KB of LDS at `to` (the same in all lanes)
__device__ __forceinline__ void to_lds(const void* from, u32x4* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                     (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// A wave's scores, weights and sums.  Addresses in LDS are kept a lane, so that a tile
// costs one addition each; all else is constant offsets.
template <int D, int KB, int BN>
struct Tile {
    static constexpr int HB = D / 32, ROW = D * 2;  // blocks of columns, bytes of a row
    typedef __attribute__((address_space(3))) const bf16x8* k_ptr;
    typedef __attribute__((address_space(3))) s16x4* v_ptr;
    f32x16 acc[HB];  // O^T, unnormalised
    float m, mc, l;  // the running maximum, m * c (0 where nothing is seen yet), the sum of this half
    unsigned k_at[D / 16], v_at[HB];

    // w0: this wave's first key of a tile
    __device__ __forceinline__ void init(int w0) {
        const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) k_at[j] = k_chunk<D>(w0 + col, 2 * j + half) * 16;
        // lane -> key rows r .. r+3 (and, 8 rows on, another 4) of column hb*32 + col
        const int r = w0 + half * 4 + ((lane & 15) >> 2);
#pragma unroll
        for (int hb = 0; hb < HB; ++hb)
            v_at[hb] = BN * ROW + v_chunk<D>(r, hb * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) * 16 + (lane & 1) * 8;
#pragma unroll
        for (int i = 0; i < HB; ++i) acc[i] = (f32x16)0.f;
        m = -INFINITY;
        mc = l = 0.f;
    }
    // this wave's 32 KB keys of the tile at `at`; where MASKED, bit i of `seen` is key i of those
    template <bool MASKED>
    __device__ __forceinline__ void take(unsigned at, const bf16x8* qf, float c, unsigned long long seen) {
        const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
        // K a block of 32 keys ahead of the products
        f32x16 s[KB];
        bf16x8 kf[D / 16];
#pragma unroll
        for (int j = 0; j < D / 16; ++j) kf[j] = *(k_ptr)(size_t)(k_at[j] + at);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            s[kb] = (f32x16)0.f;
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
                s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[j], qf[j], s[kb], 0, 0, 0);
                if (kb + 1 < KB) kf[j] = *(k_ptr)(size_t)(k_at[j] + at + (kb + 1) * 32 * ROW);
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if (MASKED && !((unsigned)(seen >> kb * 32) >> half * 4 & 1u << ((i >> 2) * 8 + (i & 3)))) s[kb][i] = -INFINITY;
                top = fmaxf(top, s[kb][i]);
            }
        top = max_halves(top);
        // the maximum follows only when a weight would pass 2^8: f32 and bf16 hold
        // that as exactly, and the accumulators are seldom rescaled
        if (__any((top - m) * c > 8.f)) {
            const float m2 = fmaxf(m, top);
            const float mc2 = m2 == -INFINITY ? 0.f : m2 * c;
            const float alpha = __builtin_amdgcn_exp2f(m * c - mc2);
            m = m2;
            mc = mc2;
            l *= alpha;
#pragma unroll
            for (int i = 0; i < HB; ++i) acc[i] *= alpha;
        }
        bf16x8 p[KB][2];
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float e = __builtin_amdgcn_exp2f(fmaf(s[kb][i], c, -mc));
                sum[i & 3] += e;
                p[kb][i >> 3][i & 7] = (__bf16)e;
            }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int hb = 0; hb < HB; ++hb) {
                    const unsigned v = v_at[hb] + at + (kb * 32 + j * 16) * ROW;
                    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((v_ptr)(size_t)v);
                    const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((v_ptr)(size_t)(v + 8 * ROW));
                    bf16x8 vf = __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
                    if (MASKED) {
                        // 0 * inf is NaN: a masked key's weight is 0, but its V must not
                        // reach the rows that do not see it.  Such values are left out
                        // here, and products of their own find the rows that they meet
                        // with a weight.
                        const u32x4 all = __builtin_bit_cast(u32x4, vf);
                        u32x4 fin;
#pragma unroll
                        for (int i = 0; i < 4; ++i) fin[i] = all[i] & ~halves_where<BAD>(all[i]);
                        vf = __builtin_bit_cast(bf16x8, fin);
                        const u32x4 cut = fin ^ all;
                        if (__any((cut[0] | cut[1] | cut[2] | cut[3]) != 0)) {
                            add_where<PLUS>(acc[hb], all, p[kb][j], INFINITY);
                            add_where<MINUS>(acc[hb], all, p[kb][j], -INFINITY);
                            add_where<NOT>(acc[hb], all, p[kb][j], NAN);
                        }
                    }
                    acc[hb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, p[kb][j], acc[hb], 0, 0, 0);
                }
    }
};

// TREE: drafted nodes with their own K/V after the context.  KV8: e4m3 cache.
// WR waves share the query rows of a tile (32 each), WK of them split its keys:
// 4 x 1 reads K/V least often, 2 x 2 makes twice the workgroups, 2 x 4 and 1 x 4 have
// twice the bytes on their way from a compute unit that has one workgroup.  A wave takes
// 64 keys of a tile, or 32 where waves split it: so 2 x 2 takes 64 KB of LDS and a compute
// unit two workgroups of it (24 prompts of 75 over 460 rows: 22 us, 34 with 64 keys and one
// workgroup; one prompt of 2048: 39 and 43), and 2 x 4, with 128 KB of tiles, fits at all.
template <bool TREE, bool KV8, int D, int WR, int WK_>
struct Shape {
    static constexpr int WK = WK_;
    static constexpr int WAVES = WR * WK;
    static constexpr int THREADS = WAVES * WAVE;
    static constexpr int KB = WK == 1 ? 2 : 1;     // blocks of 32 keys a wave takes of a tile
    static constexpr int BN = 32 * KB * WK;        // keys of a tile
    static constexpr int BM = 32 * WR;             // query rows of a workgroup
    static constexpr int TILE = 2 * BN * (D / 8);  // 16-byte chunks of a tile, K then V
    static constexpr int RAW = TILE / 2;           // the same in 8 bits
    static constexpr int RAWS = 3;
    static constexpr int CHUNKS = 2 * TILE + (KV8 ? RAWS * RAW + (TREE ? TILE : 0) : 0);
    static constexpr int SLOTS = KV8 || WK == 4 ? 256 : 512;  // workgroups that the card takes at once
    static constexpr int WAVES_A_SIMD = KV8 && WR == 2 ? 1 : WR == 1 ? 1 : 2;
};

template <bool TREE, bool KV8, int D, int WR, int WK>
__global__ void __launch_bounds__((Shape<TREE, KV8, D, WR, WK>::THREADS), (Shape<TREE, KV8, D, WR, WK>::WAVES_A_SIMD)) smg_attn_cache_t(AttnArgs a) {
    using Z = Shape<TREE, KV8, D, WR, WK>;
    constexpr int KB = Z::KB, BN = Z::BN, BM = Z::BM, WAVES = Z::WAVES, THREADS = Z::THREADS;
    constexpr int CPR = D / 8;               // 16-byte chunks a row
    constexpr int HB = D / 32;
    extern __shared__ u32x4 smem[];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave % WR, wk = wave / WR;
    const int half = lane >> 5, col = lane & 31;
    const int G = a.H / a.KVH;
    const int kvh = blockIdx.x % a.KVH;

    // Which sequence, rows and run: sequence b has ceil(rows / BM) tiles of rows, with
    // as many runs each as its last one has.
    const int length = run_length(a, BM, BN, TREE);
    int b = -1, row0 = 0, rows = a.N * G, base = 0, split = 0;
    if (TREE && a.n_split == 1) {
        const int per = (rows + BM - 1) / BM, tile = blockIdx.x / a.KVH;
        b = tile / per;
        row0 = tile % per * BM;
    } else {
        // the last ones first: they see the most keys
        const int unit = gridDim.x / a.KVH - 1 - blockIdx.x / a.KVH;
        int before = 0;
        for (int b0 = 0; b0 < a.B; b0 += WAVE) {
            int n = 0, runs = 1, first = 0, all = 0;
            if (b0 + lane < a.B) {
                const Seq s(a, b0 + lane, G, BM, BN, TREE);
                first = s.base, all = s.rows;
                runs = runs_of(a, s.key_tiles, length);
                n = s.row_tiles * runs;
            }
            int sum = n;
#pragma unroll
            for (int o = 1; o < WAVE; o <<= 1) {
                const int up = __shfl_up(sum, o, WAVE);
                if (lane >= o) sum += up;
            }
            const unsigned long long found = __ballot(before + sum > unit);
            if (found) {
                const int l = __ffsll((long long)found) - 1;
                b = b0 + l;
                base = __builtin_amdgcn_readlane(first, l);
                rows = __builtin_amdgcn_readlane(all, l);
                const int i = unit - before - __builtin_amdgcn_readlane(sum - n, l);
                runs = __builtin_amdgcn_readlane(runs, l);
                row0 = i / runs * BM;
                split = i % runs;
                break;
            }
            before += __builtin_amdgcn_readlane(sum, WAVE - 1);
        }
        if (b < 0) return;
    }
    const int slot = a.slots[b];
    const bool cached = slot >= 0 && slot < a.S;
    const int ctx = context(a, b, TREE);

    // keys of the workgroup, in tiles; a split takes a run of them
    const int last_row = min(row0 + BM, rows) - 1;
    const int kend = cached ? keys_of(a, ctx, last_row, G, TREE) : 0;
    const int ctx_tiles = (kend + BN - 1) / BN;
    const int new_tiles = TREE ? (a.N + BN - 1) / BN : 0;
    const int tiles = cached ? ctx_tiles + new_tiles : 0;
    const int most = cached ? (keys_of(a, ctx, rows - 1, G, TREE) + BN - 1) / BN + new_tiles : 0;
    const int per = run_of(a, most, length);
    const int runs = (tiles + per - 1) / per;
    if (split > 0 && split >= runs) return;
    const int t0 = split * per, t1 = min(tiles, t0 + per);

    // this lane's query row, and the last cache row that it sees
    const int row = row0 + wr * 32 + col;
    const bool live = row < rows;
    const int token = min(row, rows - 1) / G;
    const int head = kvh * G + min(row, rows - 1) % G;
    const __hip_bfloat16* qp = a.q + (TREE ? b * a.q_sb : 0) + (base + token) * a.q_st + head * a.q_sh;
    bf16x8 qf[D / 16];
#pragma unroll
    for (int j = 0; j < D / 16; ++j) qf[j] = *(const bf16x8*)(qp + j * 16 + half * 8);

    int limit;                        // cache rows <= limit
    unsigned long long nodes = 0;     // drafted nodes that this row sees
    if constexpr (TREE) {
        // A lane a node: ancestors by doubling.  A parent comes before its child;
        // anything else below -1 or not before it marks a node outside the tree,
        // which -2 hands down.
        unsigned long long m = 1ull << lane;
        int up = lane < a.N ? a.parents[(size_t)b * a.N + lane] : -2;
        if (up >= lane || up < -1) up = -2;
#pragma unroll
        for (int i = 0; i < 6; ++i) {
            const int from = max(up, 0);
            const unsigned long long m2 = __shfl(m, from, WAVE);
            const int up2 = __shfl(up, from, WAVE);
            if (up >= 0) m |= m2, up = up2;
        }
        nodes = __shfl(up == -1 ? m : 0ull, token, WAVE);
        if (!live || !cached) nodes = 0;
        limit = nodes ? ctx - 1 : -1;
    } else {
        limit = live && cached ? min(ctx + token, a.T - 1) : -1;
    }

    const size_t unit = KV8 ? 1 : 2;
    const char* kbase = (const char*)a.k + (cached ? slot * a.k_ss + kvh * a.k_sh : 0) * unit;
    const char* vbase = (const char*)a.v + (cached ? slot * a.v_ss + kvh * a.v_sh : 0) * unit;
    const __hip_bfloat16* knew = TREE ? a.k_new + b * a.kn_sb + kvh * a.kn_sh : nullptr;
    const __hip_bfloat16* vnew = TREE ? a.v_new + b * a.vn_sb + kvh * a.vn_sh : nullptr;
    const float c = a.scale * LOG2E;
    // Tiles whose every key every row sees (nodes outside the tree get their zeros at
    // the end) need no mask.  They come first, and in a loop of their own: one loop
    // that chooses would move the accumulators about.
    const int full = min(t1, (TREE ? kend : max(0, min(ctx + row0 / G + 1, kend))) / BN);

    const int w0 = wk * KB * 32;  // this wave's keys of a tile
    Tile<D, KB, BN> tile_of;
    tile_of.init(w0);
    const unsigned lds = (unsigned)(size_t)(__attribute__((address_space(3))) void*)smem;
    // tile t from LDS: of the cache, or of the drafted nodes after it
    auto take = [&](int t, int chunk, auto masked) {
        const unsigned now = lds + chunk * 16;
        if constexpr (decltype(masked)::value) {
            const bool fresh = TREE && t >= ctx_tiles;
            const int k0 = (fresh ? (t - ctx_tiles) * BN : t * BN) + w0, n = limit - k0 + 1;
            const unsigned long long seen = fresh ? (k0 < 64 ? nodes >> k0 : 0) : n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1;
            tile_of.template take<true>(now, qf, c, seen);
        } else {
            tile_of.template take<false>(now, qf, c, 0);
        }
    };
    const std::true_type masked;
    const std::false_type whole;
    // 16-bit rows n0 .. n0 + BN - 1 to LDS, permuted by where each lane reads; rows
    // past the end repeat the last.  A whole tile takes a lane's fixed offsets from
    // addresses that the wave shares (the permutation repeats every 16 rows).
    auto rows_to_lds = [&](const __hip_bfloat16* kp, const __hip_bfloat16* vp, long long ks, long long vs, int n0, int nlast, u32x4* to) {
        constexpr int RPI = WAVE / CPR, STEP = RPI * WAVES;  // rows of a wave's 1 KB, of all waves' ones
        static_assert(STEP % (D == 128 ? 16 : 8) == 0, "the permutation repeats");
        const int r0 = wave * RPI + lane / CPR, cc = lane % CPR;
        const int kc = (cc ^ (r0 & (CPR - 1))) * 8, vc = (cc ^ v_swap<D>(r0)) * 8;
        if (n0 + BN - 1 <= nlast && max(ks, vs) < (1 << 20) && min(ks, vs) >= 0) {
            const unsigned ko = (unsigned)(r0 * (int)ks + kc) * 2, vo = (unsigned)(r0 * (int)vs + vc) * 2;
#pragma unroll
            for (int i = 0; i < BN / STEP; ++i) {
                to_lds((const char*)(kp + (n0 + i * STEP) * ks) + ko, to + (i * STEP + wave * RPI) * CPR);
                to_lds((const char*)(vp + (n0 + i * STEP) * vs) + vo, to + (BN + i * STEP + wave * RPI) * CPR);
            }
        } else {
#pragma unroll
            for (int i = 0; i < BN / STEP; ++i) {
                const long long src = min(n0 + i * STEP + r0, nlast);
                to_lds(kp + src * ks + kc, to + (i * STEP + wave * RPI) * CPR);
                to_lds(vp + src * vs + vc, to + (BN + i * STEP + wave * RPI) * CPR);
            }
        }
    };
    if constexpr (!KV8) {
        // two tiles in turn: one on its way while the other is computed
        auto get = [&](int t, u32x4* to) {
            if (TREE && t >= ctx_tiles)
                rows_to_lds(knew, vnew, a.kn_st, a.vn_st, (t - ctx_tiles) * BN, a.N - 1, to);
            else
                rows_to_lds((const __hip_bfloat16*)kbase, (const __hip_bfloat16*)vbase, a.k_st, a.v_st, t * BN, kend - 1, to);
        };
        auto step = [&](int t, auto mask) {
            // tile t is there, and nobody reads the one before it any more
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (t + 1 < t1) get(t + 1, smem + ((t - t0 + 1) & 1) * Z::TILE);
            take(t, ((t - t0) & 1) * Z::TILE, mask);
        };
        if (t0 < t1) get(t0, smem);
        int t = t0;
        for (; t < full; ++t) step(t, whole);
        for (; t < t1; ++t) step(t, masked);
    } else {
        // 8-bit tiles come as they are, up to three on their way (memory is what the
        // long ones wait for), and the workgroup widens one while it computes the one
        // before it.  The drafted nodes' tile has a place of its own.
        constexpr int UPR = D / 16;                     // 16-byte units a row
        constexpr int PER = 2 * BN * UPR / THREADS;     // units a thread, of K then V
        u32x4* raws = smem + 2 * Z::TILE;
        u32x4* drafts = raws + Z::RAWS * Z::RAW;
        const int tc = min(t1, ctx_tiles);              // the cache's tiles end here
        auto get = [&](int t) {
            u32x4* to = raws + t % Z::RAWS * Z::RAW;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int u0 = (i * WAVES + wave) * WAVE;
                const bool v = u0 >= BN * UPR;
                const int r0 = (u0 - (v ? BN * UPR : 0)) / UPR;  // the wave's first row of 64 / UPR
                const char* from = v ? vbase : kbase;
                const long long st = v ? a.v_st : a.k_st;
                if (t * BN + BN <= kend && st < (1 << 20) && st >= 0)
                    to_lds(from + (t * BN + r0) * st + (unsigned)(lane / UPR * (int)st + lane % UPR * 16), to + u0);
                else
                    to_lds(from + (long long)min(t * BN + r0 + lane / UPR, kend - 1) * st + lane % UPR * 16, to + u0);
            }
        };
        auto widen = [&](int t) {
            const u32x4* from = raws + t % Z::RAWS * Z::RAW;
            u32x4* to = smem + (t & 1) * Z::TILE;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int u = i * THREADS + tid, r = u / UPR % BN, cc = u % UPR * 2;
                const bool v = u >= BN * UPR;
                const u32x4 x = from[u];
                const u32x4 lo = {fp8x2_to_bf16x2(x[0], false), fp8x2_to_bf16x2(x[0], true), fp8x2_to_bf16x2(x[1], false), fp8x2_to_bf16x2(x[1], true)};
                const u32x4 hi = {fp8x2_to_bf16x2(x[2], false), fp8x2_to_bf16x2(x[2], true), fp8x2_to_bf16x2(x[3], false), fp8x2_to_bf16x2(x[3], true)};
                to[v ? BN * CPR + v_chunk<D>(r, cc) : k_chunk<D>(r, cc)] = lo;
                to[v ? BN * CPR + v_chunk<D>(r, cc + 1) : k_chunk<D>(r, cc + 1)] = hi;
            }
        };
        static_assert(BN == 64, "one tile of drafted nodes");
        if (TREE && t1 > ctx_tiles) rows_to_lds(knew, vnew, a.kn_st, a.vn_st, 0, a.N - 1, drafts);
#pragma unroll
        for (int i = 0; i < Z::RAWS; ++i)
            if (t0 + i < tc) get(t0 + i);
        if (t0 < tc) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            widen(t0);
        }
        auto step = [&](int t, auto mask) {
            // this wave's part of raw tile t + 1 is there (t + 2 may be on its way) and
            // its part of tile t is widened: after the barrier, all are
            if (t + 2 < tc)
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(PER) : "memory");
            else
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (t + Z::RAWS < tc) get(t + Z::RAWS);  // where raw tile t was
            if (t + 1 < tc) widen(t + 1);            // where tile t - 1 was
            take(t, (t & 1) * Z::TILE, mask);
        };
        int t = t0;
        for (; t < full; ++t) step(t, whole);
        for (; t < tc; ++t) step(t, masked);
        if (TREE && t1 > ctx_tiles) {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            take(ctx_tiles, (int)(drafts - smem), masked);
        }
    }
    auto& acc = tile_of.acc;
    float m = tile_of.m, l = tile_of.l;
    l = sum_halves(l);
    if (TREE && !nodes) {
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int i = 0; i < HB; ++i) acc[i] = (f32x16)0.f;
    }

    // join the waves that took different keys: each finishes HB / WK of the columns
    constexpr int HW = HB / WK;  // WK <= HB
    if constexpr (WK > 1) {
        float* so = (float*)smem;                     // [WAVES][HB * 16][64]
        float* sm = so + WAVES * HB * 16 * WAVE;      // [WAVES][2][64]
        __syncthreads();
#pragma unroll
        for (int hb = 0; hb < HB; ++hb)
#pragma unroll
            for (int i = 0; i < 16; ++i) so[((wave * HB + hb) * 16 + i) * WAVE + lane] = acc[hb][i];
        sm[(wave * 2) * WAVE + lane] = m;
        sm[(wave * 2 + 1) * WAVE + lane] = l;
        __syncthreads();
        float f[WK], all = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < WK; ++w) all = fmaxf(all, sm[(wr + w * WR) * 2 * WAVE + lane]);
#pragma unroll
        for (int w = 0; w < WK; ++w) {
            const float mw = sm[(wr + w * WR) * 2 * WAVE + lane];
            f[w] = mw == -INFINITY ? 0.f : exp2f((mw - all) * c);
            sum += f[w] * sm[((wr + w * WR) * 2 + 1) * WAVE + lane];
        }
        m = all;
        l = sum;
#pragma unroll
        for (int hb = 0; hb < HW; ++hb)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float o = 0.f;
#pragma unroll
                for (int w = 0; w < WK; ++w)
                    o += f[w] * so[(((wr + w * WR) * HB + wk * HW + hb) * 16 + i) * WAVE + lane];
                acc[hb][i] = o;
            }
    }
    if (!live) return;
    const int hb0 = WK > 1 ? wk * HW : 0;
    if (runs > 1) {
        // by workgroup: the runs that there are at most are far more than those that
        // the card takes
        const int unit = gridDim.x / a.KVH - 1 - blockIdx.x / a.KVH;
        const size_t at = ((size_t)unit * a.KVH + kvh) * a.part_rows + wr * 32 + col;
#pragma unroll
        for (int hb = 0; hb < HW; ++hb)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *(f32x4*)(a.part_o + at * D + (hb0 + hb) * 32 + j * 8 + half * 4) =
                    (f32x4){acc[hb][j * 4], acc[hb][j * 4 + 1], acc[hb][j * 4 + 2], acc[hb][j * 4 + 3]};
        if (wk == 0 && half == 0) {
            a.part_ml[at * 2] = m;
            a.part_ml[at * 2 + 1] = l;
        }
        return;
    }
    // no key seen: zeros; NaN stays
    const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
    __hip_bfloat16* op = a.out + (TREE ? b * a.o_sb : 0) + (base + token) * a.o_st + head * a.o_sh;
#pragma unroll
    for (int hb = 0; hb < HW; ++hb)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            bf16x4 o;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = (__bf16)(acc[hb][j * 4 + i] * inv);
            *(bf16x4*)(op + (hb0 + hb) * 32 + j * 8 + half * 4) = o;
        }
}

// Joins the runs of a row that has several:
//   out = sum_s 2^((m_s - m) c) O_s / sum_s 2^((m_s - m) c) l_s.
// A wave has a (token, head); a load covers 256 / D runs, and up to 16 are on their way.
template <bool TREE, int D>
__global__ void __launch_bounds__(256) smg_attn_join_t(AttnArgs a, int BM, int BN) {
    const int lane = threadIdx.x & 63;
    const long long all_rows = TREE ? a.B * (long long)a.N : a.N;
    const long long rh = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (rh >= all_rows * a.H) return;
    const long long r = rh / a.H;
    const int h = (int)(rh % a.H), G = a.H / a.KVH;
    int b;
    if constexpr (TREE) {
        b = (int)(r / a.N);
    } else {
        // the last sequence that starts at r or before; rows outside all stay
        if (r < a.cu[0] || r >= a.cu[a.B]) return;
        int lo = 0, hi = a.B;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (a.cu[mid] <= r)
                lo = mid;
            else
                hi = mid;
        }
        b = lo;
    }
    const Seq seq(a, b, G, BM, BN, TREE);
    const int token = TREE ? (int)(r % a.N) : (int)r - seq.base;
    const int row = token * G + h % G, tile = row / BM;
    if (!seq.key_tiles || row >= seq.rows) return;
    const int last_row = min(tile * BM + BM, seq.rows) - 1;
    const int kend = keys_of(a, context(a, b, TREE), last_row, G, TREE);
    int2 mine = make_int2(0, 0);
    const int length = run_length(a, BM, BN, TREE, &mine);
    const int per = run_of(a, seq.key_tiles, length);
    const int n = ((kend + BN - 1) / BN + (TREE ? (a.N + BN - 1) / BN : 0) + per - 1) / per;
    if (n <= 1) return;
    // the workgroups before this tile's, as the other kernel counts them
    int before = lane < b ? mine.x * runs_of(a, mine.y, length) : 0;
    for (int i = lane + WAVE; i < b; i += WAVE) {
        const Seq s(a, i, G, BM, BN, TREE);
        before += s.row_tiles * runs_of(a, s.key_tiles, length);
    }
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) before += __shfl_xor(before, o, WAVE);
    const int first = before + tile * runs_of(a, seq.key_tiles, length);
    if (first < 0 || first > a.units - n) return;  // offsets that do not rise
    // a lane a run (at most 64 of them)
    const float c = a.scale * LOG2E;
    const size_t run = (size_t)a.KVH * a.part_rows, at = (size_t)first * run + (size_t)(h / G) * a.part_rows + row % BM;
    float ms = -INFINITY, ls = 0.f;
    if (lane < n) ms = a.part_ml[(lane * run + at) * 2], ls = a.part_ml[(lane * run + at) * 2 + 1];
    float top = ms;
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, WAVE));
    const float fs = ms == -INFINITY ? 0.f : exp2f((ms - top) * c);
    float sum = fs * ls;
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) sum += __shfl_xor(sum, o, WAVE);
    constexpr int LPR = D / 4, RPL = WAVE / LPR;  // lanes of a row, rows of a load
    const int e = lane % LPR * 4;
    f32x4 o = 0.f;
    for (int s0 = 0; s0 < n; s0 += 16 * RPL) {
        f32x4 part[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int s = s0 + i * RPL + lane / LPR;
            part[i] = s < n ? *(const f32x4*)(a.part_o + (s * run + at) * D + e) : (f32x4)0.f;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) o += __shfl(fs, s0 + i * RPL + lane / LPR, WAVE) * part[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int step = LPR; step < WAVE; step <<= 1) o[i] += __shfl_xor(o[i], step, WAVE);
    if (lane >= LPR) return;
    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
    __hip_bfloat16* op = (TREE ? a.out + b * a.o_sb + token * a.o_st : a.out + r * a.o_st) + h * a.o_sh + e;
    bf16x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (__bf16)(o[i] * inv);
    *(bf16x4*)op = w;
}

// `floats`, if given, gets the size of the workspace instead of a launch
template <bool TREE, bool KV8, int D, int WR, int WK>
int launch_t(AttnArgs a, hipStream_t s, long long* floats) {
    using Z = Shape<TREE, KV8, D, WR, WK>;
    constexpr int BM = Z::BM, BN = Z::BN;
    constexpr int tile_bytes = Z::CHUNKS * 16;
    constexpr int join_bytes = WK > 1 ? Z::WAVES * (D / 32 * 16 + 2) * WAVE * 4 : 0;
    constexpr int bytes = tile_bytes > join_bytes ? tile_bytes : join_bytes;
    static_assert(bytes <= 160 * 1024, "LDS of a compute unit");
    const long long G = a.H / a.KVH;
    const long long tiles = TREE ? a.B * ((a.N * G + BM - 1) / BM) : a.N * G / BM + a.B;
    // with runs: never more than `share` of them, but at least one for each tile of rows
    const long long share = Z::SLOTS / a.KVH > tiles ? Z::SLOTS / a.KVH : tiles;
    const long long units = share < tiles * a.n_split ? share : tiles * a.n_split;
    const long long grid = units * a.KVH;
    if (grid > 0x7fffffffll || share > 0x7fffffffll || a.n_split > WAVE) return -5;
    a.part_rows = (int)(a.N * G < BM ? a.N * G : BM);
    if (floats) {
        *floats = a.n_split > 1 ? grid * a.part_rows * (D + 2) : 0;
        return 0;
    }
    if (a.n_split > 1 && !a.part_o) return -3;
    a.share = (int)share;
    a.units = (int)units;
    a.part_ml = a.part_o + grid * a.part_rows * D;
    // more dynamic LDS than the default limit, once a device
    static std::atomic<unsigned long long> set{0};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return -2;
    if (dev > 63 || !(set.load(std::memory_order_relaxed) >> dev & 1)) {
        if (hipFuncSetAttribute((const void*)smg_attn_cache_t<TREE, KV8, D, WR, WK>,
                                hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
            return -2;
        if (dev <= 63) set.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    hipLaunchKernelGGL((smg_attn_cache_t<TREE, KV8, D, WR, WK>), dim3((unsigned)grid), dim3(Z::THREADS), bytes, s, a);
    if (a.n_split > 1) {
        const long long rh = (TREE ? a.B * (long long)a.N : a.N) * a.H;
        if (rh > 0x7fffffffll) return -5;
        hipLaunchKernelGGL((smg_attn_join_t<TREE, D>), dim3((unsigned)((rh + 3) / 4)), dim3(256), 0, s, a, BM, BN);
    }
    return hipGetLastError() == hipSuccess ? 0 : -2;
}

template <bool TREE, bool KV8, int D>
int launch_d(const AttnArgs& a, int wr, int wk, hipStream_t s, long long* floats) {
    if constexpr (KV8) {
        if (wr <= 2) return launch_t<TREE, true, D, 2, 2>(a, s, floats);
        if (wr == 4) return launch_t<TREE, true, D, 4, 2>(a, s, floats);
        return launch_t<TREE, true, D, 8, 1>(a, s, floats);
    } else {
        if constexpr (D == 128) {
            if (wr == 1) return launch_t<TREE, false, D, 1, 4>(a, s, floats);
            if (wr == 2 && wk == 4) return launch_t<TREE, false, D, 2, 4>(a, s, floats);
        }
        if (wr <= 2) return launch_t<TREE, false, D, 2, 2>(a, s, floats);
        return launch_t<TREE, false, D, 4, 1>(a, s, floats);
    }
}

template <bool TREE, bool KV8>
int launch(const AttnArgs& a, int D, int wr, int wk, hipStream_t s, long long* floats) {
    return D == 128 ? launch_d<TREE, KV8, 128>(a, wr, wk, s, floats) : D == 64 ? launch_d<TREE, KV8, 64>(a, wr, wk, s, floats) : -1;
}

int bad_shape(long long rows, int H, int KVH, int S, int T, int n_split) {
    if (KVH <= 0 || H <= 0 || H % KVH) return -4;
    if (rows * H > 1 << 30 || T > 1 << 30) return -5;  // row and key numbers are 32 bits
    if (S <= 0 || T <= 0 || n_split < 1) return -3;
    return 0;
}

}  // namespace

// floats of workspace that a call with n_split > 1 takes, or an error below 0
extern "C" long long smg_attn_part_floats(int tree, int B, int N, int H, int KVH, int D, int n_split, int wr, int wk, int kv_fp8) {
    if (int rc = bad_shape(tree ? (long long)B * N : N, H, KVH, 1, 1, n_split)) return rc;
    AttnArgs a = {};
    a.B = B, a.N = N, a.H = H, a.KVH = KVH, a.n_split = n_split;
    long long floats = 0;
    const int rc = tree ? kv_fp8 ? launch<true, true>(a, D, wr, wk, nullptr, &floats) : launch<true, false>(a, D, wr, wk, nullptr, &floats)
                        : kv_fp8 ? launch<false, true>(a, D, wr, wk, nullptr, &floats) : launch<false, false>(a, D, wr, wk, nullptr, &floats);
    return rc ? rc : floats;
}

// strides: q token/head, out token/head, k slot/head/row, v slot/head/row
extern "C" int smg_attn_prefill_launch(
    const void* q, const void* k, const void* v, const void* slots, const void* ctx, const void* cu,
    void* out, void* part, const long long* strides, int B, int N, int H, int KVH,
    int S, int T, int D, int n_split, int wr, int wk, float scale, int kv_fp8, void* stream) {
    if (int rc = bad_shape(N, H, KVH, S, T, n_split)) return rc;
    if (B < 1 || N < 1) return 0;
    AttnArgs a = {};
    a.q = (const __hip_bfloat16*)q;
    a.out = (__hip_bfloat16*)out;
    a.k = k;
    a.v = v;
    a.slots = (const int*)slots;
    a.ctx = (const int*)ctx;
    a.cu = (const int*)cu;
    a.part_o = (float*)part;
    a.q_st = strides[0], a.q_sh = strides[1], a.o_st = strides[2], a.o_sh = strides[3];
    a.k_ss = strides[4], a.k_sh = strides[5], a.k_st = strides[6];
    a.v_ss = strides[7], a.v_sh = strides[8], a.v_st = strides[9];
    a.B = B, a.N = N, a.H = H, a.KVH = KVH, a.S = S, a.T = T, a.n_split = n_split;
    a.scale = scale;
    return kv_fp8 ? launch<false, true>(a, D, wr, wk, (hipStream_t)stream, nullptr)
                  : launch<false, false>(a, D, wr, wk, (hipStream_t)stream, nullptr);
}

// strides: q batch/token/head, out batch/token/head, k and v as above, k_new and v_new batch/token/head
extern "C" int smg_attn_tree_launch(
    const void* q, const void* k_new, const void* v_new, const void* k, const void* v,
    const void* slots, const void* ctx, const void* parents, void* out, void* part,
    const long long* strides, int B, int N, int H, int KVH, int S, int T, int D, int n_split, int wr, int wk,
    float scale, int kv_fp8, void* stream) {
    if (int rc = bad_shape((long long)B * N, H, KVH, S, T, n_split)) return rc;
    if (N > 64) return -3;
    if (B < 1 || N < 1) return 0;
    AttnArgs a = {};
    a.q = (const __hip_bfloat16*)q;
    a.out = (__hip_bfloat16*)out;
    a.k = k;
    a.v = v;
    a.k_new = (const __hip_bfloat16*)k_new;
    a.v_new = (const __hip_bfloat16*)v_new;
    a.slots = (const int*)slots;
    a.ctx = (const int*)ctx;
    a.parents = (const int*)parents;
    a.part_o = (float*)part;
    a.q_sb = strides[0], a.q_st = strides[1], a.q_sh = strides[2];
    a.o_sb = strides[3], a.o_st = strides[4], a.o_sh = strides[5];
    a.k_ss = strides[6], a.k_sh = strides[7], a.k_st = strides[8];
    a.v_ss = strides[9], a.v_sh = strides[10], a.v_st = strides[11];
    a.kn_sb = strides[12], a.kn_st = strides[13], a.kn_sh = strides[14];
    a.vn_sb = strides[15], a.vn_st = strides[16], a.vn_sh = strides[17];
    a.B = B, a.N = N, a.H = H, a.KVH = KVH, a.S = S, a.T = T, a.n_split = n_split;
    a.scale = scale;
    return kv_fp8 ? launch<true, true>(a, D, wr, wk, (hipStream_t)stream, nullptr)
                  : launch<true, false>(a, D, wr, wk, (hipStream_t)stream, nullptr);
}
