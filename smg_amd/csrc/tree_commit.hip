// Accepting drafted tokens and committing their K/V to the slot cache — gfx950.
//
// Per sequence, over a tree of N <= 64 drafted nodes: node 0 (the token that the
// last step sampled) is always taken; from the node taken last, the walk goes
// on to its first child whose token is the one that the model sampled at that
// node (target), until there is none.  The K/V rows of the path, which lie in
// [layers, 2, B, N, KVH, D], go to rows ctx .. ctx+len-1 of the sequence's slot,
// in all layers, rounded to e4m3 where the cache holds that (to nearest even;
// beyond 464, NaN).
//
// A wave holds the tree, a node a lane, and finds a child with one ballot; each
// workgroup walks for itself and then moves its share of the planes (layer,
// K or V, kv head).  The work is latency: three dependent loads and the walk.
// One sequence of 5 nodes in 2 layers takes 2.6 us on an MI355X, about what any
// launch takes; 64 of 32 nodes in 16 layers 5.9 us for 6.3 MB that a copy would
// move in 1.4.  Walking once and copying in a second launch would cost that launch.
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>

#include <cstdint>

#define WAVE 64

namespace {

struct CommitArgs {
    const __hip_bfloat16* src;  // [L, 2, B, N, KVH, D]
    void* dst;                  // [L, 2, S, KVH, T, D] bf16 or e4m3
    const int* slots;           // [B]
    const int* ctx;             // [B]
    const int* parents;         // [B, N]
    const long long* tokens;    // [B, N]
    const long long* targets;   // [B, N]
    int* count;                 // [B]
    int* path;                  // [B, N]
    long long* next;            // [B]
    long long s_l, s_w, s_b, s_n, s_h;  // strides in elements
    long long d_l, d_w, d_s, d_h, d_t;
    int B, N, L, KVH, S, T, D;
};

__device__ __forceinline__ unsigned bf16x4_to_fp8(unsigned lo, unsigned hi) {
    unsigned r = __builtin_amdgcn_cvt_pk_fp8_f32(__uint_as_float(lo << 16), __uint_as_float(lo & 0xffff0000u), 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(__uint_as_float(hi << 16), __uint_as_float(hi & 0xffff0000u), r, true);
}

template <bool KV8>
__global__ void __launch_bounds__(256) smg_tree_commit_t(CommitArgs a) {
    const int b = blockIdx.x, lane = threadIdx.x & 63;
    const int slot = a.slots[b], ctx = a.ctx[b];
    const bool node = lane < a.N;
    const size_t at = (size_t)b * a.N + lane;
    const int parent = node ? a.parents[at] : -2;
    const long long token = node ? a.tokens[at] : 0;
    const long long target = node ? a.targets[at] : 0;

    // a slot outside the cache, no room, or a node 0 that is not a root: a padding entry
    const int room = slot >= 0 && slot < a.S && ctx >= 0 ? a.T - ctx : 0;
    int len = 0, cur = 0, mine = -1;  // lane j: the j-th node of the path
    if (room > 0 && __shfl(parent, 0, WAVE) == -1) {
        len = 1;
        if (lane == 0) mine = 0;
        while (len < room) {
            const long long want = __shfl(target, cur, WAVE);
            const unsigned long long fit = __ballot(lane > cur && parent == cur && token == want);
            if (!fit) break;
            cur = __ffsll((long long)fit) - 1;
            if (lane == len) mine = cur;
            ++len;
        }
    }
    if (blockIdx.y == 0 && threadIdx.x < WAVE) {
        if (node) a.path[at] = mine;
        if (lane == 0) a.count[b] = len;
        if (lane == cur) a.next[b] = len ? target : -1;
    }
    if (!len) return;
    // of entries that name one slot the last that is no padding writes it
    bool later = false;
    for (int i = b + 1 + lane; i < a.B; i += WAVE)
        if (a.slots[i] == slot) later |= a.ctx[i] >= 0 && a.ctx[i] < a.T && a.parents[(size_t)i * a.N] == -1;
    if (__any(later)) return;

    const int chunks = a.D / 8;
    const int planes = a.L * 2 * a.KVH;
    const int per = (planes + gridDim.y - 1) / gridDim.y;
    const int p0 = blockIdx.y * per, p1 = min(planes, p0 + per);
    const int items = (p1 - p0) * len * chunks;
    for (int i0 = 0; i0 < items; i0 += blockDim.x) {
        const int i = i0 + threadIdx.x;
        const int j = i / chunks % len;
        const int n = __shfl(mine, j, WAVE);  // by all lanes, also those past the end
        if (i >= items) continue;
        const int c = i % chunks, plane = p0 + i / (chunks * len);
        const int h = plane % a.KVH, w = plane / a.KVH % 2, l = plane / a.KVH / 2;
        const uint4 x = *(const uint4*)(a.src + l * a.s_l + w * a.s_w + b * a.s_b + n * a.s_n + h * a.s_h + c * 8);
        const long long d = l * a.d_l + w * a.d_w + slot * a.d_s + h * a.d_h + (ctx + j) * a.d_t + c * 8;
        if constexpr (KV8)
            *(uint2*)((unsigned char*)a.dst + d) = make_uint2(bf16x4_to_fp8(x.x, x.y), bf16x4_to_fp8(x.z, x.w));
        else
            *(uint4*)((__hip_bfloat16*)a.dst + d) = x;
    }
}

}  // namespace

// strides: src layer/which/batch/node/head, dst layer/which/slot/head/row
extern "C" int smg_tree_commit_launch(const void* src, void* dst, const void* slots, const void* ctx,
                                      const void* parents, const void* tokens, const void* targets,
                                      void* count, void* path, void* next, const long long* strides,
                                      int B, int N, int L, int KVH, int S, int T, int D, int kv_fp8,
                                      void* stream) {
    if (N > 64 || D % 8 || L < 1 || KVH < 1 || S < 1 || T < 1 || D < 8) return -1;
    if (B < 1 || N < 1) return 0;
    CommitArgs a = {(const __hip_bfloat16*)src, dst, (const int*)slots, (const int*)ctx, (const int*)parents,
                    (const long long*)tokens, (const long long*)targets, (int*)count, (int*)path,
                    (long long*)next,
                    strides[0], strides[1], strides[2], strides[3], strides[4],
                    strides[5], strides[6], strides[7], strides[8], strides[9],
                    B, N, L, KVH, S, T, D};
    const int planes = L * 2 * KVH;
    const dim3 grid(B, (planes + 7) / 8 > 65535 ? 65535 : (planes + 7) / 8);
    if (kv_fp8)
        hipLaunchKernelGGL(smg_tree_commit_t<true>, grid, dim3(256), 0, (hipStream_t)stream, a);
    else
        hipLaunchKernelGGL(smg_tree_commit_t<false>, grid, dim3(256), 0, (hipStream_t)stream, a);
    return hipGetLastError() == hipSuccess ? 0 : -2;
}
