"""Serving operators of the worker engine on gfx950: attention of packed prompts
and of drafted token trees over the slot cache, committing accepted drafts, and
sampling.  Each checks its tensors, launches hand-written kernels of smg_amd._core
on the current stream of the tensors' device, and neither synchronises nor copies
to the host, so all of them can be captured into graphs.

The cache is the engine's: [slots, kv heads, positions, head dim] a layer, in
bfloat16 or float8_e4m3fn; its dimensions may have any strides but the last,
which is dense.  Rows of tensors that kernels read 16 bytes at a time start at
multiples of 16 bytes.

What the host cannot see is bounded on the device: a sequence whose slot lies
outside the cache is a padding entry, lengths and offsets are cut to the tensors.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

_CACHE_TYPES = (torch.bfloat16, torch.float8_e4m3fn)
HEAD_DIMS = (64, 128)
MAX_NODES = 64
MAX_VOCAB = 1 << 20


def _core():
    from .. import _core as core

    return core


def _check(name: str, t: torch.Tensor, dtypes, dim: int, device=None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    if t.dim() != dim:
        raise ValueError(f"{name} must have {dim} dimensions, got {tuple(t.shape)}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")


def _check_rows(name: str, t: torch.Tensor) -> None:
    """The last dimension dense, and every row at a multiple of 16 bytes (8 in an 8-bit cache)."""
    e = t.element_size()
    unit = 16 if e > 1 else 8
    if t.numel() == 0:
        return
    if t.stride(-1) != 1:
        raise ValueError(f"{name} must be dense in its last dimension, strides {t.stride()}")
    if t.data_ptr() % unit or any(s * e % unit for s, n in zip(t.stride()[:-1], t.shape) if n > 1):
        raise ValueError(f"{name}: rows must start at multiples of {unit} bytes, strides {t.stride()}")


def _check_index(name: str, t: torch.Tensor, shape: tuple, device, dtype=torch.int32) -> None:
    _check(name, t, (dtype,), len(shape), device)
    if tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous {shape}, got {tuple(t.shape)} with strides {t.stride()}")


def _check_gpu(name: str, t: torch.Tensor) -> None:
    if t.device.type != "cuda":
        raise RuntimeError(f"{name} is on {t.device}: the operators run on a CUDA/HIP device")


def _check_cache(k: torch.Tensor, v: torch.Tensor, q: torch.Tensor, H: int, D: int) -> Tuple[int, int, int]:
    for name, t in (("k_cache", k), ("v_cache", v)):
        _check(name, t, _CACHE_TYPES, 4, q.device)
        _check_rows(name, t)
    if k.shape != v.shape or k.dtype != v.dtype:
        raise ValueError(f"k_cache {tuple(k.shape)} {k.dtype} and v_cache {tuple(v.shape)} {v.dtype} differ")
    S, KVH, T, d = k.shape
    if d != D or D not in HEAD_DIMS:
        raise ValueError(f"head dim must be one of {HEAD_DIMS} and equal, got {D} over a cache of {d}")
    if min(S, KVH, T) < 1 or H % KVH:
        raise ValueError(f"{H} heads over a cache of {tuple(k.shape)}")
    return S, KVH, T


def _scale(scale: Optional[float], D: int) -> float:
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    return scale


def _out_like(out: Optional[torch.Tensor], q: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _check("out", out, (torch.bfloat16,), q.dim(), q.device)
    if out.shape != q.shape:
        raise ValueError(f"out must be {tuple(q.shape)}, got {tuple(out.shape)}")
    _check_rows("out", out)
    return out


def _plan(rows: int, tiles_of, ctx: int, KVH: int, D: int) -> Tuple[int, int]:
    """(waves along the query rows, splits of the keys) for sequences of about
    `rows` rows a kv head and up to `ctx` keys; tiles_of(rows a tile) counts tiles."""
    wr = 1 if rows <= 32 and D == 128 else 2 if rows <= 64 else 4
    work = tiles_of(32 * wr) * KVH
    split = 1
    while split < 64 and work * split < 512 and ctx // (split * 2) >= 256:
        split *= 2
    return wr, split


def _parts(split: int, rows: int, D: int, device):
    if split == 1:
        return None, 0, 0
    part = torch.empty(split * rows * (D + 2), dtype=torch.float32, device=device)
    return part, part.data_ptr(), part.data_ptr() + split * rows * D * 4


def attn_prefill(
    q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor,
    starts: torch.Tensor, cu_seqlens: torch.Tensor, *, scale: Optional[float] = None,
    max_ctx: Optional[int] = None, out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Causal attention of packed prompts, or chunks of prompts, over the cache.

    q [N, H, D] bfloat16 holds the sequences one after the other: sequence b has
    the rows cu_seqlens[b] .. cu_seqlens[b+1]-1 (int32, rising, [B+1]), and its
    token i sees the rows 0 .. starts[b]+i of slot slots[b] (both int32 [B]); the
    new tokens' K/V are in the cache already.  Head h reads kv head h // (H/KVH).

    max_ctx, a bound on starts[b] plus the new tokens, only sizes the split of
    long caches over the card (default: the cache's length).  Returns out
    [N, H, D]; rows that no sequence covers are not written.  A sequence whose slot
    lies outside the cache gets zeros."""
    _check("q", q, (torch.bfloat16,), 3)
    N, H, D = q.shape
    S, KVH, T = _check_cache(k_cache, v_cache, q, H, D)
    _check_rows("q", q)
    B = slots.shape[0] if isinstance(slots, torch.Tensor) and slots.dim() else 0
    _check_index("slots", slots, (B,), q.device)
    _check_index("starts", starts, (B,), q.device)
    _check_index("cu_seqlens", cu_seqlens, (B + 1,), q.device)
    scale = _scale(scale, D)
    out = _out_like(out, q)
    _check_gpu("q", q)
    if N == 0 or B == 0:
        return out
    G = H // KVH
    ctx = T if max_ctx is None else max(1, min(int(max_ctx), T))
    wr, split = _plan(N * G // B, lambda bm: N * G // bm + B, ctx, KVH, D)
    with torch.cuda.device(q.device):
        part, po, pm = _parts(split, N * H, D, q.device)
        _core().attn_prefill(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), slots.data_ptr(), starts.data_ptr(),
            cu_seqlens.data_ptr(), out.data_ptr(), po, pm,
            [*q.stride()[:2], *out.stride()[:2], *k_cache.stride()[:3], *v_cache.stride()[:3]],
            B, N, H, KVH, S, T, D, split, wr, scale, int(k_cache.dtype == torch.float8_e4m3fn),
            torch.cuda.current_stream().cuda_stream,
        )
    return out


def attn_tree(
    q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, k_cache: torch.Tensor,
    v_cache: torch.Tensor, slots: torch.Tensor, ctx_lens: torch.Tensor, parents: torch.Tensor, *,
    scale: Optional[float] = None, max_ctx: Optional[int] = None, out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Attention of drafted token trees over the cache.

    q [B, N, H, D] and k_new, v_new [B, N, KVH, D], all bfloat16, hold N <= 64
    drafted nodes a sequence.  Node i sees the rows 0 .. ctx_lens[b]-1 of slot
    slots[b], its ancestors, and itself.  parents int32 [B, N]: the parent of a
    node, which comes before it, or -1 for a node right after the context.  Any
    other value, and a node below such a one, is padding and gets zeros, as does a
    sequence whose slot lies outside the cache.

    max_ctx, a bound on ctx_lens, only sizes the split of long caches over the
    card (default: the cache's length)."""
    _check("q", q, (torch.bfloat16,), 4)
    B, N, H, D = q.shape
    S, KVH, T = _check_cache(k_cache, v_cache, q, H, D)
    _check_rows("q", q)
    for name, t in (("k_new", k_new), ("v_new", v_new)):
        _check(name, t, (torch.bfloat16,), 4, q.device)
        if tuple(t.shape) != (B, N, KVH, D):
            raise ValueError(f"{name} must be {(B, N, KVH, D)}, got {tuple(t.shape)}")
        _check_rows(name, t)
    if N > MAX_NODES:
        raise ValueError(f"at most {MAX_NODES} drafted nodes, got {N}")
    _check_index("slots", slots, (B,), q.device)
    _check_index("ctx_lens", ctx_lens, (B,), q.device)
    _check_index("parents", parents, (B, N), q.device)
    scale = _scale(scale, D)
    out = _out_like(out, q)
    _check_gpu("q", q)
    if B == 0 or N == 0:
        return out
    G = H // KVH
    ctx = T if max_ctx is None else max(1, min(int(max_ctx), T))
    wr, split = _plan(N * G, lambda bm: B * -(-N * G // bm), ctx, KVH, D)
    with torch.cuda.device(q.device):
        part, po, pm = _parts(split, B * N * H, D, q.device)
        _core().attn_tree(
            q.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
            slots.data_ptr(), ctx_lens.data_ptr(), parents.data_ptr(), out.data_ptr(), po, pm,
            [*q.stride()[:3], *out.stride()[:3], *k_cache.stride()[:3], *v_cache.stride()[:3],
             *k_new.stride()[:3], *v_new.stride()[:3]],
            B, N, H, KVH, S, T, D, split, wr, scale, int(k_cache.dtype == torch.float8_e4m3fn),
            torch.cuda.current_stream().cuda_stream,
        )
    return out


def tree_commit(
    kv_new: torch.Tensor, kv_cache: torch.Tensor, slots: torch.Tensor, ctx_lens: torch.Tensor,
    parents: torch.Tensor, tokens: torch.Tensor, targets: torch.Tensor,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Accepts drafted tokens and writes their K/V to the cache of every layer.

    tokens int64 [B, N] are the drafted tokens, targets int64 [B, N] the ones that
    the model chose at each node; parents int32 [B, N] as in attn_tree.  Node 0 is
    always taken (it is the token of the last step); after it, as long as there is
    one, the first child of the node taken last whose token is that node's target.
    The taken nodes' rows of kv_new [L, 2, B, N, KVH, D] bfloat16 go to the rows
    ctx_lens[b] onwards of slot slots[b] in kv_cache [L, 2, S, KVH, T, D], as far
    as the cache has room.

    Returns (count int32 [B], path int32 [B, N], next int64 [B]): how many nodes
    were taken, which (-1 after the last), and the last one's target, the
    sequence's next token.  A sequence whose slot lies outside the cache, that has
    no room or whose node 0 has a parent is padding: 0, -1, -1.  Of sequences that
    name the same slot the last one's rows are written."""
    _check("kv_new", kv_new, (torch.bfloat16,), 6)
    L, two, B, N, KVH, D = kv_new.shape
    _check("kv_cache", kv_cache, _CACHE_TYPES, 6, kv_new.device)
    S, T = kv_cache.shape[2], kv_cache.shape[4]
    if two != 2 or tuple(kv_cache.shape) != (L, 2, S, KVH, T, D) or min(L, S, KVH, T, D) < 1:
        raise ValueError(f"kv_new {tuple(kv_new.shape)} does not fit kv_cache {tuple(kv_cache.shape)}")
    if D % 8:
        raise ValueError(f"head dim must be a multiple of 8, got {D}")
    _check_rows("kv_new", kv_new)
    _check_rows("kv_cache", kv_cache)
    if N > MAX_NODES or (N < 1 and B > 0):
        raise ValueError(f"1 to {MAX_NODES} drafted nodes, got {N}")
    _check_index("slots", slots, (B,), kv_new.device)
    _check_index("ctx_lens", ctx_lens, (B,), kv_new.device)
    _check_index("parents", parents, (B, N), kv_new.device)
    _check_index("tokens", tokens, (B, N), kv_new.device, torch.int64)
    _check_index("targets", targets, (B, N), kv_new.device, torch.int64)
    _check_gpu("kv_new", kv_new)
    count = torch.empty(B, dtype=torch.int32, device=kv_new.device)
    path = torch.empty(B, N, dtype=torch.int32, device=kv_new.device)
    nxt = torch.empty(B, dtype=torch.int64, device=kv_new.device)
    if B == 0:
        return count, path, nxt
    with torch.cuda.device(kv_new.device):
        _core().tree_commit(
            kv_new.data_ptr(), kv_cache.data_ptr(), slots.data_ptr(), ctx_lens.data_ptr(),
            parents.data_ptr(), tokens.data_ptr(), targets.data_ptr(), count.data_ptr(),
            path.data_ptr(), nxt.data_ptr(), [*kv_new.stride()[:5], *kv_cache.stride()[:5]],
            B, N, L, KVH, S, T, D, int(kv_cache.dtype == torch.float8_e4m3fn),
            torch.cuda.current_stream().cuda_stream,
        )
    return count, path, nxt


def sample(
    logits: torch.Tensor, u: torch.Tensor, temperature: torch.Tensor, *,
    top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None,
    min_p: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Draws a token for every row of logits [R, V] (bfloat16 or float32) from the
    uniform number u (float32 [R], in [0, 1)) of the row; int64 [R].

    With w = softmax(logits / temperature) over its largest value, and the tokens
    in falling order of their logits (equal ones by index): top_k (int32 [R], 0 for
    none) keeps the first k, top_p (float32 [R], 1 for none) of those the ones
    whose predecessors hold less than the share p of what top_k kept, and min_p
    (float32 [R], 0 for none) of those the ones with w >= min_p; the first token of
    the order is always kept.  The answer is the first token by index at which the
    kept weights add up to more than u times their sum.  Weights count in multiples
    of 2^-S, S = min(50, 62 - ceil(log2 V)), in exact sums: the answer is the same every time,
    and a token below half of that is never taken.  temperature (float32 [R]) 0
    takes the first token of the order.  -inf and NaN logits are never taken; a
    row of nothing else gives -1."""
    _check("logits", logits, (torch.bfloat16, torch.float32), 2)
    R, V = logits.shape
    if not 1 <= V <= MAX_VOCAB:
        raise ValueError(f"1 to {MAX_VOCAB} columns of logits, got {V}")
    if V > 1 and logits.stride(1) != 1:
        raise ValueError(f"logits must be dense in their last dimension, strides {logits.stride()}")
    dev = logits.device
    _check_index("u", u, (R,), dev, torch.float32)
    _check_index("temperature", temperature, (R,), dev, torch.float32)
    for name, t, dtype in (("top_k", top_k, torch.int32), ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)):
        if t is not None:
            _check_index(name, t, (R,), dev, dtype)
    if out is not None:
        _check_index("out", out, (R,), dev, torch.int64)
    _check_gpu("logits", logits)
    if out is None:
        out = torch.empty(R, dtype=torch.int64, device=dev)
    if R == 0:
        return out
    with torch.cuda.device(dev):
        _core().sample(
            logits.data_ptr(), u.data_ptr(), temperature.data_ptr(),
            0 if top_k is None else top_k.data_ptr(), 0 if top_p is None else top_p.data_ptr(),
            0 if min_p is None else min_p.data_ptr(), out.data_ptr(), logits.stride(0), R, V,
            int(logits.dtype == torch.float32), torch.cuda.current_stream().cuda_stream,
        )
    return out
