"""Serving operators of the worker engine on gfx950: attention of packed prompts
and of drafted token trees over the slot cache, committing accepted drafts, and
sampling.  Each checks its tensors, launches hand-written kernels of smg_amd._core
on the current stream of the tensors' device, and neither synchronises nor copies
to the host, so all of them can be captured into graphs.

The cache is the engine's: [slots, kv heads, positions, head dim] a layer, in
bfloat16 or float8_e4m3fn; its dimensions may have any strides but the last,
which is dense.  Rows of tensors that kernels read 16 bytes at a time start at
multiples of 16 bytes (8 where tree_commit writes an 8-bit cache).

They are forwards without a gradient, for a worker that answers: any argument that
asks for one is refused where gradients are recorded, and one with a forward-mode
tangent always.

What the host cannot see is bounded on the device: a sequence whose slot lies
outside the cache is a padding entry, lengths and offsets are cut to the tensors.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

_BF16, _FP8, _I32, _I64, _F32 = (torch.bfloat16, torch.float8_e4m3fn, torch.int32, torch.int64, torch.float32)
_CACHE_TYPES = (_BF16, _FP8)
HEAD_DIMS = (64, 128)
MAX_NODES = 64
MAX_VOCAB = 1 << 20
MAX_SEQUENCES = 1 << 16  # workgroups look through all sequences for their own

try:
    from .. import _core
except ImportError:  # refusals work without the built core
    _core = None
# a core built from older sources may lack these kernels
BUILT = all(hasattr(_core, k) for k in ("attn_prefill", "attn_tree", "attn_part_floats", "tree_commit", "sample", "sample_work_bytes"))
NOT_BUILT = "smg_amd._core lacks the gfx950 kernels of smg_amd.engine.ops: run `python -m smg_amd.csrc.build`"


# The checks are written for speed: one condition a tensor, and the reasons only
# where it fails.
def _check(name: str, t, dtypes: tuple, dim: int, dev: Optional[int]) -> None:
    if isinstance(t, torch.Tensor) and t.dtype in dtypes and t.dim() == dim and (dev is None or t.get_device() == dev):
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    if t.dim() != dim:
        raise ValueError(f"{name} must have {dim} dimensions, got {tuple(t.shape)}")
    raise ValueError(f"{name} is on {t.device}, the other tensors are not")


def _rows(name: str, t: torch.Tensor, unit: int = 16) -> tuple:
    """The strides but the last, of a tensor that is dense in its last dimension and
    whose rows start at multiples of `unit` bytes."""
    *strides, last = t.stride()
    at, e = t.data_ptr(), t.element_size()
    for s in strides:
        at |= s * e
    if (last != 1 or at % unit) and t.numel():
        if last != 1:
            raise ValueError(f"{name} must be dense in its last dimension, strides {t.stride()}")
        if t.data_ptr() % unit or any(s * e % unit for s, n in zip(strides, t.shape) if n > 1):
            raise ValueError(f"{name}: rows must start at multiples of {unit} bytes, strides {t.stride()}")
    return strides


def _index(name: str, t, shape: tuple, dev: int, dtype: torch.dtype = _I32) -> int:
    """The address of a contiguous tensor of that shape."""
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.get_device() == dev and t.is_contiguous():
        return t.data_ptr()
    _check(name, t, (dtype,), len(shape), dev)
    raise ValueError(f"{name} must be contiguous {shape}, got {tuple(t.shape)} with strides {t.stride()}")


def _cache(k: torch.Tensor, v: torch.Tensor, dev: int, H: int, D: int) -> tuple:
    """(slots, kv heads, positions) and the strides of both."""
    _check("k_cache", k, _CACHE_TYPES, 4, dev)
    _check("v_cache", v, _CACHE_TYPES, 4, dev)
    S, KVH, T, d = shape = k.shape
    if shape != v.shape or k.dtype is not v.dtype:
        raise ValueError(f"k_cache {tuple(shape)} {k.dtype} and v_cache {tuple(v.shape)} {v.dtype} differ")
    if d != D or D not in HEAD_DIMS:
        raise ValueError(f"head dim must be one of {HEAD_DIMS} and equal, got {D} over a cache of {d}")
    if S < 1 or KVH < 1 or not 1 <= T <= 1 << 30 or H < 1 or H % KVH:
        raise ValueError(f"{H} heads over a cache of {tuple(shape)}")
    return S, KVH, T, _rows("k_cache", k) + _rows("v_cache", v)


def _scale(scale: Optional[float], D: int) -> float:
    if scale is None:
        return D ** -0.5
    scale = float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    return scale


def _repeats(t: torch.Tensor) -> bool:
    """Whether several of its elements share a place in memory by a stride of 0."""
    return 0 in t.stride() and any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape))


def _out(out: Optional[torch.Tensor], q: torch.Tensor, dev: int) -> torch.Tensor:
    if out is None:
        return torch.empty_like(q, memory_format=torch.contiguous_format)
    _check("out", out, (_BF16,), q.dim(), dev)
    if out.shape != q.shape or _repeats(out):
        raise ValueError(f"out must be {tuple(q.shape)} with a place for every element, got {tuple(out.shape)} with strides {out.stride()}")
    return out


def _on_gpu(dev: int, **floats) -> None:
    """That the call can run: floats are its arguments that could ask for a gradient, the
    first argument first."""
    if torch.is_grad_enabled():
        for name, t in floats.items():
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{name} asks for a gradient, and the operators have none: detach it or use torch.no_grad()")
    if forward_ad._current_level >= 0:
        for name, t in floats.items():
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{name} has a tangent, and the operators have none: take its primal")
    if dev < 0:
        name, t = next(iter(floats.items()))
        raise RuntimeError(f"{name} is on {t.device}: the operators run on a CUDA/HIP device")
    if not BUILT:
        raise RuntimeError(NOT_BUILT)


def _launch(kernel, dev: int, *args) -> None:
    """kernel(*args, stream), on the device's current stream and with that device current."""
    stream = torch._C._cuda_getCurrentRawStream(dev)
    if torch._C._cuda_getDevice() == dev:
        kernel(*args, stream)
    else:
        with torch.cuda.device(dev):
            kernel(*args, stream)


def _shape(total: int, each: int, B: int, KVH: int, D: int, fp8: bool, ctx: int) -> Tuple[int, int, int]:
    """How attention is cut: waves of a workgroup along the query rows (32 each), waves along
    the keys, and the most runs that a row's keys are split into (the kernel sizes them by
    the sequences' lengths).  total: query rows of a kv head over all sequences, of which
    each has `each`, or any number of them if that is 0.

    More rows a workgroup read K/V less often, but few workgroups leave compute units idle:
    the most rows that fill the card are taken (16 prompts of 75 tokens over 460 rows, 4 kv
    heads: 21 us with 2 waves, 24 with 4, 37 with 1; 32 of them: 34, 32 and 63).  Where each
    workgroup has a compute unit for itself, more waves take its keys (64 trees of 16 nodes
    over 1150 rows: 38 us by 2 x 4 waves, 43 by 2 x 2; with twice the workgroups 43 and 34).
    4 waves along the rows pay in 16 bits where that leaves more workgroups than units by far
    (24 prompts, 260 workgroups: 25 us, 22 by 2; 32, 356: 30 and 32; one prompt of 3000
    tokens with 372 loses all the same: 73 and 56).  In 8 bits a unit takes one workgroup: 2
    waves until there are more of them than units (12 prompts, 124 of 4: 24 us by 2, 26 by 4;
    16, 176 of 4: 39 and 26), 8 where 4 would be more (32 prompts, 208 of 8: 34 us, 46 by 4;
    one of 3000, 184 of 8: 103 and 82).
    Splitting keys fills the card with few rows, and writes and reads partial results of as
    many rows as it takes at once: it has to save the time of about 1450 keys in 16 bits,
    650 in 8 (8 trees of 61 nodes over up to 4000 rows: 41 us split, 53 not; 16 prompts of 18
    tokens over up to 2000: 33 and 29)."""
    def work(waves: int) -> int:
        at_once = 32 * waves
        return KVH * (B * -(-each // at_once) if each else max(B, total // at_once + B // 2))

    units = 256  # compute units
    long = total > 128 * B and ctx >= 4096  # rows for 8 waves, and K/V worth reading once
    runs = max(1, min(64, ctx // 256))
    if fp8:
        four = work(4)
        if ctx * (units - four) > 650 * units:
            return (8, 1, runs) if long else (4, 2, runs)
        return (8, 1, 1) if total > 128 * B and work(8) >= 200 else (4, 2, 1) if four >= 100 else (2, 2, 1)
    two = work(2)
    if ctx * (units - two) > 1450 * units:
        return (4, 1, runs) if long else (2, 2, runs)
    if D == 128 and two <= units:
        return (1, 4, 1) if two <= 64 else (2, 4, 1)
    return (4, 1, 1) if total > 64 * B and work(4) >= 320 else (2, 2, 1)


def _parts(q: torch.Tensor, tree: bool, B: int, N: int, H: int, KVH: int, D: int, split: int, wr: int, wk: int, fp8: bool):
    """Workspace of the runs' partial results: a place for every row of the workgroups that
    the card takes at once, 17 or 34 MB at a head dim of 128, however many runs a row may have."""
    if split == 1:
        return None
    return torch.empty(_core.attn_part_floats(tree, B, N, H, KVH, D, split, wr, wk, fp8), dtype=_F32, device=q.device)


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
    [N, H, D], which may be q itself and shares no memory with the arguments otherwise;
    rows that no sequence covers are not written.  A sequence whose slot lies outside
    the cache gets zeros."""
    _check("q", q, (_BF16,), 3, None)
    dev = q.get_device()
    N, H, D = q.shape
    S, KVH, T, cache_strides = _cache(k_cache, v_cache, dev, H, D)
    B = slots.shape[0] if isinstance(slots, torch.Tensor) and slots.dim() else 0
    p_slots = _index("slots", slots, (B,), dev)
    p_starts = _index("starts", starts, (B,), dev)
    p_cu = _index("cu_seqlens", cu_seqlens, (B + 1,), dev)
    scale = _scale(scale, D)
    out = _out(out, q, dev)
    strides = _rows("q", q) + _rows("out", out) + cache_strides
    if N * H > 1 << 30 or B > MAX_SEQUENCES:
        raise ValueError(f"at most {1 << 30} rows of a head in {MAX_SEQUENCES} sequences, got {N} x {H} in {B}")
    _on_gpu(dev, q=q, k_cache=k_cache, v_cache=v_cache, out=out)
    if N == 0 or B == 0:
        return out
    total = N * (H // KVH)
    fp8 = k_cache.dtype is _FP8
    wr, wk, split = _shape(total, 0, B, KVH, D, fp8, T if max_ctx is None else min(int(max_ctx), T))
    part = _parts(q, False, B, N, H, KVH, D, split, wr, wk, fp8)
    _launch(
        _core.attn_prefill, dev, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), p_slots, p_starts, p_cu,
        out.data_ptr(), 0 if part is None else part.data_ptr(), strides, B, N, H, KVH, S, T, D, split, wr, wk, scale, fp8,
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
    card (default: the cache's length).  Returns out [B, N, H, D], which may be q
    itself and shares no memory with the arguments otherwise."""
    _check("q", q, (_BF16,), 4, None)
    dev = q.get_device()
    B, N, H, D = q.shape
    S, KVH, T, cache_strides = _cache(k_cache, v_cache, dev, H, D)
    _check("k_new", k_new, (_BF16,), 4, dev)
    _check("v_new", v_new, (_BF16,), 4, dev)
    if not k_new.shape == v_new.shape == (B, N, KVH, D):
        raise ValueError(f"k_new and v_new must be {(B, N, KVH, D)}, got {tuple(k_new.shape)} and {tuple(v_new.shape)}")
    if N > MAX_NODES:
        raise ValueError(f"at most {MAX_NODES} drafted nodes, got {N}")
    p_slots = _index("slots", slots, (B,), dev)
    p_ctx = _index("ctx_lens", ctx_lens, (B,), dev)
    p_parents = _index("parents", parents, (B, N), dev)
    scale = _scale(scale, D)
    out = _out(out, q, dev)
    strides = _rows("q", q) + _rows("out", out) + cache_strides + _rows("k_new", k_new) + _rows("v_new", v_new)
    if B * N * H > 1 << 30 or B > MAX_SEQUENCES:
        raise ValueError(f"at most {1 << 30} rows of a head in {MAX_SEQUENCES} sequences, got {B} x {N} x {H}")
    _on_gpu(dev, q=q, k_new=k_new, v_new=v_new, k_cache=k_cache, v_cache=v_cache, out=out)
    if B == 0 or N == 0:
        return out
    rows = N * (H // KVH)
    fp8 = k_cache.dtype is _FP8
    wr, wk, split = _shape(B * rows, rows, B, KVH, D, fp8, T if max_ctx is None else min(int(max_ctx), T))
    part = _parts(q, True, B, N, H, KVH, D, split, wr, wk, fp8)
    _launch(
        _core.attn_tree, dev, q.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
        p_slots, p_ctx, p_parents, out.data_ptr(), 0 if part is None else part.data_ptr(), strides, B, N, H, KVH, S, T, D, split, wr, wk, scale, fp8,
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
    no room or whose node 0 has a parent is padding: 0, -1, -1.  Of other sequences
    that name the same slot the last one's rows are written."""
    _check("kv_new", kv_new, (_BF16,), 6, None)
    dev = kv_new.get_device()
    L, two, B, N, KVH, D = kv_new.shape
    _check("kv_cache", kv_cache, _CACHE_TYPES, 6, dev)
    S, T = kv_cache.shape[2], kv_cache.shape[4]
    if two != 2 or kv_cache.shape != (L, 2, S, KVH, T, D) or min(L, S, KVH, T, D) < 1:
        raise ValueError(f"kv_new {tuple(kv_new.shape)} does not fit kv_cache {tuple(kv_cache.shape)}")
    if D % 8:
        raise ValueError(f"head dim must be a multiple of 8, got {D}")
    if B > MAX_SEQUENCES:
        raise ValueError(f"at most {MAX_SEQUENCES} sequences, got {B}")
    if _repeats(kv_cache):
        raise ValueError(f"kv_cache must have a place for every element, strides {kv_cache.stride()}")
    if N > MAX_NODES or (N < 1 and B > 0):
        raise ValueError(f"1 to {MAX_NODES} drafted nodes, got {N}")
    strides = _rows("kv_new", kv_new) + _rows("kv_cache", kv_cache, 16 if kv_cache.dtype is _BF16 else 8)
    given = (
        _index("slots", slots, (B,), dev), _index("ctx_lens", ctx_lens, (B,), dev),
        _index("parents", parents, (B, N), dev), _index("tokens", tokens, (B, N), dev, _I64),
        _index("targets", targets, (B, N), dev, _I64),
    )
    _on_gpu(dev, kv_new=kv_new, kv_cache=kv_cache)
    count, path, nxt = torch.empty_like(ctx_lens), torch.empty_like(parents), tokens.new_empty(B)
    if B:
        _launch(
            _core.tree_commit, dev, kv_new.data_ptr(), kv_cache.data_ptr(), *given, count.data_ptr(), path.data_ptr(),
            nxt.data_ptr(), strides, B, N, L, KVH, S, T, D, kv_cache.dtype is _FP8,
        )
    return count, path, nxt


def _parts_of(R: int, V: int) -> int:
    """Workgroups that share a row of logits: few long rows leave most of the card idle.
    One row of 131072 alone and shared by 8: 69 and 44 us with a top-p, 39 and 14 without a
    cut, 26 and 30 with a top-k of 50; 64 rows alone and by 4, of mixed settings: 117 and
    70.  Below 65536 the five launches cost what they save."""
    if V < 65536 or R > 128:
        return 1
    return max(1, min(16, V // 16384, 256 // R))


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
    _check("logits", logits, (_BF16, _F32), 2, None)
    dev = logits.get_device()
    R, V = logits.shape
    if not 1 <= V <= MAX_VOCAB:
        raise ValueError(f"1 to {MAX_VOCAB} columns of logits, got {V}")
    stride, dense = logits.stride()
    if V > 1 and dense != 1:
        raise ValueError(f"logits must be dense in their last dimension, strides {logits.stride()}")
    rows = (R,)
    p_u = _index("u", u, rows, dev, _F32)
    p_temperature = _index("temperature", temperature, rows, dev, _F32)
    p_k = 0 if top_k is None else _index("top_k", top_k, rows, dev)
    p_p = 0 if top_p is None else _index("top_p", top_p, rows, dev, _F32)
    p_m = 0 if min_p is None else _index("min_p", min_p, rows, dev, _F32)
    if out is not None:
        _index("out", out, rows, dev, _I64)
    _on_gpu(dev, logits=logits, u=u, temperature=temperature, top_p=top_p, min_p=min_p)
    if out is None:
        out = torch.empty(rows, dtype=_I64, device=logits.device)
    if R:
        parts = _parts_of(R, V)
        work = None if parts == 1 else torch.empty(R * _core.sample_work_bytes(), dtype=torch.uint8, device=logits.device)
        _launch(
            _core.sample, dev, logits.data_ptr(), p_u, p_temperature, p_k, p_p, p_m, out.data_ptr(),
            0 if work is None else work.data_ptr(), stride, R, V, parts, logits.dtype is _F32,
        )
    return out
