"""Cases for the worker engine's serving operators: attention of packed prompts
over the slot cache, attention of drafted token trees over it, committing the
accepted drafts, and sampling.

`run` computes a case in its plain form (elementary torch operations in 32 bits,
64 where a decision hangs on the last bits), or, where `own` is true, with the
operators of smg_amd.engine.ops.  All caches are one slot arena as the engine
lays it out: [slots, kv heads, positions, head dim] a layer.
"""
import math

import torch

own = False

DEV = "cuda:0"


# ---- cases ------------------------------------------------------------------
def listed():
    return [
        # the tiny engine configuration: a one-token prompt, an odd and a full one
        dict(name="prefill_tiny", op="prefill", B=3, new=64, hist=0, H=4, KVH=4, D=64, T=256, S=8, fp8=False),
        # 32 prefix-cache hits of the serving benchmark: 512 cached tokens, ragged
        # suffixes around its 64, grouped heads
        dict(name="prefill_cache_hits", op="prefill", B=32, new=128, hist=512, H=16, KVH=4, D=128, T=704, S=520, fp8=False),
        # a chunk of two long prompts over an 8-bit cache, every head its own K/V
        dict(name="prefill_chunk_fp8", op="prefill", B=2, new=1999, hist=6000, H=16, KVH=16, D=128, T=8192, S=4, fp8=True),
        # one whole long prompt
        dict(name="prefill_long", op="prefill", B=1, new=16384, hist=0, H=16, KVH=4, D=128, T=16384, S=1, fp8=False),
        # one request with a chain of drafts on the tiny configuration
        dict(name="tree_tiny", op="tree", B=1, N=5, ctx=77, H=4, KVH=4, D=64, T=256, S=8, fp8=False),
        # a serving batch with 16 drafted tokens each at the benchmark's lengths
        dict(name="tree_batch", op="tree", B=64, N=16, ctx=2000, H=16, KVH=4, D=128, T=2048, S=64, fp8=False),
        # few long conversations, wide trees of an odd size, 8-bit cache
        dict(name="tree_long_fp8", op="tree", B=4, N=61, ctx=65000, H=16, KVH=4, D=128, T=65536, S=5, fp8=True),
        # the commits that follow the trees: a single request, then a batch over all 16 layers
        dict(name="commit_tiny", op="commit", L=2, B=1, N=5, KVH=4, D=64, T=256, S=8, fp8=False),
        dict(name="commit_batch", op="commit", L=16, B=64, N=32, KVH=4, D=128, T=256, S=64, fp8=True),
        # one request's next token, a full serving batch, and a wide vocabulary of an odd
        # size in 32 bits
        dict(name="sample_one", op="sample", R=1, V=2048, f32=False, spread=3.0),
        dict(name="sample_batch", op="sample", R=512, V=32768, f32=False, spread=3.0),
        dict(name="sample_wide_f32", op="sample", R=64, V=131071, f32=True, spread=2.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["prefill", "tree", "commit", "sample"])
    KVH = rng.choice([1, 2, 4, 8])
    H, D, fp8 = KVH * rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 128]), rng.random() < 0.4
    if op == "prefill":
        B = _log(rng, 1, 64)
        new = _log(rng, 1, max(1, min(8192, 16384 // B)))
        hist = rng.choice([0, _log(rng, 1, 8192)])
        if B * new * (hist + new) * H > 16384 * 16384 * 16:  # as much as prefill_long
            new = max(1, 16384 * 16384 * 16 // (B * (hist + new) * H))
        T = (hist + new + rng.randrange(1, 70)) // 8 * 8 + 8
        return dict(op=op, B=B, new=new, hist=hist, H=H, KVH=KVH, D=D, T=T, S=B + rng.randrange(0, 4), fp8=fp8)
    if op == "tree":
        B, N = _log(rng, 1, 128), _log(rng, 1, 64)
        ctx = _log(rng, 1, max(16, 200_000 // B))
        return dict(op=op, B=B, N=N, ctx=ctx, H=H, KVH=KVH, D=D, T=ctx + rng.randrange(64, 100), S=B + rng.randrange(0, 4), fp8=fp8)
    if op == "commit":
        B = _log(rng, 1, 64)
        return dict(op=op, L=rng.randrange(1, 17), B=B, N=_log(rng, 1, 64), KVH=rng.choice([1, 2, 4]), D=D, T=rng.randrange(80, 256), S=B + rng.randrange(0, 4), fp8=fp8)
    V = _log(rng, 100, 131_072)
    return dict(op=op, R=_log(rng, 1, max(1, min(1024, 16_000_000 // V))), V=V, f32=rng.random() < 0.4, spread=rng.choice([1.0, 2.0, 4.0]))


def _ragged(n, most, least, salt):
    """n lengths of least..most that go by the case alone: the first is the most,
    the second (of three or more) the least."""
    if n == 1 or most <= least:
        return [most] * n
    k = [least + (i * 2654435761 + salt * 40503 + i * i * 97) % (most - least + 1) for i in range(n)]
    k[0] = most
    if n > 2:
        k[1] = least
    return k


def _lengths(case):
    if case["op"] == "prefill":
        new = _ragged(case["B"], case["new"], 1 if case["hist"] == 0 else max(1, case["new"] // 4), 3)
        return new, _ragged(case["B"], case["hist"], case["hist"] * 3 // 4, 5)
    if case["op"] == "tree":
        return [case["N"]] * case["B"], _ragged(case["B"], case["ctx"], case["ctx"] // 8, 7)
    return [case["N"]] * case["B"], _ragged(case["B"], case["T"] - case["N"], 0, 11)


# ---- inputs -----------------------------------------------------------------
def _randn(gen, *shape, scale=1.0):
    return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(torch.bfloat16)


def _arena(gen, *shape, fp8):
    t = torch.empty(*shape, dtype=torch.float8_e4m3fn if fp8 else torch.bfloat16, device=DEV)
    for part in t.view(-1, shape[-1]).split(1 << 20):  # bounds the temporaries
        part.copy_(torch.randn(part.shape, generator=gen, device=DEV))
    return t


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _trees(gen, B, N):
    """Parents of B drafted trees: every node hangs below one of the four before it."""
    i = torch.arange(N, device=DEV).expand(B, N)
    back = 1 + torch.randint(0, 4, (B, N), generator=gen, device=DEV)
    return torch.where(i == 0, -1, (i - back).clamp_min(0)).to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 17)
    st = dict(case)
    if case["op"] == "sample":
        R, V = case["R"], case["V"]
        x = torch.randn(R, V, generator=gen, device=DEV) * case["spread"]
        st["logits"] = x if case["f32"] else x.to(torch.bfloat16)
        st["u"] = torch.rand(R, generator=gen, device=DEV)

        def pick(*values):  # a batch of requests has its own settings in every row
            return torch.tensor(values, device=DEV)[torch.randint(0, len(values), (R,), generator=gen, device=DEV)]

        st["temperature"] = pick(1.0, 0.7, 0.0, 1.3)
        st["top_k"] = pick(0, 50, 0, 1000).to(torch.int32)
        st["top_p"] = pick(1.0, 0.9, 0.95)
        st["min_p"] = pick(0.0, 0.0, 0.05)
        return st
    B, KVH, D, S, T = case["B"], case["KVH"], case["D"], case["S"], case["T"]
    new, ctx = _lengths(case)
    st["slots"] = torch.randperm(S, generator=gen, device=DEV)[:B].to(torch.int32)
    st["ctx"] = _i32(ctx)
    if case["op"] == "prefill":
        st["cu"] = _i32([sum(new[:i]) for i in range(B + 1)])
        st["max_new"], st["max_ctx"] = max(new), max(a + b for a, b in zip(new, ctx))
        st["q"] = _randn(gen, sum(new), case["H"], D, scale=1.5)
    else:
        N = case["N"]
        st["parents"] = _trees(gen, B, N)
        st["max_ctx"] = max(ctx)
    if case["op"] == "tree":
        st["q"] = _randn(gen, B, N, case["H"], D, scale=1.5)
        st["k_new"], st["v_new"] = _randn(gen, B, N, KVH, D), _randn(gen, B, N, KVH, D)
    if case["op"] == "commit":
        L = case["L"]
        st["kv_new"] = _randn(gen, L, 2, B, N, KVH, D)
        st["kv"] = _arena(gen, L, 2, S, KVH, T, D, fp8=case["fp8"])
        # drafts are right about two times in three: a node's target is the token of
        # the first child it has, or a token that no node has
        st["tokens"] = torch.randint(0, 2000, (B, N), generator=gen, device=DEV)
        child = st["parents"][:, None, :] == torch.arange(N, device=DEV)[:, None]
        right = child.any(-1) & (torch.rand(B, N, generator=gen, device=DEV) < 0.66)
        st["targets"] = torch.where(right, st["tokens"].gather(1, child.to(torch.uint8).argmax(-1)), 2001)
    else:
        st["k"], st["v"] = (_arena(gen, S, KVH, T, D, fp8=case["fp8"]) for _ in range(2))
    return st


# ---- the plain forms, and the framework's operators --------------------------
def run(st):
    if own:
        return _RUN_OWN[st["op"]](st)
    return _RUN_PLAIN[st["op"]](st)


def _softmax_v(scores, mask, v):
    """softmax over the last axis where the mask holds, times v."""
    scores = scores.masked_fill_(~mask, -math.inf)
    p = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    return (p @ v) / p.sum(-1, keepdim=True)


def _prefill_plain(st):
    # every request padded to the longest; the cache rows of its slot as one window
    q, cu, H, KVH, D = st["q"], st["cu"].long(), st["H"], st["KVH"], st["D"]
    B, L, T = st["B"], st["max_new"], st["max_ctx"]
    i = torch.arange(L, device=DEV)
    lens = cu[1:] - cu[:-1]
    row = (cu[:-1, None] + i).clamp_max(q.shape[0] - 1)
    qp = q[row].float().view(B, L, KVH, H // KVH, D).permute(0, 2, 3, 1, 4).reshape(B, KVH, -1, D)
    slots = st["slots"].long()
    k, v = st["k"][slots, :, :T].float(), st["v"][slots, :, :T].float()
    seen = torch.arange(T, device=DEV) <= (st["ctx"].long()[:, None] + i)[..., None]
    scores = (qp @ k.transpose(2, 3).contiguous()).mul_(D ** -0.5).view(B, KVH, H // KVH, L, T)
    o = _softmax_v(scores, seen[:, None, None], v[:, :, None])
    o = o.permute(0, 3, 1, 2, 4).reshape(B, L, H, D)
    at = torch.arange(q.shape[0], device=DEV)
    b = torch.searchsorted(cu[1:], at, right=True)
    return o[b, at - cu[b]].to(q.dtype)


def _prefill_own(st):
    from smg_amd.engine import ops

    return ops.attn_prefill(st["q"], st["k"], st["v"], st["slots"], st["ctx"], st["cu"], max_ctx=st["max_ctx"])


def _ancestors(parents):
    """[B, N, N]: whether node j is node i or above it."""
    N = parents.shape[1]
    step = (parents[..., None] == torch.arange(N, device=DEV)).float() + torch.eye(N, device=DEV)
    for _ in range(max(1, (N - 1).bit_length())):
        step = (step @ step).clamp_(max=1.0)
    return step > 0


def _tree_plain(st):
    B, N, H, KVH, D, T = st["B"], st["N"], st["H"], st["KVH"], st["D"], st["max_ctx"]
    slots = st["slots"].long()
    k = torch.cat([st["k"][slots, :, :T].float(), st["k_new"].float().transpose(1, 2)], 2)
    v = torch.cat([st["v"][slots, :, :T].float(), st["v_new"].float().transpose(1, 2)], 2)
    old = (torch.arange(T, device=DEV) < st["ctx"].long()[:, None])[:, None].expand(B, N, T)
    seen = torch.cat([old, _ancestors(st["parents"])], 2)
    q = st["q"].float().view(B, N, KVH, H // KVH, D).permute(0, 2, 3, 1, 4).reshape(B, KVH, -1, D)
    scores = (q @ k.transpose(2, 3).contiguous()).mul_(D ** -0.5).view(B, KVH, H // KVH, N, -1)
    o = _softmax_v(scores, seen[:, None, None], v[:, :, None])
    return o.permute(0, 3, 1, 2, 4).reshape(B, N, H, D).to(st["q"].dtype)


def _tree_own(st):
    from smg_amd.engine import ops

    return ops.attn_tree(st["q"], st["k_new"], st["v_new"], st["k"], st["v"], st["slots"], st["ctx"], st["parents"], max_ctx=st["max_ctx"])


def _commit_plain(st):
    parents, tokens, targets, kv = st["parents"].long(), st["tokens"], st["targets"], st["kv"]
    B, N = parents.shape
    i = torch.arange(N, device=DEV)
    up = parents.clamp_min(0)
    # a drafted token holds if it is what its parent's target says, and the first such child
    match = (parents >= 0) & (tokens == targets.gather(1, up))
    earlier = (match[:, None] & match[..., None] & (parents[:, None] == parents[..., None]) & (i < i[:, None])).any(-1)
    holds = (match & ~earlier) | (i == 0)
    taken = (holds[:, None] | ~_ancestors(st["parents"])).all(-1)
    count = taken.sum(1)
    path = torch.where(taken, i, N + i).sort(1).values
    valid = i < count[:, None]
    path = torch.where(valid, path, 0)
    last = path.gather(1, count[:, None] - 1)
    slots, at = st["slots"].long()[:, None], st["ctx"].long()[:, None] + i
    b = torch.arange(B, device=DEV)[:, None]
    # [B, N, L, 2, KVH, D]: the new rows of the path, and the old ones elsewhere
    rows = st["kv_new"].permute(2, 3, 0, 1, 4, 5)[b, path]
    window = kv.permute(2, 4, 0, 1, 3, 5)
    keep = valid[..., None, None, None, None]
    window[slots, at] = torch.where(keep, rows.float(), window[slots, at].float()).to(kv.dtype)
    return kv, count.to(torch.int32), torch.where(valid, path, -1).to(torch.int32), targets.gather(1, last)[:, 0]


def _commit_own(st):
    from smg_amd.engine import ops

    count, path, nxt = ops.tree_commit(st["kv_new"], st["kv"], st["slots"], st["ctx"], st["parents"], st["tokens"], st["targets"])
    return st["kv"], count, path, nxt


def _sample_plain(st):
    # 64 bits: a token is right or wrong, and u may fall next to a border
    x, t = st["logits"].double(), st["temperature"].double()[:, None]
    top = x.amax(-1, keepdim=True)
    w = ((x - top) / torch.where(t > 0, t, 1.0)).exp()
    w = torch.where(t > 0, w, (x == top).double())
    order = x.sort(dim=-1, descending=True, stable=True).indices  # ties: the lowest index first
    ws = w.gather(1, order)
    place = torch.arange(x.shape[1], device=DEV)
    k = st["top_k"].long()[:, None]
    ws = torch.where((place < k) | (k <= 0), ws, 0.0)
    p = st["top_p"].double()[:, None]
    before = ws.cumsum(-1) - ws
    ws = torch.where((before < p * ws.sum(-1, keepdim=True)) | (place == 0) | (p >= 1), ws, 0.0)
    ws = torch.where(ws >= st["min_p"].double()[:, None], ws, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, ws)
    c = w.cumsum(-1)
    token = (c <= st["u"].double()[:, None] * c[:, -1:]).sum(-1)
    return torch.where(t[:, 0] > 0, token, order[:, 0])


def _sample_own(st):
    from smg_amd.engine import ops

    return ops.sample(st["logits"], st["u"], st["temperature"], top_k=st["top_k"], top_p=st["top_p"], min_p=st["min_p"])


_RUN_PLAIN = {"prefill": _prefill_plain, "tree": _tree_plain, "commit": _commit_plain, "sample": _sample_plain}
_RUN_OWN = {"prefill": _prefill_own, "tree": _tree_own, "commit": _commit_own, "sample": _sample_own}


# ---- what a pass cannot do without -------------------------------------------
def work(case):
    if case["op"] == "sample":
        return {"bytes": case["R"] * (case["V"] * (4 if case["f32"] else 2) + 28), "flops": case["R"] * case["V"]}
    new, ctx = _lengths(case)
    KVH, D, B = case["KVH"], case["D"], case["B"]
    unit = 1 if case["fp8"] else 2
    if case["op"] == "commit":
        # about two accepted rows each, read in 16 bits and written in the cache's
        return {"bytes": case["L"] * 2 * B * 2 * KVH * D * (2 + unit) + B * case["N"] * 24, "flops": B * case["N"]}
    H = case["H"]
    rows = sum(new)
    if case["op"] == "prefill":
        keys = sum(a + b for a, b in zip(new, ctx))
        pairs = sum(a * b + a * (a + 1) // 2 for a, b in zip(new, ctx))
        return {"bytes": rows * H * D * 4 + 2 * keys * KVH * D * unit, "flops": 4 * pairs * H * D}
    pairs = sum(a * b + 3 * a for a, b in zip(new, ctx))
    return {"bytes": rows * (H + KVH) * D * 4 + 2 * sum(ctx) * KVH * D * unit, "flops": 4 * pairs * H * D}


# ---- the definition, in 64 bits ------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    return _EXACT[case["op"]](st)


def _attend(q, k, v, sees):
    """One head: rows of q over the keys that sees(first row, last row) gives, a piece at a time."""
    out = torch.empty(q.shape[0], v.shape[1], dtype=torch.float64, device=DEV)
    for a in range(0, q.shape[0], 2048):
        s = (q[a:a + 2048].double() @ k.double().t().contiguous()) / math.sqrt(q.shape[1])
        s = torch.where(sees(a, a + s.shape[0]), s, -math.inf)
        out[a:a + 2048] = torch.exp(s - torch.logsumexp(s, 1, keepdim=True)) @ v.double()
    return out


def _prefill_exact(st):
    G = st["H"] // st["KVH"]
    out = torch.empty(st["q"].shape, dtype=torch.float64, device=DEV)
    cu, ctx, slots = st["cu"].tolist(), st["ctx"].tolist(), st["slots"].tolist()
    for b in range(st["B"]):
        a, z = cu[b], cu[b + 1]
        end = ctx[b] + z - a
        for h in range(st["H"]):
            k, v = st["k"][slots[b], h // G, :end], st["v"][slots[b], h // G, :end]
            at = torch.arange(end, device=DEV)
            out[a:z, h] = _attend(st["q"][a:z, h], k.float(), v.float(), lambda f, t: at <= ctx[b] + torch.arange(f, t, device=DEV)[:, None])
    return out


def _tree_exact(st):
    G, N = st["H"] // st["KVH"], st["N"]
    out = torch.empty(st["q"].shape, dtype=torch.float64, device=DEV)
    ctx, slots, parents = st["ctx"].tolist(), st["slots"].tolist(), st["parents"].tolist()
    for b in range(st["B"]):
        sees = torch.zeros(N, ctx[b] + N, dtype=torch.bool)
        sees[:, :ctx[b]] = True
        for i in range(N):
            j = i
            while j >= 0:
                sees[i, ctx[b] + j] = True
                j = parents[b][j]
        sees = sees.to(DEV)
        for h in range(st["H"]):
            k = torch.cat([st["k"][slots[b], h // G, :ctx[b]].float(), st["k_new"][b, :, h // G].float()])
            v = torch.cat([st["v"][slots[b], h // G, :ctx[b]].float(), st["v_new"][b, :, h // G].float()])
            out[b, :, h] = _attend(st["q"][b, :, h], k, v, lambda f, t: sees[f:t])
    return out


def _commit_exact(st):
    kv = st["kv"].double()
    parents, tokens, targets = st["parents"].tolist(), st["tokens"].tolist(), st["targets"].tolist()
    ctx, slots = st["ctx"].tolist(), st["slots"].tolist()
    counts, paths, nexts = [], [], []
    for b in range(st["B"]):
        path = [0]
        while True:
            below = [c for c in range(st["N"]) if parents[b][c] == path[-1] and tokens[b][c] == targets[b][path[-1]]]
            if not below:
                break
            path.append(below[0])
        kv[:, :, slots[b], :, ctx[b]:ctx[b] + len(path)] = st["kv_new"][:, :, b, path].transpose(2, 3).double()
        counts.append(len(path))
        paths.append(path + [-1] * (st["N"] - len(path)))
        nexts.append(targets[b][path[-1]])
    return kv, _i32(counts), _i32(paths), torch.tensor(nexts, device=DEV)


def _sample_exact(st):
    tokens = []
    for r in range(st["R"]):
        x, t = st["logits"][r].double(), st["temperature"][r].item()
        value, index = torch.sort(x, descending=True, stable=True)
        if t == 0:
            tokens.append(index[0].item())
            continue
        w = torch.exp(value / t - value[0] / t)
        if st["top_k"][r] > 0:
            w, index = w[:st["top_k"][r].item()], index[:st["top_k"][r].item()]
        if st["top_p"][r] < 1:
            less = torch.cat([w.new_zeros(1), w.cumsum(0)[:-1]])
            n = max(1, int((less < st["top_p"][r].double() * w.sum()).sum()))
            w, index = w[:n], index[:n]
        n = max(1, int((w >= st["min_p"][r].double()).sum()))
        w, index = w[:n], index[:n]
        index, o = torch.sort(index)
        c = w[o].cumsum(0)
        tokens.append(index[torch.searchsorted(c, st["u"][r].double() * c[-1], right=True).clamp_max(n - 1)].item())
    return torch.tensor(tokens, device=DEV)


_EXACT = {"prefill": _prefill_exact, "tree": _tree_exact, "commit": _commit_exact, "sample": _sample_exact}
