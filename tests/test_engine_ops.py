"""Serving operators of the engine (smg_amd/engine/ops.py) against plain forms in
64 bits, and their refusals."""
import math

import pytest

torch = pytest.importorskip("torch")
pytest.importorskip("smg_amd._core")

from smg_amd.engine import ops  # noqa: E402

DEV = "cuda:0"
BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn
HALF = torch.finfo(BF16).eps / 2  # a rounding to bf16 is off by at most this, relatively


def gen(seed=0, device=DEV):
    return torch.Generator(device=device).manual_seed(seed)


def randn(g, *shape, dtype=BF16, scale=1.0):
    return (torch.randn(*shape, generator=g, device=g.device) * scale).to(dtype)


def i32(v, device=DEV):
    return torch.tensor(v, dtype=torch.int32, device=device)


def attend(q, k, v, sees, scale=None):
    """softmax(scale q k^T) v of one head in 64 bits over the keys that each row sees
    (zeros where none), and the bound on the kernel's error: a half step of bf16 for
    every weight and one for the result.  The scores are sums of D products in f32,
    off by at most D 2^-24 of the sum of the products' sizes, twice that for a weight
    and its normalisation; 2^-10 of all covers that for |q . k| scale <= 60 at D = 128."""
    q, k, v = q.double(), k.double(), v.double()
    s = (q @ k.t().contiguous()) * (scale or 1 / math.sqrt(q.shape[1]))
    s = s.masked_fill(~sees, -math.inf)
    p = torch.exp(s - s.amax(1, keepdim=True).clamp_min(-1e300))
    p = p / p.sum(1, keepdim=True).clamp_min(1e-300)
    # a key that a row does not see takes no part, whatever it holds
    fin = torch.where(torch.isfinite(v), v, 0.0)
    o = p @ fin
    tol = (HALF + 2.0 ** -10) * (p @ fin.abs()) + HALF * o.abs() + 1e-30
    for x in (math.inf, -math.inf, math.nan):
        is_x = torch.isnan(v) if x != x else v == x
        o = torch.where((p > 0).double() @ is_x.double() > 0, o + x, o)
    return o, tol


def near(got, want, tol):
    got, fin = got.double(), torch.isfinite(want)
    assert ((got == want) | torch.isnan(got) & torch.isnan(want) | fin).all(), "not finite in other places"
    off = torch.where(fin, (got - want).abs() - tol, 0.0).nan_to_num(math.inf)
    assert off.max().item() <= 0, f"off by {off.max().item()} more than the roundings"


def prefill_case(lens, starts, H, KVH, D, fp8=False, T=None, seed=0, extra_slots=2):
    g = gen(seed)
    B, need = len(lens), max([a + b for a, b in zip(lens, starts)] + [1])
    T = T or need + 3
    S = B + extra_slots
    q = randn(g, sum(lens), H, D, scale=2.0)
    k, v = (randn(g, S, KVH, T, D, dtype=FP8 if fp8 else BF16) for _ in range(2))
    slots = torch.randperm(S, generator=g, device=DEV)[:B].to(torch.int32)
    cu = i32([sum(lens[:i]) for i in range(B + 1)])
    return q, k, v, slots, i32(starts), cu


def check_prefill(out, q, k, v, slots, starts, cu, scale=None):
    cu, starts, slots = cu.tolist(), starts.tolist(), slots.tolist()
    G = q.shape[1] // k.shape[1]
    for b, slot in enumerate(slots):
        a, z = cu[b], cu[b + 1]
        if z <= a:
            continue
        end = min(starts[b] + z - a, k.shape[2])
        at = torch.arange(end, device=DEV)
        sees = at <= starts[b] + torch.arange(z - a, device=DEV)[:, None]
        for h in range(q.shape[1]):
            near(out[a:z, h], *attend(q[a:z, h].float(), k[slot, h // G, :end].float(), v[slot, h // G, :end].float(), sees, scale))


@pytest.mark.gpu
class TestAttnPrefill:
    @pytest.mark.parametrize("D", [64, 128])
    @pytest.mark.parametrize("fp8", [False, True])
    @pytest.mark.parametrize("H,KVH", [(4, 4), (8, 2), (6, 2), (5, 1), (16, 1)])
    @pytest.mark.parametrize("lens,starts", [
        ([1], [0]), ([1, 1, 1], [0, 31, 64]), ([37, 1, 0, 130, 64], [0, 200, 7, 63, 1]), ([257], [0]),
    ])
    def test_matches_64_bits(self, D, fp8, H, KVH, lens, starts):
        args = prefill_case(lens, starts, H, KVH, D, fp8)
        check_prefill(ops.attn_prefill(*args), *args)

    @pytest.mark.parametrize("fp8", [False, True])
    @pytest.mark.parametrize("lens,starts,H,KVH,D", [
        ([3], [5000], 8, 2, 128), ([1, 40], [9000, 100], 4, 4, 64), ([17, 16, 2], [700, 2900, 0], 16, 4, 128),
        ([700], [1500], 4, 1, 128),
    ])
    def test_long_history_is_split(self, lens, starts, H, KVH, D, fp8):
        args = prefill_case(lens, starts, H, KVH, D, fp8, seed=1)
        check_prefill(ops.attn_prefill(*args), *args)
        # a bound that is too small costs time, not results
        check_prefill(ops.attn_prefill(*args, max_ctx=16), *args)

    def test_many_sequences(self):
        lens = [(i * 7) % 23 for i in range(150)]
        args = prefill_case(lens, [(i * 13) % 90 for i in range(150)], 8, 4, 64, seed=2)
        check_prefill(ops.attn_prefill(*args), *args)

    def test_strides_scale_and_out(self):
        lens, starts, H, KVH, D = [50, 9], [20, 70], 8, 2, 128
        q, k, v, slots, st, cu = prefill_case(lens, starts, H, KVH, D, seed=3)
        g = gen(4)
        qkv = randn(g, 59, (H + 2 * KVH) * D)  # q as a slice of a fused projection
        qs = qkv[:, :H * D].view(59, H, D)
        layers = randn(g, 3, 2, *k.shape)  # one layer of an arena
        kt = layers[1, 0].transpose(1, 2).contiguous().transpose(1, 2)  # positions before heads
        wide = torch.full((59, 2 * H, D), 7.0, dtype=BF16, device=DEV)
        out = wide[:, ::2]
        got = ops.attn_prefill(qs, kt, layers[1, 1], slots, st, cu, scale=0.03, out=out)
        assert got is out
        check_prefill(out, qs, kt, layers[1, 1], slots, st, cu, scale=0.03)
        assert (wide[:, 1::2] == 7).all()

    @pytest.mark.parametrize("lens,starts", [([70, 1, 9], [0, 30, 500]), ([3], [6000])])
    @pytest.mark.parametrize("fp8", [False, True])
    def test_out_may_be_q(self, lens, starts, fp8):
        q, *rest = prefill_case(lens, starts, 8, 2, 128, fp8, seed=9)
        want = ops.attn_prefill(q, *rest)
        assert ops.attn_prefill(q, *rest, out=q) is q and torch.equal(q, want)

    def test_rows_behind_the_last_sequence_stay(self):
        for starts in ([3, 5], [3, 4000]):  # without and with a split
            q, k, v, slots, st, cu = prefill_case([30, 10], starts, 4, 2, 128, seed=5)
            q = torch.cat([q, q])
            out = torch.full_like(q, 3.0)
            ops.attn_prefill(q, k, v, slots, st, cu, out=out)
            check_prefill(out, q, k, v, slots, st, cu)
            assert (out[40:] == 3).all()
            none = ops.attn_prefill(q, k, v, slots, st, torch.zeros_like(cu), out=torch.full_like(q, 3.0))
            assert (none == 3).all()

    def test_padding_slots_give_zeros(self):
        for starts in ([0, 40, 9], [0, 4000, 9]):
            q, k, v, slots, st, cu = prefill_case([20, 33, 5], starts, 4, 2, 128, seed=6)
            bad = slots.clone()
            bad[0], bad[2] = -1, k.shape[0]
            out = ops.attn_prefill(q, k, v, bad, st, cu)
            assert (out[:20] == 0).all() and (out[53:] == 0).all()
            check_prefill(out[20:53], q[20:53], k, v, slots[1:2], st[1:2], i32([0, 33]))

    def test_lengths_past_the_cache_are_cut(self):
        q, k, v, slots, st, cu = prefill_case([40], [100], 4, 4, 64, T=120, seed=7)
        out = ops.attn_prefill(q, k, v, slots, st, cu)
        at = torch.arange(120, device=DEV)
        for h in range(4):
            sees = at <= (100 + torch.arange(40, device=DEV))[:, None]
            near(out[:, h], *attend(q[:, h].float(), k[slots[0].item(), h].float(), v[slots[0].item(), h].float(), sees))
        # before the cache: nothing to see until its first row
        out = ops.attn_prefill(q, k, v, slots, i32([-25]), cu)
        assert (out[:25] == 0).all()
        for h in range(4):
            sees = at <= (torch.arange(15, device=DEV))[:, None]
            near(out[25:, h], *attend(q[25:, h].float(), k[slots[0].item(), h].float(), v[slots[0].item(), h].float(), sees))

    @pytest.mark.parametrize("lens,starts", [([40, 21], [9, 64]), ([5, 3], [4000, 3000])])
    def test_what_a_row_does_not_see_does_not_reach_it(self, lens, starts):
        q, k, v, slots, st, cu = prefill_case(lens, starts, 8, 2, 128, T=4100, seed=8)
        for b, slot in enumerate(slots.tolist()):
            end = starts[b] + lens[b]
            for t in (k, v):
                t[slot, :, end:] = math.nan
            v[slot, 0, end - 1, 5] = math.inf  # the last token alone sees it
            v[slot, 1, end - 2, 70] = math.nan
            k[slot, 1, end - 1] = -math.inf
        keep = torch.ones(q.shape[0], dtype=torch.bool)
        for b in range(2):
            keep[cu[b + 1] - 1] = False
        out = ops.attn_prefill(q, k, v, slots, st, cu)
        k2 = k.clone()
        for b, slot in enumerate(slots.tolist()):
            k2[slot, 1, starts[b] + lens[b] - 1] = 0
        ref = [ops.attn_prefill(q, k2, v, slots, st, cu)]
        assert torch.equal(out[keep].view(torch.int16), ref[0][keep].view(torch.int16))
        check_prefill(ref[0], q, k2, v, slots, st, cu)

    def test_far_slots_pass_32_bits(self):
        # the last slot starts past 2^32 bytes and 2^31 elements
        S, KVH, T, D = 9, 4, 1 << 19, 128
        k = torch.empty(S, KVH, T, D, dtype=BF16, device=DEV)
        g = gen(9)
        k[S - 1, 3, T - 300:] = randn(g, 300, D)
        k[S - 1, :, :300] = randn(g, 4, 300, D)
        q = randn(g, 4, 8, D)
        at = i32([296])
        out = ops.attn_prefill(q, k, k, i32([S - 1]), at, i32([0, 4]))
        check_prefill(out, q, k, k, i32([S - 1]), at, i32([0, 4]))

    def test_captured(self):
        args = prefill_case([3, 70], [1000, 0], 8, 2, 128, seed=10)
        q = args[0]
        replays(lambda: ops.attn_prefill(*args), q)


def replays(call, changing, times=3):
    """call(), captured, replayed on new contents of `changing` between eager calls."""
    outs = lambda r: list(r) if isinstance(r, (tuple, list)) else [r]  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = outs(call())
    for i in range(times):
        fresh = randn(gen(100 + i), *changing.shape, dtype=changing.dtype) if changing.dtype == BF16 else torch.rand(changing.shape, generator=gen(100 + i), device=DEV)
        changing.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, outs(call())):
            assert torch.equal(a, b)


def trees(g, B, N):
    i = torch.arange(N, device=DEV).expand(B, N)
    back = 1 + torch.randint(0, 5, (B, N), generator=g, device=DEV)
    return torch.where(i == 0, -1, (i - back).clamp_min(-1)).to(torch.int32)


def tree_case(B, N, ctx, H, KVH, D, fp8=False, T=None, seed=0):
    g = gen(seed)
    T = T or max(ctx) + 2
    q = randn(g, B, N, H, D, scale=2.0)
    kn, vn = (randn(g, B, N, KVH, D) for _ in range(2))
    k, v = (randn(g, B + 2, KVH, T, D, dtype=FP8 if fp8 else BF16) for _ in range(2))
    slots = torch.randperm(B + 2, generator=g, device=DEV)[:B].to(torch.int32)
    return [q, kn, vn, k, v, slots, i32(ctx), trees(g, B, N)]


def seen_nodes(parents):
    """Ancestors and self of every node of one tree, nothing for padding."""
    N = len(parents)
    m = torch.zeros(N, N, dtype=torch.bool)
    for i in range(N):
        at, up = i, []
        while at >= 0:
            up.append(at)
            at = parents[at] if -1 <= parents[at] < at else -2
        if at == -1:
            m[i, up] = True
    return m


def check_tree(out, q, kn, vn, k, v, slots, ctx, parents, scale=None):
    G = q.shape[2] // k.shape[1]
    for b, slot in enumerate(slots.tolist()):
        n = max(0, min(ctx[b].item(), k.shape[2]))
        m = seen_nodes(parents[b].tolist())
        sees = torch.cat([m.any(1, keepdim=True).expand(-1, n), m], 1).to(DEV)
        for h in range(q.shape[2]):
            kk = torch.cat([k[slot, h // G, :n].float(), kn[b, :, h // G].float()])
            vv = torch.cat([v[slot, h // G, :n].float(), vn[b, :, h // G].float()])
            near(out[b, :, h], *attend(q[b, :, h].float(), kk, vv, sees, scale))


@pytest.mark.gpu
class TestAttnTree:
    @pytest.mark.parametrize("D", [64, 128])
    @pytest.mark.parametrize("fp8", [False, True])
    @pytest.mark.parametrize("H,KVH", [(4, 4), (8, 2), (3, 1), (16, 2)])
    @pytest.mark.parametrize("N,ctx", [(1, [0]), (1, [77]), (5, [0, 1, 64]), (17, [63, 300]), (64, [65, 5])])
    def test_matches_64_bits(self, D, fp8, H, KVH, N, ctx):
        args = tree_case(len(ctx), N, ctx, H, KVH, D, fp8)
        check_tree(ops.attn_tree(*args), *args)

    @pytest.mark.parametrize("fp8", [False, True])
    @pytest.mark.parametrize("B,N,ctx,H,KVH,D", [
        (1, 7, [9000], 8, 2, 128), (2, 61, [5000, 0], 16, 4, 128), (1, 3, [20000], 4, 4, 64),
    ])
    def test_long_context_is_split(self, B, N, ctx, H, KVH, D, fp8):
        args = tree_case(B, N, ctx, H, KVH, D, fp8, seed=1)
        check_tree(ops.attn_tree(*args), *args)
        check_tree(ops.attn_tree(*args, max_ctx=64), *args)

    def test_padding_nodes_and_slots(self):
        for ctx in ([50, 0, 129], [5000, 0, 129]):
            args = tree_case(3, 12, ctx, 8, 2, 128, seed=2)
            parents = args[-1]
            parents[0, 4] = -2
            parents[0, 9] = 4   # below padding
            parents[1, 3] = 3   # its own parent
            parents[1, 5] = 11  # a later node
            parents[2, :] = -2
            out = ops.attn_tree(*args)
            check_tree(out, *args)
            assert (out[0, 4] == 0).all() and (out[2] == 0).all()
            slots = args[5].clone()
            slots[0], slots[1] = -3, 1 << 20
            out2 = ops.attn_tree(*args[:5], slots, *args[6:])
            assert (out2[:2] == 0).all() and torch.equal(out2[2], out[2])

    def test_context_past_the_cache_is_cut(self):
        args = tree_case(2, 6, [40, 10], 4, 4, 64, T=48, seed=3)
        args[6] = i32([1 << 30, -5])
        check_tree(ops.attn_tree(*args), *args)

    def test_strides(self):
        args = tree_case(2, 9, [70, 33], 8, 2, 128, seed=4)
        g = gen(5)
        args[0] = randn(g, 9, 2, 12, 128).transpose(0, 1)[:, :, 2:10]
        args[1] = randn(g, 2, 2, 9, 128).transpose(1, 2)
        args[3] = args[3].transpose(1, 2).contiguous().transpose(1, 2)
        out = torch.full((2, 9, 16, 128), 7.0, dtype=BF16, device=DEV)
        ops.attn_tree(*args, scale=0.05, out=out[:, :, 8:])
        check_tree(out[:, :, 8:], *args, scale=0.05)
        assert (out[:, :, :8] == 7).all()

    def test_what_a_node_does_not_see_does_not_reach_it(self):
        for ctx in ([100, 64], [5000, 64]):
            q, kn, vn, k, v, slots, st, parents = args = tree_case(2, 20, ctx, 8, 4, 128, T=5050, seed=6)
            parents[:, 1:] = 0
            for b, slot in enumerate(slots.tolist()):
                for t in (k, v):
                    t[slot, :, ctx[b]:] = math.nan
            vn[:, 7, 2, 9] = math.inf
            vn[:, 12, 0] = math.nan
            check_tree(ops.attn_tree(*args), *args)
            kn[:, 12] = math.nan
            out = ops.attn_tree(*args)
            others = [i for i in range(20) if i != 12]
            kn[:, 12] = 0
            ref = ops.attn_tree(*args)
            assert torch.equal(out[:, others].view(torch.int16), ref[:, others].view(torch.int16))

    def test_captured(self):
        args = tree_case(2, 13, [3000, 20], 8, 2, 128, seed=7)
        replays(lambda: ops.attn_tree(*args), args[0])


def commit_case(B, N, KVH, D, L=2, T=90, fp8=False, seed=0, room=None):
    g = gen(seed)
    kv_new = randn(g, L, 2, B, N, KVH, D, scale=3.0)
    kv = randn(g, L, 2, B + 2, KVH, T, D, dtype=FP8 if fp8 else BF16)
    slots = torch.randperm(B + 2, generator=g, device=DEV)[:B].to(torch.int32)
    ctx = torch.randint(0, T - N + 1, (B,), generator=g, device=DEV).to(torch.int32)
    parents = trees(g, B, N)
    tokens = torch.randint(0, 3, (B, N), generator=g, device=DEV)  # siblings often share a token
    targets = torch.randint(0, 3, (B, N), generator=g, device=DEV)
    return [kv_new, kv, slots, ctx, parents, tokens, targets]


def commit_plain(kv_new, kv, slots, ctx, parents, tokens, targets):
    kv = kv.clone()
    S, T = kv.shape[2], kv.shape[4]
    B, N = parents.shape
    real = [0 <= c < T and up == -1 for c, up in zip(ctx.tolist(), parents[:, 0].tolist())]
    count, path, nxt = [], [], []
    for b in range(B):
        p, tk, tg = parents[b].tolist(), tokens[b].tolist(), targets[b].tolist()
        slot, at = slots[b].item(), ctx[b].item()
        taken = []
        if 0 <= slot < S and real[b]:
            taken = [0]
            while len(taken) < T - at:
                below = [c for c in range(taken[-1] + 1, N) if p[c] == taken[-1] and tk[c] == tg[taken[-1]]]
                if not below:
                    break
                taken.append(below[0])
            if not any(r and s == slot for r, s in zip(real[b + 1:], slots[b + 1:].tolist())):
                kv[:, :, slot, :, at:at + len(taken)] = kv_new[:, :, b, taken].transpose(2, 3).to(kv.dtype)
        count.append(len(taken))
        path.append(taken + [-1] * (N - len(taken)))
        nxt.append(tg[taken[-1]] if taken else -1)
    return kv, count, path, nxt


def check_commit(args):
    want, count, path, nxt = commit_plain(*args)
    got = ops.tree_commit(*args)
    assert got[0].tolist() == count and got[1].tolist() == path and got[2].tolist() == nxt
    view = torch.uint8 if want.dtype == FP8 else torch.int16
    assert torch.equal(args[1].view(view), want.view(view))
    return count


# every way in which attention is cut, whatever the rule would take: waves along the rows
# and along the keys, 8 bits
SHAPES = [(1, 4, False), (2, 2, False), (2, 4, False), (4, 1, False), (2, 2, True), (4, 2, True), (8, 1, True)]


@pytest.mark.gpu
class TestAttnShapes:
    @pytest.mark.parametrize("D", [64, 128])
    @pytest.mark.parametrize("runs", [1, 5, 64])
    @pytest.mark.parametrize("wr,wk,fp8", SHAPES)
    def test_prefill(self, monkeypatch, wr, wk, fp8, runs, D):
        monkeypatch.setattr(ops, "_shape", lambda *a: (wr, wk, runs))
        args = prefill_case([1, 300, 0, 77, 130], [2100, 0, 50, 700, 3], 6, 2, D, fp8, seed=11)
        check_prefill(ops.attn_prefill(*args), *args)

    @pytest.mark.parametrize("D", [64, 128])
    @pytest.mark.parametrize("runs", [1, 5, 64])
    @pytest.mark.parametrize("wr,wk,fp8", SHAPES)
    def test_tree(self, monkeypatch, wr, wk, fp8, runs, D):
        monkeypatch.setattr(ops, "_shape", lambda *a: (wr, wk, runs))
        args = tree_case(4, 39, [0, 1500, 64, 333], 6, 2, D, fp8, seed=12)
        check_tree(ops.attn_tree(*args), *args)


class TestWorkspace:
    @pytest.mark.parametrize("N,H,KVH,T,fp8,most", [
        (2000, 16, 16, 131072, True, 256 * 256), (1000, 16, 16, 65536, False, 512 * 128), (900, 16, 4, 65536, False, 512 * 128),
        (1, 8, 2, 1 << 20, True, 64 * 8),
    ])
    def test_size_goes_by_what_the_card_takes(self, monkeypatch, N, H, KVH, T, fp8, most):
        """At most `most` rows of partial results, each of 128 values and its maximum and sum."""
        sizes = []
        monkeypatch.setattr(ops, "_on_gpu", lambda *a, **k: None)
        monkeypatch.setattr(ops, "_launch", lambda *a, **k: None)
        empty = torch.empty
        monkeypatch.setattr(torch, "empty", lambda *a, **k: sizes.append(a[0]) or empty(0))
        cache = torch.zeros(1, 1, 1, 128, dtype=FP8 if fp8 else BF16).expand(1, KVH, T, 128)
        one, new = torch.zeros(1, dtype=torch.int32), min(N, 64)
        ops.attn_prefill(torch.zeros(N, H, 128, dtype=BF16), cache, cache, one, one, torch.tensor([0, N], dtype=torch.int32))
        kn = torch.zeros(1, new, KVH, 128, dtype=BF16)
        ops.attn_tree(torch.zeros(1, new, H, 128, dtype=BF16), kn, kn, cache, cache, one, one, torch.zeros(1, new, dtype=torch.int32))
        assert len(sizes) == 2 and 0 < max(sizes) <= most * 130

    @pytest.mark.gpu
    @pytest.mark.parametrize("wr,wk,fp8", SHAPES)
    def test_calls_stay_in_it(self, monkeypatch, wr, wk, fp8):
        held = []

        def parts(q, *shape):
            n = ops._core.attn_part_floats(*shape)
            held.append(torch.full((n + 2048,), 7.0, device=DEV))
            return held[-1][1024:-1024]

        monkeypatch.setattr(ops, "_shape", lambda *a: (wr, wk, 64))
        monkeypatch.setattr(ops, "_parts", parts)
        # more sequences than lanes, some of them empty or padding, few of them long
        lens = [(i * 7) % 23 for i in range(150)]
        args = prefill_case(lens, [(3000 if i % 40 == 39 else i) for i in range(150)], 8, 4, 128, fp8, seed=2)
        args[3][70] = -1
        out = ops.attn_prefill(*args, out=torch.zeros_like(args[0]))
        cu = args[5].tolist()
        assert (out[cu[70]:cu[71]] == 0).all()
        for b in (39, 64, 69, 71, 79, 149):
            part = [args[0][cu[b]:cu[b + 1]], args[1], args[2], args[3][b:b + 1], args[4][b:b + 1], i32([0, lens[b]])]
            check_prefill(out[cu[b]:cu[b + 1]], *part)
        args = tree_case(70, 9, [(4000 if i % 33 == 32 else i) for i in range(70)], 4, 2, 128, fp8, seed=3)
        out = ops.attn_tree(*args)
        pick = [0, 32, 63, 64, 65, 69]
        check_tree(out[pick], *(t[pick] for t in args[:3]), *args[3:5], *(t[pick] for t in args[5:]))
        for t in held:
            assert (t[:1024] == 7).all() and (t[-1024:] == 7).all() and (t[1024:-1024] != 7).any()


@pytest.mark.gpu
class TestTreeCommit:
    @pytest.mark.parametrize("fp8", [False, True])
    @pytest.mark.parametrize("B,N,KVH,D,L", [(1, 1, 1, 64, 1), (3, 5, 4, 64, 2), (9, 33, 3, 128, 5), (70, 64, 2, 128, 2), (2, 8, 1, 8, 3)])
    def test_matches_plain(self, B, N, KVH, D, L, fp8):
        count = check_commit(commit_case(B, N, KVH, D, L, fp8=fp8))
        assert N < 64 or max(count) >= 3

    def test_whole_chain(self):
        args = commit_case(2, 64, 2, 64, T=200, seed=1)
        args[4] = (torch.arange(64, device=DEV) - 1).expand(2, 64).to(torch.int32).contiguous()
        args[5] = torch.arange(64, device=DEV).expand(2, 64).contiguous() + (1 << 40)
        args[6] = args[5] + 1
        assert check_commit(args) == [64, 64]

    def test_tokens_differ_in_their_high_bits(self):
        args = commit_case(1, 2, 1, 64, seed=2)
        args[4] = i32([[-1, 0]])
        args[5] = torch.tensor([[0, 5 + (1 << 33)]], device=DEV)
        args[6] = torch.tensor([[5, 6]], device=DEV)
        assert check_commit(args) == [1]

    def test_padding_and_no_room(self):
        args = commit_case(6, 9, 2, 64, T=30, seed=3)
        args[2] = i32([0, -1, 2, 8, 4, 5])  # slots 0..7 exist
        args[3] = i32([29, 3, 30, 0, -1, 27])
        args[4][:, :] = torch.arange(9, device=DEV) - 1
        args[5].fill_(1)
        args[6].fill_(1)
        assert check_commit(args) == [1, 0, 0, 0, 0, 3]
        args = commit_case(2, 4, 1, 64, seed=4)
        args[4][0, 0] = -2
        assert check_commit(args)[0] == 0

    def test_padding_may_name_a_used_slot(self):
        args = commit_case(5, 6, 2, 64, T=40, seed=9)
        args[2] = i32([3, 3, 3, 3, 3])  # one real entry, and three kinds of padding behind it
        args[3] = i32([2, 7, 40, -1, 9])
        args[4][4, 0] = -2
        assert check_commit(args)[2:] == [0, 0, 0]

    def test_same_slot_twice(self):
        args = commit_case(70, 6, 2, 64, seed=5)
        args[2][3] = args[2][66]
        args[2][10] = args[2][11]
        check_commit(args)

    def test_strides(self):
        args = commit_case(3, 7, 4, 128, L=3, seed=6)
        args[0] = args[0].permute(2, 0, 3, 1, 4, 5).contiguous().permute(1, 3, 0, 2, 4, 5)
        args[1] = args[1].permute(2, 0, 1, 4, 3, 5).contiguous().permute(1, 2, 0, 4, 3, 5)
        check_commit(args)

    def test_8_bit_rounding(self):
        # every bf16 value, to the nearest e4m3 as torch rounds it
        bits = torch.arange(1 << 16, device=DEV, dtype=torch.int32).to(torch.int16).view(BF16)
        args = commit_case(64, 1, 8, 128, L=1, T=8, fp8=True, seed=7)
        args[0] = bits[:, None].expand(-1, 2).t().reshape(2, 64, 1, 8, 128)[None].contiguous()
        args[4].fill_(-1)
        want = commit_plain(*args)[0]
        ops.tree_commit(*args)
        a, b = args[1].float(), want.float()
        assert torch.equal(torch.isnan(a), torch.isnan(b))
        assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))

    def test_captured(self):
        args = commit_case(3, 9, 2, 64, seed=8)
        replays(lambda: (*ops.tree_commit(*args), args[1].view(torch.int16).clone()), args[0])


def sample_plain(x, u, t, k=0, p=1.0, m=0.0):
    """One row in 64 bits, its weights multiples of 2^-S as documented."""
    V = len(x)
    x = x.double().cpu()
    x = torch.where(torch.isnan(x), -math.inf, x)
    if x.max() == -math.inf:
        return -1
    value, index = torch.sort(x, descending=True, stable=True)
    if not t > 0:
        return index[0].item()
    if value[0] == math.inf:
        w = (value == math.inf).double()
    else:
        w = torch.exp((value - value[0]) / t)
        w[value == -math.inf] = 0
    n = max(1, int((w >= min(m, 1.0)).sum())) if m > 0 else V
    unit = 2.0 ** min(50, 62 - (V - 1).bit_length())
    w = torch.floor(w * unit + 0.5) / unit
    if k > 0:
        w, index = w[:k], index[:k]
    if p < 1:
        before = torch.cat([w.new_zeros(1), w.cumsum(0)[:-1]])
        cut = max(1, int((before < p * w.sum()).sum()))
        w, index = w[:cut], index[:cut]
    w, index = w[:n], index[:n]
    index, o = torch.sort(index)
    c = w[o].cumsum(0)
    at = int((c <= u * c[-1]).sum())
    if at >= len(c):  # u is 1 or more: the last token with a weight
        at = int((w[o] > 0).nonzero()[-1])
    return index[at].item()


def check_sample(x, u, t, k=None, p=None, m=None):
    R = x.shape[0]
    f = lambda v, d: torch.tensor(v if isinstance(v, list) else [v] * R, dtype=d, device=DEV)  # noqa: E731
    tu, tt = f(u, torch.float32), f(t, torch.float32)
    kw = dict(top_k=None if k is None else f(k, torch.int32), top_p=None if p is None else f(p, torch.float32),
              min_p=None if m is None else f(m, torch.float32))
    got = ops.sample(x, tu, tt, **kw).tolist()
    want = [sample_plain(x[r], tu[r].item(), tt[r].item(), 0 if k is None else kw["top_k"][r].item(),
                         1.0 if p is None else kw["top_p"][r].item(), 0.0 if m is None else kw["min_p"][r].item())
            for r in range(R)]
    assert got == want
    return got


US = [0.0, 1e-30, 0.11, 0.25, 0.37, 0.5, 0.73, 0.9, 0.99999994]


@pytest.mark.gpu
class TestSample:
    @pytest.mark.parametrize("f32", [False, True])
    @pytest.mark.parametrize("V", [1, 2, 63, 64, 1000, 2048, 16385, 32768, 131071])
    @pytest.mark.parametrize("k,p,m", [(None, None, None), (40, None, None), (None, 0.9, None), (None, None, 0.02),
                                       (500, 0.95, 0.01), (1, 0.5, 0.5)])
    def test_matches_64_bits(self, V, f32, k, p, m):
        g = gen(V)
        x = randn(g, len(US), V, dtype=torch.float32 if f32 else BF16, scale=2.0)
        check_sample(x, US, [1.0, 0.6, 1.4, 0.0, 1.0, 0.8, 2.0, 0.3, 1.0], k, p, m)

    @pytest.mark.parametrize("R,V", [(300, 5000), (60, 70001), (128, 65536), (129, 65536)])
    def test_mixed_rows(self, R, V):
        g = gen(1)
        x = randn(g, R, V, scale=3.0)
        x[R // 2] = -math.inf
        x[R // 3, V // 2:] = -math.inf
        x[R // 4, 3] = x[R // 4, V - 1] = math.inf
        pick = lambda *v: [v[i] for i in torch.randint(0, len(v), (R,), generator=g, device=DEV).tolist()]  # noqa: E731
        check_sample(x, torch.rand(R, generator=g, device=DEV).tolist(), pick(0.0, 0.5, 1.0, 1.5), pick(0, 1, 7, 300, 9000),
                     pick(0.0, 0.1, 0.9, 0.99, 1.0), pick(0.0, 0.001, 0.1, 1.0))

    @pytest.mark.parametrize("V", [5, 700, 32768])
    def test_equal_logits_go_by_index(self, V):
        x = torch.full((len(US), V), 1.5, dtype=BF16, device=DEV)
        check_sample(x, US, 1.0)
        check_sample(x, US, 0.0)
        check_sample(x, US, 0.7, k=max(1, V // 3))
        check_sample(x, US, 0.7, p=0.5)
        check_sample(x, US, 1.0, k=max(2, V // 2), p=0.3, m=1.0)
        x[:, ::2] = 2.0
        check_sample(x, US, 1.0, k=V // 2 + 2, p=0.97)

    def test_zeros_of_both_signs_are_equal(self):
        x = torch.zeros(len(US), 10, dtype=torch.float32, device=DEV)
        x[:, ::3] = -0.0
        check_sample(x, US, 0.0)
        check_sample(x, US, 1.0, k=4)

    @pytest.mark.parametrize("V", [9, 3000])
    def test_masked_and_odd_logits(self, V):
        g = gen(2)
        x = randn(g, len(US), V, dtype=torch.float32, scale=2.0)
        x[torch.rand(x.shape, generator=g, device=DEV) < 0.5] = -math.inf
        x[:, 3] = math.nan
        x[1] = -math.inf
        x[2] = math.nan
        x[3, 5:8] = math.inf
        x[4] = -math.inf
        x[4, V - 1] = -3e38
        for t in (0.0, 1.0):
            got = check_sample(x, US, t)
            assert got[1] == got[2] == -1 and got[4] == V - 1
            check_sample(x, US, t, k=3, p=0.9, m=0.1)
        check_sample(x.to(BF16), US, 1.0, k=V, p=0.99)

    def test_ends_of_the_settings(self):
        g = gen(3)
        x = randn(g, len(US), 4000, dtype=torch.float32)
        check_sample(x, US, 1e-40)
        check_sample(x, US, 1e-3)
        check_sample(x, US, math.inf)
        check_sample(x, US, math.inf, k=50, p=0.5)
        check_sample(x, US, -1.0)
        check_sample(x, US, math.nan)
        check_sample(x, US, 1.0, k=[-5, 0, 1, 2, 3999, 4000, 4001, 2 ** 31 - 1, 10])
        check_sample(x, US, 1.0, p=[0.0, -1.0, 1e-30, 0.5, 0.999999, 1.0, 2.0, 1e-3, 0.99])
        check_sample(x, US, 1.0, m=[0.0, -1.0, 1.0, 2.0, 1e-30, 0.999, 0.5, 0.3, 0.1])
        check_sample(x, [0.0, -1.0, 1.0, 2.0, 1e30, 0.5, 0.1, 0.2, 0.3], 1.0, k=100)

    def test_far_off_logits(self):
        # one value far below or above, as masks of the type's lowest value leave them
        for V in (900, 40000):
            x = randn(gen(7), len(US), V, dtype=torch.float32, scale=2.0)
            x[:, 5] = -3.4e38
            check_sample(x, US, math.inf, k=V // 2, p=0.7)
            check_sample(x, US, 80.0, k=V - 2, p=0.7)
            x[:, ::3] = torch.finfo(torch.float32).min
            check_sample(x, US, 1.0, k=V // 2, p=0.9, m=0.01)
            x[:, 11] = 3.4e38
            check_sample(x, US, math.inf, k=9, p=0.7)
            check_sample(x, US, 1.0, k=9, p=0.7)
        # from one end of the type to the other, at temperatures that leave all a weight
        x = (torch.rand(len(US), 5000, generator=gen(9), device=DEV) - 0.5) * 6.8e38
        assert (x.amax(1) - x.amin(1)).isinf().all()
        for t in (3e38, math.inf):
            check_sample(x, US, t, k=4000, p=0.7)
            check_sample(x, US, t, p=0.999)
        x = randn(gen(8), len(US), 5000, dtype=torch.float32, scale=1e-42)  # denormals
        check_sample(x, US, 1.0, k=100, p=0.5)

    def test_many_values_within_one_step(self):
        x = randn(gen(9), len(US), 30000, dtype=torch.float32, scale=1e-4)
        x[:, 0] = 30.0
        check_sample(x, US, 1.0, k=10000)
        check_sample(x, US, 40.0, k=20000, p=0.6)

    def test_largest_vocabulary(self):
        x = randn(gen(10), 3, 1 << 20, scale=2.0)
        check_sample(x, [0.3, 0.6, 0.999], 1.0, k=[0, 70000, 0], p=[1.0, 0.9, 0.95])

    def test_strides(self):
        g = gen(4)
        wide = randn(g, len(US), 5003)
        check_sample(wide[:, 1:3002], US, 1.0, p=0.9)
        check_sample(wide[::2, 3:5003], US[:5], 1.0, k=99)
        check_sample(wide[:1].expand(len(US), -1), US, 1.0, p=0.95)

    def test_same_answer_every_time(self):
        g = gen(5)
        x = randn(g, 64, 30000, scale=2.0)
        u, t = torch.rand(64, generator=g, device=DEV), torch.ones(64, device=DEV)
        p = torch.full((64,), 0.97, device=DEV)
        first = ops.sample(x, u, t, top_p=p)
        for _ in range(3):
            assert torch.equal(first, ops.sample(x, u, t, top_p=p))

    def test_captured(self):
        g = gen(6)
        x = randn(g, 20, 3000, scale=2.0)
        u, t, p = torch.rand(20, generator=g, device=DEV), torch.ones(20, device=DEV), torch.full((20,), 0.9, device=DEV)
        replays(lambda: ops.sample(x, u, t, top_p=p), x)

    def test_captured_with_shared_rows(self):
        g = gen(10)
        x = randn(g, 3, 70000, scale=2.0)
        u, t, p = torch.rand(3, generator=g, device=DEV), torch.ones(3, device=DEV), torch.full((3,), 0.9, device=DEV)
        replays(lambda: ops.sample(x, u, t, top_p=p), x)

    @pytest.mark.parametrize("R,V", [(300, 3000), (2, 9000), (257, 9001)])
    def test_threads_a_row(self, R, V):
        # more rows than compute units, short rows, long ones
        x = randn(gen(11), R, V, dtype=torch.float32, scale=2.0)
        n = len(US)
        check_sample(x, (US * R)[:R], [(0.0, 1.0, 0.7)[i % 3] for i in range(R)], k=[(0, 50, 1000, V)[i // n % 4] for i in range(R)],
                     p=[(1.0, 0.9)[i % 2] for i in range(R)])


class TestRefusals:
    """Refused on the host, before anything is launched: on CPU tensors."""

    def prefill(self, **kw):
        a = dict(q=torch.zeros(6, 4, 64, dtype=BF16), k=torch.zeros(2, 2, 16, 64, dtype=BF16), v=torch.zeros(2, 2, 16, 64, dtype=BF16),
                 slots=torch.zeros(2, dtype=torch.int32), starts=torch.zeros(2, dtype=torch.int32),
                 cu=torch.tensor([0, 3, 6], dtype=torch.int32))
        extra = {k: kw.pop(k) for k in ("scale", "out") if k in kw}
        a.update(kw)
        return ops.attn_prefill(*a.values(), **extra)

    def tree(self, **kw):
        a = dict(q=torch.zeros(2, 3, 4, 64, dtype=BF16), kn=torch.zeros(2, 3, 2, 64, dtype=BF16), vn=torch.zeros(2, 3, 2, 64, dtype=BF16),
                 k=torch.zeros(2, 2, 16, 64, dtype=BF16), v=torch.zeros(2, 2, 16, 64, dtype=BF16),
                 slots=torch.zeros(2, dtype=torch.int32), ctx=torch.zeros(2, dtype=torch.int32),
                 parents=torch.full((2, 3), -1, dtype=torch.int32))
        a.update(kw)
        return ops.attn_tree(*a.values())

    def commit(self, **kw):
        a = dict(kn=torch.zeros(1, 2, 2, 3, 2, 64, dtype=BF16), kv=torch.zeros(1, 2, 4, 2, 16, 64, dtype=BF16),
                 slots=torch.zeros(2, dtype=torch.int32), ctx=torch.zeros(2, dtype=torch.int32),
                 parents=torch.full((2, 3), -1, dtype=torch.int32), tokens=torch.zeros(2, 3, dtype=torch.int64),
                 targets=torch.zeros(2, 3, dtype=torch.int64))
        a.update(kw)
        return ops.tree_commit(*a.values())

    def sample(self, **kw):
        a = dict(logits=torch.zeros(2, 9), u=torch.zeros(2), temperature=torch.ones(2))
        a.update(kw)
        return ops.sample(a.pop("logits"), a.pop("u"), a.pop("temperature"), **a)

    @pytest.mark.parametrize("call", ["prefill", "tree", "commit", "sample"])
    def test_cpu_tensors(self, call):
        with pytest.raises(RuntimeError, match="CUDA/HIP"):
            getattr(self, call)()

    @pytest.mark.parametrize("call,kw,error", [
        ("prefill", dict(q=torch.zeros(6, 4, 64)), TypeError),
        ("prefill", dict(q=torch.zeros(6, 256, dtype=BF16)), ValueError),
        ("prefill", dict(q=torch.zeros(6, 3, 64, dtype=BF16)), ValueError),
        ("prefill", dict(q=torch.zeros(6, 4, 128, dtype=BF16)), ValueError),
        ("prefill", dict(q=torch.zeros(6, 4, 128, dtype=BF16)[..., ::2]), ValueError),
        ("prefill", dict(q=torch.zeros(6, 4, 68, dtype=BF16)[..., :64]), ValueError),
        ("prefill", dict(q=torch.zeros(6 * 4 * 64 + 4, dtype=BF16)[4:].view(6, 4, 64)), ValueError),
        ("prefill", dict(q=[1, 2]), TypeError),
        ("prefill", dict(k=torch.zeros(2, 2, 17, 64, dtype=BF16)), ValueError),
        ("prefill", dict(k=torch.zeros(2, 2, 16, 64, dtype=torch.float16)), TypeError),
        ("prefill", dict(k=torch.zeros(2, 2, 16, 64, dtype=FP8)), ValueError),
        ("prefill", dict(slots=torch.zeros(2)), TypeError),
        ("prefill", dict(slots=torch.zeros(2, dtype=torch.int64)), TypeError),
        ("prefill", dict(slots=torch.zeros(4, dtype=torch.int32)[::2]), ValueError),
        ("prefill", dict(starts=torch.zeros(3, dtype=torch.int32)), ValueError),
        ("prefill", dict(cu=torch.zeros(2, dtype=torch.int32)), ValueError),
        ("prefill", dict(scale=0.0), ValueError),
        ("prefill", dict(scale=-1.0), ValueError),
        ("prefill", dict(scale=math.nan), ValueError),
        ("prefill", dict(out=torch.zeros(6, 4, 32, dtype=BF16)), ValueError),
        ("prefill", dict(out=torch.zeros(6, 4, 64)), TypeError),
        ("tree", dict(q=torch.zeros(2, 65, 4, 64, dtype=BF16)), ValueError),
        ("tree", dict(q=torch.zeros(2, 65, 4, 64, dtype=BF16), kn=torch.zeros(2, 65, 2, 64, dtype=BF16),
                      vn=torch.zeros(2, 65, 2, 64, dtype=BF16), parents=torch.zeros(2, 65, dtype=torch.int32)), ValueError),
        ("tree", dict(kn=torch.zeros(2, 3, 4, 64, dtype=BF16)), ValueError),
        ("tree", dict(vn=torch.zeros(2, 3, 2, 64, dtype=FP8)), TypeError),
        ("tree", dict(parents=torch.zeros(2, 4, dtype=torch.int32)), ValueError),
        ("tree", dict(parents=torch.zeros(2, 3, dtype=torch.int64)), TypeError),
        ("tree", dict(ctx=torch.zeros(1, dtype=torch.int32)), ValueError),
        ("commit", dict(kv=torch.zeros(1, 2, 4, 3, 16, 64, dtype=BF16)), ValueError),
        ("commit", dict(kv=torch.zeros(1, 2, 4, 2, 16, 64)), TypeError),
        ("commit", dict(kn=torch.zeros(1, 1, 2, 3, 2, 64, dtype=BF16), kv=torch.zeros(1, 1, 4, 2, 16, 64, dtype=BF16)), ValueError),
        ("commit", dict(kn=torch.zeros(1, 2, 2, 3, 2, 12, dtype=BF16), kv=torch.zeros(1, 2, 4, 2, 16, 12, dtype=BF16)), ValueError),
        ("commit", dict(tokens=torch.zeros(2, 3, dtype=torch.int32)), TypeError),
        ("commit", dict(targets=torch.zeros(3, 2, dtype=torch.int64)), ValueError),
        ("prefill", dict(out=torch.zeros(1, 4, 64, dtype=BF16).expand(6, 4, 64)), ValueError),
        ("prefill", dict(slots=torch.zeros(65537, dtype=torch.int32), starts=torch.zeros(65537, dtype=torch.int32),
                         cu=torch.zeros(65538, dtype=torch.int32)), ValueError),
        ("tree", dict(q=torch.zeros(1, 1, 4, 64, dtype=BF16).expand(65537, 1, 4, 64), kn=torch.zeros(1, 1, 2, 64, dtype=BF16).expand(65537, 1, 2, 64),
                      vn=torch.zeros(1, 1, 2, 64, dtype=BF16).expand(65537, 1, 2, 64), slots=torch.zeros(65537, dtype=torch.int32),
                      ctx=torch.zeros(65537, dtype=torch.int32), parents=torch.zeros(65537, 1, dtype=torch.int32)), ValueError),
        ("commit", dict(kn=torch.zeros(1, 2, 1, 1, 2, 64, dtype=BF16).expand(1, 2, 65537, 1, 2, 64), slots=torch.zeros(65537, dtype=torch.int32),
                        ctx=torch.zeros(65537, dtype=torch.int32), parents=torch.zeros(65537, 1, dtype=torch.int32),
                        tokens=torch.zeros(65537, 1, dtype=torch.int64), targets=torch.zeros(65537, 1, dtype=torch.int64)), ValueError),
        ("commit", dict(kv=torch.zeros(1, 2, 1, 2, 16, 64, dtype=BF16).expand(1, 2, 4, 2, 16, 64)), ValueError),
        ("prefill", dict(q=torch.zeros(6, 4, 64, dtype=BF16, requires_grad=True)), RuntimeError),
        ("tree", dict(q=torch.zeros(2, 3, 4, 64, dtype=BF16, requires_grad=True)), RuntimeError),
        ("commit", dict(kn=torch.zeros(1, 2, 2, 3, 2, 64, dtype=BF16, requires_grad=True)), RuntimeError),
        ("sample", dict(logits=torch.zeros(2, 9, requires_grad=True)), RuntimeError),
        ("sample", dict(logits=torch.zeros(2, 9, dtype=torch.float16)), TypeError),
        ("sample", dict(logits=torch.zeros(9)), ValueError),
        ("sample", dict(logits=torch.zeros(2, 0)), ValueError),
        ("sample", dict(logits=torch.zeros(2, (1 << 20) + 1)), ValueError),
        ("sample", dict(logits=torch.zeros(9, 2).t()), ValueError),
        ("sample", dict(u=torch.zeros(3)), ValueError),
        ("sample", dict(u=torch.zeros(2, dtype=torch.float64)), TypeError),
        ("sample", dict(top_k=torch.zeros(2, dtype=torch.int64)), TypeError),
        ("sample", dict(top_p=torch.zeros(1)), ValueError),
        ("sample", dict(min_p=0.1), TypeError),
        ("sample", dict(out=torch.zeros(2, dtype=torch.int32)), TypeError),
    ])
    def test_bad_arguments(self, call, kw, error):
        with pytest.raises(error):
            getattr(self, call)(**kw)


    def test_a_stride_of_one_element_does_not_matter(self):
        """Nothing but the device is wrong with these."""
        one = lambda *shape: torch.zeros(4096, dtype=BF16).as_strided(shape, (0, *torch.zeros(shape[1:]).stride()))  # noqa: E731
        cu = torch.tensor([0, 1], dtype=torch.int32)
        zero = torch.zeros(1, dtype=torch.int32)
        for call in (lambda: self.prefill(q=one(1, 4, 64), out=one(1, 4, 64), slots=zero, starts=zero, cu=cu),
                     lambda: self.commit(kn=torch.zeros(1, 2, 2, 3, 1, 8, dtype=BF16), kv=one(1, 2, 4, 1, 16, 8))):
            with pytest.raises(RuntimeError, match="CUDA/HIP"):
                call()

    @pytest.mark.parametrize("call,name,shape,dtype", [
        ("prefill", "q", (6, 4, 64), BF16), ("prefill", "k", (2, 2, 16, 64), BF16), ("prefill", "v", (2, 2, 16, 64), BF16),
        ("prefill", "out", (6, 4, 64), BF16), ("tree", "q", (2, 3, 4, 64), BF16), ("tree", "kn", (2, 3, 2, 64), BF16),
        ("tree", "vn", (2, 3, 2, 64), BF16), ("tree", "k", (2, 2, 16, 64), BF16), ("tree", "v", (2, 2, 16, 64), BF16),
        ("commit", "kn", (1, 2, 2, 3, 2, 64), BF16), ("commit", "kv", (1, 2, 4, 2, 16, 64), BF16),
        ("sample", "logits", (2, 9), torch.float32), ("sample", "u", (2,), torch.float32),
        ("sample", "temperature", (2,), torch.float32), ("sample", "top_p", (2,), torch.float32), ("sample", "min_p", (2,), torch.float32),
    ])
    def test_gradients_are_refused_for_every_argument(self, call, name, shape, dtype):
        x = torch.ones(shape, dtype=dtype)
        with pytest.raises(RuntimeError, match="gradient"):
            getattr(self, call)(**{name: x.clone().requires_grad_()})
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
            with pytest.raises(RuntimeError, match="tangent"):
                getattr(self, call)(**{name: dual})
        # and neither where there is none
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA/HIP"):
            getattr(self, call)(**{name: x.clone().requires_grad_()})


@pytest.mark.gpu
class TestTogether:
    def test_empty_batches(self):
        e = lambda *s, d=BF16: torch.empty(*s, dtype=d, device=DEV)  # noqa: E731
        k = torch.zeros(2, 2, 16, 64, dtype=BF16, device=DEV)
        none = e(0, d=torch.int32)
        assert ops.attn_prefill(e(0, 4, 64), k, k, none, none, i32([0])).shape == (0, 4, 64)
        assert (ops.attn_prefill(k[0, 0].view(16, 1, 64).expand(16, 2, 64), k, k, none, none, i32([0]),
                                 out=torch.ones(16, 2, 64, dtype=BF16, device=DEV)) == 1).all()
        assert ops.attn_tree(e(0, 3, 4, 64), e(0, 3, 2, 64), e(0, 3, 2, 64), k, k, none, none, e(0, 3, d=torch.int32)).numel() == 0
        got = ops.tree_commit(e(1, 2, 0, 3, 2, 64), k.view(1, 2, 1, 2, 16, 64).clone(), none, none, e(0, 3, d=torch.int32),
                              e(0, 3, d=torch.int64), e(0, 3, d=torch.int64))
        assert [t.numel() for t in got] == [0, 0, 0]
        assert ops.sample(e(0, 5), e(0, d=torch.float32), e(0, d=torch.float32)).numel() == 0

    @pytest.mark.parametrize("fp8", [False, True])
    def test_same_bits_every_time(self, fp8):
        cases = [(ops.attn_prefill, prefill_case(lens, starts, 8, 2, 128, fp8, seed=13))
                 for lens, starts in (([300, 1, 77], [0, 5, 64]), ([3, 40], [6000, 900]))]
        cases += [(ops.attn_tree, tree_case(len(ctx), 33, ctx, 8, 2, 128, fp8, seed=14)) for ctx in ([700] * 40, [9000, 3])]
        for call, args in cases:
            first = call(*args)
            for _ in range(5):
                assert torch.equal(first.view(torch.int16), call(*args).view(torch.int16))

    def test_on_another_stream(self):
        s = torch.cuda.Stream()
        pre, tre = prefill_case([9, 70], [3000, 4], 8, 2, 128, seed=1), tree_case(2, 9, [2500, 7], 8, 2, 128, seed=2)
        want = [ops.attn_prefill(*pre), ops.attn_tree(*tre)]
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            torch.cuda._sleep(2_000_000)
            q2 = pre[0] * 1
            got = [ops.attn_prefill(q2, *pre[1:]), ops.attn_tree(*tre)]
        s.synchronize()
        for a, b in zip(want, got):
            assert torch.equal(a, b)

    def test_draft_verify_commit_decode(self):
        """Prefill, a drafted tree, its targets, the commit, and the next tree over the
        longer context: the same as a prefill of the accepted tokens."""
        g = gen(3)
        H, KVH, D, T, B, N, V = 8, 2, 64, 256, 3, 10, 50
        slots, ctx = i32([4, 0, 2]), i32([33, 70, 1])
        kv = randn(g, 1, 2, 5, KVH, T, D)
        kv_new, parents = randn(g, 1, 2, B, N, KVH, D), trees(g, B, N)
        q = randn(g, B, N, H, D)
        out = ops.attn_tree(q, kv_new[0, 0], kv_new[0, 1], kv[0, 0], kv[0, 1], slots, ctx, parents)
        head = randn(g, H * D, V, scale=0.2)
        logits = out.view(B * N, H * D) @ head
        u, one = torch.rand(B * N, generator=g, device=DEV), torch.ones(B * N, device=DEV)
        targets = ops.sample(logits, u, one, top_k=torch.full((B * N,), 2, dtype=torch.int32, device=DEV)).view(B, N)
        tokens = targets.gather(1, parents.long().clamp_min(0))  # drafts that are right
        count, path, nxt = ops.tree_commit(kv_new, kv, slots, ctx, parents, tokens, targets)
        assert count.min() >= 1 and count.max() > 1
        for b in range(B):
            taken = path[b, :count[b]].long()
            assert nxt[b] == targets[b, taken[-1]]
            # the cache now holds the path: the same attention as a packed prompt chunk
            again = ops.attn_prefill(q[b, taken].contiguous(), kv[0, 0], kv[0, 1], slots[b:b + 1], ctx[b:b + 1], i32([0, len(taken)]))
            # both within the two roundings of the 64-bit value
            assert (again.float() - out[b, taken].float()).abs().max() <= 4 * HALF * out.abs().max().float()


def engine(device=DEV, **kw):
    from smg_amd.engine.torch_engine import TorchEngine, TorchEngineConfig

    cfg = TorchEngineConfig.tiny()
    for k, v in kw.items():
        setattr(cfg, k, v)
    return TorchEngine(cfg, device=device)


def run(eng, *rids):
    for _ in range(300):
        if all(eng.finished(r) for r in rids):
            break
        eng.step()
    return [eng.collect(r) for r in rids]


class TestEngineSampling:
    @pytest.mark.parametrize("device", ["cpu", pytest.param(DEV, marks=pytest.mark.gpu)])
    def test_requests_have_their_own_settings(self, device):
        eng, ref = engine(device), engine(device)
        prompts = [[i * 7 + j for j in range(12)] for i in range(3)]
        want = run(ref, *[ref.submit(p, 6) for p in prompts])
        # a sampled request beside greedy ones; top_k 1 and a tiny top_p leave the likeliest
        a = eng.submit(prompts[0], 6)
        b = eng.submit(prompts[1], 6, temperature=1.5, top_k=1)
        c = eng.submit(prompts[2], 6, temperature=0.7, top_p=1e-6)
        assert run(eng, a, b, c) == want
        # its slot is greedy again afterwards
        assert run(eng, *[eng.submit(p, 6) for p in prompts]) == want

    @pytest.mark.parametrize("device", ["cpu", pytest.param(DEV, marks=pytest.mark.gpu)])
    def test_draws_differ_and_repeat(self, device):
        outs = []
        for _ in range(2):
            eng = engine(device)
            outs.append(run(eng, *[eng.submit(list(range(9)), 8, temperature=2.0) for _ in range(4)]))
        assert outs[0] == outs[1]  # the engine's generator starts from its seed
        assert len({tuple(o) for o in outs[0]}) > 1
        assert all(0 <= t < 2048 for o in outs[0] for t in o)

    def test_refusals(self):
        eng = engine("cpu")
        for kw in (dict(temperature=-1.0), dict(temperature=math.inf), dict(top_p=0.0), dict(top_p=1.5), dict(min_p=-0.1), dict(min_p=2.0), dict(top_k=1 << 31)):
            with pytest.raises(ValueError):
                eng.submit([1, 2], 2, **kw)

    def test_a_temperature_beyond_float32_is_refused_before_anything_is_taken(self):
        eng = engine("cpu")
        most = torch.finfo(torch.float32).max
        for t in (1e39, most * (1 + 2.0 ** -24), 10 ** 300):
            with pytest.raises(ValueError, match="float32"):
                eng.submit([1, 2], 2, temperature=t)
            with pytest.raises(ValueError, match="float32"):
                eng.import_kv("x", torch.zeros(eng.kv_transfer_shape(3)), 3, 1, 4, temperature=t)
        assert not eng.waiting and not eng.running and len(eng._free_slots) == eng.cfg.max_slots
        rids = [eng.submit([1, 2], 3, temperature=t) for t in (most, 1e-46, 0.5)]
        assert all(len(out) == 3 for out in run(eng, *rids))
        # what the slots hold on the device is what the host takes them to hold
        for slot, s in enumerate(eng._sampling_host):
            assert [t[slot].item() for t in eng._sampling] == torch.tensor(s, dtype=torch.float32).tolist()

    def test_settings_follow_the_kv(self):
        a, b = engine("cpu"), engine("cpu")
        rid = a.submit(list(range(30)), 8, prefill_only=True, temperature=2.0)
        a.step()
        kv, plen, first = a.export_kv(rid)
        with pytest.raises(ValueError):
            b.import_kv(rid, kv, plen, first, 8, temperature=-1.0)
        assert b.import_kv(rid, kv, plen, first, 8, temperature=1.5, top_k=1)
        c = engine("cpu")
        assert c.import_kv(rid, kv, plen, first, 8)
        assert run(b, rid) == run(c, rid)

    def test_kernels_are_asked_for_on_cpu(self):
        with pytest.raises(RuntimeError, match="packed_prefill"):
            engine("cpu", packed_prefill=True)
        eng = engine("cpu")
        with pytest.raises(RuntimeError, match="step_drafts"):
            eng.step_drafts({})


    def test_a_core_without_the_kernels_is_found_out_before_a_step(self, monkeypatch):
        eng = engine("cpu")
        eng._hip_fused = eng._hip_rope_prefill = object()  # as a core from older sources has them
        assert eng._has_ops()
        monkeypatch.setattr(ops, "BUILT", False)
        assert not eng._has_ops()
        with pytest.raises(RuntimeError, match="step_drafts"):
            eng.step_drafts({})
        eng.device = torch.device(DEV)
        kv = torch.zeros(eng.kv_transfer_shape(3))
        for call in (lambda **kw: eng.submit([1, 2], 2, **kw), lambda **kw: eng.import_kv("x", kv, 3, 1, 4, **kw)):
            with pytest.raises(RuntimeError, match="csrc.build"):
                call(temperature=0.5)
        assert not eng.waiting and len(eng._free_slots) == eng.cfg.max_slots
        eng.submit([1, 2], 2)  # greedy ones do without

    def test_kernels_are_looked_for_by_name(self, monkeypatch):
        import importlib

        from smg_amd import _core

        try:
            assert ops.BUILT
            monkeypatch.delattr(_core, "tree_commit")
            assert not importlib.reload(ops).BUILT
        finally:
            monkeypatch.undo()
            assert importlib.reload(ops).BUILT


def kv_rows(eng, slot, n):
    return eng.kv[:, :, slot, :, :n].float()


@pytest.mark.parametrize("mult", [0.0, 1e-3, 0.4, 1.0, 2.5])
def test_packed_groups_follow_the_budget(monkeypatch, mult):
    """A forward takes the budget's tokens, and a chunk where that is less: all prompts end."""
    eng = engine("cpu", prefill_chunk=16, prefill_budget_mult=mult, prefix_cache_slots=0)
    eng.cfg.packed_prefill = True  # with the batched forward in the kernels' place
    taken = []

    def packed(items):
        taken.append([len(toks) for _, _, toks in items])
        return torch.cat([eng._prefill_batch([item]) for item in items])

    monkeypatch.setattr(eng, "_prefill_packed", packed)
    prompts = [list(range(n)) for n in (3, 40, 16, 17, 1)]
    got = run(eng, *[eng.submit(p, 3) for p in prompts])
    ref = engine("cpu", prefix_cache_slots=0)
    assert got == run(ref, *[ref.submit(p, 3) for p in prompts])
    assert all(0 < sum(lens) <= max(16, 16 * mult) and max(lens) <= 16 for lens in taken)


@pytest.mark.gpu
class TestEnginePaths:
    @pytest.mark.parametrize("kw", [{}, dict(n_kv_heads=2), dict(n_kv_heads=2, kv_fp8=True), dict(prefill_chunk=24, prefill_budget_mult=1.0)])
    def test_packed_prefill_fills_the_cache_as_the_batched_one(self, kw):
        base = dict(kw)
        base.pop("prefill_chunk", None), base.pop("prefill_budget_mult", None)
        g = torch.Generator().manual_seed(0)
        prompts = [torch.randint(0, 2048, (n,), generator=g).tolist() for n in (5, 130, 1, 64, 97)]
        prompts.append(prompts[1][:64] + [7, 8, 9])  # a prefix-cache hit once prompt 1 is stored
        packed, plain = engine(packed_prefill=True, **kw), engine(**base)
        for eng in (packed, plain):
            for p in prompts[:5]:
                eng.submit(p, 90, rid=str(len(p)))
            for _ in range(30):
                eng.step()
            eng.submit(prompts[5], 90, rid="hit")
            for _ in range(20):
                eng.step()
            assert eng.prefix_cache_hits >= 1
        slots = [{r.rid: s for s, r in eng.running.items()} for eng in (packed, plain)]
        for p in prompts:
            rid = "hit" if p is prompts[5] else str(len(p))
            a, b = (kv_rows(eng, sl[rid], len(p)) for eng, sl in zip((packed, plain), slots))
            # the layers' inputs differ by roundings of the layer before: bf16 steps (8-bit
            # ones of the cached K/V) of values up to a few units
            assert (a - b).abs().max() <= (0.3 if kw.get("kv_fp8") else 0.06) * max(1.0, b.abs().max().item())
            first = [eng._requests[rid].generated[0] for eng in (packed, plain)]
            assert all(0 <= t < 2048 for t in first)

    @pytest.mark.parametrize("kw", [{}, dict(n_kv_heads=1), dict(n_kv_heads=2, kv_fp8=True)])
    def test_drafts_are_verified_and_committed(self, kw):
        eng = engine(**kw)
        prompts = [list(range(3, 40)), list(range(100, 105))]
        rids = [eng.submit(p, 40) for p in prompts]
        while any(r.prefilled < len(r.tokens) for r in eng.waiting + list(eng.running.values())):
            eng.step()
        before = {r: list(eng._requests[r].generated) for r in rids}
        # what the model chooses after each node comes back; drafted again, it is accepted
        got = eng.step_drafts({r: ([], []) for r in rids})
        assert all(len(v) == 1 for v in got.values())
        for _ in range(4):
            probe = {}
            for r in rids:
                # wrong guesses beside each other, and a chain below one of them
                probe[r] = ([1, 2, 3, 4], [-1, -1, 1, 2])
            more = eng.step_drafts(probe)
            for r in rids:
                got[r] += more[r]
        events = {}
        for r, t, _ in eng.drain_events():
            events.setdefault(r, []).append(t)
        for r in rids:
            req = eng._requests[r]
            assert req.generated == before[r] + got[r] and events[r][-len(got[r]):] == got[r]
            # the cache holds the tokens but the last, as a prefill of them does
            tokens = prompts[rids.index(r)] + req.generated[:-1]
            slot = req.slot
            assert eng._seq_len_host[slot] == len(tokens) == eng.seq_len[slot].item()
            ref = engine(**kw)
            rr = ref.submit(tokens, 2)
            ref.step()
            a, b = kv_rows(eng, slot, len(tokens)), kv_rows(ref, ref._requests[rr].slot, len(tokens))
            assert (a - b).abs().max() <= (0.3 if kw.get("kv_fp8") else 0.06) * max(1.0, b.abs().max().item())

    def test_right_drafts_are_accepted(self):
        engs = [engine(), engine()]
        rids = [e.submit(list(range(50)), 30) for e in engs]
        for e, rid in zip(engs, rids):
            while not e._requests[rid].generated:
                e.step()
        # the first engine's choice is drafted, twice, in the second one
        nxt = engs[0].step_drafts({rids[0]: ([], [])})[rids[0]][0]
        eng, rid = engs[1], rids[1]
        slot = eng._requests[rid].slot
        n = int(eng._seq_len_host[slot])
        got = eng.step_drafts({rid: ([(nxt + 1) % 2048, nxt, nxt, 5], [-1, -1, -1, 1])})[rid]
        assert got[0] == nxt and len(got) >= 2
        assert eng.seq_len[slot].item() == n + len(got) == eng._seq_len_host[slot]
        assert eng._last_tok[slot].item() == got[-1]

    def test_drafts_end_with_the_request(self):
        eng = engine()
        rid = eng.submit(list(range(20)), 3)
        while not eng._requests[rid].generated:
            eng.step()
        for _ in range(3):
            if eng.finished(rid):
                break
            eng.step_drafts({rid: ([1, 2], [-1, 0])})
        assert eng.finished(rid) and len(eng.collect(rid)) == 3
        assert len(eng._free_slots) == eng.cfg.max_slots
        flags = [d for r, _, d in eng.drain_events() if r == rid]
        assert flags[-1] == 1 and not any(flags[:-1])

    def test_drafts_at_the_end_of_the_cache(self):
        eng = engine(max_seq=64)
        rid = eng.submit(list(range(55)), 100)
        while not eng._requests[rid].generated:
            eng.step()
        while not eng.finished(rid):
            eng.step_drafts({rid: (list(range(20)), [i - 1 for i in range(20)])})
        assert len(eng._free_slots) == eng.cfg.max_slots

    def test_draft_refusals(self):
        eng = engine()
        rid = eng.submit(list(range(20)), 9)
        with pytest.raises(KeyError):
            eng.step_drafts({rid: ([], [])})  # not prefilled yet
        while not eng._requests[rid].generated:
            eng.step()
        for tokens, parents in (([1], []), ([1], [0]), ([1, 2], [-1, 1]), ([1], [-2]), ([1] * 64, [-1] * 64)):
            with pytest.raises(ValueError):
                eng.step_drafts({rid: (tokens, parents)})
        assert eng.step_drafts({}) == {}
        handle = eng.step_launch()
        with pytest.raises(RuntimeError, match="finished"):
            eng.step_drafts({rid: ([], [])})
        eng.step_finish(handle)
        assert eng.step_drafts({rid: ([], [])})[rid]

    def test_sampled_drafts(self):
        eng = engine(n_kv_heads=2)
        rids = [eng.submit(list(range(9 * i, 9 * i + 9)), 20, temperature=t, top_p=0.9) for i, t in enumerate((0.0, 1.0, 0.5))]
        while any(not eng._requests[r].generated for r in rids):
            eng.step()
        for _ in range(5):
            got = eng.step_drafts({r: ([3, 4], [-1, -1]) for r in rids})
            eng.step()  # and decoding goes on in between
            assert all(got.values())


class TestStaging:
    def test_a_buffer_is_not_written_before_its_copy_ran(self, monkeypatch):
        """The ring of transfers on the CPU, with copies that run only when they are waited for."""
        stream, ran = [], []  # sources of the copies that have not run, values of those that have

        def run(n):
            ran.extend(src.tolist() for src in stream[:n])
            del stream[:n]

        class Event:
            def record(self, at):
                assert at == ("stream of", torch.device(DEV))  # the copy's, whatever device is current
                self.place = len(ran) + len(stream)

            def synchronize(self):
                run(max(0, self.place - len(ran)))

        class Device(torch.Tensor):
            def copy_(self, src, non_blocking=False):
                stream.append(src)
                return self

        empty = torch.empty

        def cpu_empty(*a, pin_memory=False, device=None, **kw):
            t = empty(*a, **kw)
            return t if device is None else t.as_subclass(Device)

        eng = engine("cpu")
        eng.device = torch.device(DEV)
        monkeypatch.setattr(torch, "empty", cpu_empty)
        monkeypatch.setattr(torch.cuda, "Event", Event)
        monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: ("stream of", device))
        sent = [[i] * (1 + i % 5) for i in range(3 * len(eng._h2d_bufs))]
        for values in sent:
            eng._h2d_i64(values)
        assert stream  # the host ran ahead
        run(len(stream))
        assert ran == sent

    @pytest.mark.gpu
    @pytest.mark.parametrize("packed", [False, True])
    def test_a_long_burst_behind_a_busy_stream(self, packed):
        outs = []
        for busy in (False, True):
            eng = engine(packed_prefill=packed, max_slots=8)
            rids = [eng.submit([(i * 37 + j) % 2048 for j in range(20 + i)], 40 + i) for i in range(6)]
            for _ in range(8):
                if busy:
                    torch.cuda._sleep(20_000_000)  # some milliseconds: the host is far ahead
                eng.step(decode_burst=16)
            assert all(eng.finished(r) for r in rids)
            outs.append([eng.collect(r) for r in rids])
        assert outs[0] == outs[1]


SD = 12 * HALF * math.sqrt(1 / 3)
"""How far a logit of the tiny engine may be off between two ways to compute it, as a
standard deviation.  Two layers of six roundings to bf16 each, were all of them half a step
in one direction, leave the last state off by 12 HALF of its length, sqrt(d).  A logit is
its product with a row of the embedding, whose direction has nothing to do with it and whose
length is sqrt(1/3): uniform numbers of up to 1/sqrt(d) in size.  8-bit K/V add half a step
of theirs, 2^-4 of what attention adds, in both layers."""
SD_FP8 = SD + 2 * 2.0 ** -4 * math.sqrt(1 / 3)


def watch(eng):
    """The logits of every choice that the engine makes from now on."""
    seen, choose = [], eng._choose

    def keep(logits, *a, **kw):
        seen.append(logits.float())
        return choose(logits, *a, **kw)

    eng._choose = keep
    return seen


def lead(logits):
    """By how much the likeliest token leads."""
    two = logits.topk(2, dim=-1).values
    return two[..., 0] - two[..., 1]


@pytest.mark.gpu
class TestEngineAnswers:
    """What the engine's ways through the operators answer, against its other ways."""

    @pytest.mark.parametrize("kw", [{}, dict(n_kv_heads=1), dict(n_kv_heads=2, kv_fp8=True)])
    def test_packed_prefill_answers_as_the_batched_one(self, kw):
        sd = SD_FP8 if kw.get("kv_fp8") else SD
        g = torch.Generator().manual_seed(1)
        prompts = [torch.randint(0, 2048, (n,), generator=g).tolist() for n in (5, 130, 1, 64, 97, 33, 200)]
        # 530 tokens, in one forward (4 chunks of 256)
        plain, packed = engine(prefix_cache_slots=0, **kw), engine(prefix_cache_slots=0, packed_prefill=True, prefill_budget_mult=4.0, **kw)
        want, got = [], watch(packed)
        for p in prompts:
            seen = watch(plain)
            plain.submit(p, 1)
            plain.step()
            want.append(seen[0][0])
        state, prefill = [], packed._prefill_packed

        def kept(items):
            nxt = prefill(items)
            state.append((items, nxt.tolist(), packed._last_tok.tolist(), packed.seq_len.tolist()))
            return nxt

        packed._prefill_packed = kept
        rids = [packed.submit(p, 9) for p in prompts]
        packed.step()
        (items, nxt, last, lens), = state
        assert len(items) == len(prompts)
        by_slot = {packed._requests[r].slot: i for i, r in enumerate(rids)}
        for row, ((slot, start, _), token) in enumerate(zip(items, nxt)):
            i = by_slot[slot]
            # 2048 logits of a few prompts stay below 6 deviations, and are rounded to bf16 twice
            assert (got[0][row] - want[i]).abs().max() <= 6 * sd + 2 * HALF * want[i].abs().max()
            assert token == got[0][row].argmax().item() == last[slot] == packed._requests[rids[i]].generated[0]
            assert start == 0 and lens[slot] == len(prompts[i])

    @pytest.mark.parametrize("kw", [{}, dict(n_kv_heads=2), dict(n_kv_heads=2, kv_fp8=True)])
    def test_drafted_steps_choose_as_decoding_does(self, kw):
        sd = SD_FP8 if kw.get("kv_fp8") else SD
        decoded, drafted = engine(max_slots=32, vocab_size=32, **kw), engine(max_slots=32, vocab_size=32, **kw)
        g = torch.Generator().manual_seed(2)
        prompts = [torch.randint(0, 32, (11 + i,), generator=g).tolist() for i in range(24)]
        rids = [[e.submit(p, 60) for p in prompts] for e in (decoded, drafted)]
        for e, rr in zip((decoded, drafted), rids):
            while any(not e._requests[r].generated for r in rr):
                e.step()
        # both chose their first tokens, and the ones of the steps so far, in the same way
        assert all(decoded._requests[a].generated == drafted._requests[b].generated for a, b in zip(*rids))
        seen, compared, clear = watch(decoded), 0, dict.fromkeys(range(len(prompts)), True)
        for _ in range(10):
            decoded.step()
            got = drafted.step_drafts({r: ([1], [-1]) for r in rids[1]})
            logits = seen[-1]
            for i, ok in clear.items():
                req = decoded._requests[rids[0][i]]
                # one that leads by less may lose: the requests' texts part from there on
                clear[i] = ok = ok and lead(logits[req.slot]).item() > 4 * math.sqrt(2) * sd and len(got[rids[1][i]]) == 1
                if ok:
                    assert got[rids[1][i]][0] == req.generated[-1]
                    compared += 1
        assert compared >= (8 if kw.get("kv_fp8") else 20)

    @pytest.mark.parametrize("settings", [{}, dict(temperature=1.5, top_k=1)])
    @pytest.mark.parametrize("kw", [{}, dict(n_kv_heads=2), dict(n_kv_heads=2, kv_fp8=True)])
    def test_a_chain_of_right_drafts_lies_in_the_cache_as_its_prefill(self, kw, settings):
        one, eng = engine(max_slots=64, vocab_size=32, **kw), engine(max_slots=64, vocab_size=32, **kw)
        g = torch.Generator().manual_seed(3)
        prompts = [torch.randint(0, 32, (20 + i % 9,), generator=g).tolist() for i in range(60)]
        # every fourth request of the second engine draws at random between the others
        heat = [dict(temperature=5.0) if i % 4 == 3 else settings for i in range(60)]
        a = [one.submit(p, 60) for p in prompts]
        b = [eng.submit(p, 60, **s) for p, s in zip(prompts, heat)]
        for e, rr in ((one, a), (eng, b)):
            while any(not e._requests[r].generated for r in rr):
                e.step()
        # the model's own texts, a token a call
        seen, texts, leads = watch(one), [[] for _ in a], []
        for _ in range(4):
            got = one.step_drafts({r: ([], []) for r in a})
            leads.append(lead(seen[-1]))
            for text, r in zip(texts, a):
                text += got[r]
        least = torch.stack(leads).amin(0).tolist()
        # drafts in 16 bits where the first engine read them in 8: 3 keys of 20 or more
        sd = SD + (2 * 2.0 ** -4 * math.sqrt(1 / 3) * 3 / 20 if kw.get("kv_fp8") else 0)
        sure = [i for i in range(60) if i % 4 != 3 and least[i] > 4 * math.sqrt(2) * sd
                and one._requests[a[i]].generated[:-4] == eng._requests[b[i]].generated]
        assert len(sure) >= 2
        before = {i: list(eng._requests[b[i]].generated) for i in sure}
        # right ones behind wrong ones beside them, and wrong ones below
        drafts = {}
        for i, r in enumerate(b):
            c1, c2, c3, _ = texts[i]
            drafts[r] = ([(c1 + 1) % 32, c1, (c2 + 1) % 32, c2, c1, (c3 + 3) % 32, c3], [-1, -1, 1, 1, 0, 3, 3])
        got = eng.step_drafts(drafts)
        for i in sure:
            req, rid = eng._requests[b[i]], b[i]
            assert got[rid] == texts[i] and req.generated == before[i] + texts[i]
            tokens = prompts[i] + req.generated[:-1]
            assert eng.seq_len[req.slot].item() == eng._seq_len_host[req.slot] == len(tokens)
            assert eng._last_tok[req.slot].item() == texts[i][-1]
            ref = engine(vocab_size=32, **kw)
            rr = ref.submit(tokens, 2)
            ref.step()
            x, y = kv_rows(eng, req.slot, len(tokens)), kv_rows(ref, ref._requests[rr].slot, len(tokens))
            # a K that is rotated by one position too few is off by about its own size
            assert (x - y).abs().max() <= (0.3 if kw.get("kv_fp8") else 0.06) * max(1.0, y.abs().max().item())
            if not kw.get("kv_fp8"):
                # row by row, what layers of 12 roundings leave
                assert ((x - y).norm(dim=-1) <= 12 * HALF * y.norm(dim=-1)).all()


@pytest.mark.gpu
def test_a_sampled_request_between_captured_forwards():
    """Captured forwards end in an argmax: a sampled request takes the others out of them and
    back, and changes none of their tokens."""
    from smg_amd.engine.torch_engine import TorchEngine

    outs = []
    for graphs in (False, True):
        eng = TorchEngine(engine("cpu").cfg, device=DEV, graphs=graphs)
        texts = []
        for wave in range(5):  # equal groups, so that prefill is captured too
            greedy = [eng.submit([(wave * 50 + i * 9 + j) % 2048 for j in range(40)], 12) for i in range(4)]
            if wave in (1, 3, 4):
                sampled = eng.submit(list(range(7)), 5, temperature=1.0, top_p=0.9)
            texts += run(eng, *greedy)
        assert eng.finished(sampled)
        assert bool(eng._graph_cache) == graphs
        outs.append(texts)
    assert outs[0] == outs[1]
